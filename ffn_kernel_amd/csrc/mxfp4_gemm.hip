// Routed GEMMs over MXFP4 operands: C[rows, N] = A[rows, K] B_g[N, K]^T, and the SwiGLU pair of them with the intermediate
// quantised in the epilogue.  The rows' codes lie as bf16 rows of a quarter of the length do - 16 bytes are 32 columns of one row -
// so the LDS panels are the bf16 GEMMs': 128-byte rows (256 columns), filled in lane order by direct global->LDS loads, XOR-swizzled
// (lds_swizzle).  A stage's scales (8 bytes a row) come two stages at a time, 16 bytes a row, and a lane reads the four it needs with
// one 32-bit read: lane half `lh` takes blocks 4 lh ... 4 lh + 3 of the stage.
#include "gemm_nt.hpp"
#include "mxfp4.hpp"

namespace ffnk {

namespace {

constexpr int kMxStageK = 256;  // columns of a stage

template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, bool DUAL_, int GROUP_M_>
struct MxTile {
  static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, GROUP_M = GROUP_M_;
  static constexpr bool DUAL = DUAL_, B_KMAJOR = false, SWAP = false;
  static constexpr int NWAVES = WAVES_M * WAVES_N, NT = NWAVES * kWave;
  static constexpr int BN_OUT = DUAL ? BN / 2 : BN, WTM = BM / WAVES_M, WTN_OUT = BN_OUT / WAVES_N;
  static constexpr int MT = 32, ACC_N = 16;
  static constexpr int TM = WTM / MT, TN_OUT = WTN_OUT / MT, TN = DUAL ? 2 * TN_OUT : TN_OUT;
  static constexpr int A_BYTES = BM * kRowBytes, STAGE_BYTES = (BM + BN) * kRowBytes;
  static constexpr int SCALE_BYTES = (BM + BN) * 16;  // of two stages
  static constexpr int LDS_BYTES = 2 * STAGE_BYTES + 2 * SCALE_BYTES;
  using Acc = f32x16_t;
  static_assert(LDS_BYTES <= 160 * 1024 && BM % 64 == 0 && (DUAL ? BN / 2 : BN) % 64 == 0 && WTN_OUT % 32 == 0 && WTM % 32 == 0, "tile");
  static_assert((BM / 8) % NWAVES == 0 && (BN / 16) % NWAVES == 0, "panel rows spread evenly over the waves, gate and up rows apart");
};

__device__ __forceinline__ const uint8_t* wave_uniform(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>(((uint64_t)hi << 32) | lo);
#else
  return p;
#endif
}

// The contraction over stages [kt0, kt1) of the tile's rows; kt0 is even.
template <class Cfg>
__device__ __forceinline__ void mx_mainloop(const MxGemmArgs& g, const TileCoord& tc, const TileLanes<Cfg>& tl, int kt0, int kt1, uint8_t* lds,
                                            f32x16_t (&acc)[Cfg::TM][Cfg::TN]) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = Cfg::NWAVES, TM = Cfg::TM, TN = Cfg::TN, BM = Cfg::BM, BN = Cfg::BN;
  constexpr int NJA = TileLanes<Cfg>::NJA, NJB = TileLanes<Cfg>::NJB;
  constexpr int NG = (BM + BN) / 64, NS = cdiv(NG, NW);  // scale loads: 64 rows each
  const int wave = tl.wave_s;
  const int nb = cdiv(g.K, kMxBlock);
  const int64_t lda = (int64_t)nb * 16, lds_row = round_up64(nb, 16);

  // Code rows.  Gathered ones are addressed from the start of A (the host checks that 32 bits reach them).
  const int64_t row0 = g.gather ? 0 : tc.row0;
  const int n_first = min(tc.n0, g.N - 1);
  auto a_row = [&](int r) {  // rows past the group's end repeat its last one; their results are not stored
    const int p = min(tc.row0 + r, tc.row_end - 1);
    return g.gather ? g.perm[p] : p - tc.row0;
  };
  auto b_row = [&](int r) { return min(tc.n0 + r, g.N - 1) - n_first; };
  __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.A.codes + row0 * lda), 0, 0xffffffff, 0x00020000);
  __amdgpu_buffer_rsrc_t rsB[2];
  rsB[0] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.B0[tc.grp].codes + n_first * lda), 0, 0xffffffff, 0x00020000);
  if (Cfg::DUAL) rsB[1] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.B1[tc.grp].codes + n_first * lda), 0, 0xffffffff, 0x00020000);
  uint32_t off_a[NJA], off_b[NJB];
#pragma unroll
  for (int j = 0; j < NJA; ++j) off_a[j] = (uint32_t)a_row(tl.load_row(j)) * (uint32_t)lda + tl.c_log * 16;
#pragma unroll
  for (int j = 0; j < NJB; ++j) {
    const int r = tl.load_row(j) - (Cfg::DUAL && j >= NJB / 2 ? BN / 2 : 0);
    off_b[j] = (uint32_t)b_row(r) * (uint32_t)lda + tl.c_log * 16;
  }
  // The last stage of a contraction that is no whole number of them: pieces past a row's end repeat its last one, and count with
  // the scale bytes behind the last block, which are 0.
  const int nk = cdiv(nb, 8), rest = nb - (nk - 1) * 8;
  const uint32_t last_back = (int)tl.c_log >= rest ? (uint32_t)((rest - 1 - (int)tl.c_log) * 16) : 0u;

  // Scale rows: group q of 64, the token rows' first.
  const uint8_t* scale_base[NS];
  uint32_t off_s[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int q = s * NW + wave;  // (uniform)
    if (q < BM / 64) {
      scale_base[s] = g.A.scales + row0 * lds_row;
      off_s[s] = (uint32_t)a_row(q * 64 + tl.lane) * (uint32_t)lds_row;
    } else {
      const int r = q * 64 - BM;
      const bool up = Cfg::DUAL && r >= BN / 2;
      scale_base[s] = (up ? g.B1[tc.grp].scales : g.B0[tc.grp].scales) + n_first * lds_row;
      off_s[s] = (uint32_t)b_row(r - (up ? BN / 2 : 0) + tl.lane) * (uint32_t)lds_row;
    }
    scale_base[s] = wave_uniform(scale_base[s]);
  }

  // Load l of stage kt (of parity u): weight rows, token rows, then - with the first of two stages - their scales.
  constexpr int LOADS = NJA + NJB;
  auto load = [&](int l, int u, int kt) {
    uint8_t* stage = lds + u * Cfg::STAGE_BYTES;
    if (l < LOADS) {
      const uint32_t back = kt == nk - 1 ? last_back : 0u;
      const int j = l < NJB ? l : l - NJB;
      if (l < NJB)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB[Cfg::DUAL && j >= NJB / 2], FFNK_LDS_PTR(stage + Cfg::A_BYTES + (j * NW + wave) * 1024), 16,
                                                 off_b[j] + back, kt * kRowBytes, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, FFNK_LDS_PTR(stage + (j * NW + wave) * 1024), 16, off_a[j] + back, kt * kRowBytes, 0, 0);
    } else {
      const int s = l - LOADS, q = s * NW + wave;
      if (NG % NW == 0 || q < NG)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(scale_base[s]), 0, 0xffffffff, 0x00020000),
            FFNK_LDS_PTR(lds + 2 * Cfg::STAGE_BYTES + ((kt >> 1) & 1) * Cfg::SCALE_BYTES + q * 1024), 16, off_s[s], (kt >> 1) * 16, 0, 0);
    }
  };

  uint32_t koff[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) koff[s] = lds_swizzle(tl.lr, 4 * tl.lh + s);
  const uint32_t a_base = (uint32_t)(tl.wm * Cfg::WTM) * kRowBytes;
  i32x4_t fa[2][TM], fb[2][TN];
  int sa[2][TM], sb[2][TN];
  // Fragment f of step s of a stage of parity u: token rows, then weight rows; their scales.
  auto read = [&](int f, int u, int s) {
    const uint8_t* stage = lds + u * Cfg::STAGE_BYTES;
    if (f < TN) fb[s & 1][f] = *reinterpret_cast<const i32x4_t*>(stage + Cfg::A_BYTES + b_frag_row<Cfg>(tl.wn, f) * kRowBytes + koff[s]);
    else fa[s & 1][f - TN] = *reinterpret_cast<const i32x4_t*>(stage + a_base + (f - TN) * 32 * kRowBytes + koff[s]);
  };
  auto read_scale = [&](int f, int u, int kt) {
    const uint8_t* scales = lds + 2 * Cfg::STAGE_BYTES + ((kt >> 1) & 1) * Cfg::SCALE_BYTES + 8 * u + 4 * tl.lh;
    if (f < TN) sb[u][f] = *reinterpret_cast<const int*>(scales + (BM + b_frag_row<Cfg>(tl.wn, f) + tl.lr) * 16);
    else sa[u][f - TN] = *reinterpret_cast<const int*>(scales + (tl.wm * Cfg::WTM + (f - TN) * 32 + tl.lr) * 16);
  };

  // A stage is four steps of 64 columns, TM x TN matrix instructions each.  Behind them, spread over the step, the next step's
  // fragments are read (the last step's early, the next stage's first ones behind the data barrier).  Two barriers a stage:
  //   RELEASE: every wave has read the last of this stage - the loads of the stage after next go into its memory from here on
  //   DATA: the next stage has landed
  // which leaves the loads 1.2 to 1.5 stages to land.
  constexpr int NM = TM * TN, NF = TM + TN, LEV = NM >= 16 ? 2 : 1;
  constexpr int RELEASE = 3 * NM - (NM >= 16 ? 4 : 1), DATA = 3 * NM + (NM >= 16 ? 6 : 1), TURN = 4 * NM;
  constexpr int FIRST = (TURN - RELEASE) / LEV, BEFORE = (DATA - RELEASE) / LEV;  // loads behind RELEASE in this stage, and of these ahead of DATA
  static_assert(FIRST <= LOADS && LOADS + NS - FIRST <= RELEASE / LEV, "the loads of a stage go out between its two RELEASE barriers");
  static_assert(NG % NW == 0, "every wave issues as many loads, which it counts");
  auto stage = [&](auto parity, int kt, auto next_, auto next2_) {
    constexpr int u = decltype(parity)::value;
    const bool next = next_, next2 = next2_;         // stages kt + 1 and kt + 2 are there
    constexpr int ALL1 = LOADS + (u == 1 ? NS : 0);  // loads of stage kt + 1 (of the other parity)
    static_for<0, 4>([&](auto step) {
      constexpr int s = decltype(step)::value;
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const int t = s * NM + m;
        if (t == RELEASE && next2) dma_wait_barrier<63>();
        if (t == DATA && next) {
          if (next2) dma_wait_barrier<BEFORE>();
          else dma_wait_barrier<0>();
        }
        __builtin_amdgcn_sched_barrier(0);
        const int i = m / TN, j = m % TN;
        acc[i][j] = mx_mfma32<s>(fb[s & 1][j], fa[s & 1][i], acc[i][j], sb[u][j], sa[u][i]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          if (s < 3 ? f * (s == 2 ? NM / 2 : NM) / NF == m : DATA + f * (TURN - DATA) / NF == t && next) {
            if (s < 3) {
              read(f, u, s + 1);
            } else {
              read_scale(f, u ^ 1, kt + 1);
              read(f, u ^ 1, 0);
            }
          }
        }
        if (t >= RELEASE) {
          if ((t - RELEASE) % LEV == LEV - 1 && next2) load((t - RELEASE) / LEV, u, kt + 2);
        } else if (t % LEV == LEV - 1 && FIRST + t / LEV < ALL1 && next) {
          load(FIRST + t / LEV, u ^ 1, kt + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  };

  zero_acc<Cfg>(acc);
#pragma unroll
  for (int l = 0; l < LOADS + NS; ++l) load(l, 0, kt0);
  if (kt0 + 1 < kt1) {
#pragma unroll
    for (int l = 0; l < FIRST; ++l) load(l, 1, kt0 + 1);
    dma_wait_barrier<FIRST>();
  } else {
    dma_wait_barrier<0>();
  }
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    read_scale(f, 0, kt0);
    read(f, 0, 0);
  }
  constexpr auto even = std::integral_constant<int, 0>{};
  constexpr auto odd = std::integral_constant<int, 1>{};
  constexpr auto yes = std::true_type{};
  int kt = kt0;
  for (; kt + 3 < kt1; kt += 2) {  // no branches inside
    stage(even, kt, yes, yes);
    stage(odd, kt + 1, yes, yes);
  }
  for (; kt < kt1; kt += 2) {
    stage(even, kt, kt + 1 < kt1, kt + 2 < kt1);
    if (kt + 1 < kt1) stage(odd, kt + 1, kt + 2 < kt1, kt + 3 < kt1);
  }
#endif
}

// Results of the wave's tile in bf16 to rows of `base`, through LDS: 16 bytes at a time where rows allow it.
template <class Cfg, bool SCATTER, class Value>
__device__ __forceinline__ void mx_store(const MxGemmArgs& g, uint16_t* base, int64_t ld, const TileCoord& tc, const TileLanes<Cfg>& tl, uint8_t* lds,
                                         Value&& value) {
  using W = WaveRows<Cfg>;
  const int p0 = tc.row0 + tl.wm * Cfg::WTM, n = tc.n0 + tl.wn * Cfg::WTN_OUT + W::col(tl.lane);
  int rows[W::ROW_REGS];
#pragma unroll
  for (int q = 0; q < W::ROW_REGS; ++q) {
    const int p = p0 + q * kWave + tl.lane;
    rows[q] = p < tc.row_end && q * kWave + tl.lane < W::ROWS ? (SCATTER ? g.perm[p] : p) : -1;
  }
  W::put(lds, tl.wave, tl.lr, tl.lh, [&](int i, int j, int q4) {
    return make_uint2(pack2bf(value(i, j, 4 * q4), value(i, j, 4 * q4 + 1)), pack2bf(value(i, j, 4 * q4 + 2), value(i, j, 4 * q4 + 3)));
  });
  const bool whole = g.N % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;  // uniform over the launch
#pragma unroll
  for (int k = 0; k < W::N; ++k) {
    const uint4 v = W::get(lds, tl.wave, tl.lane, k);
    const int row = __shfl(rows[k * W::PER / kWave], k * W::PER % kWave + tl.lane / W::CH);
    if (row < 0 || n >= g.N) continue;
    uint16_t* out = base + row * ld + n;
    if (whole) {
      *reinterpret_cast<uint4*>(out) = v;
    } else {
      const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll 1
      for (int e = 0; e < 8 && n + e < g.N; ++e) out[e] = (uint16_t)((e < 2 ? words[0] : e < 4 ? words[1] : e < 6 ? words[2] : words[3]) >> (16 * (e & 1)));
    }
  }
}

// H = Q(silu(gate) up) for the wave's tile.  An accumulator tile's 32 weight rows are one block of the intermediate: a lane holds 16 of
// a token's 32 values, the lane 32 further the other 16.
template <class Cfg>
__device__ __forceinline__ void mx_swiglu_store(const MxGemmArgs& g, const TileCoord& tc, const TileLanes<Cfg>& tl, f32x16_t (&acc)[Cfg::TM][Cfg::TN]) {
  const int nb = cdiv(g.N, kMxBlock);
  const int64_t ldh = (int64_t)nb * 16, ldsh = round_up64(nb, 16);
#pragma unroll
  for (int i = 0; i < Cfg::TM; ++i) {
    const int p = tc.row0 + tl.wm * Cfg::WTM + i * 32 + (int)tl.lr;
#pragma unroll
    for (int j = 0; j < Cfg::TN_OUT; ++j) {
      const int b = (tc.n0 + tl.wn * Cfg::WTN_OUT) / 32 + j;
      float h[16];
      uint32_t top = 0;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        h[v] = swiglu(acc[i][j][v], acc[i][j + Cfg::TN_OUT][v]);
        if (b * 32 + acc_col<Cfg>(v, (int)tl.lh) >= g.N) h[v] = 0.f;  // columns past the last one
        const uint32_t bits = __builtin_bit_cast(uint32_t, h[v]) & 0x7fffffffu;
        top = bits > top ? bits : top;
      }
      const uint32_t other = (uint32_t)__shfl_xor((int)top, 32);
      const uint32_t byte = mx_scale_byte(other > top ? other : top);
      const float inv = mx_inverse(byte);
      uint32_t c[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) c[q] = mx_codes4(h[4 * q] * inv, h[4 * q + 1] * inv, h[4 * q + 2] * inv, h[4 * q + 3] * inv);
      // run q of either half is 16 bits of dword q: half 0 stores dwords 0 and 1, half 1 the other two
      const uint32_t lo = c[0] | (c[1] << 16), hi = c[2] | (c[3] << 16);
      const uint32_t theirs = (uint32_t)__shfl_xor((int)(tl.lh == 0 ? hi : lo), 32);
      const uint32_t even = tl.lh == 0 ? lo : theirs, odd = tl.lh == 0 ? theirs : hi;
      if (p < tc.row_end && b < nb) {
        *reinterpret_cast<uint2*>(g.H + p * ldh + b * 16 + 8 * tl.lh) = make_uint2((even & 0xffffu) | (odd << 16), (even >> 16) | (odd & 0xffff0000u));
        if (tl.lh == 0) g.SH[p * ldsh + b] = (uint8_t)byte;
        if (tl.lh == 0 && b == nb - 1)
          for (int64_t z = nb; z < ldsh; ++z) g.SH[p * ldsh + z] = 0;
      }
    }
  }
}

template <class Cfg>
__global__ __launch_bounds__(Cfg::NT, 1) void mx_gemm_kernel(const MxGemmArgs g) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::LDS_BYTES];
  const int n_vis = g.counts[0];
  const int tiles = routed_tile_count(n_vis, g.M, g.N, Cfg::BM, Cfg::BN_OUT), total = tiles * g.splits;
  const int per_xcd = cdiv(total, kXcds), slot = (int)blockIdx.x / kXcds;
  const int L = ((int)blockIdx.x % kXcds) * per_xcd + slot;
  if (slot >= per_xcd || L >= total) return;
  const int split = L / tiles;
  const TileCoord tc = routed_tile_coord(L - split * tiles, n_vis, g.M, g.N, Cfg::BM, Cfg::BN_OUT, Cfg::GROUP_M);
  TileLanes<Cfg> tl;
  tl.init();
  const int nk = cdiv(g.K, kMxStageK);
  const int per_split = cdiv(cdiv(nk, 2), g.splits) * 2;  // (two stages share their scales' load)
  const int kt0 = min(split * per_split, nk), kt1 = min(kt0 + per_split, nk);
  f32x16_t acc[Cfg::TM][Cfg::TN];
  if (kt0 < kt1) mx_mainloop<Cfg>(g, tc, tl, kt0, kt1, lds, acc);
  else zero_acc<Cfg>(acc);
  if constexpr (Cfg::DUAL) {
    mx_swiglu_store<Cfg>(g, tc, tl, acc);
    if (g.pre != nullptr) {
      dma_wait_barrier<0>();
      mx_store<Cfg, false>(g, g.pre, g.ld_pre, tc, tl, lds, [&](int i, int j, int v) { return acc[i][j][v]; });
      mx_store<Cfg, false>(g, g.pre + g.N, g.ld_pre, tc, tl, lds, [&](int i, int j, int v) { return acc[i][j + Cfg::TN_OUT][v]; });
    }
  } else if (g.splits > 1) {
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
      const int p = tc.row0 + tl.wm * Cfg::WTM + i * 32 + (int)tl.lr;
      if (p >= tc.row_end) continue;
      float* row = g.P + ((int64_t)split * g.M + p) * g.N;
#pragma unroll
      for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = tc.n0 + tl.wn * Cfg::WTN_OUT + j * 32 + acc_col<Cfg>(4 * q, (int)tl.lh);
          if (n < g.N)  // (N % 4 == 0)
            *reinterpret_cast<float4*>(row + n) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
    }
  } else {
    dma_wait_barrier<0>();  // every wave has read its last fragments
    mx_store<Cfg, true>(g, g.C, g.ldc, tc, tl, lds, [&](int i, int j, int v) { return acc[i][j][v]; });
  }
}

template <class Cfg>
hipError_t launch(const MxGemmArgs& g, hipStream_t stream) {
  if (g.M <= 0 || g.N <= 0) return hipSuccess;
  if (g.K <= 0 || g.splits < 1 || (g.splits > 1 && (Cfg::DUAL || g.P == nullptr || g.N % 4 != 0))) return hipErrorInvalidValue;
  static_assert(WaveRows<Cfg>::BYTES * Cfg::NWAVES <= Cfg::LDS_BYTES, "results pass through the stages");
  const int64_t total = (int64_t)(cdiv(g.M, Cfg::BM) + 1) * cdiv(g.N, Cfg::BN_OUT) * g.splits;
  const int64_t blocks = (cdiv64(total, kXcds) + 1) * kXcds;
  if (blocks > 0xffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((mx_gemm_kernel<Cfg>), dim3((unsigned)blocks), dim3(Cfg::NT), 0, stream, g);
  return hipGetLastError();
}

template <bool DUAL>
struct MxTiles {
  using Big = MxTile<256, 256, 2, 2, DUAL, DUAL ? 8 : 4>;
  using Small = MxTile<128, 128, 2, 2, DUAL, DUAL ? 8 : 4>;
};

template <bool DUAL>
hipError_t dispatch(int tile, const MxGemmArgs& g, hipStream_t stream) {
  switch (tile) {
    case MX_256x256: return launch<typename MxTiles<DUAL>::Big>(g, stream);
    case MX_128x128: return launch<typename MxTiles<DUAL>::Small>(g, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

int mx_tile_rows(int tile) { return tile == MX_256x256 ? 256 : 128; }
int mx_tile_columns(int tile, bool dual) { return (tile == MX_256x256 ? 256 : 128) / (dual ? 2 : 1); }

hipError_t launch_mx_gemm(int tile, const MxGemmArgs& g, hipStream_t stream) { return dispatch<false>(tile, g, stream); }
hipError_t launch_mx_swiglu_gemm(int tile, const MxGemmArgs& g, hipStream_t stream) { return dispatch<true>(tile, g, stream); }

}  // namespace ffnk
