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
  static_assert((BM / 8) % NWAVES == 0 && (BN / (DUAL ? 16 : 8)) % NWAVES == 0, "panel rows spread evenly over the waves, gate and up rows apart");
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

// The tile a workgroup works on, from its operands' addresses to its sums.
template <class Cfg>
struct MxLoop {
  static constexpr int NW = Cfg::NWAVES, TM = Cfg::TM, TN = Cfg::TN, BM = Cfg::BM, BN = Cfg::BN;
  static constexpr int NJA = TileLanes<Cfg>::NJA, NJB = TileLanes<Cfg>::NJB, LOADS = NJA + NJB;
  // Scale loads: 64 rows each.  Every wave issues as many, which it counts: the last group's again where they do not come out even.
  static constexpr int NG = (BM + BN) / 64, NS = cdiv(NG, NW);
  // A stage is four steps of 64 columns, TM x TN matrix instructions each.  Behind them, spread over the step, the next step's
  // fragments are read (the last step's early, the next stage's first ones behind the data barrier).  Two barriers a stage:
  //   RELEASE: every wave has read the last of this stage - the loads of the stage after next go into its memory from here on
  //   DATA: the next stage has landed
  // which leaves the loads 1.2 to 1.5 stages to land.
  static constexpr int NM = TM * TN, NF = TM + TN, LEV = NM >= 16 ? 2 : 1, EARLY = NM >= 16 ? 4 : NM >= 8 ? 2 : 1, LATE = NM >= 16 ? 6 : NM >= 8 ? 3 : 1;
  static constexpr int RELEASE = 3 * NM - EARLY, DATA = 3 * NM + LATE, TURN = 4 * NM;
  static constexpr int FIRST = (TURN - RELEASE) / LEV, BEFORE = (DATA - RELEASE) / LEV;  // loads behind RELEASE in a stage, and of these ahead of DATA
  static_assert(FIRST <= LOADS && LOADS + NS - FIRST <= RELEASE / LEV, "the loads of a stage go out between its two RELEASE barriers");

  TileLanes<Cfg> tl;
  uint8_t* lds;
  int nb, nk;
  uint32_t koff[4], a_base;
  // of the tile
  int kt0, kt1;
  const uint8_t* code_base[3];  // token rows, weight rows (SwiGLU: gate, up)
  uint32_t off_a[NJA], off_b[NJB], last_back;
  const uint8_t* scale_base[NS];
  uint32_t off_s[NS];
  int64_t scale_turn[NS];  // from one 512 columns to the next

  __device__ __forceinline__ void init(const MxGemmArgs& g, uint8_t* lds_) {
    tl.init();
    lds = lds_;
    nb = cdiv(g.K, kMxBlock);
    nk = cdiv(nb, 8);
#pragma unroll
    for (int s = 0; s < 4; ++s) koff[s] = lds_swizzle(tl.lr, 4 * tl.lh + s);
    a_base = (uint32_t)(tl.wm * Cfg::WTM) * kRowBytes;
    // The last stage of a contraction that is no whole number of them: pieces past a row's end repeat its last one, and count with
    // the scale bytes behind the last block, which are 0.
    const int rest = nb - (nk - 1) * 8;
    last_back = (int)tl.c_log >= rest ? (uint32_t)((rest - 1 - (int)tl.c_log) * 16) : 0u;
  }

  // Addresses, and the loads ahead of the first stage.  The token rows' places come from memory: all of them are asked for at once, and the
  // weight rows' loads go out before they are there.
  __device__ __forceinline__ void begin(const MxGemmArgs& g, const TileCoord& tc, int first_stage, int end_stage) {
    kt0 = first_stage;
    kt1 = end_stage;
    const int64_t lda = (int64_t)nb * 16;
    auto a_place = [&](int r) { return min(tc.row0 + r, tc.row_end - 1); };  // rows past the group's end repeat its last one; their results are not stored
    int place[NJA], scale_place[NS];
#pragma unroll
    for (int j = 0; j < NJA; ++j) place[j] = g.perm[a_place(tl.load_row(j))];
#pragma unroll
    for (int s = 0; s < NS; ++s) scale_place[s] = g.perm[a_place(min(s * NW + tl.wave_s, NG - 1) * 64 + tl.lane)];
    __builtin_amdgcn_sched_barrier(0);
    const int n_first = min(tc.n0, g.N - 1);
    auto b_row = [&](int r) { return min(tc.n0 + r, g.N - 1) - n_first; };
    code_base[1] = g.B0[tc.grp].codes + n_first * lda;
    if (Cfg::DUAL) code_base[2] = g.B1[tc.grp].codes + n_first * lda;
#pragma unroll
    for (int j = 0; j < NJB; ++j) {
      const int r = tl.load_row(j) - (Cfg::DUAL && j >= NJB / 2 ? BN / 2 : 0);
      off_b[j] = (uint32_t)b_row(r) * (uint32_t)lda + tl.c_log * 16;
    }
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int l = 0; l < NJB; ++l) load(l, 0, kt0);
#endif
    __builtin_amdgcn_sched_barrier(0);
    // Gathered rows are addressed from the start of A (the host checks that 32 bits reach them).
    const int64_t row0 = g.gather ? 0 : tc.row0;
    auto a_row = [&](int r, int gathered) { return g.gather ? gathered : a_place(r) - tc.row0; };
    code_base[0] = g.A.codes + row0 * lda;
#pragma unroll
    for (int j = 0; j < NJA; ++j) off_a[j] = (uint32_t)a_row(tl.load_row(j), place[j]) * (uint32_t)lda + tl.c_log * 16;
    // Scale rows: group q of 64, the token rows' first.
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int q = min(s * NW + tl.wave_s, NG - 1);  // (uniform)
      if (q < BM / 64) {
        scale_base[s] = g.A.scales + row0 * 16;
        off_s[s] = (uint32_t)a_row(q * 64 + tl.lane, scale_place[s]) * 16u;
      } else {
        const int r = q * 64 - BM;
        const bool up = Cfg::DUAL && r >= BN / 2;
        scale_base[s] = (up ? g.B1[tc.grp].scales : g.B0[tc.grp].scales) + n_first * 16;
        off_s[s] = (uint32_t)b_row(r - (up ? BN / 2 : 0) + tl.lane) * 16u;
      }
      scale_base[s] = wave_uniform(scale_base[s]);
      scale_turn[s] = (int64_t)(q < BM / 64 ? g.M : g.N) * 16;
    }
#if defined(__HIP_DEVICE_COMPILE__)
    // (the rest of it, and of the second stage what the stage before would have issued)
#pragma unroll
    for (int l = NJB; l < LOADS + NS; ++l) load(l, 0, kt0);
    if (kt0 + 1 < kt1)
#pragma unroll
      for (int l = 0; l < FIRST; ++l) load(l, 1, kt0 + 1);
#endif
  }

#if defined(__HIP_DEVICE_COMPILE__)
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const uint8_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, 0xffffffff, 0x00020000);
  }
  // Load l of stage kt (of parity u): weight rows, token rows, then - with the first of two stages - their scales.
  __device__ __forceinline__ void load(int l, int u, int kt) const {
    uint8_t* stage = lds + u * Cfg::STAGE_BYTES;
    if (l < LOADS) {
      const uint32_t back = kt == nk - 1 ? last_back : 0u;
      const int j = l < NJB ? l : l - NJB;
      if (l < NJB)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(code_base[Cfg::DUAL && j >= NJB / 2 ? 2 : 1]),
                                                 FFNK_LDS_PTR(stage + Cfg::A_BYTES + (j * NW + tl.wave_s) * 1024), 16, off_b[j] + back, kt * kRowBytes, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(code_base[0]), FFNK_LDS_PTR(stage + (j * NW + tl.wave_s) * 1024), 16, off_a[j] + back,
                                                 kt * kRowBytes, 0, 0);
    } else {
      const int s = l - LOADS, q = min(s * NW + tl.wave_s, NG - 1);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(scale_base[s] + (kt >> 1) * scale_turn[s]),
                                               FFNK_LDS_PTR(lds + 2 * Cfg::STAGE_BYTES + ((kt >> 1) & 1) * Cfg::SCALE_BYTES + q * 1024), 16, off_s[s],
                                               0, 0, 0);
    }
  }
  // The contraction over stages [kt0, kt1), kt0 even, whose head has been issued.
  __device__ __forceinline__ void run(f32x16_t (&acc)[TM][TN]) const {
    i32x4_t fa[2][TM], fb[2][TN];
    int sa[2][TM], sb[2][TN];
    // Fragment f of step s of a stage of parity u: weight rows, then token rows; their scales.
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
    constexpr f32x16_t kZero = {};
    auto stage = [&](auto parity, auto first, int kt, auto next_, auto next2_) {
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
          acc[i][j] = mx_mfma32<s>(fb[s & 1][j], fa[s & 1][i], decltype(first)::value && s == 0 ? kZero : acc[i][j], sb[u][j], sa[u][i]);
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

    if (kt0 + 1 < kt1) dma_wait_barrier<FIRST>();
    else dma_wait_barrier<0>();
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      read_scale(f, 0, kt0);
      read(f, 0, 0);
    }
    constexpr auto even = std::integral_constant<int, 0>{};
    constexpr auto odd = std::integral_constant<int, 1>{};
    constexpr auto yes = std::true_type{};
    constexpr auto no = std::false_type{};
    stage(even, yes, kt0, kt0 + 1 < kt1, kt0 + 2 < kt1);
    int kt = kt0 + 1;
    for (; kt + 3 < kt1; kt += 2) {  // no branches inside
      stage(odd, no, kt, yes, yes);
      stage(even, no, kt + 1, yes, yes);
    }
    for (; kt < kt1; kt += 2) {
      stage(odd, no, kt, kt + 1 < kt1, kt + 2 < kt1);
      if (kt + 1 < kt1) stage(even, no, kt + 1, kt + 2 < kt1, kt + 3 < kt1);
    }
  }
#else
  __device__ void run(f32x16_t (&acc)[TM][TN]) const {}
#endif
};

// 32 x 32 results of the wave in bf16: token row lr of `base` at element `row` (-1: not stored), columns n0 ... n0 + 31.  A lane has runs
// of four columns, the lane 32 further the runs between them: of two runs each hands one over, and both store eight columns.
template <class Cfg>
__device__ __forceinline__ void mx_store32(const f32x16_t& v, uint16_t* base, int64_t row, int n0, int N, uint32_t lh, bool whole) {
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    uint32_t w[4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x2_t x = lane_swap32(pack2bf(v[4 * q + 2 * half], v[4 * q + 2 * half + 1]), pack2bf(v[4 * q + 4 + 2 * half], v[4 * q + 5 + 2 * half]));
      w[half] = x[0];
      w[2 + half] = x[1];
    }
    const int n = n0 + 8 * q + 8 * (int)lh;
    if (row < 0 || n >= N) continue;
    uint16_t* out = base + row + n;
    if (whole) {
      *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < N) out[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
  }
}

__device__ __forceinline__ bool whole_chunks(const uint16_t* base, int64_t ld, int N) {
  return N % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
}

// H = Q(silu(gate) up) for the wave's tile.  An accumulator tile's 32 weight rows are one block of the intermediate: a lane holds 16 of
// a token's 32 values, the lane 32 further the other 16.
template <class Cfg, bool WHOLE>  // WHOLE: no column past the last one
__device__ __forceinline__ void mx_swiglu_store(const MxGemmArgs& g, const TileCoord& tc, const TileLanes<Cfg>& tl,
                                                const f32x16_t (&acc)[Cfg::TM][Cfg::TN]) {
  const int nb = cdiv(g.N, kMxBlock);
  const int64_t ldh = (int64_t)nb * 16;
#pragma unroll
  for (int i = 0; i < Cfg::TM; ++i) {
    const int p = tc.row0 + tl.wm * Cfg::WTM + i * 32 + (int)tl.lr;
#pragma unroll
    for (int j = 0; j < Cfg::TN_OUT; ++j) {
      const int b = (tc.n0 + tl.wn * Cfg::WTN_OUT) / 32 + j;
      float h[16], top = 0.f;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        h[v] = swiglu(acc[i][j][v], acc[i][j + Cfg::TN_OUT][v]);
        if (!WHOLE && b * 32 + acc_col<Cfg>(v, (int)tl.lh) >= g.N) h[v] = 0.f;
      }
#pragma unroll
      for (int v = 0; v < 16; v += 2) top = mx_top(top, h[v], h[v + 1]);
      const uint32_t byte = mx_scale_byte(mx_top_across32(top));
      uint32_t c[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) c[q] = mx_codes4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3], byte);
      // run q of either half is 16 bits of dword q: half 0 stores dwords 0 and 1, half 1 the other two
      const u32x2_t w = lane_swap32(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
      if (p < tc.row_end && (WHOLE || b < nb)) {
        *reinterpret_cast<uint2*>(g.H + p * ldh + b * 16 + 8 * tl.lh) = make_uint2((w[0] & 0xffffu) | (w[1] << 16), (w[0] >> 16) | (w[1] & 0xffff0000u));
        if (tl.lh == 0) {
          uint8_t* s = g.SH + mx_scale_at(p, b, g.M);
          *s = (uint8_t)byte;
          if (b == nb - 1)
            for (int z = 1; (b + z) % 16 != 0; ++z) s[z] = 0;
        }
      }
    }
  }
}

// LDS operations of a wave's lanes before and behind it keep their order.
__device__ __forceinline__ void wave_turn() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#endif
}

// The results of one tile.  KEEP (SwiGLU): the projections too (MxGemmArgs::pre).
template <class Cfg, bool KEEP>
__device__ __forceinline__ void mx_epilogue(const MxGemmArgs& g, const TileCoord& tc, int split, const TileLanes<Cfg>& tl, const int (&out_rows)[Cfg::TM],
                                            const f32x16_t (&acc)[Cfg::TM][Cfg::TN], uint8_t* lds) {
  const int p0 = tc.row0 + tl.wm * Cfg::WTM + (int)tl.lr, n0 = tc.n0 + tl.wn * Cfg::WTN_OUT;
  if constexpr (Cfg::DUAL) {
    if (tc.n0 + Cfg::BN_OUT <= g.N) mx_swiglu_store<Cfg, true>(g, tc, tl, acc);
    else mx_swiglu_store<Cfg, false>(g, tc, tl, acc);
    if constexpr (KEEP) {
      // 32 x 32 projections at a time through LDS, so that a store writes whole lines of them, past the caches: M = 4096, d = 4096, h = 14336
      // with its backward 1890 us, 1895 - 1902 without the hint, 1910 straight from the accumulators, 2140 so with the hint.  (bf16 projections
      // took 1762, and left the gradient half as much again off: 0.0034 of its norm against 0.0023.)
      const bool whole = (reinterpret_cast<uintptr_t>(g.pre) & 15) == 0 && (g.ld_pre | g.N) % 4 == 0;
      __syncthreads();  // every wave has read its last fragments
      float4* const turn = reinterpret_cast<float4*>(lds + tl.wave * 4096);
      const int out_row = tl.lane / 8, n = n0 + 4 * (tl.lane % 8);
#pragma unroll
      for (int i = 0; i < Cfg::TM; ++i) {
        const int p = p0 - (int)tl.lr + i * 32 + out_row;
        float* out = g.pre + (int64_t)p * g.ld_pre + n;
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j) {
          const int nj = (j % Cfg::TN_OUT) * 32, at = nj + (j < Cfg::TN_OUT ? 0 : g.N);
          wave_turn();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            turn[tl.lr * 8 + ((2 * q + tl.lh) ^ (tl.lr & 7))] =
                make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
          wave_turn();
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 v = turn[(out_row + 8 * r) * 8 + ((tl.lane % 8) ^ out_row)];
            if (p + 8 * r >= tc.row_end) continue;
            float* dst = out + (int64_t)(8 * r) * g.ld_pre + at;
            if (whole) {
              if (n + nj < g.N) __builtin_nontemporal_store(f32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<f32x4_t*>(dst));
            } else {
              const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (n + nj + k < g.N) dst[k] = e[k];
            }
          }
        }
      }
    }
  } else if (g.splits > 1) {
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
      const int p = p0 + i * 32;
      if (p >= tc.row_end) continue;
      float* row = g.P + ((int64_t)split * g.M + p) * g.N;
#pragma unroll
      for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + j * 32 + acc_col<Cfg>(4 * q, (int)tl.lh);
          if (n < g.N)  // (N % 4 == 0)
            *reinterpret_cast<float4*>(row + n) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
    }
  } else {
    const bool whole = whole_chunks(g.C, g.ldc, g.N);
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
      const int64_t row = out_rows[i] < 0 ? -1 : out_rows[i] * g.ldc;
#pragma unroll
      for (int j = 0; j < Cfg::TN; ++j) mx_store32<Cfg>(acc[i][j], g.C, row, n0 + j * 32, g.N, tl.lh, whole);
    }
  }
}

// One tile a workgroup; every XCD takes an eighth of the order.  On v_mfma_scale_f32_32x32x64_f8f6f4 (from registers alone 7.8 PFLOP/s on all
// CUs, the 16x16x128 form 5.0).  A tile costs 11 - 14 us beyond its stages: first loads, the SwiGLU epilogue and the results.
// M = 32768, d = 4096, h = 14336: SwiGLU 1840 - 1910 us (4.1 PFLOP/s, matrix pipes 54 % busy at a held clock of 1.81 GHz of 2.4),
// down projection 800 - 890 us (4.6 PFLOP/s, 61 % at 1.72 GHz).  M = 300: 38 us for 125 MB of weights, down 27 for 62 MB and 5 for the
// sum over its K ranges: every stage waits for its weights.
template <class Cfg, bool KEEP>
__global__ __launch_bounds__(Cfg::NT, 1) void mx_gemm_kernel(const MxGemmArgs g) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::LDS_BYTES];
  const int n_vis = g.counts[0];
  const int tiles = routed_tile_count(n_vis, g.M, g.N, Cfg::BM, Cfg::BN_OUT), total = tiles * g.splits;
  const int per_xcd = cdiv(total, kXcds), slot = (int)blockIdx.x / kXcds;
  const int L = ((int)blockIdx.x % kXcds) * per_xcd + slot;
  if (slot >= per_xcd || L >= total) return;
  const int split = L / tiles;
  const TileCoord tc = routed_tile_coord(L - split * tiles, n_vis, g.M, g.N, Cfg::BM, Cfg::BN_OUT, Cfg::GROUP_M);
  const int nk = cdiv(g.K, kMxStageK), per_split = cdiv(cdiv(nk, 2), g.splits) * 2;  // (two stages share their scales' load)
  MxLoop<Cfg> loop;
  loop.init(g, lds);
  // Where the results' rows go: asked for ahead of the contraction, which hides the round trip, where registers are left for it.
  constexpr bool AHEAD = Cfg::BM < 256;
  int out_rows[Cfg::TM];
  auto ask = [&]() {
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
      const int p = tc.row0 + loop.tl.wm * Cfg::WTM + i * 32 + (int)loop.tl.lr;
      const int place = Cfg::DUAL ? p : g.perm[min(p, tc.row_end - 1)];
      out_rows[i] = p < tc.row_end ? place : -1;
    }
  };
  if (AHEAD) ask();
  loop.begin(g, tc, split * per_split, min((split + 1) * per_split, nk));
  f32x16_t acc[Cfg::TM][Cfg::TN];
  loop.run(acc);
  if (!AHEAD) ask();
  mx_epilogue<Cfg, KEEP>(g, tc, split, loop.tl, out_rows, acc, lds);
}

template <class Cfg>
hipError_t launch(const MxGemmArgs& g, hipStream_t stream) {
  if (g.M <= 0 || g.N <= 0) return hipSuccess;
  if (g.K <= 0 || g.splits < 1 || (g.splits > 1 && (Cfg::DUAL || g.P == nullptr || g.N % 4 != 0))) return hipErrorInvalidValue;
  const int pairs = cdiv(cdiv(g.K, kMxStageK), 2);
  if ((g.splits - 1) * cdiv(pairs, g.splits) >= pairs) return hipErrorInvalidValue;  // an empty K range
  const int64_t total = (int64_t)(cdiv(g.M, Cfg::BM) + 1) * cdiv(g.N, Cfg::BN_OUT) * g.splits;
  if (total > kMxMaxWorkgroups) return hipErrorInvalidValue;
  const dim3 blocks((unsigned)round_up64(total, kXcds));
  if constexpr (Cfg::DUAL) {
    if (g.pre != nullptr) {
      hipLaunchKernelGGL((mx_gemm_kernel<Cfg, true>), blocks, dim3(Cfg::NT), 0, stream, g);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((mx_gemm_kernel<Cfg, false>), blocks, dim3(Cfg::NT), 0, stream, g);
  return hipGetLastError();
}

template <bool DUAL>
struct MxTiles {
  static constexpr int G = DUAL ? 8 : 4;
  using T0 = MxTile<256, 256, 2, 2, DUAL, G>;
  using T1 = MxTile<128, 128, 2, 2, DUAL, G>;
  using T2 = MxTile<64, 128, 2, 2, DUAL, G>;
};

template <bool DUAL>
hipError_t dispatch(int tile, const MxGemmArgs& g, hipStream_t stream) {
  switch (tile) {
    case MX_256x256: return launch<typename MxTiles<DUAL>::T0>(g, stream);
    case MX_128x128: return launch<typename MxTiles<DUAL>::T1>(g, stream);
    case MX_64x128: return launch<typename MxTiles<DUAL>::T2>(g, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

int mx_tile_rows(int tile) { return tile == MX_256x256 ? 256 : tile == MX_64x128 ? 64 : 128; }
int mx_tile_columns(int tile, bool dual) { return (tile == MX_256x256 ? 256 : 128) / (dual ? 2 : 1); }

hipError_t launch_mx_gemm(int tile, const MxGemmArgs& g, hipStream_t stream) { return dispatch<false>(tile, g, stream); }
hipError_t launch_mx_swiglu_gemm(int tile, const MxGemmArgs& g, hipStream_t stream) { return dispatch<true>(tile, g, stream); }

}  // namespace ffnk
