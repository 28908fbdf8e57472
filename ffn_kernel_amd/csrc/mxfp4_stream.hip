// Up to 64 token rows over MXFP4 weights: bound by reading each present modality's weights once.
//
// A workgroup takes a few 16-row weight tiles and its wavefronts an equal part of the contraction each, so that most of the matrix is
// in flight at once.  For every group of 512 columns a tile's rows are 256 bytes of codes, which four loads of 4 rows x 256 bytes
// fetch - whole cache lines; the matrix cores' operands, 16 rows x 64 bytes, are put together in a piece of LDS of the wavefront's own
// - and 16 scale bytes.  The token rows are the other operand: MXFP4 rows read from cache, or up to 16 bf16 rows that the workgroup
// quantises into LDS while its weights are on their way.  The wavefronts' sums meet in LDS in a fixed order.
// d = 4096, h = 14336: M = 1 62 MB in 13.2 us and 31 MB (down projection) in 7.7, M = 27 over both modalities 125 MB in 25 - 26 and 62 MB in
// 15.2: 4 us to start and end, and the bytes at about 6 TB/s (6.9 from one size to the next).
#include "mxfp4.hpp"

namespace ffnk {

namespace {

constexpr int kGroupK = 512, kGroupBlocks = kGroupK / kMxBlock;  // columns that share a row's 16 scale bytes

// A block of 32 bf16 values, 64 bytes -> its codes; the scale byte.
__device__ __forceinline__ i32x4_t quantise_block(const uint4 (&v)[4], uint32_t* byte) {
  i32x4_t codes = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
  uint32_t w[16];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[4 * q] = v[q].x;
    w[4 * q + 1] = v[q].y;
    w[4 * q + 2] = v[q].z;
    w[4 * q + 3] = v[q].w;
  }
  u16x2_t top = {0, 0};  // magnitudes of bf16 order like their bits, a NaN above all
#pragma unroll
  for (int i = 0; i < 16; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
  const uint16_t lo = top[0], hi = top[1];
  *byte = mx_scale_byte(bf2f(lo > hi ? lo : hi));
  const float scale = __builtin_bit_cast(float, *byte << 23);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2_t, w[4 * q]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[4 * q + 1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[4 * q + 2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[4 * q + 3]), scale, 3);
    codes[q] = (int)c;
  }
#endif
  return codes;
}

// Rows in LDS: 16 bytes of codes per block and one block more, so that 16 rows' blocks lie in different banks; scales behind all rows.
__host__ __device__ constexpr int fused_code_stride(int nb) { return (nb + 1) * 16; }
__host__ __device__ constexpr int fused_scale_stride(int nb) { return (nb + 15) / 16 * 16 + 16; }
__host__ __device__ constexpr int fused_bytes(int rows, int nb) { return rows * (fused_code_stride(nb) + fused_scale_stride(nb)); }
constexpr int kFusedRows = 16, kFusedK = 8192;
// Every workgroup quantises all rows: worth a launch less (2.4 us) up to two blocks a thread.  SwiGLU projections, d = 4096,
// h = 14336: M = 1 13.0 us, M = 16 (eight blocks) 22.4 against 20.3 and the launch.
constexpr int kFusedBlocks = 512;  // (9.4 KB of LDS at the most; with room for 16 rows whatever M is, M = 1, K = N = 8192 took 11.6 us, not 9.9)

// 0, which the compiler does not know: a read of LDS at an index with it may be of any slot, so the wavefront's writes ahead of it stay
// ahead of it, and those behind it behind, also where no lane reads what it wrote itself.  The hardware runs a wavefront's LDS
// operations in order, so the lanes then see one another's.  (A fence around the turn orders the weights' loads as well: two groups'
// in flight take past 256 registers, d = 4096, h = 14336, both modalities, M = 27 44.5 us -> 50, M = 48 51 -> 59.)
__device__ __forceinline__ int any_slot() {
  int slot = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("" : "+v"(slot));
#endif
  return slot;
}

// What a workgroup knows of its rows.
struct StreamJob {
  int grp, rows;
  int token;          // of the lane's rank: row `lane` of the modality
  uint8_t* fused;     // FUSED: room for their codes and scales
  i32x4_t* turn;      // 256 slots of the wavefront's own
  float* sums;        // [WAVES - 1][NW][NT][256]
};

// NT: 16-row token tiles at most.  TILES: 16-row weight tiles of a workgroup (SwiGLU: that many of the gate and of the up weight).
// FUSED: bf16 rows (MxStreamArgs::x), quantised here.
template <int NT, bool DUAL, int TILES, int WAVES, bool FUSED>
__device__ __forceinline__ void stream_body(const MxStreamArgs& a, const StreamJob& job) {
  constexpr int NW = TILES * (DUAL ? 2 : 1), NTHREADS = WAVES * kWave;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lr = lane & 15, lg = lane >> 4, rows = job.rows, grp = job.grp;
  int token[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) token[t] = __shfl(job.token, min(t * 16 + lr, rows - 1));  // rows past the last repeat it; not stored

  const int nb = cdiv(a.K, kMxBlock), groups = cdiv(a.K, kGroupK);
  const int64_t ld = (int64_t)nb * 16;
  const int pad = cdiv(nb, 16) * 16 - nb;
  const int n0 = (int)blockIdx.x * TILES * 16;

  f32x4_t acc[NW][NT];
#pragma unroll
  for (int r = 0; r < NW; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  struct Weights {
    i32x4_t codes[NW][4], scales[NW];
  };
  struct Tokens {
    i32x4_t codes[NT][4], scales[NT];
  };
  // Rows and blocks past the last ones repeat them; the blocks count with scale bytes of 0.
  auto load_weights = [&](int g, Weights& v) {
    const uint32_t piece = (uint32_t)(min(g * kGroupBlocks + lr, nb - 1) * 16);
#pragma unroll
    for (int r = 0; r < NW; ++r) {
      const MxRows& w = DUAL && r >= TILES ? a.B1[grp] : a.B0[grp];
      const int first = min(n0 + (r % TILES) * 16, a.N - 1), left = a.N - 1 - first;  // (uniform)
      const uint8_t *codes = w.codes + first * ld, *scales = w.scales + ((int64_t)g * a.N + first) * 16;
      v.scales[r] = *reinterpret_cast<const i32x4_t*>(scales + min(lr, left) * 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) v.codes[r][q] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(codes + ((uint32_t)min(4 * q + lg, left) * (uint32_t)ld + piece)));
    }
  };
  auto load_tokens = [&](int g, Tokens& v) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t > 0 && t * 16 >= rows) continue;  // uniform
      const uint8_t *codes, *scales;
      if constexpr (FUSED) {
        codes = job.fused + min(lr, rows - 1) * fused_code_stride(nb);
        scales = job.fused + a.M * fused_code_stride(nb) + min(lr, rows - 1) * fused_scale_stride(nb) + g * 16;
      } else {
        codes = a.A.codes + token[t] * ld;
        scales = a.A.scales + ((int64_t)g * a.M + token[t]) * 16;
      }
      v.scales[t] = *reinterpret_cast<const i32x4_t*>(scales);
#pragma unroll
      for (int i = 0; i < 4; ++i) v.codes[t][i] = *reinterpret_cast<const i32x4_t*>(codes + min(g * kGroupBlocks + 4 * i + lg, nb - 1) * 16);
    }
  };
  auto multiply = [&](const Weights& w, const Tokens& x) {
#pragma unroll
    for (int r = 0; r < NW; ++r) {
      // slot row * 16 + (piece ^ row): rows as loaded, and one piece of 16 rows, lie in different banks
#pragma unroll
      for (int q = 0; q < 4; ++q) job.turn[(4 * q + lg) * 16 + (lr ^ (4 * q + lg))] = w.codes[r][q];
      const int from = lr * 16 + any_slot();
      i32x4_t f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = job.turn[from + ((4 * i + lg) ^ lr)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int sw = (int)((uint32_t)w.scales[r][i] >> (8 * lg));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (t > 0 && t * 16 >= rows) continue;
          acc[r][t] = mx_mfma16(f[i], x.codes[t][i], acc[r][t], sw, (int)((uint32_t)x.scales[t][i] >> (8 * lg)));
        }
      }
    }
  };

  const int per_wave = cdiv(groups, WAVES), g0 = wave * per_wave, g1 = min(g0 + per_wave, groups);
  // Two groups' loads in flight where registers allow it.
  constexpr bool PAIRS = NT == 1 || (!DUAL && NT == 2);
  if constexpr (FUSED) {
    // The rows' blocks are dealt to the threads; their loads go out ahead of the weights'.
    const int blocks = rows * nb;
    uint4 v[4];
    auto load_block = [&](int b) {  // (every lane of a wavefront is here: they look their row up in one another)
      b = min(b, blocks - 1);
      const int r = b / nb;
      const uint4* p = reinterpret_cast<const uint4*>(a.x + __shfl(job.token, r) * a.ldx + (b - r * nb) * kMxBlock);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = p[q];
    };
    auto put_block = [&](int b) {
      if (b >= blocks) return;
      const int r = b / nb;
      uint32_t byte;
      const i32x4_t codes = quantise_block(v, &byte);
      *reinterpret_cast<i32x4_t*>(job.fused + r * fused_code_stride(nb) + (b - r * nb) * 16) = codes;
      job.fused[a.M * fused_code_stride(nb) + r * fused_scale_stride(nb) + (b - r * nb)] = (uint8_t)byte;
    };
    auto put_rows = [&]() {
      // scale bytes behind the last block
      for (int z = (int)threadIdx.x; z < rows * pad; z += NTHREADS) {
        const int r = z / pad;
        job.fused[a.M * fused_code_stride(nb) + r * fused_scale_stride(nb) + nb + z - r * pad] = 0;
      }
      put_block((int)threadIdx.x);
      for (int first = NTHREADS; first < blocks; first += NTHREADS) {
        load_block(first + (int)threadIdx.x);
        put_block(first + (int)threadIdx.x);
      }
      __syncthreads();
    };
    load_block((int)threadIdx.x);
    Weights w;
    Tokens x;
    // How many groups' weights are on their way meanwhile is the same for every wavefront of the workgroup, which meets in put_rows; a
    // wavefront without that many of its own asks for the last group's again.
    const int last = groups - 1;
    if (per_wave > 1) {
      Weights w2;
      load_weights(min(g0, last), w);
      load_weights(min(g0 + 1, last), w2);
      put_rows();
      if (g0 < g1) {
        load_tokens(g0, x);
        multiply(w, x);
      }
      if (g0 + 1 < g1) {
        load_tokens(g0 + 1, x);
        multiply(w2, x);
      }
    } else {
      load_weights(min(g0, last), w);
      put_rows();
      if (g0 < g1) {
        load_tokens(g0, x);
        multiply(w, x);
      }
    }
    for (int g = g0 + 2; g < g1; ++g) {
      load_weights(g, w);
      load_tokens(g, x);
      multiply(w, x);
    }
  } else {
    int g = g0;
    Weights w;
    Tokens x;
    if constexpr (PAIRS)
      for (; g + 1 < g1; g += 2) {
        Weights w2;
        Tokens x2;
        load_tokens(g, x);
        load_weights(g, w);
        load_tokens(g + 1, x2);
        load_weights(g + 1, w2);
        multiply(w, x);
        multiply(w2, x2);
      }
    for (; g < g1; ++g) {
      load_tokens(g, x);
      load_weights(g, w);
      multiply(w, x);
    }
  }

  // Sum over the wavefronts, in their order; wavefront 0 finishes.
  if (wave > 0)
#pragma unroll
    for (int r = 0; r < NW; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(&job.sums[(((wave - 1) * NW + r) * NT + t) * 256 + lane * 4]) = acc[r][t];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
#pragma unroll
    for (int r = 0; r < NW; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[r][t] += *reinterpret_cast<const f32x4_t*>(&job.sums[(((w - 1) * NW + r) * NT + t) * 256 + lane * 4]);

  // A lane holds token row lr of a token tile and weight rows 4 lg ... 4 lg + 3 of a weight tile.
  if constexpr (DUAL) {
    static_assert(TILES == 2, "a block of the intermediate");
    const int nbh = cdiv(a.N, kMxBlock), b = (int)blockIdx.x;
    const int64_t ldh = (int64_t)nbh * 16;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t * 16 >= rows) continue;
      float h[8], top = 0.f;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        h[v] = swiglu(acc[v / 4][t][v % 4], acc[TILES + v / 4][t][v % 4]);
        if (n0 + v / 4 * 16 + lg * 4 + v % 4 >= a.N) h[v] = 0.f;
      }
#pragma unroll
      for (int v = 0; v < 8; v += 2) top = mx_top(top, h[v], h[v + 1]);
      const uint32_t byte = mx_scale_byte(mx_top_across32(mx_top_across16(top)));
      if (t * 16 + lr >= rows) continue;
      uint8_t* hc = a.H + token[t] * ldh + b * 16 + lg * 2;
      *reinterpret_cast<uint16_t*>(hc) = (uint16_t)mx_codes4(h[0], h[1], h[2], h[3], byte);
      *reinterpret_cast<uint16_t*>(hc + 8) = (uint16_t)mx_codes4(h[4], h[5], h[6], h[7], byte);
      if (lg == 0) {
        uint8_t* s = a.SH + mx_scale_at(token[t], b, a.M);
        *s = (uint8_t)byte;
        if (b == nbh - 1)
          for (int z = 1; (b + z) % 16 != 0; ++z) s[z] = 0;
      }
    }
  } else {
    const bool whole = a.N % 4 == 0 && a.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(a.C) & 7) == 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t * 16 + lr >= rows) continue;
#pragma unroll
      for (int r = 0; r < TILES; ++r) {
        const int n = n0 + r * 16 + lg * 4;
        if (n >= a.N) continue;
        uint16_t* out = a.C + token[t] * a.ldc + n;
        if (whole) {
          *reinterpret_cast<uint2*>(out) = make_uint2(pack2bf(acc[r][t][0], acc[r][t][1]), pack2bf(acc[r][t][2], acc[r][t][3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.N) out[e] = f2bf(acc[r][t][e]);
        }
      }
    }
  }
}

// NT: 16-row token tiles that the call's rows could fill; a modality with at most 16 of them runs as for one.
template <int NT, bool DUAL, int TILES, int WAVES, bool FUSED>
__global__ __launch_bounds__(WAVES * kWave) void mx_stream_kernel(const MxStreamArgs a) {
  constexpr int NW = TILES * (DUAL ? 2 : 1);
  extern __shared__ __attribute__((aligned(16))) uint8_t s_rows[];
  __shared__ float s_sum[(WAVES - 1) * NW * NT * 256];
  __shared__ i32x4_t s_turn[WAVES * 256];
  static_assert(!FUSED || NT == 1, "up to 16 rows");
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;

  // This workgroup's modality and its rows, in order.
  const bool visual_row = lane < a.M && a.mask[lane] != 0;
  const unsigned long long visual = __ballot(visual_row), all = a.M >= 64 ? ~0ull : (1ull << a.M) - 1;
  const int grp = (int)blockIdx.y ^ first_group(__popcll(visual));
  const unsigned long long mine = grp == 0 ? visual : all & ~visual;
  const int rows = __popcll(mine);
  if (rows == 0) return;
  // Row index of rank r, to lane r (the other lanes take the places behind the last rank: every lane sends and receives one).
  int token = lane;
#if defined(__HIP_DEVICE_COMPILE__)
  const unsigned long long below = (1ull << lane) - 1;
  token = __builtin_amdgcn_ds_permute(((mine >> lane & 1) ? __popcll(mine & below) : rows + __popcll(~mine & below)) * 4, lane);
#endif
  const StreamJob job{grp, rows, token, s_rows, s_turn + wave * 256, s_sum};
  if (NT > 1 && rows <= 16) stream_body<1, DUAL, TILES, WAVES, FUSED>(a, job);
  else stream_body<NT, DUAL, TILES, WAVES, FUSED>(a, job);
}

template <int NT, bool DUAL, int TILES, int WAVES, bool FUSED>
hipError_t launch_waves(const MxStreamArgs& a, hipStream_t stream) {
  const int nb = cdiv(a.K, kMxBlock);
  const size_t lds = FUSED ? fused_bytes(a.M, nb) : 0;
  hipLaunchKernelGGL((mx_stream_kernel<NT, DUAL, TILES, WAVES, FUSED>), dim3((unsigned)cdiv(a.N, TILES * 16), 2), dim3(WAVES * kWave), lds, stream, a);
  return hipGetLastError();
}

// Wavefronts of a workgroup by the 512-column groups that there are, as far as a wavefront's registers allow.
template <int NT, bool DUAL, int TILES, bool FUSED>
hipError_t launch_tiles(const MxStreamArgs& a, hipStream_t stream) {
  const int groups = cdiv(a.K, kGroupK);
  if (groups <= 2) return launch_waves<NT, DUAL, TILES, 2, FUSED>(a, stream);
  if constexpr (!DUAL && NT == 1 && !FUSED)  // (FUSED: up to kFusedK)
    if (groups > 16) return launch_waves<NT, DUAL, TILES, 16, FUSED>(a, stream);
  if constexpr (!DUAL)
    if (groups > 4) return launch_waves<NT, DUAL, TILES, 8, FUSED>(a, stream);
  return launch_waves<NT, DUAL, TILES, 4, FUSED>(a, stream);
}

template <bool DUAL, int TILES>
hipError_t launch(const MxStreamArgs& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  if (a.M > (DUAL ? kMxStreamFfnRows : kMxStreamRows) || a.K <= 0 || (a.x != nullptr && !mx_stream_takes(a.M, a.K, a.x, a.ldx))) return hipErrorInvalidValue;
  switch (cdiv(a.M, 16)) {
    case 1: return a.x != nullptr ? launch_tiles<1, DUAL, TILES, true>(a, stream) : launch_tiles<1, DUAL, TILES, false>(a, stream);
    case 2: return launch_tiles<2, DUAL, TILES, false>(a, stream);
    case 3: return launch_tiles<3, DUAL, TILES, false>(a, stream);
    default:
      if constexpr (DUAL) return hipErrorInvalidValue;
      else return launch_tiles<4, DUAL, TILES, false>(a, stream);
  }
}

}  // namespace

bool mx_stream_takes(int64_t M, int64_t K, const uint16_t* x, int64_t ldx) {
  return M <= kFusedRows && K <= kFusedK && K % kMxBlock == 0 && M * (K / kMxBlock) <= kFusedBlocks && ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

hipError_t launch_mx_stream(const MxStreamArgs& a, hipStream_t stream) { return launch<false, 1>(a, stream); }
hipError_t launch_mx_stream_swiglu(const MxStreamArgs& a, hipStream_t stream) { return launch<true, 2>(a, stream); }

}  // namespace ffnk
