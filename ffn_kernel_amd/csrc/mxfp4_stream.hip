// Up to 64 token rows over MXFP4 weights: bound by reading each present modality's weights once.
//
// A workgroup takes a few 16-row weight tiles and its wavefronts an equal part of the contraction each, so that the whole matrix is
// in flight at once.  Weight rows go from memory to the matrix cores' operands as they lie: 16 rows x 64 bytes a load (16 x 128
// columns), four loads and the 16 scale bytes of a row for every 512 columns.  The token rows are the other operand, read from
// cache.  The wavefronts' sums meet in LDS in a fixed order.
#include "mxfp4.hpp"

namespace ffnk {

namespace {

constexpr int kGroupK = 512;  // columns that share a row's 16 scale bytes

// NT: 16-row token tiles at most.  TILES: 16-row weight tiles of a workgroup (SwiGLU: that many of the gate and of the up weight).
template <int NT, bool DUAL, int TILES, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void mx_stream_kernel(const MxStreamArgs a) {
  constexpr int NW = TILES * (DUAL ? 2 : 1);
  __shared__ float s_sum[WAVES > 1 ? (WAVES - 1) * NW * NT * 256 : 1];
  __shared__ int s_token[kMxStreamRows];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int lr = lane & 15, lg = lane >> 4;

  // This workgroup's modality and its rows, in order.
  const bool visual_row = lane < a.M && a.mask[lane] != 0;
  const unsigned long long visual = __ballot(visual_row), all = a.M >= 64 ? ~0ull : (1ull << a.M) - 1;
  const int grp = (int)blockIdx.y ^ first_group(__popcll(visual));
  const unsigned long long mine = grp == 0 ? visual : all & ~visual;
  const int rows = __popcll(mine);
  if (rows == 0) return;
  if (wave == 0 && (mine >> lane & 1)) s_token[__popcll(mine & ((1ull << lane) - 1))] = lane;
  __syncthreads();
  int token[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) token[t] = s_token[min(t * 16 + lr, rows - 1)];  // rows past the last repeat it; not stored

  const int nb = cdiv(a.K, kMxBlock), groups = cdiv(a.K, kGroupK);
  const int64_t ld = (int64_t)nb * 16, ld_s = round_up64(nb, 16);
  const int n0 = (int)blockIdx.x * TILES * 16;
  const uint8_t *w_codes[NW], *w_scales[NW], *t_codes[NT], *t_scales[NT];
#pragma unroll
  for (int r = 0; r < NW; ++r) {
    const MxRows& w = DUAL && r >= TILES ? a.B1[grp] : a.B0[grp];
    const int64_t n = min(n0 + (r % TILES) * 16 + lr, a.N - 1);
    w_codes[r] = w.codes + n * ld;
    w_scales[r] = w.scales + n * ld_s;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    t_codes[t] = a.A.codes + token[t] * ld;
    t_scales[t] = a.A.scales + token[t] * ld_s;
  }

  f32x4_t acc[NW][NT];
#pragma unroll
  for (int r = 0; r < NW; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int per_wave = cdiv(groups, WAVES), g0 = wave * per_wave, g1 = min(g0 + per_wave, groups);
#pragma unroll 2
  for (int g = g0; g < g1; ++g) {
    i32x4_t wc[NW][4], ws[NW], tc[NT][4], ts[NT];
    // Blocks past the last one repeat it and count with scale bytes of 0.
#pragma unroll
    for (int r = 0; r < NW; ++r) {
      ws[r] = *reinterpret_cast<const i32x4_t*>(w_scales[r] + g * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) wc[r][i] = *reinterpret_cast<const i32x4_t*>(w_codes[r] + min(g * 16 + 4 * i + lg, nb - 1) * 16);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t > 0 && t * 16 >= rows) continue;  // uniform
      ts[t] = *reinterpret_cast<const i32x4_t*>(t_scales[t] + g * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) tc[t][i] = *reinterpret_cast<const i32x4_t*>(t_codes[t] + min(g * 16 + 4 * i + lg, nb - 1) * 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t > 0 && t * 16 >= rows) continue;
        const int st = (int)((uint32_t)ts[t][i] >> (8 * lg));
#pragma unroll
        for (int r = 0; r < NW; ++r) acc[r][t] = mx_mfma16(wc[r][i], tc[t][i], acc[r][t], (int)((uint32_t)ws[r][i] >> (8 * lg)), st);
      }
  }

  // Sum over the wavefronts, in their order; wavefront 0 finishes.
  if (WAVES > 1) {
    if (wave > 0)
#pragma unroll
      for (int r = 0; r < NW; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(&s_sum[(((wave - 1) * NW + r) * NT + t) * 256 + lane * 4]) = acc[r][t];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
      for (int r = 0; r < NW; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[r][t] += *reinterpret_cast<const f32x4_t*>(&s_sum[(((w - 1) * NW + r) * NT + t) * 256 + lane * 4]);
  }

  // A lane holds token row lr of a token tile and weight rows 4 lg ... 4 lg + 3 of a weight tile.
  if constexpr (DUAL) {
    static_assert(TILES == 2, "a block of the intermediate");
    const int nbh = cdiv(a.N, kMxBlock), b = (int)blockIdx.x;
    const int64_t ldh = (int64_t)nbh * 16, ldsh = round_up64(nbh, 16);
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
        uint8_t* hs = a.SH + token[t] * ldsh;
        hs[b] = (uint8_t)byte;
        if (b == nbh - 1)
          for (int64_t z = nbh; z < ldsh; ++z) hs[z] = 0;
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

template <bool DUAL, int TILES, int WAVES>
hipError_t launch(const MxStreamArgs& a, hipStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return hipSuccess;
  if (a.M > kMxStreamRows || a.K <= 0) return hipErrorInvalidValue;
  const dim3 grid((unsigned)cdiv(a.N, TILES * 16), 2), threads(WAVES * kWave);
  switch (cdiv(a.M, 16)) {
    case 1: hipLaunchKernelGGL((mx_stream_kernel<1, DUAL, TILES, WAVES>), grid, threads, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((mx_stream_kernel<2, DUAL, TILES, WAVES>), grid, threads, 0, stream, a); break;
    case 3: hipLaunchKernelGGL((mx_stream_kernel<3, DUAL, TILES, WAVES>), grid, threads, 0, stream, a); break;
    default: hipLaunchKernelGGL((mx_stream_kernel<4, DUAL, TILES, WAVES>), grid, threads, 0, stream, a); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_stream(const MxStreamArgs& a, hipStream_t stream) { return launch<false, 1, 8>(a, stream); }
hipError_t launch_mx_stream_swiglu(const MxStreamArgs& a, hipStream_t stream) { return launch<true, 2, 4>(a, stream); }

}  // namespace ffnk
