// Quantisation to MXFP4 and back.  Both are bound by memory: each value is read and written once.  32768 x 4096 bf16, from memory:
// 66 us and 54 us, 340 MB each way (5.1 and 6.3 TB/s; a plain copy of 1 GiB reaches 5.1).
#include <hip/hip_fp16.h>

#include "mxfp4.hpp"
#include "route_block.hpp"

namespace ffnk {

namespace {

constexpr int kItem = 8;  // columns of a lane: a quad of lanes holds a block

template <int TYPE>
struct MxElement;
template <>
struct MxElement<MX_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float load(T v) { return bf2f(v); }
  static __device__ __forceinline__ T store(float v) { return f2bf(v); }
};
template <>
struct MxElement<MX_FP16> {
  typedef __half T;
  static __device__ __forceinline__ float load(T v) { return __half2float(v); }
  static __device__ __forceinline__ T store(float v) { return __float2half_rn(v); }
};
template <>
struct MxElement<MX_FP32> {
  typedef float T;
  static __device__ __forceinline__ float load(T v) { return v; }
  static __device__ __forceinline__ T store(float v) { return v; }
};

static_assert(kRouteThreads == 256, "blocks of both kinds in one launch");

template <class T>
struct alignas(16) Run {
  T v[kItem];
};

typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
// A run's pieces of 16 bytes; STREAM: past the caches, which hold little of a long tensor and write others' lines back to make room (32768 x
// 4096: 94 -> 66 us and 59 -> 54; a layer's backward, which reads the values next, M = 4096, 1788 -> 1765 us with its forward).
template <bool STREAM, class T>
__device__ __forceinline__ Run<T> load_run(const T* p) {
  if constexpr (!STREAM) return *reinterpret_cast<const Run<T>*>(p);
  Run<T> v;
#pragma unroll
  for (int i = 0; i < (int)sizeof(Run<T>) / 16; ++i) {
    const U32x4 w = __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(p) + i);
    __builtin_memcpy(reinterpret_cast<char*>(&v) + 16 * i, &w, 16);
  }
  return v;
}
template <bool STREAM, class T>
__device__ __forceinline__ void store_run(T* p, const Run<T>& v) {
  if constexpr (!STREAM) *reinterpret_cast<Run<T>*>(p) = v;
  else
#pragma unroll
    for (int i = 0; i < (int)sizeof(Run<T>) / 16; ++i) {
      U32x4 w;
      __builtin_memcpy(&w, reinterpret_cast<const char*>(&v) + 16 * i, 16);
      __builtin_nontemporal_store(w, reinterpret_cast<U32x4*>(p) + i);
    }
}

// Which row and run of kItem columns item `j` of a workgroup is.  Rows of at least kWgItems runs take several workgroups each,
// shorter ones share a workgroup.
struct ItemAt {
  int row, run;
};
struct ItemShape {
  int runs;         // of a row
  int wgs_per_row;  // 0: rows_per_wg instead
  int rows_per_wg;
  uint32_t inverse; // cdiv(2^20, runs): j / runs == j * inverse >> 20 for j, runs <= 1024
};
inline ItemShape item_shape(int runs, int wg_items) {
  ItemShape s{runs, 0, 0, 0};
  if (runs >= wg_items) s.wgs_per_row = cdiv(runs, wg_items);
  else {
    s.rows_per_wg = wg_items / runs;
    s.inverse = (uint32_t)((1u << 20) + runs - 1) / (uint32_t)runs;
  }
  return s;
}
inline int64_t item_blocks(const ItemShape& s, int rows) { return s.wgs_per_row > 0 ? (int64_t)rows * s.wgs_per_row : cdiv64(rows, s.rows_per_wg); }
template <int WG_ITEMS>
__device__ __forceinline__ ItemAt item_at(const ItemShape& s, uint32_t block, int j) {
  if (s.wgs_per_row > 0) {
    const uint32_t row = block / (uint32_t)s.wgs_per_row;
    return {(int)row, (int)(block - row * (uint32_t)s.wgs_per_row) * WG_ITEMS + j};
  }
  const int r = (int)(((uint32_t)j * s.inverse) >> 20);
  return {r < s.rows_per_wg ? (int)block * s.rows_per_wg + r : 0x7fffffff, j - r * s.runs};
}

template <int PATTERN>
__device__ __forceinline__ float quad_lane(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), PATTERN, 0xf, 0xf, true));
#else
  return v;
#endif
}

// U items of a lane, their loads in flight together.  VEC: rows are whole, aligned 16-byte pieces.  The partition's blocks come first:
// a launch of its own takes 3.3 us at M = 2048, and the GEMM behind both waits for either.
template <int TYPE, int U, bool VEC>
__global__ __launch_bounds__(256) void mx_quantise_kernel(const MxQuantiseArgs a, const ItemShape shape, const int nb,
                                                          const RouteShape route) {
  if ((int)blockIdx.x < route.blocks) {
    route_block(a.mask, a.rows, a.part_perm, a.part_counts, route.chunks_per_block, (int)blockIdx.x);
    return;
  }
  const uint32_t block = blockIdx.x - (uint32_t)route.blocks;
  using E = MxElement<TYPE>;
  using T = typename E::T;
  constexpr int WG_ITEMS = 256 * U;
  Run<T> v[U];
  ItemAt at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    at[u] = item_at<WG_ITEMS>(shape, block, u * 256 + (int)threadIdx.x);
    const int column = at[u].run * kItem;
#pragma unroll
    for (int e = 0; e < kItem; ++e) v[u].v[e] = E::store(0.f);
    if (at[u].row < a.rows && column < a.columns) {
      const int64_t row = a.perm != nullptr ? a.perm[at[u].row] : at[u].row;
      const T* p = static_cast<const T*>(a.x) + row * a.ldx + column;
      if (VEC) v[u] = load_run<(U > 1)>(p);
      else
#pragma unroll
        for (int e = 0; e < kItem; ++e)
          if (column + e < a.columns) v[u].v[e] = p[e];
    }
  }
  const int64_t ldc = (int64_t)nb * 16;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[kItem], top = 0.f;
#pragma unroll
    for (int e = 0; e < kItem; ++e) f[e] = E::load(v[u].v[e]);
#pragma unroll
    for (int e = 0; e < kItem; e += 2) top = mx_top(top, f[e], f[e + 1]);
    // the quad's largest (a quad's items are one block: runs is a multiple of 4, and so is every workgroup's first item)
    top = mx_top(top, quad_lane<0xb1>(top), quad_lane<0x4e>(top));  // lanes 1 0 3 2, lanes 2 3 0 1
    top = mx_top(top, quad_lane<0xb1>(top), 0.f);
    const uint32_t byte = mx_scale_byte(top);
    if (at[u].row >= a.rows || at[u].run >= 4 * nb) continue;
    const uint32_t lo = mx_codes4(f[0], f[1], f[2], f[3], byte);
    const uint32_t hi = mx_codes4(f[4], f[5], f[6], f[7], byte);
    *reinterpret_cast<uint32_t*>(a.codes + at[u].row * ldc + at[u].run * 4) = lo | (hi << 16);
    if ((at[u].run & 3) == 0) {
      const int b = at[u].run >> 2;
      uint8_t* s = a.scales + mx_scale_at(at[u].row, b, a.rows);
      *s = (uint8_t)byte;
      if (b == nb - 1)
        for (int z = 1; (b + z) % 16 != 0; ++z) s[z] = 0;
    }
  }
}

template <int TYPE, int U, bool VEC>
__global__ __launch_bounds__(256) void mx_dequantise_kernel(const MxDequantiseArgs a, const ItemShape shape, const int nb) {
  using E = MxElement<TYPE>;
  using T = typename E::T;
  constexpr int WG_ITEMS = 256 * U;
  if (a.counts != nullptr && a.counts[blockIdx.y] == 0) return;
  const MxRows x = a.x[blockIdx.y];
  const int64_t ldc = (int64_t)nb * 16;
  uint32_t codes[U], byte[U];
  ItemAt at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    at[u] = item_at<WG_ITEMS>(shape, blockIdx.x, u * 256 + (int)threadIdx.x);
    codes[u] = byte[u] = 0;
    if (at[u].row < a.rows && at[u].run * kItem < a.columns) {
      codes[u] = *reinterpret_cast<const uint32_t*>(x.codes + at[u].row * ldc + at[u].run * 4);
      byte[u] = x.scales[mx_scale_at(at[u].row, at[u].run >> 2, a.rows)];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int column = at[u].run * kItem;
    if (at[u].row >= a.rows || column >= a.columns) continue;
    Run<T> v;
#if defined(__HIP_DEVICE_COMPILE__)
    const float scale = mx_scale(byte[u]);
#define FFNK_MX_PAIR(I)                                                              \
  {                                                                                  \
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], 1.0f, I);      \
    v.v[2 * I] = E::store(p[0] * scale);                                             \
    v.v[2 * I + 1] = E::store(p[1] * scale);                                         \
  }
    FFNK_MX_PAIR(0) FFNK_MX_PAIR(1) FFNK_MX_PAIR(2) FFNK_MX_PAIR(3)
#undef FFNK_MX_PAIR
#endif
    T* p = static_cast<T*>(a.y[blockIdx.y]) + at[u].row * a.ldy + column;
    if (VEC) store_run<(U > 1)>(p, v);
    else
#pragma unroll
      for (int e = 0; e < kItem; ++e)
        if (column + e < a.columns) p[e] = v.v[e];
  }
}

bool whole_runs(const void* p, int64_t ld, int columns, int type) {
  const int size = type == MX_FP32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && columns % kItem == 0 && ld * size % 16 == 0;
}

// Four items a lane (64 bytes of bf16) once there are two workgroups of them for every CU; fewer rows are spread wider (32768 x 4096
// with two 64.7 and 54.7 us, four 66.6 and 53.5; eight, before the loads passed the caches, 93 and 66 against 94 and 59).
constexpr int kManyItems = 4;
bool many_items(int64_t runs, int64_t rows) { return runs * rows >= (int64_t)256 * kManyItems * 512; }

template <int TYPE>
hipError_t quantise(const MxQuantiseArgs& a, hipStream_t stream) {
  const int nb = (int)mx_blocks(a.columns), runs = 4 * nb;
  const bool vec = whole_runs(a.x, a.ldx, a.columns, TYPE), many = many_items(runs, a.rows);
  const ItemShape s = item_shape(runs, many ? 256 * kManyItems : 256);
  const RouteShape route = a.mask != nullptr ? route_shape(a.rows) : RouteShape{0, 0};
  const int64_t blocks = item_blocks(s, a.rows) + route.blocks;
  if (blocks > 0xffffff) return hipErrorInvalidValue;  // (2^32 threads)
  const dim3 grid((unsigned)blocks), threads(256);
  if (many && vec) hipLaunchKernelGGL((mx_quantise_kernel<TYPE, kManyItems, true>), grid, threads, 0, stream, a, s, nb, route);
  else if (many) hipLaunchKernelGGL((mx_quantise_kernel<TYPE, kManyItems, false>), grid, threads, 0, stream, a, s, nb, route);
  else if (vec) hipLaunchKernelGGL((mx_quantise_kernel<TYPE, 1, true>), grid, threads, 0, stream, a, s, nb, route);
  else hipLaunchKernelGGL((mx_quantise_kernel<TYPE, 1, false>), grid, threads, 0, stream, a, s, nb, route);
  return hipGetLastError();
}

template <int TYPE>
hipError_t dequantise(const MxDequantiseArgs& a, hipStream_t stream) {
  const int nb = (int)mx_blocks(a.columns), runs = 4 * nb, n = a.x[1].codes != nullptr ? 2 : 1;
  const bool vec = whole_runs(a.y[0], a.ldy, a.columns, TYPE) && (n == 1 || whole_runs(a.y[1], a.ldy, a.columns, TYPE));
  const bool many = many_items(runs, a.rows);
  const ItemShape s = item_shape(runs, many ? 256 * kManyItems : 256);
  const int64_t blocks = item_blocks(s, a.rows);
  if (blocks > 0xffffff) return hipErrorInvalidValue;  // (2^32 threads)
  const dim3 grid((unsigned)blocks, (unsigned)n), threads(256);
  if (many && vec) hipLaunchKernelGGL((mx_dequantise_kernel<TYPE, kManyItems, true>), grid, threads, 0, stream, a, s, nb);
  else if (many) hipLaunchKernelGGL((mx_dequantise_kernel<TYPE, kManyItems, false>), grid, threads, 0, stream, a, s, nb);
  else if (vec) hipLaunchKernelGGL((mx_dequantise_kernel<TYPE, 1, true>), grid, threads, 0, stream, a, s, nb);
  else hipLaunchKernelGGL((mx_dequantise_kernel<TYPE, 1, false>), grid, threads, 0, stream, a, s, nb);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantise(const MxQuantiseArgs& a, hipStream_t stream) {
  if (a.rows <= 0 || a.columns <= 0) return hipSuccess;
  switch (a.type) {
    case MX_BF16: return quantise<MX_BF16>(a, stream);
    case MX_FP16: return quantise<MX_FP16>(a, stream);
    case MX_FP32: return quantise<MX_FP32>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_mx_dequantise(const MxDequantiseArgs& a, hipStream_t stream) {
  if (a.rows <= 0 || a.columns <= 0) return hipSuccess;
  switch (a.type) {
    case MX_BF16: return dequantise<MX_BF16>(a, stream);
    case MX_FP16: return dequantise<MX_FP16>(a, stream);
    case MX_FP32: return dequantise<MX_FP32>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ffnk
