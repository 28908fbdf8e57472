// MXFP4 (OCP Microscaling): 32 neighbours of a row share a power-of-two scale, each is a 4-bit number.
//   value = number * 2^(scale byte - 127),  numbers 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (E2M1);  scale byte 255: NaN
// A tensor of [rows, columns] is held as whole blocks: nb = cdiv(columns, 32) blocks of a row, 16 bytes of codes each (the even
// column in a byte's low half, rows one after the other), and one scale byte each.  The scale bytes of 16 blocks (512 columns) lie
// together, and those of all rows behind one another, [cdiv(nb, 16)][rows][16]: the products want them for many rows at a time, and
// a load of 64 rows of a tile is 1 KB in one piece instead of 64 cache lines.  Codes past the last column are 0; so are the scale
// bytes past the last block, which lets the products run over whole groups of blocks: a code read there is some finite number, and
// the two operands' scales of 2^-127 take its product below the smallest fp32.
#pragma once
#include "common.hpp"

namespace ffnk {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

constexpr int kMxBlock = 32;

__host__ __device__ constexpr int64_t mx_blocks(int64_t columns) { return cdiv64(columns, kMxBlock); }
__host__ __device__ constexpr int64_t mx_code_stride(int64_t columns) { return mx_blocks(columns) * 16; }
__host__ __device__ constexpr int64_t mx_scale_bytes(int64_t rows, int64_t columns) { return rows * round_up64(mx_blocks(columns), 16); }
__host__ __device__ constexpr int64_t mx_scale_at(int64_t row, int64_t block, int64_t rows) { return (block / 16 * rows + row) * 16 + block % 16; }

// Scale byte of a block whose largest magnitude is `top`: the largest power of two not above it over 4, the largest power of two of
// the numbers, so that the largest one lands in [4, 8) and saturates at 6.  Blocks with an infinity or a NaN are NaN as a whole.
__device__ __forceinline__ uint32_t mx_scale_byte(float top) {
  const uint32_t e = __builtin_bit_cast(uint32_t, top) >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// The largest of `top` and the magnitudes of a and b; a NaN if one of them is.
__device__ __forceinline__ float mx_top(float top, float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_fabsf(b)), top);
#else
  return top;
#endif
}

// Lane l exchanges with lane l + 32 (16: with lane l + 16 of its half).
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;
__device__ __forceinline__ u32x2_t lane_swap32(uint32_t a, uint32_t b) {  // {a, a of lane + 32} below, {b of lane - 32, b} above
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_permlane32_swap(a, b, false, false);
#else
  return u32x2_t{a, b};
#endif
}
__device__ __forceinline__ u32x2_t lane_swap16(uint32_t a, uint32_t b) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_permlane16_swap(a, b, false, false);
#else
  return u32x2_t{a, b};
#endif
}
__device__ __forceinline__ float mx_top_of(u32x2_t v) {
  const uint32_t a = v[0], b = v[1];  // (a bit cast of an element as such reads the first one)
  return mx_top(0.f, __builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float mx_top_across32(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  return mx_top_of(lane_swap32(bits, bits));
}
__device__ __forceinline__ float mx_top_across16(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  return mx_top_of(lane_swap16(bits, bits));
}

// Codes of four values of a block in the low 16 bits: divided by its scale (the instruction takes the exponent of its operand,
// which for byte 0 is that of 2^-127 as well), rounded to the nearest number, ties to the even code, saturated.
__device__ __forceinline__ uint32_t mx_codes4(float a, float b, float c, float d, uint32_t byte) {
#if defined(__HIP_DEVICE_COMPILE__)
  const float scale = __builtin_bit_cast(float, byte << 23);
  const uint32_t v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, scale, 0);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, c, d, scale, 1);
#else
  return 0;
#endif
}

// acc += W T^T over 64 columns: 32 weight rows x 32 token rows.  A lane brings 32 columns (16 bytes) of row lane % 32 of either
// operand, and their scales in byte SEL of `sw` and `st`; which 32 columns is free as long as both operands agree.  Results: token row lane % 32, weight rows 8 * (v / 4) + 4 * (lane / 32) + v % 4.
template <int SEL>
__device__ __forceinline__ f32x16_t mx_mfma32(i32x4_t w, i32x4_t t, f32x16_t acc, int sw, int st) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8_t w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, t8 = {t[0], t[1], t[2], t[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, t8, acc, 4, 4, SEL, sw, SEL, st);
#else
  return acc;
#endif
}
// The same over 128 columns of 16 weight rows x 16 token rows (lane % 16; results: weight rows 4 * (lane / 16) + v), scales in byte 0.
__device__ __forceinline__ f32x4_t mx_mfma16(i32x4_t w, i32x4_t t, f32x4_t acc, int sw, int st) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8_t w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, t8 = {t[0], t[1], t[2], t[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, t8, acc, 4, 4, 0, sw, 0, st);
#else
  return acc;
#endif
}

// A tensor's memory.
struct MxRows {
  const uint8_t* codes;
  const uint8_t* scales;
};

// ---- mxfp4_convert.hip ----
enum MxType : int { MX_BF16 = 0, MX_FP16 = 1, MX_FP32 = 2 };
struct MxQuantiseArgs {
  const void* x; int64_t ldx;      // [rows, columns], columns contiguous
  int type;                        // MxType
  const int32_t* perm;             // row r of the result is row perm[r] of x (NULL: row r)
  uint8_t *codes, *scales;
  int rows, columns;
  // With a mask (rows entries) the launch also makes their partition, in blocks ahead of the others.
  const uint8_t* mask = nullptr;
  int32_t *part_perm = nullptr, *part_counts = nullptr;
};
hipError_t launch_mx_quantise(const MxQuantiseArgs& a, hipStream_t stream);
struct MxDequantiseArgs {
  MxRows x[2];                     // x[1].codes == NULL: one tensor
  int type;
  void* y[2]; int64_t ldy;
  int rows, columns;               // columns [columns, ldy) of y are left alone
  const int32_t* counts;           // tensor i is left out where counts[i] is 0 (NULL: neither)
};
hipError_t launch_mx_dequantise(const MxDequantiseArgs& a, hipStream_t stream);

// ---- mxfp4_gemm.hip ----
struct MxGemmArgs {
  MxRows A;                        // token rows: [*, K]
  int gather;                      // row p of the partition is row perm[p] of A (0: row p)
  MxRows B0[2], B1[2];             // per modality (0 = visual): weight rows [N, K]; B1: the up projection of the SwiGLU kernels
  uint16_t* C; int64_t ldc;        // single weight: bf16 [M, N], in token order
  uint8_t *H, *SH;                 // SwiGLU: the intermediate as MXFP4 [M, N], rows in routed order
  float* pre; int64_t ld_pre;      // SwiGLU, optional: both projections, pre[p, n] and pre[p, N + n]
  const int32_t *perm, *counts;
  int M, N, K;
  int splits; float* P;            // single weight, splits > 1: fp32 sums of a K range at P[split][p][N]
};
enum MxTileId : int { MX_256x256 = 0, MX_128x128 = 1, MX_64x128 = 2 };
constexpr int64_t kMxMaxWorkgroups = 0xffff00;  // (2^32 threads)
int mx_tile_rows(int tile);
int mx_tile_columns(int tile, bool dual);  // output columns
hipError_t launch_mx_gemm(int tile, const MxGemmArgs& g, hipStream_t stream);
hipError_t launch_mx_swiglu_gemm(int tile, const MxGemmArgs& g, hipStream_t stream);

// ---- mxfp4_stream.hip: up to kMxStreamRows token rows; a feed-forward layer, whose SwiGLU streams hold two weights' sums, up to
// kMxStreamFfnRows ----
// Streams against tiles, weights from memory, rows of one modality / of both, us: linear K = N = 4096, M = 64 10.5 / 12.6 against
// 14.7 / 14.6.  Feed-forward, 48 rows (40 rows where the tiles lead there too):
//   d = 1024, h = 2816    13.8 / 12.4 against 18.4 / 18.5      d = 4096, h = 14336   38.9 / 51.3 against 39.0 / 48.5 (36.4 / 49.4, 38.8 / 48.0)
//   d = 2048, h = 5632    18.7 / 18.8 against 25.6 / 26.7      d = 5120, h = 13824   54.0 / 61.3 against 44.3 / 56.3 (50.4 / 60.3, 44.1 / 56.0)
//   d = 4096, h = 8192    26.9 / 34.4 against 33.3 / 37.0      d = 8192, h = 20480   87.1 / 119.2 against 80.4 / 138.6 (82.4 / 113.3, 79.5 / 137.4)
// 12 % ahead at 48 rows in the geometric mean, with the tiles up to 18 % ahead; 56 rows on streams of four token tiles, which are not
// there any more, took 45.9 / 61.0 against 36.5 / 48.5 at d = 4096, h = 14336.
constexpr int kMxStreamRows = 64, kMxStreamFfnRows = 48;
struct MxStreamArgs {
  MxRows A;                        // [M, K], token order
  const uint16_t* x; int64_t ldx;  // or bf16 rows, quantised by every workgroup (mx_stream_takes); NULL: A
  MxRows B0[2], B1[2];
  const uint8_t* mask;
  uint16_t* C; int64_t ldc;        // single weight: bf16 [M, N]
  uint8_t *H, *SH;                 // SwiGLU: MXFP4 [M, N], token order
  int M, N, K;
};
bool mx_stream_takes(int64_t M, int64_t K, const uint16_t* x, int64_t ldx);
hipError_t launch_mx_stream(const MxStreamArgs& a, hipStream_t stream);
hipError_t launch_mx_stream_swiglu(const MxStreamArgs& a, hipStream_t stream);

}  // namespace ffnk
