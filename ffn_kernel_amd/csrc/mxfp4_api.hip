// C ABI of the MXFP4 operators (declared in include/ffnk.h): argument checks, workspace carving and kernel sequencing.
#include "../../include/ffnk.h"

#include "capi_parts.hpp"
#include "gemm_sched.hpp"
#include "launch.hpp"
#include "mxfp4.hpp"

using namespace ffnk;

namespace {

constexpr int64_t k4g = (int64_t)1 << 32;
constexpr int kMaxSplits = 8;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int element_size(int dtype) { return dtype == FFNK_DT_FP32 ? 4 : 2; }

int check_tensor(const ffnk_mxfp4_t* t, const char* name) {
  if (!t || !t->codes || !t->scales) return api_fail(FFNK_E_NULL, "%s, its codes or its scales is NULL", name);
  if (!aligned(t->codes, 16) || !aligned(t->scales, 16)) return api_fail(FFNK_E_ALIGN, "%s: codes or scales not 16-byte aligned", name);
  return FFNK_OK;
}
MxRows rows_of(const ffnk_mxfp4_t* t) { return {t->codes, t->scales}; }

size_t tensor_bytes(int64_t rows, int64_t columns) {
  return ws_align((size_t)(rows * mx_code_stride(columns))) + ws_align((size_t)mx_scale_bytes(rows, columns));
}
struct Room {
  uint8_t *codes, *scales;
};
Room carve_tensor(uint8_t* ws, int64_t rows, int64_t columns) { return {ws, ws + ws_align((size_t)(rows * mx_code_stride(columns)))}; }

// Tile and K ranges of a GEMM over [M, K] x [N, K]^T: the cheapest by a model of the launch, in us.  A round of tiles (`slots` at once)
// costs a fixed time and a time per stage of 256 columns, both at most half full and quite full, in between by its share.  The costs are
// fits to launches that find their weights in memory, as a layer of a model does (256x256 / 128x128 / 64x128, half of the rows in either modality):
//   N 4096, K 14336: M 300 81.6 / 48.7 / 46.5, M 700 83.5 / 50.0 / 51.6, M 1411 87.0 / 63.0 / 90.8, M 4096 107 / 132 / 197
//   M 8192, N = K = 2048 28.1 / 28.2 / 37.3    M 2048, N = K = 1024 16.4 / 7.4 / 6.5    M 3001, N 1544, K 2056 23.5 / 15.3 / 18.8
//   SwiGLU, K = 4096, 14336 columns: M 300 37.4 / 42.9 / 52.6, M 700 69.2 / 66.0 / 98.2, M 1411 107.5 / 123.2 / 181.3
// (128x256 had the least by the model in 6 of 4914 shapes from M 49 to 32768, and is not there.)  K ranges add a pass over their sums:
// N 4096, K 14336 on 128x128 in one / two / four ranges and that pass: M 300 48.7, 30.1 + 4.8, 26.0 + 6; M 1411 63.0, 69.5 + 8.
struct Plan {
  int tile, splits;
};
struct TileCost {
  int slots;
  float fixed, stage, fixed_full, stage_full;
};
constexpr TileCost kTileCosts[] = {{256, 12.7f, 1.2f, 14.5f, 1.7f}, {512, 5.f, 0.78f, 7.5f, 1.2f}, {512, 4.5f, 0.74f, 4.f, 0.85f}};
float launch_us(const TileCost& c, int64_t workgroups, float stages) {
  const float half = c.fixed + stages * c.stage, full = c.fixed_full + stages * c.stage_full;
  const float share = (float)(workgroups % c.slots) / (float)c.slots;
  return (float)(workgroups / c.slots) * full + (share == 0.f ? 0.f : share <= 0.5f ? half : half + (full - half) * (2.f * share - 1.f));
}
Plan plan_gemm(bool dual, int64_t M, int64_t N, int64_t K) {
  const int64_t pairs = cdiv64(K, 512);  // two stages each: K ranges are whole pairs
  Plan best{MX_256x256, 1};
  float best_us = 1e30f;
  for (int tile = MX_256x256; tile <= MX_64x128; ++tile) {
    const TileCost& c = kTileCosts[tile];
    // The mask decides between cdiv(M, rows) M-tiles and one more, which it is where the first modality's rows leave fewer past their
    // whole tiles than all rows do.
    const int64_t rows = mx_tile_rows(tile), tiles_n = cdiv64(N, mx_tile_columns(tile, dual)), fewer = cdiv64(M, rows) * tiles_n, tiles = fewer + tiles_n;
    const float more = (float)(M - (cdiv64(M, rows) - 1) * rows) / (float)rows;
    if (tile != MX_256x256 && tiles > kMxMaxWorkgroups) break;
    for (int splits = 1; splits <= kMaxSplits; ++splits) {
      if (splits > 1 && (dual || N % 4 != 0 || M >= 65536 || splits * 2 > pairs || tiles * splits > c.slots)) break;
      const int64_t per_range = cdiv64(pairs, splits);
      if (per_range * (splits - 1) >= pairs) continue;  // an empty range
      const float stages = splits > 1 ? (float)(2 * per_range) : (float)cdiv64(K, 256);
      float us = (1.f - more) * launch_us(c, fewer * splits, stages) + more * launch_us(c, tiles * splits, stages);
      if (splits > 1) us += 2.5f + (float)(splits * M * N) * 4.f / 4e6f;
      if (us < best_us) {
        best_us = us;
        best = {tile, splits};
      }
    }
  }
  return best;
}
size_t partial_bytes(const Plan& p, int64_t M, int64_t N) { return p.splits > 1 ? ws_align((size_t)p.splits * M * N * 4) : 0; }

int check_call(int64_t M, int64_t K, int64_t N) {
  if (int e = api_check_extents(M, K, N)) return e;
  return K == 0 || N == 0 ? api_fail(FFNK_E_SHAPE, "MXFP4 layers need K > 0 and N > 0") : FFNK_OK;
}
int check_rows(const uint16_t* x, int64_t x_stride_m, const ffnk_mxfp4_t* xq, int64_t K) {
  if (xq) return x ? api_fail(FFNK_E_NULL, "x and xq are both given") : check_tensor(xq, "xq");
  if (!x) return api_fail(FFNK_E_NULL, "x and xq are both NULL");
  if (!aligned(x, 2)) return api_fail(FFNK_E_ALIGN, "x not 2-byte aligned");
  return x_stride_m < K ? api_fail(FFNK_E_STRIDE, "x_stride_m=%lld < K=%lld", (long long)x_stride_m, (long long)K) : FFNK_OK;
}
int check_ws(const void* ws, size_t have, size_t need) {
  if (need == 0) return FFNK_OK;
  if (!ws || have < need) return api_fail(FFNK_E_WORKSPACE, "workspace %zu < %zu bytes", have, need);
  return aligned(ws, 16) ? FFNK_OK : api_fail(FFNK_E_ALIGN, "workspace not 16-byte aligned");
}

// The rows of a streamed call: the caller's MXFP4 ones, bf16 ones that the stream quantises itself, or x quantised into `room`.
int stream_rows(const uint16_t* x, int64_t x_stride_m, const ffnk_mxfp4_t* xq, const Room& room, int64_t M, int64_t K, hipStream_t stream, MxStreamArgs* a) {
  if (xq) {
    a->A = rows_of(xq);
    return FFNK_OK;
  }
  if (mx_stream_takes(M, K, x, x_stride_m)) {
    a->x = x;
    a->ldx = x_stride_m;
    return FFNK_OK;
  }
  const MxQuantiseArgs q{x, x_stride_m, MX_BF16, nullptr, room.codes, room.scales, (int)M, (int)K};
  FFNK_TRY_HIP(launch_mx_quantise(q, stream), "quantise kernel");
  a->A = {room.codes, room.scales};
  return FFNK_OK;
}

// ... with the partition (the caller's, or one in `ws`), which the quantising launch makes where it is still to be made.  The GEMM finds
// its rows through it; where 32-bit offsets do not reach them, x is quantised in routed order instead.
struct RoutedRows {
  const int32_t *perm, *counts;
  MxRows A;
  int gather;
};
int routed_rows(const uint16_t* x, int64_t x_stride_m, const ffnk_mxfp4_t* xq, const uint8_t* mask, const ffnk_routing_t* routing, int made, uint8_t* ws,
                const Room& room, int64_t M, int64_t K, hipStream_t stream, RoutedRows* out) {
  const bool reach = M * mx_code_stride(K) < k4g;
  if (xq && !reach) return api_fail(FFNK_E_SHAPE, "xq: 32-bit offsets do not reach %lld rows of %lld columns", (long long)M, (long long)K);
  if (int e = routing_room(routing, ws, M, &out->perm, &out->counts)) return e;
  const bool make = routing == nullptr || !made;
  int32_t *perm = const_cast<int32_t*>(out->perm), *counts = const_cast<int32_t*>(out->counts);
  if (make && (xq || !reach)) FFNK_TRY_HIP(launch_route(mask, (int)M, perm, counts, stream), "route kernel");
  out->gather = reach;
  if (xq) {
    out->A = rows_of(xq);
    return FFNK_OK;
  }
  MxQuantiseArgs q{x, x_stride_m, MX_BF16, reach ? nullptr : perm, room.codes, room.scales, (int)M, (int)K};
  if (make && reach) {
    q.mask = mask;
    q.part_perm = perm;
    q.part_counts = counts;
  }
  FFNK_TRY_HIP(launch_mx_quantise(q, stream), "quantise kernel");
  out->A = {room.codes, room.scales};
  return FFNK_OK;
}
// Paths without a partition leave the caller's all the same.
int leave_routing(const ffnk_routing_t* routing, int made, const uint8_t* mask, int64_t M, hipStream_t stream) {
  if (routing == nullptr || made) return FFNK_OK;
  if (!routing->perm || !routing->counts) return api_fail(FFNK_E_NULL, "routing: perm or counts is NULL");
  FFNK_TRY_HIP(launch_route(mask, (int)M, const_cast<int32_t*>(routing->perm), const_cast<int32_t*>(routing->counts), stream), "route kernel");
  return FFNK_OK;
}

// out[m] = A[m] W_grp^T on the tiled kernels, A in routed order or gathered.
int tiled_product(const Plan& plan, const MxRows& A, bool gather, const MxRows (&W)[2], const int32_t* perm, const int32_t* counts, uint16_t* out,
                  int64_t out_stride_m, int64_t M, int64_t K, int64_t N, float* P, hipStream_t stream) {
  MxGemmArgs g{};
  g.A = A; g.gather = gather;
  g.B0[0] = W[0]; g.B0[1] = W[1];
  g.C = out; g.ldc = out_stride_m;
  g.perm = perm; g.counts = counts;
  g.M = (int)M; g.N = (int)N; g.K = (int)K;
  g.splits = plan.splits; g.P = P;
  FFNK_TRY_HIP(launch_mx_gemm(plan.tile, g, stream), "MXFP4 GEMM");
  if (plan.splits > 1)
    FFNK_TRY_HIP(launch_routed_reduce(P, plan.splits, plan.splits, mx_tile_rows(plan.tile), (int)M, (int)N, counts, perm, out, out_stride_m, stream),
                 "reduce kernel");
  return FFNK_OK;
}

struct LinearRoom {
  Plan plan;
  size_t x, p, total;
};
LinearRoom linear_room(int64_t M, int64_t K, int64_t N) {
  LinearRoom r{};
  if (M <= kMxStreamRows) {
    r.total = tensor_bytes(M, K);
    return r;
  }
  r.plan = plan_gemm(false, M, N, K);
  r.x = routing_bytes(M);
  r.p = r.x + tensor_bytes(M, K);
  r.total = r.p + partial_bytes(r.plan, M, N);
  return r;
}
// ... of a call with these rows (x NULL: MXFP4 ones): none where a stream takes them as they are.
size_t linear_need(const LinearRoom& room, int64_t M, int64_t K, const uint16_t* x, int64_t x_stride_m) {
  return M <= kMxStreamRows && (x == nullptr || mx_stream_takes(M, K, x, x_stride_m)) ? 0 : room.total;
}
// `tiled`: on the tiled kernels whatever M is (a forward that keeps its pre-activations).
struct FfnRoom {
  Plan up, down;
  size_t x, h, p, total;
};
FfnRoom ffn_room(int64_t M, int64_t d, int64_t h, bool tiled) {
  FfnRoom r{};
  const bool stream = M <= kMxStreamFfnRows && !tiled;
  r.x = stream ? 0 : routing_bytes(M);
  r.h = r.x + tensor_bytes(M, d);
  r.p = r.h + tensor_bytes(M, h);
  r.total = r.p;
  if (!stream) {
    r.up = plan_gemm(true, M, h, d);
    r.down = plan_gemm(false, M, d, h);
    r.total += partial_bytes(r.down, M, d);
  }
  return r;
}

size_t weight_bytes(int64_t rows, int64_t columns) { return ws_align((size_t)rows * columns * 2); }

size_t linear_bwd_bytes(int64_t M, int64_t K, int64_t N) { return routing_bytes(M) + 2 * weight_bytes(N, K); }
size_t ffn_bwd_bytes(int64_t M, int64_t d, int64_t h) { return routing_bytes(M) + 6 * weight_bytes(h, d) + ffn_dx_bytes(M, d, h); }

// Both modalities' weights [rows, columns] as bf16 in `room`, where the modality has rows.
int dequantise_pair(const ffnk_mxfp4_t* v, const ffnk_mxfp4_t* t, int64_t rows, int64_t columns, const int32_t* counts, uint8_t* room,
                    const uint16_t* (&out)[2], hipStream_t stream) {
  uint8_t* second = room + weight_bytes(rows, columns);
  const MxDequantiseArgs a{{rows_of(v), rows_of(t)}, MX_BF16, {room, second}, columns, (int)rows, (int)columns, counts};
  FFNK_TRY_HIP(launch_mx_dequantise(a, stream), "dequantise kernel");
  out[0] = reinterpret_cast<const uint16_t*>(room);
  out[1] = reinterpret_cast<const uint16_t*>(second);
  return FFNK_OK;
}

int check_dx(const uint16_t* g, const uint8_t* mask, const uint16_t* dx, int64_t dx_stride_m, int64_t columns) {
  if (!g || !mask || !dx) return api_fail(FFNK_E_NULL, "g, mask or dx is NULL");
  if (dx_stride_m < columns || !aligned(dx, 2)) return api_fail(FFNK_E_STRIDE, "dx_stride_m=%lld < %lld, or dx not 2-byte aligned", (long long)dx_stride_m, (long long)columns);
  return FFNK_OK;
}

}  // namespace

extern "C" {

int ffnk_mxfp4_quantise(const void* x, int dtype, int64_t x_stride_m, const ffnk_mxfp4_t* out, int64_t rows, int64_t columns, void* stream) {
  if (int e = api_check_extents(rows, columns, 0)) return e;
  if (dtype < FFNK_DT_BF16 || dtype > FFNK_DT_FP32) return api_fail(FFNK_E_OP, "unknown dtype %d", dtype);
  if (rows == 0 || columns == 0) return FFNK_OK;
  if (!x) return api_fail(FFNK_E_NULL, "x is NULL");
  if (int e = check_tensor(out, "out")) return e;
  if (!aligned(x, element_size(dtype))) return api_fail(FFNK_E_ALIGN, "x not aligned to its elements");
  if (x_stride_m < columns) return api_fail(FFNK_E_STRIDE, "x_stride_m=%lld < columns=%lld", (long long)x_stride_m, (long long)columns);
  const MxQuantiseArgs a{x, x_stride_m, dtype, nullptr, const_cast<uint8_t*>(out->codes), const_cast<uint8_t*>(out->scales), (int)rows, (int)columns};
  FFNK_TRY_HIP(launch_mx_quantise(a, (hipStream_t)stream), "quantise kernel");
  return FFNK_OK;
}

int ffnk_mxfp4_dequantise(const ffnk_mxfp4_t* x, void* y, int dtype, int64_t y_stride_m, int64_t rows, int64_t columns, void* stream) {
  if (int e = api_check_extents(rows, columns, 0)) return e;
  if (dtype < FFNK_DT_BF16 || dtype > FFNK_DT_FP32) return api_fail(FFNK_E_OP, "unknown dtype %d", dtype);
  if (rows == 0 || columns == 0) return FFNK_OK;
  if (!y) return api_fail(FFNK_E_NULL, "y is NULL");
  if (int e = check_tensor(x, "x")) return e;
  if (!aligned(y, element_size(dtype))) return api_fail(FFNK_E_ALIGN, "y not aligned to its elements");
  if (y_stride_m < columns) return api_fail(FFNK_E_STRIDE, "y_stride_m=%lld < columns=%lld", (long long)y_stride_m, (long long)columns);
  const MxDequantiseArgs a{{rows_of(x), {nullptr, nullptr}}, dtype, {y, nullptr}, y_stride_m, (int)rows, (int)columns, nullptr};
  FFNK_TRY_HIP(launch_mx_dequantise(a, (hipStream_t)stream), "dequantise kernel");
  return FFNK_OK;
}

size_t ffnk_mxfp4_workspace_bytes(int op, int64_t M, int64_t K, int64_t N) {
  if (check_call(M, K, N)) return (size_t)-1;
  switch (op) {
    case FFNK_OP_LINEAR_FWD: return linear_room(M, K, N).total;
    case FFNK_OP_FFN_FWD: {  // either kind of forward
      const size_t plain = ffn_room(M, K, N, false).total, kept = ffn_room(M, K, N, true).total;
      return plain > kept ? plain : kept;
    }
    case FFNK_OP_LINEAR_BWD: return linear_bwd_bytes(M, K, N);
    case FFNK_OP_FFN_BWD: return ffn_bwd_bytes(M, K, N);
    default:
      api_fail(FFNK_E_OP, "no workspace for op %d", op);
      return (size_t)-1;
  }
}

size_t ffnk_mxfp4_workspace_bytes_linear_fwd(const uint16_t* x, int64_t x_stride_m, int64_t M, int64_t K, int64_t N) {
  return check_call(M, K, N) ? (size_t)-1 : linear_need(linear_room(M, K, N), M, K, x, x_stride_m);
}

int ffnk_mxfp4_linear_fwd(const uint16_t* x, int64_t x_stride_m, const ffnk_mxfp4_t* xq, const ffnk_mxfp4_t* Wv, const ffnk_mxfp4_t* Wt,
                          const uint8_t* mask, uint16_t* y, int64_t y_stride_m, int64_t M, int64_t K, int64_t N, void* ws, size_t ws_bytes,
                          void* stream_, const ffnk_routing_t* routing, int made) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int e = check_call(M, K, N)) return e;
  if (M == 0) return leave_routing(routing, made, mask, M, stream);
  if (int e = check_rows(x, x_stride_m, xq, K)) return e;
  if (int e = check_tensor(Wv, "Wv")) return e;
  if (int e = check_tensor(Wt, "Wt")) return e;
  if (!mask || !y) return api_fail(FFNK_E_NULL, "mask or y is NULL");
  if (!aligned(y, 2) || y_stride_m < N) return api_fail(FFNK_E_STRIDE, "y_stride_m=%lld < N=%lld, or y not 2-byte aligned", (long long)y_stride_m, (long long)N);
  const LinearRoom room = linear_room(M, K, N);
  if (int e = check_ws(ws, ws_bytes, linear_need(room, M, K, xq ? nullptr : x, x_stride_m))) return e;
  uint8_t* wsb = static_cast<uint8_t*>(ws);
  if (M <= kMxStreamRows) {
    if (int e = leave_routing(routing, made, mask, M, stream)) return e;
    MxStreamArgs a{};
    if (int e = stream_rows(x, x_stride_m, xq, carve_tensor(wsb, M, K), M, K, stream, &a)) return e;
    a.B0[0] = rows_of(Wv); a.B0[1] = rows_of(Wt);
    a.mask = mask; a.C = y; a.ldc = y_stride_m;
    a.M = (int)M; a.N = (int)N; a.K = (int)K;
    FFNK_TRY_HIP(launch_mx_stream(a, stream), "MXFP4 stream");
    return FFNK_OK;
  }
  RoutedRows r;
  if (int e = routed_rows(x, x_stride_m, xq, mask, routing, made, wsb, carve_tensor(wsb + room.x, M, K), M, K, stream, &r)) return e;
  const MxRows W[2] = {rows_of(Wv), rows_of(Wt)};
  return tiled_product(room.plan, r.A, r.gather, W, r.perm, r.counts, y, y_stride_m, M, K, N, reinterpret_cast<float*>(wsb + room.p), stream);
}

int ffnk_mxfp4_ffn_fwd(const uint16_t* x, int64_t x_stride_m, const ffnk_mxfp4_t* xq, const ffnk_mxfp4_t* W1, const ffnk_mxfp4_t* W2,
                       const ffnk_mxfp4_t* W3, const ffnk_mxfp4_t* U1, const ffnk_mxfp4_t* U2, const ffnk_mxfp4_t* U3, const uint8_t* mask,
                       uint16_t* out, int64_t out_stride_m, float* pre, int64_t M, int64_t d, int64_t h, void* ws, size_t ws_bytes, void* stream_,
                       const ffnk_routing_t* routing, int made) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int e = check_call(M, d, h)) return e;
  if (M == 0) return leave_routing(routing, made, mask, M, stream);
  if (int e = check_rows(x, x_stride_m, xq, d)) return e;
  const ffnk_mxfp4_t* weights[6] = {W1, W2, W3, U1, U2, U3};
  const char* names[6] = {"W1", "W2", "W3", "U1", "U2", "U3"};
  for (int i = 0; i < 6; ++i)
    if (int e = check_tensor(weights[i], names[i])) return e;
  if (!mask || !out) return api_fail(FFNK_E_NULL, "mask or out is NULL");
  if (!aligned(out, 2) || out_stride_m < d) return api_fail(FFNK_E_STRIDE, "out_stride_m=%lld < d=%lld, or out not 2-byte aligned", (long long)out_stride_m, (long long)d);
  if (!aligned(pre, 4)) return api_fail(FFNK_E_ALIGN, "pre not 4-byte aligned");
  const FfnRoom room = ffn_room(M, d, h, pre != nullptr);
  if (int e = check_ws(ws, ws_bytes, room.total)) return e;
  uint8_t* wsb = static_cast<uint8_t*>(ws);
  const Room hidden = carve_tensor(wsb + room.h, M, h);
  if (M <= kMxStreamFfnRows && !pre) {
    if (int e = leave_routing(routing, made, mask, M, stream)) return e;
    MxStreamArgs a{};
    if (int e = stream_rows(x, x_stride_m, xq, carve_tensor(wsb + room.x, M, d), M, d, stream, &a)) return e;
    a.B0[0] = rows_of(W1); a.B0[1] = rows_of(U1); a.B1[0] = rows_of(W3); a.B1[1] = rows_of(U3);
    a.mask = mask; a.H = hidden.codes; a.SH = hidden.scales;
    a.M = (int)M; a.N = (int)h; a.K = (int)d;
    FFNK_TRY_HIP(launch_mx_stream_swiglu(a, stream), "MXFP4 SwiGLU stream");
    MxStreamArgs b{};
    b.A = {hidden.codes, hidden.scales};
    b.B0[0] = rows_of(W2); b.B0[1] = rows_of(U2);
    b.mask = mask; b.C = out; b.ldc = out_stride_m;
    b.M = (int)M; b.N = (int)d; b.K = (int)h;
    FFNK_TRY_HIP(launch_mx_stream(b, stream), "MXFP4 stream");
    return FFNK_OK;
  }
  RoutedRows r;
  if (int e = routed_rows(x, x_stride_m, xq, mask, routing, made, wsb, carve_tensor(wsb + room.x, M, d), M, d, stream, &r)) return e;
  MxGemmArgs g{};
  g.A = r.A; g.gather = r.gather;
  g.B0[0] = rows_of(W1); g.B0[1] = rows_of(U1); g.B1[0] = rows_of(W3); g.B1[1] = rows_of(U3);
  g.H = hidden.codes; g.SH = hidden.scales;
  g.pre = pre; g.ld_pre = 2 * h;
  g.perm = r.perm; g.counts = r.counts;
  g.M = (int)M; g.N = (int)h; g.K = (int)d;
  g.splits = 1;
  FFNK_TRY_HIP(launch_mx_swiglu_gemm(room.up.tile, g, stream), "MXFP4 SwiGLU GEMM");
  const MxRows W[2] = {rows_of(W2), rows_of(U2)};
  return tiled_product(room.down, {hidden.codes, hidden.scales}, false, W, r.perm, r.counts, out, out_stride_m, M, h, d,
                       reinterpret_cast<float*>(wsb + room.p), stream);
}

int ffnk_mxfp4_linear_bwd(const uint16_t* g, int64_t g_stride_m, const ffnk_mxfp4_t* Wv, const ffnk_mxfp4_t* Wt, const uint8_t* mask, uint16_t* dx,
                          int64_t dx_stride_m, int64_t M, int64_t K, int64_t N, void* ws, size_t ws_bytes, void* stream_, const ffnk_routing_t* routing) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int e = check_call(M, K, N)) return e;
  if (M == 0) return FFNK_OK;
  if (int e = check_dx(g, mask, dx, dx_stride_m, K)) return e;
  if (int e = check_tensor(Wv, "Wv")) return e;
  if (int e = check_tensor(Wt, "Wt")) return e;
  if (g_stride_m % 8 != 0 || g_stride_m < N || !aligned(g, 16) || !linear_dx_ok(M, K, N, g_stride_m))
    return api_fail(FFNK_E_STRIDE, "MXFP4 linear backward: K and N must be multiples of 8, N a multiple of 64 or at least 128, and the rows of g 16-byte "
                                   "aligned and within 32-bit offsets");
  if (int e = check_ws(ws, ws_bytes, linear_bwd_bytes(M, K, N))) return e;
  uint8_t* wsb = static_cast<uint8_t*>(ws);
  const int32_t *perm, *counts;
  if (int e = make_routing(routing, wsb, mask, M, stream, &perm, &counts)) return e;
  const uint16_t* W[2];
  if (int e = dequantise_pair(Wv, Wt, N, K, counts, wsb + routing_bytes(M), W, stream)) return e;
  return linear_dx(g, g_stride_m, W, perm, counts, dx, dx_stride_m, M, K, N, stream);
}

int ffnk_mxfp4_ffn_bwd(const uint16_t* g, int64_t g_stride_m, const ffnk_mxfp4_t* W1, const ffnk_mxfp4_t* W2, const ffnk_mxfp4_t* W3,
                       const ffnk_mxfp4_t* U1, const ffnk_mxfp4_t* U2, const ffnk_mxfp4_t* U3, const uint8_t* mask, const float* pre, uint16_t* dx,
                       int64_t dx_stride_m, int64_t M, int64_t d, int64_t h, void* ws, size_t ws_bytes, void* stream_, const ffnk_routing_t* routing) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int e = check_call(M, d, h)) return e;
  if (M == 0) return FFNK_OK;
  if (int e = check_dx(g, mask, dx, dx_stride_m, d)) return e;
  const ffnk_mxfp4_t* weights[6] = {W1, W2, W3, U1, U2, U3};
  const char* names[6] = {"W1", "W2", "W3", "U1", "U2", "U3"};
  for (int i = 0; i < 6; ++i)
    if (int e = check_tensor(weights[i], names[i])) return e;
  if (!pre) return api_fail(FFNK_E_NULL, "pre is NULL");
  if (g_stride_m % 8 != 0 || g_stride_m < d || !aligned(g, 16) || !aligned(pre, 16) || !ffn_dx_ok(M, d, h, g_stride_m))
    return api_fail(FFNK_E_STRIDE, "MXFP4 FFN backward: d and h must be multiples of 8, d a multiple of 64 or at least 128, and the rows of g 16-byte "
                                   "aligned and within 32-bit offsets");
  if (int e = check_ws(ws, ws_bytes, ffn_bwd_bytes(M, d, h))) return e;
  uint8_t* wsb = static_cast<uint8_t*>(ws);
  const int32_t *perm, *counts;
  if (int e = make_routing(routing, wsb, mask, M, stream, &perm, &counts)) return e;
  uint8_t* at = wsb + routing_bytes(M);
  const size_t pair = 2 * weight_bytes(h, d);
  const uint16_t *w1[2], *w2[2], *w3[2];
  if (int e = dequantise_pair(W2, U2, d, h, counts, at, w2, stream)) return e;
  if (int e = dequantise_pair(W1, U1, h, d, counts, at + pair, w1, stream)) return e;
  if (int e = dequantise_pair(W3, U3, h, d, counts, at + 2 * pair, w3, stream)) return e;
  return ffn_dx(g, g_stride_m, pre, w1, w3, w2, perm, counts, dx, dx_stride_m, M, d, h, at + 3 * pair, stream);
}

}  // extern "C"
