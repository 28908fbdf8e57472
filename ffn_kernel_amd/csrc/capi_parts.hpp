// What capi.hip shares with the other files of the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ffnk.h"

namespace ffnk {

// Set the calling thread's ffnk_last_error() text; return the code.
int api_fail(int code, const char* fmt, ...);
int api_hip_fail(hipError_t e, const char* what);
int api_check_extents(int64_t M, int64_t K, int64_t N);

#define FFNK_TRY_HIP(expr, what)                              \
  do {                                                        \
    hipError_t e__ = (expr);                                  \
    if (e__ != hipSuccess) return ::ffnk::api_hip_fail(e__, what); \
  } while (0)

// The partition a call works with: the caller's, or one made in `ws`, which holds routing_bytes(M).
size_t routing_bytes(int64_t M);
int routing_room(const ffnk_routing_t* caller, uint8_t* ws, int64_t M, const int32_t** perm, const int32_t** counts);  // made or not
int make_routing(const ffnk_routing_t* caller, uint8_t* ws, const uint8_t* mask, int64_t M, hipStream_t stream, const int32_t** perm,
                 const int32_t** counts);

// Gradients of a routed layer's rows alone, over bf16 weights as nn.Linear holds them ([out, in] rows without gaps, 16-byte aligned);
// g: [M, out] rows.  Both are the dx GEMMs of the layers' backward.
//   linear: dx[m] = g[m] W_grp
//   ffn:    dh = g W2_grp; (dt1 | dt3) = dh * the SwiGLU derivative at `pre` (gate | up, rows in routed order); dx = dt1 W1_grp + dt3 W3_grp
bool linear_dx_ok(int64_t M, int64_t K, int64_t N, int64_t g_stride_m);
int linear_dx(const uint16_t* g, int64_t g_stride_m, const uint16_t* const (&W)[2], const int32_t* perm, const int32_t* counts, uint16_t* dx,
              int64_t dx_stride_m, int64_t M, int64_t K, int64_t N, hipStream_t stream);
bool ffn_dx_ok(int64_t M, int64_t d, int64_t h, int64_t g_stride_m);
size_t ffn_dx_bytes(int64_t M, int64_t d, int64_t h);
int ffn_dx(const uint16_t* g, int64_t g_stride_m, const float* pre, const uint16_t* const (&W1)[2], const uint16_t* const (&W3)[2],
           const uint16_t* const (&W2)[2], const int32_t* perm, const int32_t* counts, uint16_t* dx, int64_t dx_stride_m, int64_t M, int64_t d, int64_t h,
           uint8_t* ws, hipStream_t stream);

}  // namespace ffnk
