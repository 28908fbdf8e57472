// Row partition by modality: mask[M] -> perm[M] (visual rows first, each group in ascending
// row order) and counts[2].  The reference tests mask rows inside every GEMM tile
// (ffn_kernel/linear.py:120-149); here the same row -> weight assignment is made once,
// as an integer permutation, so that GEMM tiles never mix modalities.
//
// One launch, no inter-block dependency: every block re-counts the visual rows that
// precede its rows (and the total) straight from the mask, which is at most M bytes of
// L2-resident reads per block, then places its own rows, 1024 at a time.  The launch has at most
// kRouteMaxBlocks blocks (each takes more 1024-row chunks instead), so the counting reads stay
// linear in M: kRouteMaxBlocks * M bytes.
#include "common.hpp"
#include "launch.hpp"
#include "route_block.hpp"

namespace ffnk {

__global__ __launch_bounds__(kRouteThreads) void route_kernel(const uint8_t* __restrict__ mask, int M,
                                                               int32_t* __restrict__ perm,
                                                               int32_t* __restrict__ counts, int chunks_per_block) {
  route_block(mask, M, perm, counts, chunks_per_block, blockIdx.x);
}

hipError_t launch_route(const uint8_t* mask, int M, int32_t* perm, int32_t* counts, hipStream_t stream) {
  const RouteShape r = route_shape(M);
  hipLaunchKernelGGL(route_kernel, dim3(r.blocks), dim3(kRouteThreads), 0, stream, mask, M, perm, counts, r.chunks_per_block);
  return hipGetLastError();
}

}  // namespace ffnk
