// dH GEMM of the feed-forward backward over weights that are constant: from fp32 pre-activations, without the intermediate.
#include "gemm_tiles.hpp"

namespace ffnk {

namespace {
struct Tiles {
  using K = KMajorTiles<true, false>;
  using T0 = Pre32<K::T0>;
  using T1 = T0;  // (the four-wave tile has no registers left for the epilogue)
  using T2 = Pre32<K::T2>;
  using T3 = Pre32<K::T3>;
  using T4 = Pre32<K::T4>;
  using T6 = Pre32<K::T6>;
  using T7 = Pre32<K::T7>;
};
}  // namespace

hipError_t launch_gather_gemm_kmajor32(int tile, const GemmArgs& g, hipStream_t stream) { return dispatch_tile_with_tail<Tiles>(tile, g, stream); }

}  // namespace ffnk
