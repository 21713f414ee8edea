// Instantiations and launcher of the tile attention (serve_tile.cuh).
#include "launch.h"
#include "serve_tile.cuh"

namespace tttj {

namespace {
template <int HD, bool BF16>
cudaError_t launch(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const TileParams& p,
                   int grid, cudaStream_t stream) {
  auto kern = tile_kernel<HD, BF16>;
  constexpr int smem = TileSmem<HD>::ALL;
  static_assert(smem <= 232448, "shared memory exceeds the 227 KB per-CTA limit");
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(tile_plan_kernel, dim3(1), dim3(TILE_PLAN_THREADS), 0, stream, p, tile_nt(HD), grid);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kern, dim3(grid), dim3(TileSmem<HD>::THREADS), smem, stream, tm_q, tm_k, tm_v, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(tile_join_kernel<HD, BF16>, dim3(8 * grid), dim3(32 * TILE_JOIN_WARPS), 0, stream, p);
}
}  // namespace

cudaError_t tile_launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileParams& p,
                        int head_dim, int bf16, int grid, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return bf16 ? launch<32, true>(q, k, v, p, grid, stream) : launch<32, false>(q, k, v, p, grid, stream);
    case 64: return bf16 ? launch<64, true>(q, k, v, p, grid, stream) : launch<64, false>(q, k, v, p, grid, stream);
    case 128: return bf16 ? launch<128, true>(q, k, v, p, grid, stream) : launch<128, false>(q, k, v, p, grid, stream);
    case 256: return bf16 ? launch<256, true>(q, k, v, p, grid, stream) : launch<256, false>(q, k, v, p, grid, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tttj
