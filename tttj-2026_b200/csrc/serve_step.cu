// Instantiations and launcher of the few-row attention (serve_step.cuh).
#include "launch.h"
#include "serve_step.cuh"

namespace tttj {

namespace {
template <int HD, bool BF16>
cudaError_t launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const StepParams& p, int grid,
                   cudaStream_t stream) {
  const int prefix = (p.s.batch + 1) * (int)sizeof(long);
  const int smem = StepSmem<HD>::FIXED + prefix;
  auto kern = step_kernel<HD, BF16>;
  // The limit is the kernel's, not the launch's: set to the most that any call needs, so that a
  // call of another thread does not lower it between here and the launch.
  constexpr int most = StepSmem<HD>::FIXED + (SRV_MAX_BATCH + 1) * (int)sizeof(long);
  static_assert(most <= 232448, "shared memory exceeds the 227 KB per-CTA limit");
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kern, dim3(grid), dim3(STEP_THREADS), smem, stream, tm_k, tm_v, p);
  if (e != cudaSuccess) return e;
  const long rows = (long)p.s.tokens * p.heads;
  const int blocks = (int)((rows + STEP_JOIN_WARPS - 1) / STEP_JOIN_WARPS);
  return launch_pdl(step_join_kernel<HD, BF16>, dim3(blocks), dim3(32 * STEP_JOIN_WARPS), prefix, stream,
                    p, grid);
}
}  // namespace

cudaError_t step_launch(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const StepParams& p,
                        int head_dim, int bf16, int grid, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return bf16 ? launch<32, true>(tm_k, tm_v, p, grid, stream) : launch<32, false>(tm_k, tm_v, p, grid, stream);
    case 64: return bf16 ? launch<64, true>(tm_k, tm_v, p, grid, stream) : launch<64, false>(tm_k, tm_v, p, grid, stream);
    case 128: return bf16 ? launch<128, true>(tm_k, tm_v, p, grid, stream) : launch<128, false>(tm_k, tm_v, p, grid, stream);
    case 256: return bf16 ? launch<256, true>(tm_k, tm_v, p, grid, stream) : launch<256, false>(tm_k, tm_v, p, grid, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tttj
