// Instantiations and launcher of the attention mass (serve_mass.cuh).
#include "launch.h"
#include "serve_mass.cuh"

namespace tttj {

namespace {
template <int HD, bool BF16>
cudaError_t launch(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const MassParams& p, int grid,
                   cudaStream_t stream) {
  auto kern = mass_kernel<HD, BF16>;
  const int smem = MassSmem<HD>::FIXED + p.s.batch * ((int)sizeof(SrvSeq) + 8) + 4;
  // The most that any call needs, for every call: the limit is the kernel's, and a call of another
  // thread must not lower it between here and the launch.
  constexpr int most = MassSmem<HD>::FIXED + SRV_MAX_BATCH * ((int)sizeof(SrvSeq) + 8) + 4;
  static_assert(most <= 232448, "shared memory exceeds the 227 KB per-CTA limit");
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(grid), dim3(MASS_THREADS), smem, stream, tm_q, tm_k, p);
}
}  // namespace

cudaError_t mass_launch(const CUtensorMap& q, const CUtensorMap& k, const MassParams& p, int head_dim, int bf16,
                        int grid, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return bf16 ? launch<32, true>(q, k, p, grid, stream) : launch<32, false>(q, k, p, grid, stream);
    case 64: return bf16 ? launch<64, true>(q, k, p, grid, stream) : launch<64, false>(q, k, p, grid, stream);
    case 128: return bf16 ? launch<128, true>(q, k, p, grid, stream) : launch<128, false>(q, k, p, grid, stream);
    case 256: return bf16 ? launch<256, true>(q, k, p, grid, stream) : launch<256, false>(q, k, p, grid, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tttj
