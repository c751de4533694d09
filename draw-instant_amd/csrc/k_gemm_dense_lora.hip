// k_gemm instantiations: dense A with low-rank adapters beside the product.
#include "k_gemm_families.h"
#include "k_gemm_kernel.h"

namespace di {

void gemm_fast_lora(const GemmArgs& g, int tile_cfg, hipStream_t s) {
  launch_fast_d<A_DENSE, 2, EX_LORA>(g, tile_cfg, s);
}

void gemm_slow_lora(const GemmArgs& g, int elem, int tile_cfg, hipStream_t s) {
  if (elem == DI_F32) launch_slow<float, A_DENSE, B_NK, float, EX_LORA>(g, tile_cfg, s);
  else launch_slow<f16, A_DENSE, B_NK, f16, EX_LORA>(g, tile_cfg, s);
}

}  // namespace di
