// bf16 instantiations of the feed-forward products (v_mfma_f32_16x16x32_bf16)
#include "ffn_gemm.h"

namespace ddl {
namespace ffn {
void launch_gemm_bf16(const GemmArgs& a, int cfg, hipStream_t s) {
  if (cfg == TILE_256x256) run_big<__bf16, 256, 256, 4, 2, 2>(a, s);
  else if (cfg == TILE_256x128) run_big<__bf16, 256, 128, 4, 2, 3>(a, s);
  else run_small<__bf16>(a, cfg, s);
}
}  // namespace ffn
}  // namespace ddl
