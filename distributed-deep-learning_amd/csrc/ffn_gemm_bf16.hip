// bf16 instantiations of the feed-forward products (v_mfma_f32_16x16x32_bf16)
#include "ffn_gemm.h"

namespace ddl {
namespace ffn {
void launch_gemm_bf16(const GemmArgs& a, int cfg, hipStream_t s) {
  if (cfg == 0) run_cfg<__bf16, 128, 32, 2, 1>(a, s);
  else if (cfg == 1) run_cfg<__bf16, 128, 128, 2, 2>(a, s);
  else run_big<__bf16>(a, s);
}
}  // namespace ffn
}  // namespace ddl
