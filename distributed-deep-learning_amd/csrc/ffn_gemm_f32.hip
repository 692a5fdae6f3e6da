// fp32 instantiations of the feed-forward products (v_mfma_f32_16x16x4_f32: exact fp32, 1/16 of the bf16 rate).  No 256 x 256
// tile: the fp32 MFMA takes eight times as long per LDS byte, so the 128 x 128 tile already keeps it fed.
#include "ffn_gemm.h"

namespace ddl {
namespace ffn {
void launch_gemm_f32(const GemmArgs& a, int cfg, hipStream_t s) { run_small<float>(a, cfg, s); }
}  // namespace ffn
}  // namespace ddl
