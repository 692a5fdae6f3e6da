// Launchers of dropout and of the residual / norm kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace ddl {
namespace ffn {

struct DropoutArgs {
  const void* x = nullptr;
  const void* residual = nullptr;
  void* y = nullptr;
  long n = 0;
  const int64_t* key = nullptr;          // device: (seed, call)
  double p = 0.;
};
void launch_dropout(int dtype, const DropoutArgs& a, hipStream_t s);
void launch_rng_keys(int64_t* state /*[2]*/, int64_t* keys /*[n][2]*/, int n, hipStream_t s);

// r = x + scale * gate * post(y);  h = pre(r)
enum GateKind : int { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_FULL = 2 };
struct NormArgs {
  int M = 0, C = 0;
  bool layer = false;                    // layer norm (mean and variance) or RMS norm
  float eps = 1e-6f, scale = 1.f;
  bool post = false, pre = false;        // which norms there are
  int gate_kind = GATE_NONE;
  bool param_f32 = false;                // weights, biases and a channel gate in fp32 beside 16-bit rows
  bool vec = false;                      // C a multiple of 16 bytes, every row 16-byte aligned
  const void *x = nullptr, *y = nullptr, *gate = nullptr;      // y null: r = x
  const void *post_w = nullptr, *post_b = nullptr, *pre_w = nullptr, *pre_b = nullptr;
  void *r = nullptr, *h = nullptr;
  float* stats = nullptr;                // [4][M]: post mean, post rstd, pre mean, pre rstd (null: not kept)
  // backward
  const void *dr = nullptr, *dh = nullptr;                     // either may be null (zero)
  void *dx = nullptr, *dy = nullptr, *dgate = nullptr;         // dgate: full gates only
  float* part = nullptr;                 // [groups][5][C]: dgate, dpost_w, dpost_b, dpre_w, dpre_b
  float* means = nullptr;                // [2][M], wide rows with `part`: what the rows' pass leaves for the columns' pass
  int groups = 0;
};
constexpr int NORM_MAX_C = 16384;
int norm_bwd_groups(int M, int C);
bool norm_bwd_wants_means(int C);
void launch_norm_fwd(int dtype, const NormArgs& a, hipStream_t s);
void launch_norm_bwd(int dtype, const NormArgs& a, hipStream_t s);

}  // namespace ffn
}  // namespace ddl
