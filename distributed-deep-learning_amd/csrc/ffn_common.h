// Shared by the feed-forward operators (ffn_*.hip): element types, activations and their derivatives, the argument
// structs of the launchers and the epilogue of the matrix products.
//
// Element types T: __bf16, _Float16, float.  Every sum, activation and norm runs in fp32; a value is rounded to T once,
// where it is stored.
#pragma once
#include <hip/hip_runtime.h>
#include <cfloat>
#include <cmath>
#include <cstdint>

namespace ddl {
namespace ffn {

// ---- activations: act(z) and act'(z) ---------------------------------------------------------------------------------
enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SIGMOID = 5 };
constexpr int N_ACT = 6;
enum DType : int { F32 = 0, BF16 = 1, F16 = 2 };
inline int esize(int dtype) { return dtype == F32 ? 4 : 2; }

// 1 / (1 + e^-z): e^-z overflows to infinity below -88, and the quotient is then the right limit, zero
__device__ __forceinline__ float sigmoid_f(float z) { return 1.0f / (1.0f + expf(-z)); }

// gelu_tanh uses 0.5 (1 + tanh(v)) = sigmoid(2 v)
__device__ __forceinline__ float gelu_tanh_arg(float z) { return 1.5957691216057308f * (z + 0.044715f * z * z * z); }

__device__ __forceinline__ float act_fwd(int act, float z) {
  switch (act) {
    case ACT_RELU: return z < 0.f ? 0.f : z;             // a NaN passes
    case ACT_SILU: return z * sigmoid_f(z);
    case ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case ACT_GELU_TANH: return z * sigmoid_f(gelu_tanh_arg(z));
    case ACT_SIGMOID: return sigmoid_f(z);
    default: return z;
  }
}

// derivative; also returns act(z) for the gated block
__device__ __forceinline__ float act_grad(int act, float z, float& a) {
  switch (act) {
    case ACT_RELU: a = z < 0.f ? 0.f : z; return z <= 0.f ? 0.f : 1.f;
    case ACT_SILU: {
      const float s = sigmoid_f(z);
      a = z * s;
      return s * (1.0f + z * (1.0f - s));
    }
    case ACT_GELU: {
      const float cdf = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
      a = z * cdf;
      return cdf + z * 0.3989422804014327f * expf(-0.5f * z * z);
    }
    case ACT_GELU_TANH: {
      const float s = sigmoid_f(gelu_tanh_arg(z));
      a = z * s;
      // beyond 12 s is 0 or 1, and the second term nothing: from 2e19 on its square would be infinite (a NaN stays one)
      const float c = z > 12.f ? 12.f : z < -12.f ? -12.f : z;
      return s + c * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * c * c);
    }
    case ACT_SIGMOID: a = sigmoid_f(z); return a * (1.0f - a);
    default: a = z; return 1.f;
  }
}

// ---- loads / stores with conversion ----------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }    // round to nearest even

template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack { T v[N]; };

// N consecutive values at an address that is aligned to min(16, N * sizeof(T)) bytes
template <typename T, int N> __device__ __forceinline__ void load_vec(const T* p, float* out) {
  const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_f(x.v[i]);
}
template <typename T, int N> __device__ __forceinline__ void store_vec(T* p, const float* in) {
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = from_f<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = x;
}
// n <= N valid values; `vec`: the address is aligned as above and all N are valid
template <typename T, int N> __device__ __forceinline__ void load_some(const T* p, float* out, int n, bool vec) {
  if (vec) { load_vec<T, N>(p, out); return; }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = i < n ? to_f(p[i]) : 0.f;
}
template <typename T, int N> __device__ __forceinline__ void store_some(T* p, const float* in, int n, bool vec) {
  if (vec) { store_vec<T, N>(p, in); return; }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) p[i] = from_f<T>(in[i]);
}

// ---- epilogue of a product: what becomes of the fp32 sums ------------------------------------------------------------
//   single:  z = sum + bias0;             out = act(z) + residual            (z kept in fp32 where training needs it)
//   dual:    g = sum0 + bias0, u = sum1 + bias1;  out = act(g) * u           (g, u kept likewise)
struct Epilogue {
  void* out[2] = {nullptr, nullptr};      // [1]: second output of a product with two (weight gradients of a gated block)
  long ldo = 0;
  const void* bias[2] = {nullptr, nullptr};
  const void* residual = nullptr;
  long ldr = 0;
  float* z[2] = {nullptr, nullptr};
  long ldz = 0;
  int act = ACT_NONE;
  bool out_vec = false, res_vec = false, bias_vec = false;   // rows start 16-byte aligned
  const float* scale = nullptr;           // fp16 gradients: the power of two that dz is held in (device; see act_bwd_rescale_kernel)
};

// act over V values; one switch for all of them
template <int V> __device__ __forceinline__ void act_fwd_all(int act, float* v) {
#define DDL_ACT_CASE(A)                                   \
  case A:                                                 \
    _Pragma("unroll") for (int i = 0; i < V; ++i) v[i] = act_fwd(A, v[i]); \
    break;
  switch (act) {
    DDL_ACT_CASE(ACT_RELU)
    DDL_ACT_CASE(ACT_SILU)
    DDL_ACT_CASE(ACT_GELU)
    DDL_ACT_CASE(ACT_GELU_TANH)
    DDL_ACT_CASE(ACT_SIGMOID)
    default: break;
  }
#undef DDL_ACT_CASE
}

// bias of the columns n .. n+V-1 (zeros where there is none)
template <typename T, int V> __device__ __forceinline__ void load_bias(const Epilogue& e, int which, int n, int N, bool aligned, float* b) {
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = 0.f;
  if (e.bias[which] != nullptr && n < N) load_some<T, V>((const T*)e.bias[which] + n, b, N - n, N - n >= V && aligned && e.bias_vec);
}

// V consecutive outputs (row m, columns n .. n+V-1); v: the sums, w: the second product's (dual only); b0, b1: their biases.
// z rows are padded to 16 values, so z is stored in whole vectors where n is `aligned` (to the vector).  PLAIN: neither bias, activation nor residual.
template <typename T, bool DUAL, bool PLAIN, int V>
__device__ __forceinline__ void epilogue_store(const Epilogue& e, int which, long m, int n, int N, bool aligned, float* v, float* w,
                                               const float* b0, const float* b1) {
  const int left = N - n;
  if (left <= 0) return;
  const bool full = left >= V && aligned;
  if (!PLAIN) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += b0[i];
    if (DUAL) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] += b1[i];
    }
    if (e.z[0] != nullptr) {
      store_some<float, V>(e.z[0] + m * e.ldz + n, v, left, aligned);
      if (DUAL) store_some<float, V>(e.z[1] + m * e.ldz + n, w, left, aligned);
    }
    act_fwd_all<V>(e.act, v);
    if (DUAL) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= w[i];
    } else if (e.residual != nullptr) {
      float r[V];
      load_some<T, V>((const T*)e.residual + m * e.ldr + n, r, left, full && e.res_vec);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += r[i];
    }
  }
  store_some<T, V>((T*)e.out[which] + m * e.ldo + n, v, left, full && e.out_vec);
}

// ---- a product --------------------------------------------------------------------------------------------------------
//   out[m][n] = epilogue( sum over segments s, k of P_s(n, k) * Q_s(m, k) )
// P's direction n is contiguous in the output.  An operand is k-contiguous (element (r, k) at r * ld + k) or
// k-strided (at k * ld + r).  All vector accesses are 16 bytes: bases aligned, ld and the contiguous extent multiples of
// 16 bytes (`pack` brings other operands into that form).
struct GemmArgs {
  const void* p[2] = {nullptr, nullptr};  // dual: gate and up; nseg = 2: the operand of each contraction segment
  const void* q[2] = {nullptr, nullptr};  // nseg = 2: of each segment; nout = 2: of each output
  long ldp[2] = {0, 0}, ldq[2] = {0, 0};
  int N = 0, M = 0, K = 0;                // K: contraction length of ONE segment
  int nseg = 1, nout = 1;
  bool p_kc = true, q_kc = true, dual = false;
  bool halves = false;                    // outputs m and m + M / 2 are one output's sums: joined (M / 2 rows of out)
  float* partial = nullptr;               // split contraction: [splits][nout * (1 + dual)][M][ldw] sums instead of out
  long ldw = 0;
  int splits = 1;
  Epilogue ep;
};
enum Tile : int { TILE_128x32 = 0, TILE_64x32 = 1, TILE_64x64 = 2, TILE_128x128 = 3, TILE_256x128 = 4, TILE_256x256 = 5, N_TILES = 6 };
// Tile (rows and columns of the output) and split of a launch; partial_floats: the floats `partial` needs with that split (0: none)
struct GemmPlan { int cfg = 0, splits = 1, bm = 0, bn = 0; long ldw = 0; long partial_floats = 0; };
GemmPlan gemm_plan(int dtype, const GemmArgs& a);                                   // bm == 0: no tile fits a launch
void launch_gemm(int dtype, GemmArgs a, const GemmPlan& plan, hipStream_t s);      // + the joining launch if split
void launch_gemm_f32(const GemmArgs& a, int cfg, hipStream_t s);
void launch_gemm_bf16(const GemmArgs& a, int cfg, hipStream_t s);
void launch_gemm_f16(const GemmArgs& a, int cfg, hipStream_t s);

// few rows: weights streamed once from memory into the matrix-core operands, no LDS staging
struct FewRowsArgs {
  const void* w[2] = {nullptr, nullptr};
  const void* x = nullptr;
  long ldw[2] = {0, 0}, ldx = 0;
  int N = 0, M = 0, K = 0;
  bool dual = false, vec = true;
  Epilogue ep;
};
constexpr int FEW_ROWS = 32;
void launch_few_rows(int dtype, const FewRowsArgs& a, hipStream_t s);

// ---- pointwise companions (ffn_pointwise.hip) --------------------------------------------------------------------------
// dst [rows][ld] = src with any strides, columns from `cols` on zero
struct PackItem { const void* src = nullptr; void* dst = nullptr; long s_row = 0, s_col = 0, ld = 0, rows = 0; int cols = 0; };
struct PackArgs { PackItem item[4]; int count = 0; };
void launch_pack(int dtype, const PackArgs& a, hipStream_t s);
void launch_join(int dtype, const float* partial, const GemmArgs& a, hipStream_t s);
struct ActBwdArgs {
  const void* dy = nullptr;
  long ldy = 0;                           // rows contiguous, any alignment (dy_vec says 16-byte)
  bool dy_vec = false;
  const float* z[2] = {nullptr, nullptr}; // linear: z; dual: g, u.  null: dz = dy (column sums only)
  long ldz = 0;
  void* dz[2] = {nullptr, nullptr};       // padded rows; may be null where only the column sums are wanted
  long ldd = 0;
  bool two = false;                       // dz in two parts: rounded, and what that lacks in rows M ..
  float* range = nullptr;                 // fp16 with dz: [act_bwd_tiles] largest finite |dz| of each workgroup
  float* scale = nullptr;                 // fp16 with dz: the power of two that dz is held in
  int act = ACT_NONE;
  bool dual = false;
  int M = 0, N = 0;
  float* part = nullptr;                  // [chunks][1 + dual][N] column sums of dz, null: none
  void* db[2] = {nullptr, nullptr};       // instead, with one chunk: the column sums themselves, in the element type
  int chunks = 0;
};
// few rows: out[which][n][k] = sum over m of dz[which][m][n] x[m][k], rows of K; two: dz in two parts (see above)
struct OuterArgs {
  const void* dz[2] = {nullptr, nullptr};
  const void* x = nullptr;
  void* out[2] = {nullptr, nullptr};
  long ldd = 0, ldx = 0;
  int M = 0, N = 0, K = 0, nout = 1;
  int rows = 0, strips = 0;               // of the output: rows a workgroup writes, strips of 1024 columns (the launcher's)
  bool two = false, x_vec = false, out_vec = false;
  const float* scale = nullptr;           // of dz (fp16), null: 1
};
void launch_outer(int dtype, const OuterArgs& a, hipStream_t s);
int act_bwd_chunks(int dtype, int M, int N);
int act_bwd_tiles(int dtype, const ActBwdArgs& a);         // workgroups of the launch
void launch_act_bwd(int dtype, const ActBwdArgs& a, hipStream_t s);
// out[which][n] = sum over chunks of part[chunk][which][n]
void launch_colsum(int out_dtype, const float* part, int chunks, int nvec, long n, void* const* out, hipStream_t s);

}  // namespace ffn
}  // namespace ddl
