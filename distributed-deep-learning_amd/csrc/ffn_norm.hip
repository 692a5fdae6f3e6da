// Residual join between two blocks with the norms on both sides of it:
//     n = post(y),  r = x + scale * gate * n,  h = pre(r)          (layer or RMS norm; either norm may be absent)
//
// Bound by memory: x and y are read once, r and h written once.  A row lives in the registers of one wave (up to 1024
// columns) or one workgroup, so the mean, the variance about the mean and the normalised values all come from one read.
// Statistics, sums and the joined row stay in fp32; h is taken from the unrounded r.
//
// Backward: r is computed again from x and y (reading it instead would cost the same bytes and bring its rounding into the
// weights' gradients).  With d = dh * w_pre:  dr' = dr + rstd (d - mean(d) - rhat mean(d rhat));  dx = dr';
// dn = scale * gate * dr';  dy the same formula for the post norm;  the vectors' gradients are sums over rows: workgroups
// stride over the rows, keep their columns' sums in registers and write one row of partials each (`launch_colsum` adds them
// in order).
#include "ffn_common.h"
#include "ffn_misc.h"
#include "ddl_kernels.h"
#include <type_traits>

namespace ddl {
namespace ffn {
namespace {

// The EL elements of a row that a thread holds: VEC: 16-byte chunks t, t + TPR, ...; otherwise single elements.
template <typename T, int TPR, int EL, bool VEC> struct Row {
  static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, NV = EL / V;
  static __device__ __forceinline__ int col(int t, int j) { return (j * TPR + t) * V; }
  template <typename S> static __device__ __forceinline__ void load(const S* p, int t, int C, float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col(t, j);
      if (c < C) {
        load_vec<S, V>(p + c, o + j * V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[j * V + e] = 0.f;
      }
    }
  }
  template <typename S> static __device__ __forceinline__ void store(S* p, int t, int C, const float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col(t, j);
      if (c < C) store_vec<S, V>(p + c, o + j * V);
    }
  }
  static __device__ __forceinline__ bool in(int t, int e, int C) { return col(t, e / V) < C; }   // C % V == 0
  // a parameter vector (fp32 or T); null: the constant
  static __device__ __forceinline__ void param(const void* p, bool f32, float none, int t, int C, float (&o)[EL]) {
    if (p == nullptr) {
#pragma unroll
      for (int e = 0; e < EL; ++e) o[e] = none;
    } else if (f32) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = col(t, j);
#pragma unroll
        for (int e = 0; e < V; ++e) o[j * V + e] = c < C ? ((const float*)p)[c + e] : 0.f;
      }
    } else {
      load<T>((const T*)p, t, C, o);
    }
  }
};

// sums of two values over the TPR threads of a row; every thread gets them
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float (*red)[2]) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
  if (TPR > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();                                       // the previous sums have been read
    if ((threadIdx.x & 63) == 0) { red[w][0] = a; red[w][1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) { a += red[i][0]; b += red[i][1]; }
  }
}

// hat = (v - mean) rstd over the row; layer norm takes the variance about the mean, in a second sum over the registers
template <typename R, int TPR, int EL>
__device__ __forceinline__ void normalise(const float (&v)[EL], float (&hat)[EL], bool layer, float eps, int t, int C, float& mean,
                                          float& rstd, float (*red)[2]) {
  float s = 0.f, q = 0.f;
  mean = 0.f;
  if (layer) {
#pragma unroll
    for (int e = 0; e < EL; ++e) s += v[e];
    row_sum2<TPR>(s, q, red);
    mean = s / C;
  }
  q = 0.f;
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    hat[e] = R::in(t, e, C) ? v[e] - mean : 0.f;
    q += hat[e] * hat[e];
  }
  s = 0.f;
  row_sum2<TPR>(q, s, red);
  rstd = 1.0f / sqrtf(q / C + eps);
#pragma unroll
  for (int e = 0; e < EL; ++e) hat[e] *= rstd;
}

template <typename T, int TPR, int EL, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_fwd_kernel(NormArgs a) {
  using R = Row<T, TPR, EL, VEC>;
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[16][2];
  const int t = threadIdx.x % TPR, C = a.C;
  const long m = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  if (m >= a.M) return;                                    // whole waves (TPR = 64) or the whole workgroup
  float r[EL], n[EL], w[EL], hat[EL];
  R::template load<T>((const T*)a.x + m * C, t, C, r);
  if (a.y != nullptr) {
    R::template load<T>((const T*)a.y + m * C, t, C, n);
    if (a.post) {
      float mean, rstd;
      normalise<R, TPR, EL>(n, hat, a.layer, a.eps, t, C, mean, rstd, red);
      R::param(a.post_w, a.param_f32, 1.f, t, C, w);
      R::param(a.post_b, a.param_f32, 0.f, t, C, n);
#pragma unroll
      for (int e = 0; e < EL; ++e) n[e] += hat[e] * w[e];
      if (a.stats != nullptr && t == 0) { a.stats[m] = mean; a.stats[a.M + m] = rstd; }
    }
    if (a.gate_kind == GATE_FULL) R::template load<T>((const T*)a.gate + m * C, t, C, w);
    else R::param(a.gate, a.param_f32, 1.f, t, C, w);
#pragma unroll
    for (int e = 0; e < EL; ++e) r[e] += a.scale * w[e] * n[e];
    R::template store<T>((T*)a.r + m * C, t, C, r);
  }
  if (a.pre) {
    float mean, rstd;
    normalise<R, TPR, EL>(r, hat, a.layer, a.eps, t, C, mean, rstd, red);
    R::param(a.pre_w, a.param_f32, 1.f, t, C, w);
    R::param(a.pre_b, a.param_f32, 0.f, t, C, n);
#pragma unroll
    for (int e = 0; e < EL; ++e) n[e] += hat[e] * w[e];
    R::template store<T>((T*)a.h + m * C, t, C, n);
    if (a.stats != nullptr && t == 0) { a.stats[2 * (long)a.M + m] = mean; a.stats[3 * (long)a.M + m] = rstd; }
  }
}

// d -> rstd (d - mean(d) - hat mean(d hat)); d of columns beyond C is zero
template <typename R, int TPR, int EL>
__device__ __forceinline__ void norm_back(float (&d)[EL], const float (&hat)[EL], float rstd, bool layer, int C,
                                          float (*red)[2]) {
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int e = 0; e < EL; ++e) { s += d[e]; q += d[e] * hat[e]; }
  row_sum2<TPR>(s, q, red);
  s = layer ? s / C : 0.f;
  q /= C;
#pragma unroll
  for (int e = 0; e < EL; ++e) d[e] = rstd * (d[e] - s - hat[e] * q);
}

template <typename T, int TPR, int EL, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_bwd_kernel(NormArgs a) {
  using R = Row<T, TPR, EL, VEC>;
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[16][2];
  __shared__ float join[RPB > 1 ? RPB * TPR * EL : 1];
  const int t = threadIdx.x % TPR, C = a.C, sub = threadIdx.x / TPR;
  float acc[5][EL];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int e = 0; e < EL; ++e) acc[k][e] = 0.f;
  // a row group walks its rows; all threads of a row take the same turns (the row sums meet in barriers only if TPR > 64)
  for (long m = (long)blockIdx.x * RPB + sub; m < a.M; m += (long)gridDim.x * RPB) {
    float r[EL], n[EL], nhat[EL], g[EL], w[EL], dr[EL];
    float prstd = 0.f;
    if (a.y != nullptr) {
      R::template load<T>((const T*)a.y + m * C, t, C, n);
      if (a.post) {
        const float mean = a.stats[m];
        prstd = a.stats[a.M + m];
#pragma unroll
        for (int e = 0; e < EL; ++e) nhat[e] = R::in(t, e, C) ? (n[e] - mean) * prstd : 0.f;
        R::param(a.post_w, a.param_f32, 1.f, t, C, w);
        R::param(a.post_b, a.param_f32, 0.f, t, C, n);
#pragma unroll
        for (int e = 0; e < EL; ++e) n[e] += nhat[e] * w[e];
      }
      if (a.gate_kind == GATE_FULL) R::template load<T>((const T*)a.gate + m * C, t, C, g);
      else R::param(a.gate, a.param_f32, 1.f, t, C, g);
    }
    if (a.dr != nullptr) {
      R::template load<T>((const T*)a.dr + m * C, t, C, dr);
    } else {
#pragma unroll
      for (int e = 0; e < EL; ++e) dr[e] = 0.f;
    }
    if (a.dh != nullptr) {
      float d[EL];
      R::template load<T>((const T*)a.x + m * C, t, C, r);
      const float mean = a.stats[2 * (long)a.M + m], rstd = a.stats[3 * (long)a.M + m];
      if (a.y != nullptr) {
#pragma unroll
        for (int e = 0; e < EL; ++e) r[e] += a.scale * g[e] * n[e];
      }
#pragma unroll
      for (int e = 0; e < EL; ++e) r[e] = R::in(t, e, C) ? (r[e] - mean) * rstd : 0.f;      // rhat
      R::template load<T>((const T*)a.dh + m * C, t, C, d);
      R::param(a.pre_w, a.param_f32, 1.f, t, C, w);
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        acc[3][e] += d[e] * r[e];
        acc[4][e] += d[e];
        d[e] *= w[e];
      }
      norm_back<R, TPR, EL>(d, r, rstd, a.layer, C, red);
#pragma unroll
      for (int e = 0; e < EL; ++e) dr[e] += d[e];
    }
    if (a.dx != nullptr) R::template store<T>((T*)a.dx + m * C, t, C, dr);
    if (a.y != nullptr) {
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        dr[e] *= a.scale;
        const float dg = dr[e] * n[e];
        acc[0][e] += dg;
        dr[e] *= g[e];                                     // dn
        g[e] = dg;
      }
      if (a.gate_kind == GATE_FULL && a.dgate != nullptr) R::template store<T>((T*)a.dgate + m * C, t, C, g);
      if (a.post) {
        R::param(a.post_w, a.param_f32, 1.f, t, C, w);
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          acc[1][e] += dr[e] * nhat[e];
          acc[2][e] += dr[e];
          dr[e] *= w[e];
        }
        norm_back<R, TPR, EL>(dr, nhat, prstd, a.layer, C, red);
      }
      if (a.dy != nullptr) R::template store<T>((T*)a.dy + m * C, t, C, dr);
    }
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    float* out = a.part + ((long)blockIdx.x * 5 + k) * C;
    if (RPB > 1) {                                         // the workgroup's row groups, in order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EL; ++e) join[(sub * EL + e) * TPR + t] = acc[k][e];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          float s = 0.f;
#pragma unroll
          for (int q = 0; q < RPB; ++q) s += join[(q * EL + e) * TPR + t];
          acc[k][e] = s;
        }
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int j = 0; j < R::NV; ++j) {
        const int c = R::col(t, j);
#pragma unroll
        for (int e = 0; e < R::V; ++e)
          if (c < C) out[c + e] = acc[k][j * R::V + e];
      }
    }
  }
}

// Threads of a row: eight elements each as long as a workgroup can hold the row so, since the backward pass keeps five column
// sums an element in registers beside the row (sixteen elements over 512 threads spilled at 256 registers).
template <typename F> void by_width(int C, F f) {
  if (C <= 64 * 8) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
  else if (C <= 64 * 16) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
  else if (C <= 256 * 8) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  else if (C <= 512 * 8) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 8>{});
  else if (C <= 1024 * 8) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 16>{});
}

template <typename T> void fwd(const NormArgs& a, hipStream_t s) {
  by_width(a.C, [&](auto tpr, auto el) {
    constexpr int TPR = decltype(tpr)::value, EL = decltype(el)::value, RPB = TPR < 256 ? 256 / TPR : 1;
    const dim3 grid((a.M + RPB - 1) / RPB), block(TPR < 256 ? 256 : TPR);
    if (a.vec) hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, EL, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, EL, false>), grid, block, 0, s, a);
  });
}
template <typename T> void bwd(const NormArgs& a, hipStream_t s) {
  by_width(a.C, [&](auto tpr, auto el) {
    constexpr int TPR = decltype(tpr)::value, EL = decltype(el)::value;
    const dim3 grid(a.groups), block(TPR < 256 ? 256 : TPR);
    if (a.vec) hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, EL, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, EL, false>), grid, block, 0, s, a);
  });
}
}  // namespace

// workgroups of the backward pass: as many as the chip holds at once, no more than there are rows
int norm_bwd_groups(int M, int C) {
  const int rpb = C <= 64 * 16 ? 4 : 1, most = (M + rpb - 1) / rpb, want = C > 512 * 8 ? 256 : 512;
  return most < want ? most : want;
}

void launch_norm_fwd(int dtype, const NormArgs& a, hipStream_t s) {
  if (dtype == F32) fwd<float>(a, s);
  else if (dtype == BF16) fwd<__bf16>(a, s);
  else fwd<_Float16>(a, s);
  DDL_HIP_CHECK(hipGetLastError());
}
void launch_norm_bwd(int dtype, const NormArgs& a, hipStream_t s) {
  if (dtype == F32) bwd<float>(a, s);
  else if (dtype == BF16) bwd<__bf16>(a, s);
  else bwd<_Float16>(a, s);
  DDL_HIP_CHECK(hipGetLastError());
}

}  // namespace ffn
}  // namespace ddl
