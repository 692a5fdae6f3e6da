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
//
// 16384 x 4096 bf16, both layer norms and a gate: forward 134 to 152 us (537 MB, 3.5 to 4 TB/s: two exchanges a row, each a
// barrier), backward 240 us (805 MB, 3.4 TB/s: four exchanges); 8192 x 8192 backward 410 us in two passes.  One row of 4096: 6 us, a
// launch.
#include "ffn_common.h"
#include "ffn_misc.h"
#include "ddl_kernels.h"
#include <type_traits>

namespace ddl {
namespace ffn {
namespace {

// threads of a workgroup: four rows where a row is one wave (rows of more waves meet in barriers, so they have a workgroup each)
constexpr int block_of(int tpr) { return tpr == 64 ? 256 : tpr; }

// A launch has fewer than 2^32 threads along x, and a row has up to 1024: workgroup ids go on along y.
__device__ __forceinline__ long group_id() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }
inline dim3 grid_of(long groups) {
  const long y = (groups + 65535) / 65536;
  return dim3((unsigned)((groups + y - 1) / y), (unsigned)y);
}

// The EL elements of a row that a thread holds: VEC: 16-byte chunks t, t + TPR, ...; otherwise single elements.
template <typename T, int TPR, int EL, bool VEC> struct Row {
  static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, NV = EL / V;
  static __device__ __forceinline__ int col(int t, int j) { return (j * TPR + t) * V; }
  template <typename S> static __device__ __forceinline__ void load(const S* p, int t, int C, float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col(t, j);
      load_vec<S, V>(p + (c < C ? c : 0), o + j * V);
#pragma unroll
      for (int e = 0; e < V; ++e) o[j * V + e] = c < C ? o[j * V + e] : 0.f;
    }
  }
  template <typename S> static __device__ __forceinline__ void store(S* p, int t, int C, const float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col(t, j);
      if (c < C) store_vec<S, V>(p + c, o + j * V);
    }
  }
  // a row's values as they come from memory; threads beyond the last column hold the first one's
  struct Raw { Pack<T, V> p[NV]; };
  static __device__ __forceinline__ void load_raw(const T* p, int t, int C, Raw& o) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = col(t, j);
      o.p[j] = *reinterpret_cast<const Pack<T, V>*>(p + (c < C ? c : 0));
    }
  }
  template <bool ZERO> static __device__ __forceinline__ void unpack(const Raw& r, int t, int C, float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool ok = !ZERO || col(t, j) < C;              // ZERO: zero beyond the last column
#pragma unroll
      for (int e = 0; e < V; ++e) o[j * V + e] = ok ? to_f(r.p[j].v[e]) : 0.f;
    }
  }
  // (v - mean) rstd, zero beyond the last column
  static __device__ __forceinline__ void centre(const float (&v)[EL], float mean, float rstd, int t, int C, float (&o)[EL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float f = col(t, j) < C ? rstd : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) o[j * V + e] = (v[j * V + e] - mean) * f;
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

// What the waves of a row exchange in LDS.  Successive exchanges alternate between two buffers, so that one barrier each is enough.
struct Exchange {
  float (*buf)[16][2];
  int turn = 0;
  __device__ explicit Exchange(float (*b)[16][2]) : buf(b) {}
};

// sum over a wave, in every lane: prefix sums inside rows of 16 lanes, then of the rows, by lane-shifting adds (an exchange through LDS
// costs about ten times as long)
__device__ __forceinline__ float wave_sum(float v) {
#define DDL_DPP_ADD(ctrl, rows) \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, true))
  DDL_DPP_ADD(0x111, 0xf);                                 // row_shr 1, 2, 4, 8
  DDL_DPP_ADD(0x112, 0xf);
  DDL_DPP_ADD(0x114, 0xf);
  DDL_DPP_ADD(0x118, 0xf);
  DDL_DPP_ADD(0x142, 0xa);                                 // row_bcast 15 into rows 1 and 3, then 31 into rows 2 and 3
  DDL_DPP_ADD(0x143, 0xc);
#undef DDL_DPP_ADD
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// sums of one or two values over the TPR threads of a row; every thread gets them
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, Exchange& x) {
  a = wave_sum(a);
  b = wave_sum(b);
  if (TPR > 64) {
    const int w = threadIdx.x >> 6;
    float(*red)[2] = x.buf[x.turn];
    x.turn ^= 1;
    if ((threadIdx.x & 63) == 0) { red[w][0] = a; red[w][1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) { a += red[i][0]; b += red[i][1]; }
  }
}
template <int TPR> __device__ __forceinline__ float row_sum(float a, Exchange& x) {
  a = wave_sum(a);
  if (TPR > 64) {
    float(*red)[2] = x.buf[x.turn];
    x.turn ^= 1;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = a;
    __syncthreads();
    a = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) a += red[i][0];
  }
  return a;
}

// hat = (v - mean) rstd over the row; layer norm takes the variance about the mean, in a second sum over the registers
template <typename R, int TPR, int EL>
__device__ __forceinline__ void normalise(const float (&v)[EL], float (&hat)[EL], bool layer, float eps, int t, int C, float& mean,
                                          float& rstd, Exchange& x) {
  float s = 0.f, q = 0.f;
  mean = 0.f;
  if (layer) {
#pragma unroll
    for (int e = 0; e < EL; ++e) s += v[e];                // zero beyond C
    mean = row_sum<TPR>(s, x) / C;
  }
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    hat[e] = R::in(t, e, C) ? v[e] - mean : 0.f;
    q += hat[e] * hat[e];
  }
  rstd = 1.0f / sqrtf(row_sum<TPR>(q, x) / C + eps);
#pragma unroll
  for (int e = 0; e < EL; ++e) hat[e] *= rstd;
}

template <typename T, int TPR, int EL, bool VEC>
__global__ void __launch_bounds__(block_of(TPR)) norm_fwd_kernel(NormArgs a) {
  using R = Row<T, TPR, EL, VEC>;
  constexpr int RPB = block_of(TPR) / TPR;
  __shared__ float xbuf[2][16][2];
  Exchange red(xbuf);
  const int t = threadIdx.x % TPR, C = a.C;
  const long m = group_id() * RPB + threadIdx.x / TPR;
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

// d -> rstd (d - s - hat q), s and q the row's means of d (layer norm) and d hat; d and hat are zero beyond the last column (by zero
// weights and `centre`)
template <int TPR, int EL>
__device__ __forceinline__ void norm_back(float (&d)[EL], const float (&hat)[EL], float rstd, bool layer, int C, Exchange& x, float& s,
                                          float& q) {
  s = q = 0.f;
#pragma unroll
  for (int e = 0; e < EL; ++e) { s += d[e]; q += d[e] * hat[e]; }
  row_sum2<TPR>(s, q, x);
  s = layer ? s / C : 0.f;
  q /= C;
#pragma unroll
  for (int e = 0; e < EL; ++e) d[e] = rstd * (d[e] - s - hat[e] * q);
}

// SUMS: the vectors' gradients are summed on the way.  A thread then keeps its columns' weights and sums in registers and, while it
// works on a row, the next row's values as they came from memory: at one or two workgroups a CU the loads of one row in flight
// would not cover their latency.  That takes up to 256 registers, so rows wider than 512 threads leave the sums to
// `norm_cols_kernel` and keep only the two means of the pre norm's backward formula for it (8192 x 8192 bf16: 910 us with the
// sums in spilled registers).
template <typename T, int TPR, int EL, bool VEC, bool SUMS>
__global__ void __launch_bounds__(block_of(TPR)) norm_bwd_kernel(NormArgs a) {
  using R = Row<T, TPR, EL, VEC>;
  constexpr int RPB = block_of(TPR) / TPR, S = SUMS ? EL : 1;
  __shared__ float xbuf[2][16][2];
  __shared__ float join[RPB > 1 ? RPB * TPR * EL : 1];
  Exchange red(xbuf);
  const int t = threadIdx.x % TPR, C = a.C, sub = threadIdx.x / TPR;
  const bool has_y = a.y != nullptr, full = a.gate_kind == GATE_FULL;
  float acc[5][S], post_w[EL], post_b[EL], pre_w[EL], gate[EL];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int e = 0; e < S; ++e) acc[k][e] = 0.f;
  auto load_post = [&]() { R::param(a.post_w, a.param_f32, 1.f, t, C, post_w); };
  auto load_post_b = [&]() { R::param(a.post_b, a.param_f32, 0.f, t, C, post_b); };
  auto load_pre = [&]() { R::param(a.pre_w, a.param_f32, 1.f, t, C, pre_w); };
  auto load_gate = [&]() {                                 // scale * gate
    if (full) return;
    R::param(a.gate, a.param_f32, 1.f, t, C, gate);
#pragma unroll
    for (int e = 0; e < EL; ++e) gate[e] *= a.scale;
  };
  if (SUMS) { load_post(); load_post_b(); load_pre(); load_gate(); }
  typename R::Raw xr, yr, gr, rr, hr;
  float st[4] = {0.f, 0.f, 0.f, 0.f};                      // post mean and rstd, pre mean and rstd
  const long stride = (long)gridDim.x * RPB;
  auto ahead = [&](long m) {
    if (a.dh != nullptr) { R::load_raw((const T*)a.dh + m * C, t, C, hr); R::load_raw((const T*)a.x + m * C, t, C, xr); }
    if (has_y) R::load_raw((const T*)a.y + m * C, t, C, yr);
    if (full) R::load_raw((const T*)a.gate + m * C, t, C, gr);
    if (a.dr != nullptr) R::load_raw((const T*)a.dr + m * C, t, C, rr);
    if (has_y && a.post) { st[0] = a.stats[m]; st[1] = a.stats[a.M + m]; }
    if (a.dh != nullptr) { st[2] = a.stats[2 * (long)a.M + m]; st[3] = a.stats[3 * (long)a.M + m]; }
  };
  long m = group_id() * RPB + sub;
  if (SUMS && m < a.M) ahead(m);
  // a row group walks its rows; all threads of a row take the same turns (the row sums meet in barriers only if TPR > 64)
  for (; m < a.M; m += stride) {
    float n[EL], nhat[EL], dr[EL], r[EL], d[EL];
    float prstd = 0.f, mean = 0.f, rstd = 0.f, s, q;
    if (!SUMS && has_y && a.post) { st[0] = a.stats[m]; st[1] = a.stats[a.M + m]; }
    if (!SUMS && has_y) R::load_raw((const T*)a.y + m * C, t, C, yr);
    if (!SUMS && full) R::load_raw((const T*)a.gate + m * C, t, C, gr);
    if (has_y) {
      R::template unpack<false>(yr, t, C, n);
      if (a.post) {
        if (!SUMS) { load_post(); load_post_b(); }
        const float pmean = st[0];
        prstd = st[1];
        R::centre(n, pmean, prstd, t, C, nhat);
#pragma unroll
        for (int e = 0; e < EL; ++e) n[e] = nhat[e] * post_w[e] + post_b[e];
      }
      if (!SUMS) load_gate();
      if (full) {
        R::template unpack<false>(gr, t, C, gate);
#pragma unroll
        for (int e = 0; e < EL; ++e) gate[e] *= a.scale;
      }
    }
    if (!SUMS && a.dh != nullptr) {
      R::load_raw((const T*)a.dh + m * C, t, C, hr);
      R::load_raw((const T*)a.x + m * C, t, C, xr);
      st[2] = a.stats[2 * (long)a.M + m];
      st[3] = a.stats[3 * (long)a.M + m];
    }
    if (!SUMS && a.dr != nullptr) R::load_raw((const T*)a.dr + m * C, t, C, rr);
    if (a.dr != nullptr) {
      R::template unpack<false>(rr, t, C, dr);
    } else {
#pragma unroll
      for (int e = 0; e < EL; ++e) dr[e] = 0.f;
    }
    if (a.dh != nullptr) {
      R::template unpack<false>(xr, t, C, r);
      R::template unpack<false>(hr, t, C, d);
      mean = st[2];
      rstd = st[3];
    }
    if (SUMS && m + stride < a.M) ahead(m + stride);
    if (a.dh != nullptr) {
      if (!SUMS) load_pre();
      if (has_y) {
#pragma unroll
        for (int e = 0; e < EL; ++e) r[e] += gate[e] * n[e];
      }
      R::centre(r, mean, rstd, t, C, r);                   // rhat
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        if constexpr (SUMS) {
          acc[3][e] += d[e] * r[e];
          acc[4][e] += d[e];
        }
        d[e] *= pre_w[e];
      }
      norm_back<TPR, EL>(d, r, rstd, a.layer, C, red, s, q);
      if (!SUMS && a.means != nullptr && t == 0) { a.means[m] = s; a.means[a.M + m] = q; }
#pragma unroll
      for (int e = 0; e < EL; ++e) dr[e] += d[e];
    }
    if (a.dx != nullptr) R::template store<T>((T*)a.dx + m * C, t, C, dr);
    if (has_y) {
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        if constexpr (SUMS) acc[0][e] += n[e] * dr[e];     // dgate / scale
        n[e] *= dr[e] * a.scale;
        dr[e] *= gate[e];                                  // dn
      }
      if (full && a.dgate != nullptr) R::template store<T>((T*)a.dgate + m * C, t, C, n);
      if (a.post) {
        if (!SUMS) load_post();
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          if constexpr (SUMS) {
            acc[1][e] += dr[e] * nhat[e];
            acc[2][e] += dr[e];
          }
          dr[e] *= post_w[e];
        }
        norm_back<TPR, EL>(dr, nhat, prstd, a.layer, C, red, s, q);
      }
      if (a.dy != nullptr) R::template store<T>((T*)a.dy + m * C, t, C, dr);
    }
    if (!SUMS) break;                                      // a workgroup a row
  }
  if constexpr (SUMS) {
    if (a.part == nullptr) return;
#pragma unroll
    for (int e = 0; e < EL; ++e) acc[0][e] *= a.scale;
#pragma unroll
    for (int k = 0; k < 5; ++k) {
      float* out = a.part + ((long)blockIdx.x * 5 + k) * C;
      if (RPB > 1) {                                       // the workgroup's row groups, in order
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EL; ++e) join[(sub * EL + e) * TPR + t] = acc[k][e];
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int e = 0; e < EL; ++e) {
            float v = 0.f;
#pragma unroll
            for (int g = 0; g < RPB; ++g) v += join[(g * EL + e) * TPR + t];
            acc[k][e] = v;
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
}

// The vectors' gradients of wide rows: with the rows' statistics and means known every term is element-wise, so threads own columns and
// stream down a chunk of rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) norm_cols_kernel(NormArgs a) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, TX = 32, TY = 8;
  __shared__ float red[TY][TX * V + 1];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, C = a.C, c = (blockIdx.x * TX + tx) * V;
  const int per = (a.M + a.groups - 1) / a.groups, m0 = blockIdx.y * per, m1 = min(a.M, m0 + per);
  const bool has_y = a.y != nullptr, full = a.gate_kind == GATE_FULL;
  auto vec = [&](const void* p, float none, float (&o)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = p == nullptr ? none : a.param_f32 ? ((const float*)p)[c + e] : to_f(((const T*)p)[c + e]);
  };
  float acc[5][V];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[k][e] = 0.f;
  if (c < C) {
    float post_w[V], post_b[V], pre_w[V], gate[V];
    vec(a.post_w, 1.f, post_w);
    vec(a.post_b, 0.f, post_b);
    vec(a.pre_w, 1.f, pre_w);
    vec(full ? nullptr : a.gate, 1.f, gate);
#pragma unroll 1
    for (long m = m0 + ty; m < m1; m += TY) {
      float n[V], nhat[V], dr[V];
#pragma unroll
      for (int e = 0; e < V; ++e) n[e] = nhat[e] = dr[e] = 0.f;
      if (has_y) {
        load_vec<T, V>((const T*)a.y + m * C + c, n);
        if (full) load_vec<T, V>((const T*)a.gate + m * C + c, gate);
        if (a.post) {
          const float mean = a.stats[m], rstd = a.stats[a.M + m];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            nhat[e] = (n[e] - mean) * rstd;
            n[e] = nhat[e] * post_w[e] + post_b[e];
          }
        }
      }
      if (a.dr != nullptr) load_vec<T, V>((const T*)a.dr + m * C + c, dr);
      if (a.dh != nullptr) {
        float r[V], d[V];
        load_vec<T, V>((const T*)a.x + m * C + c, r);
        load_vec<T, V>((const T*)a.dh + m * C + c, d);
        const float mean = a.stats[2 * (long)a.M + m], rstd = a.stats[3 * (long)a.M + m], s = a.means[m], q = a.means[a.M + m];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (has_y) r[e] += a.scale * gate[e] * n[e];
          r[e] = (r[e] - mean) * rstd;
          acc[3][e] += d[e] * r[e];
          acc[4][e] += d[e];
          dr[e] += rstd * (d[e] * pre_w[e] - s - r[e] * q);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dr[e] *= a.scale;
        acc[0][e] += dr[e] * n[e];
        dr[e] *= gate[e];
        acc[1][e] += dr[e] * nhat[e];
        acc[2][e] += dr[e];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) red[ty][tx * V + e] = acc[k][e];
    __syncthreads();
    for (int i = threadIdx.x; i < TX * V; i += 256) {
      const int col = blockIdx.x * TX * V + i;
      if (col >= C) continue;
      float v = 0.f;
#pragma unroll
      for (int y = 0; y < TY; ++y) v += red[y][i];
      a.part[((long)blockIdx.y * 5 + k) * C + col] = v;
    }
  }
}

// Threads of a row: eight elements each as far as a workgroup reaches (16384 x 4096 bf16 forward: 512 x 8 threads x elements 141 us,
// 256 x 16 177 us; more waves hide the memory better than fewer exchanges).
constexpr int SUMS_MAX_C = 4096;
template <typename F> void by_width(int C, bool forward, F f) {
  if (C <= 64 * 8) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
  else if (forward && C <= 64 * 16) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
  else if (C <= 256 * 8) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  else if (C <= 512 * 8) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 8>{});
  else if (C <= 1024 * 8) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 16>{});
}

template <typename T> void fwd(const NormArgs& a, hipStream_t s) {
  by_width(a.C, true, [&](auto tpr, auto el) {
    constexpr int TPR = decltype(tpr)::value, EL = decltype(el)::value, RPB = block_of(TPR) / TPR;
    const dim3 grid = grid_of(((long)a.M + RPB - 1) / RPB), block(block_of(TPR));
    if (a.vec) hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, EL, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, EL, false>), grid, block, 0, s, a);
  });
}
template <typename T> void bwd(const NormArgs& a, hipStream_t s) {
  by_width(a.C, false, [&](auto tpr, auto el) {
    constexpr int TPR = decltype(tpr)::value, EL = decltype(el)::value;
    constexpr bool SUMS = TPR * EL <= SUMS_MAX_C;
    const dim3 grid = SUMS ? dim3(a.groups) : grid_of(a.M), block(block_of(TPR));
    if (a.vec) hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, EL, true, SUMS>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, EL, false, SUMS>), grid, block, 0, s, a);
    if (!SUMS && a.part != nullptr) {
      const int width = 32 * (a.vec ? 16 / (int)sizeof(T) : 1);
      const dim3 cols((a.C + width - 1) / width, a.groups);
      if (a.vec) hipLaunchKernelGGL((norm_cols_kernel<T, true>), cols, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((norm_cols_kernel<T, false>), cols, dim3(256), 0, s, a);
    }
  });
}
}  // namespace

bool norm_bwd_wants_means(int C) { return C > SUMS_MAX_C; }

// rows of the table of partial column sums: about as many workgroups as the chip holds at once, no more than there are rows
int norm_bwd_groups(int M, int C) {
  const int rpb = C <= 64 * 8 ? 4 : C > SUMS_MAX_C ? 8 : 1, most = (M + rpb - 1) / rpb;
  const int want = C > SUMS_MAX_C ? 64 : C > 256 * 8 ? 256 : 512;
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
