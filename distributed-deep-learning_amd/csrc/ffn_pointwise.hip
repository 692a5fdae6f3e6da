// Pointwise companions of the feed-forward products: operand packing, joining of split contractions, the activation's
// backward pass with the bias gradients' column sums.  All are bound by memory: one pass, 16-byte accesses.
#include "ffn_common.h"
#include "ddl_kernels.h"

namespace ddl {
namespace ffn {
namespace {

// ---- pack: any strides -> rows of 16-byte multiples, padding zero (it enters sums over k) -------------------------------
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* __restrict__ src, long s_row, long s_col, T* __restrict__ dst,
                                                   long ld, long rows, int cols) {
  constexpr int V = 16 / sizeof(T);
  const long per = ld / V, total = rows * per;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const long r = i / per;
    const int c = (int)(i - r * per) * V;
    Pack<T, V> x;
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = c + e < cols ? src[r * s_row + (c + e) * s_col] : (T)0.f;
    *reinterpret_cast<Pack<T, V>*>(dst + r * ld + c) = x;
  }
}

// ---- join: the splits' sums in split order, then the product's epilogue -------------------------------------------------
template <typename T, bool DUAL>
__global__ void __launch_bounds__(256) join_kernel(GemmArgs a) {
  constexpr int V = 4;
  const int per = (int)(a.ldw / V), planes = a.nout * (DUAL ? 2 : 1);
  const long rows = (long)a.M * a.nout, total = rows * per, plane = (long)a.M * a.ldw;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const long row = i / per;
    const int n = (int)(i - row * per) * V, which = (int)(row / a.M);
    const long m = row - (long)which * a.M;
    if (n >= a.N) continue;
    const float* p = a.partial + which * plane + m * a.ldw + n;
    float v[V] = {0.f, 0.f, 0.f, 0.f}, w[V] = {0.f, 0.f, 0.f, 0.f}, b0[V], b1[V];
    for (int s = 0; s < a.splits; ++s) {
      float t[V];
      load_vec<float, V>(p, t);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += t[e];
      if (DUAL) {
        load_vec<float, V>(p + plane, t);
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] += t[e];
      }
      p += planes * plane;
    }
    load_bias<T, V>(a.ep, 0, n, a.N, true, b0);
    load_bias<T, V>(a.ep, 1, n, a.N, true, b1);
    epilogue_store<T, DUAL, false, V>(a.ep, which, m, n, a.N, true, v, w, b0, b1);
  }
}

// ---- backward of the activation -----------------------------------------------------------------------------------------
//   linear:  dz = dy act'(z);      dual:  dg = dy u act'(g), du = dy act(g);      without z: dz = dy
// z, g and u are the fp32 sums of the forward pass, so dz is rounded once.  The bias gradients are column sums of the
// unrounded dz: a workgroup adds its rows in registers, then in LDS in a fixed order; `launch_colsum` adds the chunks.
// Columns N .. ldd-1 of dz are written as zeros (they enter the sums of the products that read dz).
template <typename T, bool DUAL>
__global__ void __launch_bounds__(256) act_bwd_kernel(ActBwdArgs a) {
  constexpr int V = 16 / sizeof(T), TX = 32, TY = 8, D = DUAL ? 2 : 1;
  __shared__ float red[TY][TX * V + 4];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int n = (blockIdx.x * TX + tx) * V, left = a.N - n;
  const bool full = left >= V;
  const int per = (a.M + a.chunks - 1) / a.chunks, m0 = blockIdx.y * per, m1 = min(a.M, m0 + per);
  float sum[D][V];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[d][e] = 0.f;
  if (n < a.N || n < a.ldd) {
    for (int m = m0 + ty; m < m1; m += TY) {
      float dy[V], d0[V], d1[V];
      load_some<T, V>((const T*)a.dy + m * a.ldy + n, dy, left, full && a.dy_vec);
#pragma unroll
      for (int e = 0; e < V; ++e) d0[e] = dy[e];
      if (a.z[0] != nullptr) {                             // rows of z are padded to 16 values
        float z[V], u[V];
        if (left > 0) {
          load_vec<float, V>(a.z[0] + m * a.ldz + n, z);
          if (DUAL) load_vec<float, V>(a.z[1] + m * a.ldz + n, u);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float act;
          const float da = act_grad(a.act, z[e], act);
          const bool in = e < left;
          d0[e] = in ? dy[e] * (DUAL ? u[e] * da : da) : 0.f;
          if (DUAL) d1[e] = in ? dy[e] * act : 0.f;
        }
      }
      if (a.dz[0] != nullptr && n < a.ldd) {
        store_vec<T, V>((T*)a.dz[0] + m * a.ldd + n, d0);
        if (DUAL) store_vec<T, V>((T*)a.dz[1] + m * a.ldd + n, d1);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sum[0][e] += d0[e];
        if (DUAL) sum[D - 1][e] += d1[e];
      }
    }
  }
  if (a.part == nullptr) return;                           // uniform over the grid
#pragma unroll
  for (int d = 0; d < D; ++d) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) red[ty][tx * V + e] = sum[d][e];
    __syncthreads();
    for (int c = threadIdx.x; c < TX * V; c += 256) {
      const int col = blockIdx.x * TX * V + c;
      if (col >= a.N) continue;
      float s = 0.f;
#pragma unroll
      for (int y = 0; y < TY; ++y) s += red[y][c];
      a.part[((long)blockIdx.y * D + d) * a.N + col] = s;
    }
  }
}

// ---- column sums over chunks --------------------------------------------------------------------------------------------
struct ColsumOuts { void* out[8]; };
template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const float* __restrict__ part, int chunks, int nvec, long n,
                                                     ColsumOuts o) {
  __shared__ float red[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, vec = blockIdx.y;
  const long c = blockIdx.x * 64L + tx;
  float s = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int k = ty; k < chunks; k += 4) s += part[((long)k * nvec + vec) * n + c];
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < n && o.out[vec] != nullptr)
    ((T*)o.out[vec])[c] = from_f<T>((red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]));
}

unsigned grid_for(long items) {
  const long g = (items + 255) / 256;
  return (unsigned)(g < 1 ? 1 : g > 8192 ? 8192 : g);
}
}  // namespace

#define DDL_BY_TYPE(dtype, CALL)                                  \
  do {                                                            \
    if ((dtype) == F32) { using T = float; CALL; }                \
    else if ((dtype) == BF16) { using T = __bf16; CALL; }         \
    else { using T = _Float16; CALL; }                            \
    DDL_HIP_CHECK(hipGetLastError());                             \
  } while (0)

void launch_pack(int dtype, const void* src, long s_row, long s_col, void* dst, long ld_dst, long rows, int cols,
                 hipStream_t s) {
  if (rows <= 0 || ld_dst <= 0) return;
  DDL_BY_TYPE(dtype, hipLaunchKernelGGL(pack_kernel<T>, dim3(grid_for(rows * ld_dst * sizeof(T) / 16)), dim3(256), 0, s,
                                        (const T*)src, s_row, s_col, (T*)dst, ld_dst, rows, cols));
}

void launch_join(int dtype, const float* partial, const GemmArgs& a0, hipStream_t s) {
  GemmArgs a = a0;
  a.partial = const_cast<float*>(partial);
  const dim3 grid(grid_for((long)a.M * a.nout * (a.ldw / 4)));
  if (a.dual) DDL_BY_TYPE(dtype, hipLaunchKernelGGL((join_kernel<T, true>), grid, dim3(256), 0, s, a));
  else DDL_BY_TYPE(dtype, hipLaunchKernelGGL((join_kernel<T, false>), grid, dim3(256), 0, s, a));
}

// rows are dealt to so many workgroups that the grid holds about 2048 of them, eight rows at least each
int act_bwd_chunks(int dtype, int M, int N) {
  const int cols = 32 * 16 / esize(dtype), nb = (N + cols - 1) / cols;
  int c = 2048 / (nb < 1 ? 1 : nb);
  const int most = (M + 7) / 8;
  c = c > most ? most : c;
  return c < 1 ? 1 : c;
}

void launch_act_bwd(int dtype, const ActBwdArgs& a, hipStream_t s) {
  const int cols = 32 * 16 / esize(dtype);
  const int width = a.ldd > a.N ? (int)a.ldd : a.N;
  const dim3 grid((width + cols - 1) / cols, a.chunks);
  if (a.dual) DDL_BY_TYPE(dtype, hipLaunchKernelGGL((act_bwd_kernel<T, true>), grid, dim3(256), 0, s, a));
  else DDL_BY_TYPE(dtype, hipLaunchKernelGGL((act_bwd_kernel<T, false>), grid, dim3(256), 0, s, a));
}

void launch_colsum(int out_dtype, const float* part, int chunks, int nvec, long n, void* const* out, hipStream_t s) {
  ColsumOuts o = {};
  for (int i = 0; i < nvec; ++i) o.out[i] = out[i];
  const dim3 grid((unsigned)((n + 63) / 64), nvec);
  DDL_BY_TYPE(out_dtype, hipLaunchKernelGGL(colsum_kernel<T>, grid, dim3(256), 0, s, part, chunks, nvec, n, o));
}

// ---- choice of tile and split -------------------------------------------------------------------------------------------
GemmPlan gemm_plan(int dtype, const GemmArgs& a) {
  auto tiles = [&](int bn, int bm) {
    const long w = a.dual ? bn / 2 : bn;
    return ((a.N + w - 1) / w) * (long)((a.M + bm - 1) / bm) * a.nout;
  };
  GemmPlan p;
  p.ldw = (a.N + 15) / 16 * 16;
  const bool same = a.nseg == 1 || (a.ldp[0] == a.ldp[1] && a.ldq[0] == a.ldq[1]);
  const bool holds = a.M >= 256 && a.N >= (a.dual ? 128 : 256) && same;
  if (dtype != F32 && holds && tiles(256, 256) >= 192) p.cfg = 2;
  else if (a.M > 64) p.cfg = 1;
  else p.cfg = 0;
  const long t = p.cfg == 2 ? tiles(256, 256) : p.cfg == 1 ? tiles(128, 128) : tiles(128, 32);
  const int tk = 128 / esize(dtype);
  const long slabs = (long)((a.K + tk - 1) / tk) * a.nseg;
  const long want = p.cfg == 2 ? 1 : (p.cfg == 1 ? 384 : 1024) / (t < 1 ? 1 : t);
  long s = want;
  if (s > slabs / 4) s = slabs / 4;
  if (s > 32) s = 32;
  p.splits = s < 2 ? 1 : (int)s;
  if (p.splits > 1) {                                      // no empty splits
    const long per = (slabs + p.splits - 1) / p.splits;
    p.splits = (int)((slabs + per - 1) / per);
    p.partial_floats = (long)p.splits * a.nout * (a.dual ? 2 : 1) * a.M * p.ldw;
  }
  return p;
}

void launch_gemm(int dtype, GemmArgs a, const GemmPlan& plan, hipStream_t s) {
  a.splits = plan.splits;
  a.ldw = plan.ldw;
  if (plan.splits == 1) a.partial = nullptr;
  if (dtype == F32) launch_gemm_f32(a, plan.cfg, s);
  else if (dtype == BF16) launch_gemm_bf16(a, plan.cfg, s);
  else launch_gemm_f16(a, plan.cfg, s);
  DDL_HIP_CHECK(hipGetLastError());
  if (plan.splits > 1) launch_join(dtype, a.partial, a, s);
}

}  // namespace ffn
}  // namespace ddl
