// Pointwise companions of the feed-forward products: operand packing, joining of split contractions, the activation's
// backward pass with the bias gradients' column sums.  All are bound by memory: one pass, 16-byte accesses.
#include "ffn_common.h"
#include "ddl_kernels.h"
#include <type_traits>

namespace ddl {
namespace ffn {
namespace {

// ---- pack: any strides -> rows of 16-byte multiples, padding zero (it enters sums over k); one launch for a product's operands -----
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(PackArgs a) {
  constexpr int V = 16 / sizeof(T);
  const PackItem& it = a.item[blockIdx.y];
  const T* src = (const T*)it.src;
  const long per = it.ld / V, total = it.rows * per;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < total; i += gridDim.x * 256L) {
    const long r = i / per;
    const int c = (int)(i - r * per) * V;
    Pack<T, V> x;
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = c + e < it.cols ? src[r * it.s_row + (c + e) * it.s_col] : (T)0.f;
    *reinterpret_cast<Pack<T, V>*>((T*)it.dst + r * it.ld + c) = x;
  }
}

// ---- join: the splits' sums, then the product's epilogue -----------------------------------------------------------------
// Four groups of threads take every fourth split each and meet in LDS in a fixed order: with up to 32 splits of few rows one thread
// an output would wait for memory 32 times.
template <typename T, bool DUAL>
__global__ void __launch_bounds__(256) join_kernel(GemmArgs a) {
  constexpr int V = 4, GROUPS = 4, TX = 64, D = DUAL ? 2 : 1;
  __shared__ float red[GROUPS - 1][TX][D * V + 1];
  const int per = (int)(a.ldw / V), planes = a.nout * D, tx = threadIdx.x % TX, g = threadIdx.x / TX;
  const long rows = (long)a.M * a.nout, total = rows * per, plane = (long)a.M * a.ldw, step = planes * plane;
  const long i = blockIdx.x * (long)TX + tx, row = i / per;
  const int n = (int)(i - row * per) * V, which = (int)(row / a.M);
  const long m = row - (long)which * a.M;
  const bool in = i < total && n < a.N;
  float v[D * V];
#pragma unroll
  for (int e = 0; e < D * V; ++e) v[e] = 0.f;
  if (in) {
    const float* p = a.partial + which * plane + m * a.ldw + n;
#pragma unroll 4
    for (int s = g; s < a.splits; s += GROUPS) {
      float t[D * V];
      load_vec<float, V>(p + s * step, t);
      if (DUAL) load_vec<float, V>(p + s * step + plane, t + (D - 1) * V);
#pragma unroll
      for (int e = 0; e < D * V; ++e) v[e] += t[e];
    }
  }
  if (g > 0) {
#pragma unroll
    for (int e = 0; e < D * V; ++e) red[g - 1][tx][e] = v[e];
  }
  __syncthreads();
  if (g > 0 || !in) return;
#pragma unroll
  for (int q = 0; q < GROUPS - 1; ++q)
#pragma unroll
    for (int e = 0; e < D * V; ++e) v[e] += red[q][tx][e];
  if constexpr (std::is_same<T, _Float16>::value && !DUAL) {
    if (a.ep.scale != nullptr) {
      const float scale = *a.ep.scale;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= scale;
    }
  }
  float b0[V], b1[V];
  load_bias<T, V>(a.ep, 0, n, a.N, true, b0);
  load_bias<T, V>(a.ep, 1, n, a.N, true, b1);
  epilogue_store<T, DUAL, false, V>(a.ep, which, m, n, a.N, true, v, v + (D - 1) * V, b0, b1);
}

// ---- backward of the activation -----------------------------------------------------------------------------------------
//   linear:  dz = dy act'(z);      dual:  dg = dy u act'(g), du = dy act(g);      without z: dz = dy
// z, g and u are the fp32 sums of the forward pass, so dz is rounded once (`two`: and what the rounding took off is kept as well).  The bias gradients are column sums of the
// unrounded dz: a workgroup adds its rows in registers, then in LDS in a fixed order; `launch_colsum` adds the chunks.
// Columns N .. ldd-1 of dz are written as zeros (they enter the sums of the products that read dz).
// Bound by memory: 8192 x 4096 bf16 with bias sums 52 us for 268 MB (5.1 TB/s, the rate of a copy).
// what rounding took off v (nothing where it left no finite value: the sum of both parts is that value)
template <typename T, int V> __device__ __forceinline__ void store_lack(T* dst, const float* v) {
  float lack[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float r = to_f(from_f<T>(v[e])), d = v[e] - r;
    lack[e] = fabsf(r) <= FLT_MAX ? d : 0.f;
  }
  store_vec<T, V>(dst, lack);
}
// The rows of one tile (strip of 32 vectors of columns, chunk of rows).
// STORE: dz, its sums, and in fp16 the largest |dz|;  STORE_SCALED: dz times `inv`;  FINITE_TOP: nothing but the largest finite |dz|
enum RowsPass : int { STORE, STORE_SCALED, FINITE_TOP };
template <typename T, bool DUAL, int PASS>
__device__ __forceinline__ void act_bwd_rows(const ActBwdArgs& a, int strip, int chunk, float inv,
                                             float (&sum)[DUAL ? 2 : 1][16 / sizeof(T)], float& top) {
  constexpr int V = 16 / sizeof(T), TX = 32, TY = 8, D = DUAL ? 2 : 1;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int n = (strip * TX + tx) * V, left = a.N - n;
  const bool full = left >= V;
  const int per = (a.M + a.chunks - 1) / a.chunks, m0 = chunk * per, m1 = min(a.M, m0 + per);
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
      if (PASS == STORE) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sum[0][e] += d0[e];
          if (DUAL) sum[D - 1][e] += d1[e];
          if (std::is_same<T, _Float16>::value) {          // a NaN is passed over
            top = fmaxf(top, fabsf(d0[e]));
            if (DUAL) top = fmaxf(top, fabsf(d1[e]));
          }
        }
      }
      if (PASS == FINITE_TOP) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (fabsf(d0[e]) <= FLT_MAX) top = fmaxf(top, fabsf(d0[e]));
          if (DUAL && fabsf(d1[e]) <= FLT_MAX) top = fmaxf(top, fabsf(d1[e]));
        }
        continue;
      }
      if (PASS == STORE_SCALED) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          d0[e] *= inv;
          if (DUAL) d1[e] *= inv;
        }
      }
      if (a.dz[0] != nullptr && n < a.ldd) {
        store_vec<T, V>((T*)a.dz[0] + m * a.ldd + n, d0);
        if (DUAL) store_vec<T, V>((T*)a.dz[1] + m * a.ldd + n, d1);
        if (a.two) {
          store_lack<T, V>((T*)a.dz[0] + (m + a.M) * a.ldd + n, d0);
          if (DUAL) store_lack<T, V>((T*)a.dz[1] + (m + a.M) * a.ldd + n, d1);
        }
      }
    }
  }
}
// largest of a workgroup of 256, in every thread; values are not negative
__device__ __forceinline__ float group_max(float v, float (&red)[4]) {
#pragma unroll
  for (int i = 32; i > 0; i /= 2) v = fmaxf(v, __shfl_xor(v, i));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

template <typename T, bool DUAL>
__global__ void __launch_bounds__(256) act_bwd_kernel(ActBwdArgs a) {
  constexpr int V = 16 / sizeof(T), TX = 32, TY = 8, D = DUAL ? 2 : 1;
  __shared__ float red[TY][TX * V + 4];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  float sum[D][V], top = 0.f;
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[d][e] = 0.f;
  act_bwd_rows<T, DUAL, STORE>(a, blockIdx.x, blockIdx.y, 1.f, sum, top);
  if constexpr (std::is_same<T, _Float16>::value) {
    __shared__ float tops[4];
    if (a.range != nullptr) {                              // uniform over the grid
      top = group_max(top, tops);
      if (top > FLT_MAX) {                                 // an infinity is nothing to scale by: look again
        top = 0.f;
        act_bwd_rows<T, DUAL, FINITE_TOP>(a, blockIdx.x, blockIdx.y, 1.f, sum, top);
        __syncthreads();
        top = group_max(top, tops);
      }
      if (threadIdx.x == 0) a.range[blockIdx.y * gridDim.x + blockIdx.x] = top;
    }
  }
  if (a.part == nullptr && a.db[0] == nullptr) return;      // uniform over the grid
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
      if (a.db[0] != nullptr) ((T*)a.db[d])[col] = from_f<T>(s);
      else a.part[((long)blockIdx.y * D + d) * a.N + col] = s;
    }
  }
}

// fp16 has five exponent bits, and dz is no input or result: dy u act' may pass 65504, or lie where fp16 counts in steps of 2^-24, while the
// gradients made of it are ordinary numbers.  So dz is held times one power of two for the call.  It is 1 where the largest finite |dz|
// lies in [2^-8, 65504]; then nothing is done here (a launch that reads one number a workgroup of the pass before).  Otherwise dz is
// written again with the largest in [2^14, 2^15), and the products scale their fp32 sums back.  2^-8: below it the steps of 2^-24
// would be more than dz's own rounding for values of a sixteenth of the largest, about their root mean square.  fp16 gradients with the
// scale at 1, both and the biases': 20 x 1024 x 4096 26.4 us without this launch, 29.3 with it; 777 x 1021 x 1531 49.4 and 53.1;
// 8192 x 4096 x 4096 503 and 510.
template <bool DUAL>
__global__ void __launch_bounds__(256) act_bwd_rescale_kernel(ActBwdArgs a, int strips) {
  __shared__ float tops[4];
  const int tiles = strips * a.chunks;
  float top = 0.f;
  for (int i = threadIdx.x; i < tiles; i += 256) top = fmaxf(top, a.range[i]);
  top = group_max(top, tops);
  int e = 0;
  if (top > 65504.f || (top > 0.f && top < 0x1p-8f)) {
    e = (int)(__builtin_bit_cast(unsigned, top) >> 23) - 126 - 15;   // top in [2^(e + 14), 2^(e + 15))
    e = e < -60 ? -60 : e;
  }
  const float scale = __builtin_bit_cast(float, (unsigned)(127 + e) << 23), inv = __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.scale = scale;
  if (e == 0) return;
  float sum[DUAL ? 2 : 1][8];
  for (int i = blockIdx.x; i < tiles; i += gridDim.x) act_bwd_rows<_Float16, DUAL, STORE_SCALED>(a, i % strips, i / strips, inv, sum, top);
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

void launch_pack(int dtype, const PackArgs& a, hipStream_t s) {
  long most = 0;
  for (int i = 0; i < a.count; ++i) {
    const long v = a.item[i].rows * a.item[i].ld * esize(dtype) / 16;
    most = v > most ? v : most;
  }
  if (most == 0) return;
  DDL_BY_TYPE(dtype, hipLaunchKernelGGL(pack_kernel<T>, dim3(grid_for(most), a.count), dim3(256), 0, s, a));
}

void launch_join(int dtype, const float* partial, const GemmArgs& a0, hipStream_t s) {
  GemmArgs a = a0;
  a.partial = const_cast<float*>(partial);
  const dim3 grid((unsigned)(((long)a.M * a.nout * (a.ldw / 4) + 63) / 64));
  if (a.dual) DDL_BY_TYPE(dtype, hipLaunchKernelGGL((join_kernel<T, true>), grid, dim3(256), 0, s, a));
  else DDL_BY_TYPE(dtype, hipLaunchKernelGGL((join_kernel<T, false>), grid, dim3(256), 0, s, a));
}

// Rows are dealt to so many workgroups that the grid holds about 2048 of them, eight rows at least each.  Up to 32 rows are one
// chunk: four turns of a thread cost less than the second launch (a step over 30 x 4096 fp32: 4 + 2.4 us as two); the eight turns of
// 64 x 4096 bf16 cost 16 us.
int act_bwd_chunks(int dtype, int M, int N) {
  if (M <= 32) return 1;
  const int cols = 32 * 16 / esize(dtype), nb = (N + cols - 1) / cols;
  int c = 2048 / (nb < 1 ? 1 : nb);
  const int most = (M + 7) / 8;
  c = c > most ? most : c;
  return c < 1 ? 1 : c;
}

int act_bwd_strips(int dtype, const ActBwdArgs& a) {
  const int cols = 32 * 16 / esize(dtype);
  const int width = a.ldd > a.N ? (int)a.ldd : a.N;
  return (width + cols - 1) / cols;
}
int act_bwd_tiles(int dtype, const ActBwdArgs& a) { return act_bwd_strips(dtype, a) * a.chunks; }

void launch_act_bwd(int dtype, const ActBwdArgs& a, hipStream_t s) {
  const int strips = act_bwd_strips(dtype, a);
  const dim3 grid(strips, a.chunks);
  if (a.dual) DDL_BY_TYPE(dtype, hipLaunchKernelGGL((act_bwd_kernel<T, true>), grid, dim3(256), 0, s, a));
  else DDL_BY_TYPE(dtype, hipLaunchKernelGGL((act_bwd_kernel<T, false>), grid, dim3(256), 0, s, a));
  if (a.range != nullptr) {
    const int tiles = strips * a.chunks;
    const dim3 again(tiles < 512 ? tiles : 512);
    if (a.dual) hipLaunchKernelGGL(act_bwd_rescale_kernel<true>, again, dim3(256), 0, s, a, strips);
    else hipLaunchKernelGGL(act_bwd_rescale_kernel<false>, again, dim3(256), 0, s, a, strips);
    DDL_HIP_CHECK(hipGetLastError());
  }
}

void launch_colsum(int out_dtype, const float* part, int chunks, int nvec, long n, void* const* out, hipStream_t s) {
  ColsumOuts o = {};
  for (int i = 0; i < nvec; ++i) o.out[i] = out[i];
  const dim3 grid((unsigned)((n + 63) / 64), nvec);
  DDL_BY_TYPE(out_dtype, hipLaunchKernelGGL(colsum_kernel<T>, grid, dim3(256), 0, s, part, chunks, nvec, n, o));
}

// ---- choice of tile and split -------------------------------------------------------------------------------------------
// The estimate in microseconds that picks both: a launch, then the fullest CU's workgroups.  `one` / `two`: what 128 bytes of k of one
// workgroup alone / of two side by side on a CU cost, `end`: a tile's epilogue.  Fitted to graphs of 20 calls of every tile and split
// over twelve shapes from 40 x 256 x 512 to 1024 x 2048 x 2048 (rows x columns x k); its choice was 1.3% behind the best of them on
// the geometric mean, and these are some of the sides, bf16:
//   256 x 4096 x 1024:   64 x 64 tiles 8.3 us, 128 x 32 9.3, 128 x 128 17.4;     its d_x: 128 x 32 in 4 splits 14.1, 64 x 32 in 2 15.7
//   512 x 1024 x 1024:   64 x 32 7.5 us, 64 x 64 8.1, 128 x 32 8.7, 64 x 64 in 2 splits 11.2;     its d_w: 128 x 32 6.3, 64 x 32 7.9
//   1500 x 5000 x 5000:  256 x 128 88 us, 256 x 256 122, 128 x 128 100;          8192 x 8192 x 8192: 256 x 256 first
// A split writes its sums in fp32 and a second launch joins them: 3 us and the bytes at 2 TB/s.
namespace {
struct TileCost { int bn, bm, threads; double one, two, end; };
constexpr TileCost COST16[N_TILES] = {{128, 32, 512, .30, .56, .4}, {64, 32, 512, .22, .40, .5}, {64, 64, 512, .30, .53, .4},
                                      {128, 128, 256, .80, 1.40, 1.}, {256, 128, 512, 1.05, 2.1, 2.5}, {256, 256, 512, 1.7, 3.4, 5.}};
constexpr TileCost COST32[N_TILES] = {{128, 32, 512, .71, 1.35, .6}, {64, 32, 512, .42, .75, .6}, {64, 64, 512, .66, 1.23, .7},
                                      {128, 128, 256, 2.4, 3.9, 2.}, {}, {}};
}  // namespace

GemmPlan gemm_plan(int dtype, const GemmArgs& a) {
  GemmPlan best;
  best.ldw = (a.N + 15) / 16 * 16;
  const int tk = 128 / esize(dtype);
  const long slabs = (long)((a.K + tk - 1) / tk) * a.nseg;
  const bool same = a.nseg == 1 || (a.ldp[0] == a.ldp[1] && a.ldq[0] == a.ldq[1]);
  double best_us = 1e300;
  for (int cfg = 0; cfg < N_TILES; ++cfg) {
    const TileCost& c = (dtype == F32 ? COST32 : COST16)[cfg];
    const int width = a.dual ? c.bn / 2 : c.bn;
    if (c.bn == 0 || (cfg >= TILE_256x128 && !(same && a.N >= width && a.M >= c.bm))) continue;     // tiles without edges
    // k-strided 16-bit operands of 64 columns: every read of LDS is a transposing one, half as wide
    const double f = dtype != F32 && cfg == TILE_64x64 && !(a.p_kc && a.q_kc) ? 1.2 : 1.0;
    const long tiles = ((a.N + width - 1) / width) * (long)((a.M + c.bm - 1) / c.bm) * a.nout;
    if (tiles * c.threads >= 1l << 32) continue;           // more threads than a launch may have
    for (long s = 1; s <= 32; s *= 2) {
      if (s > 1 && (s > slabs / 2 || tiles * s > 2048)) break;
      const long per = (slabs + s - 1) / s, splits = slabs > 0 ? (slabs + per - 1) / per : 1;      // no empty splits
      const long wgs = (tiles * splits + 255) / 256;
      const double turns = cfg <= TILE_64x64 ? (per + 1) / 2 * 2 : per;     // slabs in pairs
      double us = 3.5 + turns * f * ((wgs / 2) * c.two + (wgs % 2) * c.one) + wgs * c.end;
      const double floats = (double)splits * a.nout * (a.dual ? 2 : 1) * a.M * best.ldw;
      const bool join = splits > 1 || a.halves;
      if (join) us += 3.0 + floats * 4 / 2e6;
      if (us < best_us) {
        best_us = us;
        best.cfg = cfg;
        best.bm = c.bm;
        best.bn = width;
        best.splits = (int)splits;
        best.partial_floats = join ? (long)floats : 0;
      }
    }
  }
  return best;
}

void launch_gemm(int dtype, GemmArgs a, const GemmPlan& plan, hipStream_t s) {
  a.splits = plan.splits;
  a.ldw = plan.ldw;
  if (plan.partial_floats == 0) a.partial = nullptr;
  if (dtype == F32) launch_gemm_f32(a, plan.cfg, s);
  else if (dtype == BF16) launch_gemm_bf16(a, plan.cfg, s);
  else launch_gemm_f16(a, plan.cfg, s);
  DDL_HIP_CHECK(hipGetLastError());
  if (a.halves) {                                          // the two halves of the rows lie like two splits
    a.M /= 2;
    a.splits *= 2;
  }
  if (plan.partial_floats > 0) launch_join(dtype, a.partial, a, s);
}

}  // namespace ffn
}  // namespace ddl
