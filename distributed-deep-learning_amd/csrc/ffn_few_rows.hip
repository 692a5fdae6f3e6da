// Products with few rows (inference on one or a few rows): out[m][n] = epilogue(sum_k w(n, k) x(m, k)), up to 32 rows m.
//
// Bound by reading the weights once: 2 N K bytes in 16 bits against 2 M N K operations.  A workgroup owns 16 weight rows and
// streams them from memory straight into the matrix cores' A operand (lane: 16 bytes of one row), eight waves splitting k;
// the few rows of x come out of L2 as the B operand.  The waves' sums meet in LDS in a fixed order, so the result does not
// depend on timing.  With 16 rows a workgroup even N = 4096 gives every CU a workgroup of eight waves.
// bf16: gated 1 x 11264 x 4096 39 us with all weights from memory (185 MB at 4.7 TB/s; a large copy moves 5.1), 31 to 35 where repeated
// calls find part of them in the Infinity Cache; linear 1 x 4096 x 4096 8.5 us and 6.4 to 7.4, a launch and 34 MB; fp32
// 30 x 4096 x 1024 10.2 us and 8.7 to 9.3.
// Rows of x beyond M repeat row 0 (their sums are dropped).
#include "ffn_common.h"
#include "ffn_mma.h"
#include "ddl_kernels.h"

namespace ddl {
namespace ffn {
namespace {

constexpr int NW = 8, U = 8, OUTER_ROWS = 64;

template <typename T, bool VEC>
__device__ __forceinline__ typename Mma<T>::Frag load_chunk(const T* row, int k, int K) {
  using Frag = typename Mma<T>::Frag;
  constexpr int EPC = 16 / sizeof(T);
  Frag f;
  if (VEC) {                                               // K is a multiple of the chunk: all of it or nothing
    if (k < K) f = *reinterpret_cast<const Frag*>(row + k);
    else f = Frag{};
  } else {
#pragma unroll
    for (int e = 0; e < EPC; ++e) f[e] = k + e < K ? row[k + e] : (T)0.f;
  }
  return f;
}

template <typename T, int MT, bool DUAL, bool VEC>
__global__ void __launch_bounds__(NW * 64) few_rows_kernel(FewRowsArgs a) {
  using Frag = typename Mma<T>::Frag;
  constexpr int EPC = 16 / sizeof(T), KS = 4 * EPC;        // k of one step of a wave
  constexpr int D = DUAL ? 2 : 1;
  __shared__ float red[NW][D][MT * 16][16];
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
  const int n0 = blockIdx.x * 16, n = min(n0 + i, a.N - 1);
  const T* w[D];
  const T* x[MT];
#pragma unroll
  for (int d = 0; d < D; ++d) w[d] = (const T*)a.w[d] + (long)n * a.ldw[d];
#pragma unroll
  for (int u = 0; u < MT; ++u) x[u] = (const T*)a.x + (u * 16 + i < a.M ? (long)(u * 16 + i) * a.ldx : 0);

  f32x4 acc[D][MT];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[d][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave * KS * U; kb < a.K; kb += NW * KS * U) {
    Frag wf[D][U], xf[MT][U];
#pragma unroll
    for (int s = 0; s < U; ++s) {
#pragma unroll
      for (int d = 0; d < D; ++d) wf[d][s] = load_chunk<T, VEC>(w[d], kb + s * KS + kg * EPC, a.K);
#pragma unroll
      for (int u = 0; u < MT; ++u) xf[u][s] = load_chunk<T, VEC>(x[u], kb + s * KS + kg * EPC, a.K);
    }
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[d][u] = Mma<T>::mma(wf[d][s], xf[u][s], acc[d][u]);
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int u = 0; u < MT; ++u) *reinterpret_cast<f32x4*>(&red[wave][d][u * 16 + i][4 * kg]) = acc[d][u];
  __syncthreads();
  const int o = threadIdx.x, m = o >> 4, nn = n0 + (o & 15);
  if (o >= MT * 256 || m >= a.M || nn >= a.N) return;
  float v = 0.f, v1 = 0.f;
#pragma unroll
  for (int q = 0; q < NW; ++q) {
    v += red[q][0][m][o & 15];
    if (DUAL) v1 += red[q][D - 1][m][o & 15];
  }
  float b0, b1;
  load_bias<T, 1>(a.ep, 0, nn, a.N, true, &b0);
  load_bias<T, 1>(a.ep, 1, nn, a.N, true, &b1);
  epilogue_store<T, DUAL, false, 1>(a.ep, 0, m, nn, a.N, true, &v, &v1, &b0, &b1);
}

template <typename T, int MT, bool DUAL> void run_vec(const FewRowsArgs& a, hipStream_t s) {
  const dim3 grid((a.N + 15) / 16), block(NW * 64);
  if (a.vec) hipLaunchKernelGGL((few_rows_kernel<T, MT, DUAL, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((few_rows_kernel<T, MT, DUAL, false>), grid, block, 0, s, a);
}
template <typename T> void run(const FewRowsArgs& a, hipStream_t s) {
  if (a.dual) {
    if (a.M <= 16) run_vec<T, 1, true>(a, s); else run_vec<T, 2, true>(a, s);
  } else {
    if (a.M <= 16) run_vec<T, 1, false>(a, s); else run_vec<T, 2, false>(a, s);
  }
}

// ---- the weights' gradient of few rows: a sum of outer products --------------------------------------------------------------
// Bound by writing the result: 2 M operations an output.  A thread keeps four or eight columns of x in registers, all rows of them, and
// walks down the rows of the result; dz lies in LDS as [row of the result][m] and is read by all lanes at once; a wave writes 64
// such runs.  A tile on the matrix cores would live for one slab and wait for it.  Tiles and this, the activation's gradient
// included: gated 10 x 9408 x 6080 fp32 234 us and 97 (457 MB, 4.7 TB/s), 30 x 4096 x 4096 73 and 49; bf16 1 x 11264 x 4096 57 and
// 51, 10 x 9408 x 6080 72 and 75.
// `two`: both parts of dz are added in fp32 first.
template <typename T, int V, int MR>
__global__ void __launch_bounds__(256) outer_kernel(OuterArgs a) {
  __shared__ __attribute__((aligned(16))) float dz[OUTER_ROWS][MR];
  const int strip = blockIdx.x % a.strips, k = (strip * 256 + threadIdx.x) * V, left = a.K - k, which = blockIdx.y;
  const long n0 = (long)(blockIdx.x / a.strips) * a.rows;
  const int count = (int)min((long)a.rows, a.N - n0);
  const T* src = (const T*)a.dz[which] + n0;
  const float scale = a.scale != nullptr ? *a.scale : 1.f;
  for (int i = threadIdx.x; i < a.rows * MR; i += 256) {
    const int n = i % a.rows, m = i / a.rows;
    float v = 0.f;
    if (m < a.M && n < count) {
      v = to_f(src[m * a.ldd + n]);
      if (a.two) v += to_f(src[(m + a.M) * a.ldd + n]);
      v *= scale;
    }
    dz[n][m] = v;
  }
  float x[MR][V];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    if (m < a.M && left > 0) load_some<T, V>((const T*)a.x + m * a.ldx + k, x[m], left, a.x_vec && left >= V);
    else
#pragma unroll
      for (int e = 0; e < V; ++e) x[m][e] = 0.f;
  }
  __syncthreads();
  if (left <= 0) return;
  T* out = (T*)a.out[which] + n0 * a.K + k;
#pragma unroll 2
  for (int n = 0; n < count; ++n) {
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const float f = dz[n][m];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += f * x[m][e];
    }
    store_some<T, V>(out, v, left, a.out_vec && left >= V);
    out += a.K;
  }
}
// Rows of a workgroup: as many as leave the grid enough workgroups, so that x is read from L2 seldom.
template <typename T, int V, int MR> void run_outer(OuterArgs a, hipStream_t s) {
  a.strips = (a.K + 256 * V - 1) / (256 * V);
  a.rows = OUTER_ROWS;
  while (a.rows > 8 && (long)a.strips * ((a.N + a.rows - 1) / a.rows) * a.nout < (MR <= 8 ? 2048 : 1024)) a.rows /= 2;
  const dim3 grid((unsigned)((long)a.strips * ((a.N + a.rows - 1) / a.rows)), a.nout), block(256);
  hipLaunchKernelGGL((outer_kernel<T, V, MR>), grid, block, 0, s, a);
}
// 16 bytes of columns a thread where its rows of x fit into 128 registers
template <typename T> void run_outer(const OuterArgs& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (a.M <= 1) run_outer<T, V, 1>(a, s);
  else if (a.M <= 4) run_outer<T, V, 4>(a, s);
  else if (a.M <= 8) run_outer<T, V, 8>(a, s);
  else if (a.M <= 12) run_outer<T, V, 12>(a, s);
  else if (a.M <= 16) run_outer<T, V, 16>(a, s);
  else if (a.M <= 24) run_outer<T, 4, 24>(a, s);
  else run_outer<T, 4, 32>(a, s);
}
}  // namespace

void launch_few_rows(int dtype, const FewRowsArgs& a, hipStream_t s) {
  if (dtype == F32) run<float>(a, s);
  else if (dtype == BF16) run<__bf16>(a, s);
  else run<_Float16>(a, s);
  DDL_HIP_CHECK(hipGetLastError());
}

void launch_outer(int dtype, const OuterArgs& a, hipStream_t s) {
  if (dtype == F32) run_outer<float>(a, s);
  else if (dtype == BF16) run_outer<__bf16>(a, s);
  else run_outer<_Float16>(a, s);
  DDL_HIP_CHECK(hipGetLastError());
}

}  // namespace ffn
}  // namespace ddl
