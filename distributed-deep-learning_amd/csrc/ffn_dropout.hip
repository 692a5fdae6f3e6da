// Dropout whose mask is never stored: element e of a call stays iff word e % 4 of Philox4x32-7 at counter (e / 4, call) under
// the key `seed` is at least p 2^32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011;
// seven rounds is the smallest count the paper reports as passing every statistical test).  The backward pass draws the same words
// again, so training keeps 16 bytes of key instead of a mask.
//
// Bound by memory: one read (two with the residual) and one write per element.  Four elements share one generator block; seven
// rounds are 14 32 x 32 -> 64 bit multiplies, which run at a quarter of the fp32 rate.  16384 x 8192 bf16: 124 us (4.3 TB/s; the
// multiplies show), with the residual 159 us (5.1 TB/s, the rate of a copy).
#include "ffn_common.h"
#include "ffn_misc.h"
#include "ddl_kernels.h"

namespace ddl {
namespace ffn {
namespace {

struct Key { unsigned s0, s1, c0, c1; };

__device__ __forceinline__ void philox7(const Key& k, unsigned long long block, unsigned (&w)[4]) {
  unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = k.c0, c3 = k.c1, k0 = k.s0, k1 = k.s1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long a = 0xD2511F53ull * c0, b = 0xCD9E8D57ull * c2;
    const unsigned n0 = (unsigned)(b >> 32) ^ c1 ^ k0, n2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c1 = (unsigned)b;
    c3 = (unsigned)a;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// V elements from element e (a multiple of 4 and of V); n: how many of them exist
template <typename T, int V, bool RES, bool VEC>
__device__ __forceinline__ void drop_some(const T* x, const T* res, T* y, long e, int n, const Key& key, unsigned threshold,
                                          bool none, float scale) {
  float v[V], r[V];
  load_some<T, V>(x + e, v, n, VEC && n >= V);
  if (RES) load_some<T, V>(res + e, r, n, VEC && n >= V);
#pragma unroll
  for (int b = 0; b < V / 4; ++b) {
    unsigned w[4];
    philox7(key, (unsigned long long)e / 4 + b, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // a dropped element contributes zero whatever it holds: an infinity or NaN in it does not pass
      const float kept = !none && w[i] >= threshold ? v[4 * b + i] * scale : 0.f;
      v[4 * b + i] = RES ? r[4 * b + i] + kept : kept;
    }
  }
  store_some<T, V>(y + e, v, n, VEC && n >= V);
}

template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
                                                      long n, const long long* __restrict__ key_t, unsigned threshold,
                                                      bool none, float scale) {
  constexpr int V = 16 / sizeof(T);
  const unsigned long long seed = (unsigned long long)key_t[0], call = (unsigned long long)key_t[1];
  const Key key = {(unsigned)seed, (unsigned)(seed >> 32), (unsigned)call, (unsigned)(call >> 32)};
  const long stride = (long)gridDim.x * 256 * V;
  for (long e = ((long)blockIdx.x * 256 + threadIdx.x) * V; e < n; e += stride) {
    const long left = n - e;
    drop_some<T, V, RES, VEC>(x, res, y, e, left < V ? (int)left : V, key, threshold, none, scale);
  }
}

// keys[i] = (seed, call + i), call += n.  One atomic add: calls from several streams take disjoint ranges.
__global__ void rng_keys_kernel(long long* __restrict__ state, long long* __restrict__ keys, int n) {
  __shared__ unsigned long long base;
  if (threadIdx.x == 0) base = atomicAdd((unsigned long long*)state + 1, (unsigned long long)n);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 64) {
    keys[2 * i] = state[0];
    keys[2 * i + 1] = (long long)(base + i);
  }
}

template <typename T> void run(const DropoutArgs& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const long items = (a.n + V - 1) / V;
  long g = (items + 255) / 256;
  if (g > 256 * 16) g = 256 * 16;
  const dim3 grid((unsigned)g), block(256);
  const T *x = (const T*)a.x, *r = (const T*)a.residual;
  T* y = (T*)a.y;
  auto al = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const bool vec = al(a.x) && al(a.residual) && al(a.y);
  const unsigned long long thr = (unsigned long long)(a.p * 4294967296.0);
  const bool none = thr > 0xffffffffull;                   // p = 1
  const float scale = none ? 0.f : (float)(1.0 / (1.0 - a.p));
#define DDL_DROP(RES, VEC)                                                                                            \
  hipLaunchKernelGGL((dropout_kernel<T, RES, VEC>), grid, block, 0, s, x, r, y, a.n, (const long long*)a.key, (unsigned)thr, \
                     none, scale)
  if (r != nullptr) { if (vec) DDL_DROP(true, true); else DDL_DROP(true, false); }
  else { if (vec) DDL_DROP(false, true); else DDL_DROP(false, false); }
#undef DDL_DROP
  DDL_HIP_CHECK(hipGetLastError());
}
}  // namespace

void launch_dropout(int dtype, const DropoutArgs& a, hipStream_t s) {
  if (a.n <= 0) return;
  if (dtype == F32) run<float>(a, s);
  else if (dtype == BF16) run<__bf16>(a, s);
  else run<_Float16>(a, s);
}

void launch_rng_keys(int64_t* state, int64_t* keys, int n, hipStream_t s) {
  hipLaunchKernelGGL(rng_keys_kernel, dim3(1), dim3(64), 0, s, (long long*)state, (long long*)keys, n);
  DDL_HIP_CHECK(hipGetLastError());
}

}  // namespace ffn
}  // namespace ddl
