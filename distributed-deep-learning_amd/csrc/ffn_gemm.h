// Matrix products of the feed-forward operators on the CDNA4 matrix cores, one translation unit per element type
// (ffn_gemm_{f32,bf16,f16}.hip include this and instantiate the kernels).
//
//   out[m][n] = epilogue( sum_k P(n, k) Q(m, k) )
//
// P sits on the A side of the MFMA and Q on the B side, so that a lane's accumulators are 16 CONSECUTIVE outputs of one row
// (rows n of a wave are dealt to the MFMA's A rows as n = 16 (i / 4) + 4 t + i % 4 for tile t): bias, residual and result move
// as 16-byte vectors without a detour through LDS.
//
// Tiles: LDS holds a 128-byte wide k slab (64 values of 16 bits, 32 of fp32) of both operands, filled by direct
// global -> LDS loads of 16 bytes a lane, double buffered: slab t+1 is in flight while slab t is multiplied.  A lane whose
// 16 bytes lie outside the operand reads a block of zeros in global memory instead, so edges cost no branch and no
// masked arithmetic, and an infinity beyond the edge cannot turn into NaN.
// LDS image of a k-contiguous operand: [row][8 chunks of 16 B]; of a k-strided one: [k][rows].  Chunks are permuted inside a
// row by an XOR with bits of the row (applied to the global address, since the direct loads write LDS linearly) so that the
// operand reads spread over the banks.  16-bit k-strided operands are read with the transposing ds_read_b64_tr_b16.
#pragma once
#include "ffn_common.h"
#include "ffn_mma.h"

namespace ddl {
namespace ffn {
namespace {
__device__ __attribute__((aligned(16))) const unsigned g_zeros[4] = {0, 0, 0, 0};

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
__device__ __forceinline__ void load_to_lds(const char* src, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((glb_void*)src, (lds_void*)lds_wave_base, 16, 0, 0);
}

// 4 k x 16 columns of 16-bit values, transposed: the lane's 8 bytes in, four k of one column out (two of them)
template <typename T> __device__ __forceinline__ typename Mma<T>::Frag read_transposed(const char* a, const char* b) {
  typedef __attribute__((address_space(3))) i16x4 L;
  const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)b);
  return __builtin_bit_cast(typename Mma<T>::Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- one operand's staging and reading -----------------------------------------------------------------------------
// R: rows of the tile; G: how the wave's tiles are dealt to rows (see `row_of`); SIDE_P: the A side
template <typename T, int R, int THREADS, bool KC, bool SIDE_P, bool DUAL, int G>
struct Operand {
  static constexpr int ES = sizeof(T), EPC = 16 / ES, TK = 128 / ES;
  static constexpr int CPR = KC ? 8 : R * ES / 16;         // 16-byte chunks per LDS row
  static constexpr int ROUNDS = R * 8 / THREADS;           // chunks each thread moves per slab
  static constexpr int BYTES = R * 128;
  static_assert(ROUNDS >= 1 && R * 8 % THREADS == 0, "tile / workgroup size");
  static constexpr bool F32 = ES == 4;

  static __device__ __forceinline__ int swizzle(int row) {
    if (KC) {
      if (SIDE_P) return DUAL ? (row & 3) | ((row >> 3) & 1) << 2 : (row & 3) | ((row >> 4) & 1) << 2;
      return F32 && G > 1 ? (row / G) & 7 : row & 7;
    }
    if (F32) return 0;                                     // 16 lanes read 256 contiguous bytes of one k
    if (SIDE_P) return ((row & 1) | ((row >> 1) & 1) << 3) & (CPR - 1);
    return ((row & 3) << 1 | ((row >> 3) & 1) << 3) & (CPR - 1);
  }

  const char* ptr[ROUNDS];
  bool ok[ROUNDS];
  int kpos[ROUNDS];                                        // k of the chunk (k-contiguous: its first k) inside a slab
  long step;

  // rows row0 .. of an operand of `rows` rows; b1, ld1: second matrix of a dual operand (rows R/2 ..)
  __device__ __forceinline__ void init(const T* b0, long ld0, const T* b1, long ld1, int row0, int rows, int k0) {
    step = KC ? 128 : (long)TK * ld0 * ES;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int idx = r * THREADS + threadIdx.x, lrow = idx / CPR, c = (idx % CPR) ^ swizzle(lrow);
      const T* base = b0;
      long ld = ld0;
      int row;
      if (KC) {
        row = row0 + lrow;
        if (DUAL && lrow >= R / 2) { base = b1; ld = ld1; row = row0 + lrow - R / 2; }
        kpos[r] = c * EPC;
        ptr[r] = (const char*)(base + (long)row * ld + k0 + kpos[r]);
      } else {
        row = row0 + c * EPC;
        kpos[r] = lrow;
        ptr[r] = (const char*)(base + (long)(k0 + lrow) * ld + row);
      }
      ok[r] = row < rows;
    }
  }
  // issue the loads of the slab at the current position, `left` k remaining, and move on
  __device__ __forceinline__ void stage(char* lds, int left) {
    char* w = lds + (threadIdx.x & ~63) * 16;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const char* src = ok[r] && kpos[r] < left ? ptr[r] : (const char*)g_zeros;
      load_to_lds(src, w + r * THREADS * 16);
      ptr[r] += step;
    }
  }

  // rows of the operand that lane index i (0..15) of tile t stands for, inside a wave's rows starting at w0
  static __device__ __forceinline__ int row_of(int w0, int t, int i) {
    if (SIDE_P) {
      if (DUAL) return (t >= 2 ? R / 2 : 0) + w0 + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
      if (F32 && !KC) return w0 + 4 * i + t;
      return w0 + 16 * (i >> 2) + 4 * t + (i & 3);
    }
    if (F32) return w0 + 16 * G * (t / G) + G * i + t % G;
    return w0 + 16 * t + i;
  }

  using Frag = typename Mma<T>::Frag;
  // operand of k step s (half of the slab); `lds` is the slab, w0 the wave's first row
  template <int NT> static __device__ __forceinline__ void read(const char* lds, int w0, int s, Frag (&f)[NT]) {
    const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
    if (KC) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int row = row_of(w0, t, i);
        f[t] = *reinterpret_cast<const Frag*>(lds + row * 128 + (((s * 4 + kg) ^ swizzle(row)) * 16));
      }
    } else if constexpr (F32) {
      // one 16-byte read per k covers four tiles (G = 4) or one 8-byte read two (G = 2)
#pragma unroll
      for (int t = 0; t < NT; t += G) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = s * 16 + kg * 4 + e;
          const float* p = reinterpret_cast<const float*>(lds + k * (R * 4)) + row_of(w0, t, i);
#pragma unroll
          for (int j = 0; j < G; ++j) f[t + j][e] = p[j];
        }
      }
    } else {
      const int q = i >> 2, pp = i & 3;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // columns of this lane's 8 bytes: four consecutive rows of the operand
        const int col = SIDE_P ? w0 + 16 * pp + 4 * t : w0 + 16 * t + 4 * pp;
        const int k0 = s * 32 + kg * 8 + q, k1 = k0 + 4;
        const char* a = lds + k0 * (R * 2) + ((col / 8) ^ swizzle(k0)) * 16 + (col & 4) * 2;
        const char* b = lds + k1 * (R * 2) + ((col / 8) ^ swizzle(k1)) * 16 + (col & 4) * 2;
        f[t] = read_transposed<T>(a, b);
      }
    }
  }
};

// ---- the kernel ---------------------------------------------------------------------------------------------------------
template <typename T, int BN, int BM, int WN, int WM, bool PKC, bool QKC, bool DUAL>
__global__ void __launch_bounds__(WN * WM * 64) gemm_kernel(GemmArgs a) {
  constexpr int THREADS = WN * WM * 64;
  constexpr int NT = BN / WN / 16, MT = BM / WM / 16;
  static_assert(NT == 4, "a wave covers 64 rows of P");
  static_assert(!DUAL || PKC, "dual products: k-contiguous weights");
  constexpr int G = sizeof(T) == 4 ? (MT >= 4 ? 4 : MT) : 1;
  constexpr int TN = DUAL ? BN / 2 : BN;                   // output columns of a tile
  using P = Operand<T, BN, THREADS, PKC, true, DUAL, 4>;
  using Q = Operand<T, BM, THREADS, QKC, false, false, G>;
  constexpr int TK = P::TK, SLAB = P::BYTES + Q::BYTES;
  __shared__ __attribute__((aligned(1024))) char lds[2 * SLAB];

  // tile of this workgroup.  Consecutive workgroup ids go round the 8 XCDs: give each XCD a contiguous run of tiles (its L2
  // then sees neighbours), and walk the tiles in groups of 8 row tiles so that a run shares operands in both directions.
  const int tn = (a.N + TN - 1) / TN, tm1 = (a.M + BM - 1) / BM, tm = tm1 * a.nout;
  const int total = tn * tm;
  int id = blockIdx.x;
  {
    const int q = total / 8, r = total % 8, x = id % 8;
    id = x * q + (x < r ? x : r) + id / 8;
  }
  constexpr int GROUP = 8;
  const int g0 = id / (GROUP * tn) * GROUP, gm = min(GROUP, tm - g0), in = id - g0 * tn;
  const int mt_all = g0 + in % gm, nt_ = in / gm;
  const int which = mt_all / tm1, m0 = (mt_all - which * tm1) * BM, n0 = nt_ * TN;
  const int split = blockIdx.y;

  // contraction: a.nseg segments of `slabs` slabs each; this split takes [s_begin, s_end) of all of them
  const int slabs = (a.K + TK - 1) / TK, all = slabs * a.nseg;
  const int per = (all + a.splits - 1) / a.splits, s_begin = split * per, s_end = min(all, s_begin + per);

  const int wave = threadIdx.x >> 6, wn = wave % WN, wm = wave / WN;
  const int pw0 = DUAL ? wn * 32 : wn * 64, qw0 = wm * (BM / WM);

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  P pop;
  Q qop;
  auto seek = [&](int slab) {                              // position both operands at a global slab index
    const int seg = slab / slabs, k0 = (slab - seg * slabs) * TK;
    pop.init((const T*)a.p[seg], a.ldp[seg], (const T*)a.p[1], a.ldp[1], n0, a.N, k0);
    qop.init((const T*)a.q[seg + which], a.ldq[seg + which], nullptr, 0, m0, a.M, k0);
  };
  auto issue = [&](int slab, int buf) {
    const int seg = slab / slabs, ks = slab - seg * slabs;
    if (slab != s_begin && ks == 0) seek(slab);            // the next segment
    const int left = a.K - ks * TK;
    pop.stage(lds + buf * SLAB, left);
    qop.stage(lds + buf * SLAB + P::BYTES, left);
  };
  if (s_begin < s_end) {
    seek(s_begin);
    issue(s_begin, 0);
    for (int slab = s_begin; slab < s_end; ++slab) {
      const int buf = (slab - s_begin) & 1;
      if (slab + 1 < s_end) {
        issue(slab + 1, buf ^ 1);
        __builtin_amdgcn_s_waitcnt(0xF70 | ((P::ROUNDS + Q::ROUNDS) & 15));    // vmcnt: slab's loads have landed
      } else {
        __builtin_amdgcn_s_waitcnt(0xF70);
      }
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const char* ps = lds + buf * SLAB;
      const char* qs = ps + P::BYTES;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        typename P::Frag pf[NT];
        typename Q::Frag qf[MT];
        P::template read<NT>(ps, pw0, s, pf);
        Q::template read<MT>(qs, qw0, s, qf);
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][u] = Mma<T>::mma(pf[t], qf[u], acc[t][u]);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();                        // everyone has read this slab: it may be overwritten
    }
  }

  // lane: rows 4 kg + r of each MFMA tile (columns of the output), column i (a row of the output)
  const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
  const int n = n0 + pw0 + (DUAL ? 8 : 16) * kg;
  constexpr bool PLAIN = !(PKC && QKC);                    // gradients take neither bias nor activation
  constexpr int V = DUAL ? 8 : 16;
  float b0[V], b1[V];
  if (!PLAIN) {
    load_bias<T, V>(a.ep, 0, n, a.N, b0);
    if (DUAL) load_bias<T, V>(a.ep, 1, n, a.N, b1);
  }
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int m = m0 + Q::row_of(qw0, u, i);
    if (m >= a.M) continue;
    float v[16];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[(sizeof(T) == 4 && !PKC) ? 4 * r + t : 4 * t + r] = acc[t][u][r];
    if (a.partial != nullptr) {
      if (n < a.N) {                                       // ldw is N rounded up to 16: whole vectors stay inside a row
        float* d = a.partial + (((long)split * (a.nout * (DUAL ? 2 : 1)) + which) * a.M + m) * a.ldw + n;
        store_vec<float, V>(d, v);
        if (DUAL) store_vec<float, V>(d + a.M * a.ldw, v + 8);
      }
    } else {
      epilogue_store<T, DUAL, PLAIN, V>(a.ep, which, m, n, a.N, v, v + (DUAL ? 8 : 0), b0, b1);
    }
  }
}

template <typename T, int BN, int BM, int WN, int WM> void run_cfg(const GemmArgs& a, hipStream_t s) {
  const long tn = (a.N + (a.dual ? BN / 2 : BN) - 1) / (a.dual ? BN / 2 : BN), tm = (long)((a.M + BM - 1) / BM) * a.nout;
  const dim3 grid((unsigned)(tn * tm), (unsigned)a.splits), block(WN * WM * 64);
  if (a.dual) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, true, true, true>), grid, block, 0, s, a);
  else if (a.p_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, true, true, false>), grid, block, 0, s, a);
  else if (a.q_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, false, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, false, false, false>), grid, block, 0, s, a);
}
}  // namespace
}  // namespace ffn
}  // namespace ddl
