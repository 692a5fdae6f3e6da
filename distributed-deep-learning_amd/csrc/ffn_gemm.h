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
#include <type_traits>

namespace ddl {
namespace ffn {
namespace {
__device__ __attribute__((aligned(16))) const unsigned g_zeros[4] = {0, 0, 0, 0};

// 16 bytes a lane from memory to lds_wave_base + 16 lane.  Written as assembly because the compiler, which cannot tell the buffer
// being filled from the one being read, waits for every such load in front of a transposing LDS read; here the waits are `meet`'s.
// The instruction has no result register; its LDS address goes through m0, which wants one wait state.
__device__ __forceinline__ void load_to_lds(const char* src, char* lds_wave_base) {
  typedef __attribute__((address_space(3))) char lds_char;
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(lds_char*)lds_wave_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(src) : "m0");
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

  // Rounds r, r + CLS, ... of a thread lie a constant distance apart: their swizzles agree.  So it carries CLS pointers.
  static constexpr int STEP_ROWS = THREADS / CPR;          // LDS rows from one round to the next
  static constexpr int CLS = KC && SIDE_P && STEP_ROWS < 32 ? 2 : 1;
  static_assert(ROUNDS == 1 || STEP_ROWS >= (KC ? (SIDE_P ? 16 : 8 * G) : F32 ? 1 : SIDE_P ? 4 : 16), "rounds swizzle differently");
  const char* ptr[CLS];
  int kpos[CLS];                                           // k inside a slab of round 0 (1) of the class
  long stride, step;                                       // bytes between rounds of a class; between slabs
  unsigned ok;                                             // bit r: round r lies inside the operand's rows

  // rows row0 .. of an operand of `rows` rows; b1, ld1: second matrix of a dual operand (rows R/2 ..)
  __device__ __forceinline__ void init(const T* b0, long ld0, const T* b1, long ld1, int row0, int rows, int k0) {
    ok = 0;
    const int first = threadIdx.x / CPR;
    step = KC ? 128 : (long)TK * ld0 * ES;
    stride = (long)CLS * STEP_ROWS * ld0 * ES;
#pragma unroll
    for (int r = 0; r < CLS; ++r) {
      const int lrow = first + r * STEP_ROWS, c = (threadIdx.x % CPR) ^ swizzle(lrow);
      if (KC) {
        kpos[r] = c * EPC;
        ptr[r] = (const char*)(b0 + (long)(row0 + lrow) * ld0 + k0 + kpos[r]);
      } else {
        kpos[r] = lrow;
        ptr[r] = (const char*)(b0 + (long)(k0 + lrow) * ld0 + row0 + c * EPC);
        if (row0 + c * EPC < rows) ok = ~0u;
      }
    }
    if (KC) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) ok |= (row0 + (first + r * STEP_ROWS) % (DUAL ? R / 2 : R) < rows ? 1u : 0u) << r;
    }
    if (DUAL) {                                            // rounds of the second half read b1: same rows, same columns
      lead = ld1 - ld0;
      half = reinterpret_cast<const char*>(b1) - reinterpret_cast<const char*>(b0) - (long)(R / 2) * ld0 * ES + row0 * lead * ES;
    }
  }
  long half, lead;                                         // dual only

  // round r of a slab that lies inside
  __device__ __forceinline__ void stage_round(char* lds, int r) const {
    const char* src = ptr[r % CLS] + (r / CLS) * stride;
    if (DUAL && r * STEP_ROWS >= R / 2) src += half + ((int)(threadIdx.x / CPR) + r * STEP_ROWS - R / 2) * lead * ES;
    load_to_lds(src, lds + (threadIdx.x & ~63) * 16 + r * THREADS * 16);
  }
  __device__ __forceinline__ void advance(long by) {
#pragma unroll
    for (int r = 0; r < CLS; ++r) ptr[r] += by;
  }
  // the slab at the current position, `left` k remaining, with its edges; moves on
  __device__ __forceinline__ void stage(char* lds, int left) {
    char* w = lds + (threadIdx.x & ~63) * 16;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const char* src = ptr[r % CLS] + (r / CLS) * stride;
      if (DUAL && r * STEP_ROWS >= R / 2) src += half + ((int)(threadIdx.x / CPR) + r * STEP_ROWS - R / 2) * lead * ES;
      const int k = KC ? kpos[r % CLS] : kpos[0] + r * STEP_ROWS;
      if (!((ok >> r) & 1) || k >= left) src = (const char*)g_zeros;
      load_to_lds(src, w + r * THREADS * 16);
    }
    advance(step);
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
  // tile t of k half s of the slab at `lds`; w0: the wave's first row
  static __device__ __forceinline__ Frag read_one(const char* lds, int w0, int s, int t) {
    const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
    if constexpr (KC) {
      const int row = row_of(w0, t, i);
      return *reinterpret_cast<const Frag*>(lds + row * 128 + (((s * 4 + kg) ^ swizzle(row)) * 16));
    } else {
      static_assert(!F32, "fp32 tiles are read in groups");
      // columns of this lane's 8 bytes: four consecutive rows of the operand
      const int q = i >> 2, pp = i & 3, col = SIDE_P ? w0 + 16 * pp + 4 * t : w0 + 16 * t + 4 * pp;
      const int k0 = s * 32 + kg * 8 + q, k1 = k0 + 4;
      return read_transposed<T>(lds + k0 * (R * 2) + ((col / 8) ^ swizzle(k0)) * 16 + (col & 4) * 2,
                                lds + k1 * (R * 2) + ((col / 8) ^ swizzle(k1)) * 16 + (col & 4) * 2);
    }
  }
  template <int NT> static __device__ __forceinline__ void read(const char* lds, int w0, int s, Frag (&f)[NT]) {
    if constexpr (F32 && !KC) {
      // one 16-byte read per k covers four tiles (G = 4) or one 8-byte read two (G = 2)
      const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
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
#pragma unroll
      for (int t = 0; t < NT; ++t) f[t] = read_one(lds, w0, s, t);
    }
  }
};

// ---- pieces of the kernels ------------------------------------------------------------------------------------------------
// Tile of this workgroup.  Consecutive workgroup ids go round the 8 XCDs: give each XCD a contiguous run of tiles (its L2 then sees
// neighbours), and walk the tiles in groups of 8 row tiles so that a run shares operands in both directions.
__device__ __forceinline__ void tile_of(int id, int tn, int tm, int& nt, int& mt) {
  const int total = tn * tm, q = total / 8, r = total % 8, x = id % 8;
  id = x * q + (x < r ? x : r) + id / 8;
  constexpr int GROUP = 8;
  const int g0 = id / (GROUP * tn) * GROUP, gm = min(GROUP, tm - g0), in = id - g0 * tn;
  mt = g0 + in % gm;
  nt = in / gm;
}

// Results of a wave: lane holds rows 4 kg + r of each MFMA tile (16 or 2 x 8 consecutive columns of the output), column i (a row of
// the output).  n: first column; aligned: it is a multiple of 8.
template <typename T, typename P, typename Q, bool PKC, bool QKC, bool DUAL, int NT, int MT>
__device__ __forceinline__ void finish(const GemmArgs& a, const f32x4 (&acc)[NT][MT], int n0, int pw0, int m0, int qw0, int which,
                                       int split) {
  const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
  const int n = n0 + pw0 + (DUAL ? 8 : 16) * kg;
  const bool aligned = (n0 & 7) == 0;
  constexpr bool PLAIN = !(PKC && QKC);                    // gradients take neither bias nor activation
  constexpr int V = DUAL ? 8 : 16;
  float b0[V], b1[V];
  if (!PLAIN && a.partial == nullptr) {
    load_bias<T, V>(a.ep, 0, n, a.N, aligned, b0);
    if (DUAL) load_bias<T, V>(a.ep, 1, n, a.N, aligned, b1);
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
    if (a.partial != nullptr) {                            // rows of whole vectors: ldw is N rounded up to 16
      float* d = a.partial + (((long)split * (a.nout * (DUAL ? 2 : 1)) + which) * a.M + m) * a.ldw + n;
      store_some<float, V>(d, v, a.N - n, aligned && n < a.N);
      if (DUAL) store_some<float, V>(d + a.M * a.ldw, v + 8, a.N - n, aligned && n < a.N);
    } else {
      epilogue_store<T, DUAL, PLAIN, V>(a.ep, which, m, n, a.N, aligned, v, v + (DUAL ? 8 : 0), b0, b1);
    }
  }
}

// this wave's LDS reads and loads are done; behind the barrier so are the others'
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                      // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- tiles of any size, with their edges: latency and ragged shapes -------------------------------------------------------
// Double buffered slabs of 128 bytes of k; slab t + 1 is in flight while slab t is multiplied.
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

  const int tm1 = (a.M + BM - 1) / BM;
  int nt, mt;
  tile_of(blockIdx.x, (a.N + TN - 1) / TN, tm1 * a.nout, nt, mt);
  const int which = mt / tm1, m0 = (mt - which * tm1) * BM, n0 = nt * TN, split = blockIdx.y;

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
  auto issue = [&](int slab, int buf) {
    const int seg = slab / slabs, ks = slab - seg * slabs;
    if (slab == s_begin || ks == 0) {
      pop.init((const T*)a.p[seg], a.ldp[seg], (const T*)a.p[1], a.ldp[1], n0, a.N, ks * TK);
      qop.init((const T*)a.q[seg + which], a.ldq[seg + which], nullptr, 0, m0, a.M, ks * TK);
    }
    pop.stage(lds + buf * SLAB, a.K - ks * TK);
    qop.stage(lds + buf * SLAB + P::BYTES, a.K - ks * TK);
  };
  if (s_begin < s_end) {
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
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        typename P::Frag pf[NT];
        typename Q::Frag qf[MT];
        P::template read<NT>(lds + buf * SLAB, pw0, s, pf);
        Q::template read<MT>(lds + buf * SLAB + P::BYTES, qw0, s, qf);
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][u] = Mma<T>::mma(pf[t], qf[u], acc[t][u]);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();                        // everyone has read this slab: it may be overwritten
    }
  }
  finish<T, P, Q, PKC, QKC, DUAL, NT, MT>(a, acc, n0, pw0, m0, qw0, which, split);
}

// ---- 256 x 256 tiles of 16-bit operands -------------------------------------------------------------------------------------
// Bound by the matrix cores; what keeps them from their rate is everything that is not a product between two barriers.  So the
// loop over slabs is one block of straight-line code with ONE barrier, in which the LDS reads and the loads are dealt out between
// the products:
//   half 0's products   beside   the LDS reads of half 1
//   -- all waves have read this slab, and the next one has landed --
//   half 1's products   beside   the LDS reads of the next slab's half 0 and the loads of the slab after it
// P's registers are double, Q's mostly single: a Q tile is replaced right behind its last product.  The last two tiles are double
// too, so that the reads end before the products do and the wait in front of the barrier finds them done.
// No edges in the loop: the slab with the end of k comes first (the order of a sum is free), and a tile that would reach beyond the
// output is moved back inside (it computes some results a second time; both writers hold the same bits).  So N and M are at
// least a tile.  The second contraction segment has the first one's strides and is reached by a jump.
template <typename T, bool PKC, bool QKC, bool DUAL>
__global__ void __launch_bounds__(512) gemm_big_kernel(GemmArgs a) {
  constexpr int BN = 256, BM = 256, THREADS = 512, WN = 4, NT = 4, MT = 8, DBL = 2, SNG = MT - DBL;
  constexpr int TN = DUAL ? BN / 2 : BN, EPC = 16 / sizeof(T);
  using P = Operand<T, BN, THREADS, PKC, true, DUAL, 4>;
  using Q = Operand<T, BM, THREADS, QKC, false, false, 1>;
  constexpr int TK = P::TK, SLAB = P::BYTES + Q::BYTES;
  static_assert(P::ROUNDS == 4 && Q::ROUNDS == 4 && P::CLS == 1 && Q::CLS == 1, "one load of the slab per row of products");
  __shared__ __attribute__((aligned(1024))) char lds[2 * SLAB];

  const int tm1 = (a.M + BM - 1) / BM;
  int nt, mt;
  tile_of(blockIdx.x, (a.N + TN - 1) / TN, tm1 * a.nout, nt, mt);
  const int which = mt / tm1, split = blockIdx.y;
  auto inside = [&](int at, int size, int extent, bool kc) {         // k-strided rows are padded to whole chunks
    const int e = kc ? extent : (extent + EPC - 1) / EPC * EPC;
    return at + size > e ? e - size : at;
  };
  const int n0 = inside(nt * TN, TN, a.N, PKC), m0 = inside((mt - which * tm1) * BM, BM, a.M, QKC);

  // slabs in order: the partial ones of each segment, then the full ones of the first and of the second
  const int full = a.K / TK, tails = a.K % TK ? a.nseg : 0, all = tails + full * a.nseg;
  const int per = (all + a.splits - 1) / a.splits, s_begin = split * per, s_end = min(all, s_begin + per);
  const int wave = threadIdx.x >> 6, wn = wave % WN, wm = wave / WN;
  const int pw0 = DUAL ? wn * 32 : wn * 64, qw0 = wm * (BM / 2);

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  P pop;
  Q qop;
  auto seek = [&](int slab) {
    const bool tail = slab < tails;
    const int seg = tail ? slab : full > 0 ? (slab - tails) / full : 0, k0 = (tail ? full : slab - tails - seg * full) * TK;
    pop.init((const T*)a.p[seg], a.ldp[seg], (const T*)a.p[1], a.ldp[1], n0, a.N, k0);
    qop.init((const T*)a.q[seg + which], a.ldq[seg + which], nullptr, 0, m0, a.M, k0);
    return a.K - k0;
  };
  typename P::Frag pf[2][NT];
  typename Q::Frag q1[SNG], q2[2][DBL];
  auto products = [&](int s, int u) {
    const typename Q::Frag q = u < SNG ? q1[u < SNG ? u : 0] : q2[s][u < SNG ? 0 : u - SNG];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][u] = Mma<T>::mma(pf[s][t], q, acc[t][u]);
  };
  // half s's products of the slab in buffer `buf`; NEXT: read the following half (of this slab, or of the other buffer's);
  // LOAD: fill this buffer anew
  auto phase = [&](auto half, auto with_next, auto with_load, int buf) {
    constexpr int s = decltype(half)::value;
    constexpr bool NEXT = decltype(with_next)::value, LOAD = decltype(with_load)::value;
    const char* next = lds + (s == 0 ? buf : buf ^ 1) * SLAB;
    char* load = lds + buf * SLAB;
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      if constexpr (NEXT) {
        if (u < NT) pf[s ^ 1][u] = P::read_one(next, pw0, s ^ 1, u);
        if (u < DBL) q2[s ^ 1][u] = Q::read_one(next + P::BYTES, qw0, s ^ 1, SNG + u);
      }
      if constexpr (LOAD) {
        if (u < 4) pop.stage_round(load, u);
        else qop.stage_round(load + P::BYTES, u - 4);
      }
      products(s, u);
      if constexpr (NEXT) {
        if (u < SNG) q1[u] = Q::read_one(next + P::BYTES, qw0, s ^ 1, u);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, 0> H0{};
  constexpr std::integral_constant<int, 1> H1{};
  constexpr std::true_type YES{};
  constexpr std::false_type NO{};
  const int count = s_end - s_begin;
  if (count > 0) {
    int left = seek(s_begin);
    pop.stage(lds, left);
    qop.stage(lds + P::BYTES, left);
    if (count > 1) {
      left = seek(s_begin + 1);
      pop.stage(lds + SLAB, left);
      qop.stage(lds + SLAB + P::BYTES, left);
    }
    meet();
    P::template read<NT>(lds, pw0, 0, pf[0]);
#pragma unroll
    for (int u = 0; u < SNG; ++u) q1[u] = Q::read_one(lds + P::BYTES, qw0, 0, u);
#pragma unroll
    for (int u = 0; u < DBL; ++u) q2[0][u] = Q::read_one(lds + P::BYTES, qw0, 0, SNG + u);
    int buf = 0;
    if (count > 2) {
      seek(s_begin + 2);
      // slabs until the jump to the second segment (0: none), and its distance from where the first one ends
      int to_jump = a.nseg == 2 ? tails + full - (s_begin + 2) : 0;
      const long p_jump = a.nseg == 2 ? (const char*)a.p[1] - (const char*)a.p[0] - full * pop.step : 0;
      const long q_jump = a.nseg == 2 ? (const char*)a.q[1] - (const char*)a.q[0] - full * qop.step : 0;
      for (int i = 0; i < count - 2; ++i) {
        phase(H0, YES, NO, buf);
        meet();
        phase(H1, YES, YES, buf);
        const bool jump = --to_jump == 0;
        pop.advance(pop.step + (jump ? p_jump : 0));
        qop.advance(qop.step + (jump ? q_jump : 0));
        buf ^= 1;
      }
    }
    phase(H0, YES, NO, buf);
    if (count > 1) {
      meet();
      phase(H1, YES, NO, buf);
      buf ^= 1;
      phase(H0, YES, NO, buf);
    }
    phase(H1, NO, NO, buf);
  }
  finish<T, P, Q, PKC, QKC, DUAL, NT, MT>(a, acc, n0, pw0, m0, qw0, which, split);
}

template <typename T, int BN, int BM, int WN, int WM> void run_cfg(const GemmArgs& a, hipStream_t s) {
  const long tn = (a.N + (a.dual ? BN / 2 : BN) - 1) / (a.dual ? BN / 2 : BN), tm = (long)((a.M + BM - 1) / BM) * a.nout;
  const dim3 grid((unsigned)(tn * tm), (unsigned)a.splits), block(WN * WM * 64);
  if (a.dual) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, true, true, true>), grid, block, 0, s, a);
  else if (a.p_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, true, true, false>), grid, block, 0, s, a);
  else if (a.q_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, false, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, false, false, false>), grid, block, 0, s, a);
}
template <typename T> void run_big(const GemmArgs& a, hipStream_t s) {
  const int tn = a.dual ? 128 : 256;
  const dim3 grid((unsigned)((long)((a.N + tn - 1) / tn) * ((a.M + 255) / 256) * a.nout), (unsigned)a.splits), block(512);
  if (a.dual) hipLaunchKernelGGL((gemm_big_kernel<T, true, true, true>), grid, block, 0, s, a);
  else if (a.p_kc) hipLaunchKernelGGL((gemm_big_kernel<T, true, true, false>), grid, block, 0, s, a);
  else if (a.q_kc) hipLaunchKernelGGL((gemm_big_kernel<T, false, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_big_kernel<T, false, false, false>), grid, block, 0, s, a);
}
}  // namespace
}  // namespace ffn
}  // namespace ddl
