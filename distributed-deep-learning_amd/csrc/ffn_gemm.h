// Matrix products of the feed-forward operators on the CDNA4 matrix cores, one translation unit per element type
// (ffn_gemm_{f32,bf16,f16}.hip include this and instantiate the kernels).
//
//   out[m][n] = epilogue( sum_k P(n, k) Q(m, k) )
//
// P sits on the A side of the MFMA and Q on the B side, so that a lane's accumulators are consecutive outputs of one row, 16 bytes of
// them, and four lanes hold 64 bytes: 16 bits: rows n of a wave are dealt to the MFMA's A rows as n = 32 (t / 2) + 8 (i / 4) +
// 4 (t % 2) + i % 4 for tile t, so that a pair of tiles gives eight values; fp32: n = 16 t + i, four values a tile.  Bias, residual
// and result move as such vectors without a detour through LDS.
//
// Tiles: LDS holds 128-byte wide k slabs (64 values of 16 bits, 32 of fp32) of both operands in a ring of two or three, filled by
// direct global -> LDS loads of 16 bytes a lane: the next slabs are in flight while one is multiplied.  A lane whose
// 16 bytes lie outside the operand reads a block of zeros in global memory instead, so edges cost no masked
// arithmetic, and an infinity beyond the edge cannot turn into NaN.
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
// R: rows of the tile; SIDE_P: the A side
template <typename T, int R, int THREADS, bool KC, bool SIDE_P, bool DUAL>
struct Operand {
  static constexpr int ES = sizeof(T), EPC = 16 / ES, TK = 128 / ES;
  static constexpr int CPR = KC ? 8 : R * ES / 16;         // 16-byte chunks per LDS row
  static constexpr int ROUNDS = R * 8 / THREADS;           // chunks each thread moves per slab
  static constexpr int BYTES = R * 128;
  static_assert(ROUNDS >= 1 && R * 8 % THREADS == 0, "tile / workgroup size");
  static constexpr bool F32 = ES == 4;
  static_assert((THREADS & (THREADS - 1)) == 0, "groups of threads");
  static __device__ __forceinline__ int tid() { return (int)threadIdx.x & (THREADS - 1); }     // in the group that stages a slab

  // bits of the LDS row that differ between the lanes of one read place the 16-byte chunks
  static __device__ __forceinline__ int swizzle(int row) {
    if (KC) return SIDE_P && !F32 ? (row & 3) | ((row >> 3) & 1) << 2 : row & 7;
    if (F32) return 0;                                     // 16 lanes read 64 contiguous bytes of one k
    if (SIDE_P) return ((row & 3) << 2) & (CPR - 1);
    return ((row & 3) << 1 | ((row >> 3) & 1) << 3) & (CPR - 1);
  }

  // Rounds r, r + CLS, ... of a thread lie a constant distance apart: their swizzles agree.  So it carries CLS pointers.
  static constexpr int STEP_ROWS = THREADS / CPR;          // LDS rows from one round to the next
  static constexpr int CLS = KC && STEP_ROWS < 16 ? 2 : 1;
  static_assert(ROUNDS == 1 || STEP_ROWS >= (KC ? (SIDE_P && !F32 ? 16 : 8) : F32 ? 1 : SIDE_P ? 4 : 16), "rounds swizzle differently");
  static_assert(!DUAL || STEP_ROWS <= R / 2, "a round of a dual operand lies in one of its matrices");
  const char* ptr[CLS];
  int kpos[CLS];                                           // k inside a slab of round 0 (1) of the class
  long stride, step;                                       // bytes between rounds of a class; between slabs
  unsigned ok;                                             // bit r: round r lies inside the operand's rows

  // rows row0 .. of an operand of `rows` rows; b1, ld1: second matrix of a dual operand (rows R/2 ..)
  __device__ __forceinline__ void init(const T* b0, long ld0, const T* b1, long ld1, int row0, int rows, int k0) {
    ok = 0;
    const int first = tid() / CPR;
    step = KC ? 128 : (long)TK * ld0 * ES;
    stride = (long)CLS * STEP_ROWS * ld0 * ES;
#pragma unroll
    for (int r = 0; r < CLS; ++r) {
      const int lrow = first + r * STEP_ROWS, c = (tid() % CPR) ^ swizzle(lrow);
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
    if (DUAL && r * STEP_ROWS >= R / 2) src += half + (tid() / CPR + r * STEP_ROWS - R / 2) * lead * ES;
    load_to_lds(src, lds + (tid() & ~63) * 16 + r * THREADS * 16);
  }
  __device__ __forceinline__ void advance(long by) {
#pragma unroll
    for (int r = 0; r < CLS; ++r) ptr[r] += by;
  }
  // the slab at the current position, `left` k remaining, with its edges; moves on
  __device__ __forceinline__ void stage(char* lds, int left) {
    char* w = lds + (tid() & ~63) * 16;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const char* src = ptr[r % CLS] + (r / CLS) * stride;
      if (DUAL && r * STEP_ROWS >= R / 2) src += half + (tid() / CPR + r * STEP_ROWS - R / 2) * lead * ES;
      const int k = KC ? kpos[r % CLS] : kpos[0] + r * STEP_ROWS;
      if (!((ok >> r) & 1) || k >= left) src = (const char*)g_zeros;
      load_to_lds(src, w + r * THREADS * 16);
    }
    advance(step);
  }
  static __device__ __forceinline__ void stage_zeros(char* lds) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) load_to_lds((const char*)g_zeros, lds + (tid() & ~63) * 16 + r * THREADS * 16);
  }
  // the same where nothing lies outside
  __device__ __forceinline__ void stage_inside(char* lds) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) stage_round(lds, r);
    advance(step);
  }

  // rows of the operand that lane index i (0..15) of tile t stands for, inside a wave's rows starting at w0
  static __device__ __forceinline__ int row_of(int w0, int t, int i) {
    if (SIDE_P) {
      if (DUAL && t >= 2) { w0 += R / 2; t -= 2; }
      return F32 ? w0 + 16 * t + i : w0 + 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
    }
    return w0 + 16 * t + i;
  }

  using Frag = typename Mma<T>::Frag;
  // tile t of k half s of the slab at `lds`; w0: the wave's first row
  static __device__ __forceinline__ Frag read_one(const char* lds, int w0, int s, int t) {
    const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
    if constexpr (KC) {
      const int row = row_of(w0, t, i);
      return *reinterpret_cast<const Frag*>(lds + row * 128 + (((s * 4 + kg) ^ swizzle(row)) * 16));
    } else if constexpr (F32) {
      Frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = reinterpret_cast<const float*>(lds + (s * 16 + kg * 4 + e) * (R * 4))[row_of(w0, t, i)];
      return f;
    } else {
      // columns of this lane's 8 bytes: four consecutive rows of the operand
      const int q = i >> 2, pp = i & 3, col = SIDE_P ? w0 + 32 * (t >> 1) + 8 * pp + 4 * (t & 1) : w0 + 16 * t + 4 * pp;
      const int k0 = s * 32 + kg * 8 + q, k1 = k0 + 4;
      return read_transposed<T>(lds + k0 * (R * 2) + ((col / 8) ^ swizzle(k0)) * 16 + (col & 4) * 2,
                                lds + k1 * (R * 2) + ((col / 8) ^ swizzle(k1)) * 16 + (col & 4) * 2);
    }
  }
  template <int NT> static __device__ __forceinline__ void read(const char* lds, int w0, int s, Frag (&f)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) f[t] = read_one(lds, w0, s, t);
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

// What lanes of this wave wrote to LDS before is what its other lanes read behind.  LDS serves a wave in order, so this costs no
// instruction: it keeps the compiler from moving one lane's read in front of another's write, of which it cannot know.
__device__ __forceinline__ void wave_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Results of a wave: lane holds rows 4 kg + r of each MFMA tile, i.e. V consecutive columns of the output for every tile (fp32) or pair
// of tiles (16 bits), and column i (a row of the output).  Dual products: the upper half of the tiles belongs to the second weight.
// CHUNK > 0: the sums go through LDS, CHUNK of the wave's row tiles at a time, so that one piece of code serves them in a loop: unrolled over
// all of them with the activations inside, it outgrows the instruction cache, and a tile waits for its code (8192 x 4096 x 4096 bf16 with
// gelu and residual: 285 us unrolled, 252 so).  The ring is no longer read then; `lds` is this wave's part: each lane reads back what it
// wrote, and where the kept sums of a dual product are stored by rows, what other lanes of the wave wrote.
template <typename T, typename P, typename Q, bool PKC, bool QKC, bool DUAL, int NT, int MT, int CHUNK>
__device__ __forceinline__ void finish(const GemmArgs& a, const f32x4 (&acc)[NT][MT], int n0, int pw0, int m0, int qw0, int which,
                                       int split, char* lds) {
  constexpr bool PLAIN = !(PKC && QKC);                    // gradients take neither bias nor activation
  constexpr int V = 16 / sizeof(T), TPV = V / 4, PARTS = (DUAL ? NT / 2 : NT) / TPV;
  const int l = threadIdx.x & 63, i = l & 15, kg = l >> 4;
  const int n1 = n0 + pw0 + V * kg;                        // part p: columns n1 + 4 V p ..
  const bool aligned = n0 % V == 0;
  float b0[PARTS][V], b1[PARTS][V];
  if (!PLAIN && a.partial == nullptr) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      load_bias<T, V>(a.ep, 0, n1 + 4 * V * p, a.N, aligned, b0[p]);
      if (DUAL) load_bias<T, V>(a.ep, 1, n1 + 4 * V * p, a.N, aligned, b1[p]);
    }
  }
  constexpr bool Z_ROWS = DUAL && CHUNK > 0;               // z is written by itself below
  constexpr bool SCALED = PLAIN && std::is_same<T, _Float16>::value;
  float scale = 1.f;
  if (SCALED && a.partial == nullptr && a.ep.scale != nullptr) scale = *a.ep.scale;
  // the sums of row m
  auto row = [&](int m, const f32x4 (&sums)[NT]) {
    if (m >= a.M) return;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int n = n1 + 4 * V * p;
      float v[V], w[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = sums[p * TPV + e / 4][e % 4];
        if (SCALED) v[e] *= scale;
        w[e] = DUAL ? sums[(DUAL ? NT / 2 : 0) + p * TPV + e / 4][e % 4] : 0.f;
      }
      if (a.partial != nullptr) {                          // rows of whole vectors: ldw is N rounded up to 16
        float* d = a.partial + (((long)split * (a.nout * (DUAL ? 2 : 1)) + which) * a.M + m) * a.ldw + n;
        store_some<float, V>(d, v, a.N - n, aligned && n < a.N);
        if (DUAL) store_some<float, V>(d + a.M * a.ldw, w, a.N - n, aligned && n < a.N);
      } else {
        if constexpr (Z_ROWS) {
          Epilogue ep = a.ep;
          ep.z[0] = nullptr;
          epilogue_store<T, DUAL, PLAIN, V>(ep, which, m, n, a.N, aligned, v, w, b0[p], b1[p]);
        } else {
          epilogue_store<T, DUAL, PLAIN, V>(a.ep, which, m, n, a.N, aligned, v, w, b0[p], b1[p]);
        }
      }
    }
  };
  f32x4 sums[NT];
  if constexpr (CHUNK == 0) {
#pragma unroll
    for (int u = 0; u < MT; ++u) {
#pragma unroll
      for (int t = 0; t < NT; ++t) sums[t] = acc[t][u];
      row(m0 + Q::row_of(qw0, u, i), sums);
    }
  } else {
    // z of dual products: 16 lanes take the 2 x 32 sums of a row, four each (16 bits: tile t holds columns 32 (t / 2) + 8 kg + 4 (t % 2);
    // fp32: 16 t + 4 kg), so that a store covers whole lines; as the lanes hold them, 16 of every 32 bytes.  Keeping the sums
    // adds 30 us to 2011 x 2708 x 1000 bf16 the latter way, 16 by rows.  Single products keep the lanes' way: a training step over
    // 8192 x 4096 x 4096 took 754 us with it, 806 by rows.
    const int zq = l & 15, zt = V == 8 ? 2 * (zq >> 3) + (zq & 1) : zq >> 2, zkg = V == 8 ? (zq & 7) >> 1 : zq & 3;
    const bool up = zt >= NT / 2, keep = Z_ROWS && a.ep.z[0] != nullptr && a.partial == nullptr;
    const int zn = n0 + pw0 + 4 * (zq & 7);
    float zb[4] = {0.f, 0.f, 0.f, 0.f};
    if (keep) load_bias<T, 4>(a.ep, up, zn, a.N, aligned, zb);
    f32x4* mine = reinterpret_cast<f32x4*>(lds) + l;
#pragma unroll
    for (int u0 = 0; u0 < MT; u0 += CHUNK) {
#pragma unroll
      for (int u = 0; u < CHUNK; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) mine[(u * NT + t) * 64] = acc[t][u0 + u];
      wave_meet();
#pragma unroll 1
      for (int u = 0; u < CHUNK; ++u) {
        if (keep) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int zi = 4 * j + (l >> 4), m = m0 + Q::row_of(qw0, u0 + u, zi);
            const f32x4 q = reinterpret_cast<f32x4*>(lds)[(u * NT + zt) * 64 + zkg * 16 + zi];
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q[e] + zb[e];
            if (m < a.M && zn < a.N) store_some<float, 4>(a.ep.z[up] + m * a.ep.ldz + zn, v, a.N - zn, aligned);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) sums[t] = mine[(u * NT + t) * 64];
        row(m0 + Q::row_of(qw0, u0 + u, i), sums);
      }
      wave_meet();                                         // the next chunk is written where this one was read
    }
  }
}

// this wave's LDS reads are done, and all but its last N loads; behind the barrier so are the others'
template <int N> __device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- tiles of any size, with their edges: small and fp32 products -----------------------------------------------------------
// A ring of slabs of 128 bytes of k; while some are multiplied, the next ones are in flight.  One barrier a turn: behind it the
// turn's slabs have landed for everyone, and everyone is done with the previous turn's, whose buffers are filled anew.
// Small tiles give a CU too little to do: a wave alone on its SIMD stands still in front of every barrier, LDS read and load.  So more
// waves share a tile along k: WK = 2 groups take one k half of a slab each, and with GROUPS = 2 a turn has two slabs, each staged
// and multiplied by a group of its own.  Their sums meet in LDS at the end, in a fixed order.  One slab a turn and one group, bf16:
// 256 x 4096 x 1024 10.0 us, gated 512 x 1024 x 1024 10.9; two groups 8.3 and 8.6.  A ring of three turns for 64 x 64 leaves a CU one
// workgroup instead of two: 512 x 4096 x 1024 bf16 13.6 us with two, 20.8 with three.
// fp32 is bound by its matrix rate (4096 x 4096 x 4096: 1.06 to 1.12 ms, 123 to 130 TFLOP/s; the library 137), small products by the
// latency of a load, a barrier and a launch (512 x 1024 x 1024 bf16 7.5 us, fp32 18).
template <typename T, int BN, int BM, int WN, int WM, int WK, int GROUPS, int RING, bool PKC, bool QKC, bool DUAL>
__global__ void __launch_bounds__(WN * WM * WK * GROUPS * 64) gemm_kernel(GemmArgs a) {
  constexpr int WAVES = WN * WM, THREADS = WAVES * WK * 64, SETS = WK * GROUPS;
  constexpr int NT = BN / WN / 16, MT = BM / WM / 16;
  static_assert(NT == 4, "a wave covers 64 rows of P");
  static_assert(!DUAL || PKC, "dual products: k-contiguous weights");
  constexpr int TN = DUAL ? BN / 2 : BN;                   // output columns of a tile
  using P = Operand<T, BN, THREADS, PKC, true, DUAL>;
  using Q = Operand<T, BM, THREADS, QKC, false, false>;
  constexpr int TK = P::TK, SLAB = P::BYTES + Q::BYTES, LOADS = P::ROUNDS + Q::ROUNDS;
  constexpr int AHEAD = (RING - 2) * LOADS;                // a wave's loads behind the turn's own
  static_assert(RING >= 2 && AHEAD <= 63, "loads in flight beyond the counter");
  __shared__ __attribute__((aligned(1024))) char lds[RING * GROUPS * SLAB];

  const int tm1 = (a.M + BM - 1) / BM;
  int nt, mt;
  tile_of(blockIdx.x, (a.N + TN - 1) / TN, tm1 * a.nout, nt, mt);
  const int which = mt / tm1, m0 = (mt - which * tm1) * BM, n0 = nt * TN, split = blockIdx.y;

  // contraction: a.nseg segments of `slabs` slabs each; this split takes [s_begin, s_end) of all of them, GROUPS a turn
  const int slabs = (a.K + TK - 1) / TK, all = slabs * a.nseg;
  const int per = (all + a.splits - 1) / a.splits, s_begin = split * per, s_end = min(all, s_begin + per);
  const int turns = (s_end - s_begin + GROUPS - 1) / GROUPS;         // no work: 0 or less
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wm = wave / WN % WM;
  const int set = wave / WAVES, wk = set % WK, group = set / WK;
  const int pw0 = DUAL ? wn * 32 : wn * 64, qw0 = wm * (BM / WM);

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  P pop;
  Q qop;
  const bool inside = n0 + TN <= a.N && m0 + BM <= a.M;
  int next = s_begin + group, seg = -1, fill = 0;          // this group's slab issued next, the segment its pointers are in
  auto issue = [&]() {
    char* at = lds + (fill * GROUPS + group) * SLAB;
    if (next < s_end) {
      const int sg = next / slabs, left = a.K - (next - sg * slabs) * TK;
      if (sg != seg) {
        seg = sg;
        pop.init((const T*)a.p[seg], a.ldp[seg], (const T*)a.p[1], a.ldp[1], n0, a.N, a.K - left);
        qop.init((const T*)a.q[seg + which], a.ldq[seg + which], nullptr, 0, m0, a.M, a.K - left);
      }
      if (inside && left >= TK) {
        pop.stage_inside(at);
        qop.stage_inside(at + P::BYTES);
      } else {
        pop.stage(at, left);
        qop.stage(at + P::BYTES, left);
      }
      if (GROUPS > 1) {                                    // the other groups' slabs
        pop.advance((GROUPS - 1) * pop.step);
        qop.advance((GROUPS - 1) * qop.step);
      }
    } else {                                               // a turn that is not full: zeros
      P::stage_zeros(at);
      Q::stage_zeros(at + P::BYTES);
    }
    next += GROUPS;
    fill = fill + 1 == RING ? 0 : fill + 1;
  };
  for (int i = 0; i < RING - 1 && i < turns; ++i) issue();
  int at = 0;
  for (int turn = 0; turn < turns; ++turn) {
    asm volatile("" ::: "memory");
    if (turn + RING - 2 < turns) __builtin_amdgcn_s_waitcnt(0x0F70 | (AHEAD & 15) | (AHEAD >> 4) << 14);
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (turn + RING - 1 < turns) issue();
    const char* ps = lds + (at * GROUPS + group) * SLAB;
    constexpr int HALVES = 2 / WK;
    typename P::Frag pf[HALVES][NT];                       // all reads first: the second half's run beside the first's products
    typename Q::Frag qf[HALVES][MT];
#pragma unroll
    for (int s = 0; s < HALVES; ++s) {
      P::template read<NT>(ps, pw0, WK == 2 ? wk : s, pf[s]);
      Q::template read<MT>(ps + P::BYTES, qw0, WK == 2 ? wk : s, qf[s]);
    }
#pragma unroll
    for (int s = 0; s < HALVES; ++s) mma_tiles<T, NT, MT>(pf[s], qf[s], acc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // this wave has read its slab before it meets the others
    at = at + 1 == RING ? 0 : at + 1;
  }
  if constexpr (SETS > 1) {
    static_assert((SETS - 1) * WAVES * 64 * NT * MT * 16 <= RING * GROUPS * SLAB, "sums of the other waves");
    f32x4* join = reinterpret_cast<f32x4*>(lds) + (wave % WAVES) * 64 * NT * MT + (threadIdx.x & 63);
    __syncthreads();                                       // the ring has been read
    if (set > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) join[(set - 1) * WAVES * 64 * NT * MT + (t * MT + u) * 64] = acc[t][u];
    }
    __syncthreads();
    if (set > 0) return;
#pragma unroll
    for (int i = 0; i < SETS - 1; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] += join[i * WAVES * 64 * NT * MT + (t * MT + u) * 64];
  }
  constexpr int CHUNK = MT > 1 ? MT : 0;
  static_assert(CHUNK == 0 || (SETS == 1 && WAVES * NT * CHUNK * 1024 <= RING * GROUPS * SLAB), "sums in LDS");
  if (CHUNK > 0) __syncthreads();                          // the ring has been read
  finish<T, P, Q, PKC, QKC, DUAL, NT, MT, CHUNK>(a, acc, n0, pw0, m0, qw0, which, split, lds + wave * NT * CHUNK * 1024);
}

// ---- large products of 16-bit operands ----------------------------------------------------------------------------------------
// Bound by the matrix cores; what keeps them from their rate is everything that is not a product between two barriers.  So the
// loop over slabs is one block of straight-line code with ONE barrier, in which the LDS reads and the loads are dealt out between
// the products:
//   half 0's products   beside   the LDS reads of half 1
//   -- all waves have read this slab, and the next one has landed --
//   half 1's products   beside   the LDS reads of the next slab's half 0 and the loads of the slab RING later
// P's registers are double, Q's mostly single: a Q tile is replaced right behind its last product.  The last two tiles are double
// too, so that the reads end before the products do and the wait in front of the barrier finds them done.
// No edges in the loop: the slab with the end of k comes first (the order of a sum is free), and a tile that would reach beyond the
// output is moved back inside (it computes some results a second time; both writers hold the same bits).  So N and M are at
// least a tile.  The second contraction segment has the first one's strides and is reached by a jump.
// bf16: 8192 x 8192 x 8192 forward 850 us, d_x 795, d_w 825 (1290 to 1380 TFLOP/s; the library 840, 965, 1080); 8192 x 4096 x 4096 205
// to 215 us in all three directions once the clocks are up (1300; the library 175 to 245).  A CU's fill of LDS, 40 to 47 GB/s, bounds
// what is left; a ring of 32-value slabs (two barriers for 64 k) reached 783 TFLOP/s where this did 1008.
template <typename T, int BN, int BM, int WN, int WM, int RING, bool PKC, bool QKC, bool DUAL>
__global__ void __launch_bounds__(WN * WM * 64) gemm_big_kernel(GemmArgs a) {
  constexpr int THREADS = WN * WM * 64, NT = 4, MT = BM / WM / 16, DBL = 2, SNG = MT - DBL;
  static_assert(BN / WN == 64, "a wave covers 64 rows of P");
  constexpr int TN = DUAL ? BN / 2 : BN, EPC = 16 / sizeof(T);
  using P = Operand<T, BN, THREADS, PKC, true, DUAL>;
  using Q = Operand<T, BM, THREADS, QKC, false, false>;
  constexpr int TK = P::TK, SLAB = P::BYTES + Q::BYTES;
  constexpr int LOADS = P::ROUNDS + Q::ROUNDS;             // loads of a slab, dealt out over the rows of products
  static_assert(NT <= MT && P::CLS == 1 && Q::CLS == 1, "dealing of reads and loads");
  __shared__ __attribute__((aligned(1024))) char lds[RING * SLAB];
  static_assert(RING >= 2 && (RING - 2) * LOADS <= 63, "loads in flight beyond the counter");

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
  const int pw0 = DUAL ? wn * 32 : wn * 64, qw0 = wm * (BM / WM);

  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  P pop;
  Q qop;
  // Each XCD starts at another eighth of k: tiles in step, with rows a power of two apart, ask the same memory channels at the same
  // time (8192 x 8192 x 8192 forward 872 -> 853 us, 8192 x 4096 x 16384 878 -> 842, bf16; 4096 x 4096 unchanged).
  // Only where no tile was moved: both writers of an output have to sum in the same order.
  const bool whole = a.N % TN == 0 && a.M % BM == 0 && tails == 0;
  const int skew = whole && a.nseg == 1 && a.splits == 1 ? full * (int)(blockIdx.x % 8) / 8 : 0;
  auto seek = [&](int slab) {
    slab += skew;
    if (slab >= all) slab -= all;
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
  // half s's products of the slab in buffer `buf`; NEXT: read the following half (of this slab, or of the next buffer's);
  // LOAD: fill this buffer anew
  auto phase = [&](auto half, auto with_next, auto with_load, int buf) {
    constexpr int s = decltype(half)::value;
    constexpr bool NEXT = decltype(with_next)::value, LOAD = decltype(with_load)::value;
    const char* next = lds + (s == 0 ? buf : buf + 1 == RING ? 0 : buf + 1) * SLAB;
    char* load = lds + buf * SLAB;
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      if constexpr (NEXT) {
        if (u < NT) pf[s ^ 1][u] = P::read_one(next, pw0, s ^ 1, u);
        if (u < DBL) q2[s ^ 1][u] = Q::read_one(next + P::BYTES, qw0, s ^ 1, SNG + u);
      }
      if constexpr (LOAD) {
#pragma unroll
        for (int r = u * LOADS / MT; r < (u + 1) * LOADS / MT; ++r) {
          if (r < P::ROUNDS) pop.stage_round(load, r);
          else qop.stage_round(load + P::BYTES, r - P::ROUNDS);
        }
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
    for (int i = 0; i < RING && i < count; ++i) {
      const int left = seek(s_begin + i);
      pop.stage(lds + i * SLAB, left);
      qop.stage(lds + i * SLAB + P::BYTES, left);
    }
    meet<0>();
    P::template read<NT>(lds, pw0, 0, pf[0]);
#pragma unroll
    for (int u = 0; u < SNG; ++u) q1[u] = Q::read_one(lds + P::BYTES, qw0, 0, u);
#pragma unroll
    for (int u = 0; u < DBL; ++u) q2[0][u] = Q::read_one(lds + P::BYTES, qw0, 0, SNG + u);
    int buf = 0;
    if (count > RING) {
      seek(s_begin + RING);
      // slabs until the jump to the second segment (0: none), and its distance from where the first one ends
      int to_jump = a.nseg == 2 ? tails + full - (s_begin + RING) : 0;
      long p_jump = a.nseg == 2 ? (const char*)a.p[1] - (const char*)a.p[0] - full * pop.step : 0;
      long q_jump = a.nseg == 2 ? (const char*)a.q[1] - (const char*)a.q[0] - full * qop.step : 0;
      if (skew > 0) {
        to_jump = full - (s_begin + RING + skew);
        p_jump = -full * pop.step;
        q_jump = -full * qop.step;
      }
      for (int i = 0; i < count - RING; ++i) {
        phase(H0, YES, NO, buf);
        meet<(RING - 2) * LOADS>();                        // the next slab has landed; later ones stay in flight
        phase(H1, YES, YES, buf);
        const bool jump = --to_jump == 0;
        pop.advance(pop.step + (jump ? p_jump : 0));
        qop.advance(qop.step + (jump ? q_jump : 0));
        buf = buf + 1 == RING ? 0 : buf + 1;
      }
    }
    for (int i = min(count, RING) - 1; i > 0; --i) {
      phase(H0, YES, NO, buf);
      meet<0>();
      phase(H1, YES, NO, buf);
      buf = buf + 1 == RING ? 0 : buf + 1;
    }
    phase(H0, YES, NO, buf);
    phase(H1, NO, NO, buf);
  }
  constexpr int CHUNK = 4;
  static_assert(MT % CHUNK == 0 && WN * WM * NT * CHUNK * 1024 <= RING * SLAB, "sums in LDS");
  __syncthreads();                                         // the ring has been read
  finish<T, P, Q, PKC, QKC, DUAL, NT, MT, CHUNK>(a, acc, n0, pw0, m0, qw0, which, split, lds + wave * NT * CHUNK * 1024);
}

template <typename T, int BN, int BM, int WN, int WM, int WK, int GROUPS, int RING> void run_cfg(const GemmArgs& a, hipStream_t s) {
  const long tn = (a.N + (a.dual ? BN / 2 : BN) - 1) / (a.dual ? BN / 2 : BN), tm = (long)((a.M + BM - 1) / BM) * a.nout;
  const dim3 grid((unsigned)(tn * tm), (unsigned)a.splits), block(WN * WM * WK * GROUPS * 64);
  if (a.dual) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, WK, GROUPS, RING, true, true, true>), grid, block, 0, s, a);
  else if (a.p_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, WK, GROUPS, RING, true, true, false>), grid, block, 0, s, a);
  else if (a.q_kc) hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, WK, GROUPS, RING, false, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_kernel<T, BN, BM, WN, WM, WK, GROUPS, RING, false, false, false>), grid, block, 0, s, a);
}
template <typename T, int BN, int BM, int WN, int WM, int RING> void run_big(const GemmArgs& a, hipStream_t s) {
  const int tn = a.dual ? BN / 2 : BN;
  const dim3 grid((unsigned)((long)((a.N + tn - 1) / tn) * ((a.M + BM - 1) / BM) * a.nout), (unsigned)a.splits), block(WN * WM * 64);
  if (a.dual) hipLaunchKernelGGL((gemm_big_kernel<T, BN, BM, WN, WM, RING, true, true, true>), grid, block, 0, s, a);
  else if (a.p_kc) hipLaunchKernelGGL((gemm_big_kernel<T, BN, BM, WN, WM, RING, true, true, false>), grid, block, 0, s, a);
  else if (a.q_kc) hipLaunchKernelGGL((gemm_big_kernel<T, BN, BM, WN, WM, RING, false, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_big_kernel<T, BN, BM, WN, WM, RING, false, false, false>), grid, block, 0, s, a);
}
template <typename T> void run_small(const GemmArgs& a, int cfg, hipStream_t s) {
  if (cfg == TILE_128x32) run_cfg<T, 128, 32, 2, 2, 1, 2, 2>(a, s);
  else if (cfg == TILE_64x32) run_cfg<T, 64, 32, 1, 2, 2, 2, 3>(a, s);
  else if (cfg == TILE_64x64) run_cfg<T, 64, 64, 1, 4, 1, 2, 2>(a, s);
  else run_cfg<T, 128, 128, 2, 2, 1, 1, 2>(a, s);
}
}  // namespace
}  // namespace ffn
}  // namespace ddl
