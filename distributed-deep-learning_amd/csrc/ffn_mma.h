// Matrix-core operand types and products of the feed-forward operators, by element type.
// A: lane holds row (lane & 15), 16 bytes of k at chunk (lane >> 4); B likewise; D: lane holds column (lane & 15) and the rows
// 4 (lane >> 4) + 0..3.
#pragma once
#include <hip/hip_runtime.h>

namespace ddl {
namespace ffn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mma;
template <> struct Mma<__bf16> {
  using Frag = bf16x8;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<_Float16> {
  using Frag = f16x8;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<float> {          // four 16x16x4 products over the four k of a 16-byte chunk
  using Frag = f32x4;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// acc += P Q for NT x MT tiles.  fp32: all tiles of one k before the next k, since a product that waits for the one before it on the
// same accumulator leaves the matrix core idle.
template <typename T, int NT, int MT>
__device__ __forceinline__ void mma_tiles(const typename Mma<T>::Frag (&p)[NT], const typename Mma<T>::Frag (&q)[MT],
                                          f32x4 (&acc)[NT][MT]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[t][e], q[u][e], acc[t][u], 0, 0, 0);
  } else {
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][u] = Mma<T>::mma(p[t], q[u], acc[t][u]);
  }
}

}  // namespace ffn
}  // namespace ddl
