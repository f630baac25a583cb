// fp32 numbers as three bf16 numbers, and products of them as six bf16 products (sdpa_fp32_tc.cu has the reasons).
#pragma once

#include <stdint.h>

#include "sm100_primitives.cuh"

namespace nb200 {

#ifdef __CUDACC__
// eight fp32 as three words of eight bf16 each, by truncation
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&w)[3]) {
  uint32_t r[8], o[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(x[i]);
#pragma unroll
  for (int p = 0; p < 3; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __byte_perm(r[2 * i], r[2 * i + 1], 0x7632);
    w[p] = make_uint4(o[0], o[1], o[2], o[3]);
    if (p < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) - __uint_as_float(r[i] & 0xffff0000u));
    }
  }
}

// the six products, small ones first: (plane of the left operand, plane of the right one)
inline constexpr int kProducts = 6;
__device__ __forceinline__ constexpr int left_plane(int i) { return i == 0 ? 2 : (i == 1 ? 0 : (i == 2 ? 1 : (i == 3 ? 1 : 0))); }
__device__ __forceinline__ constexpr int right_plane(int i) { return i == 0 ? 0 : (i == 1 ? 2 : (i == 2 ? 1 : (i == 3 ? 0 : (i == 4 ? 1 : 0)))); }
#endif

}  // namespace nb200
