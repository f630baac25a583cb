// The codes of a cache in few bits: how values become codes and back, and the checks of its pages.
//
//   a = max x if max x >= -min x else min x,  step = fp16(-a / 2^(b-1)),  code = rint(x / step) + 2^(b-1),
//   value = step (code - 2^(b-1))                                          per group of 32 elements of a head's row
//
// The element of largest size has the code 0, so that all 2^b codes are in use and the step is as small as they allow; of the
// other sign's side, values beyond the last code are cut to it (by half a step and more of rounding at most one).
//
// A row of codes is (8, groups, b / 2) bytes: the elements 4 j .. 4 j + 3 of every group lie together, the first in the lowest bits.
// A part j of the row then holds as much of every group, which is what the lanes of a warp-level MMA need (decode_quantized.cu).
#pragma once

#include "nitrix_b200_cache.h"
#include "sdpa_common.cuh"

namespace nb200 {
namespace {

constexpr int kGroup = 32;      // elements with one step

#ifdef __CUDACC__
// Codes of a lane's 8 elements: with 4 bits in `lo` alone, with 8 the first four in `lo`.
template <int kBits>
struct Quantized {
  uint32_t lo, hi;
  uint16_t step;
};

__device__ __forceinline__ float larger(float a, float b) {      // a NaN on either side comes out
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// 8 elements of a group whose other elements the lanes beside (of a multiple of four) have.  All lanes of the warp call it.
template <int kBits, typename T>
__device__ __forceinline__ Quantized<kBits> quantize(const uint4 (&words)[sizeof(T) / 2]) {
  constexpr float kHalf = float(1 << (kBits - 1));
  const T* e = reinterpret_cast<const T*>(words);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
  float high = x[0], low = -x[0];      // the largest value, and the smallest one's opposite
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    high = larger(high, x[i]);
    low = larger(low, -x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    high = larger(high, __shfl_xor_sync(0xffffffffu, high, o));
    low = larger(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  const bool finite = high < INFINITY && low < INFINITY;      // (false for a NaN)
  const float a = high >= low ? high : -low;
  const __half step = __float2half_rn(fminf(fmaxf(a * (-1.f / kHalf), -65504.f), 65504.f));
  const float s = __half2float(step);
  const float inverse = finite && s != 0.f ? __frcp_rn(s) : 0.f;
  Quantized<kBits> q;
  q.step = finite ? __half_as_ushort(step) : uint16_t(0x7fff);
  uint32_t c[8];
  // (adding 1.5 2^23 + half rounds to whole numbers, halves to even, and leaves the code in the lowest bits)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = finite ? fminf(fmaxf(__fmul_rn(x[i], inverse), -kHalf), kHalf - 1.f) : 0.f;
    c[i] = __float_as_uint(__fadd_rn(z, 12582912.f + kHalf)) & ((1u << kBits) - 1u);
  }
  if constexpr (kBits == 4) {
    q.lo = c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12 | c[4] << 16 | c[5] << 20 | c[6] << 24 | c[7] << 28;
    q.hi = 0;
  } else {
    q.lo = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    q.hi = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
  }
  return q;
}

// The codes of elements 8 u .. 8 u + 7 of a group: parts 2 u and 2 u + 1 of the row.
template <int kBits>
__device__ __forceinline__ void store_codes(uint8_t* row, int groups, int group, int u, const Quantized<kBits>& q) {
  if constexpr (kBits == 4) {
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + 2 * u * groups + group;
    p[0] = uint16_t(q.lo);
    p[groups] = uint16_t(q.lo >> 16);
  } else {
    uint32_t* p = reinterpret_cast<uint32_t*>(row) + 2 * u * groups + group;
    p[0] = q.lo;
    p[groups] = q.hi;
  }
}
// A part's four codes of a group, less the half of their range.
template <int kBits>
__device__ __forceinline__ void load_codes(const uint8_t* row, int groups, int group, int part, float (&c)[4]) {
  constexpr float kHalf = float(1 << (kBits - 1));
  const uint32_t w = kBits == 4 ? uint32_t(__ldg(reinterpret_cast<const uint16_t*>(row) + part * groups + group))
                                : __ldg(reinterpret_cast<const uint32_t*>(row) + part * groups + group);
  // (a code in the lowest bits of 2^23 is 2^23 + code)
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __uint_as_float(0x4b000000u | (w >> (kBits * i) & ((1u << kBits) - 1u))) - (8388608.f + kHalf);
}
#endif

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_steps(const nb200_cache_pages& c, const nb200_cache_steps& s, const char* what) {
  if (s.bits != 4 && s.bits != 8) { set_error("%s: codes of %d bits, 4 or 8 are possible", what, s.bits); return NB200_ERR_INVALID; }
  if (c.pages && (!s.k || !s.v)) { set_error("%s: NULL steps", what); return NB200_ERR_INVALID; }
  if (c.head_dim % kGroup) { set_error("%s: head dim %d must be a multiple of %d", what, c.head_dim, kGroup); return NB200_ERR_UNSUPPORTED; }
  const int groups = c.head_dim / kGroup;
  bool ok = aligned16(s.k) && aligned16(s.v);
  for (int i = 0; i < 3; ++i) ok = ok && s.k_stride[i] % groups == 0 && s.v_stride[i] % groups == 0;
  if (!ok) { set_error("%s: the rows of the steps must begin at multiples of their size from a 16-byte boundary", what); return NB200_ERR_ALIGNMENT; }
  return NB200_OK;
}

}  // namespace
}  // namespace nb200
