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
__device__ __forceinline__ float smaller(float a, float b) {
  float m;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// 8 elements of a group whose other elements the lanes beside (of a multiple of four) have.  All lanes of the warp call it.
template <int kBits, typename T>
__device__ __forceinline__ Quantized<kBits> quantize(const uint4 (&words)[sizeof(T) / 2]) {
  constexpr int kHalf = 1 << (kBits - 1);
  const T* e = reinterpret_cast<const T*>(words);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
  float high = x[0], low = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    high = larger(high, x[i]);
    low = smaller(low, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    high = larger(high, __shfl_xor_sync(0xffffffffu, high, o));
    low = smaller(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  const bool finite = high < INFINITY && low > -INFINITY;      // (false for a NaN)
  const float a = high >= -low ? high : low;
  const __half step = __float2half_rn(fminf(fmaxf(a * (-1.f / kHalf), -65504.f), 65504.f));
  const float s = __half2float(step);
  // (1 / s rounded to nearest: an approximation good to one unit and one step of Newton's method give that for every fp16 number)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  const float inverse = s != 0.f ? __fmaf_rn(r, __fmaf_rn(-s, r, 1.f), r) : 0.f;
  Quantized<kBits> q;
  q.step = finite ? __half_as_ushort(step) : uint16_t(0x7fff);
  // Adding M = 1.5 2^23 + half rounds to whole numbers, halves to even, and leaves the code in the lowest bits of a number whose
  // others are known: codes are put side by side by adding these numbers up, shifted, and taking the known bits off at the end.
  constexpr float kM = 12582912.f + kHalf;
  constexpr uint32_t kBase = 0x4b400000u, kKnown = kBits == 4 ? kBase * 0x11111111u : kBase * 0x01010101u;
  // A quotient is at most half (1 + 2^-11) in size, so that only the far end has to be cut, unless the step has been cut itself or has
  // lost bits as one of fp16's smallest numbers.
  float2 z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    z[i] = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(inverse, inverse));
    z[i] = make_float2(fminf(z[i].x, kHalf - 1.f), fminf(z[i].y, kHalf - 1.f));
  }
  const float size = fabsf(s);
  if (__any_sync(0xffffffffu, size < 6.103515625e-05f || size >= 65504.f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = make_float2(fmaxf(z[i].x, float(-kHalf)), fmaxf(z[i].y, float(-kHalf)));
  }
  uint32_t w[8 * kBits / 32] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 c = __fadd2_rn(z[i], make_float2(kM, kM));
    w[2 * i * kBits / 32] += (__float_as_uint(c.x) << (2 * i * kBits % 32)) + (__float_as_uint(c.y) << ((2 * i + 1) * kBits % 32));
  }
  // (what is not finite, and a step of zero, has the codes of zero: z is zero in the second case)
  constexpr uint32_t kZero = kBits == 4 ? 0x88888888u : 0x80808080u;
  q.lo = finite ? w[0] - kKnown : kZero;
  q.hi = kBits == 4 ? 0u : finite ? w[8 * kBits / 32 - 1] - kKnown : kZero;
  return q;
}

// The codes of elements 8 u .. 8 u + 7 of a group are in parts 2 u and 2 u + 1 of the row.
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
// Those of all groups at once lie side by side, kGroups kBits / 4 words.
template <int n, typename P>
__device__ __forceinline__ void store_words(P* to, const uint32_t (&w)[n]) {
  if constexpr (n == 1) *reinterpret_cast<uint32_t*>(to) = w[0];
  else if constexpr (n == 2) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  else
#pragma unroll
    for (int i = 0; i < n / 4; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}
template <int n, typename P>
__device__ __forceinline__ void load_words(uint32_t (&w)[n], const P* from) {
  if constexpr (n == 1) {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(from));
  } else if constexpr (n == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(from));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < n / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(from) + i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}
template <int kBits, int kGroups>
__device__ __forceinline__ void store_quarter(uint8_t* row, int u, const Quantized<kBits> (&q)[kGroups]) {
  constexpr int n = kGroups * kBits / 4;
  uint32_t w[n];
#pragma unroll
  for (int i = 0; i < n / 2; ++i) {
    w[i] = kBits == 4 ? __byte_perm(q[(2 * i) % kGroups].lo, q[(2 * i + 1) % kGroups].lo, 0x5410) : q[i % kGroups].lo;
    w[n / 2 + i] = kBits == 4 ? __byte_perm(q[(2 * i) % kGroups].lo, q[(2 * i + 1) % kGroups].lo, 0x7632) : q[i % kGroups].hi;
  }
  store_words(row + u * n * 4, w);
}
// Values of 8 elements, from the words of their codes (one in 4 bits).
template <int kBits>
__device__ __forceinline__ void values_of(uint32_t lo, uint32_t hi, float step, float2 (&x)[4]) {
  // A code in the bits from p on of 2^23 is 2^23 + 2^p code: the half of the range and 2^23 come off exactly, the step takes 2^-p.
  constexpr int kEach = 16 / kBits;      // codes of 16 bits
  constexpr float kHalf = float(1 << (kBits - 1));
#pragma unroll
  for (int h = 0; h < 8 / kEach; ++h) {
    const uint32_t word = kBits == 8 && h >= 2 ? hi : lo, part = h & 1 ? word >> 16 : word;
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
      const float p0 = float(1u << (i * kBits)), p1 = float(1u << ((i + 1) * kBits));
      const uint32_t mask = (1u << kBits) - 1u;
      const float2 c = make_float2(__uint_as_float(0x4b000000u | (part & mask << (i * kBits))), __uint_as_float(0x4b000000u | (part & mask << ((i + 1) * kBits))));
      x[(h * kEach + i) / 2] = __fmul2_rn(__fadd2_rn(c, make_float2(-8388608.f - kHalf * p0, -8388608.f - kHalf * p1)), make_float2(step * (1.f / p0), step * (1.f / p1)));
    }
  }
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
