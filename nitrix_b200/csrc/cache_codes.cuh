// The codes of a cache in few bits: how values become codes and back, and the checks of its pages.
//
//   a = max x if max x >= -min x else min x,  step = fp16(-a / 2^(b-1)),  code = rint(x (1 / step)) + 2^(b-1),
//   value = step (code - 2^(b-1))                                          per group of 32 elements of a head's row
//
// with 1 / step and the product rounded to fp32.  The element of largest size has the code 0, so that all 2^b codes are in use and the
// step is as small as they allow.  The other sign has one code less: values beyond its last one are cut to it, by a step at most.
//
// A row of codes is (8, groups, b / 2) bytes: the elements 4 j .. 4 j + 3 of every group lie together, the first in the lowest bits.
// A part j of the row then holds as much of every group, which is what the lanes of a warp-level MMA need (decode_quantized.cu).
#pragma once

#include <type_traits>

#include "nitrix_b200_cache.h"
#include "sdpa_common.cuh"

namespace nb200 {
namespace {

constexpr int kGroup = 32;      // elements with one step

#ifdef __CUDACC__
// Codes of a lane's 8 elements of n groups: with 4 bits in `lo` alone, with 8 the first four in `lo`.  The four lanes of a group share
// out the steps: this lane has that of group `step_of(lane)`.
template <int kBits, int n>
struct Quantized {
  uint32_t lo[n], hi[n];
  uint16_t step;
  static __device__ __forceinline__ int step_of(int lane) { return (lane & 3) * n / 4; }
  static __device__ __forceinline__ int first_lane(int group) { return group * (4 / n); }      // of those that have a group's
};

// The largest of two or three; a NaN anywhere comes out.
__device__ __forceinline__ float larger(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float larger(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {      // of the two halves of a word
  uint32_t m;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t smaller2(uint32_t a, uint32_t b) {
  uint32_t m;
  if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
// max x and -min x of elements
template <typename T>
struct Extremes {      // (a word: the two as halves)
  uint32_t m;
  __device__ __forceinline__ explicit Extremes(const uint4 (&words)[1]) {
    const uint4 w = words[0];
    const uint32_t high = larger2<T>(larger2<T>(w.x, w.y), larger2<T>(w.z, w.w)), low = smaller2<T>(smaller2<T>(w.x, w.y), smaller2<T>(w.z, w.w)) ^ 0x80008000u;
    m = larger2<T>(__byte_perm(high, low, 0x5410), __byte_perm(high, low, 0x7632));
  }
  __device__ __forceinline__ void join(uint32_t from, int lanes) { m = larger2<T>(m, __shfl_xor_sync(0xffffffffu, from, lanes)); }
  __device__ __forceinline__ float high() const { return to_f32<T>(reinterpret_cast<const T*>(&m)[0]); }
  __device__ __forceinline__ float minus_low() const { return to_f32<T>(reinterpret_cast<const T*>(&m)[1]); }
};
template <>
struct Extremes<float> {
  float2 m;
  __device__ __forceinline__ explicit Extremes(const uint4 (&words)[2]) {
    const float* x = reinterpret_cast<const float*>(words);
    m = make_float2(larger(larger(x[0], x[1], x[2]), larger(x[3], x[4], x[5]), larger(x[6], x[7])),
                    larger(larger(-x[0], -x[1], -x[2]), larger(-x[3], -x[4], -x[5]), larger(-x[6], -x[7])));
  }
  __device__ __forceinline__ void join(float2 from, int lanes) {
    m = make_float2(larger(m.x, __shfl_xor_sync(0xffffffffu, from.x, lanes)), larger(m.y, __shfl_xor_sync(0xffffffffu, from.y, lanes)));
  }
  __device__ __forceinline__ float high() const { return m.x; }
  __device__ __forceinline__ float minus_low() const { return m.y; }
};

// 8 elements each of n groups (1, 2 or 4) whose other elements the lanes beside (of a multiple of four) have.  All lanes of the warp
// call it.
template <int kBits, typename T, int n>
__device__ __forceinline__ Quantized<kBits, n> quantize(const uint4 (&words)[n][sizeof(T) / 2]) {
  constexpr int kHalf = 1 << (kBits - 1);
  const int lane = threadIdx.x & 31;
  Quantized<kBits, n> q;
  // extremes of the lane's own group of the n, from the other lanes, as they get those of theirs
  Extremes<T> m(words[0]);
  if constexpr (n == 4) {
    const Extremes<T> m1(words[1]), m2(words[2]), m3(words[3]);
    const bool upper = lane & 2, odd = lane & 1;
    Extremes<T> k0 = upper ? m2 : m, k1 = upper ? m3 : m1;
    k0.join(upper ? m.m : m2.m, 2);
    k1.join(upper ? m1.m : m3.m, 2);
    m = odd ? k1 : k0;
    m.join(odd ? k0.m : k1.m, 1);
  } else {
    if constexpr (n == 2) {
      const Extremes<T> m0 = m, m1(words[1]);
      const bool upper = lane & 2;
      m = upper ? m1 : m0;
      m.join(upper ? m0.m : m1.m, 2);
    } else {
      m.join(m.m, 2);
    }
    m.join(m.m, 1);
  }
  const float high = m.high(), low = -m.minus_low();
  const bool finite = high < INFINITY && low > -INFINITY;      // (false for a NaN)
  const float a = high >= -low ? high : low;
  const __half step = __float2half_rn(fminf(fmaxf(a * (-1.f / kHalf), -65504.f), 65504.f));
  q.step = finite ? __half_as_ushort(step) : uint16_t(0x7fff);
  const float s = __half2float(step), size = fabsf(s);
  // (1 / s rounded to nearest: an approximation good to one unit and one step of Newton's method give that for every fp16 number)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  float inverse = s != 0.f ? __fmaf_rn(r, __fmaf_rn(-s, r, 1.f), r) : 0.f;
  if (!finite) inverse = __uint_as_float(0x7fffffffu);
  // A quotient is at most half (1 + 2^-11) in size, so that only the far end of the codes has to be cut, unless the step has been cut
  // itself or has lost bits as one of fp16's smallest numbers.
  const bool rare = __any_sync(0xffffffffu, !finite || size < 6.103515625e-05f || size >= 65504.f);
#pragma unroll
  for (int g = 0; g < n; ++g) {
    const T* e = reinterpret_cast<const T*>(words[g]);
    const float by = __shfl_sync(0xffffffffu, inverse, (lane & ~3) + Quantized<kBits, n>::first_lane(g));
    float2 z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __fmul2_rn(make_float2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1])), make_float2(by, by));
    if (rare) {
      // (what is not finite, and a step of zero, has the codes of zero)
      const auto cut = [by](float x) { return by == by ? fminf(fmaxf(x, float(-kHalf)), kHalf - 1.f) : 0.f; };
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = make_float2(cut(z[i].x), cut(z[i].y));
    }
    // Adding 1.5 2^23 + half rounds to whole numbers, halves to even, and leaves the code in the lowest 16 bits, of which those of two
    // elements are put side by side.
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr float kM = 12582912.f + kHalf;
      const float2 y = __fadd2_rn(z[i], make_float2(kM, kM));
      c[2 * i] = __float_as_uint(y.x);
      c[2 * i + 1] = __float_as_uint(y.y);
    }
    const auto pair = [&c](int i, int j) {
      constexpr uint32_t kMost = (2 * kHalf - 1) * 0x10001u;
      uint32_t p;
      asm("min.u16x2 %0, %1, %2;" : "=r"(p) : "r"(__byte_perm(c[i], c[j], 0x5410)), "r"(kMost));
      return p;
    };
    if constexpr (kBits == 4) {
      q.lo[g] = pair(0, 4) + pair(1, 5) * 16u + pair(2, 6) * 256u + pair(3, 7) * 4096u;
      q.hi[g] = 0;
    } else {
      q.lo[g] = pair(0, 2) + pair(1, 3) * 256u;
      q.hi[g] = pair(4, 6) + pair(5, 7) * 256u;
    }
  }
  return q;
}

// The codes of elements 8 u .. 8 u + 7 of a group are in parts 2 u and 2 u + 1 of the row.
template <int kBits>
__device__ __forceinline__ void store_codes(uint8_t* row, int groups, int group, int u, const Quantized<kBits, 1>& q) {
  if constexpr (kBits == 4) {
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + 2 * u * groups + group;
    p[0] = uint16_t(q.lo[0]);
    p[groups] = uint16_t(q.lo[0] >> 16);
  } else {
    uint32_t* p = reinterpret_cast<uint32_t*>(row) + 2 * u * groups + group;
    p[0] = q.lo[0];
    p[groups] = q.hi[0];
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
__device__ __forceinline__ void store_quarter(uint8_t* row, int u, const Quantized<kBits, kGroups>& q) {
  constexpr int n = kGroups * kBits / 4;
  uint32_t w[n];
#pragma unroll
  for (int i = 0; i < n / 2; ++i) {
    w[i] = kBits == 4 ? __byte_perm(q.lo[(2 * i) % kGroups], q.lo[(2 * i + 1) % kGroups], 0x5410) : q.lo[i % kGroups];
    w[n / 2 + i] = kBits == 4 ? __byte_perm(q.lo[(2 * i) % kGroups], q.lo[(2 * i + 1) % kGroups], 0x7632) : q.hi[i % kGroups];
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
  if (int64_t(c.heads) * c.head_dim > 0x3fffffff) { set_error("%s: rows too large", what); return NB200_ERR_UNSUPPORTED; }      // (counted in 32 bits)
  const int groups = c.head_dim / kGroup;
  bool ok = aligned16(s.k) && aligned16(s.v);
  for (int i = 0; i < 3; ++i) ok = ok && s.k_stride[i] % groups == 0 && s.v_stride[i] % groups == 0;
  if (!ok) { set_error("%s: the rows of the steps must begin at multiples of their size from a 16-byte boundary", what); return NB200_ERR_ALIGNMENT; }
  return NB200_OK;
}

}  // namespace
}  // namespace nb200
