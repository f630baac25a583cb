// Root-mean-square norm over the trailing axis with the addition of a residual stream, forward and backward, and with an output
// in 8 bits.
//
//   forward   h = x + r (rounded to the storage type),  s = (mean h^2 + eps)^-1/2,  y = h s w
//             8 bits: a = max |y| of a row or group of channels, scale = a / 448, code = e4m3(y 448 / a)
//   backward  n = h s,  g = dy w,  dx = dh + s (g - n mean(g n)),  dw = sum_rows dy n
//
// Bound by HBM: every stream is read once and written once, so a row is held in registers between its sum and its output: by
// tpr threads (whole warps; a power of two where rows share a CTA), kPer chunks of kVec elements each.  kVec is a 16-byte word's elements, or one where rows do not
// begin on 16-byte boundaries.  CTAs walk the rows with a stride and ask for the next row before they work on the present one.
// Elements are taken in pairs, two fp32 operations per instruction: with 16-bit storage the conversions and the arithmetic take as
// many issue slots as the loads leave.  Rows that are too long to be held are read once more (the *_wide kernels).
//
// Launches by themselves with cold caches (ncu).  bf16, 16384 x 4096 with a residual: forward 81 us (6.6 TB/s of what has to be moved, the
// rate of a copy), backward 87 (6.2), and the sums of dw take 6 more; e4m3, 16384 x 8192: with a scale per 128 channels 154 us (149 in a
// captured graph, 6.3 TB/s), with one per row 5 more.  fp32, 4099 rows of 1001 channels, by elements: 17 and 22 us.  Scalar arithmetic and
// conversions, one row at a time: 107, 136 and 279 us.
#include <cuda_fp8.h>
#include <math.h>

#include <type_traits>

#include "dependent_launch.cuh"
#include "nitrix_b200_rms_norm.h"
#include "sdpa_tc_common.cuh"

namespace nb200 {
namespace {

constexpr int kMaxWarps = 16;

// Threads of all CTAs of an SM, by the registers that a thread takes (the kernels' launch bounds), and CTAs of `threads`.
constexpr int fwd_threads(int per, int vec) { return per <= (vec == 1 ? 8 : 2) ? 1024 : 512; }
constexpr int bwd_threads(int elements) { return elements <= 8 ? 1024 : elements <= 16 ? 768 : 512; }
constexpr int ctas_of(int all, int threads) { return all < threads ? 1 : all / threads; }

struct RmsArgs {
  const void* x;
  const void* r;
  const void* w;
  void* y;
  void* sum;
  float* rstd;
  float* scales;
  const void* dy;
  const void* dsum;
  void* dx;
  float* part;      // [CTA][C]: partial sums of dw
  int64_t rows;
  int C;
  int group;        // channels of a scale; its power of two, where rows have several
  int group_shift;
  float eps, inv_c;
  double eps64;     // (not flushed where it is one of fp32's smallest numbers)
};

// kVec consecutive elements as they lie in memory, and as pairs (one element: with a zero behind it).
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (sizeof(T) == 4) return make_float2(0.f, 0.f);
  else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t word_of(float2 v) {
  return tc::pack2<!std::is_same<T, __half>::value>(v.x, v.y);
}
template <typename T, int kVec>
struct Chunk {
  static constexpr int kPairs = kVec / 2, kWords = kVec * int(sizeof(T)) / 16;
  uint4 w[kWords];
  __device__ __forceinline__ static Chunk load(const T* p) {
    Chunk c;
#pragma unroll
    for (int i = 0; i < kWords; ++i) c.w[i] = sm100::ldg_no_allocate(reinterpret_cast<const uint4*>(p) + i);
    return c;
  }
  __device__ __forceinline__ static Chunk load_cached(const T* p) {
    Chunk c;
#pragma unroll
    for (int i = 0; i < kWords; ++i) c.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return c;
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float2 (&f)[kPairs]) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      f[i] = sizeof(T) == 4 ? make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])) : pair_of<T>(u[i]);
  }
  __device__ __forceinline__ static Chunk of(const float2 (&f)[kPairs]) {
    Chunk c;
    uint32_t* u = reinterpret_cast<uint32_t*>(c.w);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      if constexpr (sizeof(T) == 4) {
        u[2 * i] = __float_as_uint(f[i].x);
        u[2 * i + 1] = __float_as_uint(f[i].y);
      } else {
        u[i] = word_of<T>(f[i]);
      }
    }
    return c;
  }
  __device__ __forceinline__ static Chunk zero() {
    Chunk c;
#pragma unroll
    for (int i = 0; i < kWords; ++i) c.w[i] = make_uint4(0, 0, 0, 0);
    return c;
  }
};
template <typename T>
struct Chunk<T, 1> {
  static constexpr int kPairs = 1;
  T v;
  __device__ __forceinline__ static Chunk load(const T* p) { return Chunk{__ldg(p)}; }
  __device__ __forceinline__ static Chunk load_cached(const T* p) { return Chunk{*p}; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float2 (&f)[1]) const { f[0] = make_float2(to_f32<T>(v), 0.f); }
  __device__ __forceinline__ static Chunk of(const float2 (&f)[1]) { return Chunk{from_f32<T>(f[0].x)}; }
  __device__ __forceinline__ static Chunk zero() { return Chunk{from_f32<T>(0.f)}; }
};

// Weights of a chunk, of their own type; ones without a weight.
template <typename W, int kVec>
__device__ __forceinline__ Chunk<W, kVec> weights(const void* w, int c, bool in) {
  using C = Chunk<W, kVec>;
  if (w && in) return C::load_cached(static_cast<const W*>(w) + c);
  float2 ones[C::kPairs];
#pragma unroll
  for (int i = 0; i < C::kPairs; ++i) ones[i] = make_float2(1.f, 1.f);
  return C::of(ones);
}

// Elements times their row's factor, without a flush of small numbers: of rows of the largest numbers the factor is one of fp32's
// smallest.
__device__ __forceinline__ float2 times(float2 a, float factor) {
  float2 c;
  asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %4};\nmul.rn.f32x2 c, a, b;\nmov.b64 {%0, %1}, c;\n}" : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(factor));
  return c;
}

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN on either side comes out
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// `op` over the tpr threads that share a row.  `red` holds kMaxWarps floats per use; uses that follow one another take other ones, so
// that one barrier each is enough.  All threads of the CTA call it.
template <float (*op)(float, float)>
__device__ __forceinline__ float over_row(float v, int tpr, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, warps = tpr >> 5, first = tpr == int(blockDim.x) ? 0 : warp & ~(warps - 1);
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const float2* sums = reinterpret_cast<const float2*>(red + first);
    v = op(sums[0].x, sums[0].y);
    for (int i = 1; i < warps / 2; ++i) v = op(v, op(sums[i].x, sums[i].y));
    if (warps & 1) v = op(v, red[first + warps - 1]);
  }
  return v;
}

// A row's factor where its squares leave fp32 or vanish from it: in 64 bits, by every warp of the row for itself.  (Infinities and NaN end
// up here as well and give 0 and NaN, rows of zeros without an eps infinity.)
constexpr float kMostFactor = 1125899906842624.f;     // 2^50: squares below 2^-126 are flushed, which a mean of 2^-100 does not feel
// (fp16 has no such numbers: its squares lie between 2^-48 and 2^32; infinities and NaN need nothing else.)
template <typename T>
constexpr bool kLeaves = !std::is_same<T, __half>::value;
template <typename T>
__device__ __forceinline__ bool leaves_fp32(float factor) { return kLeaves<T> && !(factor > 0.f && factor < kMostFactor); }
template <typename T>
__device__ __noinline__ float far_factor(const T* x, const T* r, int C, double eps) {
  double sum = 0.0;
#pragma unroll 1
  for (int c = threadIdx.x & 31; c < C; c += 32) {
    float h = to_f32<T>(x[c]);
    if (r) h = to_f32<T>(from_f32<T>(h + to_f32<T>(r[c])));
    sum += double(h) * double(h);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float s;      // (down to 2^-128 without a flush)
  asm("cvt.rn.f32.f64 %0, %1;" : "=f"(s) : "d"(rsqrt(sum / C + eps)));
  return s;
}

// codes of a chunk's values, each times `inv`
template <int kVec, int kPairs>
__device__ __forceinline__ void store_codes(uint8_t* p, const float2 (&y)[kPairs], float inv) {
  uint32_t c[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) c[i] = __nv_cvt_float2_to_fp8x2(__fmul2_rn(y[i], make_float2(inv, inv)), __NV_SATFINITE, __NV_E4M3);
  if constexpr (kVec == 1) *p = uint8_t(c[0]);
  else if constexpr (kVec == 4) *reinterpret_cast<uint32_t*>(p) = c[0] | c[1] << 16;
  else *reinterpret_cast<uint2*>(p) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}
constexpr float kLeast = 7.888609052210118e-31f;      // 2^-100
template <int kPairs>
__device__ __forceinline__ float top_of(const float2 (&y)[kPairs], float top) {
  // (abs without a flush of small numbers, which is an operand's modifier; fabsf is an instruction here)
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    asm("{\n.reg .f32 a, b;\nabs.f32 a, %1;\nabs.f32 b, %2;\nmax.NaN.f32 a, a, b;\nmax.NaN.f32 %0, %0, a;\n}" : "+f"(top) : "f"(y[i].x), "f"(y[i].y));
  return top;
}
// The scale for a largest magnitude, and what the values are multiplied by: 448 / top, from the reciprocal of the scale (2^-109 or more),
// which is good to 2^-22, by one step of Newton's method; an infinity has a factor of zero, a NaN a NaN.
__device__ __forceinline__ float scale_of(float top) { return top * (1.f / 448.f); }
__device__ __forceinline__ float inverse_of(float top, float scale) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  const float e = fmaf(-top, r, 448.f);
  return e == e ? fmaf(r * (1.f / 448.f), e, r) : r;
}
// The same of a group of lanes' values; its first lane writes the scale.
__device__ __forceinline__ float group_scale(float top, int lanes, float* scale, bool write) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = scale_of(top);
  if (write && (threadIdx.x & (lanes - 1)) == 0) *scale = s;
  return inverse_of(top, s);
}

// The rows of a CTA, from `block` on, whose squares leave fp32: rms_fwd_kernel has left NaN in all that a warp writes of them.  Called behind
// its loop, with arguments of its own, so that nothing is held for it meanwhile: as a call within the loop 105 us instead of 93 (16384 x 4096
// bf16 with a residual), 194 instead of 152 (16384 x 8192 to e4m3).
template <typename T, typename W, int kVec, bool kEight>
__device__ __noinline__ void far_rows(const RmsArgs* pa, int tpr, int64_t block) {
  const RmsArgs a = *pa;
  using C = Chunk<T, kVec>;
  constexpr int kPairs = C::kPairs;
  const int groups = blockDim.x / tpr, mine = groups == 1 ? 0 : threadIdx.x / tpr, tin = threadIdx.x - mine * tpr, lane = threadIdx.x & 31;
  const int step = tpr * kVec, own = tin * kVec;
#pragma unroll 1
  for (;; block += gridDim.x) {
    const int64_t row = block * groups + mine, base = row * a.C;
    if (row >= a.rows) return;
    bool good = false;      // (a thread reads back what it has written itself)
    if (own < a.C) {
      if constexpr (kEight) good = (static_cast<const uint8_t*>(a.y)[base + own] & 0x7f) != 0x7f;
      else good = to_f32<T>(static_cast<const T*>(a.y)[base + own]) == to_f32<T>(static_cast<const T*>(a.y)[base + own]);
    }
    if (own - lane * kVec >= a.C || __any_sync(0xffffffffu, good)) continue;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* r = a.r ? static_cast<const T*>(a.r) + base : nullptr;
    const float s = far_factor(x, r, a.C, a.eps64);
    if (tin == 0 && a.rstd) a.rstd[row] = s;
    auto output = [&](int c, float2 (&f)[kPairs]) {
      float2 v[kPairs];
      C::load_cached(x + c).get(f);
      if (r) {
        C::load_cached(r + c).get(v);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) f[i] = __fadd2_rn(f[i], v[i]);
        C::of(f).get(f);
      }
      weights<W, kVec>(a.w, c, true).get(v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = __fmul2_rn(times(f[i], s), v[i]);
    };
    float inv = 0.f;
    if constexpr (kEight) {
      if (a.group == a.C) {
        float top = kLeast;
#pragma unroll 1
        for (int c = lane * kVec; c < a.C; c += 32 * kVec) {
          float2 f[kPairs];
          output(c, f);
          top = top_of(f, top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float scale = scale_of(top);
        if (tin == 0) a.scales[row] = scale;
        inv = inverse_of(top, scale);
      }
    }
#pragma unroll 1
    for (int c0 = own - lane * kVec; c0 < a.C; c0 += step) {
      const int c = c0 + lane * kVec;
      const bool in = c < a.C;
      float2 f[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = make_float2(0.f, 0.f);
      if (in) output(c, f);
      if constexpr (kEight) {
        if (a.group != a.C) inv = group_scale(top_of(f, kLeast), a.group / kVec, a.scales + ((base + c) >> a.group_shift), in);
        if (in) store_codes<kVec>(static_cast<uint8_t*>(a.y) + base + c, f, inv);
      } else {
        if (in) C::of(f).store(static_cast<T*>(a.y) + base + c);
      }
    }
  }
}

template <typename T, typename W, int kVec, int kPer, int kThreads, bool kEight>
__global__ void __launch_bounds__(kThreads, ctas_of(fwd_threads(kPer, kVec), kThreads)) rms_fwd_kernel(const __grid_constant__ RmsArgs a, int tpr) {
  __shared__ __align__(16) float red[4 * kMaxWarps];
  __shared__ uint8_t far[kMaxWarps];
  using C = Chunk<T, kVec>;
  constexpr int kPairs = C::kPairs;
  const int groups = blockDim.x / tpr, mine = groups == 1 ? 0 : threadIdx.x / tpr, tin = threadIdx.x - mine * tpr;
  const unsigned rows = unsigned(a.rows), blocks = (rows + groups - 1) / groups;      // (counted in 32 bits: registers are what is short here)
  auto column = [&](int p) { return (p * tpr + tin) * kVec; };
  C nx[kPer], nr[kPer];
  auto fetch = [&](unsigned block) {
    const unsigned row = block * groups + mine;
    const bool in_rows = block < blocks && row < rows;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const bool in = in_rows && column(p) < a.C;
      const int64_t at = in ? int64_t(row) * a.C + column(p) : 0;
      nx[p] = in ? C::load(static_cast<const T*>(a.x) + at) : C::zero();
      if (a.r) nr[p] = in ? C::load(static_cast<const T*>(a.r) + at) : C::zero();
    }
  };
  fetch(blockIdx.x);
  // (fp32 with two chunks a thread has no registers for the weights beside the next row: 121 us held, 94 from L1, 8192 x 4096)
  constexpr bool kHeld = !(sizeof(T) == 4 && kVec > 1 && kPer == 2);
  Chunk<W, kVec> w[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p)
    if (kHeld) w[p] = weights<W, kVec>(a.w, column(p), column(p) < a.C);
  int turn = 0;
  if constexpr (kLeaves<T>) {
    if ((threadIdx.x & 31) == 0) far[threadIdx.x >> 5] = 0;      // (of the warp: a flag in a register is one more than there are)
    __syncwarp();
  }
  for (unsigned block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    const unsigned row = block * groups + mine;
    const int64_t base = int64_t(row) * a.C;
    const bool in_rows = row < rows;
    C h[kPer];
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      h[p] = nx[p];
      float2 f[kPairs];
      h[p].get(f);
      if (a.r) {
        float2 g[kPairs];
        nr[p].get(g);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) f[i] = __fadd2_rn(f[i], g[i]);
        h[p] = C::of(f);
        if (in_rows && column(p) < a.C) h[p].store(static_cast<T*>(a.sum) + base + column(p));
        h[p].get(f);
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) ss = __ffma2_rn(f[i], f[i], ss);
    }
    fetch(block + gridDim.x);
    float s = rsqrtf(fmaf(over_row<add>(ss.x + ss.y, tpr, red + turn * kMaxWarps), a.inv_c, a.eps));
    if (leaves_fp32<T>(s)) {
      far[threadIdx.x >> 5] = 1;
      s = __uint_as_float(0x7fffffffu);
    }
    if (tin == 0 && in_rows && a.rstd) a.rstd[row] = s;
    auto output = [&](int p, float2 (&f)[kPairs]) {
      float2 v[kPairs];
      h[p].get(f);
      if (kHeld) w[p].get(v);
      else weights<W, kVec>(a.w, column(p), column(p) < a.C).get(v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = __fmul2_rn(times(f[i], s), v[i]);
    };
    float inv = 0.f;
    if constexpr (kEight) {
      if (a.group == a.C) {
        float top = kLeast;
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          float2 f[kPairs];
          output(p, f);
          top = top_of(f, top);
        }
        top = over_row<max_nan>(top, tpr, red + (2 + turn) * kMaxWarps);
        const float scale = scale_of(top);
        if (tin == 0 && in_rows) a.scales[row] = scale;
        inv = inverse_of(top, scale);
      }
    }
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      float2 f[kPairs];
      output(p, f);
      const bool in = in_rows && column(p) < a.C;
      if constexpr (kEight) {
        if (a.group != a.C)
          inv = group_scale(top_of(f, kLeast), a.group / kVec, a.scales + ((base + column(p)) >> a.group_shift), in);
        if (in) store_codes<kVec>(static_cast<uint8_t*>(a.y) + base + column(p), f, inv);
      } else {
        if (in) C::of(f).store(static_cast<T*>(a.y) + base + column(p));
      }
    }
  }
  if constexpr (kLeaves<T>) {
    __syncwarp();
    if (far[threadIdx.x >> 5]) {
      const RmsArgs* args = &a;
      int threads = tpr;
      asm volatile("" : "+l"(args), "+r"(threads));      // (not what the loop has worked out of them)
      far_rows<T, W, kVec, kEight>(args, threads, blockIdx.x);
    }
  }
}

constexpr int kWide = 256;      // threads of a row that is not held

// A sum over a thread's chunks of a row of any length, kPairs pairs each: fp32, folded into 64 bits every 64 terms.  (One by one in
// fp32, 2^16 terms of one size are 2e-4 off.)  term(c, sum) adds the chunk at column c.
template <int kPairs, int kVec, typename Term>
__device__ __forceinline__ float long_sum(int C, Term term) {
  constexpr int kStep = kWide * kVec;
  double all = 0.0;
  for (int c = threadIdx.x * kVec; c < C;) {
    float2 sum = make_float2(0.f, 0.f);
    const int end = min(C, c + 64 / kPairs * kStep);      // (2^30 + 2^17 at most)
#pragma unroll 4
    for (; c < end; c += kStep) term(c, sum);
    all += double(sum.x) + double(sum.y);
  }
  return float(all);
}

// A row per CTA, read again for its output (and, for one scale of the row, for that).
template <typename T, typename W, int kVec, bool kEight>
__global__ void __launch_bounds__(kWide) rms_fwd_wide_kernel(const RmsArgs a) {
  __shared__ __align__(16) float red[2 * kMaxWarps];
  using C = Chunk<T, kVec>;
  constexpr int kPairs = C::kPairs;
  const int64_t row = blockIdx.x, base = row * a.C;
  const T* x = static_cast<const T*>(a.x) + base;
  const auto square = [&](int c, float2& sum) {
    C h = C::load_cached(x + c);
    float2 f[kPairs], g[kPairs];
    h.get(f);
    if (a.r) {
      C::load_cached(static_cast<const T*>(a.r) + base + c).get(g);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = __fadd2_rn(f[i], g[i]);
      h = C::of(f);
      h.store(static_cast<T*>(a.sum) + base + c);
      h.get(f);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum = __ffma2_rn(f[i], f[i], sum);
  };
  float s = rsqrtf(fmaf(over_row<add>(long_sum<kPairs, kVec>(a.C, square), kWide, red), a.inv_c, a.eps));
  if (leaves_fp32<T>(s)) s = far_factor(x, a.r ? static_cast<const T*>(a.r) + base : nullptr, a.C, a.eps64);
  if (threadIdx.x == 0 && a.rstd) a.rstd[row] = s;
  const T* h = a.r ? static_cast<const T*>(a.sum) + base : x;      // (every thread reads back what it has written itself)
  auto output = [&](int c, float2 (&f)[kPairs]) {
    float2 v[kPairs];
    C::load_cached(h + c).get(f);
    weights<W, kVec>(a.w, c, true).get(v);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) f[i] = __fmul2_rn(times(f[i], s), v[i]);
  };
  float inv = 0.f;
  if constexpr (kEight) {
    if (a.group == a.C) {
      float top = kLeast;
      for (int c = threadIdx.x * kVec; c < a.C; c += kWide * kVec) {
        float2 f[kPairs];
        output(c, f);
        top = top_of(f, top);
      }
      top = over_row<max_nan>(top, kWide, red + kMaxWarps);
      const float scale = scale_of(top);
      if (threadIdx.x == 0) a.scales[row] = scale;
      inv = inverse_of(top, scale);
    }
  }
  // (whole warps go round together: a group's lanes are in one)
  for (int c0 = (threadIdx.x & ~31) * kVec; c0 < a.C; c0 += kWide * kVec) {
    const int c = c0 + (threadIdx.x & 31) * kVec;
    const bool in = c < a.C;
    float2 f[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) f[i] = make_float2(0.f, 0.f);
    if (in) output(c, f);
    if constexpr (kEight) {
      if (a.group != a.C)
        inv = group_scale(top_of(f, kLeast), a.group / kVec, a.scales + ((base + c) >> a.group_shift), in);
      if (in) store_codes<kVec>(static_cast<uint8_t*>(a.y) + base + c, f, inv);
    } else {
      if (in) C::of(f).store(static_cast<T*>(a.y) + base + c);
    }
  }
}

// Backward.  A thread always has the same columns, whose part of dw stays in its registers; it copies its own chunks of the next
// kAhead rows into its own places of a ring in shared memory, so that no barrier is needed for them.
template <int kPer, int kThreads, int kChunkBytes>
struct Ring {
  static constexpr int kThread = 3 * kPer * kChunkBytes;                        // h, dy and dsum of a row, of a thread
  static constexpr int kAhead = kThread * kThreads <= 24576 ? 2 : 1;
  __host__ __device__ static constexpr int bytes(int threads) { return (kAhead + 1) * kThread * threads; }
};
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool in) {
  const uint32_t d = uint32_t(__cvta_generic_to_shared(dst));
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(in ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(in ? 4 : 0) : "memory");
}

template <typename T, typename W, int kVec, int kPer, int kThreads, int kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) rms_bwd_kernel(const RmsArgs a, int tpr) {
  using Ch = Chunk<T, kVec>;
  constexpr int kPairs = Ch::kPairs, kSize = kVec * int(sizeof(T));
  using Rg = Ring<kPer, kThreads, kSize>;
  extern __shared__ __align__(16) char ring[];
  __shared__ __align__(16) float red[2 * kMaxWarps];
  const int groups = blockDim.x / tpr, mine = groups == 1 ? 0 : threadIdx.x / tpr, tin = threadIdx.x - mine * tpr;
  auto column = [&](int p) { return (p * tpr + tin) * kVec; };
  float2 dw[kPer][kPairs];
  Chunk<W, kVec> w[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) dw[p][i] = make_float2(0.f, 0.f);
    w[p] = weights<W, kVec>(a.w, column(p), column(p) < a.C);
  }
  const int64_t blocks = (a.rows + groups - 1) / groups;
  auto place = [&](int stage, int which, int p) { return ring + (((stage * 3 + which) * kPer + p) * int(blockDim.x) + threadIdx.x) * kSize; };
  auto fetch = [&](int64_t block, int stage) {
    const int64_t row = block * groups + mine;
    const bool in_rows = block < blocks && row < a.rows;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const bool in = in_rows && column(p) < a.C;
      const int64_t at = in ? row * a.C + column(p) : 0;
      if constexpr (kSize >= 4) {
        copy_async<kSize>(place(stage, 0, p), static_cast<const T*>(a.x) + at, in);
        copy_async<kSize>(place(stage, 1, p), static_cast<const T*>(a.dy) + at, in);
        if (a.dsum) copy_async<kSize>(place(stage, 2, p), static_cast<const T*>(a.dsum) + at, in);
      } else {      // (no asynchronous copies of two bytes)
        (in ? Ch::load(static_cast<const T*>(a.x) + at) : Ch::zero()).store(reinterpret_cast<T*>(place(stage, 0, p)));
        (in ? Ch::load(static_cast<const T*>(a.dy) + at) : Ch::zero()).store(reinterpret_cast<T*>(place(stage, 1, p)));
        if (a.dsum) (in ? Ch::load(static_cast<const T*>(a.dsum) + at) : Ch::zero()).store(reinterpret_cast<T*>(place(stage, 2, p)));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return in_rows ? __ldg(a.rstd + row) : 0.f;
  };
  float rstds[Rg::kAhead];
#pragma unroll
  for (int i = 0; i < Rg::kAhead; ++i) rstds[i] = fetch(blockIdx.x + int64_t(i) * gridDim.x, i);
  int stage = 0, turn = 0;
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    const int64_t row = block * groups + mine;
    const float rstd = rstds[0];
    if constexpr (Rg::kAhead == 2) rstds[0] = rstds[1];
    // (into the stage before this one, which this thread has left)
    rstds[Rg::kAhead - 1] = fetch(block + int64_t(Rg::kAhead) * gridDim.x, stage == 0 ? Rg::kAhead : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(Rg::kAhead) : "memory");
    float2 t2 = make_float2(0.f, 0.f), n[kPer][kPairs], g[kPer][kPairs];
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      float2 v[kPairs];
      Ch::load_cached(reinterpret_cast<const T*>(place(stage, 0, p))).get(n[p]);
      Ch::load_cached(reinterpret_cast<const T*>(place(stage, 1, p))).get(g[p]);
      w[p].get(v);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        n[p][i] = times(n[p][i], rstd);
        dw[p][i] = __ffma2_rn(g[p][i], n[p][i], dw[p][i]);
        g[p][i] = __fmul2_rn(g[p][i], v[i]);
        t2 = __ffma2_rn(g[p][i], n[p][i], t2);
      }
    }
    const float mean = over_row<add>(t2.x + t2.y, tpr, red + turn * kMaxWarps) * a.inv_c;
    const float2 by = make_float2(-mean, -mean), s2 = make_float2(rstd, rstd);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      if (row >= a.rows || column(p) >= a.C) continue;
      float2 d[kPairs];
      if (a.dsum) {
        Ch::load_cached(reinterpret_cast<const T*>(place(stage, 2, p))).get(d);
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) d[i] = make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) d[i] = __ffma2_rn(s2, __ffma2_rn(n[p][i], by, g[p][i]), d[i]);
      Ch::of(d).store(static_cast<T*>(a.dx) + row * a.C + column(p));
    }
    stage = stage == Rg::kAhead ? 0 : stage + 1;
  }
  if (!a.part) return;
  if (groups > 1) {      // one group after the other, so that the sums have one order
    float* columns = reinterpret_cast<float*>(ring);
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int k = 0; k < groups; ++k) {
      __syncthreads();
      if (mine == k) {
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          const float* own = reinterpret_cast<const float*>(dw[p]);
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (column(p) < a.C) columns[column(p) + i] = own[i] + (k ? columns[column(p) + i] : 0.f);
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) a.part[int64_t(blockIdx.x) * a.C + c] = columns[c];
    return;
  }
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    if (column(p) >= a.C) continue;
    float* to = a.part + int64_t(blockIdx.x) * a.C + column(p);
    if constexpr (kVec == 1) {
      *to = dw[p][0].x;
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; i += 2) *reinterpret_cast<float4*>(to + 2 * i) = make_float4(dw[p][i].x, dw[p][i].y, dw[p][i + 1].x, dw[p][i + 1].y);
    }
  }
}

// dx of a row per CTA, read twice.
template <typename T, typename W, int kVec>
__global__ void __launch_bounds__(kWide) rms_bwd_wide_kernel(const RmsArgs a) {
  __shared__ __align__(16) float red[kMaxWarps];
  using Ch = Chunk<T, kVec>;
  constexpr int kPairs = Ch::kPairs;
  const int64_t row = blockIdx.x, base = row * a.C;
  const float rstd = a.rstd[row];
  const float2 s2 = make_float2(rstd, rstd);
  auto operands = [&](int c, float2 (&n)[kPairs], float2 (&g)[kPairs]) {      // n, and dy w
    float2 v[kPairs];
    Ch::load_cached(static_cast<const T*>(a.x) + base + c).get(n);
    Ch::load_cached(static_cast<const T*>(a.dy) + base + c).get(g);
    weights<W, kVec>(a.w, c, true).get(v);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      n[i] = times(n[i], rstd);
      g[i] = __fmul2_rn(g[i], v[i]);
    }
  };
  const auto product = [&](int c, float2& sum) {
    float2 n[kPairs], g[kPairs];
    operands(c, n, g);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum = __ffma2_rn(g[i], n[i], sum);
  };
  const float mean = over_row<add>(long_sum<kPairs, kVec>(a.C, product), kWide, red) * a.inv_c;
  for (int c = threadIdx.x * kVec; c < a.C; c += kWide * kVec) {
    float2 n[kPairs], g[kPairs], d[kPairs];
    operands(c, n, g);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) d[i] = make_float2(0.f, 0.f);
    if (a.dsum) Ch::load_cached(static_cast<const T*>(a.dsum) + base + c).get(d);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) d[i] = __ffma2_rn(s2, __ffma2_rn(n[i], make_float2(-mean, -mean), g[i]), d[i]);
    Ch::of(d).store(static_cast<T*>(a.dx) + base + c);
  }
}
// Sums of dw are fp32 over that many rows of a thread at most (2^14 rows of one size are 1e-4 off); what they come to is added in 64 bits.
constexpr int kChain = 256;

// dw of wide rows: a thread has a column, a CTA row the rows of its part.
template <typename T>
__global__ void __launch_bounds__(kWide) rms_dweight_wide_kernel(const RmsArgs a) {
  const int c = blockIdx.x * kWide + threadIdx.x;
  if (c >= a.C) return;
  const int64_t r1 = a.rows * (blockIdx.y + 1) / gridDim.y;
  const auto chain = [&](int64_t r, int64_t end) {
    float sum = 0.f;
#pragma unroll 4
    for (; r < end; ++r)
      sum = fmaf(to_f32<T>(static_cast<const T*>(a.dy)[r * a.C + c]), times(make_float2(to_f32<T>(static_cast<const T*>(a.x)[r * a.C + c]), 0.f), a.rstd[r]).x, sum);
    return sum;
  };
  int64_t r = a.rows * blockIdx.y / gridDim.y;
  float sum = chain(r, min(r1, r + kChain));
  if (r1 - r > kChain) {
    double all = sum;
    for (r += kChain; r < r1; r += kChain) all += chain(r, min(r1, r + kChain));
    sum = float(all);
  }
  a.part[int64_t(blockIdx.y) * a.C + c] = sum;
}

// The sum of the partial rows, 32 columns per CTA, every 32nd row per warp, in one order.
template <typename W>
__global__ void __launch_bounds__(1024) rms_dweight_kernel(const float* part, int rows, int C, W* out) {
  __shared__ float sums[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  wait_for_previous();
  if (c < C) {
    const auto chain = [&](int r, int end) {
      float part_sum = 0.f;
#pragma unroll 4
      for (; r < end; r += 32) part_sum += __ldcg(part + int64_t(r) * C + c);
      return part_sum;
    };
    sum = chain(threadIdx.y, min(rows, 1024));
    if (rows > 1024) {
      double all = sum;
      for (int r = 1024; r < rows; r += 1024) all += chain(r + threadIdx.y, min(rows, r + 1024));
      sum = float(all);
    }
  }
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  float v = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < C) out[blockIdx.x * 32 + threadIdx.y] = from_f32<W>(v);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a row is divided: by `tpr` threads, a power of two that shares a CTA of 256 with other rows, or from 160 on a CTA of its own.
struct Shape {
  bool vec;
  int tpr, threads;
  int per;       // chunks of a thread: least_per, two, four or (forward) eight times that; 0: the row is too wide to be held
};
constexpr int least_per(bool vec) { return vec ? 1 : 4; }

// The backward takes one chunk a thread as long as 512 threads hold the row (16384 rows of 4096, bf16: two chunks of 256 threads 124 us,
// one of 512 90; 1024 threads for 8192 channels 89, two chunks of 512 78), the forward two (93 us either way, and fewer shuffles).
Shape shape_of(int C, int esz, bool vec, bool backward) {
  Shape s{vec, 0, 0, 0};
  const int chunks = vec ? C / (16 / esz) : C, least = least_per(vec);
  for (int per = backward ? least : 2 * least; per <= (backward ? 4 : 8) * least; per *= 2) {
    const int threads = (chunks + per - 1) / per;
    if (threads > 512) continue;
    s.per = per;
    if (threads > 128) {
      s.tpr = s.threads = (threads + 31) / 32 * 32;
    } else {
      s.threads = 256;
      for (s.tpr = 32; s.tpr < threads;) s.tpr *= 2;
      if (!backward && s.tpr * least >= chunks) s.per = least;      // (short rows, of a warp)
    }
    return s;
  }
  return s;
}

int check(const nb200_rms_norm_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_rms_norm_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  if (p->dtype != NB200_F32 && p->dtype != NB200_BF16 && p->dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (p->weight_dtype != p->dtype && p->weight_dtype != NB200_F32) { set_error("%s: the weight must be of the operands' dtype or fp32", what); return NB200_ERR_INVALID; }
  if (p->rows < 0 || p->channels <= 0) { set_error("%s: bad extents", what); return NB200_ERR_INVALID; }
  if (p->channels > 1 << 30) { set_error("%s: %d channels, at most 2^30", what, p->channels); return NB200_ERR_UNSUPPORTED; }      // (counted in 32 bits)
  if (p->rows > 0x7fffffff) { set_error("%s: %lld rows, at most 2^31 - 1", what, static_cast<long long>(p->rows)); return NB200_ERR_UNSUPPORTED; }
  return NB200_OK;
}

// Rows of 16-byte words that all pointers are aligned to.
bool vectors(const nb200_rms_norm_params* p, bool backward) {
  if (int64_t(p->channels) * dtype_size(p->dtype) % 16) return false;
  if (!aligned16(p->x) || !aligned16(p->weight)) return false;
  if (backward) return aligned16(p->dy) && aligned16(p->dsum) && aligned16(p->dx);
  return aligned16(p->residual) && aligned16(p->sum) && aligned16(p->y);
}

// Calls f with the kernel's (kVec, kPer, kThreads: the most threads of a CTA).
template <typename T, bool kForward, typename F>
int with_shape(const Shape& s, F f) {
  constexpr int kVec = 16 / int(sizeof(T));
  auto with_per = [&](auto vec, auto threads) {
    constexpr int kLeast = least_per(decltype(vec)::value > 1);
    if (s.per == kLeast) return f(vec, std::integral_constant<int, kLeast>{}, threads);
    if (s.per == 2 * kLeast) return f(vec, std::integral_constant<int, 2 * kLeast>{}, threads);
    if constexpr (decltype(threads)::value == 512) {      // (smaller CTAs have rows of few chunks a thread)
      if (s.per == 4 * kLeast) return f(vec, std::integral_constant<int, 4 * kLeast>{}, threads);
      if constexpr (kForward) return f(vec, std::integral_constant<int, 8 * kLeast>{}, threads);
    }
    set_error("rms_norm: no kernel for %d chunks a thread", s.per);
    return int(NB200_ERR_UNSUPPORTED);
  };
  auto with_threads = [&](auto vec) {
    return s.threads <= 256 ? with_per(vec, std::integral_constant<int, 256>{}) : with_per(vec, std::integral_constant<int, 512>{});
  };
  return s.vec ? with_threads(std::integral_constant<int, kVec>{}) : with_threads(std::integral_constant<int, 1>{});
}

// The backward's shape, its shared memory and CTAs; the rows of a launch, and the rows of partial sums that all launches leave, one per CTA.
struct BwdPlan {
  Shape s;
  int smem, ctas;
  int64_t launch_rows;
  int parts;
};
template <typename T>
BwdPlan bwd_plan(int C, int64_t rows, bool vec) {
  BwdPlan pl{shape_of(C, int(sizeof(T)), vec, true), 0, 0, rows, 0};
  if (rows == 0) return pl;
  if (pl.s.per == 0) {
    pl.parts = int(rows < 64 ? rows : 64);
    return pl;
  }
  with_shape<T, false>(pl.s, [&](auto kv, auto kp, auto kt) {
    constexpr int kVec = decltype(kv)::value, kPer = decltype(kp)::value, kThreads = decltype(kt)::value;
    // (the sums of rows that share a CTA are joined in the ring)
    const int ring = Ring<kPer, kThreads, kVec * int(sizeof(T))>::bytes(pl.s.threads), columns = pl.s.tpr < pl.s.threads ? C * 4 : 0;
    pl.smem = ring > columns ? ring : columns;
    const int by_threads = ctas_of(bwd_threads(kPer * kVec), pl.s.threads), by_room = 227 * 1024 / (pl.smem + 2048);
    const int64_t groups = pl.s.threads / pl.s.tpr, blocks = (rows + groups - 1) / groups;
    const int64_t most = int64_t(tc::sm_count()) * (by_threads < by_room ? by_threads : by_room);
    pl.ctas = int(blocks < most ? blocks : most);
    // (a launch for each kChain rows of a thread: 0.4 ms of work and more)
    const int64_t launch_blocks = int64_t(pl.ctas) * kChain, whole = blocks / launch_blocks, rest = blocks % launch_blocks;
    pl.launch_rows = launch_blocks * groups;
    pl.parts = int(whole * pl.ctas + (rest < pl.ctas ? rest : pl.ctas));
    return int(NB200_OK);
  });
  return pl;
}
BwdPlan bwd_plan(const nb200_rms_norm_params* p) {
  const bool vec = vectors(p, true);
  return p->dtype == NB200_F32 ? bwd_plan<float>(p->channels, p->rows, vec) : bwd_plan<__half>(p->channels, p->rows, vec);
}

template <typename T, typename W, bool kEight>
int launch_fwd(const RmsArgs& a, const Shape& s, cudaStream_t st) {
  constexpr int kVec = 16 / int(sizeof(T));
  if (s.per == 0) {
    if (s.vec) rms_fwd_wide_kernel<T, W, kVec, kEight><<<unsigned(a.rows), kWide, 0, st>>>(a);
    else rms_fwd_wide_kernel<T, W, 1, kEight><<<unsigned(a.rows), kWide, 0, st>>>(a);
    count_launch();
    return check_launch("rms_fwd_wide_kernel");
  }
  return with_shape<T, true>(s, [&](auto kv, auto kp, auto kt) {
    constexpr int kV = decltype(kv)::value, kPer = decltype(kp)::value, kThreads = decltype(kt)::value;
    const int64_t groups = s.threads / s.tpr, blocks = (a.rows + groups - 1) / groups;
    const int64_t most = int64_t(tc::sm_count()) * ctas_of(fwd_threads(kPer, kV), s.threads);
    rms_fwd_kernel<T, W, kV, kPer, kThreads, kEight><<<unsigned(blocks < most ? blocks : most), s.threads, 0, st>>>(a, s.tpr);
    count_launch();
    return check_launch("rms_fwd_kernel");
  });
}
template <typename T, typename W>
int launch_fwd(const RmsArgs& a, const Shape& s, cudaStream_t st) {
  return a.scales ? launch_fwd<T, W, true>(a, s, st) : launch_fwd<T, W, false>(a, s, st);
}

template <typename T, typename W>
int launch_rows(const RmsArgs& a, const BwdPlan& pl, cudaStream_t st) {
  constexpr int kVec = 16 / int(sizeof(T));
  if (pl.s.per == 0) {
    if (pl.s.vec) rms_bwd_wide_kernel<T, W, kVec><<<unsigned(a.rows), kWide, 0, st>>>(a);
    else rms_bwd_wide_kernel<T, W, 1><<<unsigned(a.rows), kWide, 0, st>>>(a);
    count_launch();
    if (int rc = check_launch("rms_bwd_wide_kernel")) return rc;
    if (!a.part) return NB200_OK;
    rms_dweight_wide_kernel<T><<<dim3(unsigned((a.C + kWide - 1) / kWide), unsigned(pl.parts)), kWide, 0, st>>>(a);
    count_launch();
    return check_launch("rms_dweight_wide_kernel");
  }
  return with_shape<T, false>(pl.s, [&](auto kv, auto kp, auto kt) {
    constexpr int kV = decltype(kv)::value, kPer = decltype(kp)::value, kThreads = decltype(kt)::value;
    auto kernel = rms_bwd_kernel<T, W, kV, kPer, kThreads, ctas_of(bwd_threads(kPer * kV), kThreads)>;
    if (pl.smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pl.smem) != cudaSuccess) return check_launch("rms_bwd_kernel");
    for (int64_t r0 = 0; r0 < a.rows; r0 += pl.launch_rows) {
      const int64_t at = r0 * a.C;
      RmsArgs b = a;
      b.x = static_cast<const T*>(a.x) + at; b.dy = static_cast<const T*>(a.dy) + at; b.dx = static_cast<T*>(a.dx) + at;
      if (a.dsum) b.dsum = static_cast<const T*>(a.dsum) + at;
      b.rstd = a.rstd + r0;
      b.rows = a.rows - r0 < pl.launch_rows ? a.rows - r0 : pl.launch_rows;
      if (a.part) b.part = a.part + r0 / pl.launch_rows * pl.ctas * a.C;
      const int64_t groups = pl.s.threads / pl.s.tpr, blocks = (b.rows + groups - 1) / groups;
      kernel<<<unsigned(blocks < pl.ctas ? blocks : pl.ctas), pl.s.threads, pl.smem, st>>>(b, pl.s.tpr);
      count_launch();
      if (int rc = check_launch("rms_bwd_kernel")) return rc;
    }
    return int(NB200_OK);
  });
}
template <typename T, typename W>
int launch_bwd(const RmsArgs& a, const BwdPlan& pl, void* dweight, cudaStream_t st) {
  if (int rc = launch_rows<T, W>(a, pl, st)) return rc;
  if (!a.part) return NB200_OK;
  if (launch_dependent(rms_dweight_kernel<W>, dim3(unsigned((a.C + 31) / 32)), dim3(32, 32), 0, st, static_cast<const float*>(a.part), pl.parts, a.C, static_cast<W*>(dweight)) != cudaSuccess)
    return check_launch("rms_dweight_kernel");
  count_launch();
  return check_launch("rms_dweight_kernel");
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_rms_norm_workspace_bytes(const nb200_rms_norm_params* p, size_t* bytes) {
  if (!bytes) { set_error("bytes out-pointer is NULL"); return NB200_ERR_INVALID; }
  if (int rc = check(p, "rms_norm_workspace_bytes")) return rc;
  *bytes = size_t(bwd_plan(p).parts) * size_t(p->channels) * sizeof(float);
  return NB200_OK;
}

extern "C" NB200_API int nb200_rms_norm_fwd(const nb200_rms_norm_params* p, void* cuda_stream) {
  if (int rc = check(p, "rms_norm_fwd")) return rc;
  if (p->rows == 0) return NB200_OK;
  if (!p->x || !p->y || (p->residual && !p->sum)) { set_error("rms_norm_fwd: NULL operand"); return NB200_ERR_INVALID; }
  const bool vec = vectors(p, false);
  if (p->scales && p->group) {
    if ((p->group != 32 && p->group != 64 && p->group != 128) || p->channels % p->group) {
      set_error("rms_norm_fwd: groups of %d of %d channels; 32, 64 or 128 that divide them are possible", p->group, p->channels);
      return NB200_ERR_UNSUPPORTED;
    }
    if (!vec) { set_error("rms_norm_fwd: with groups the operands must begin on 16-byte boundaries"); return NB200_ERR_ALIGNMENT; }
  }
  RmsArgs a{};
  a.x = p->x; a.r = p->residual; a.w = p->weight; a.y = p->y; a.sum = p->sum; a.rstd = p->rstd; a.scales = p->scales;
  a.rows = p->rows; a.C = p->channels;
  a.group = p->group ? p->group : p->channels;
  a.group_shift = p->group == 32 ? 5 : p->group == 64 ? 6 : 7;
  a.eps = p->eps;
  a.eps64 = p->eps;
  a.inv_c = float(1.0 / p->channels);
  const Shape s = shape_of(p->channels, dtype_size(p->dtype), vec, false);
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  const bool wide_weight = p->weight_dtype == NB200_F32;
  if (p->dtype == NB200_F32) return launch_fwd<float, float>(a, s, st);
  if (p->dtype == NB200_BF16) return wide_weight ? launch_fwd<__nv_bfloat16, float>(a, s, st) : launch_fwd<__nv_bfloat16, __nv_bfloat16>(a, s, st);
  return wide_weight ? launch_fwd<__half, float>(a, s, st) : launch_fwd<__half, __half>(a, s, st);
}

extern "C" NB200_API int nb200_rms_norm_bwd(const nb200_rms_norm_params* p, void* cuda_stream) {
  if (int rc = check(p, "rms_norm_bwd")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  if (p->rows == 0) {
    if (p->dweight && cudaMemsetAsync(p->dweight, 0, size_t(p->channels) * dtype_size(p->weight_dtype), st) != cudaSuccess) return check_launch("rms_norm_bwd: clearing dweight");
    return NB200_OK;
  }
  if (!p->x || !p->dy || !p->dx || !p->rstd) { set_error("rms_norm_bwd: NULL operand"); return NB200_ERR_INVALID; }
  const BwdPlan pl = bwd_plan(p);
  RmsArgs a{};
  a.x = p->x; a.w = p->weight; a.rstd = p->rstd; a.dy = p->dy; a.dsum = p->dsum; a.dx = p->dx;
  a.rows = p->rows; a.C = p->channels;
  a.inv_c = float(1.0 / p->channels);
  if (p->dweight) {
    const size_t need = size_t(pl.parts) * size_t(p->channels) * sizeof(float);
    if (!p->workspace || p->workspace_bytes < need) {
      set_error("rms_norm_bwd: workspace of %zu bytes needed (nb200_rms_norm_workspace_bytes), %zu given", need, p->workspace_bytes);
      return NB200_ERR_WORKSPACE;
    }
    if (!aligned16(p->workspace)) { set_error("rms_norm_bwd: the workspace must begin on a 16-byte boundary"); return NB200_ERR_ALIGNMENT; }
    a.part = static_cast<float*>(p->workspace);
  }
  prof_call_begin(st);
  const bool wide_weight = p->weight_dtype == NB200_F32;
  if (p->dtype == NB200_F32) return launch_bwd<float, float>(a, pl, p->dweight, st);
  if (p->dtype == NB200_BF16)
    return wide_weight ? launch_bwd<__nv_bfloat16, float>(a, pl, p->dweight, st) : launch_bwd<__nv_bfloat16, __nv_bfloat16>(a, pl, p->dweight, st);
  return wide_weight ? launch_bwd<__half, float>(a, pl, p->dweight, st) : launch_bwd<__half, __half>(a, pl, p->dweight, st);
}
