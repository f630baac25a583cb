// Root-mean-square norm over the trailing axis with the addition of a residual stream, forward and backward, and with an output
// in 8 bits.
//
//   forward   h = x + r (rounded to the storage type),  s = (mean h^2 + eps)^-1/2,  y = h s w
//             8 bits: a = max |y| of a row or group of channels, scale = a / 448, code = e4m3(y 448 / a)
//   backward  n = h s,  g = dy w,  dx = dh + s (g - n mean(g n)),  dw = sum_rows dy n
//
// Bound by HBM: every stream is read once and written once, so a row is held in registers between its sum and its output: by
// tpr threads (a power of two, up to the CTA's 256), kPer chunks of kVec elements each.  kVec is a 16-byte word's elements, or
// one where rows do not begin on 16-byte boundaries.  Rows that are too long for that are read once more (the *_wide kernels).
#include <cuda_fp8.h>
#include <math.h>

#include "nitrix_b200_rms_norm.h"
#include "sdpa_tc_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

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
  int group;        // channels of a scale
  float eps, inv_c;
};

// kVec consecutive elements as they lie in memory.
template <typename T, int kVec>
struct Chunk {
  uint4 w;
  __device__ __forceinline__ static Chunk load(const T* p) { return Chunk{sm100::ldg_no_allocate(reinterpret_cast<const uint4*>(p))}; }
  __device__ __forceinline__ static Chunk load_cached(const T* p) { return Chunk{*reinterpret_cast<const uint4*>(p)}; }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ void get(float (&f)[kVec]) const {
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = to_f32<T>(e[i]);
  }
  __device__ __forceinline__ static Chunk of(const float (&f)[kVec]) {
    Chunk c;
    T* e = reinterpret_cast<T*>(&c.w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) e[i] = from_f32<T>(f[i]);
    return c;
  }
  __device__ __forceinline__ static Chunk zero() { return Chunk{make_uint4(0, 0, 0, 0)}; }
};
template <typename T>
struct Chunk<T, 1> {
  T v;
  __device__ __forceinline__ static Chunk load(const T* p) { return Chunk{__ldg(p)}; }
  __device__ __forceinline__ static Chunk load_cached(const T* p) { return Chunk{*p}; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f32<T>(v); }
  __device__ __forceinline__ static Chunk of(const float (&f)[1]) { return Chunk{from_f32<T>(f[0])}; }
  __device__ __forceinline__ static Chunk zero() { return Chunk{from_f32<T>(0.f)}; }
};

// kVec weights of type W (ones without a weight)
template <typename W, int kVec>
__device__ __forceinline__ void weights(const void* w, int c, float (&f)[kVec]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = 1.f;
    return;
  }
  const W* p = static_cast<const W*>(w) + c;
  if constexpr (kVec == 1) {
    f[0] = to_f32<W>(__ldg(p));
  } else {
    constexpr int kWords = kVec * int(sizeof(W)) / 16, kEach = kVec / kWords;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const uint4 word = __ldg(reinterpret_cast<const uint4*>(p) + j);
      const W* e = reinterpret_cast<const W*>(&word);
#pragma unroll
      for (int i = 0; i < kEach; ++i) f[j * kEach + i] = to_f32<W>(e[i]);
    }
  }
}

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN on either side comes out
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// `op` over the tpr threads that share a row.  `red` holds kWarps floats per use; uses that follow one another take other ones, so
// that one barrier each is enough.  All threads of the CTA call it.
template <float (*op)(float, float)>
__device__ __forceinline__ float over_row(float v, int tpr, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, warps = tpr >> 5, first = warp & ~(warps - 1);
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[first];
    for (int i = 1; i < warps; ++i) v = op(v, red[first + i]);
  }
  return v;
}

// codes of kVec values, each times `inv`
template <int kVec>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[kVec], float inv) {
  if constexpr (kVec == 1) {
    *p = __nv_cvt_float_to_fp8(y[0] * inv, __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[kVec / 4];
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i] * inv, y[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * i + 2] * inv, y[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    }
    if constexpr (kVec == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}
constexpr float kLeast = 7.888609052210118e-31f;      // 2^-100
template <int kVec>
__device__ __forceinline__ float top_of(const float (&y)[kVec], float top) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) top = max_nan(top, fabsf(y[i]));
  return top;
}
// The scale of a group of lanes' values, written by its first lane; what the values are multiplied by.
__device__ __forceinline__ float group_scale(float top, int lanes, float* scale) {
  for (int o = lanes >> 1; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & (lanes - 1)) == 0 && scale) *scale = __fdiv_rn(top, 448.f);
  return __fdiv_rn(448.f, top);
}

template <typename T, typename W, int kVec, int kPer, bool kEight>
__global__ void __launch_bounds__(kThreads, kPer <= 2 ? 4 : 2) rms_fwd_kernel(const RmsArgs a, int tpr) {
  __shared__ float red[2 * kWarps];
  using C = Chunk<T, kVec>;
  const int tin = threadIdx.x & (tpr - 1);
  const int64_t row = int64_t(blockIdx.x) * (kThreads / tpr) + threadIdx.x / tpr;
  const bool in_rows = row < a.rows;
  const int64_t base = in_rows ? row * a.C : 0;
  auto column = [&](int p) { return (p * tpr + tin) * kVec; };
  C h[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) h[p] = in_rows && column(p) < a.C ? C::load(static_cast<const T*>(a.x) + base + column(p)) : C::zero();
  if (a.r) {
    C r[kPer];
#pragma unroll
    for (int p = 0; p < kPer; ++p) r[p] = in_rows && column(p) < a.C ? C::load(static_cast<const T*>(a.r) + base + column(p)) : C::zero();
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      float f[kVec], g[kVec];
      h[p].get(f);
      r[p].get(g);
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] += g[i];
      h[p] = C::of(f);
      if (in_rows && column(p) < a.C) h[p].store(static_cast<T*>(a.sum) + base + column(p));
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    float f[kVec];
    h[p].get(f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) ss = fmaf(f[i], f[i], ss);
  }
  const float s = __frsqrt_rn(fmaf(over_row<add>(ss, tpr, red), a.inv_c, a.eps));
  if (tin == 0 && in_rows && a.rstd) a.rstd[row] = s;
  auto output = [&](int p, float (&f)[kVec]) {
    float w[kVec];
    h[p].get(f);
    if (column(p) < a.C) weights<W, kVec>(a.w, column(p), w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = column(p) < a.C ? f[i] * s * w[i] : 0.f;
  };
  float inv = 0.f;
  if constexpr (kEight) {
    if (a.group == a.C) {
      float top = kLeast;
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        float f[kVec];
        output(p, f);
        top = top_of(f, top);
      }
      top = over_row<max_nan>(top, tpr, red + kWarps);
      if (tin == 0 && in_rows) a.scales[row] = __fdiv_rn(top, 448.f);
      inv = __fdiv_rn(448.f, top);
    }
  }
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    float f[kVec];
    output(p, f);
    const bool in = in_rows && column(p) < a.C;
    if constexpr (kEight) {
      if (a.group != a.C)
        inv = group_scale(top_of(f, kLeast), a.group / kVec, in ? a.scales + row * (a.C / a.group) + column(p) / a.group : nullptr);
      if (in) store_codes<kVec>(static_cast<uint8_t*>(a.y) + base + column(p), f, inv);
    } else {
      if (in) C::of(f).store(static_cast<T*>(a.y) + base + column(p));
    }
  }
}

// A row per CTA, read again for its output (and, for one scale of the row, for that).
template <typename T, typename W, int kVec, bool kEight>
__global__ void __launch_bounds__(kThreads) rms_fwd_wide_kernel(const RmsArgs a) {
  __shared__ float red[2 * kWarps];
  using C = Chunk<T, kVec>;
  const int64_t row = blockIdx.x, base = row * a.C;
  const T* x = static_cast<const T*>(a.x) + base;
  float ss = 0.f;
  for (int c = threadIdx.x * kVec; c < a.C; c += kThreads * kVec) {
    C h = C::load_cached(x + c);
    float f[kVec], g[kVec];
    h.get(f);
    if (a.r) {
      C::load_cached(static_cast<const T*>(a.r) + base + c).get(g);
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[i] += g[i];
      h = C::of(f);
      h.store(static_cast<T*>(a.sum) + base + c);
      h.get(f);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) ss = fmaf(f[i], f[i], ss);
  }
  const float s = __frsqrt_rn(fmaf(over_row<add>(ss, kThreads, red), a.inv_c, a.eps));
  if (threadIdx.x == 0 && a.rstd) a.rstd[row] = s;
  const T* h = a.r ? static_cast<const T*>(a.sum) + base : x;      // (every thread reads back what it has written itself)
  auto output = [&](int c, float (&f)[kVec]) {
    float w[kVec];
    C::load_cached(h + c).get(f);
    weights<W, kVec>(a.w, c, w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = f[i] * s * w[i];
  };
  float inv = 0.f;
  if constexpr (kEight) {
    if (a.group == a.C) {
      float top = kLeast;
      for (int c = threadIdx.x * kVec; c < a.C; c += kThreads * kVec) {
        float f[kVec];
        output(c, f);
        top = top_of(f, top);
      }
      top = over_row<max_nan>(top, kThreads, red + kWarps);
      if (threadIdx.x == 0) a.scales[row] = __fdiv_rn(top, 448.f);
      inv = __fdiv_rn(448.f, top);
    }
  }
  // (whole warps go round together: a group's lanes are in one)
  for (int c0 = (threadIdx.x & ~31) * kVec; c0 < a.C; c0 += kThreads * kVec) {
    const int c = c0 + (threadIdx.x & 31) * kVec;
    const bool in = c < a.C;
    float f[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = 0.f;
    if (in) output(c, f);
    if constexpr (kEight) {
      if (a.group != a.C)
        inv = group_scale(top_of(f, kLeast), a.group / kVec, in ? a.scales + row * (a.C / a.group) + c / a.group : nullptr);
      if (in) store_codes<kVec>(static_cast<uint8_t*>(a.y) + base + c, f, inv);
    } else {
      if (in) C::of(f).store(static_cast<T*>(a.y) + base + c);
    }
  }
}

// Backward.  CTAs walk the rows with a stride; a thread always has the same columns, whose part of dw stays in its registers, and
// asks for its chunks of the next row before it works on the present one.
template <typename T, typename W, int kVec, int kPer>
__global__ void __launch_bounds__(kThreads, kPer * kVec <= 8 ? 4 : kPer * kVec <= 16 ? 3 : kPer * kVec <= 32 ? 2 : 1)
rms_bwd_kernel(const RmsArgs a, int tpr) {
  extern __shared__ float columns[];      // [C], where rows share a CTA
  __shared__ float red[2][kWarps];
  using Ch = Chunk<T, kVec>;
  const int tin = threadIdx.x & (tpr - 1), mine = threadIdx.x / tpr, groups = kThreads / tpr;
  auto column = [&](int p) { return (p * tpr + tin) * kVec; };
  float dw[kPer][kVec];
#pragma unroll
  for (int p = 0; p < kPer; ++p)
#pragma unroll
    for (int i = 0; i < kVec; ++i) dw[p][i] = 0.f;
  const int64_t blocks = (a.rows + groups - 1) / groups;
  Ch h[kPer], dy[kPer], ds[kPer];
  float s = 0.f;
  auto fetch = [&](int64_t block) {
    const int64_t row = block * groups + mine;
    const bool in_rows = block < blocks && row < a.rows;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const bool in = in_rows && column(p) < a.C;
      const int64_t at = in ? row * a.C + column(p) : 0;
      h[p] = in ? Ch::load(static_cast<const T*>(a.x) + at) : Ch::zero();
      dy[p] = in ? Ch::load(static_cast<const T*>(a.dy) + at) : Ch::zero();
      ds[p] = in && a.dsum ? Ch::load(static_cast<const T*>(a.dsum) + at) : Ch::zero();
    }
    s = in_rows ? __ldg(a.rstd + row) : 0.f;
  };
  fetch(blockIdx.x);
  int turn = 0;
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    const int64_t row = block * groups + mine;
    Ch hc[kPer], gc[kPer], sc[kPer];
#pragma unroll
    for (int p = 0; p < kPer; ++p) { hc[p] = h[p]; gc[p] = dy[p]; sc[p] = ds[p]; }
    const float rstd = s;
    fetch(block + gridDim.x);
    float t = 0.f;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      float n[kVec], g[kVec], w[kVec];
      hc[p].get(n);
      gc[p].get(g);
      if (column(p) < a.C) {
        weights<W, kVec>(a.w, column(p), w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          n[i] *= rstd;
          dw[p][i] = fmaf(g[i], n[i], dw[p][i]);
          t = fmaf(g[i] * w[i], n[i], t);
        }
      }
    }
    const float mean = over_row<add>(t, tpr, red[turn]) * a.inv_c;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      if (row >= a.rows || column(p) >= a.C) continue;
      float n[kVec], g[kVec], w[kVec], d[kVec];
      hc[p].get(n);
      gc[p].get(g);
      sc[p].get(d);
      weights<W, kVec>(a.w, column(p), w);
#pragma unroll
      for (int i = 0; i < kVec; ++i) d[i] += rstd * (g[i] * w[i] - n[i] * rstd * mean);
      Ch::of(d).store(static_cast<T*>(a.dx) + row * a.C + column(p));
    }
  }
  if (!a.part) return;
  if (groups > 1) {      // one group after the other, so that the sums have one order
    for (int g = 0; g < groups; ++g) {
      __syncthreads();
      if (mine == g) {
#pragma unroll
        for (int p = 0; p < kPer; ++p)
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (column(p) < a.C) columns[column(p) + i] = dw[p][i] + (g ? columns[column(p) + i] : 0.f);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += kThreads) a.part[int64_t(blockIdx.x) * a.C + c] = columns[c];
    return;
  }
#pragma unroll
  for (int p = 0; p < kPer; ++p)
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (column(p) < a.C) a.part[int64_t(blockIdx.x) * a.C + column(p) + i] = dw[p][i];
}

// dx of a row per CTA, read twice.
template <typename T, typename W, int kVec>
__global__ void __launch_bounds__(kThreads) rms_bwd_wide_kernel(const RmsArgs a) {
  __shared__ float red[kWarps];
  using Ch = Chunk<T, kVec>;
  const int64_t row = blockIdx.x, base = row * a.C;
  const float rstd = a.rstd[row];
  float t = 0.f;
  for (int c = threadIdx.x * kVec; c < a.C; c += kThreads * kVec) {
    float n[kVec], g[kVec], w[kVec];
    Ch::load_cached(static_cast<const T*>(a.x) + base + c).get(n);
    Ch::load_cached(static_cast<const T*>(a.dy) + base + c).get(g);
    weights<W, kVec>(a.w, c, w);
#pragma unroll
    for (int i = 0; i < kVec; ++i) t = fmaf(g[i] * w[i], n[i] * rstd, t);
  }
  const float mean = over_row<add>(t, kThreads, red) * a.inv_c;
  for (int c = threadIdx.x * kVec; c < a.C; c += kThreads * kVec) {
    float n[kVec], g[kVec], w[kVec], d[kVec];
    Ch::load_cached(static_cast<const T*>(a.x) + base + c).get(n);
    Ch::load_cached(static_cast<const T*>(a.dy) + base + c).get(g);
    weights<W, kVec>(a.w, c, w);
    if (a.dsum) Ch::load_cached(static_cast<const T*>(a.dsum) + base + c).get(d);
#pragma unroll
    for (int i = 0; i < kVec; ++i) d[i] = (a.dsum ? d[i] : 0.f) + rstd * (g[i] * w[i] - n[i] * rstd * mean);
    Ch::of(d).store(static_cast<T*>(a.dx) + base + c);
  }
}
// dw of wide rows: a thread has a column, a CTA row the rows of its part.
template <typename T>
__global__ void __launch_bounds__(kThreads) rms_dweight_wide_kernel(const RmsArgs a) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.C) return;
  const int64_t r0 = a.rows * blockIdx.y / gridDim.y, r1 = a.rows * (blockIdx.y + 1) / gridDim.y;
  float sum = 0.f;
  for (int64_t r = r0; r < r1; ++r)
    sum = fmaf(to_f32<T>(static_cast<const T*>(a.dy)[r * a.C + c]), to_f32<T>(static_cast<const T*>(a.x)[r * a.C + c]) * a.rstd[r], sum);
  a.part[int64_t(blockIdx.y) * a.C + c] = sum;
}

// The sum of the partial rows, 32 columns per CTA, every 32nd row per warp, in one order.
template <typename W>
__global__ void __launch_bounds__(1024) rms_dweight_kernel(const float* part, int rows, int C, W* out) {
  __shared__ float sums[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (c < C)
    for (int r = threadIdx.y; r < rows; r += 32) sum += part[int64_t(r) * C + c];
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  float v = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < C) out[blockIdx.x * 32 + threadIdx.y] = from_f32<W>(v);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a row is divided.
struct Shape {
  bool vec;
  int tpr;       // threads of a row
  int per;       // chunks of a thread; 0: the row is too wide to be held
};
constexpr int kMostVec = 8, kMostScalar = 32;      // chunks of a thread

Shape shape_of(int C, int esz, bool vec) {
  Shape s{vec, 32, 0};
  const int chunks = vec ? C * esz / 16 : C, least = vec ? 2 : 4, most = vec ? kMostVec : kMostScalar;
  while (s.tpr < kThreads && s.tpr * least < chunks) s.tpr *= 2;
  for (int per = vec ? 1 : 4; per <= most; per *= 2)
    if (s.tpr * per >= chunks) { s.per = per; break; }
  return s;
}

int bwd_ctas(const Shape& s, int vec_elements) {      // resident per SM, as the launch bounds say
  const int elements = s.per * vec_elements;
  return elements <= 8 ? 4 : elements <= 16 ? 3 : elements <= 32 ? 2 : 1;
}

int check(const nb200_rms_norm_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_rms_norm_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  if (p->dtype != NB200_F32 && p->dtype != NB200_BF16 && p->dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (p->weight_dtype != p->dtype && p->weight_dtype != NB200_F32) { set_error("%s: the weight must be of the operands' dtype or fp32", what); return NB200_ERR_INVALID; }
  if (p->rows < 0 || p->channels <= 0) { set_error("%s: bad extents", what); return NB200_ERR_INVALID; }
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

// The backward's shape and the rows of partial sums that it leaves.
struct BwdPlan {
  Shape s;
  int parts;
};
BwdPlan bwd_plan(const nb200_rms_norm_params* p, bool vec) {
  const int esz = dtype_size(p->dtype);
  BwdPlan pl{shape_of(p->channels, esz, vec), 0};
  if (pl.s.per == 0) {
    pl.parts = int(p->rows < 64 ? p->rows : 64);
  } else {
    const int64_t blocks = (p->rows + kThreads / pl.s.tpr - 1) / (kThreads / pl.s.tpr);
    const int64_t most = int64_t(tc::sm_count()) * bwd_ctas(pl.s, vec ? 16 / esz : 1);
    pl.parts = int(blocks < most ? blocks : most);
  }
  return pl;
}

template <typename T, typename W, int kVec, bool kEight>
int launch_fwd(const RmsArgs& a, const Shape& s, cudaStream_t st) {
  const unsigned grid = unsigned((a.rows + kThreads / s.tpr - 1) / (kThreads / s.tpr));
  constexpr int k = kVec == 1 ? 4 : 1;
  if (s.per == 0) rms_fwd_wide_kernel<T, W, kVec, kEight><<<unsigned(a.rows), kThreads, 0, st>>>(a);
  else if (s.per == k) rms_fwd_kernel<T, W, kVec, k, kEight><<<grid, kThreads, 0, st>>>(a, s.tpr);
  else if (s.per == 2 * k) rms_fwd_kernel<T, W, kVec, 2 * k, kEight><<<grid, kThreads, 0, st>>>(a, s.tpr);
  else if (s.per == 4 * k) rms_fwd_kernel<T, W, kVec, 4 * k, kEight><<<grid, kThreads, 0, st>>>(a, s.tpr);
  else rms_fwd_kernel<T, W, kVec, 8 * k, kEight><<<grid, kThreads, 0, st>>>(a, s.tpr);
  count_launch();
  return check_launch("rms_fwd_kernel");
}
template <typename T, typename W>
int launch_fwd(const RmsArgs& a, const Shape& s, cudaStream_t st) {
  constexpr int kVec = 16 / int(sizeof(T));
  if (a.scales) return s.vec ? launch_fwd<T, W, kVec, true>(a, s, st) : launch_fwd<T, W, 1, true>(a, s, st);
  return s.vec ? launch_fwd<T, W, kVec, false>(a, s, st) : launch_fwd<T, W, 1, false>(a, s, st);
}

template <typename T, typename W, int kVec>
int launch_bwd(const RmsArgs& a, const BwdPlan& pl, cudaStream_t st) {
  const Shape& s = pl.s;
  constexpr int k = kVec == 1 ? 4 : 1;
  if (s.per == 0) {
    rms_bwd_wide_kernel<T, W, kVec><<<unsigned(a.rows), kThreads, 0, st>>>(a);
    count_launch();
    if (int rc = check_launch("rms_bwd_wide_kernel")) return rc;
    if (a.part) {
      rms_dweight_wide_kernel<T><<<dim3(unsigned((a.C + kThreads - 1) / kThreads), unsigned(pl.parts)), kThreads, 0, st>>>(a);
      count_launch();
      return check_launch("rms_dweight_wide_kernel");
    }
    return NB200_OK;
  }
  const size_t smem = s.tpr < kThreads && a.part ? size_t(a.C) * sizeof(float) : 0;
  if (s.per == k) rms_bwd_kernel<T, W, kVec, k><<<unsigned(pl.parts), kThreads, smem, st>>>(a, s.tpr);
  else if (s.per == 2 * k) rms_bwd_kernel<T, W, kVec, 2 * k><<<unsigned(pl.parts), kThreads, smem, st>>>(a, s.tpr);
  else if (s.per == 4 * k) rms_bwd_kernel<T, W, kVec, 4 * k><<<unsigned(pl.parts), kThreads, smem, st>>>(a, s.tpr);
  else rms_bwd_kernel<T, W, kVec, 8 * k><<<unsigned(pl.parts), kThreads, smem, st>>>(a, s.tpr);
  count_launch();
  return check_launch("rms_bwd_kernel");
}
template <typename T, typename W>
int launch_bwd(const RmsArgs& a, const BwdPlan& pl, void* dweight, cudaStream_t st) {
  constexpr int kVec = 16 / int(sizeof(T));
  if (int rc = pl.s.vec ? launch_bwd<T, W, kVec>(a, pl, st) : launch_bwd<T, W, 1>(a, pl, st)) return rc;
  if (!a.part) return NB200_OK;
  rms_dweight_kernel<W><<<unsigned((a.C + 31) / 32), dim3(32, 32), 0, st>>>(a.part, pl.parts, a.C, static_cast<W*>(dweight));
  count_launch();
  return check_launch("rms_dweight_kernel");
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_rms_norm_workspace_bytes(const nb200_rms_norm_params* p, size_t* bytes) {
  if (!bytes) { set_error("bytes out-pointer is NULL"); return NB200_ERR_INVALID; }
  if (int rc = check(p, "rms_norm_workspace_bytes")) return rc;
  *bytes = size_t(bwd_plan(p, vectors(p, true)).parts) * size_t(p->channels) * sizeof(float);
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
  a.eps = p->eps;
  a.inv_c = float(1.0 / p->channels);
  const Shape s = shape_of(p->channels, dtype_size(p->dtype), vec);
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
  const BwdPlan pl = bwd_plan(p, vectors(p, true));
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
