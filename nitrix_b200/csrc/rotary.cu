// Rotary positions of one or several axes, applied to queries and keys by ONE launch; the gradient is the same kernel
// turning the other way.
//
//   (x1, x2) -> (x1 cos - x2 sin, x1 sin + x2 cos),   phase = position[token][axis of the pair] * frequency[pair]
//
// Bound by HBM: every element is read and written once, and a pair costs three multiply-adds.  The cosines and sines are
// the same for every head of a token, so a CTA takes all heads of its tokens and forms their table once, in shared memory.  The
// phase is formed with the rounding errors of its products, so that a position of 2^40 is as good as one of 1: as one product of
// two fp32 numbers it is off by 0.008 at position 131072.  16384 bf16 tokens, 16 + 16 heads of 128, forward and gradient: 96 to
// 100 us, 5.4 to 5.6 TB/s, with small CTAs and one row per thread in flight; 256 or 512 threads 101 and 108, two or four rows in flight 104 and
// 100, cosines and sines in registers of a thread that goes over the heads 115, loads that do not stay in L2 115.
#include <math.h>

#include <type_traits>

#include "nitrix_b200_rotary.h"
#include "sdpa_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxPairs = 128;      // head dim 256
// 1 / (2 pi) in two doubles
constexpr double kTurnHigh = 0.15915494309189535, kTurnLow = -9.839338337591243e-18;
// and in two fp32 numbers
constexpr float kTurnHigh32 = 0.15915494f, kTurnLow32 = float(kTurnHigh - double(kTurnHigh32));
constexpr float kFp32Positions = 16777216.f;

struct RotaryTensor {
  const void* x;
  void* y;
  int64_t xs[3];
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[2];
  const void* positions;
  const float* frequencies;
  int tokens, length;         // B * S, S
  int D, pairs, axes;
  int bound[NB200_ROTARY_MAX_AXES];   // pairs of the axes up to and with this one
  int position_dtype;
  int interleaved;
  float sign;                 // -1: the other way
  int tokens_per_cta;
  uint32_t heads_magic;       // ceil(2^32 / heads of both tensors): row of a CTA -> its token, exact below 2^16 (one head: not used)
};

// cos and sin of a pair's phase at a token.  position * frequency / (2 pi) is formed with the rounding errors of its products,
// less whole turns: in pairs of fp32 numbers below 2^24, where a position is one, in pairs of fp64 ones from there on (2^24 + 1
// rounds to 2^24).  (64-bit units are few: with them alone the training pass of 16384 tokens took 102 us at its best.)
template <typename T>
__device__ __forceinline__ float2 turn_of(const RotaryArgs& a, int token, int pair) {
  int axis = 0;
  while (axis + 1 < a.axes && pair >= a.bound[axis]) ++axis;
  const int64_t i = int64_t(token) * a.axes + axis;
  double exact = 0.0;
  float p;
  if (a.position_dtype == NB200_POS_I32) {
    const int32_t n = static_cast<const int32_t*>(a.positions)[i];
    p = float(n);
    if (fabsf(p) >= kFp32Positions) exact = double(n);
  } else if (a.position_dtype == NB200_POS_I64) {
    const int64_t n = static_cast<const int64_t*>(a.positions)[i];
    p = float(n);
    if (fabsf(p) >= kFp32Positions) exact = double(n);
  } else {
    p = static_cast<const float*>(a.positions)[i];
    if (fabsf(p) >= kFp32Positions) exact = double(p);
  }
  const float f = a.frequencies[pair];
  float part;      // of a turn
  if (fabsf(p) >= kFp32Positions) {
    const double phase = exact * f, phase_low = fma(exact, double(f), -phase);
    const double turns = phase * kTurnHigh, turns_low = fma(phase, kTurnHigh, -turns) + fma(phase, kTurnLow, phase_low * kTurnHigh);
    part = float((turns - rint(turns)) + turns_low);
  } else {
    const float step = f * kTurnHigh32, step_low = fmaf(f, kTurnLow32, fmaf(f, kTurnHigh32, -step));      // turns per position
    const float turns = p * step, turns_low = fmaf(p, step_low, fmaf(p, step, -turns));
    part = (turns - rintf(turns)) + turns_low;
  }
  float s, c;
  if constexpr (sizeof(T) == 4) {
    sincospif(2.f * part, &s, &c);
  } else {
    __sincosf(part * 6.283185307f, &s, &c);      // within 5e-7, a thousandth of the result's rounding
  }
  return make_float2(c, a.sign * s);
}

// One (token, head) row's word `c` (and, for split pairs, its partner P elements on) in registers.
template <typename T, bool kInterleaved>
struct Piece {
  static constexpr int kVec = 16 / int(sizeof(T));
  uint4 lo, hi;
  __device__ __forceinline__ void load(const T* x, int c, int pairs, bool rotated) {
    lo = *reinterpret_cast<const uint4*>(x + c * kVec);
    if (!kInterleaved && rotated) hi = *reinterpret_cast<const uint4*>(x + c * kVec + pairs);
  }
  __device__ __forceinline__ void turn(const float2* table, int c) {
    T* e = reinterpret_cast<T*>(&lo);
    if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) {
        const float2 cs = table[c * (kVec / 2) + i];
        const float x1 = to_f32<T>(e[2 * i]), x2 = to_f32<T>(e[2 * i + 1]);
        e[2 * i] = from_f32<T>(x1 * cs.x - x2 * cs.y);
        e[2 * i + 1] = from_f32<T>(x1 * cs.y + x2 * cs.x);
      }
    } else {
      T* f = reinterpret_cast<T*>(&hi);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float2 cs = table[c * kVec + i];
        const float x1 = to_f32<T>(e[i]), x2 = to_f32<T>(f[i]);
        e[i] = from_f32<T>(x1 * cs.x - x2 * cs.y);
        f[i] = from_f32<T>(x1 * cs.y + x2 * cs.x);
      }
    }
  }
  __device__ __forceinline__ void store(T* y, int c, int pairs, bool rotated) const {
    *reinterpret_cast<uint4*>(y + c * kVec) = lo;
    if (!kInterleaved && rotated) *reinterpret_cast<uint4*>(y + c * kVec + pairs) = hi;
  }
};

// kLanes threads (a power of two) share a (token, head) row; thread c takes rotated word c, threads behind those the words that
// pass unchanged.  A CTA takes all heads of its tokens, a row per group of threads at a time; the first are on their way while
// the tokens' table is formed.
template <typename T, bool kInterleaved, int kLanes>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  constexpr int kVec = 16 / int(sizeof(T)), kGroups = kThreads / kLanes;
  extern __shared__ float2 table[];     // [token of the CTA][pair]
  const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int token0 = blockIdx.x * a.tokens_per_cta;
  const int n_tokens = min(a.tokens_per_cta, a.tokens - token0);
  const int heads = a.t[0].heads + a.t[1].heads;
  const int rows = n_tokens * heads;
  const int words = kInterleaved ? 2 * a.pairs / kVec : a.pairs / kVec;      // rotated words (for split pairs: of the first halves)
  const int pass0 = 2 * a.pairs / kVec, passing = a.D / kVec - pass0;        // words that pass unchanged
  const bool rotated = c < words, takes = rotated || c - words < passing;
  const int word = rotated ? c : pass0 + c - words;

  Piece<T, kInterleaved> piece;
  T* y = nullptr;
  int token = 0;           // of the CTA
  auto load = [&](int row) {
    token = heads == 1 ? row : int(__umulhi(uint32_t(row), a.heads_magic));
    int head = row - token * heads;
    const int n = token0 + token;
    const bool second = head >= a.t[0].heads;
    const RotaryTensor& t = second ? a.t[1] : a.t[0];
    if (second) head -= a.t[0].heads;
    const int b = n / a.length, s = n - b * a.length;
    y = static_cast<T*>(t.y) + (int64_t(n) * t.heads + head) * a.D;
    piece.load(static_cast<const T*>(t.x) + (b * t.xs[0] + s * t.xs[1] + head * t.xs[2]), word, a.pairs, rotated);
  };
  if (group < rows && takes) load(group);
  for (int i = threadIdx.x; i < n_tokens * a.pairs; i += kThreads) {
    const int tl = i / a.pairs;
    table[i] = turn_of<T>(a, token0 + tl, i - tl * a.pairs);
  }
  __syncthreads();
  for (int row = group; row < rows && takes; row += kGroups) {
    if (row != group) load(row);
    if (rotated) piece.turn(table + token * a.pairs, word);
    piece.store(y, word, a.pairs, rotated);
  }
}

// Any head dim, alignment and stride: one thread per pair or passing element.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_generic_kernel(const RotaryArgs a) {
  extern __shared__ float2 table[];
  const int token = blockIdx.x;
  for (int i = threadIdx.x; i < a.pairs; i += kThreads) table[i] = turn_of<T>(a, token, i);
  __syncthreads();
  const int b = token / a.length, s = token - b * a.length;
  const int per_head = a.D - a.pairs;      // pairs, then passing elements
  const int heads = a.t[0].heads + a.t[1].heads;
  for (int i = threadIdx.x; i < heads * per_head; i += kThreads) {
    int head = i / per_head;
    const int e = i - head * per_head;
    const RotaryTensor& t = head < a.t[0].heads ? a.t[0] : a.t[1];
    if (head >= a.t[0].heads) head -= a.t[0].heads;
    const T* x = static_cast<const T*>(t.x) + (b * t.xs[0] + s * t.xs[1] + head * t.xs[2]);
    T* y = static_cast<T*>(t.y) + (int64_t(token) * t.heads + head) * a.D;
    if (e >= a.pairs) {
      y[a.pairs + e] = x[a.pairs + e];
      continue;
    }
    const int e1 = a.interleaved ? 2 * e : e, e2 = a.interleaved ? 2 * e + 1 : e + a.pairs;
    const float x1 = to_f32<T>(x[e1]), x2 = to_f32<T>(x[e2]);
    y[e1] = from_f32<T>(x1 * table[e].x - x2 * table[e].y);
    y[e2] = from_f32<T>(x1 * table[e].y + x2 * table[e].x);
  }
}

template <typename T, bool kInterleaved, int kLanes>
int launch_lanes(RotaryArgs a, cudaStream_t st) {
  const int heads = a.t[0].heads + a.t[1].heads;
  // Tokens of a CTA: as many as give every group a row, one where that leaves the GPU short of CTAs.
  int per = kThreads / kLanes / heads;
  per = per < 1 || a.tokens / per < 4 * 148 ? 1 : per;
  a.tokens_per_cta = per;
  a.heads_magic = uint32_t(((uint64_t(1) << 32) + uint32_t(heads) - 1) / uint32_t(heads));
  const unsigned grid = unsigned((a.tokens + per - 1) / per);
  rotary_kernel<T, kInterleaved, kLanes><<<grid, kThreads, sizeof(float2) * size_t(per) * a.pairs, st>>>(a);
  count_launch();
  return check_launch("rotary_kernel");
}

template <typename T>
int launch_typed(const RotaryArgs& a, bool words, cudaStream_t st) {
  if (!words) {
    rotary_generic_kernel<T><<<unsigned(a.tokens), kThreads, sizeof(float2) * size_t(a.pairs), st>>>(a);
    count_launch();
    return check_launch("rotary_generic_kernel");
  }
  constexpr int kVec = 16 / int(sizeof(T));
  const int lanes = a.D / kVec - (a.interleaved ? 0 : a.pairs / kVec);
  auto go = [&](auto interleaved) {
    constexpr bool kI = decltype(interleaved)::value;
    if (lanes <= 4) return launch_lanes<T, kI, 4>(a, st);
    if (lanes <= 8) return launch_lanes<T, kI, 8>(a, st);
    if (lanes <= 16) return launch_lanes<T, kI, 16>(a, st);
    if (lanes <= 32) return launch_lanes<T, kI, 32>(a, st);
    return launch_lanes<T, kI, 64>(a, st);
  };
  return a.interleaved ? go(std::true_type()) : go(std::false_type());
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace nb200

extern "C" NB200_API int nb200_rotary(const nb200_rotary_params* p, void* cuda_stream) {
  using namespace nb200;
  if (!p || p->struct_size != sizeof(nb200_rotary_params)) { set_error("rotary: NULL params or wrong struct_size"); return NB200_ERR_INVALID; }
  if (p->dtype != NB200_F32 && p->dtype != NB200_BF16 && p->dtype != NB200_F16) { set_error("rotary: bad dtype"); return NB200_ERR_INVALID; }
  if (p->position_dtype < NB200_POS_I32 || p->position_dtype > NB200_POS_F32) { set_error("rotary: bad position dtype"); return NB200_ERR_INVALID; }
  if (p->batch < 0 || p->length < 0 || p->q.heads < 0 || p->k.heads < 0 || p->head_dim <= 0) { set_error("rotary: bad extents"); return NB200_ERR_INVALID; }
  if (p->axes < 1 || p->axes > NB200_ROTARY_MAX_AXES) { set_error("rotary: %d axes, 1 to %d are supported", p->axes, NB200_ROTARY_MAX_AXES); return NB200_ERR_UNSUPPORTED; }
  RotaryArgs a{};
  int64_t pairs = 0;
  for (int i = 0; i < p->axes; ++i) {
    if (p->sections[i] < 0) { set_error("rotary: section %d has %d pairs", i, p->sections[i]); return NB200_ERR_INVALID; }
    pairs += p->sections[i];
    a.bound[i] = int(pairs > kMaxPairs ? kMaxPairs + 1 : pairs);
  }
  if (p->head_dim > 2 * kMaxPairs) { set_error("rotary: head dim %d, at most %d", p->head_dim, 2 * kMaxPairs); return NB200_ERR_UNSUPPORTED; }
  if (2 * pairs > p->head_dim) { set_error("rotary: %lld pairs do not fit head dim %d", (long long)pairs, p->head_dim); return NB200_ERR_INVALID; }
  const int64_t tokens = int64_t(p->batch) * p->length, heads = int64_t(p->q.heads) + p->k.heads;
  if (tokens == 0 || heads == 0) return NB200_OK;
  if (tokens > 0x7fffffff || heads > 16384) { set_error("rotary: too many tokens or heads"); return NB200_ERR_UNSUPPORTED; }
  if ((pairs && !p->frequencies) || !p->positions) { set_error("rotary: NULL positions or frequencies"); return NB200_ERR_INVALID; }
  const int vec = p->dtype == NB200_F32 ? 4 : 8;
  bool words = p->head_dim % vec == 0 && (p->interleaved ? 2 * pairs : pairs) % vec == 0;
  const nb200_rotary_tensor* in[2] = {&p->q, &p->k};
  for (int i = 0; i < 2; ++i) {
    if (in[i]->heads == 0) continue;
    if (!in[i]->x || !in[i]->y) { set_error("rotary: NULL tensor"); return NB200_ERR_INVALID; }
    words = words && aligned16(in[i]->x) && aligned16(in[i]->y);
    for (int s = 0; s < 3; ++s) words = words && in[i]->x_stride[s] % vec == 0;
    a.t[i] = RotaryTensor{in[i]->x, in[i]->y, {in[i]->x_stride[0], in[i]->x_stride[1], in[i]->x_stride[2]}, in[i]->heads};
  }
  a.positions = p->positions; a.frequencies = p->frequencies;
  a.tokens = int(tokens); a.length = p->length; a.D = p->head_dim; a.pairs = int(pairs); a.axes = p->axes;
  a.position_dtype = p->position_dtype; a.interleaved = p->interleaved != 0;
  a.sign = p->inverse ? -1.f : 1.f;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  switch (p->dtype) {
    case NB200_F32: return launch_typed<float>(a, words, st);
    case NB200_BF16: return launch_typed<__nv_bfloat16>(a, words, st);
    default: return launch_typed<__half>(a, words, st);
  }
}
