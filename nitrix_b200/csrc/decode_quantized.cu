// Attention of one new token per sequence over a paged cache in 4 or 8 bits, divided and joined as decode.cuh says.
//
//   s_t = scale q . k_t,  p = softmax(s),  out = sum_t p_t v_t,     k_t, v_t = step (code - 2^(b-1)) per group of 32 elements
//
// Every code and step is read once, 72 bytes per 128 elements in 4 bits, which HBM would deliver faster than the codes can be taken
// apart: 16 tokens of a head of 128 take a warp 322 instructions, 140 of them on the integer pipe at two cycles each, and the
// schedulers issue 0.6 per cycle with three or four warps each.
//
// 64 sequences of up to 8192 tokens (266 k in all), 8 key heads: bf16 4 bits, 4 x 128: 83 us, 3.7 TB/s; 8 bits, 5 x 64: 63, 4.6 TB/s; 4 of
// up to 131072 tokens, f16 4 bits, 8 x 128: 91, 4.1 TB/s.  32 such sequences in fp32, 4 bits, head dim 128, 1 / 2 / 4 / 8 query heads per
// key head: 102 / 124 / 183 / 337 us; bf16 52 with 1, 103 with 16.  On the way, for the first of these cases: fp32 units 792 us, MMAs with
// loads into registers 124, places as constants of a lane 102, the ring 98, two blocks a turn and beginnings counted 89.
#include <type_traits>

#include "cache_codes.cuh"
#include "decode.cuh"

namespace nb200 {
namespace {

struct QuantizedArgs : DecodeArgs {      // k, v: codes
  const uint16_t* k_steps;
  const uint16_t* v_steps;
  int kss[3], vss[3];      // head's rows of steps, over (page, head, slot)
  int groups;
};

// CTAs of an SM, which the loops' registers allow and the division of the work counts on.
constexpr int fma_ctas(int heads_by_groups) { return heads_by_groups <= 4 ? 4 : heads_by_groups <= 8 ? 3 : 2; }
// (head dim 128: three CTAs per SM without spills 97 us over long contexts, four with them 99, five 142)
constexpr int mma_ctas(int head_dim, int bits, int heads) { return heads == 8 ? (head_dim == 64 ? 4 : bits == 4 ? 3 : 2) : head_dim == 64 ? 3 : 2; }

__device__ __forceinline__ const uint16_t* steps_of(const uint16_t* base, const int (&stride)[3], int groups, int kv_head, Where w) {
  return base + (int64_t(w.page) * stride[0] + int64_t(kv_head) * stride[1] + int64_t(w.slot) * stride[2]) * groups;
}

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}

// fp32 multiply-adds, two per instruction.  Eight lanes share a token, a part of its row of codes each; a warp's four groups take tokens
// of their own, kAhead at a time: the next ones' codes are on their way while these are worked on.  The query heads' sums are scattered
// over the lanes as they are reduced, so that a lane has one head's scores.
//
// A code in the bits from p on of 2^23 is 2^23 + 2^p code, from which the offset comes off exactly; the queries have 2^-p, the output
// gets it at the end.
//
// kExact: the row has kGroups groups, so that a part's codes of all of them are one load; otherwise at most as many.
template <typename T, int kBits, int kGroups, bool kExact, int kNumHeads>
struct QuantizedFmaLoop {
  static constexpr const char* kName = "decode_kernel<quantized>";
  static constexpr int kRing = 0;
  static constexpr int kHeads = kNumHeads;
  static constexpr int kSlots = 4;
  static constexpr int kMinCtas = fma_ctas(kHeads * kGroups);
  static constexpr int kAhead = 2;
  static constexpr int kLanes = 8, kSteps = kHeads == 4 ? 2 : kHeads == 2 ? 1 : 0;      // of the reduce-scatter
  static constexpr int kWords = (kGroups * kBits + 7) / 8, kStepWords = (kGroups + 1) / 2;
  static constexpr float kHalf = float(1 << (kBits - 1));
  float2 o[kHeads][kGroups][2];
  float m, l;             // of this lane's head

  __device__ __forceinline__ static int my_head(int c) {   // the reduce-scatter's choices, high to low
    int h = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) h = 2 * h + ((c & (kLanes >> (s + 1))) ? 1 : 0);
    return h;
  }
  // the first lane (of a group) that holds head h
  __device__ __forceinline__ static int lane_of(int h) {
    int c = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (h & (kHeads >> (s + 1))) c += kLanes >> (s + 1);
    return c;
  }
  // 2^-p of element i of four: with 8 bits the upper two are shifted down
  __device__ __forceinline__ static float2 unit(int i) {
    return kBits == 4 ? (i ? make_float2(1.f / 256.f, 1.f / 4096.f) : make_float2(1.f, 1.f / 16.f)) : make_float2(1.f, 1.f / 256.f);
  }
  // four codes of group g, each times its 2^p
  __device__ __forceinline__ static void codes(const uint32_t (&w)[kWords], int g, float2 (&c)[2]) {
    const uint32_t part = kBits == 4 ? (g % 2 ? w[g / 2] >> 16 : w[g / 2]) : w[g];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = kBits == 8 && i ? part >> 16 : part;
      const int p0 = kBits == 4 ? 8 * i : 0, p1 = kBits == 4 ? 8 * i + 4 : 8;
      constexpr uint32_t mask = (1u << kBits) - 1u;
      c[i] = __fadd2_rn(make_float2(__uint_as_float(0x4b000000u | (x & mask << p0)), __uint_as_float(0x4b000000u | (x & mask << p1))),
                        make_float2(-8388608.f - kHalf * float(1 << p0), -8388608.f - kHalf * float(1 << p1)));
    }
  }
  __device__ __forceinline__ static float step_of(const uint32_t (&w)[kStepWords], int g) {
    return __half2float(__ushort_as_half(uint16_t(g % 2 ? w[g / 2] >> 16 : w[g / 2])));
  }
  __device__ __forceinline__ static void load(const QuantizedArgs& a, const uint8_t* row, const uint16_t* steps, int part, uint32_t (&w)[kWords], uint32_t (&s)[kStepWords]) {
    if constexpr (kExact) {
      load_words(w, row + part * kWords * 4);
      load_words(s, steps);
    } else {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const bool in = g < a.groups;
        const uint32_t step = in ? __ldg(steps + g) : 0;
        s[g / 2] = g % 2 ? s[g / 2] | step << 16 : step;
        if constexpr (kBits == 4) {
          const uint32_t c = in ? __ldg(reinterpret_cast<const uint16_t*>(row) + part * a.groups + g) : 0;
          w[g / 2] = g % 2 ? w[g / 2] | c << 16 : c;
        } else {
          w[g] = in ? __ldg(reinterpret_cast<const uint32_t*>(row) + part * a.groups + g) : 0;
        }
      }
    }
  }

  __device__ __forceinline__ void run(const QuantizedArgs& a, const int* row_table, int kv_head, const void* q_row, int heads, int t0, int t1,
                                      int wi, int wn) {
    const T* q = static_cast<const T*>(q_row);
    const int lane = threadIdx.x & 31, part = lane % kLanes;
    const int first = wi * kSlots, group = first + lane / kLanes, groups = wn * kSlots;
    float2 qf[kHeads][kGroups][2];
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const T* e = q + h * a.qs[1] + g * kGroup + part * 4;
        const bool in = h < heads && (kExact || g < a.groups);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          qf[h][g][i] = in ? __fmul2_rn(make_float2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1])), unit(i)) : make_float2(0.f, 0.f);
          o[h][g][i] = make_float2(0.f, 0.f);
        }
      }
    m = -INFINITY;
    l = 0.f;
    const uint4* kbase = a.k + int64_t(kv_head) * a.ks[1];
    const uint4* vbase = a.v + int64_t(kv_head) * a.vs[1];
    const int last = t1 - 1;
    uint32_t kw[kAhead][kWords], vw[kAhead][kWords], kt[kAhead][kStepWords], vt[kAhead][kStepWords];
    Where at[kAhead];       // of the tokens whose keys were asked for last
    // (behind the last token that one's rows are read again, with a probability of zero)
    auto load_k = [&](int b) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        at[j] = where(a, row_table, min(b + group + j * groups, last));
        load(a, reinterpret_cast<const uint8_t*>(row_of(kbase, a.ks, at[j])), steps_of(a.k_steps, a.kss, a.groups, kv_head, at[j]), part, kw[j], kt[j]);
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        load(a, reinterpret_cast<const uint8_t*>(row_of(vbase, a.vs, at[j])), steps_of(a.v_steps, a.vss, a.groups, kv_head, at[j]), part, vw[j], vt[j]);
    };
    // (every group of a warp makes as many turns as its first, which has the most: the shuffles below are warp-wide)
    int b = t0;
    if (b + first >= t1) return;
    load_k(b);
    load_v();
    for (; b + first < t1; b += groups * kAhead) {
      const int next = b + groups * kAhead;
      float x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float2 s2[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s2[h] = make_float2(0.f, 0.f);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float2 c[2];
          codes(kw[j], g, c);
          const float step = step_of(kt[j], g);
#pragma unroll
          for (int h = 0; h < kHeads; ++h)
            s2[h] = __ffma2_rn(__ffma2_rn(qf[h][g][1], c[1], __fmul2_rn(qf[h][g][0], c[0])), make_float2(step, step), s2[h]);
        }
        float s[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s[h] = s2[h].x + s2[h].y;
        // reduce-scatter: every step halves the heads that a lane still sums; then what is left of the lanes
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          const int off = kLanes >> (step + 1), n = kHeads >> (step + 1);
          const bool upper = (part & off) != 0;
#pragma unroll
          for (int h = 0; h < kHeads / 2; ++h) {
            if (h >= n) continue;
            const float keep = upper ? s[h + n] : s[h], send = upper ? s[h] : s[h + n];
            s[h] = keep + __shfl_xor_sync(0xffffffffu, send, off);
          }
        }
#pragma unroll
        for (int off = kLanes >> (kSteps + 1); off > 0; off >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
        x[j] = b + group + j * groups < t1 ? s[0] * a.mul : -INFINITY;
      }
      if (next + first < t1) load_k(next);
      float m_new = m;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) m_new = fmaxf(m_new, x[j]);
      const float shift = m_new == -INFINITY ? 0.f : m_new;
      if (__any_sync(0xffffffffu, m_new > m)) {
        const float alpha = ex2(m - shift);
        l *= alpha;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float ah = __shfl_sync(0xffffffffu, alpha, (lane & ~(kLanes - 1)) + lane_of(h));
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) o[h][g][i] = __fmul2_rn(o[h][g][i], make_float2(ah, ah));
        }
      }
      m = m_new;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float pr = ex2(x[j] - shift);
        l += pr;
        float ph[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) ph[h] = __shfl_sync(0xffffffffu, pr, (lane & ~(kLanes - 1)) + lane_of(h));
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float2 c[2];
          codes(vw[j], g, c);
          const float step = step_of(vt[j], g);
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            const float w = ph[h] * step;
#pragma unroll
            for (int i = 0; i < 2; ++i) o[h][g][i] = __ffma2_rn(make_float2(w, w), c[i], o[h][g][i]);
          }
        }
      }
      if (next + first < t1) load_v();
    }
  }

  __device__ __forceinline__ void store(const QuantizedArgs& a, float* dst) const {
    const int part = threadIdx.x % kLanes;
    float* slot = dst + threadIdx.x / kLanes * kHeads * (a.D + 2);
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (kExact || g < a.groups)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<float2*>(slot + h * (a.D + 2) + g * kGroup + part * 4 + 2 * i) = __fmul2_rn(o[h][g][i], unit(i));
    if ((part & ((kLanes >> kSteps) - 1)) == 0) {
      float* row = slot + my_head(part) * (a.D + 2);
      row[a.D] = m;
      row[a.D + 1] = l;
    }
  }
};

// 16-bit queries, head dim 64 or 128: warp-level MMAs.  Tokens are the M side of the scores (S^T = K Q^T), elements that of the output
// (O^T = V^T P^T), as in decode.cu.
//
// Codes become operands without a conversion: the bits of a whole number below 1024 in an fp16 are that number times 2^-24, so a
// mask of a word that holds codes of two operands' halves gives both (in 4 bits every other element's code stands four bits up,
// which is times 16: the queries have 1/16 there, the output's rows get it at the end).  Queries are fp16, by a power of two per head
// that brings the largest to 2^9 .. 2^10: fp16's bits are all kept down to 2^-23 of it, bf16's to 2^-26 (with the 1/16 to 2^-19 and 2^-22),
// and smaller elements are off by 2^-34 (2^-30) of it.
// Steps: those of a key's groups multiply the groups' sums, fp32, of which the half of the codes' range has been taken off
// beforehand (the accumulators begin with it); those of a value's groups multiply its probability before that is rounded to fp16,
// once, for each group.  The reference maximum is that of score + log2 of the value's largest step, so that no product leaves
// fp16 and those of small steps keep their bits: a token's largest is at 2^7 .. 2^15 at the reference, so that a rounding is 2^-11 of the
// product or 2^-32 of the largest one; the sum of the probabilities is fp32.  Values' codes lose the half of
// their range before the product, two at a time: taken off the sums instead, by MMAs of their own, it leaves errors of 2^-18 of it.
//
// A warp takes two blocks of 16 tokens at a turn, which come through a ring in shared memory by asynchronous copies, the next turn's
// while it works on this one: of pages of 16, 32, ... slots that lie side by side (kDense) as they are, of others row by row.
template <typename T, int D, int kBits, int kTiles, bool kDense>
struct QuantizedMmaLoop {
  static constexpr const char* kName = "decode_kernel<quantized>";
  static constexpr int kHeads = 8 * kTiles;
  static constexpr int kBlock = 16, kTurn = 32;  // tokens
  static constexpr int kSlots = 1;
  static constexpr int kMinCtas = mma_ctas(D, kBits, kHeads);
  static constexpr int kG = D / kGroup;          // groups
  static constexpr int kW = kG * kBits / 8;      // words of a part of a row of codes
  static constexpr int kRow = D * kBits / 8;     // bytes of a row of codes
  // a stage: rows of codes of keys, of values, rows of steps of keys, of values
  static constexpr int kStages = 2;
  static constexpr int kValuesAt = kTurn * kRow, kStepsAt = 2 * kTurn * kRow, kValueStepsAt = kStepsAt + kTurn * 2 * kG;
  static constexpr int kStage = kStepsAt + kTurn * 4 * kG;
  static constexpr int kRing = kStages * kStage;
  static constexpr float kUp = 7.f;              // log2 of what probabilities are kept at: their products are below 2^15
  static constexpr float kLag = 8.f;             // log2 of how far a token may pass the reference
  float o[kTiles][D / 16][4];
  float m[kTiles][2];                            // reference maxima, and kLag
  float2 l[kTiles];

  template <int n>
  __device__ __forceinline__ static void load_words(uint32_t (&w)[n], const char* p) {
    if constexpr (n == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (n == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < n / 4; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    }
  }
  // Elements 0 .. 3 of group i of two parts (or of two tokens' same part), as halves of four words.
  __device__ __forceinline__ static void codes(uint32_t (&e)[4], const uint32_t* a, const uint32_t* b, int i) {
    if constexpr (kBits == 4) {
      const uint32_t x = __byte_perm(a[i / 2], b[i / 2], i % 2 ? 0x7632 : 0x5410), y = x >> 8;
      e[0] = x & 0x000f000fu; e[1] = x & 0x00f000f0u; e[2] = y & 0x000f000fu; e[3] = y & 0x00f000f0u;
    } else {
      const uint32_t x = __byte_perm(a[i], b[i], 0x5410), y = __byte_perm(a[i], b[i], 0x7632);
      e[0] = x & 0x00ff00ffu; e[1] = x >> 8 & 0x00ff00ffu; e[2] = y & 0x00ff00ffu; e[3] = y >> 8 & 0x00ff00ffu;
    }
  }
  // minus the half of the range, for even and odd elements
  static constexpr uint32_t kEven = kBits == 4 ? 0x80088008u : 0x80808080u, kOdd = 0x80808080u;
  __device__ __forceinline__ static uint32_t plus(uint32_t a, uint32_t b) {
    uint32_t c;
    asm("add.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
  }
  // d = c + A B
  __device__ __forceinline__ static void mma(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
  __device__ __forceinline__ static float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  // step of group i
  __device__ __forceinline__ static float step(const uint32_t (&w)[kG / 2], int i) { return i % 2 ? halves(w[i / 2]).y : halves(w[i / 2]).x; }

  __device__ __forceinline__ void run(const QuantizedArgs& a, const int* row_table, int kv_head, const void* q_row, int heads, int t0, int t1,
                                      int wi, int wn, char* ring) {
    const T* q = static_cast<const T*>(q_row);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t qf[kTiles][kG][4];
    float mul[kTiles][2], half[kTiles][kG][4];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float x[kG][8], top = 0.f;
#pragma unroll
      for (int i = 0; i < kG; ++i) {
        const uint4 w = n * 8 + g < heads ? *reinterpret_cast<const uint4*>(q + (n * 8 + g) * a.qs[1] + i * kGroup + t * 8) : make_uint4(0, 0, 0, 0);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[i][j] = to_f32<T>(e[j]);
          top = fmaxf(top, fabsf(x[i][j]));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int size = min(max(int(__float_as_uint(top) >> 23) - 127, -100), 100);
      const float up = __uint_as_float(uint32_t(127 + 9 - size) << 23), down = __uint_as_float(uint32_t(127 + 15 + size) << 23) * a.mul;
      mul[n][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      mul[n][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
      for (int i = 0; i < kG; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = kBits == 4 && e % 2 ? up * (1.f / 16.f) : up;
          qf[n][i][e] = pack2<false>(x[i][e] * f, x[i][4 + e] * f);
        }
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        mma(half[n][i], zero, kEven, kEven, kOdd, kOdd, qf[n][i][0], qf[n][i][1]);
        mma(half[n][i], half[n][i], kEven, kEven, kOdd, kOdd, qf[n][i][2], qf[n][i][3]);
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n] = make_float2(0.f, 0.f);
    }
    const int last = t1 - 1;
    // Row r of a product's 16 is token `token_of(r)` of the block: with this order the rows that a lane's neighbours read side by side
    // lie in different banks.
    auto token_of = [](int r) { return (r & 8) + ((r & 1) ? 4 + ((r >> 1 & 3) ^ 1) : r >> 1 & 3); };
    const int mine = token_of(g);      // and mine + 8: this lane's tokens of the scores; t, 4 + (t ^ 1) and these + 8 are those of the values
    const uint32_t to = uint32_t(__cvta_generic_to_shared(ring)) + lane * 16;
    const uint4* k_from = a.k + int64_t(kv_head) * a.ks[1] + (kDense ? lane : 0);
    const uint4* v_from = a.v + int64_t(kv_head) * a.vs[1] + (kDense ? lane : 0);
    const char* steps_from = reinterpret_cast<const char*>(lane < 16 ? steps_of(a.k_steps, a.kss, kG, kv_head, Where{0, 0})
                                                                    : steps_of(a.v_steps, a.vss, kG, kv_head, Where{0, 0})) + (kDense ? (lane & 15) * 16 : 0);
    // (kDense: a page's steps are whole 16-byte words, as are 16 tokens')
    const int page_words = a.kss[0] * kG / 8, page_mask = a.page_size - 1;
    const bool has_steps = (lane & 15) < 2 * kG;
    auto page_of = [&](int b) { return kDense ? page_at(a, row_table, min(b, last) >> a.page_shift) : 0; };
    // block u of the turn at b; behind the last token what stands in its page, or that token's rows again
    auto fetch = [&](int b, int u, int page, uint32_t dst) {
      if constexpr (kDense) {
        const int slot = b & page_mask;
        const int64_t at = int64_t(page) * a.ks[0] + slot * (kRow / 16), steps = int64_t(page) * page_words + (slot * kG >> 3);
#pragma unroll
        for (int i = 0; i < kRow / 32; ++i) copy_async<16>(dst + u * kBlock * kRow + i * 512, k_from + at + i * 32);
#pragma unroll
        for (int i = 0; i < kRow / 32; ++i) copy_async<16>(dst + kValuesAt + u * kBlock * kRow + i * 512, v_from + at + i * 32);
        if (has_steps) copy_async<16>(dst + kStepsAt + u * kBlock * 2 * kG + (lane < 16 ? 0 : kTurn * 2 * kG - 256), reinterpret_cast<const uint4*>(steps_from) + steps);
      } else {
#pragma unroll
        for (int i = 0; i < kRow / 32; ++i) {
          const int at = lane * 16 + i * 512;
          const Where w = where(a, row_table, min(b + at / kRow, last));
          const int64_t k_row = int64_t(w.page) * a.ks[0] + int64_t(w.slot) * a.ks[2], v_row = int64_t(w.page) * a.vs[0] + int64_t(w.slot) * a.vs[2];
          copy_async<16>(dst + u * kBlock * kRow + i * 512, k_from + k_row + at % kRow / 16);
          copy_async<16>(dst + kValuesAt + u * kBlock * kRow + i * 512, v_from + v_row + at % kRow / 16);
        }
        const Where w = where(a, row_table, min(b + (lane & 15), last));
        const int64_t row = lane < 16 ? int64_t(w.page) * a.kss[0] + int64_t(w.slot) * a.kss[2] : int64_t(w.page) * a.vss[0] + int64_t(w.slot) * a.vss[2];
        copy_async<2 * kG>(dst - lane * 16 + (lane < 16 ? kStepsAt : kValueStepsAt) + (u * kBlock + (lane & 15)) * 2 * kG, steps_from + row * (2 * kG));
      }
    };
    int page[2];
    auto fetch_turn = [&](int b, int stage) {
      const uint32_t dst = to + stage * kStage;
      if (b < t1) {
        fetch(b, 0, page[0], dst);
        fetch(b + kBlock, 1, page[1], dst);      // (of which there may be nothing: then another block's rows, for no one)
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // One turn; kTail: the last of the tokens, of which it may hold any number.
    auto turn = [&](int b0, const char* at, auto tail) {
      constexpr bool kTail = decltype(tail)::value;
      float s[2][kTiles][4];      // of rows g, g + 8: heads 2t, 2t + 1
      uint32_t vt[2][2][kG / 2];
      float log_step[2][2];       // log2 of the largest step of the values of rows g, g + 8
      bool in[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t kw[2][2 * kW], kt[2][kG / 2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = u * kBlock + mine + 8 * r;
          load_words(kw[r], at + row * kRow + t * 8 * kW);
          load_words(kt[r], at + kStepsAt + row * 2 * kG);
          load_words(vt[u][r], at + kValueStepsAt + row * 2 * kG);
          in[u][r] = !kTail || b0 + row < t1;
          if (kTail && !in[u][r])
#pragma unroll
            for (int i = 0; i < kG / 2; ++i) kt[r][i] = vt[u][r][i] = 0;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < kG; ++i) top = fmaxf(top, fabsf(step(vt[u][r], i)));
          log_step[u][r] = in[u][r] ? fmaxf(__log2f(top), -24.f) : -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][n][j] = 0.f;
#pragma unroll
        for (int i = 0; i < kG; ++i) {
          uint32_t e0[4], e1[4];
          codes(e0, kw[0], kw[0] + kW, i);
          codes(e1, kw[1], kw[1] + kW, i);
          const float k0 = step(kt[0], i), k1 = step(kt[1], i);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            float c[4];
            mma(c, half[n][i], e0[0], e1[0], e0[1], e1[1], qf[n][i][0], qf[n][i][1]);
            mma(c, c, e0[2], e1[2], e0[3], e1[3], qf[n][i][2], qf[n][i][3]);
            s[u][n][0] = fmaf(k0, c[0], s[u][n][0]);
            s[u][n][1] = fmaf(k0, c[1], s[u][n][1]);
            s[u][n][2] = fmaf(k1, c[2], s[u][n][2]);
            s[u][n][3] = fmaf(k1, c[3], s[u][n][3]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        // The reference maximum moves only when a token passes it by more than 2^kLag.
        float most[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          most[j] = fmaxf(fmaxf(fmaf(s[0][n][j], mul[n][j], log_step[0][0]), fmaf(s[0][n][2 + j], mul[n][j], log_step[0][1])),
                          fmaxf(fmaf(s[1][n][j], mul[n][j], log_step[1][0]), fmaf(s[1][n][2 + j], mul[n][j], log_step[1][1])));
        if (__any_sync(0xffffffffu, most[0] > m[n][0] || most[1] > m[n][1])) {
          float c[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) most[j] = fmaxf(most[j], __shfl_xor_sync(0xffffffffu, most[j], off));
            const float to = fmaxf(most[j] + kLag, m[n][j]);
            c[j] = to > m[n][j] ? ex2(m[n][j] - to) : 1.f;
            m[n][j] = to;
          }
          l[n].x *= c[0];
          l[n].y *= c[1];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[n][i][0] *= c[0]; o[n][i][1] *= c[1]; o[n][i][2] *= c[0]; o[n][i][3] *= c[1];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (kTail && u == 1 && b0 + kBlock >= t1) break;
        uint32_t vw[4][kW], pt[kTiles][kG][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) load_words(vw[r], at + kValuesAt + (u * kBlock + (r & 1 ? 4 + (t ^ 1) : t) + (r >> 1) * 8) * kRow + g * 4 * kW);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float up = m[n][j & 1] == -INFINITY ? kUp : kUp + kLag - m[n][j & 1];
            p[j] = in[u][j >> 1] ? ex2(fmaf(s[u][n][j], mul[n][j & 1], up)) : 0.f;
          }
          l[n].x += p[0] + p[2];
          l[n].y += p[1] + p[3];
#pragma unroll
          for (int i = 0; i < kG; ++i) {
            const float v0 = step(vt[u][0], i), v1 = step(vt[u][1], i);
            pt[n][i][0] = transpose8x8(pack2<false>(p[0] * v0, p[1] * v0));
            pt[n][i][1] = transpose8x8(pack2<false>(p[2] * v1, p[3] * v1));
          }
        }
#pragma unroll
        for (int i = 0; i < kG; ++i) {
          uint32_t e0[4], e1[4];      // of rows 2t, 2t + 1 and 2t + 8, 2t + 9
          codes(e0, vw[0], vw[1], i);
          codes(e1, vw[2], vw[3], i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            e0[e] = plus(e0[e], e % 2 ? kOdd : kEven);
            e1[e] = plus(e1[e], e % 2 ? kOdd : kEven);
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            mma(o[n][2 * i], o[n][2 * i], e0[0], e0[1], e1[0], e1[1], pt[n][i][0], pt[n][i][1]);
            mma(o[n][2 * i + 1], o[n][2 * i + 1], e0[2], e0[3], e1[2], e1[3], pt[n][i][0], pt[n][i][1]);
          }
        }
      }
    };
    int b0 = t0 + wi * kTurn;
    if (b0 >= t1) return;
    const int stride = wn * kTurn;
    auto pages = [&](int b) { page[0] = page_of(b); page[1] = page_of(b + kBlock); };
    pages(b0);
    fetch_turn(b0, 0);
    pages(b0 + stride);
    int stage = 0;
    for (; b0 < t1; b0 += stride) {
      __syncwarp();      // all have left the turn before, whose stage the next copies take
      fetch_turn(b0 + stride, stage ^ 1);
      pages(b0 + 2 * stride);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      const char* at = ring + stage * kStage;
      stage ^= 1;
      if (b0 + kTurn <= t1) turn(b0, at, std::false_type{});
      else turn(b0, at, std::true_type{});
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[n].x += __shfl_xor_sync(0xffffffffu, l[n].x, off);
        l[n].y += __shfl_xor_sync(0xffffffffu, l[n].y, off);
      }
  }

  __device__ __forceinline__ void store(const QuantizedArgs& a, float* dst) const {
    constexpr float kScale = 16777216.f, kOddScale = kBits == 4 ? kScale / 16.f : kScale;      // of codes as fp16
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    static_assert(kRing >= kHeads * (D + 2) * int(sizeof(float)), "a warp's results lie in its ring");
    float* slot = dst + (threadIdx.x >> 5) * (kRing / 4);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float* row = slot + (n * 8 + 2 * t + hh) * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float2*>(row + (i / 2) * kGroup + 4 * g + 2 * (i & 1)) = make_float2(o[n][i][hh] * kScale, o[n][i][2 + hh] * kOddScale);
        if (g == 0) {
          row[D] = m[n][hh] == -INFINITY ? -INFINITY : m[n][hh] - kLag - kUp;
          row[D + 1] = hh ? l[n].y : l[n].x;
        }
      }
  }
};

struct Plan {
  bool mma;
  int heads, side, chunks;      // query heads of a chunk, chunks side by side, times that a group is taken
  int unit, extra, workers;
  size_t bytes;
};

int check(const nb200_decode_quantized_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_decode_quantized_params) || p->decode.struct_size != sizeof(nb200_decode_params)) {
    set_error("%s: NULL params or wrong struct_size", what);
    return NB200_ERR_INVALID;
  }
  const nb200_decode_params& d = p->decode;
  const nb200_cache_pages& c = d.pages;
  if (c.dtype != NB200_F32 && c.dtype != NB200_BF16 && c.dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (c.pages < 0 || c.heads <= 0 || c.page_size <= 0 || c.head_dim <= 0 || d.rows < 0 || d.width < 0 || d.q_heads <= 0) {
    set_error("%s: bad extents", what);
    return NB200_ERR_INVALID;
  }
  if (d.q_heads % c.heads) { set_error("%s: %d query heads are no multiple of %d key heads", what, d.q_heads, c.heads); return NB200_ERR_INVALID; }
  if (c.head_dim > 256) { set_error("%s: head dim %d is more than 256", what, c.head_dim); return NB200_ERR_UNSUPPORTED; }
  if (d.rows > 65535) { set_error("%s: %d sequences, at most 65535", what, d.rows); return NB200_ERR_UNSUPPORTED; }
  return check_steps(c, p->steps, what);
}

// groups of the fp32 loops that take a head dim
int groups_of(int head_dim) { return head_dim == 64 ? 2 : head_dim <= 128 ? 4 : 8; }

Plan plan(const nb200_decode_params* p, int bits) {
  const nb200_cache_pages& c = p->pages;
  Plan pl{};
  const int group = p->q_heads / c.heads;
  bool q_words = aligned16(p->q);
  for (int i = 0; i < 2; ++i) q_words = q_words && p->q_stride[i] % 8 == 0;
  pl.mma = c.dtype != NB200_F32 && (c.head_dim == 64 || c.head_dim == 128) && q_words;
  int ctas;
  if (pl.mma) {
    pl.heads = group > 8 ? 16 : 8;
    ctas = mma_ctas(c.head_dim, bits, pl.heads);
  } else {
    const int most = c.head_dim > 128 ? 2 : 4;
    pl.heads = group >= most ? most : group == 3 ? 4 : group;
    ctas = fma_ctas(pl.heads * groups_of(c.head_dim));
  }
  const int chunks = (group + pl.heads - 1) / pl.heads;
  pl.side = chunks == 1 ? 1 : chunks == 2 ? 2 : 4;
  pl.chunks = (chunks + pl.side - 1) / pl.side;
  pl.unit = 64;
  const int64_t units = (int64_t(p->width) * c.page_size + pl.unit - 1) / pl.unit * p->rows * c.heads * pl.chunks;
  const int64_t most = int64_t(tc::sm_count()) * ctas;
  pl.workers = int(units < most ? (units > 0 ? units : 1) : most);
  // Beginning with a (sequence, key head) costs a CTA about as much as two units: the queries, the first page, the join of its warps (64
  // sequences of up to 8192 tokens, 8 heads of 128, 4 bits: none 103 to 107 us, one 93 to 99, two 89 to 94).  Where every unit has a CTA
  // of its own there is nothing to balance.
  pl.extra = units < most ? 0 : 2;
  pl.bytes = size_t(pl.workers) * 2 * pl.side * pl.heads * (c.head_dim + 4) * sizeof(float);
  return pl;
}

template <typename T, int kBits, int kGroups, bool kExact>
int launch_fma(const QuantizedArgs& a, int heads, int side, cudaStream_t st) {
  if (heads == 1) return launch<T, QuantizedFmaLoop<T, kBits, kGroups, kExact, 1>, true>(a, side, st);
  if constexpr (kGroups <= 4) {
    if (heads == 4) return launch<T, QuantizedFmaLoop<T, kBits, kGroups, kExact, 4>, false>(a, side, st);
    return launch<T, QuantizedFmaLoop<T, kBits, kGroups, kExact, 2>, true>(a, side, st);
  } else {
    return launch<T, QuantizedFmaLoop<T, kBits, kGroups, kExact, 2>, false>(a, side, st);
  }
}
template <typename T, int kBits>
int launch_fma(const QuantizedArgs& a, int heads, int side, cudaStream_t st) {
  if (a.groups == 2) return launch_fma<T, kBits, 2, true>(a, heads, side, st);
  if (a.groups == 4) return launch_fma<T, kBits, 4, true>(a, heads, side, st);
  if (a.groups < 4) return launch_fma<T, kBits, 4, false>(a, heads, side, st);
  if (a.groups == 8) return launch_fma<T, kBits, 8, true>(a, heads, side, st);
  return launch_fma<T, kBits, 8, false>(a, heads, side, st);
}

template <typename T, int D, int kBits, bool kDense>
int launch_mma(const QuantizedArgs& a, int heads, int side, cudaStream_t st) {
  return heads == 8 ? launch<T, QuantizedMmaLoop<T, D, kBits, 1, kDense>, true>(a, side, st) : launch<T, QuantizedMmaLoop<T, D, kBits, 2, kDense>, false>(a, side, st);
}
template <typename T, int kBits>
int launch_mma(const QuantizedArgs& a, int heads, int side, cudaStream_t st) {
  // (places within a page, and steps' pages, as 32-bit numbers of words)
  bool dense = a.page_shift >= 4 && a.page_shift <= 24 && a.ks[2] == a.D * kBits / 128 && a.kss[2] == 1;
  dense = dense && int64_t(a.kss[0]) * a.groups <= 0x7fffffff && int64_t(a.kss[0]) * a.groups >= -0x7fffffff;
  for (int i = 0; i < 3; ++i) dense = dense && a.ks[i] == a.vs[i] && a.kss[i] == a.vss[i];
  for (int i = 0; i < 2; ++i) dense = dense && int64_t(a.kss[i]) * a.groups % 8 == 0;      // (16-byte copies of steps)
  if (a.D == 64) return dense ? launch_mma<T, 64, kBits, true>(a, heads, side, st) : launch_mma<T, 64, kBits, false>(a, heads, side, st);
  return dense ? launch_mma<T, 128, kBits, true>(a, heads, side, st) : launch_mma<T, 128, kBits, false>(a, heads, side, st);
}

template <typename T>
int launch_16(const QuantizedArgs& a, const Plan& pl, bool four, cudaStream_t st) {
  if (pl.mma) return four ? launch_mma<T, 4>(a, pl.heads, pl.side, st) : launch_mma<T, 8>(a, pl.heads, pl.side, st);
  return four ? launch_fma<T, 4>(a, pl.heads, pl.side, st) : launch_fma<T, 8>(a, pl.heads, pl.side, st);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_decode_quantized_workspace_bytes(const nb200_decode_quantized_params* p, size_t* bytes) {
  if (!bytes) { set_error("bytes out-pointer is NULL"); return NB200_ERR_INVALID; }
  if (int rc = check(p, "decode_quantized_workspace_bytes")) return rc;
  *bytes = plan(&p->decode, p->steps.bits).bytes;
  return NB200_OK;
}

extern "C" NB200_API int nb200_decode_quantized(const nb200_decode_quantized_params* qp, void* cuda_stream) {
  const char* what = "decode_quantized";
  if (int rc = check(qp, what)) return rc;
  const nb200_decode_params* p = &qp->decode;
  if (p->rows == 0) return NB200_OK;
  const nb200_cache_pages& c = p->pages;
  if (!p->q || !p->out || !p->lengths || (p->width && !p->table) || (c.pages && (!c.k || !c.v))) { set_error("%s: NULL operand", what); return NB200_ERR_INVALID; }
  const int groups = c.head_dim / kGroup;
  bool ok = aligned16(c.k) && aligned16(c.v), near = true;
  auto fits = [&](int64_t stride) { near = near && stride <= 0x7fffffff && stride >= -0x7fffffff; return int(stride); };
  QuantizedArgs a{};
  for (int i = 0; i < 3; ++i) {
    ok = ok && c.k_stride[i] % 16 == 0 && c.v_stride[i] % 16 == 0;
    a.ks[i] = fits(c.k_stride[i] / 16);
    a.vs[i] = fits(c.v_stride[i] / 16);
    a.kss[i] = fits(qp->steps.k_stride[i] / groups);
    a.vss[i] = fits(qp->steps.v_stride[i] / groups);
  }
  if (!ok) { set_error("%s: the rows of the pages must begin on 16-byte boundaries", what); return NB200_ERR_ALIGNMENT; }
  if (!near) { set_error("%s: a stride of the pages is 2^31 words of 16 bytes, or rows of steps, or more", what); return NB200_ERR_UNSUPPORTED; }
  const Plan pl = plan(p, qp->steps.bits);
  if (!p->workspace || p->workspace_bytes < pl.bytes) {
    set_error("%s: workspace of %zu bytes needed (nb200_decode_quantized_workspace_bytes), %zu given", what, pl.bytes, p->workspace_bytes);
    return NB200_ERR_WORKSPACE;
  }
  if (!aligned16(p->workspace)) { set_error("%s: the workspace must begin on a 16-byte boundary", what); return NB200_ERR_ALIGNMENT; }
  a.k = static_cast<const uint4*>(c.k);
  a.v = static_cast<const uint4*>(c.v);
  a.k_steps = static_cast<const uint16_t*>(qp->steps.k);
  a.v_steps = static_cast<const uint16_t*>(qp->steps.v);
  a.groups = groups;
  a.pages = c.pages; a.kv_heads = c.heads; a.page_size = c.page_size; a.D = c.head_dim;
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page_size == 1 << s) a.page_shift = s;
  a.table = p->table; a.lengths = p->lengths; a.rows = p->rows;
  a.width = c.pages ? p->width : 0;      // (without pages every sequence is empty)
  a.q = p->q; a.qs[0] = p->q_stride[0]; a.qs[1] = p->q_stride[1];
  a.out = p->out;
  a.q_heads = p->q_heads; a.group = p->q_heads / c.heads;
  a.chunks = pl.chunks;
  a.mul = p->scale * kLog2e;
  a.unit = pl.unit;
  a.extra = pl.extra;
  a.part = static_cast<float*>(p->workspace);
  a.workers = pl.workers;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  const bool four = qp->steps.bits == 4;
  if (c.dtype == NB200_F32) return four ? launch_fma<float, 4>(a, pl.heads, pl.side, st) : launch_fma<float, 8>(a, pl.heads, pl.side, st);
  return c.dtype == NB200_BF16 ? launch_16<__nv_bfloat16>(a, pl, four, st) : launch_16<__half>(a, pl, four, st);
}
