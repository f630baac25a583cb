// Attention of one new token per sequence over the paged cache, split over the sequences' lengths and joined.
//
//   s_t = scale q . k_t,  p = softmax(s),  out = sum_t p_t v_t       for every query head, t < length of its sequence
//
// Bound by HBM: every kept key and value is read once, by the CTA that serves all query heads of its key head, and with G
// query heads per key head a byte of the cache takes G multiply-adds.  The lengths are known on the device only, and the grid
// is the same whatever they are: the tokens of all (sequence, key head) items, in units, are dealt in equal contiguous shares
// to as many CTAs as the GPU holds, so that one long sequence, many short ones and any mix end together.  A CTA's share is a
// run of pieces of items; a piece that is a whole item is finished on the spot, one that is not leaves its maximum, sum and
// unnormalised output (fp32) in the workspace: at most two per CTA, the share's first and last.  decode_join_kernel adds up
// those pieces, in order; it is set up while the main kernel runs.
//
// Two inner loops:
//  * 16-bit operands, head dim 64 or 128: warp-level MMAs on operands that go from global memory straight into registers, no
//    shared memory and no barrier in the loop.  Keys are the M side (S^T = K Q^T, O^T = V^T P^T), so that up to 8 query heads
//    are one N = 8 tile and nothing is wasted on padding to 16.  The order of the head dim inside a product is free, so a
//    lane's 16-byte words of K serve as the fragments of two steps; V's fragments pair two keys of one element, which is one
//    byte permutation of words loaded from the two keys' rows.  P^T goes from accumulator to operand layout by movmatrix.
//    P is rounded to the operand type for the product with V; its sum is of the unrounded values, in fp32.
//  * anything else: fp32 multiply-adds, two per instruction, lanes along the head dim, a reduce-scatter of the query heads' sums.
// In both, the next tokens' keys are asked for as soon as the scores have used the last ones, their values after the output.
//
// 32 sequences, 400 MB of cache: bf16, head dim 128, 8 key heads with 1 / 4 / 8 query heads each 6.0 / 5.6 / 5.0 TB/s, 4 with 16
// each 4.3; f32 1 / 4 / 8 5.3 / 4.7 / 3.4.  bf16 of head dim 80, 96 and 256, four query heads per key head: 1.2, 1.4 and 1.9.  One key
// head with 128 query heads: 0.67.  Four sequences of up to 131072 tokens, f16, 8 x 8 heads of 128: 201 to 208 us, 6.4 to 6.7 TB/s
// (of reads alone, which may pass a copy's 6.56).
#include "decode.cuh"

namespace nb200 {
namespace {

// Part `wi` of `wn` of a piece, for one warp: blocks of 16 tokens wi, wi + wn, ... of [t0, t1) of a sequence.
template <int D, int kTiles, bool kBf16>
struct MmaLoop {
  static constexpr int kHeads = 8 * kTiles;      // query heads of a chunk
  static constexpr int kBlock = 16;              // tokens
  static constexpr const char* kName = "decode_kernel";
  static constexpr int kRing = 0;
  static constexpr int kSlots = 1;               // partial results of a warp
  // (head dim 128, one tile: four CTAs per SM spill, 5280 GB/s of cache, three 5675; 64: four 5510, five 5616)
  static constexpr int kMinCtas = kTiles == 1 ? (D == 64 ? 5 : 3) : D == 64 ? 4 : 2;
  float o[kTiles][D / 16][4];                    // O^T: lane (g, t): head 2t (+1), see store
  float m[kTiles][2], l[kTiles][2];              // of heads 2t, 2t + 1; l: this lane's keys

  __device__ __forceinline__ void run(const DecodeArgs& a, const int* row_table, int kv_head, const void* q_row, int heads,
                                      int t0, int t1, int wi, int wn) {
    const uint16_t* q = static_cast<const uint16_t*>(q_row);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint4* kbase = a.k + int64_t(kv_head) * a.ks[1];
    const uint4* vbase = a.v + int64_t(kv_head) * a.vs[1];
    uint4 qf[kTiles][D / 32];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        qf[n][i] = n * 8 + g < heads ? *reinterpret_cast<const uint4*>(q + (n * 8 + g) * a.qs[1] + (i * 4 + t) * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    const int last = t1 - 1;
    uint4 kf[2][D / 32], vf[4][D / 64];
    // Blocks begin at multiples of 16 tokens, so that a block lies in one page where pages are of 16, 32, ... slots: the page is
    // looked up once, a turn ahead.
    const bool one_page = a.page_shift >= 4;
    auto page_of_block = [&](int b) { return one_page && b < t1 ? page_at(a, row_table, b >> a.page_shift) : 0; };
    auto place = [&](int b, int page, int token) {
      token = min(token, last);
      if (one_page) return Where{page, (b & (a.page_size - 1)) + token - b};
      return where(a, row_table, token);
    };
    auto load_k = [&](int b, int page) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint4* row = row_of(kbase, a.ks, place(b, page, b + g + 8 * r));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) kf[r][i] = sm100::ldg_no_allocate(row + i * 4 + t);
      }
    };
    // (zeros behind the last token: another's value there would be multiplied by a probability of zero, which an infinity survives)
    auto load_v = [&](int b, int page) {
      if (b + kBlock <= t1) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint4* row = row_of(vbase, a.vs, place(b, page, b + 2 * t + (r & 1) + (r >> 1) * 8));
#pragma unroll
          for (int i = 0; i < D / 64; ++i) vf[r][i] = sm100::ldg_no_allocate(row + i * 8 + g);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = b + 2 * t + (r & 1) + (r >> 1) * 8;
          const uint4* row = row_of(vbase, a.vs, place(b, page, token));
#pragma unroll
          for (int i = 0; i < D / 64; ++i) vf[r][i] = token <= last ? sm100::ldg_no_allocate(row + i * 8 + g) : make_uint4(0, 0, 0, 0);
        }
      }
    };
    int b0 = t0 + wi * kBlock;
    if (b0 >= t1) return;
    int next_page = page_of_block(b0);
    load_k(b0, next_page);
    load_v(b0, next_page);
    next_page = page_of_block(b0 + wn * kBlock);
    const float thr = a.mul > 0.f ? 8.f / a.mul : INFINITY;
    for (; b0 < t1; b0 += wn * kBlock) {
      const int next = b0 + wn * kBlock;
      float s[kTiles][4];
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          mma16816<kBf16>(s[n], kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, qf[n][i].x, qf[n][i].y);
          mma16816<kBf16>(s[n], kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, qf[n][i].z, qf[n][i].w);
        }
      if (next < t1) load_k(next, next_page);      // (the keys are used: their registers take the next block's)
      uint32_t pt[kTiles][2];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        if (b0 + g >= t1) s[n][0] = s[n][1] = -INFINITY;
        if (b0 + g + 8 >= t1) s[n][2] = s[n][3] = -INFINITY;
        // The reference maximum moves only when a score passes it by more than 2^8 (p <= 256; sums and outputs are fp32).
        const float mx0 = fmaxf(s[n][0], s[n][2]), mx1 = fmaxf(s[n][1], s[n][3]);
        if (__any_sync(0xffffffffu, mx0 > m[n][0] + thr || mx1 > m[n][1] + thr)) {
          float x0 = mx0, x1 = mx1;
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
          }
          x0 = fmaxf(x0, m[n][0]);
          x1 = fmaxf(x1, m[n][1]);
          const float c0 = x0 > m[n][0] ? ex2((m[n][0] - x0) * a.mul) : 1.f, c1 = x1 > m[n][1] ? ex2((m[n][1] - x1) * a.mul) : 1.f;
          m[n][0] = x0;
          m[n][1] = x1;
          l[n][0] *= c0;
          l[n][1] *= c1;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[n][i][0] *= c0; o[n][i][1] *= c1; o[n][i][2] *= c0; o[n][i][3] *= c1;
          }
        }
        const float n0 = m[n][0] == -INFINITY ? 0.f : -m[n][0] * a.mul, n1 = m[n][1] == -INFINITY ? 0.f : -m[n][1] * a.mul;
        const float p0 = ex2(fmaf(s[n][0], a.mul, n0)), p1 = ex2(fmaf(s[n][1], a.mul, n1));
        const float p2 = ex2(fmaf(s[n][2], a.mul, n0)), p3 = ex2(fmaf(s[n][3], a.mul, n1));
        l[n][0] += p0 + p2;
        l[n][1] += p1 + p3;
        pt[n][0] = transpose8x8(pack2<kBf16>(p0, p1));
        pt[n][1] = transpose8x8(pack2<kBf16>(p2, p3));
      }
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint32_t* w[4] = {&vf[0][i].x, &vf[1][i].x, &vf[2][i].x, &vf[3][i].x};
#pragma unroll
        for (int e = 0; e < 4; ++e) {      // elements i * 64 + g * 8 + 2 e, + 1
          const uint32_t a0 = __byte_perm(w[0][e], w[1][e], 0x5410), a1 = __byte_perm(w[0][e], w[1][e], 0x7632);
          const uint32_t a2 = __byte_perm(w[2][e], w[3][e], 0x5410), a3 = __byte_perm(w[2][e], w[3][e], 0x7632);
#pragma unroll
          for (int n = 0; n < kTiles; ++n) mma16816<kBf16>(o[n][i * 4 + e], a0, a1, a2, a3, pt[n][0], pt[n][1]);
        }
      }
      if (next < t1) load_v(next, next_page);
      next_page = page_of_block(next + wn * kBlock);
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], off);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], off);
      }
  }

  // output, maximum (base 2) and sum of this warp's part: [head][D + 2] floats
  __device__ __forceinline__ void store(const DecodeArgs& a, float* dst) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float* slot = dst + (threadIdx.x >> 5) * kHeads * (D + 2);
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float* row = slot + (n * 8 + 2 * t + hh) * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float2*>(row + (i / 4) * 64 + g * 8 + 2 * (i & 3)) = make_float2(o[n][i][hh], o[n][i][2 + hh]);
        if (g == 0) {
          row[D] = m[n][hh] == -INFINITY ? -INFINITY : m[n][hh] * a.mul;
          row[D + 1] = l[n][hh];
        }
      }
  }
};

// ---- fp32 multiply-adds ----------------------------------------------------------------------------------------------------
// kLanes lanes share a token's row, kPer 16-byte words each.  A warp's 32 / kLanes groups take tokens of their own, kAhead at a
// time: the next ones' keys are on their way from the scores on, their values from the end of the output sums on.
template <typename T, int kLanes, int kPer, int kNumHeads>
struct FmaLoop {
  static constexpr int kHeads = kNumHeads;
  static constexpr int kVec = 16 / int(sizeof(T));
  static constexpr const char* kName = "decode_kernel";
  static constexpr int kRing = 0;
  static constexpr int kSlots = 32 / kLanes;
  static constexpr int kAhead = sizeof(T) == 4 && kPer == 1 ? 4 : 2;
  // (eight heads: two, three, four, five CTAs per SM 2730, 3330, 3030, 2470 GB/s)
  static constexpr int kMinCtas = sizeof(T) == 4 && kPer == 1 ? (kNumHeads == 8 ? 3 : 4) : 2;
  static constexpr int kSteps = kHeads == 8 ? 3 : kHeads == 4 ? 2 : kHeads == 2 ? 1 : 0;   // of the reduce-scatter
  float2 o[kHeads][kPer][kVec / 2];      // (pairs: two multiply-adds per instruction)
  float m, l;             // of the head that the reduce-scatter leaves in this lane

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

  __device__ __forceinline__ void run(const DecodeArgs& a, const int* row_table, int kv_head, const void* q_row, int heads, int t0,
                                      int t1, int wi, int wn) {
    const T* q = static_cast<const T*>(q_row);
    const int c = threadIdx.x % kLanes, lane = threadIdx.x & 31;
    const int first = wi * kSlots, group = first + lane / kLanes, groups = wn * kSlots;
    const int words = a.D / kVec;
    float2 qf[kHeads][kPer][kVec / 2];
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const bool in = h < heads && c + p * kLanes < words;
        const T* e = q + h * a.qs[1] + (c + p * kLanes) * kVec;
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          qf[h][p][i] = in ? make_float2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1])) : make_float2(0.f, 0.f);
          o[h][p][i] = make_float2(0.f, 0.f);
        }
      }
    m = -INFINITY;
    l = 0.f;
    const uint4* kbase = a.k + int64_t(kv_head) * a.ks[1];
    const uint4* vbase = a.v + int64_t(kv_head) * a.vs[1];
    const int last = t1 - 1;
    uint4 kw[kAhead][kPer], vw[kAhead][kPer];
    Where at[kAhead];       // of the tokens whose keys were asked for last
    auto load = [&](uint4 (&w)[kAhead][kPer], const uint4* base, const int (&stride)[3], auto wanted) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint4* row = row_of(base, stride, at[j]);
#pragma unroll
        for (int p = 0; p < kPer; ++p) w[j][p] = c + p * kLanes < words && wanted(j) ? __ldg(row + c + p * kLanes) : make_uint4(0, 0, 0, 0);
      }
    };
    auto load_k = [&](int b) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) at[j] = where(a, row_table, min(b + group + j * groups, last));
      load(kw, kbase, a.ks, [](int) { return true; });
    };
    // (zeros behind the last token: another's value there would be multiplied by a probability of zero, which an infinity survives)
    auto load_v = [&](int b) {
      load(vw, vbase, a.vs, [&](int j) { return b + group + j * groups <= last; });
    };
    // (every group of a warp makes as many turns as its first, which has the most: the shuffles below are warp-wide)
    int b = t0;
    if (b + first >= t1) return;
    load_k(b);
    load_v(b);
    for (; b + first < t1; b += groups * kAhead) {
      const int next = b + groups * kAhead;
      float x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float2 s2[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s2[h] = make_float2(0.f, 0.f);
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          const T* e = reinterpret_cast<const T*>(&kw[j][p]);
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) {
            const float2 x2 = make_float2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1]));
#pragma unroll
            for (int h = 0; h < kHeads; ++h) s2[h] = __ffma2_rn(qf[h][p][i], x2, s2[h]);
          }
        }
        float s[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s[h] = s2[h].x + s2[h].y;
        // reduce-scatter: every step halves the heads that a lane still sums; then what is left of the lanes
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          const int off = kLanes >> (step + 1), n = kHeads >> (step + 1);
          const bool upper = (c & off) != 0;
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
      const float alpha = ex2(m - shift);
      if (__any_sync(0xffffffffu, m_new > m)) {
        l *= alpha;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float ah = __shfl_sync(0xffffffffu, alpha, (lane & ~(kLanes - 1)) + lane_of(h));
#pragma unroll
          for (int p = 0; p < kPer; ++p)
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) o[h][p][i] = __fmul2_rn(o[h][p][i], make_float2(ah, ah));
        }
      }
      m = m_new;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float pr = ex2(x[j] - shift);
        l += pr;
        float2 ph[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          ph[h].x = __shfl_sync(0xffffffffu, pr, (lane & ~(kLanes - 1)) + lane_of(h));
          ph[h].y = ph[h].x;
        }
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          const T* e = reinterpret_cast<const T*>(&vw[j][p]);
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) {
            const float2 x2 = make_float2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1]));
#pragma unroll
            for (int h = 0; h < kHeads; ++h) o[h][p][i] = __ffma2_rn(ph[h], x2, o[h][p][i]);
          }
        }
      }
      if (next + first < t1) load_v(next);
    }
  }
  __device__ __forceinline__ void store(const DecodeArgs& a, float* dst) const {
    const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    float* slot = dst + group * kHeads * (a.D + 2);
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int p = 0; p < kPer; ++p)
        if (c + p * kLanes < a.D / kVec)
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) *reinterpret_cast<float2*>(slot + h * (a.D + 2) + (c + p * kLanes) * kVec + 2 * i) = o[h][p][i];
    if ((c & ((kLanes >> kSteps) - 1)) == 0) {
      float* row = slot + my_head(c) * (a.D + 2);
      row[a.D] = m;
      row[a.D + 1] = l;
    }
  }
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What a call runs as, which the size of its workspace depends on.
struct Plan {
  bool mma;
  int heads;       // query heads of a chunk
  int side, chunks;
  int unit, workers;
  size_t bytes;
};

int check(const nb200_decode_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_decode_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  const nb200_cache_pages& c = p->pages;
  if (c.dtype != NB200_F32 && c.dtype != NB200_BF16 && c.dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (c.pages < 0 || c.heads <= 0 || c.page_size <= 0 || c.head_dim <= 0 || p->rows < 0 || p->width < 0 || p->q_heads <= 0) {
    set_error("%s: bad extents", what);
    return NB200_ERR_INVALID;
  }
  if (p->q_heads % c.heads) { set_error("%s: %d query heads are no multiple of %d key heads", what, p->q_heads, c.heads); return NB200_ERR_INVALID; }
  const int vec = c.dtype == NB200_F32 ? 4 : 8;
  if (c.head_dim % vec || c.head_dim > 256) {
    set_error("%s: head dim %d must be a multiple of %d and at most 256", what, c.head_dim, vec);
    return NB200_ERR_UNSUPPORTED;
  }
  if (p->rows > 65535) { set_error("%s: %d sequences, at most 65535", what, p->rows); return NB200_ERR_UNSUPPORTED; }
  return NB200_OK;
}

Plan plan(const nb200_decode_params* p) {
  const nb200_cache_pages& c = p->pages;
  Plan pl{};
  const int group = p->q_heads / c.heads;
  bool q_words = aligned16(p->q);
  for (int i = 0; i < 2; ++i) q_words = q_words && p->q_stride[i] % 8 == 0;
  // (with a scale below 1e-30 the MMA loop's threshold, 8 / scale, comes near the end of fp32)
  pl.mma = c.dtype != NB200_F32 && (c.head_dim == 64 || c.head_dim == 128) && q_words && p->scale > 1e-30f;
  int ctas;      // resident per SM: the loops' kMinCtas
  if (pl.mma) {
    pl.heads = group > 8 ? 16 : 8;
    ctas = pl.heads == 8 ? (c.head_dim == 64 ? 5 : 3) : c.head_dim == 64 ? 4 : 2;
  } else if (c.dtype == NB200_F32) {
    pl.heads = group == 1 ? 1 : group == 2 ? 2 : group <= 4 ? 4 : 8;
    ctas = c.head_dim <= 128 ? (pl.heads == 8 ? 3 : 4) : 2;
  } else {
    pl.heads = 8;
    ctas = 2;
  }
  // A group of several chunks: warps side by side take them over the same tokens, which come from HBM once.
  const int chunks = (group + pl.heads - 1) / pl.heads;
  pl.side = chunks == 1 ? 1 : chunks == 2 ? 2 : 4;
  pl.chunks = (chunks + pl.side - 1) / pl.side;
  pl.unit = 64;
  const int64_t units = (int64_t(p->width) * c.page_size + pl.unit - 1) / pl.unit * p->rows * c.heads * pl.chunks;
  const int64_t most = int64_t(tc::sm_count()) * ctas;
  pl.workers = int(units < most ? (units > 0 ? units : 1) : most);
  pl.bytes = size_t(pl.workers) * 2 * pl.side * pl.heads * (c.head_dim + 4) * sizeof(float);
  return pl;
}

template <typename T, int kHeads>
int launch_fma(const DecodeArgs& a, int side, cudaStream_t st) {
  constexpr bool kWhole = kHeads < 8;
  const int words = a.D / (16 / int(sizeof(T)));
  if (words <= 8) return launch<T, FmaLoop<T, 8, 1, kHeads>, kWhole>(a, side, st);
  if (words <= 16) return launch<T, FmaLoop<T, 16, 1, kHeads>, kWhole>(a, side, st);
  if constexpr (sizeof(T) == 4) {
    if (words > 32) return launch<T, FmaLoop<T, 32, 2, kHeads>, kWhole>(a, side, st);
  }
  return launch<T, FmaLoop<T, 32, 1, kHeads>, kWhole>(a, side, st);      // (16-bit heads of 256 are 32 words)
}

int launch_f32(const DecodeArgs& a, int heads, int side, cudaStream_t st) {
  switch (heads) {
    case 1: return launch_fma<float, 1>(a, side, st);
    case 2: return launch_fma<float, 2>(a, side, st);
    case 4: return launch_fma<float, 4>(a, side, st);
    default: return launch_fma<float, 8>(a, side, st);
  }
}

template <typename T, bool kBf16>
int launch_mma(const DecodeArgs& a, int heads, int side, cudaStream_t st) {
  if (a.D == 64) return heads == 8 ? launch<T, MmaLoop<64, 1, kBf16>, true>(a, side, st) : launch<T, MmaLoop<64, 2, kBf16>, false>(a, side, st);
  return heads == 8 ? launch<T, MmaLoop<128, 1, kBf16>, true>(a, side, st) : launch<T, MmaLoop<128, 2, kBf16>, false>(a, side, st);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_decode_workspace_bytes(const nb200_decode_params* p, size_t* bytes) {
  if (!bytes) { set_error("bytes out-pointer is NULL"); return NB200_ERR_INVALID; }
  if (int rc = check(p, "decode_workspace_bytes")) return rc;
  *bytes = plan(p).bytes;
  return NB200_OK;
}

extern "C" NB200_API int nb200_decode(const nb200_decode_params* p, void* cuda_stream) {
  if (int rc = check(p, "decode")) return rc;
  if (p->rows == 0) return NB200_OK;
  const nb200_cache_pages& c = p->pages;
  if (!p->q || !p->out || !p->lengths || (p->width && !p->table) || (c.pages && (!c.k || !c.v))) { set_error("decode: NULL operand"); return NB200_ERR_INVALID; }
  const int vec = c.dtype == NB200_F32 ? 4 : 8;
  bool ok = aligned16(c.k) && aligned16(c.v), near = true;
  for (int i = 0; i < 3; ++i) {
    for (const int64_t stride : {c.k_stride[i], c.v_stride[i]}) {
      ok = ok && stride % vec == 0;
      near = near && stride / vec <= 0x7fffffff && stride / vec >= -0x7fffffff;
    }
  }
  if (!ok) { set_error("decode: the rows of the pages must begin on 16-byte boundaries"); return NB200_ERR_ALIGNMENT; }
  if (!near) { set_error("decode: a stride of the pages is 2^31 words of 16 bytes or more"); return NB200_ERR_UNSUPPORTED; }
  const Plan pl = plan(p);
  if (!p->workspace || p->workspace_bytes < pl.bytes) {
    set_error("decode: workspace of %zu bytes needed (nb200_decode_workspace_bytes), %zu given", pl.bytes, p->workspace_bytes);
    return NB200_ERR_WORKSPACE;
  }
  if (!aligned16(p->workspace)) { set_error("decode: the workspace must begin on a 16-byte boundary"); return NB200_ERR_ALIGNMENT; }
  DecodeArgs a{};
  a.k = static_cast<const uint4*>(c.k);
  a.v = static_cast<const uint4*>(c.v);
  for (int i = 0; i < 3; ++i) { a.ks[i] = int(c.k_stride[i] / vec); a.vs[i] = int(c.v_stride[i] / vec); }
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
  a.part = static_cast<float*>(p->workspace);
  a.workers = pl.workers;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  if (c.dtype == NB200_F32) return launch_f32(a, pl.heads, pl.side, st);
  if (c.dtype == NB200_BF16)
    return pl.mma ? launch_mma<__nv_bfloat16, true>(a, pl.heads, pl.side, st) : launch_fma<__nv_bfloat16, 8>(a, pl.side, st);
  return pl.mma ? launch_mma<__half, false>(a, pl.heads, pl.side, st) : launch_fma<__half, 8>(a, pl.side, st);
}
