// Attention over packed sequences on the fp32 units: every type, head dim up to 256, group size and stride, forward and
// backward, each sum in one order (no atomics).  The tensor-core kernels take what they cover; this is the rest,
// short fp32 sequences and the backward of fp32 operands of head dim 128 among it.
//
// The query heads of one key head are rows of the same matrix: row r of a sequence is query r / G, head r % G, so that a tile
// of rows reads its keys once for the whole group whatever G is, and dK and dV sum over the group by themselves.
//   forward   a tile of kT rows walks over key tiles with the running maximum and sum of a softmax
//   dq        the same walk with P = exp2(S - lse), dS = P (dO V^T - delta), dQ += dS K
//   dk, dv    a tile of kT keys walks over row tiles, dV += P^T dO, dK += dS^T Q
// Bound by the fp32 units: 256 threads as 16 x 16, each with a (kT / 16)-square piece of the scores and kT / 16 rows of the
// outputs in registers, operands in shared memory as fp32 with rows padded by four words (16-byte reads of 8 rows meet no bank
// twice), two multiply-adds per instruction.  Tiles are 64 rows up to head dim 128, and 32 above, where four operands of 64 rows
// would not fit.  fp32 rows of whole words are copied while the tile before is worked on.  f32, 2048 tokens, 16 heads on 4, head dim
// 128, causal: forward 516 us (33 TFLOP/s), dq 729, dk and dv 1060; both directions 2.36 ms.  bf16 takes a tenth longer: head dim 80 or
// 96 forward 572 to 598 us, both directions 2.5 to 2.6 ms; 256 2.2 and 8.3 ms.
#include <math.h>

#include <type_traits>

#include "packed.cuh"
#include "sm100_primitives.cuh"

namespace nb200 {
namespace packed {
namespace {

constexpr int kThreads = 256;

template <int kD>
struct Tile {
  static constexpr int kT = kD > 128 ? 32 : 64;
  static constexpr int kM = kT / 16;            // rows and score columns of a thread
  static constexpr int kStride = kD + 4;
  static constexpr int kCols = kD / 64;         // 16-byte pieces of an output row of a thread
  static constexpr int kPStride = kT + 4;
  static constexpr int kOperand = kT * kStride;
  static constexpr int kScores = kT * kPStride;
};

// Element offsets of a tile's rows, one thread per row: an index division per row, not per element.
template <int kT, typename Offset>
__device__ __forceinline__ void row_offsets(int64_t* dst, int n, Offset offset) {
  if (threadIdx.x < kT) dst[threadIdx.x] = int(threadIdx.x) < n ? offset(threadIdx.x) : 0;
}

// Rows `first` .. n - 1 of a tile from `offset(row)` elements on; zeros elsewhere.  kWords: rows of whole 16-byte words.
template <typename T, int kD, bool kWords, typename Offset>
__device__ __forceinline__ void load_tile(float* dst, const void* base, int n, int D, Offset offset, int first = 0) {
  using L = Tile<kD>;
  const T* x = static_cast<const T*>(base);
  if constexpr (kWords) {
    constexpr int kVec = 16 / int(sizeof(T)), kRow = kD / kVec;
#pragma unroll
    for (int i = threadIdx.x; i < L::kT * kRow; i += kThreads) {
      const int r = i / kRow, d = (i - r * kRow) * kVec;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (r >= first && r < n && d < D) w = *reinterpret_cast<const uint4*>(x + offset(r) + d);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int j = 0; j < kVec; j += 4)
        *reinterpret_cast<float4*>(dst + r * L::kStride + d + j) = make_float4(to_f32<T>(e[j]), to_f32<T>(e[j + 1]), to_f32<T>(e[j + 2]), to_f32<T>(e[j + 3]));
    }
  } else {
    for (int i = threadIdx.x; i < L::kT * kD; i += kThreads) {
      const int r = i / kD, d = i - r * kD;
      dst[r * L::kStride + d] = r >= first && r < n && d < D ? to_f32<T>(x[offset(r) + d]) : 0.f;
    }
  }
}

// The same for fp32 rows of whole words, by copies that this thread waits for later.
template <int kD, typename Offset>
__device__ __forceinline__ void copy_tile(float* dst, const void* base, int n, int D, Offset offset, int first = 0) {
  using L = Tile<kD>;
  constexpr int kRow = kD / 4;
#pragma unroll
  for (int i = threadIdx.x; i < L::kT * kRow; i += kThreads) {
    const int r = i / kRow, d = (i - r * kRow) * 4;
    float* to = dst + r * L::kStride + d;
    if (r >= first && r < n && d < D) sm100::cp_async16(sm100::smem_u32(to), static_cast<const float*>(base) + offset(r) + d);
    else *reinterpret_cast<float4*>(to) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the last group of copies have landed
__device__ __forceinline__ void wait_copies_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// A key or value tile: copied (fp32 words; what follows has to wait) or loaded.
template <typename T, int kD, bool kWords, typename Offset>
__device__ __forceinline__ void fetch_tile(float* dst, const void* base, int n, int D, Offset offset, int first = 0) {
  if constexpr (kWords && sizeof(T) == 4) copy_tile<kD>(dst, base, n, D, offset, first);
  else load_tile<T, kD, kWords>(dst, base, n, D, offset, first);
  commit_copies();
}

// s[i][j] = A row (ty * kM + i) . B row (tx + 16 j)
template <int kD>
__device__ __forceinline__ void products(float (&s)[Tile<kD>::kM][Tile<kD>::kM], const float* A, const float* B) {
  using L = Tile<kD>;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float2 t[L::kM][L::kM];      // sums over even and over odd columns: two multiply-adds per instruction
#pragma unroll
  for (int i = 0; i < L::kM; ++i)
#pragma unroll
    for (int j = 0; j < L::kM; ++j) t[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int d = 0; d < kD; d += 4) {
    float4 a[L::kM], b[L::kM];
#pragma unroll
    for (int i = 0; i < L::kM; ++i) {
      a[i] = *reinterpret_cast<const float4*>(A + (ty * L::kM + i) * L::kStride + d);
      b[i] = *reinterpret_cast<const float4*>(B + (tx + 16 * i) * L::kStride + d);
    }
#pragma unroll
    for (int i = 0; i < L::kM; ++i)
#pragma unroll
      for (int j = 0; j < L::kM; ++j) {
        t[i][j] = __ffma2_rn(make_float2(a[i].x, a[i].y), make_float2(b[j].x, b[j].y), t[i][j]);
        t[i][j] = __ffma2_rn(make_float2(a[i].z, a[i].w), make_float2(b[j].z, b[j].w), t[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < L::kM; ++i)
#pragma unroll
    for (int j = 0; j < L::kM; ++j) s[i][j] = t[i][j].x + t[i][j].y;
}

// acc[i] += sum_c W(row ty * kM + i, c) B row c; W is kT x kT in shared memory, read along rows or (transposed) columns.
// Columns of a thread: tx * 4 + 64 j.
template <int kD, bool kTransposed>
__device__ __forceinline__ void accumulate(float4 (&acc)[Tile<kD>::kM][Tile<kD>::kCols], const float* W, const float* B) {
  using L = Tile<kD>;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  // four columns of W at a time: its words are read whole, along rows or (transposed) down the rows of this thread
  static_assert(L::kM == 4 || L::kM == 2, "rows of a thread");
#pragma unroll 2
  for (int c0 = 0; c0 < L::kT; c0 += 4) {
    float w[L::kM][4];
    if constexpr (kTransposed) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float* x = W + (c0 + c) * L::kPStride + ty * L::kM;
        if constexpr (L::kM == 4) {
          const float4 v = *reinterpret_cast<const float4*>(x);
          w[0][c] = v.x; w[1][c] = v.y; w[2][c] = v.z; w[3][c] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(x);
          w[0][c] = v.x; w[1][c] = v.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < L::kM; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(W + (ty * L::kM + i) * L::kPStride + c0);
        w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < L::kCols; ++j) {
        const float4 b = *reinterpret_cast<const float4*>(B + (c0 + c) * L::kStride + tx * 4 + 64 * j);
#pragma unroll
        for (int i = 0; i < L::kM; ++i) {
          const float2 ww = make_float2(w[i][c], w[i][c]);
          const float2 lo = __ffma2_rn(ww, make_float2(b.x, b.y), make_float2(acc[i][j].x, acc[i][j].y));
          const float2 hi = __ffma2_rn(ww, make_float2(b.z, b.w), make_float2(acc[i][j].z, acc[i][j].w));
          acc[i][j] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
      }
  }
}

template <int kD>
__device__ __forceinline__ void clear(float4 (&acc)[Tile<kD>::kM][Tile<kD>::kCols]) {
#pragma unroll
  for (int i = 0; i < Tile<kD>::kM; ++i)
#pragma unroll
    for (int j = 0; j < Tile<kD>::kCols; ++j) acc[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
}

template <typename T, int kD>
__device__ __forceinline__ void store_row(T* dst, const float4 (&row)[Tile<kD>::kCols], float mul, int D) {
  const int tx = threadIdx.x & 15;
#pragma unroll
  for (int j = 0; j < Tile<kD>::kCols; ++j) {
    const float v[4] = {row[j].x, row[j].y, row[j].z, row[j].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = tx * 4 + 64 * j + e;
      if (d < D) dst[d] = from_f32<T>(v[e] * mul);
    }
  }
}

// Rows of a sequence of one key head: query r / G, head r % G.
struct Rows {
  int2 q, k;           // first token, tokens
  int kv_head, group, heads;
  int64_t n;           // rows
  __device__ __forceinline__ Rows(const PackedArgs& a, int sequence, int kv)
      : q(sequence_span(a.offsets_q, sequence, a.tokens_q)), k(sequence_span(a.offsets_k, sequence, a.tokens_k)), kv_head(kv),
        group(a.group), heads(a.heads), n(int64_t(q.y) * a.group) {}
  __device__ __forceinline__ int token(int64_t r) const { return q.x + int(r / group); }
  __device__ __forceinline__ int head(int64_t r) const { return kv_head * group + int(r % group); }
  __device__ __forceinline__ int64_t at(int64_t r, const int64_t (&stride)[2]) const { return token(r) * stride[0] + head(r) * stride[1]; }
  // (token, head) index of a dense array
  __device__ __forceinline__ int64_t flat(int64_t r) const { return int64_t(token(r)) * heads + head(r); }
  // keys that row r sees: the first `seen` of the sequence
  __device__ __forceinline__ int seen(int64_t r, int causal) const {
    return causal ? min(k.y, max(int(r / group) + 1 + k.y - q.y, 0)) : k.y;
  }
};

template <typename T, int kD, bool kWords>
__global__ void __launch_bounds__(kThreads, kD > 64 ? 1 : 2) packed_fwd_simt_kernel(const PackedArgs a) {
  using L = Tile<kD>;
  extern __shared__ __align__(16) float smem[];
  float *sq = smem, *sk = sq + L::kOperand, *sv = sk + L::kOperand, *sp = sv + L::kOperand;
  const Place place = find_place(blockIdx.x, a.sequences, [&](int i) { return int((int64_t(sequence_span(a.offsets_q, i, a.tokens_q).y) * a.group + L::kT - 1) / L::kT); });
  if (place.index < 0) return;
  const Rows rows(a, place.sequence, blockIdx.y);
  // (the last tiles of a sequence see the most keys: they go first)
  const int64_t r0 = ((rows.n - 1) / L::kT - place.index) * L::kT;
  const int n = int(min(int64_t(L::kT), rows.n - r0));
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float mul = a.scale * kLog2e;
  __shared__ int64_t at_q[L::kT];
  row_offsets<L::kT>(at_q, n, [&](int r) { return rows.at(r0 + r, a.qs); });
  __syncthreads();
  load_tile<T, kD, kWords>(sq, a.q, n, a.D, [&](int r) { return at_q[r]; });
  float m[L::kM], l[L::kM];
  int seen[L::kM];
  float4 acc[L::kM][L::kCols];
  clear<kD>(acc);
#pragma unroll
  for (int i = 0; i < L::kM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    seen[i] = ty * L::kM + i < n ? rows.seen(r0 + ty * L::kM + i, a.causal) : 0;
  }
  const int keys = rows.seen(r0 + n - 1, a.causal);     // the tile's last row sees the most
  // The next tile's keys are on their way from the scores on, its values from the end of the output products on.
  auto fetch = [&](float* dst, const void* base, const int64_t (&stride)[2], int k0) {
    if (k0 < keys)
      fetch_tile<T, kD, kWords>(dst, base, min(L::kT, rows.k.y - k0), a.D, [&](int r) { return (int64_t(rows.k.x) + k0 + r) * stride[0] + rows.kv_head * stride[1]; });
    else
      commit_copies();
  };
  fetch(sk, a.k, a.ks, 0);
  fetch(sv, a.v, a.vs, 0);
  for (int k0 = 0; k0 < keys; k0 += L::kT) {
    wait_copies_but_one();
    __syncthreads();
    float s[L::kM][L::kM];
    products<kD>(s, sq, sk);
    __syncthreads();
    fetch(sk, a.k, a.ks, k0 + L::kT);
#pragma unroll
    for (int i = 0; i < L::kM; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < L::kM; ++j) {
        s[i][j] = k0 + tx + 16 * j < seen[i] ? s[i][j] * mul : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float shift = mx == -INFINITY ? 0.f : mx, alpha = exp2f(m[i] - shift);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < L::kM; ++j) {
        const float p = exp2f(s[i][j] - shift);
        sum += p;
        sp[(ty * L::kM + i) * L::kPStride + tx + 16 * j] = p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = l[i] * alpha + sum;
      m[i] = mx;
#pragma unroll
      for (int j = 0; j < L::kCols; ++j) {
        acc[i][j].x *= alpha; acc[i][j].y *= alpha; acc[i][j].z *= alpha; acc[i][j].w *= alpha;
      }
    }
    wait_copies_but_one();
    __syncthreads();
    accumulate<kD, false>(acc, sp, sv);
    __syncthreads();
    fetch(sv, a.v, a.vs, k0 + L::kT);
  }
#pragma unroll
  for (int i = 0; i < L::kM; ++i) {
    const int r = ty * L::kM + i;
    if (r >= n) continue;
    const int64_t at = rows.flat(r0 + r);
    const bool empty = seen[i] == 0;
    store_row<T, kD>(static_cast<T*>(a.out) + at * a.D, acc[i], empty ? 0.f : 1.f / l[i], a.D);
    if (tx == 0) a.lse[at] = empty ? -INFINITY : m[i] + log2f(l[i]);
  }
}

// P and dS of a (row tile, key tile) pair into shared memory; row statistics in `stat` (lse, delta per row)
template <int kD>
__device__ __forceinline__ void score_gradients(const float* sq, const float* sdo, const float* sk, const float* sv, float* sp,
                                                float* sds, const float* stat, const int* seen, int k0, float mul) {
  using L = Tile<kD>;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float s[L::kM][L::kM], dp[L::kM][L::kM];
  products<kD>(s, sq, sk);
  products<kD>(dp, sdo, sv);
#pragma unroll
  for (int i = 0; i < L::kM; ++i)
#pragma unroll
    for (int j = 0; j < L::kM; ++j) {
      const int r = ty * L::kM + i, c = tx + 16 * j;
      const bool in = k0 + c < seen[r];
      const float p = in ? exp2f(s[i][j] * mul - stat[2 * r]) : 0.f;
      if (sp) sp[r * L::kPStride + c] = p;
      sds[r * L::kPStride + c] = in ? p * (dp[i][j] - stat[2 * r + 1]) : 0.f;
    }
}

template <int kT>
__device__ __forceinline__ void load_stats(const PackedArgs& a, const Rows& rows, int64_t r0, int n, float* stat, int* seen) {
  if (threadIdx.x < kT) {
    const int r = threadIdx.x;
    const int64_t at = r < n ? rows.flat(r0 + r) : 0;
    stat[2 * r] = r < n ? a.lse[at] : 0.f;
    stat[2 * r + 1] = r < n ? a.delta[at] : 0.f;
    seen[r] = r < n ? rows.seen(r0 + r, a.causal) : 0;
  }
}

template <typename T, int kD, bool kWords>
__global__ void __launch_bounds__(kThreads, 1) packed_dq_simt_kernel(const PackedArgs a) {
  using L = Tile<kD>;
  extern __shared__ __align__(16) float smem[];
  __shared__ float stat[2 * L::kT];
  __shared__ int seen[L::kT];
  __shared__ int64_t at_q[L::kT], at_do[L::kT];
  float *sq = smem, *sdo = sq + L::kOperand, *sk = sdo + L::kOperand, *sv = sk + 2 * L::kOperand, *sds = sv + L::kOperand;
  const Place place = find_place(blockIdx.x, a.sequences, [&](int i) { return int((int64_t(sequence_span(a.offsets_q, i, a.tokens_q).y) * a.group + L::kT - 1) / L::kT); });
  if (place.index < 0) return;
  const Rows rows(a, place.sequence, blockIdx.y);
  // (the last tiles of a sequence see the most keys: they go first)
  const int64_t r0 = ((rows.n - 1) / L::kT - place.index) * L::kT;
  const int n = int(min(int64_t(L::kT), rows.n - r0));
  const int ty = threadIdx.x >> 4;
  row_offsets<L::kT>(at_q, n, [&](int r) { return rows.at(r0 + r, a.qs); });
  row_offsets<L::kT>(at_do, n, [&](int r) { return rows.at(r0 + r, a.dos); });
  __syncthreads();
  load_tile<T, kD, kWords>(sq, a.q, n, a.D, [&](int r) { return at_q[r]; });
  load_tile<T, kD, kWords>(sdo, a.dout, n, a.D, [&](int r) { return at_do[r]; });
  load_stats<L::kT>(a, rows, r0, n, stat, seen);
  float4 acc[L::kM][L::kCols];
  clear<kD>(acc);
  const int keys = rows.seen(r0 + n - 1, a.causal);
  // Keys in two buffers (they are needed to the end of a turn), values in one: the next tile is on its way from the scores on.
  auto fetch = [&](float* dst, const void* base, const int64_t (&stride)[2], int k0) {
    if (k0 < keys)
      fetch_tile<T, kD, kWords>(dst, base, min(L::kT, rows.k.y - k0), a.D, [&](int r) { return (int64_t(rows.k.x) + k0 + r) * stride[0] + rows.kv_head * stride[1]; });
    else
      commit_copies();
  };
  fetch(sk, a.k, a.ks, 0);
  fetch(sv, a.v, a.vs, 0);
  for (int k0 = 0, turn = 0; k0 < keys; k0 += L::kT, ++turn) {
    const float* keys_now = sk + (turn & 1) * L::kOperand;
    fetch(sk + (~turn & 1) * L::kOperand, a.k, a.ks, k0 + L::kT);      // (its last readers passed the barrier at the end of their turn)
    wait_copies_but_one();
    __syncthreads();
    score_gradients<kD>(sq, sdo, keys_now, sv, nullptr, sds, stat, seen, k0, a.scale * kLog2e);
    __syncthreads();
    fetch(sv, a.v, a.vs, k0 + L::kT);
    accumulate<kD, false>(acc, sds, keys_now);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < L::kM; ++i) {
    const int r = ty * L::kM + i;
    if (r < n) store_row<T, kD>(static_cast<T*>(a.dq) + rows.flat(r0 + r) * a.D, acc[i], a.scale, a.D);
  }
}

template <typename T, int kD, bool kWords>
__global__ void __launch_bounds__(kThreads, 1) packed_dkv_simt_kernel(const PackedArgs a) {
  using L = Tile<kD>;
  extern __shared__ __align__(16) float smem[];
  __shared__ float stat[2][2 * L::kT];
  __shared__ int seen[2][L::kT];
  __shared__ int64_t at_q[2][L::kT], at_do[2][L::kT];
  float *sq = smem, *sdo = sq + L::kOperand, *sk = sdo + L::kOperand, *sv = sk + L::kOperand, *sp = sv + L::kOperand,
        *sds = sp + L::kScores;
  const Place place = find_place(blockIdx.x, a.sequences, [&](int i) { return int((int64_t(sequence_span(a.offsets_k, i, a.tokens_k).y) + L::kT - 1) / L::kT); });
  if (place.index < 0) return;
  const Rows rows(a, place.sequence, blockIdx.y);
  const int k0 = place.index * L::kT, nk = min(L::kT, rows.k.y - k0);
  const int ty = threadIdx.x >> 4;
  load_tile<T, kD, kWords>(sk, a.k, nk, a.D, [&](int r) { return (int64_t(rows.k.x) + k0 + r) * a.ks[0] + rows.kv_head * a.ks[1]; });
  load_tile<T, kD, kWords>(sv, a.v, nk, a.D, [&](int r) { return (int64_t(rows.k.x) + k0 + r) * a.vs[0] + rows.kv_head * a.vs[1]; });
  float4 dk[L::kM][L::kCols], dv[L::kM][L::kCols];
  clear<kD>(dk);
  clear<kD>(dv);
  // the first query that sees this tile's first key; the row tiles from there on are dealt to gridDim.z CTAs in turn
  const int64_t first = a.causal ? int64_t(max(k0 - (rows.k.y - rows.q.y), 0)) * a.group : 0;
  const int64_t step = int64_t(gridDim.z) * L::kT, begin = (first / L::kT + blockIdx.z) * L::kT;
  auto count = [&](int64_t r0) { return r0 < rows.n ? int(min(int64_t(L::kT), rows.n - r0)) : 0; };
  auto place_rows = [&](int buf, int64_t r0) {      // where the rows lie, and their statistics
    const int n = count(r0);
    row_offsets<L::kT>(at_q[buf], n, [&](int r) { return rows.at(r0 + r, a.qs); });
    row_offsets<L::kT>(at_do[buf], n, [&](int r) { return rows.at(r0 + r, a.dos); });
    if (n > 0) load_stats<L::kT>(a, rows, r0, n, stat[buf], seen[buf]);
  };
  // (rows of queries that see no key are left out: a probability of zero makes a NaN of what is not a number in them)
  const int64_t blind = a.causal ? int64_t(max(rows.q.y - rows.k.y, 0)) * a.group : 0;
  auto fetch = [&](float* dst, const void* base, const int64_t* at, int64_t r0) {
    if (r0 < rows.n)
      fetch_tile<T, kD, kWords>(dst, base, count(r0), a.D, [&](int r) { return at[r]; }, int(min(max(blind - r0, int64_t(0)), int64_t(L::kT))));
  };
  place_rows(0, begin);
  __syncthreads();
  fetch(sq, a.q, at_q[0], begin);
  fetch(sdo, a.dout, at_do[0], begin);
  int buf = 0;
  for (int64_t r0 = begin; r0 < rows.n; r0 += step, buf ^= 1) {
    sm100::cp_async_wait_all();
    __syncthreads();
    score_gradients<kD>(sq, sdo, sk, sv, sp, sds, stat[buf], seen[buf], k0, a.scale * kLog2e);
    place_rows(buf ^ 1, r0 + step);
    __syncthreads();
    accumulate<kD, true>(dv, sp, sdo);
    __syncthreads();
    fetch(sdo, a.dout, at_do[buf ^ 1], r0 + step);      // under the products of dk
    accumulate<kD, true>(dk, sds, sq);
    __syncthreads();
    fetch(sq, a.q, at_q[buf ^ 1], r0 + step);
  }
#pragma unroll
  for (int i = 0; i < L::kM; ++i) {
    const int r = ty * L::kM + i;
    if (r >= nk) continue;
    const int64_t at = (int64_t(rows.k.x) + k0 + r) * a.kv_heads + rows.kv_head;
    if (gridDim.z == 1) {
      store_row<T, kD>(static_cast<T*>(a.dk) + at * a.D, dk[i], a.scale, a.D);
      store_row<T, kD>(static_cast<T*>(a.dv) + at * a.D, dv[i], 1.f, a.D);
    } else {
      const int64_t all = int64_t(a.tokens_k) * a.kv_heads * a.D;
      store_row<float, kD>(a.parts + 2 * blockIdx.z * all + at * a.D, dk[i], a.scale, a.D);
      store_row<float, kD>(a.parts + (2 * blockIdx.z + 1) * all + at * a.D, dv[i], 1.f, a.D);
    }
  }
}

// dk and dv as the sums of their parts, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) packed_dkv_sum_kernel(const PackedArgs a, int parts) {
  const int64_t row = int64_t(a.kv_heads) * a.D, all = a.tokens_k * row;
  const int64_t first = tokens_before(a.offsets_k, a.sequences, a.tokens_k) * row, end = covered_tokens(a.offsets_k, a.sequences, a.tokens_k) * row;
  for (int64_t i = first + int64_t(blockIdx.x) * kThreads + threadIdx.x; i < end; i += int64_t(gridDim.x) * kThreads) {
    float dk = 0.f, dv = 0.f;
    for (int p = 0; p < parts; ++p) {
      dk += a.parts[2 * p * all + i];
      dv += a.parts[(2 * p + 1) * all + i];
    }
    static_cast<T*>(a.dk)[i] = from_f32<T>(dk);
    static_cast<T*>(a.dv)[i] = from_f32<T>(dv);
  }
}

// delta[token][head] = sum_d out dout: a warp per row
template <typename T>
__global__ void __launch_bounds__(kThreads) packed_delta_kernel(const PackedArgs a) {
  const int64_t row = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= int64_t(a.tokens_q) * a.heads) return;
  const int64_t token = row / a.heads;
  const int head = int(row - token * a.heads);
  const T* o = static_cast<const T*>(a.out) + row * a.D;
  const T* g = static_cast<const T*>(a.dout) + token * a.dos[0] + head * a.dos[1];
  float sum = 0.f;
  for (int d = lane; d < a.D; d += 32) sum = fmaf(to_f32<T>(o[d]), to_f32<T>(g[d]), sum);
#pragma unroll
  for (int o2 = 16; o2 > 0; o2 >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
  if (lane == 0) a.delta[row] = sum;
}

// The tokens of no sequence: before the first and behind the last.
template <typename T>
__global__ void __launch_bounds__(kThreads) packed_clear_kernel(const PackedArgs a, bool backward) {
  const int64_t step = int64_t(gridDim.x) * kThreads, at = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int q0 = tokens_before(a.offsets_q, a.sequences, a.tokens_q), q1 = covered_tokens(a.offsets_q, a.sequences, a.tokens_q);
  clear_outside(static_cast<T*>(backward ? a.dq : a.out), int64_t(a.heads) * a.D, q0, q1, a.tokens_q, from_f32<T>(0.f), at, step);
  if (!backward) {
    clear_outside(a.lse, a.heads, q0, q1, a.tokens_q, -INFINITY, at, step);
    return;
  }
  const int k0 = tokens_before(a.offsets_k, a.sequences, a.tokens_k), k1 = covered_tokens(a.offsets_k, a.sequences, a.tokens_k);
  clear_outside(static_cast<T*>(a.dk), int64_t(a.kv_heads) * a.D, k0, k1, a.tokens_k, from_f32<T>(0.f), at, step);
  clear_outside(static_cast<T*>(a.dv), int64_t(a.kv_heads) * a.D, k0, k1, a.tokens_k, from_f32<T>(0.f), at, step);
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == NB200_F32) return f(float());
  if (dtype == NB200_BF16) return f(__nv_bfloat16());
  return f(__half());
}
template <int kN>
struct Int {
  static constexpr int value = kN;
};
template <typename F>
int by_head_dim(int D, F f) {
  if (D <= 64) return f(Int<64>());
  if (D <= 128) return f(Int<128>());
  return f(Int<256>());
}

template <typename F>
int by_words(bool words, F f) {
  return words ? f(std::true_type()) : f(std::false_type());
}
// rows of whole 16-byte words on 16-byte boundaries
bool words(const PackedArgs& a, size_t size, bool backward) {
  const int64_t vec = int64_t(16 / size);
  auto fits = [&](const void* p, const int64_t (&st)[2]) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % vec == 0 && st[1] % vec == 0; };
  return a.D % vec == 0 && fits(a.q, a.qs) && fits(a.k, a.ks) && fits(a.v, a.vs) && (!backward || fits(a.dout, a.dos));
}

template <typename Kernel>
int configure(Kernel kernel, size_t smem, const char* what) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return check_launch(what);
  return NB200_OK;
}

// most tiles that sequences of `tokens` tokens together can have
unsigned most_tiles(int64_t rows, int sequences, int tile) { return unsigned(rows / tile + sequences); }

}  // namespace

int launch_clear_uncovered(const PackedArgs& a, int dtype, bool backward, cudaStream_t st) {
  return by_type(dtype, [&](auto t) {
    packed_clear_kernel<decltype(t)><<<32, kThreads, 0, st>>>(a, backward);
    count_launch();
    return check_launch("packed_clear_kernel");
  });
}

int launch_packed_delta(const PackedArgs& a, int dtype, cudaStream_t st) {
  return by_type(dtype, [&](auto t) {
    const int64_t rows = int64_t(a.tokens_q) * a.heads;
    packed_delta_kernel<decltype(t)><<<unsigned((rows + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(a);
    count_launch();
    return check_launch("packed_delta_kernel");
  });
}

int simt_packed_fwd(const PackedArgs& a, int dtype, cudaStream_t st) {
  return by_type(dtype, [&](auto t) {
    return by_head_dim(a.D, [&](auto d) {
      return by_words(words(a, sizeof(t), false), [&](auto w) {
        constexpr int kD = decltype(d)::value;
        using L = Tile<kD>;
        auto kernel = packed_fwd_simt_kernel<decltype(t), kD, decltype(w)::value>;
        constexpr size_t smem = sizeof(float) * (3 * L::kOperand + L::kScores);
        static_assert(smem + 1024 <= 232448, "shared memory of a CTA");
        if (int rc = configure(kernel, smem, "packed_fwd_simt_kernel")) return rc;
        kernel<<<dim3(most_tiles(int64_t(a.tokens_q) * a.group, a.sequences, L::kT), unsigned(a.kv_heads)), kThreads, smem, st>>>(a);
        count_launch();
        return check_launch("packed_fwd_simt_kernel");
      });
    });
  });
}

// Parts that a key tile's rows are taken in, up to eight where the key tiles alone are fewer than eight per SM: the tiles of a causal
// sequence differ in length, and a group's rows all fall to one key head (f32, 2048 tokens, 16 heads on one, head dim 128, one
// part: 32 CTAs, 19 ms).
int dkv_parts(const PackedArgs& a) {
  const int64_t ctas = int64_t(most_tiles(a.tokens_k, a.sequences, a.D > 128 ? 32 : 64)) * a.kv_heads;
  const int64_t parts = (8 * 148 + ctas - 1) / (ctas < 1 ? 1 : ctas);
  return int(parts < 1 ? 1 : parts > 8 ? 8 : parts);
}

size_t simt_packed_bwd_bytes(const PackedArgs& a) {
  const int parts = dkv_parts(a);
  return parts > 1 ? size_t(parts) * 2 * size_t(a.tokens_k) * a.kv_heads * a.D * sizeof(float) : 0;
}

int simt_packed_bwd(const PackedArgs& a, int dtype, cudaStream_t st) {
  return by_type(dtype, [&](auto t) {
    return by_head_dim(a.D, [&](auto d) {
      return by_words(words(a, sizeof(t), true), [&](auto w) {
        constexpr int kD = decltype(d)::value;
        using L = Tile<kD>;
        constexpr size_t smem_dq = sizeof(float) * (5 * L::kOperand + L::kScores), smem_dkv = sizeof(float) * (4 * L::kOperand + 2 * L::kScores);
        static_assert(smem_dkv + 2048 <= 232448 && smem_dq + 2048 <= 232448, "shared memory of a CTA");
        if (a.tokens_q > 0) {
          auto kernel = packed_dq_simt_kernel<decltype(t), kD, decltype(w)::value>;
          if (int rc = configure(kernel, smem_dq, "packed_dq_simt_kernel")) return rc;
          kernel<<<dim3(most_tiles(int64_t(a.tokens_q) * a.group, a.sequences, L::kT), unsigned(a.kv_heads)), kThreads, smem_dq, st>>>(a);
          count_launch();
          if (int rc = check_launch("packed_dq_simt_kernel")) return rc;
        }
        if (a.tokens_k == 0) return int(NB200_OK);
        auto kernel = packed_dkv_simt_kernel<decltype(t), kD, decltype(w)::value>;
        if (int rc = configure(kernel, smem_dkv, "packed_dkv_simt_kernel")) return rc;
        const int parts = dkv_parts(a);
        kernel<<<dim3(most_tiles(a.tokens_k, a.sequences, L::kT), unsigned(a.kv_heads), unsigned(parts)), kThreads, smem_dkv, st>>>(a);
        count_launch();
        if (int rc = check_launch("packed_dkv_simt_kernel")) return rc;
        if (parts == 1) return int(NB200_OK);
        const int64_t n = int64_t(a.tokens_k) * a.kv_heads * a.D;
        packed_dkv_sum_kernel<decltype(t)><<<unsigned(n / kThreads + 1 < 148 * 8 ? n / kThreads + 1 : 148 * 8), kThreads, 0, st>>>(a, parts);
        count_launch();
        return check_launch("packed_dkv_sum_kernel");
      });
    });
  });
}

}  // namespace packed
}  // namespace nb200
