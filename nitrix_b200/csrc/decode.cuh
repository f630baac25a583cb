// What the kernels of attention of one new token over a paged cache share (decode.cu, decode_quantized.cu): the division of the
// work, the kernel around a loop over the tokens, and the joining of pieces.
//
// A loop has kName, its name in a profile; kHeads, the query heads that it takes; kSlots, the partial results that a warp leaves; kMinCtas;
// kRing, bytes of shared memory that a warp has to itself, or 0;
// run(args, row of the table, key head, queries, heads, t0, t1, wi, wn), which takes part `wi` of `wn` of the tokens t0 .. t1 for one
// warp; and store(args, dst), which leaves output, maximum (base 2) and sum of every head and slot.
#pragma once

#include <math.h>

#include "dependent_launch.cuh"
#include "nitrix_b200_cache.h"
#include "sdpa_tc_common.cuh"

namespace nb200 {
namespace {

using tc::ex2;
using tc::pack2;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct DecodeArgs {
  const uint4* k;
  const uint4* v;
  int ks[3], vs[3];          // 16-byte words, over (page, head, slot): 32 bits, so that an offset is one wide multiply-add each
  int pages, kv_heads, page_size, page_shift;   // page_shift: log2 of page_size, or -1
  int D;
  const int* table;
  const int* lengths;
  int rows, width;
  const void* q;
  int64_t qs[2];
  void* out;
  int q_heads, group;        // query heads, and those of one key head
  int chunks;                // times that a key head's group is taken, kSide chunks of query heads side by side each
  float mul;                 // scale * log2 e
  int unit;                  // tokens per unit of work
  int extra;                 // units that beginning with a (sequence, key head) counts for
  float* part;               // pieces: [2 * CTAs][heads of a chunk][D + 4]: output, maximum (base 2), sum
  int workers;               // most CTAs of the main kernel that get work
};

__device__ __forceinline__ int length_of(const DecodeArgs& a, int row) {
  return int(min(int64_t(min(max(a.lengths[row], 0), NB200_CACHE_MOST_TOKENS)), int64_t(a.width) * a.page_size));
}
__device__ __forceinline__ int units_of_length(const DecodeArgs& a, int length) { return length > 0 ? (length + a.unit - 1) / a.unit + a.extra : 0; }
__device__ __forceinline__ int units_of(const DecodeArgs& a, int row) { return units_of_length(a, length_of(a, row)); }

// Work position: units of all rows times (key head, chunk), row-major.  All lanes of a warp hold the same values.
struct Share {
  int64_t total;             // units of work
  int workers;               // with a unit at least
  __device__ __forceinline__ Share(const DecodeArgs& a, int64_t units) : total(units), workers(int(min(int64_t(a.workers), units))) {}
  __device__ __forceinline__ int64_t begin(int worker) const { return total * worker / workers; }
  // the worker whose share holds position u < total
  __device__ __forceinline__ int worker_of(int64_t u) const {
    int w = int(u * workers / total);
    while (begin(w + 1) <= u) ++w;        // (begin rounds down, so that the estimate may be one short)
    return w;
  }
};

__device__ __forceinline__ Share share_of(const DecodeArgs& a, int lane) {
  int64_t units = 0;
  for (int i = lane; i < a.rows; i += 32) units += units_of(a, i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
  return Share(a, units * a.kv_heads * a.chunks);
}

// the row that position u < total lies in, and the position of its first unit
__device__ __forceinline__ void find_row(const DecodeArgs& a, int lane, int64_t u, int* row, int64_t* row_begin) {
  const int per = a.kv_heads * a.chunks;
  int64_t before = 0;
  for (int row0 = 0; row0 < a.rows; row0 += 32) {
    int64_t upto = row0 + lane < a.rows ? int64_t(units_of(a, row0 + lane)) * per : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    const unsigned above = __ballot_sync(0xffffffffu, before + upto > u);
    if (above) {
      const int j = __ffs(above) - 1;
      const int64_t prev = __shfl_sync(0xffffffffu, upto, j > 0 ? j - 1 : 0);
      *row = row0 + j;
      *row_begin = before + (j > 0 ? prev : 0);
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  *row = a.rows;
  *row_begin = before;
}

// Where a token's row lies: its page (cut to the pool) and slot.
struct Where {
  int page, slot;
};
__device__ __forceinline__ int page_at(const DecodeArgs& a, const int* row_table, int column) {
  return min(max(__ldg(row_table + column), 0), a.pages - 1);
}
__device__ __forceinline__ Where where(const DecodeArgs& a, const int* row_table, int token) {
  const int column = a.page_shift >= 0 ? token >> a.page_shift : token / a.page_size;
  return Where{page_at(a, row_table, column), token - (a.page_shift >= 0 ? column << a.page_shift : column * a.page_size)};
}
__device__ __forceinline__ const uint4* row_of(const uint4* base, const int (&stride)[3], Where w) {
  return base + int64_t(w.page) * stride[0] + int64_t(w.slot) * stride[2];
}

// ---- warp-level MMA ------------------------------------------------------------------------------------------------------
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Floats of shared memory from one slot's results to the next one's; a loop with a ring leaves its results there.
template <typename Loop>
__host__ __device__ constexpr int slot_stride(int D) { return Loop::kRing > 0 ? Loop::kRing / 4 : Loop::kHeads * (D + 2); }

// kSide chunks of query heads are taken by the warps of a CTA side by side.
template <typename T, typename Loop, int kSide, typename Args>
__global__ void __launch_bounds__(kThreads, Loop::kMinCtas) decode_kernel(const Args a) {
  extern __shared__ __align__(16) float merge[];      // [slot][head][D + 2], or the warps' rings
  allow_dependents();
  const int lane = threadIdx.x & 31;
  const Share share = share_of(a, lane);
  if (int(blockIdx.x) >= share.workers) return;
  int64_t u = share.begin(blockIdx.x);
  const int64_t u_end = share.begin(blockIdx.x + 1);
  const int per = a.kv_heads * a.chunks;
  int row;
  int64_t row_begin;
  find_row(a, lane, u, &row, &row_begin);
  while (u < u_end) {
    const int length = length_of(a, row);
    const int units = units_of_length(a, length);
    if (units == 0) { ++row; continue; }
    const int item = int((u - row_begin) / units);
    const int64_t item_begin = row_begin + int64_t(item) * units;
    const int kv_head = item / a.chunks, chunk = item - kv_head * a.chunks;
    const int ub = int(u - item_begin), ue = int(min(int64_t(units), u_end - item_begin));
    const int in_group = chunk * kSide * Loop::kHeads;                 // the first query head within its group
    const int heads = min(kSide * Loop::kHeads, a.group - in_group);   // of all chunks that are taken side by side
    const int head0 = kv_head * a.group + in_group;
    const bool whole = ub == 0 && ue == units;
    constexpr int wn = kWarps / kSide;                                  // warps of a chunk
    const int own = (threadIdx.x >> 5) / wn;                            // this warp's chunk
    if (own * Loop::kHeads < heads) {
      Loop loop;
      const int t0 = max(ub - a.extra, 0) * a.unit, t1 = min(length, max(ue - a.extra, 0) * a.unit);
      const T* q = static_cast<const T*>(a.q) + row * a.qs[0] + (head0 + own * Loop::kHeads) * a.qs[1];
      const int* row_table = a.table + int64_t(row) * a.width;
      const int own_heads = min(Loop::kHeads, heads - own * Loop::kHeads), wi = (threadIdx.x >> 5) % wn;
      if constexpr (Loop::kRing > 0)
        loop.run(a, row_table, kv_head, q, own_heads, t0, t1, wi, wn, reinterpret_cast<char*>(merge) + (threadIdx.x >> 5) * Loop::kRing);
      else
        loop.run(a, row_table, kv_head, q, own_heads, t0, t1, wi, wn);
      loop.store(a, merge);
    }
    __syncthreads();
    // the CTA's result: sums over the slots of a head's warps, relative to their largest maximum
    float* part = a.part + int64_t(2 * blockIdx.x + (ub == 0 ? 1 : 0)) * kSide * Loop::kHeads * (a.D + 4);
    constexpr int slots = wn * Loop::kSlots;
    const int step = slot_stride<Loop>(a.D);
    for (int i = threadIdx.x; i < heads * a.D; i += kThreads) {
      const int h = i / a.D, d = i - h * a.D, of = h / Loop::kHeads;
      const float* col = merge + of * slots * step + (h - of * Loop::kHeads) * (a.D + 2);
      float mx = -INFINITY;
#pragma unroll
      for (int s = 0; s < slots; ++s) mx = fmaxf(mx, col[s * step + a.D]);
      const float shift = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int s = 0; s < slots; ++s) {
        const float w = ex2(col[s * step + a.D] - shift);
        sum = fmaf(w, col[s * step + a.D + 1], sum);
        acc = fmaf(w, col[s * step + d], acc);
      }
      if (whole) {
        static_cast<T*>(a.out)[(int64_t(row) * a.q_heads + head0 + h) * a.D + d] = from_f32<T>(acc / sum);
      } else {
        part[h * (a.D + 4) + d] = acc;
        if (d == 0) *reinterpret_cast<float2*>(part + h * (a.D + 4) + a.D) = make_float2(mx, sum);
      }
    }
    __syncthreads();
    u += ue - ub;
    if (u == row_begin + int64_t(units) * per) { row_begin = u; ++row; }
  }
}

// Sums of pieces w, w + stride, ... up to w1 of one query head, a lane's 16-byte words of them.
struct Joined {
  float top, sum;
  float4 acc[2];
};
template <typename Piece>
__device__ __forceinline__ Joined join_pieces(int w, int w1, int stride, int D, Piece piece) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 31, words = D / 4;
  Joined r{-INFINITY, 0.f, {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)}};
  for (; w <= w1; w += stride * kAhead) {
    float2 st[kAhead];
    float4 v[kAhead][2];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int wj = w + j * stride;
      st[j] = make_float2(-INFINITY, 0.f);
      if (wj > w1) continue;
      const float* p = piece(wj);
      st[j] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < words) v[j][i] = reinterpret_cast<const float4*>(p)[lane + 32 * i];
    }
    float next = r.top;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) next = fmaxf(next, st[j].x);
    const float shift = next == -INFINITY ? 0.f : next, old = ex2(r.top - shift);
    r.sum *= old;
#pragma unroll
    for (int i = 0; i < 2; ++i) { r.acc[i].x *= old; r.acc[i].y *= old; r.acc[i].z *= old; r.acc[i].w *= old; }
    r.top = next;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (w + j * stride > w1) continue;
      const float f = ex2(st[j].x - shift);
      r.sum = fmaf(f, st[j].y, r.sum);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (lane + 32 * i >= words) continue;
        r.acc[i].x = fmaf(f, v[j][i].x, r.acc[i].x); r.acc[i].y = fmaf(f, v[j][i].y, r.acc[i].y);
        r.acc[i].z = fmaf(f, v[j][i].z, r.acc[i].z); r.acc[i].w = fmaf(f, v[j][i].w, r.acc[i].w);
      }
    }
  }
  return r;
}

// The pieces of items that no CTA had the whole of; zeros for a sequence without a token.
//  kByItem: a CTA per (row, key head and chunk), a warp per query head: where there are items for every SM, they have few pieces
//  otherwise a CTA per (row, query head), whose warps take every fourth piece
template <typename T, bool kByItem>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const DecodeArgs a, int heads_per_item) {
  constexpr int kMaxWords = 64;             // 16-byte words of a head of 256
  __shared__ float4 outs[kWarps][kMaxWords];
  __shared__ float sums[kWarps], tops[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = a.D / 4;
  const int row = blockIdx.y;
  int item, h0, heads, head0;               // within the row's items; query heads of this CTA in the item; its first query head
  if constexpr (kByItem) {
    item = blockIdx.x;
    const int kv_head = item / a.chunks, in_group = (item - kv_head * a.chunks) * heads_per_item;
    h0 = 0;
    heads = min(heads_per_item, a.group - in_group);
    head0 = kv_head * a.group + in_group;
  } else {
    head0 = blockIdx.x;
    const int kv_head = head0 / a.group, in_group = head0 - kv_head * a.group, chunk = in_group / heads_per_item;
    item = kv_head * a.chunks + chunk;
    h0 = in_group - chunk * heads_per_item;
    heads = 1;
  }
  T* out = static_cast<T*>(a.out) + (int64_t(row) * a.q_heads + head0) * a.D;
  const int units = units_of(a, row);
  if (units == 0) {
    wait_for_previous();
    for (int i = threadIdx.x; i < heads * a.D; i += kThreads) out[i] = from_f32<T>(0.f);
    return;
  }
  const int per = a.kv_heads * a.chunks;
  int64_t total = 0, before = 0;
  for (int i = lane; i < a.rows; i += 32) {
    const int64_t n = int64_t(units_of(a, i)) * per;
    total += n;
    if (i < row) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const Share share(a, total);
  const int64_t begin = before + int64_t(item) * units;
  const int w0 = share.worker_of(begin), w1 = share.worker_of(begin + units - 1);
  wait_for_previous();      // (the lengths are the caller's: what is above needs no wait)
  if (w0 == w1) return;     // finished by the CTA that had all of it
  const int64_t step = int64_t(heads_per_item) * (a.D + 4);
  // the first piece begins the item (slot 1 of its worker); the others begin inside it (slot 0)
  auto piece_of = [&](int h) {
    return [&, h](int w) { return a.part + (2 * int64_t(w) + (w == w0 ? 1 : 0)) * step + h * (a.D + 4); };
  };
  if constexpr (kByItem) {
    for (int h = warp; h < heads; h += kWarps) {
      const Joined r = join_pieces(w0, w1, 1, a.D, piece_of(h));
      const float inv = 1.f / r.sum;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (lane + 32 * i >= words) continue;
        T* to = out + h * a.D + (lane + 32 * i) * 4;
        to[0] = from_f32<T>(r.acc[i].x * inv); to[1] = from_f32<T>(r.acc[i].y * inv);
        to[2] = from_f32<T>(r.acc[i].z * inv); to[3] = from_f32<T>(r.acc[i].w * inv);
      }
    }
  } else {
    const Joined r = join_pieces(w0 + warp, w1, kWarps, a.D, piece_of(h0));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i < words) outs[warp][lane + 32 * i] = r.acc[i];
    if (lane == 0) {
      sums[warp] = r.sum;
      tops[warp] = r.top;
    }
    __syncthreads();
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) most = fmaxf(most, tops[i]);
    const float shift = most == -INFINITY ? 0.f : most;
    float f[kWarps], all = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      f[i] = ex2(tops[i] - shift);
      all = fmaf(f[i], sums[i], all);
    }
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) x = fmaf(f[i], reinterpret_cast<const float*>(outs[i])[d], x);
      out[d] = from_f32<T>(x / all);
    }
  }
}

template <typename T, typename Loop, int kSide, typename Args>
int launch_side(const Args& a, cudaStream_t st) {
  const size_t smem = size_t(kWarps) * Loop::kSlots * slot_stride<Loop>(a.D) * sizeof(float);
  if (Loop::kRing > 0 && cudaFuncSetAttribute(decode_kernel<T, Loop, kSide, Args>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
    return check_launch(Loop::kName);
  decode_kernel<T, Loop, kSide, Args><<<unsigned(a.workers), kThreads, smem, st>>>(a);
  count_launch();
  if (int rc = check_launch(Loop::kName)) return rc;
  const int items = a.kv_heads * a.chunks;      // of a row
  const bool by_item = int64_t(items) * a.rows >= tc::sm_count();
  if (launch_dependent(by_item ? decode_join_kernel<T, true> : decode_join_kernel<T, false>, dim3(unsigned(by_item ? items : a.q_heads), unsigned(a.rows)),
                       kThreads, 0, st, static_cast<const DecodeArgs&>(a), kSide * Loop::kHeads) != cudaSuccess)
    return check_launch("decode_join_kernel");
  count_launch();
  return check_launch("decode_join_kernel");
}

// (loops of few query heads take the whole of a group that small)
template <typename T, typename Loop, bool kWholeGroup, typename Args>
int launch(const Args& a, int side, cudaStream_t st) {
  if constexpr (!kWholeGroup) {
    if (side == 2) return launch_side<T, Loop, 2>(a, st);
    if (side == 4) return launch_side<T, Loop, 4>(a, st);
  }
  return launch_side<T, Loop, 1>(a, st);
}

}  // namespace
}  // namespace nb200
