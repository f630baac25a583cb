// The paged key / value cache: append, fork (and free), compact.
//
// All bookkeeping runs on the device, so that a generation step needs no host round trip and can be captured into a graph.
// It is whole numbers throughout and has one outcome whatever the order in which CTAs run: pages are given out in the free
// list's order to the sequences in order, lists are ascending.  Every page index and position is checked before it is used.
//
// Bound by HBM where tokens or pages are moved (each read and written once, in 16-byte words with eight in flight per
// thread), by launches and latency where a step adds one token per sequence: append is ONE launch, in which every warp finds
// its tokens' sequence and the number of pages that the sequences before it take by one pass over `offsets` and `lengths`;
// fork is a memset and two launches, compact a memset and three, each set up while the one before runs.  33 k tokens of bf16, 8
// heads of 128, 50 us (5.5 TB/s); 2100 pages of 64 KB moved among 8300, 60 us (4.5 TB/s), 48 of them the moves; 256 single tokens 7.6 and
// a fork of 64 rows 10.5 in a captured graph, 15 and 21 where the host makes the calls.
//
// Tokens for a cache in few bits are quantised on the way (cache_codes.cuh): 34 k tokens of bf16, 8 heads of 128, into 4 bits in 42 us (39
// by itself), 4.3 TB/s of what is read and written; two thirds of the issue slots are busy, with 47 instructions for a lane's 8 elements
// and some 300 for a token's place.  On the way: one group a lane and 16-bit stores of codes 78 us, steps worked out by every lane of a
// group 52, three CTAs per SM without spills 49, places in 64 bits and elements asked for when the place is known 45; four tokens a warp
// 46.  The same in fp32: 49 (6.4 TB/s); 78 with two CTAs per SM and loads past L1, which holds a sector's other half for the second load.
#include <algorithm>

#include "cache_codes.cuh"
#include "dependent_launch.cuh"
#include "sm100_primitives.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;

// Pages as 16-byte words.
struct Pages {
  uint4* k;
  uint4* v;
  int64_t ks[3], vs[3];     // words, over (page, head, slot)
  int pages, heads, page_size, words;   // words of a head's row
};

// The steps of a cache in few bits.
struct StepPages {
  uint16_t* k;
  uint16_t* v;
  int64_t ks[3], vs[3];     // elements, over (page, head, slot)
  int groups;               // of a head's row
};

// ---- append ---------------------------------------------------------------------------------------------------------------
struct AppendArgs {
  Pages p;
  int* table;
  const int* lengths;
  const int* offsets;
  const int* free_pages;
  const int* free_range;
  int rows, width;
  int* new_lengths;
  int* new_free_range;
  int* shortfall;
  const uint4* k;
  const uint4* v;
  int64_t ks[2], vs[2];     // words, over (token, head)
  int tokens, tokens_per_warp;
  int capacity;             // tokens that a row of the table has places for
  StepPages steps;
  // Strides where tokens are quantised, of keys and values, so that an offset is one wide multiply-add each: of codes and tokens in
  // 16-byte words, of steps in rows, over (page, head, slot) and (token, head).
  int codes_stride[2][3], steps_stride[2][3], from_stride[2][2];
};

struct RowPlan {
  int held, want, have, need;   // tokens held and to be held, pages held and asked for
};

// Offsets that leave the tokens are cut to them.
__device__ __forceinline__ int first_of(const AppendArgs& a, int row) { return min(max(a.offsets[row], 0), a.tokens); }

__device__ __forceinline__ RowPlan plan_row(const AppendArgs& a, int row) {
  RowPlan r;
  const int lo = first_of(a, row), hi = first_of(a, row + 1);
  r.held = min(max(a.lengths[row], 0), a.capacity);
  r.want = int(min(unsigned(r.held) + unsigned(max(hi - lo, 0)), unsigned(NB200_CACHE_MOST_TOKENS)));
  r.have = int((unsigned(r.held) + unsigned(a.p.page_size - 1)) / unsigned(a.p.page_size));      // (below 2^32)
  const int pages = int((unsigned(r.want) + unsigned(a.p.page_size - 1)) / unsigned(a.p.page_size));
  r.need = max(min(pages, a.width) - r.have, 0);
  return r;
}

// The pages given to a row when `before` have gone to the rows before it, and the tokens it then holds.
__device__ __forceinline__ int pages_got(const RowPlan& r, int64_t avail, int64_t before) {
  return int(min(max(avail - before, int64_t(0)), int64_t(r.need)));
}
__device__ __forceinline__ int tokens_kept(const RowPlan& r, int got, int page_size) {
  return int(min(int64_t(r.want), (int64_t(r.have) + got) * page_size));
}

__device__ __forceinline__ void free_bounds(const int* range, int pages, int* begin, int* end) {
  *begin = min(max(range[0], 0), pages);
  *end = min(max(range[1], *begin), pages);
}

// A token that is quantised, by a warp.  With kGroups, those of a head's row, a lane takes 8 elements of each of them, so that its
// codes lie side by side; otherwise, for any number of groups, 8 elements.  Four lanes share a group's elements.
template <int kBits, typename T, int kGroups>
struct Quantizer {
  static constexpr int kWords = sizeof(T) == 4 ? 2 : 1, kEach = kGroups ? kGroups : 1;
  uint4 x[2][kEach][kWords];      // of the lane's first elements of the token that comes next

  // the lane's head and place within its row at a turn that begins with w0 (whole warps go round together: a group's lanes exchange
  // their maxima)
  struct Turn {
    int n, h, c;
    __device__ __forceinline__ Turn(const AppendArgs& a, int w0) {
      const int lane = threadIdx.x & 31, units = (kGroups ? kGroups : a.steps.groups) * 4 / kEach;
      n = a.p.heads * units;
      const int w = min(w0 + lane, n - 4 + (lane & 3));      // (n is a multiple of 4)
      h = w / units;
      c = w - h * units;
    }
  };
  __device__ __forceinline__ void load(const AppendArgs& a, int t, const Turn& at) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint4* from = (which ? a.v : a.k) + int64_t(t) * a.from_stride[which][0] + int64_t(at.h) * a.from_stride[which][1] + at.c * kWords;
#pragma unroll
      for (int g = 0; g < kEach; ++g)
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[which][g][i] = kWords == 1 ? sm100::ldg_no_allocate(from + g * 4 * kWords + i) : __ldg(from + g * 4 * kWords + i);
    }
  }
  __device__ __forceinline__ void load(const AppendArgs& a, int t) { load(a, t, Turn(a, 0)); }
  __device__ __forceinline__ void store(const AppendArgs& a, int t, int page, int slot) {
    const int lane = threadIdx.x & 31, u = lane & 3, groups = kGroups ? kGroups : a.steps.groups;
    Turn at(a, 0);
    for (int w0 = 0;;) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int (&cs)[3] = a.codes_stride[which], (&ss)[3] = a.steps_stride[which];
        const Quantized<kBits, kEach> q = quantize<kBits, T, kEach>(x[which]);
        if (w0 + lane >= at.n) continue;
        uint8_t* codes = reinterpret_cast<uint8_t*>((which ? a.p.v : a.p.k) + int64_t(page) * cs[0] + int64_t(at.h) * cs[1] + int64_t(slot) * cs[2]);
        uint16_t* steps = (which ? a.steps.v : a.steps.k) + (int64_t(page) * ss[0] + int64_t(at.h) * ss[1] + int64_t(slot) * ss[2]) * groups;
        if constexpr (kGroups > 0) {
          store_quarter<kBits, kGroups>(codes, u, q);
          const int g = q.step_of(u);
          if (u == q.first_lane(g)) steps[g] = q.step;
        } else {
          store_codes(codes, groups, at.c >> 2, u, q);
          if (u == 0) steps[at.c >> 2] = q.step;
        }
      }
      w0 += 32;
      if (w0 >= at.n) return;
      at = Turn(a, w0);
      load(a, t, at);
    }
  }
};
// A token that is copied.
struct Copier {
  __device__ __forceinline__ void load(const AppendArgs&, int) {}
  __device__ __forceinline__ void store(const AppendArgs& a, int t, int page, int slot) {
    uint4* kd = a.p.k + page * a.p.ks[0] + slot * a.p.ks[2];
    uint4* vd = a.p.v + page * a.p.vs[0] + slot * a.p.vs[2];
    const uint4* kx = a.k + int64_t(t) * a.ks[0];
    const uint4* vx = a.v + int64_t(t) * a.vs[0];
    const int n = a.p.heads * a.p.words;
    for (int w0 = threadIdx.x & 31; w0 < n; w0 += 128) {
      uint4 kw[4], vw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int w = w0 + 32 * i, h = w / a.p.words, c = w - h * a.p.words;
        if (w < n) {
          kw[i] = __ldg(kx + h * a.ks[1] + c);
          vw[i] = __ldg(vx + h * a.vs[1] + c);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int w = w0 + 32 * i, h = w / a.p.words, c = w - h * a.p.words;
        if (w < n) {
          kd[h * a.p.ks[1] + c] = kw[i];
          vd[h * a.p.vs[1] + c] = vw[i];
        }
      }
    }
  }
};

// Tokens t0 .. t1, by a warp.  Where one comes from does not depend on where it goes: its elements are on their way meanwhile.
template <typename Token>
__device__ __forceinline__ void append_tokens(const AppendArgs& a, int begin, int64_t avail, int t0, int t1) {
  const int lane = threadIdx.x & 31;
  if (t0 >= t1) return;
  Token token;
  token.load(a, t0);
  int row = -1, next = 0, first = 0, got = 0, before = 0;
  RowPlan r{0, 0, 0, 0};
  for (int t = t0;;) {
    if (row < 0 || t >= next) {
      // the token's sequence, and the pages that those before it take
      int count = 0;
      int64_t need = 0;
      bool descend = false;
      for (int i = lane; i < a.rows; i += 32) {
        descend = descend || a.offsets[i] > a.offsets[i + 1];
        if (a.offsets[i + 1] <= t) {
          ++count;
          need += plan_row(a, i).need;
        }
      }
      // (more than there are free pages is as good as all of them, and fits 32 bits; a sum of 32 such numbers takes two)
      const unsigned few = unsigned(min(need, avail));
      need = int64_t(__reduce_add_sync(0xffffffffu, few & 0xffffu)) + (int64_t(__reduce_add_sync(0xffffffffu, few >> 16)) << 16);
      row = __reduce_add_sync(0xffffffffu, count);
      if (row >= a.rows || __any_sync(0xffffffffu, descend)) return;     // (tokens behind the last offset)
      r = plan_row(a, row);
      first = first_of(a, row);
      next = a.offsets[row + 1];
      got = pages_got(r, avail, need);
      before = int(min(need, avail));
    }
    int page = -1, slot = 0;
    const unsigned pos = unsigned(r.held) + unsigned(t - first);
    if (t >= first && pos < unsigned(tokens_kept(r, got, a.p.page_size))) {
      const int column = int(pos / unsigned(a.p.page_size));
      slot = int(pos) - column * a.p.page_size;
      if (column >= r.have) {
        page = a.free_pages[begin + before + column - r.have];
        if (slot == 0 && lane == 0) a.table[int64_t(row) * a.width + column] = page;
      } else if (column < a.width) {
        page = a.table[int64_t(row) * a.width + column];
      }
    }
    if (page >= 0 && page < a.p.pages) token.store(a, t, page, slot);
    if (++t >= t1) return;
    token.load(a, t);
  }
}

// kBits 0: the tokens' rows are copied; otherwise T is their type.
template <int kBits, typename T>
__global__ void __launch_bounds__(kThreads, kBits == 0 || sizeof(T) == 4 ? 3 : 4) cache_append_kernel(const AppendArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int begin, end;
  free_bounds(a.free_range, a.p.pages, &begin, &end);
  const int64_t avail = end - begin;
  if (blockIdx.x == 0) {
    // the state after the call: one CTA, 256 rows at a time
    __shared__ int64_t part[kThreads / 32];
    __shared__ unsigned long long dropped;
    if (threadIdx.x == 0) dropped = 0;
    // (offsets that descend name no row's tokens: every row keeps what it holds, as the other CTAs store nothing)
    bool descend = false;
    for (int row = threadIdx.x; row < a.rows; row += kThreads) descend = descend || a.offsets[row] > a.offsets[row + 1];
    descend = __syncthreads_or(descend);
    int64_t before = 0;
    for (int row0 = 0; row0 < a.rows; row0 += kThreads) {
      const int row = row0 + threadIdx.x;
      RowPlan r{0, 0, 0, 0};
      if (row < a.rows) r = plan_row(a, row);
      if (descend) r = RowPlan{r.held, r.held, r.have, 0};
      int64_t upto = r.need;      // inclusive sum over the warp, then over the warps before
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      __syncthreads();
      if (lane == 31) part[warp] = upto;
      __syncthreads();
      int64_t total = 0;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) upto += part[w];
        total += part[w];
      }
      if (row < a.rows) {
        const int kept = tokens_kept(r, pages_got(r, avail, before + upto - r.need), a.p.page_size);
        a.new_lengths[row] = kept;
        const int64_t asked = descend ? 0 : int64_t(a.offsets[row + 1]) - a.offsets[row], stored = max(kept - r.held, 0);
        if (asked > stored) atomicAdd(&dropped, static_cast<unsigned long long>(asked - stored));
      }
      before += total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      a.new_free_range[0] = begin + int(min(before, avail));
      a.new_free_range[1] = end;
      *a.shortfall = int(min(descend ? static_cast<unsigned long long>(a.tokens) : dropped, 0x7fffffffull));
    }
    return;
  }
  const int t0 = int(min((int64_t(blockIdx.x - 1) * (kThreads / 32) + warp) * a.tokens_per_warp, int64_t(a.tokens)));
  const int t1 = t0 + min(a.tokens_per_warp, a.tokens - t0);
  if constexpr (kBits == 0) append_tokens<Copier>(a, begin, avail, t0, t1);
  else if (a.steps.groups == 4) append_tokens<Quantizer<kBits, T, 4>>(a, begin, avail, t0, t1);
  else if (a.steps.groups == 2) append_tokens<Quantizer<kBits, T, 2>>(a, begin, avail, t0, t1);
  else append_tokens<Quantizer<kBits, T, 0>>(a, begin, avail, t0, t1);
}

// ---- fork and compact -----------------------------------------------------------------------------------------------------
// Workspace: [0] dropped tokens, [1] pages to move, [2 .. 4) unused, then one bit per page (live), then (compact) the live pages
// before each word of bits, the free pages in ascending order, the live pages that move in ascending order.
struct Layout {
  int words;                                  // of 32 pages
  size_t bits, before, holes, moves, total;   // offsets in ints
};
Layout layout(int pages) {
  Layout l{};
  l.words = (pages + 31) / 32;
  l.bits = 4;
  l.before = l.bits + size_t(l.words);
  l.holes = l.before + size_t(l.words);
  l.moves = l.holes + size_t(pages);
  l.total = l.moves + size_t(pages);
  return l;
}

struct MoveArgs {
  Pages p;
  StepPages steps;
  const int* table;
  const int* lengths;
  const int* free_pages;
  const int* free_range;
  int rows, width, new_rows;
  const int* parents;
  const uint8_t* finished;
  int* new_table;
  int* new_lengths;
  int* new_free_pages;
  int* new_free_range;
  int* shortfall;
  int* dropped;
  unsigned* bits;
  int* before;
  int* holes;
  int* moves;
  int* n_moves;
};

__device__ __forceinline__ int parent_of(const MoveArgs& a, int row) {
  const int parent = a.parents ? a.parents[row] : (a.finished[row] ? -1 : row);
  return parent >= 0 && parent < a.rows ? parent : -1;
}
// tokens of a row, of which a table of this width can hold the pages
__device__ __forceinline__ int64_t held_by(const MoveArgs& a, int row) {
  return min(int64_t(max(a.lengths[row], 0)), int64_t(a.width) * a.p.page_size);
}
__device__ __forceinline__ void mark(const MoveArgs& a, int page) {
  if (page >= 0 && page < a.p.pages) atomicOr(a.bits + (page >> 5), 1u << (page & 31));
}

// `slots` slots of every head of a page, by the CTAs `part` of `parts`: rows of `words` units, strides in units
template <typename U>
__device__ __forceinline__ void copy_rows(U* k, U* v, const int64_t (&ks)[3], const int64_t (&vs)[3], int heads, int words, int src, int dst, int slots,
                                          int part, int parts) {
  const int per_head = slots * words, n = heads * per_head, stride = parts * kThreads;
  for (int i0 = part * kThreads + int(threadIdx.x); i0 < n; i0 += 4 * stride) {
    U kw[4], vw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * stride, h = i / per_head, rem = i - h * per_head, s = rem / words, c = rem - s * words;
      if (i < n) {
        kw[j] = __ldcs(k + src * ks[0] + h * ks[1] + s * ks[2] + c);
        vw[j] = __ldcs(v + src * vs[0] + h * vs[1] + s * vs[2] + c);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * stride, h = i / per_head, rem = i - h * per_head, s = rem / words, c = rem - s * words;
      if (i < n) {
        k[dst * ks[0] + h * ks[1] + s * ks[2] + c] = kw[j];
        v[dst * vs[0] + h * vs[1] + s * vs[2] + c] = vw[j];
      }
    }
  }
}
// (rows of steps begin at multiples of their size: as the largest words that this allows)
template <typename U>
__device__ __forceinline__ void copy_steps(const StepPages& p, int heads, int src, int dst, int slots, int part, int parts) {
  constexpr int n = int(sizeof(U)) / 2;
  const int64_t ks[3] = {p.ks[0] / n, p.ks[1] / n, p.ks[2] / n}, vs[3] = {p.vs[0] / n, p.vs[1] / n, p.vs[2] / n};
  copy_rows(reinterpret_cast<U*>(p.k), reinterpret_cast<U*>(p.v), ks, vs, heads, p.groups / n, src, dst, slots, part, parts);
}
template <bool kSteps>
__device__ __forceinline__ void copy_page(const MoveArgs& a, int src, int dst, int slots, int part, int parts) {
  copy_rows(a.p.k, a.p.v, a.p.ks, a.p.vs, a.p.heads, a.p.words, src, dst, slots, part, parts);
  if constexpr (kSteps) {
    if (a.steps.groups % 4 == 0) copy_steps<uint2>(a.steps, a.p.heads, src, dst, slots, part, parts);
    else if (a.steps.groups % 2 == 0) copy_steps<uint32_t>(a.steps, a.p.heads, src, dst, slots, part, parts);
    else copy_steps<uint16_t>(a.steps, a.p.heads, src, dst, slots, part, parts);
  }
}

// One row of the result per blockIdx.x, its page copy in gridDim.y parts.  A row's rank among the rows that copy is the number
// of rows before it with an open page less the number of their distinct parents, which a bit per parent counts.
template <bool kSteps>
__global__ void __launch_bounds__(kThreads) cache_fork_rows_kernel(const MoveArgs a) {
  extern __shared__ unsigned seen[];       // one bit per row of the old table
  allow_dependents();
  __shared__ int open_rows, distinct;
  const int row = blockIdx.x, words = (a.rows + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kThreads) seen[i] = 0;
  if (threadIdx.x == 0) open_rows = distinct = 0;
  __syncthreads();
  const int parent = parent_of(a, row);
  const int64_t held = parent < 0 ? 0 : held_by(a, parent);
  const int full = int(held / a.p.page_size), part = int(held - int64_t(full) * a.p.page_size);
  int mine = 0;
  bool same = false;
  for (int i = threadIdx.x; i < row; i += kThreads) {
    const int other = parent_of(a, i);
    if (other < 0) continue;
    same = same || other == parent;
    if (part > 0 && held_by(a, other) % a.p.page_size != 0) {
      ++mine;
      atomicOr(seen + (other >> 5), 1u << (other & 31));
    }
  }
  const bool first = !__syncthreads_or(same);
  int bits = 0;
  for (int i = threadIdx.x; i < words; i += kThreads) bits += __popc(seen[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mine += __shfl_xor_sync(0xffffffffu, mine, o);
    bits += __shfl_xor_sync(0xffffffffu, bits, o);
  }
  if ((threadIdx.x & 31) == 0) {
    atomicAdd(&open_rows, mine);
    atomicAdd(&distinct, bits);
  }
  __syncthreads();
  const bool copies = part > 0 && !first;
  const int rank = open_rows - distinct;
  int begin, end;
  free_bounds(a.free_range, a.p.pages, &begin, &end);
  const bool served = copies && rank < end - begin;
  const int fresh = served ? a.free_pages[begin + rank] : -1;
  const int kept = copies && !served ? 0 : part;      // tokens of the open page
  const int pages = full + (kept > 0 ? 1 : 0);
  const int* from = a.table + int64_t(parent < 0 ? 0 : parent) * a.width;
  if (blockIdx.y == 0) {
    int* to = a.new_table + int64_t(row) * a.width;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const int page = c >= pages ? -1 : served && c == full ? fresh : from[c];
      to[c] = page;
      // (pages that are shared are marked by the first child)
      if (c < pages && (first || c == full)) mark(a, page);
    }
    if (threadIdx.x == 0) {
      a.new_lengths[row] = int(int64_t(full) * a.p.page_size + kept);
      if (part > kept) atomicAdd(a.dropped, part - kept);
    }
  }
  if (served) {
    const int src = from[full];
    if (src >= 0 && src < a.p.pages && fresh >= 0 && fresh < a.p.pages) copy_page<kSteps>(a, src, fresh, part, blockIdx.y, gridDim.y);
  }
}

__global__ void __launch_bounds__(kThreads) cache_mark_kernel(const MoveArgs a) {
  allow_dependents();
  const int row = blockIdx.x;
  const int pages = int((held_by(a, row) + a.p.page_size - 1) / a.p.page_size);
  for (int c = threadIdx.x; c < pages; c += kThreads) mark(a, a.table[int64_t(row) * a.width + c]);
}

constexpr int kListWords = 64;      // words of bits per CTA of the listing kernel

// The pages without a bit, ascending, -1 behind them.  Every CTA counts the bits before its own anew, which costs a reading of
// the bits (32 KB for 256 K pages) and saves a launch.  For compact: also the live pages before each word, and the live pages
// that have to move, which are those at or behind the number of live ones.
template <bool kCompact>
__global__ void __launch_bounds__(kThreads) cache_list_kernel(const MoveArgs a, int words, int* list, int* range) {
  __shared__ int sums[3];
  allow_dependents();
  wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w0 = blockIdx.x * kListWords;
  if (threadIdx.x < 3) sums[threadIdx.x] = 0;
  __syncthreads();
  int earlier = 0, all = 0;
  for (int w = threadIdx.x; w < words; w += kThreads) {
    const int n = __popc(a.bits[w]);
    all += n;
    if (w < w0) earlier += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    earlier += __shfl_xor_sync(0xffffffffu, earlier, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    atomicAdd(&sums[0], earlier);
    atomicAdd(&sums[1], all);
  }
  __syncthreads();
  const int live = sums[1], n_free = a.p.pages - live;
  int stay = 0;             // live pages in front of the live-th
  if constexpr (kCompact) {
    for (int w = threadIdx.x; w <= live >> 5 && w < words; w += kThreads) stay += __popc(a.bits[w] & (w < live >> 5 ? ~0u : (1u << (live & 31)) - 1u));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) stay += __shfl_xor_sync(0xffffffffu, stay, o);
    if (lane == 0) atomicAdd(&sums[2], stay);
    __syncthreads();
    stay = sums[2];
  }
  int base = sums[0];       // live pages before word w0; then before word w
  for (int w = w0; w < min(w0 + kListWords, words); ++w) {
    const unsigned word = a.bits[w];
    if (((w - w0) & (kThreads / 32 - 1)) == warp) {
      const int page = w * 32 + lane;
      if (kCompact && lane == 0) a.before[w] = base;
      if (page < a.p.pages) {
        const int rank = base + __popc(word & ((1u << lane) - 1u));      // live pages before this one
        if (!((word >> lane) & 1u)) list[page - rank] = page;
        else if (kCompact && page >= live) a.moves[rank - stay] = page;
        if (page >= n_free) list[page] = -1;
      }
    }
    base += __popc(word);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    range[0] = 0;
    range[1] = n_free;
    *a.shortfall = *a.dropped;
    if (kCompact) *a.n_moves = live - stay;
  }
}

// Live pages at or behind the number of live pages go to the lowest free ones, in order: free pages are the only ones
// written, live ones the only ones read, so that moves cannot meet.
template <bool kSteps>
__global__ void __launch_bounds__(kThreads) cache_move_kernel(const MoveArgs a, int parts) {
  wait_for_previous();
  const int n_free = a.new_free_range[1], live = a.p.pages - n_free, kept = live - *a.n_moves;      // kept: live pages that stay
  auto live_before = [&](int page) { return a.before[page >> 5] + __popc(a.bits[page >> 5] & ((1u << (page & 31)) - 1u)); };
  auto moved_to = [&](int page) { return page < live ? page : a.holes[live_before(page) - kept]; };
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int pages = int((held_by(a, row) + a.p.page_size - 1) / a.p.page_size);
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const int page = c < pages ? a.table[int64_t(row) * a.width + c] : -1;
      a.new_table[int64_t(row) * a.width + c] = page >= 0 && page < a.p.pages ? moved_to(page) : page;
    }
  }
  // a page in `parts` parts, all parts of all pages dealt to the CTAs in turn
  const int n = *a.n_moves * parts;
  for (int i = blockIdx.x; i < n; i += gridDim.x) copy_page<kSteps>(a, a.moves[i / parts], a.holes[i / parts], a.p.page_size, i % parts, parts);
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < a.p.pages; i += gridDim.x * kThreads)
    a.new_free_pages[i] = i < n_free ? live + i : -1;
}

// `steps`: of a cache in few bits, whose pages hold codes; otherwise NULL
int check_pages(const nb200_cache_pages& c, const nb200_cache_steps* steps, const char* what, Pages* out) {
  if (c.dtype != NB200_F32 && c.dtype != NB200_BF16 && c.dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (c.pages < 0 || c.heads <= 0 || c.page_size <= 0 || c.head_dim <= 0 || (c.pages && (!c.k || !c.v))) {
    set_error("%s: bad extents of the pages, or NULL pages", what);
    return NB200_ERR_INVALID;
  }
  if (steps)
    if (int rc = check_steps(c, *steps, what)) return rc;
  const int vec = steps ? 16 : c.dtype == NB200_F32 ? 4 : 8;      // elements of a word, bytes of codes
  const int row = steps ? c.head_dim / 8 * steps->bits : c.head_dim;
  bool ok = row % vec == 0 && aligned16(c.k) && aligned16(c.v);
  for (int i = 0; i < 3; ++i) ok = ok && c.k_stride[i] % vec == 0 && c.v_stride[i] % vec == 0;
  if (!ok) { set_error("%s: the rows of the pages must begin on 16-byte boundaries", what); return NB200_ERR_ALIGNMENT; }
  if (int64_t(c.heads) * c.page_size * (row / vec) > 0x3fffffff) { set_error("%s: pages too large", what); return NB200_ERR_UNSUPPORTED; }
  out->k = static_cast<uint4*>(c.k);
  out->v = static_cast<uint4*>(c.v);
  for (int i = 0; i < 3; ++i) {
    out->ks[i] = c.k_stride[i] / vec;
    out->vs[i] = c.v_stride[i] / vec;
  }
  out->pages = c.pages; out->heads = c.heads; out->page_size = c.page_size; out->words = row / vec;
  return NB200_OK;
}

StepPages step_pages(const nb200_cache_pages& c, const nb200_cache_steps* s) {
  StepPages p{};
  if (!s) return p;
  p.k = static_cast<uint16_t*>(s->k);
  p.v = static_cast<uint16_t*>(s->v);
  for (int i = 0; i < 3; ++i) { p.ks[i] = s->k_stride[i]; p.vs[i] = s->v_stride[i]; }
  p.groups = c.head_dim / kGroup;
  return p;
}

int check_state(const nb200_cache_params* p, const nb200_cache_steps* steps, const char* what, Pages* pages) {
  if (!p || p->struct_size != sizeof(nb200_cache_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  if (int rc = check_pages(p->pages, steps, what, pages)) return rc;
  if (p->rows < 0 || p->width <= 0) { set_error("%s: bad extents of the table", what); return NB200_ERR_INVALID; }
  if ((p->rows && (!p->table || !p->lengths)) || !p->free_range || (p->pages.pages && !p->free_pages)) {
    set_error("%s: NULL table, lengths, free_pages or free_range", what);
    return NB200_ERR_INVALID;
  }
  return NB200_OK;
}

int move_args(const nb200_cache_params* p, const nb200_cache_steps* steps, const char* what, const Pages& pages, MoveArgs* a, Layout* l, cudaStream_t st) {
  *l = layout(pages.pages);
  if (!p->workspace || p->workspace_bytes < l->total * sizeof(int)) {
    set_error("%s: workspace of %zu bytes needed (nb200_cache_workspace_bytes), %zu given", what, l->total * sizeof(int), p->workspace_bytes);
    return NB200_ERR_WORKSPACE;
  }
  int* ws = static_cast<int*>(p->workspace);
  *a = MoveArgs{};
  a->p = pages;
  a->steps = step_pages(p->pages, steps);
  a->table = p->table; a->lengths = p->lengths; a->free_pages = p->free_pages; a->free_range = p->free_range;
  a->rows = p->rows; a->width = p->width; a->new_rows = p->new_rows;
  a->new_table = p->new_table; a->new_lengths = p->new_lengths;
  a->new_free_pages = p->new_free_pages; a->new_free_range = p->new_free_range;
  a->dropped = ws;
  a->bits = reinterpret_cast<unsigned*>(ws + l->bits);
  a->before = ws + l->before;
  a->holes = ws + l->holes;
  a->moves = ws + l->moves;
  a->n_moves = ws + 1;
  if (cudaMemsetAsync(ws, 0, (l->bits + size_t(l->words)) * sizeof(int), st) != cudaSuccess) return check_launch("cache: clearing the workspace");
  return NB200_OK;
}

// parts that a page is copied in: 32 KB of keys and values, which eight words in flight per thread cover in one turn
int page_parts(const Pages& p) {
  const int64_t bytes = int64_t(p.heads) * p.page_size * p.words * 32;
  return int(bytes <= 32768 ? 1 : bytes >= 16 * 32768 ? 16 : (bytes + 32767) / 32768);
}

unsigned list_grid(const Layout& l) { return l.words ? unsigned((l.words + kListWords - 1) / kListWords) : 1u; }

int append(const nb200_cache_params* p, const nb200_cache_steps* steps, const char* what, void* cuda_stream) {
  AppendArgs a{};
  if (int rc = check_state(p, steps, what, &a.p)) return rc;
  if (p->rows == 0) { set_error("%s: no rows", what); return NB200_ERR_INVALID; }
  if (p->tokens < 0 || p->tokens > 0x7fffffff || !p->offsets || !p->new_lengths || !p->new_free_range || !p->shortfall ||
      (p->tokens && (!p->new_k || !p->new_v))) {
    set_error("%s: NULL operand or bad number of tokens", what);
    return NB200_ERR_INVALID;
  }
  const int vec = p->pages.dtype == NB200_F32 ? 4 : 8;
  bool ok = aligned16(p->new_k) && aligned16(p->new_v);
  for (int i = 0; i < 2; ++i) ok = ok && p->new_k_stride[i] % vec == 0 && p->new_v_stride[i] % vec == 0;
  if (!ok) { set_error("%s: the rows of k and v must begin on 16-byte boundaries", what); return NB200_ERR_ALIGNMENT; }
  a.table = p->table; a.lengths = p->lengths; a.offsets = p->offsets; a.free_pages = p->free_pages; a.free_range = p->free_range;
  a.rows = p->rows; a.width = p->width;
  a.new_lengths = p->new_lengths; a.new_free_range = p->new_free_range; a.shortfall = p->shortfall;
  a.k = static_cast<const uint4*>(p->new_k); a.v = static_cast<const uint4*>(p->new_v);
  for (int i = 0; i < 2; ++i) {
    a.ks[i] = p->new_k_stride[i] / vec;
    a.vs[i] = p->new_v_stride[i] / vec;
  }
  a.tokens = int(p->tokens);
  a.capacity = int(std::min<int64_t>(int64_t(p->width) * p->pages.page_size, NB200_CACHE_MOST_TOKENS));
  if (steps) {
    bool near = true;
    auto fits = [&](int64_t stride) { near = near && stride <= 0x7fffffff && stride >= -0x7fffffff; return int(stride); };
    const int groups = p->pages.head_dim / kGroup;
    for (int i = 0; i < 3; ++i) {
      a.codes_stride[0][i] = fits(a.p.ks[i]); a.codes_stride[1][i] = fits(a.p.vs[i]);
      a.steps_stride[0][i] = fits(steps->k_stride[i] / groups); a.steps_stride[1][i] = fits(steps->v_stride[i] / groups);
    }
    for (int i = 0; i < 2; ++i) { a.from_stride[0][i] = fits(a.ks[i]); a.from_stride[1][i] = fits(a.vs[i]); }
    if (!near) { set_error("%s: a stride of the pages or tokens is 2^31 words of 16 bytes, or rows of steps, or more", what); return NB200_ERR_UNSUPPORTED; }
  }
  // one token per warp while that does not fill the GPU's warps; then two, which share a sequence's search (33 k tokens of bf16,
  // 8 heads of 128: one 55.9 us, two 51.4, four 53.9, eight 60.2)
  a.tokens_per_warp = p->tokens < 148 * 64 ? 1 : 2;
  const int64_t per_cta = int64_t(a.tokens_per_warp) * (kThreads / 32);
  const unsigned grid = unsigned((p->tokens + per_cta - 1) / per_cta) + 1u;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  a.steps = step_pages(p->pages, steps);
  void (*kernel)(AppendArgs) = cache_append_kernel<0, uint4>;
  if (steps) {
    const bool four = steps->bits == 4;
    kernel = p->pages.dtype == NB200_F32    ? four ? cache_append_kernel<4, float> : cache_append_kernel<8, float>
             : p->pages.dtype == NB200_BF16 ? four ? cache_append_kernel<4, __nv_bfloat16> : cache_append_kernel<8, __nv_bfloat16>
             : four                         ? cache_append_kernel<4, __half> : cache_append_kernel<8, __half>;
  }
  kernel<<<grid, kThreads, 0, st>>>(a);
  count_launch();
  return check_launch(steps ? "cache_append_kernel<quantized>" : "cache_append_kernel");
}

int fork(const nb200_cache_params* p, const nb200_cache_steps* steps, const char* what, void* cuda_stream) {
  Pages pages;
  if (int rc = check_state(p, steps, what, &pages)) return rc;
  if (p->new_rows < 0 || !p->new_free_range || !p->shortfall || (pages.pages && !p->new_free_pages) ||
      (p->new_rows && (!p->new_table || !p->new_lengths || (!p->parents && !p->finished)))) {
    set_error("%s: NULL operand or bad number of rows", what);
    return NB200_ERR_INVALID;
  }
  if (p->new_rows && !p->parents && p->new_rows != p->rows) { set_error("%s: finished names %d rows of %d", what, p->new_rows, p->rows); return NB200_ERR_INVALID; }
  if (p->rows > 262144) { set_error("%s: %d rows, at most 262144", what, p->rows); return NB200_ERR_UNSUPPORTED; }   // bits in shared memory
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  MoveArgs a;
  Layout l;
  if (int rc = move_args(p, steps, what, pages, &a, &l, st)) return rc;
  a.parents = p->parents; a.finished = p->finished; a.shortfall = p->shortfall;
  if (p->new_rows > 0) {
    (steps ? cache_fork_rows_kernel<true> : cache_fork_rows_kernel<false>)<<<dim3(unsigned(p->new_rows), unsigned(page_parts(pages))), kThreads, size_t((p->rows + 31) / 32) * sizeof(unsigned), st>>>(a);
    count_launch();
    if (int rc = check_launch("cache_fork_rows_kernel")) return rc;
  }
  if (launch_dependent(cache_list_kernel<false>, list_grid(l), kThreads, 0, st, a, l.words, a.new_free_pages, a.new_free_range) != cudaSuccess)
    return check_launch("cache_list_kernel");
  count_launch();
  return check_launch("cache_list_kernel");
}

int compact(const nb200_cache_params* p, const nb200_cache_steps* steps, const char* what, void* cuda_stream) {
  Pages pages;
  if (int rc = check_state(p, steps, what, &pages)) return rc;
  if ((p->rows && !p->new_table) || (pages.pages && !p->new_free_pages) || !p->new_free_range || !p->shortfall) { set_error("%s: NULL operand", what); return NB200_ERR_INVALID; }
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  MoveArgs a;
  Layout l;
  if (int rc = move_args(p, steps, what, pages, &a, &l, st)) return rc;
  a.shortfall = p->shortfall;      // (nothing is dropped)
  if (p->rows > 0) {
    cache_mark_kernel<<<unsigned(p->rows), kThreads, 0, st>>>(a);
    count_launch();
    if (int rc = check_launch("cache_mark_kernel")) return rc;
  }
  if (launch_dependent(cache_list_kernel<true>, list_grid(l), kThreads, 0, st, a, l.words, a.holes, a.new_free_range) != cudaSuccess)
    return check_launch("cache_list_kernel");
  count_launch();
  if (int rc = check_launch("cache_list_kernel")) return rc;
  // a CTA per part of a page that may have to move, which half of the pages at most have
  const int parts = page_parts(pages);
  int64_t grid = int64_t(pages.pages + 1) / 2 * parts;
  if (grid < p->rows) grid = p->rows;
  grid = grid < 1 ? 1 : grid > 65536 ? 65536 : grid;
  if (launch_dependent(steps ? cache_move_kernel<true> : cache_move_kernel<false>, unsigned(grid), kThreads, 0, st, a, parts) != cudaSuccess) return check_launch("cache_move_kernel");
  count_launch();
  return check_launch("cache_move_kernel");
}

// A parameter block of a cache in few bits is one around the other cache's.
int check_quantized(const nb200_cache_quantized_params* p, const char* what) {
  if (p && p->struct_size == sizeof(nb200_cache_quantized_params)) return NB200_OK;
  set_error("%s: NULL params or wrong struct_size", what);
  return NB200_ERR_INVALID;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_cache_workspace_bytes(const nb200_cache_params* p, size_t* bytes) {
  if (!p || p->struct_size != sizeof(nb200_cache_params) || !bytes) { set_error("cache_workspace_bytes: NULL or wrong struct_size"); return NB200_ERR_INVALID; }
  if (p->pages.pages < 0) { set_error("cache_workspace_bytes: bad extents"); return NB200_ERR_INVALID; }
  *bytes = layout(p->pages.pages).total * sizeof(int);
  return NB200_OK;
}

extern "C" NB200_API int nb200_cache_append(const nb200_cache_params* p, void* cuda_stream) { return append(p, nullptr, "cache_append", cuda_stream); }
extern "C" NB200_API int nb200_cache_fork(const nb200_cache_params* p, void* cuda_stream) { return fork(p, nullptr, "cache_fork", cuda_stream); }
extern "C" NB200_API int nb200_cache_compact(const nb200_cache_params* p, void* cuda_stream) { return compact(p, nullptr, "cache_compact", cuda_stream); }

extern "C" NB200_API int nb200_cache_append_quantized(const nb200_cache_quantized_params* p, void* cuda_stream) {
  if (int rc = check_quantized(p, "cache_append_quantized")) return rc;
  return append(&p->cache, &p->steps, "cache_append_quantized", cuda_stream);
}
extern "C" NB200_API int nb200_cache_fork_quantized(const nb200_cache_quantized_params* p, void* cuda_stream) {
  if (int rc = check_quantized(p, "cache_fork_quantized")) return rc;
  return fork(&p->cache, &p->steps, "cache_fork_quantized", cuda_stream);
}
extern "C" NB200_API int nb200_cache_compact_quantized(const nb200_cache_quantized_params* p, void* cuda_stream) {
  if (int rc = check_quantized(p, "cache_compact_quantized")) return rc;
  return compact(&p->cache, &p->steps, "cache_compact_quantized", cuda_stream);
}
