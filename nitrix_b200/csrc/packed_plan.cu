// Work lists of the tensor-core kernels of attention over packed sequences.
//
// The lengths are in device memory, so the blocks of all sequences are listed there, by one CTA.  Two things decide their
// order.  CTAs that work on one sequence side by side share its keys in L2 (forward), or its queries and the sums of dq, which
// every key block adds to (backward: with all sequences' blocks sorted by length alone, 16 documents of up to 4096 tokens, the
// sums alone are 284 MB and the kernel takes 1252 us for 1054).  And the longest blocks of what is left should come first, so that
// short ones even out the end.  So the sequences, longest first, are cut into groups of at least one block per SM (two: 1078 us, three: 1089), and within a
// group the blocks are sorted by their length in tiles; blocks of one length come in any order, which changes no result.
// The other CTAs clear the outputs of tokens that belong to no sequence, and reduce what the fp16 backward wants the maxima of.
#include "dependent_launch.cuh"
#include "packed_tc.cuh"

namespace nb200 {
namespace packed {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kClearCtas = 31;
constexpr int kBuckets = 1024;         // group, then length
constexpr int kLengths = 64;           // of them per group, longest first
constexpr int kGroups = kBuckets / kLengths;
constexpr int kGroupItems = 148;       // (block, key head) pairs that a group has at least

struct PlanArgs {
  PackedArgs a;
  int backward;
  int halves;            // of an element of the outputs, 16 bits each
  int block, step_tokens;
  int shift;             // lengths in tiles are counted in units of 2^shift
  int kv_heads;
  int grouped;           // more than one group is possible
  // Entries and (backward) steps that there is room for: as many as sequences that follow one another have.  Offsets that run
  // backwards describe sequences that overlap, of which those that do not fit are left out.
  int most;
  int64_t most_steps;
  int* count;
  WorkItem* items;
};

// Blocks of a sequence.
__device__ __forceinline__ int blocks_of(const PlanArgs& p, int s) {
  const int n = p.backward ? sequence_span(p.a.offsets_k, s, p.a.tokens_k).y : sequence_span(p.a.offsets_q, s, p.a.tokens_q).y;
  return (n + p.block - 1) / p.block;
}

// Group of every sequence into `group`; up to kPlanThreads sequences (more of them are one group).
__device__ __forceinline__ void form_groups(const PlanArgs& p, uint8_t* group, int* blocks, int* sorted) {
  const int n = p.a.sequences, i = threadIdx.x, lane = i & 31, warp = i >> 5;
  __shared__ int sums[kPlanThreads / 32];
  if (i < n) blocks[i] = blocks_of(p, i);
  sorted[i] = 0;
  __syncthreads();
  int rank = 0;
  if (i < n) {
    const int mine = blocks[i];
    for (int j = 0; j < n; ++j) rank += blocks[j] > mine || (blocks[j] == mine && j < i) ? 1 : 0;
    sorted[rank] = mine;
  }
  __syncthreads();
  const int own = sorted[i];
  int64_t upto = own;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += other;
  }
  if (lane == 31) sums[warp] = int(upto);
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
  }
  const int64_t items = max(int64_t(kGroupItems), (total * p.kv_heads + kGroups - 1) / kGroups);
  sorted[i] = int(min((upto - own) * p.kv_heads / items, int64_t(kGroups - 1)));      // the group of rank i
  __syncthreads();
  if (i < n) group[i] = uint8_t(sorted[rank]);
  __syncthreads();
}

template <typename Visit>
__device__ __forceinline__ void for_each_block(const PlanArgs& p, const uint8_t* group, Visit visit) {
  const PackedArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t steps_before = 0;  // backward: 64-row steps of the sequences before, every warp for itself
  int at = 0;
  for (int s = warp; s < a.sequences; s += kPlanThreads / 32) {
    const int2 q = sequence_span(a.offsets_q, s, a.tokens_q), k = sequence_span(a.offsets_k, s, a.tokens_k);
    if (p.backward) {
      int64_t more = 0;
      for (int i = at + lane; i < s; i += 32) more += (sequence_span(a.offsets_q, i, a.tokens_q).y + p.step_tokens - 1) / p.step_tokens;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
      steps_before += more;
      at = s;
    }
    if (p.backward && steps_before + (q.y + p.step_tokens - 1) / p.step_tokens > p.most_steps) break;
    const int2 own = p.backward ? k : q, other = p.backward ? q : k;
    const int shift = k.y - q.y;       // query i sees keys up to i + shift
    for (int b = lane; int64_t(b) * p.block < own.y; b += 32) {
      WorkItem w;
      const int first = b * p.block;
      w.begin = own.x + first;
      w.n = min(p.block, own.y - first);
      w.other = other.x;
      w.other_n = other.y;
      w.steps = int(steps_before);
      w.index = b;
      w.sequence = s;
      int length;        // tokens of the other side
      if (p.backward) {
        w.seen = first - shift;
        length = other.y - (a.causal ? min(max(w.seen, 0), other.y) : 0);
      } else {
        w.seen = first + 1 + shift;
        length = a.causal ? min(max(w.seen + w.n - 1, 0), other.y) : other.y;
      }
      visit(w, (group ? group[s] : 0) * kLengths + kLengths - 1 - min((length / 128) >> p.shift, kLengths - 1));
    }
  }
}

// The largest of value(row) >= 0 over every sequence's rows, `heads` a token, into to[kMosts * sequence].  The tokens are dealt to the
// warps in contiguous shares, so that nobody looks a row's sequence up by itself.
template <typename Value>
__device__ __forceinline__ void raise_largest(const int* offsets, int sequences, int tokens, int heads, unsigned* to, Value value) {
  const int lane = threadIdx.x & 31, warps = kClearCtas * (kPlanThreads / 32);
  const int share = (tokens + warps - 1) / warps;
  const int64_t t0 = (int64_t(blockIdx.x - 1) * (kPlanThreads / 32) + (threadIdx.x >> 5)) * share;
  const int64_t t1 = min(t0 + share, int64_t(tokens));
  if (t0 >= t1) return;
  int s0 = 0, n = sequences;      // the last sequence that begins at t0 or before it is one of s0 .. s0 + n - 1
  while (n > 1) {
    const int step = (n + 31) / 32, i = lane * step;
    const int skip = max(__popc(__ballot_sync(0xffffffffu, i < n && offsets[s0 + i] <= t0)) - 1, 0) * step;
    s0 += skip;
    n = min(step, n - skip);
  }
  for (; s0 < sequences; s0 += 32) {
    const int2 span = s0 + lane < sequences ? sequence_span(offsets, s0 + lane, tokens) : make_int2(tokens, 0);
    unsigned some = __ballot_sync(0xffffffffu, span.y > 0 && span.x < t1 && int64_t(span.x) + span.y > t0);
    for (; some; some &= some - 1) {
      const int j = __ffs(some) - 1, first = __shfl_sync(0xffffffffu, span.x, j), length = __shfl_sync(0xffffffffu, span.y, j);
      const int64_t end = min(t1, int64_t(first) + length) * heads;
      float most = 0.f;
#pragma unroll 4
      for (int64_t row = max(t0, int64_t(first)) * heads + lane; row < end; row += 32) most = fmaxf(most, value(row));
      const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));      // (numbers >= 0 have the order of their bits)
      unsigned* at = to + kMosts * int64_t(s0 + j);
      if (lane == 0 && bits > *reinterpret_cast<volatile unsigned*>(at)) atomicMax(at, bits);
    }
    if (__any_sync(0xffffffffu, span.x >= t1)) break;
  }
}

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const PlanArgs p) {
  allow_dependents();
  const PackedArgs& a = p.a;
  if (blockIdx.x > 0) {
    if (p.halves == 0) return;
    const int q0 = tokens_before(a.offsets_q, a.sequences, a.tokens_q), q1 = covered_tokens(a.offsets_q, a.sequences, a.tokens_q);
    const int64_t row = int64_t(a.heads) * a.D * p.halves;
    const int64_t at = int64_t(blockIdx.x - 1) * kPlanThreads + threadIdx.x, step = int64_t(kClearCtas) * kPlanThreads;
    clear_outside<uint16_t>(static_cast<uint16_t*>(p.backward ? a.dq : a.out), row, q0, q1, a.tokens_q, 0, at, step);      // (a zero has no bits)
    if (!p.backward) {
      clear_outside<float>(a.lse, a.heads, q0, q1, a.tokens_q, -INFINITY, at, step);
    } else {
      const int k0 = tokens_before(a.offsets_k, a.sequences, a.tokens_k), k1 = covered_tokens(a.offsets_k, a.sequences, a.tokens_k);
      const int64_t krow = int64_t(a.kv_heads) * a.D * p.halves;
      clear_outside<uint16_t>(static_cast<uint16_t*>(a.dk), krow, k0, k1, a.tokens_k, 0, at, step);
      clear_outside<uint16_t>(static_cast<uint16_t*>(a.dv), krow, k0, k1, a.tokens_k, 0, at, step);
      if (a.largest) {
        // (a NaN counts as infinite; a query without a key has no gradient)
        auto size = [](float x) { return fabsf(x) < INFINITY ? fabsf(x) : INFINITY; };
        const float inv_mul = 1.f / (a.scale * kLog2e);
        raise_largest(a.offsets_q, a.sequences, a.tokens_q, a.heads, a.largest + kMostDout,
                      [&](int64_t row) { return a.lse[row] == -INFINITY ? 0.f : size(a.squares[row]); });
        raise_largest(a.offsets_q, a.sequences, a.tokens_q, a.heads, a.largest + kMostOfAddends, [&](int64_t row) {
          const float lse = a.lse[row];
          return lse == -INFINITY ? 0.f : fmaxf(size((lse - float(kPShift)) * inv_mul), size(a.delta[row]));
        });
        const float* values = a.squares + int64_t(a.tokens_q) * a.heads;
        raise_largest(a.offsets_k, a.sequences, a.tokens_k, a.kv_heads, a.largest + kMostV, [&](int64_t row) { return size(values[row]); });
      }
    }
    return;
  }
  __shared__ int buckets[kBuckets];      // blocks of each group and length, then the place of the next one
  __shared__ int sums[32];
  __shared__ uint8_t groups[kPlanThreads];
  __shared__ int scratch[kPlanThreads];
  if (p.grouped) form_groups(p, groups, buckets, scratch);
  const uint8_t* group = p.grouped ? groups : nullptr;
  for (int i = threadIdx.x; i < kBuckets; i += kPlanThreads) buckets[i] = 0;
  __syncthreads();
  for_each_block(p, group, [&](const WorkItem&, int bucket) { atomicAdd(&buckets[bucket], 1); });
  __syncthreads();
  // places
  static_assert(kBuckets == kPlanThreads, "a bucket per thread");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int own = buckets[threadIdx.x];
  int upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += other;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += sums[w];
  buckets[threadIdx.x] = upto - own;
  if (threadIdx.x == kPlanThreads - 1) {
    p.count[0] = min(upto, p.most);
    p.count[1] = 0;
  }
  __syncthreads();
  for_each_block(p, group, [&](const WorkItem& w, int bucket) {
    const int place = atomicAdd(&buckets[bucket], 1);
    if (place >= p.most) return;
    int4* dst = reinterpret_cast<int4*>(p.items + place);
    dst[0] = make_int4(w.begin, w.n, w.other, w.other_n);
    dst[1] = make_int4(w.seen, w.steps, w.index, w.sequence);
  });
}

}  // namespace

int launch_plan(const PackedArgs& a, bool backward, int block, int step_tokens, void* list, cudaStream_t st, int element) {
  PlanArgs p{};
  p.a = a;
  p.backward = backward;
  p.halves = element / 2;
  p.block = block;
  p.kv_heads = a.kv_heads;
  p.grouped = a.sequences > 1 && a.sequences <= kPlanThreads && most_blocks(backward ? a.tokens_k : a.tokens_q, a.sequences, block) * a.kv_heads > kGroupItems;
  p.step_tokens = step_tokens;
  const int64_t tiles = (backward ? a.tokens_q : a.tokens_k) / 128;
  while ((tiles >> p.shift) >= kLengths) ++p.shift;
  p.most = int(most_blocks(backward ? a.tokens_k : a.tokens_q, a.sequences, block));
  p.most_steps = most_blocks(a.tokens_q, a.sequences, step_tokens);
  p.count = static_cast<int*>(list);
  p.items = reinterpret_cast<WorkItem*>(static_cast<char*>(list) + 16);
  packed_plan_kernel<<<1 + kClearCtas, kPlanThreads, 0, st>>>(p);
  count_launch();
  return check_launch("packed_plan_kernel");
}

}  // namespace packed
}  // namespace nb200
