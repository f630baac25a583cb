// The tensor-core kernels of attention over packed sequences: work lists and launches.
#pragma once

#include "packed.cuh"
#include "sdpa_tc_common.cuh"

namespace nb200 {
namespace packed {

// One entry of a work list: a block of one sequence, for every key head.
//   forward   queries begin .. begin + n of the packed tensor, of which the first sees the sequence's first `seen` keys (causal)
//   backward  keys begin .. begin + n, of which the first is seen by the queries from `seen` on (counted within the sequence)
// Under causal `seen` may lie outside the sequence; it means nothing otherwise.
struct __align__(16) WorkItem {
  int begin;        // first token of the block
  int n;            // tokens of the block
  int other;        // first token of the sequence on the other side: its keys (forward), its queries (backward)
  int other_n;      // tokens there
  int seen;         // see above
  int steps;        // backward: first 64-row step of the sequence's rows in the gradient sums of dq
  int index;        // number of the block in its sequence
  int sequence;
};
static_assert(sizeof(WorkItem) == 32, "two 16-byte loads");

// List in device memory: 16 bytes of header (the number of entries; the pieces of work taken so far, zero to begin with), then
// the entries (packed_plan.cu: their order).
struct WorkList {
  const int* count;
  int* taken;
  const WorkItem* items;
};
inline size_t work_list_bytes(int64_t most) { return (16 + size_t(most) * sizeof(WorkItem) + 255) / 256 * 256; }
// most blocks of `block` tokens that sequences of `tokens` tokens together have
inline int64_t most_blocks(int64_t tokens, int sequences, int block) { return tokens / block + sequences; }

// Fills the list (and clears the outputs of tokens that no sequence covers, and takes the maxima that the fp16 backward asks for,
// which would be launches of their own).
// `element`: bytes of an element of the outputs; 0: they are left alone.
// `block`: queries (forward) or keys (backward) of a block; `step_tokens` (backward): queries of a 64-row step.
int launch_plan(const PackedArgs& a, bool backward, int block, int step_tokens, void* list, cudaStream_t st, int element = 2);

// fp16 backward: a power of two on P, and what is known of each sequence (over its queries that see a key): the largest squared
// norm of a row of dout and of v, the largest size of what is added to a product (lse - kPShift over scale log2 e, and delta).
constexpr int kPShift = 10;
enum SequenceMost { kMostDout = 0, kMostV = 1, kMostOfAddends = 2, kMosts = 4 };

// Rows of a query tile are, token after token, the query heads of one key head: this many tokens fit.
__host__ __device__ inline int tile_tokens(int rows, int group) { return rows / group; }

bool tc_packed_supported(const PackedArgs& a, int dtype);
size_t tc_packed_fwd_bytes(const PackedArgs& a);
int tc_packed_fwd(const PackedArgs& a, int dtype, void* ws, cudaStream_t st);
bool tc_packed_bwd_supported(const PackedArgs& a, int dtype);
size_t tc_packed_bwd_bytes(const PackedArgs& a, int dtype);
int tc_packed_bwd(const PackedArgs& a, int dtype, void* ws, cudaStream_t st);

// fp32 operands as three bf16 planes (packed_fp32_tc.cu)
bool fp32_packed_supported(const PackedArgs& a, int dtype);
size_t fp32_packed_fwd_bytes(const PackedArgs& a);
int fp32_packed_fwd(const PackedArgs& a, void* ws, cudaStream_t st);
bool fp32_packed_bwd_supported(const PackedArgs& a, int dtype);
size_t fp32_packed_bwd_bytes(const PackedArgs& a);
int fp32_packed_bwd(const PackedArgs& a, void* ws, cudaStream_t st);

#ifdef __CUDACC__
__device__ __forceinline__ WorkItem load_item(const WorkItem* p) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(p)), b = __ldg(reinterpret_cast<const int4*>(p) + 1);
  WorkItem w;
  w.begin = a.x; w.n = a.y; w.other = a.z; w.other_n = a.w; w.seen = b.x; w.steps = b.y; w.index = b.z; w.sequence = b.w;
  return w;
}
#endif

}  // namespace packed
}  // namespace nb200
