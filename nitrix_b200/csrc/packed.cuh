// Shared pieces of the kernels of attention over packed sequences (packed_simt.cu, packed_tc_*.cu).
#pragma once

#include "nitrix_b200_packed.h"
#include "sdpa_common.cuh"

namespace nb200 {
namespace packed {

struct PackedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;                // (tokens_q, heads)
  const void* dout;
  void* dq;
  void* dk;
  void* dv;
  const int* offsets_q;
  const int* offsets_k;
  int64_t qs[2], ks[2], vs[2], dos[2];
  int tokens_q, tokens_k, sequences;
  int heads, kv_heads, group;       // group: query heads of a key head
  int D;
  int causal;
  float scale;
  float* delta;              // (tokens_q, heads): rowsum(out * dout)
};

#ifdef __CUDACC__
// First token and number of tokens of a sequence; offsets that make no sense are cut to the tensors.
__device__ __forceinline__ int2 sequence_span(const int* offsets, int i, int tokens) {
  const int begin = min(max(offsets[i], 0), tokens), end = min(max(offsets[i + 1], begin), tokens);
  return make_int2(begin, end - begin);
}
__device__ __forceinline__ int covered_tokens(const int* offsets, int sequences, int tokens) {
  return sequences > 0 ? min(max(offsets[sequences], 0), tokens) : 0;
}
#endif

// out = zeros for the tokens behind the last sequence (and lse = -inf, where `lse` is given): part of every pass
int launch_clear_uncovered(const PackedArgs& a, int dtype, bool backward, cudaStream_t st);
int launch_packed_delta(const PackedArgs& a, int dtype, cudaStream_t st);
int simt_packed_fwd(const PackedArgs& a, int dtype, cudaStream_t st);
int simt_packed_bwd(const PackedArgs& a, int dtype, cudaStream_t st);

}  // namespace packed
}  // namespace nb200
