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
  float* squares;            // fp16 on the tensor cores: squared norms of the rows of dout (tokens_q, heads), then of v
  unsigned* largest;         // and maxima over each sequence (SequenceMost), as the bits of fp32 numbers
  float* parts;              // fp32 units: parts of dk and dv, [part][dk, dv][token][key head][D]
};

#ifdef __CUDACC__
// First token and number of tokens of a sequence; offsets that make no sense are cut to the tensors.
__device__ __forceinline__ int2 sequence_span(const int* offsets, int i, int tokens) {
  const int begin = min(max(offsets[i], 0), tokens), end = min(max(offsets[i + 1], begin), tokens);
  return make_int2(begin, end - begin);
}
// Tokens before the first sequence, and up to the end of the last one: those outside belong to no sequence.
__device__ __forceinline__ int tokens_before(const int* offsets, int sequences, int tokens) {
  return sequences > 0 ? min(max(offsets[0], 0), tokens) : 0;
}
__device__ __forceinline__ int covered_tokens(const int* offsets, int sequences, int tokens) {
  return sequences > 0 ? min(max(offsets[sequences], 0), tokens) : 0;
}

// Elements of the rows, `row` elements each, that lie outside [first, last); every `step`-th of them from `at` on.
template <typename T>
__device__ __forceinline__ void clear_outside(T* base, int64_t row, int first, int last, int rows, T value, int64_t at, int64_t step) {
  for (int64_t i = at; i < first * row; i += step) base[i] = value;
  for (int64_t i = last * row + at; i < rows * row; i += step) base[i] = value;
}

// The sequence that piece `index` of all sequences' `count(i)` pieces belongs to, and its number there (-1: there is no such
// piece).  For a whole warp.
struct Place {
  int sequence, index;
};
template <typename Count>
__device__ __forceinline__ Place find_place(int index, int sequences, Count count) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < sequences; s0 += 32) {
    int upto = s0 + lane < sequences ? count(s0 + lane) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    const unsigned above = __ballot_sync(0xffffffffu, before + upto > index);
    if (above) {
      const int j = __ffs(above) - 1;
      const int prev = __shfl_sync(0xffffffffu, upto, j > 0 ? j - 1 : 0);
      return Place{s0 + j, index - before - (j > 0 ? prev : 0)};
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Place{0, -1};
}
#endif

// out = zeros for the tokens of no sequence (and lse = -inf), or zero gradients: part of every pass
int launch_clear_uncovered(const PackedArgs& a, int dtype, bool backward, cudaStream_t st);
int launch_packed_delta(const PackedArgs& a, int dtype, cudaStream_t st);
int simt_packed_fwd(const PackedArgs& a, int dtype, cudaStream_t st);
size_t simt_packed_bwd_bytes(const PackedArgs& a);
int simt_packed_bwd(const PackedArgs& a, int dtype, cudaStream_t st);

}  // namespace packed
}  // namespace nb200
