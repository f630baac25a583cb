/*
 * nitrix_b200_rotary.h -- C ABI of the rotary position embedding of the B200 (sm_100a) library, behind the same shared
 * library, status codes and dtype codes as the attention path (nitrix_b200_attention.h).
 *
 *   nb200_rotary   queries and keys (either may be left out) in one launch
 *
 * Head dim D; the first 2 P elements of a head are P pairs, the others pass unchanged.  Pair j belongs to axis a(j): the
 * axes' pairs follow one another, `sections[a]` of them for axis a.  With phase = positions[token][a(j)] * frequencies[j],
 *
 *   (x1, x2) -> (x1 cos phase - x2 sin phase,  x1 sin phase + x2 cos phase)
 *
 * where a pair is elements (j, j + P), or (2 j, 2 j + 1) with `interleaved`.  `inverse` turns the other way: it is the
 * gradient, since the rotation is orthogonal.  Phases are formed with the rounding errors of their products and
 * reduced to one turn, so that they are as good at position 2^40 as at 1; the rotation itself is fp32, rounded once to the operands' type.
 *
 * Layout.  x is (B, S, heads, D) described by three element strides (unit stride on D), y is dense.  positions are dense
 * (B, S, axes), frequencies dense fp32 (P).  Every pointer is a device pointer; the work is enqueued on the caller's
 * stream and nothing is allocated.
 */
#ifndef NITRIX_B200_ROTARY_H_
#define NITRIX_B200_ROTARY_H_

#include "nitrix_b200_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NB200_ROTARY_MAX_AXES 8

enum nb200_position_dtype { NB200_POS_I32 = 0, NB200_POS_I64 = 1, NB200_POS_F32 = 2 };

typedef struct nb200_rotary_tensor {
  const void* x;
  void* y;                 /* dense (B, S, heads, D); must not overlap x */
  int64_t x_stride[3];     /* elements, over (B, S, heads) */
  int32_t heads;           /* 0: the tensor is left out */
  int32_t reserved;
} nb200_rotary_tensor;

typedef struct nb200_rotary_params {
  size_t struct_size;      /* sizeof(nb200_rotary_params) */
  nb200_rotary_tensor q, k;
  const void* positions;
  const float* frequencies;
  int32_t batch, length;   /* B, S */
  int32_t head_dim;
  int32_t axes;
  int32_t sections[NB200_ROTARY_MAX_AXES];   /* pairs of each axis; their sum is P, 2 P <= head_dim */
  int32_t position_dtype;  /* nb200_position_dtype */
  int32_t dtype;           /* nb200_dtype of x and y */
  int32_t interleaved;
  int32_t inverse;
} nb200_rotary_params;

NB200_API int nb200_rotary(const nb200_rotary_params* p, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* NITRIX_B200_ROTARY_H_ */
