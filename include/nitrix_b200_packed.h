/*
 * nitrix_b200_packed.h -- C ABI of attention over packed sequences of the B200 (sm_100a) library, behind the same shared
 * library, status codes and dtype codes as the attention path (nitrix_b200_attention.h).
 *
 *   nb200_packed_fwd   out and lse
 *   nb200_packed_bwd   dq, dk, dv
 *
 * Sequences of unequal length lie one after the other without padding: sequence i has the queries offsets_q[i] ..
 * offsets_q[i + 1) and the keys offsets_k[i] .. offsets_k[i + 1), lq and lk of them.  q is (tokens_q, heads, D), k and v are
 * (tokens_k, kv_heads, D); query head h reads key head h / (heads / kv_heads).  With `causal`, query i of a sequence sees its
 * keys up to i + lk - lq: the last query sees all of them.  A query that sees no key gives zeros, lse = -inf and zero
 * gradients.  Tokens before offsets[0] and behind offsets[sequences] belong to no sequence; their rows of every output are
 * zeros.  lse is (tokens_q, heads) fp32, the base-2 log-sum-exp of the scaled scores.
 *
 * q, k, v and dout are described by two element strides (token, head; unit stride on D); out, dq, dk and dv are dense.  The
 * offsets are device memory: nothing is read on the host.  Every pointer is a device pointer; all work is enqueued on the
 * caller's stream; nothing is allocated.
 */
#ifndef NITRIX_B200_PACKED_H_
#define NITRIX_B200_PACKED_H_

#include "nitrix_b200_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nb200_packed_params {
  size_t struct_size;        /* sizeof(nb200_packed_params) */
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
  const void* dout;          /* backward, with dq, dk and dv */
  void* dq;
  void* dk;
  void* dv;
  const int32_t* offsets_q;  /* (sequences + 1) */
  const int32_t* offsets_k;
  int64_t q_stride[2], k_stride[2], v_stride[2], dout_stride[2];
  int32_t tokens_q, tokens_k;
  int32_t sequences;
  int32_t heads, kv_heads, head_dim;
  int32_t dtype;             /* nb200_dtype */
  int32_t causal;
  float scale;
  int32_t kernel;            /* nb200_kernel: AUTO or SIMT */
  void* workspace;           /* nb200_packed_workspace_bytes of the pass, asked for with the same operands; 256-byte aligned */
  size_t workspace_bytes;
} nb200_packed_params;

NB200_API int nb200_packed_fwd(const nb200_packed_params* p, void* cuda_stream);
NB200_API int nb200_packed_bwd(const nb200_packed_params* p, void* cuda_stream);
/* pass: nb200_pass */
NB200_API int nb200_packed_workspace_bytes(const nb200_packed_params* p, int pass, size_t* bytes);
/* The family that runs the pass: NB200_KERNEL_TCGEN05 (fp32 as three bf16 planes among it) or NB200_KERNEL_SIMT. */
NB200_API int nb200_packed_plan(const nb200_packed_params* p, int pass, int* kernel);

#ifdef __cplusplus
}
#endif
#endif /* NITRIX_B200_PACKED_H_ */
