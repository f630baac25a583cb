/*
 * nitrix_b200_rms_norm.h -- C ABI of the root-mean-square norm of the B200 (sm_100a) library, behind the same shared library,
 * status codes and dtype codes as the attention path (nitrix_b200_attention.h).
 *
 *   nb200_rms_norm_fwd   y, or its e4m3 codes and their scales; with a residual also the sum of the two streams
 *   nb200_rms_norm_bwd   dx (the gradient of either stream) and dweight
 *
 * Per row of `channels` elements, in fp32 whatever the storage dtype (rows whose squares leave fp32, above or below, in fp64):
 *
 *   h = x + residual, rounded to the dtype (x without a residual);   rstd = (mean h^2 + eps)^-1/2;   y = h rstd weight
 *
 * With `scales`, y is e4m3: of every `group` channels (0: of the row) a = max(max |y|, 2^-100), scale = a / 448 (fp32,
 * [row][group]), code = y (448 / a) rounded to e4m3, of the y that has not been rounded before.  A NaN makes all of its row NaN.  An
 * infinity has the mean square infinite and rstd 0: its own y is NaN and the others of its row are 0, so that the codes and the scale
 * of its group (or row) are NaN, those of the row's other groups zeros under the least scale.  With g = dy weight and n = h rstd, the
 * backward is
 *
 *   dx = dsum + rstd (g - n mean(g n)),   dweight = sum over rows of dy n
 *
 * Layout.  x, residual, y, sum, dy, dsum, dx are dense [rows][channels]; weight and dweight [channels], of the same dtype or
 * fp32.  Rows of a multiple of 16 bytes and 16-byte aligned pointers take kernels that move 16-byte words and read
 * a row once up to 64 KB (backward: 32 KB); anything else runs the same kernels element by element, up to 16384 (8192) channels at
 * one reading.  Sums have one order.  Every pointer is a
 * device pointer; all work is enqueued on the caller's stream; nothing is allocated.
 */
#ifndef NITRIX_B200_RMS_NORM_H_
#define NITRIX_B200_RMS_NORM_H_

#include "nitrix_b200_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct nb200_rms_norm_params {
  size_t struct_size;      /* sizeof(nb200_rms_norm_params) */
  const void* x;           /* backward: the rows that were normalised, h */
  const void* residual;    /* forward: NULL, or the second stream */
  const void* weight;      /* NULL: no scaling */
  void* y;                 /* forward output; no output may overlap an input */
  void* sum;               /* forward, with a residual: h */
  float* rstd;             /* [rows]: written by the forward when non-NULL, read by the backward */
  float* scales;           /* forward: NULL, or the scales of an e4m3 y */
  const void* dy;          /* backward */
  const void* dsum;        /* backward: the gradient of `sum`, or NULL */
  void* dx;
  void* dweight;           /* backward: NULL: not wanted */
  void* workspace;         /* backward with dweight: nb200_rms_norm_workspace_bytes of the same block (the operands' alignment
                              counts); 16-byte aligned */
  size_t workspace_bytes;
  int64_t rows;
  int32_t channels;        /* at most 2^30 */
  int32_t dtype;           /* nb200_dtype of x, residual, y, sum, dy, dsum, dx */
  int32_t weight_dtype;    /* of weight and dweight: dtype or NB200_F32 */
  int32_t group;           /* with scales: 0, 32, 64 or 128 channels; a group divides the channels */
  float eps;
  int32_t reserved;
} nb200_rms_norm_params;

NB200_API int nb200_rms_norm_fwd(const nb200_rms_norm_params* p, void* cuda_stream);
NB200_API int nb200_rms_norm_bwd(const nb200_rms_norm_params* p, void* cuda_stream);
NB200_API int nb200_rms_norm_workspace_bytes(const nb200_rms_norm_params* p, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* NITRIX_B200_RMS_NORM_H_ */
