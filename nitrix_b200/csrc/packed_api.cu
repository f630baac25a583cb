// Entry points of attention over packed sequences: checks, choice of the kernel family, scratch.
#include "packed_tc.cuh"

namespace nb200 {
namespace packed {
namespace {

int check(const nb200_packed_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_packed_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  if (p->dtype != NB200_F32 && p->dtype != NB200_BF16 && p->dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (p->kernel != NB200_KERNEL_AUTO && p->kernel != NB200_KERNEL_SIMT) { set_error("%s: bad kernel", what); return NB200_ERR_INVALID; }
  if (p->tokens_q < 0 || p->tokens_k < 0 || p->sequences < 0 || p->heads <= 0 || p->kv_heads <= 0 || p->head_dim <= 0) {
    set_error("%s: bad extents", what);
    return NB200_ERR_INVALID;
  }
  if (p->heads % p->kv_heads) { set_error("%s: %d query heads are no multiple of %d key heads", what, p->heads, p->kv_heads); return NB200_ERR_INVALID; }
  if (p->head_dim > 256) { set_error("%s: head dim %d, at most 256", what, p->head_dim); return NB200_ERR_UNSUPPORTED; }
  if (p->kv_heads > 65535 || int64_t(p->tokens_q) * (p->heads / p->kv_heads) / 32 + p->sequences > 0x7fffffff) {
    set_error("%s: too many heads or tokens", what);
    return NB200_ERR_UNSUPPORTED;
  }
  return NB200_OK;
}

PackedArgs lower(const nb200_packed_params* p) {
  PackedArgs a{};
  a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.lse = p->lse;
  a.dout = p->dout; a.dq = p->dq; a.dk = p->dk; a.dv = p->dv;
  a.offsets_q = p->offsets_q; a.offsets_k = p->offsets_k;
  for (int i = 0; i < 2; ++i) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.dos[i] = p->dout_stride[i]; }
  a.tokens_q = p->tokens_q; a.tokens_k = p->tokens_k; a.sequences = p->sequences;
  a.heads = p->heads; a.kv_heads = p->kv_heads; a.group = p->heads / p->kv_heads;
  a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  return a;
}

size_t delta_bytes(const nb200_packed_params* p) { return (size_t(p->tokens_q) * size_t(p->heads) * sizeof(float) + 255) / 256 * 256; }

bool tensor_cores(const nb200_packed_params* p, const PackedArgs& a, int pass) {
  if (p->kernel != NB200_KERNEL_AUTO) return false;
  return pass == NB200_PASS_FWD ? tc_packed_supported(a, p->dtype) : tc_packed_bwd_supported(a, p->dtype);
}

// fp32 on the tensor cores
bool fp32_tensor_cores(const nb200_packed_params* p, const PackedArgs& a, int pass) {
  if (p->kernel != NB200_KERNEL_AUTO) return false;
  return pass == NB200_PASS_FWD ? fp32_packed_supported(a, p->dtype) : fp32_packed_bwd_supported(a, p->dtype);
}

size_t workspace(const nb200_packed_params* p, const PackedArgs& a, int pass) {
  if (fp32_tensor_cores(p, a, pass)) return pass == NB200_PASS_FWD ? fp32_packed_fwd_bytes(a) : delta_bytes(p) + fp32_packed_bwd_bytes(a);
  if (tensor_cores(p, a, pass)) return pass == NB200_PASS_FWD ? tc_packed_fwd_bytes(a) : tc_packed_bwd_bytes(a, p->dtype);
  return pass == NB200_PASS_FWD ? 0 : delta_bytes(p) + simt_packed_bwd_bytes(a);
}

int check_workspace(const nb200_packed_params* p, const PackedArgs& a, int pass, const char* what) {
  const size_t need = workspace(p, a, pass);
  if (need && (!p->workspace || p->workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes needed (nb200_packed_workspace_bytes), %zu given", what, need, p->workspace_bytes);
    return NB200_ERR_WORKSPACE;
  }
  if (need && reinterpret_cast<uintptr_t>(p->workspace) % 256) { set_error("%s: the workspace must begin on a 256-byte boundary", what); return NB200_ERR_ALIGNMENT; }
  return NB200_OK;
}

int check_operands(const nb200_packed_params* p, const char* what, bool backward) {
  const bool q = p->tokens_q > 0, k = p->tokens_k > 0;
  bool ok = p->offsets_q && p->offsets_k && (!q || (p->q && p->out && p->lse)) && (!k || (p->k && p->v));
  if (backward) ok = ok && (!q || (p->dout && p->dq)) && (!k || (p->dk && p->dv));
  if (!ok) { set_error("%s: NULL operand", what); return NB200_ERR_INVALID; }
  return NB200_OK;
}

}  // namespace
}  // namespace packed
}  // namespace nb200

using namespace nb200;
using namespace nb200::packed;

extern "C" NB200_API int nb200_packed_plan(const nb200_packed_params* p, int pass, int* kernel) {
  if (int rc = check(p, "packed_plan")) return rc;
  if (!kernel || (pass != NB200_PASS_FWD && pass != NB200_PASS_BWD)) { set_error("packed_plan: NULL result or bad pass"); return NB200_ERR_INVALID; }
  const PackedArgs a = lower(p);
  *kernel = tensor_cores(p, a, pass) || fp32_tensor_cores(p, a, pass) ? NB200_KERNEL_TCGEN05 : NB200_KERNEL_SIMT;
  return NB200_OK;
}

extern "C" NB200_API int nb200_packed_workspace_bytes(const nb200_packed_params* p, int pass, size_t* bytes) {
  if (int rc = check(p, "packed_workspace_bytes")) return rc;
  if (!bytes || (pass != NB200_PASS_FWD && pass != NB200_PASS_BWD)) { set_error("packed_workspace_bytes: NULL result or bad pass"); return NB200_ERR_INVALID; }
  *bytes = workspace(p, lower(p), pass);
  return NB200_OK;
}

extern "C" NB200_API int nb200_packed_fwd(const nb200_packed_params* p, void* cuda_stream) {
  if (int rc = check(p, "packed_fwd")) return rc;
  if (p->tokens_q == 0) return NB200_OK;
  if (int rc = check_operands(p, "packed_fwd", false)) return rc;
  const PackedArgs a = lower(p);
  if (int rc = check_workspace(p, a, NB200_PASS_FWD, "packed_fwd")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  if (tensor_cores(p, a, NB200_PASS_FWD)) return tc_packed_fwd(a, p->dtype, p->workspace, st);
  if (fp32_tensor_cores(p, a, NB200_PASS_FWD)) return fp32_packed_fwd(a, p->workspace, st);
  if (int rc = launch_clear_uncovered(a, p->dtype, false, st)) return rc;
  if (p->sequences == 0) return NB200_OK;
  return simt_packed_fwd(a, p->dtype, st);
}

extern "C" NB200_API int nb200_packed_bwd(const nb200_packed_params* p, void* cuda_stream) {
  if (int rc = check(p, "packed_bwd")) return rc;
  if (p->tokens_q == 0 && p->tokens_k == 0) return NB200_OK;
  if (int rc = check_operands(p, "packed_bwd", true)) return rc;
  PackedArgs a = lower(p);
  if (int rc = check_workspace(p, a, NB200_PASS_BWD, "packed_bwd")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  if (tensor_cores(p, a, NB200_PASS_BWD)) return tc_packed_bwd(a, p->dtype, p->workspace, st);
  a.delta = static_cast<float*>(p->workspace);
  if (fp32_tensor_cores(p, a, NB200_PASS_BWD)) {
    if (int rc = launch_packed_delta(a, p->dtype, st)) return rc;
    return fp32_packed_bwd(a, static_cast<char*>(p->workspace) + delta_bytes(p), st);
  }
  a.parts = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + delta_bytes(p));
  if (int rc = launch_clear_uncovered(a, p->dtype, true, st)) return rc;
  if (p->sequences == 0) return NB200_OK;
  if (p->tokens_q > 0) {
    if (int rc = launch_packed_delta(a, p->dtype, st)) return rc;
  }
  return simt_packed_bwd(a, p->dtype, st);
}
