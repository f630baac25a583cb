// The differentiable operations of nitrix_b200.nn as C++ autograd functions over the library's C ABI.
//
// A training pass of a small problem is bound by the host.  As Python autograd functions with ctypes calls, a forward and
// backward with 13 us of library calls took 180 us (fp32 attention, 64 x 64; an empty autograd function takes 67), most of
// it filling parameter blocks, allocating through Python and taking the interpreter lock on the engine's device thread;
// here it takes 103, an inference call 16 instead of 38, LayerNorm's pass 81 instead of 131, the scan's 117 instead of 193.
// Nothing is kept between calls: every call asks the library for its plan and its scratch anew (about a microsecond).
//
// The library is the one ctypes has loaded: bind() receives the addresses of its entry points.
#include <limits>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>

#include "nitrix_b200_attention.h"
#include "nitrix_b200_cache.h"
#include "nitrix_b200_norm.h"
#include "nitrix_b200_packed.h"
#include "nitrix_b200_rms_norm.h"
#include "nitrix_b200_rotary.h"
#include "nitrix_b200_scan.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using MaybeTensor = std::optional<Tensor>;

#define NB200_ENTRY_POINTS(X)                                                                                              \
  X(nb200_last_error) X(nb200_sdpa_plan) X(nb200_sdpa_workspace_bytes) X(nb200_sdpa_workspace_least_bytes)                 \
  X(nb200_sdpa_fwd) X(nb200_sdpa_bwd) X(nb200_mask_pack_bytes) X(nb200_mask_pack) X(nb200_qk_rms_norm)                     \
  X(nb200_qk_rms_norm_grad) X(nb200_layer_norm_fwd) X(nb200_layer_norm_bwd) X(nb200_layer_norm_workspace_bytes)            \
  X(nb200_selective_scan_fwd) X(nb200_selective_scan_bwd) X(nb200_selective_scan_checkpoint_bytes)                         \
  X(nb200_selective_scan_workspace_bytes) X(nb200_rotary) X(nb200_cache_append) X(nb200_cache_fork) X(nb200_cache_compact)  \
  X(nb200_cache_workspace_bytes) X(nb200_decode) X(nb200_decode_workspace_bytes) X(nb200_packed_plan) X(nb200_packed_fwd)  \
  X(nb200_packed_bwd) X(nb200_packed_workspace_bytes) X(nb200_rms_norm_fwd) X(nb200_rms_norm_bwd)                          \
  X(nb200_rms_norm_workspace_bytes) X(nb200_cache_append_quantized) X(nb200_cache_fork_quantized)                          \
  X(nb200_cache_compact_quantized) X(nb200_cache_read) X(nb200_decode_quantized) X(nb200_decode_quantized_workspace_bytes)

struct Library {
#define X(name) decltype(&::name) name = nullptr;
  NB200_ENTRY_POINTS(X)
#undef X
} lib;

void bind(const std::map<std::string, uintptr_t>& addresses) {
#define X(name) lib.name = reinterpret_cast<decltype(&::name)>(addresses.at(#name));
  NB200_ENTRY_POINTS(X)
#undef X
}

std::vector<std::string> entry_points() {
  std::vector<std::string> names;
#define X(name) names.push_back(#name);
  NB200_ENTRY_POINTS(X)
#undef X
  return names;
}

void check(int rc, const char* what) {
  if (rc != NB200_OK) throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(rc) + "): " + lib.nb200_last_error());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({int64_t(bytes)}, like.options().dtype(at::kByte));
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? NB200_F32 : t == at::kBFloat16 ? NB200_BF16 : t == at::kHalf ? NB200_F16 : -1;
}

bool has_expanded_axis(const Tensor& t) {
  for (int64_t a = 0; a < t.dim(); ++a)
    if (t.stride(a) == 0 && t.size(a) > 1) return true;
  return false;
}

// There are no forward-mode rules.  (torch's own refusal for C++ functions is a RuntimeError, after the kernels have run.)
bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const MaybeTensor& t) { return t && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* what, const T&... operands) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(operands) || ...), what, ": forward-mode differentiation is not implemented");
}

Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }

void copy_strides(int64_t (&dst)[4], const Tensor& t) {
  for (int a = 0; a < 4; ++a) dst[a] = t.stride(a);
}
// 0 on every axis that t broadcasts over
void copy_strides(int64_t (&dst)[4], const Tensor& t, const int64_t (&full)[4]) {
  for (int a = 0; a < 4; ++a) dst[a] = (t.size(a) == 1 && full[a] != 1) ? 0 : t.stride(a);
}

// ---- attention ---------------------------------------------------------------------------------------------------------
struct Attention {
  Tensor q, k, v;            // (B, H, S, D), (B, H, T, D), (B, H, T, Dv)
  Tensor bias, mask;         // own extent (1 or full) on four axes, or undefined
  Tensor packed;             // the mask's bits as nb200_mask_pack writes them, or undefined
  double scale;
  bool causal;
  int kernel;
  // The mask's strides when it was packed, which are the layout of its bits.  A saved-tensor hook may hand the backward the
  // mask in another layout: an expanded axis, which has no bits of its own, comes back from t.cpu() as a dense one.
  std::vector<int64_t> packed_strides;

  nb200_sdpa_params params() const {
    nb200_sdpa_params p{};
    p.struct_size = sizeof(p);
    p.dtype = dtype_code(q.scalar_type());
    p.B = int32_t(q.size(0)); p.H = int32_t(q.size(1)); p.S = int32_t(q.size(2)); p.D = int32_t(q.size(3));
    p.T = int32_t(k.size(2)); p.Dv = int32_t(v.size(3));
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr();
    copy_strides(p.q_stride, q); copy_strides(p.k_stride, k); copy_strides(p.v_stride, v);
    const int64_t full[4] = {p.B, p.H, p.S, p.T};
    if (bias.defined()) {
      p.bias = bias.data_ptr();
      p.bias_dtype = dtype_code(bias.scalar_type());
      copy_strides(p.bias_stride, bias, full);
    }
    if (mask.defined()) {
      p.mask = static_cast<const uint8_t*>(packed.defined() ? packed.data_ptr() : mask.data_ptr());
      if (packed.defined()) std::copy(packed_strides.begin(), packed_strides.end(), p.mask_stride);
      else copy_strides(p.mask_stride, mask, full);
      p.mask_is_bitpacked = packed.defined() ? 2 : 0;
    }
    p.scale = float(scale);
    p.causal = causal;
    p.kernel = kernel;
    p.bh_end = p.B * p.H;
    return p;
  }

  // Kernel family of a pass (no launch; the planner dereferences nothing, q stands in for what does not exist yet)
  int plan(int pass, bool want_dbias) const {
    nb200_sdpa_params p = params();
    p.out = q.data_ptr();
    p.lse = static_cast<float*>(q.data_ptr());
    p.dout = p.dq = p.dk = p.dv = q.data_ptr();
    copy_strides(p.out_stride, q); copy_strides(p.dout_stride, q); copy_strides(p.dq_stride, q);
    copy_strides(p.dk_stride, k); copy_strides(p.dv_stride, v);
    if (want_dbias && pass == NB200_PASS_BWD) {
      p.want_dbias = 1;
      int64_t st = 1;
      for (int a = 3; a >= 0; --a) { p.dbias_stride[a] = st; st *= bias.size(a); }
    }
    int chosen = 0;
    check(lib.nb200_sdpa_plan(&p, pass, &chosen), "nb200_sdpa_plan");
    return chosen;
  }

  // Scratch of a pass; a device without room for all of it gets the least with which the pass runs (the planes of fp32
  // operands take up to 1 GiB that the other kernels do without).
  Tensor workspace(nb200_sdpa_params& p, int pass) const {
    size_t need = 0;
    check(lib.nb200_sdpa_workspace_bytes(&p, pass, &need), "nb200_sdpa_workspace_bytes");
    Tensor ws;
    if (need) {
      try {
        ws = scratch(need, q);
      } catch (const c10::OutOfMemoryError&) {
        size_t least = 0;
        check(lib.nb200_sdpa_workspace_least_bytes(&p, pass, &least), "nb200_sdpa_workspace_least_bytes");
        if (least >= need) throw;
        need = least;
        if (need) ws = scratch(need, q);
      }
    }
    p.workspace = need ? ws.data_ptr() : nullptr;
    p.workspace_bytes = need;
    return ws;
  }

  // The problem as the packing entry points take it, and the bytes its bits take.
  nb200_sdpa_params pack_params(size_t* bytes) const {
    nb200_sdpa_params p = params();
    p.out = q.data_ptr();
    p.lse = static_cast<float*>(q.data_ptr());
    copy_strides(p.out_stride, q);
    p.bias = nullptr;
    p.mask_is_bitpacked = 0;
    check(lib.nb200_mask_pack_bytes(&p, 1, bytes), "nb200_mask_pack_bytes");
    return p;
  }

  void pack_mask() {
    size_t need = 0;
    const nb200_sdpa_params p = pack_params(&need);
    Tensor bits = scratch(need ? need : 1, q);
    check(lib.nb200_mask_pack(&p, 1, bits.data_ptr(), size_t(bits.numel()), stream_of(q)), "nb200_mask_pack");
    packed = bits;
    packed_strides.assign(p.mask_stride, p.mask_stride + 4);
  }

  // Bits of another layout than the one described would be read out of their buffer.
  void check_packed() const {
    if (!packed.defined()) return;
    size_t need = 0;
    pack_params(&need);
    TORCH_CHECK(size_t(packed.numel()) == (need ? need : 1), "scaled_dot_product_attention: the packed mask holds ", packed.numel(),
                " bytes, its layout takes ", need);
  }

  std::pair<Tensor, Tensor> forward() const {
    Tensor out = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
    Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    nb200_sdpa_params p = params();
    p.out = out.data_ptr();
    p.lse = lse.data_ptr<float>();
    copy_strides(p.out_stride, out);
    const Tensor ws = workspace(p, NB200_PASS_FWD);   // (same-stream reuse is ordered by the caching allocator)
    check(lib.nb200_sdpa_fwd(&p, stream_of(q)), "nb200_sdpa_fwd");
    return {out, lse};
  }

  tensor_list backward(const Tensor& out, const Tensor& lse, Tensor dout, bool want_dbias) const {
    // (e.g. the cotangent of out.sum() or out.mean(0) arrives as an expanded view)
    if (dout.stride(3) != 1 || has_expanded_axis(dout)) dout = dout.contiguous();
    Tensor dq = dense_like(q), dk = dense_like(k), dv = dense_like(v), dbias;
    nb200_sdpa_params p = params();
    p.out = out.data_ptr();
    p.lse = lse.data_ptr<float>();
    p.dout = dout.data_ptr(); p.dq = dq.data_ptr(); p.dk = dk.data_ptr(); p.dv = dv.data_ptr();
    copy_strides(p.out_stride, out); copy_strides(p.dout_stride, dout); copy_strides(p.dq_stride, dq);
    copy_strides(p.dk_stride, dk); copy_strides(p.dv_stride, dv);
    if (want_dbias) {
      dbias = dense_like(bias);
      p.dbias = dbias.data_ptr();
      copy_strides(p.dbias_stride, dbias);
    }
    check_packed();
    const Tensor ws = workspace(p, NB200_PASS_BWD);
    check(lib.nb200_sdpa_bwd(&p, stream_of(q)), "nb200_sdpa_bwd");
    return {dq, dk, dv, dbias};
  }
};

// Differentiation rule of the fused path (reference src/nitrix/_kernels/cuda/attention.py:661-700): residuals
// (q, k, v, bias, mask, out, lse), cotangents (dq, dk, dv, dbias or none).
struct AttentionRule : torch::autograd::Function<AttentionRule> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& bias,
                             const MaybeTensor& mask, double scale, bool causal, int64_t kernel, bool tensor_core) {
    Attention a{q, k, v, bias.value_or(Tensor()), mask.value_or(Tensor()), Tensor(), scale, causal, int(kernel), {}};
    const bool want_dbias = bias && bias->requires_grad();
    // (a stride of 0 is a broadcast axis to the library, which has one gradient for it)
    if (want_dbias && has_expanded_axis(a.bias)) a.bias = a.bias.contiguous();
    // On the tensor-core path the mask is bit-packed once, with the key-major copy, and the same bits serve both passes;
    // otherwise each pass reads the byte mask.
    if (tensor_core && mask && a.plan(NB200_PASS_BWD, want_dbias) == NB200_KERNEL_TCGEN05) a.pack_mask();
    auto [out, lse] = a.forward();
    ctx->save_for_backward({q, k, v, a.bias, a.mask, out, lse});
    if (a.packed.defined()) {
      ctx->saved_data["packed"] = a.packed;
      ctx->saved_data["packed_strides"] = a.packed_strides;
    }
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["flags"] = (kernel << 2) | (int64_t(want_dbias) << 1) | int64_t(causal);
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);   // (no zeros for lse's cotangent: an allocation and a launch per backward)
    return {out, lse};
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    if (!grads[0].defined()) return tensor_list(9);
    const auto s = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const auto packed = ctx->saved_data.find("packed");
    const c10::cuda::CUDAGuard guard(s[0].device());
    Attention a{s[0], s[1], s[2], s[3], s[4], Tensor(), ctx->saved_data["scale"].toDouble(), (flags & 1) != 0, int(flags >> 2), {}};
    if (packed != ctx->saved_data.end()) {
      a.packed = packed->second.toTensor();
      a.packed_strides = ctx->saved_data["packed_strides"].toIntVector();
    }
    tensor_list g = a.backward(s[5], s[6], grads[0], (flags & 2) != 0);
    g.resize(9);
    return g;
  }
};

// Operands as the library takes them: four axes, one batch and head count, unit stride on the head dim, nothing expanded
// (the tensor-core kernels address q, k, v by absolute (batch, head)); bias and mask with each axis 1 or full.
bool operands_fit(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& bias, const MaybeTensor& mask) {
  for (const Tensor* t : {&q, &k, &v})
    if (t->dim() != 4 || !t->is_cuda() || t->device() != q.device() || t->scalar_type() != q.scalar_type() ||
        t->size(0) != q.size(0) || t->size(1) != q.size(1) || t->stride(3) != 1 || has_expanded_axis(*t))
      return false;
  if (dtype_code(q.scalar_type()) < 0 || k.size(2) != v.size(2) || k.size(3) != q.size(3)) return false;
  const int64_t full[4] = {q.size(0), q.size(1), q.size(2), k.size(2)};
  for (const MaybeTensor* t : {&bias, &mask}) {
    if (!*t) continue;
    if ((*t)->dim() != 4 || (*t)->device() != q.device()) return false;
    for (int a = 0; a < 4; ++a)
      if ((*t)->size(a) != 1 && (*t)->size(a) != full[a]) return false;
  }
  if (bias && dtype_code(bias->scalar_type()) < 0) return false;
  return !mask || mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte;
}

// (out, lse, true); or without tensors: false where the operands have to be brought into shape first, true where the problem
// leaves the tensor-core families and the caller has not allowed that.
using AttentionResult = std::tuple<MaybeTensor, MaybeTensor, bool>;
AttentionResult attention(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& bias, const MaybeTensor& mask,
                          double scale, bool causal, int64_t kernel, bool any_family) {
  refuse_tangents("scaled_dot_product_attention", q, k, v, bias);
  if (!operands_fit(q, k, v, bias, mask)) return {std::nullopt, std::nullopt, false};
  const c10::cuda::CUDAGuard guard(q.device());
  const Attention a{q, k, v, bias.value_or(Tensor()), mask.value_or(Tensor()), Tensor(), scale, causal, int(kernel), {}};
  int family = NB200_KERNEL_SIMT;
  if (kernel == NB200_KERNEL_AUTO) {
    family = a.plan(NB200_PASS_FWD, false);
    if (!any_family && family != NB200_KERNEL_TCGEN05 && family != NB200_KERNEL_MMA_TF32X3) return {std::nullopt, std::nullopt, true};
  }
  if (c10::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad() || (bias && bias->requires_grad()))) {
    tensor_list r = AttentionRule::apply(q, k, v, bias, mask, scale, causal, kernel, family == NB200_KERNEL_TCGEN05);
    return {r[0], r[1], true};
  }
  auto [out, lse] = a.forward();
  return {out, lse, true};
}

// ---- QK-norm pre-op ------------------------------------------------------------------------------------------------------
// x viewed as (B, H, N, D), leading axes flattened
nb200_qk_norm_tensor norm_desc(const Tensor& x, const Tensor& y, const Tensor& g) {
  const Tensor x4 = x.dim() == 4 ? x : x.reshape({-1, x.size(-3), x.size(-2), x.size(-1)});
  nb200_qk_norm_tensor t{};
  t.x = x4.data_ptr();
  t.y = y.data_ptr();
  t.g = g.defined() ? g.data_ptr() : nullptr;
  for (int a = 0; a < 3; ++a) t.xs[a] = x4.stride(a);
  t.B = int32_t(x4.size(0)); t.H = int32_t(x4.size(1)); t.N = int32_t(x4.size(2));
  return t;
}

struct QkNormRule : torch::autograd::Function<QkNormRule> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k) {
    const Tensor qn = dense_like(q), kn = dense_like(k);
    const nb200_qk_norm_tensor dq = norm_desc(q, qn, Tensor()), dk = norm_desc(k, kn, Tensor());
    check(lib.nb200_qk_rms_norm(&dq, &dk, int(q.size(-1)), dtype_code(q.scalar_type()), stream_of(q)), "nb200_qk_rms_norm");
    ctx->save_for_backward({q, k});
    return {qn, kn};
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor q = s[0], k = s[1];
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor gq = grads[0].contiguous().to(q.scalar_type()), gk = grads[1].contiguous().to(k.scalar_type());
    const Tensor dq = dense_like(q), dk = dense_like(k);
    const nb200_qk_norm_tensor tq = norm_desc(q, dq, gq), tk = norm_desc(k, dk, gk);
    check(lib.nb200_qk_rms_norm_grad(&tq, &tk, int(q.size(-1)), dtype_code(q.scalar_type()), stream_of(q)), "nb200_qk_rms_norm_grad");
    return {dq, dk};
  }
};

// The kernel's layout rules: same device, type and head dim, rows of 16-byte words.
bool qk_norm_fits(const Tensor& q, const Tensor& k) {
  if (!q.is_cuda() || !k.is_cuda() || q.device() != k.device() || q.scalar_type() != k.scalar_type() ||
      dtype_code(q.scalar_type()) < 0 || q.dim() < 3 || k.dim() < 3)
    return false;
  const int64_t d = q.size(-1), vec = 16 / int64_t(q.element_size());
  if (k.size(-1) != d || d % vec || d > 256) return false;
  for (const Tensor* z : {&q, &k}) {
    if (z->stride(-1) != 1 || reinterpret_cast<uintptr_t>(z->data_ptr()) % 16 || (z->dim() != 4 && !z->is_contiguous())) return false;
    for (int64_t a = z->dim() - 2; a >= std::max<int64_t>(0, z->dim() - 4); --a)
      if (z->stride(a) % vec) return false;
  }
  return true;
}

std::tuple<Tensor, Tensor> qk_norm(const Tensor& q, const Tensor& k) {
  const c10::cuda::CUDAGuard guard(q.device());
  refuse_tangents("qk_rms_norm", q, k);
  const tensor_list r = QkNormRule::apply(q, k);
  return {r[0], r[1]};
}

// ---- LayerNorm -----------------------------------------------------------------------------------------------------------
nb200_layer_norm_params norm_params(const Tensor& x2, const Tensor& weight, double eps, double out_scale) {
  nb200_layer_norm_params p{};
  p.struct_size = sizeof(p);
  p.rows = x2.size(0);
  p.channels = int32_t(x2.size(1));
  p.dtype = dtype_code(x2.scalar_type());
  p.eps = float(eps);
  p.out_scale = float(out_scale);
  p.x = x2.data_ptr();
  p.weight = weight.defined() ? weight.data_ptr() : nullptr;
  return p;
}

// Saves (x, weight, mean, rstd), returns (dx, dweight, dbias).
struct LayerNormRule : torch::autograd::Function<LayerNormRule> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                        double out_scale) {
    const Tensor x2 = x.reshape({-1, x.size(-1)}).contiguous();
    const Tensor w = weight ? weight->to(x.scalar_type()).contiguous() : Tensor();
    const Tensor b = bias ? bias->to(x.scalar_type()).contiguous() : Tensor();
    const Tensor y = dense_like(x2);
    const Tensor mean = at::empty({x2.size(0)}, x.options().dtype(at::kFloat)), rstd = dense_like(mean);
    nb200_layer_norm_params p = norm_params(x2, w, eps, out_scale);
    p.bias = b.defined() ? b.data_ptr() : nullptr;
    p.y = y.data_ptr();
    p.mean = mean.data_ptr<float>();
    p.rstd = rstd.data_ptr<float>();
    check(lib.nb200_layer_norm_fwd(&p, stream_of(x)), "nb200_layer_norm_fwd");
    ctx->save_for_backward({x2, w, mean, rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["out_scale"] = out_scale;
    ctx->saved_data["shape"] = x.sizes().vec();
    // the types that dweight and dbias leave in; -1: not wanted
    ctx->saved_data["dw"] = weight && weight->requires_grad() ? int64_t(weight->scalar_type()) : int64_t(-1);
    ctx->saved_data["db"] = bias && bias->requires_grad() ? int64_t(bias->scalar_type()) : int64_t(-1);
    return y.reshape(x.sizes());
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor x2 = s[0], mean = s[2], rstd = s[3];
    const c10::cuda::CUDAGuard guard(x2.device());
    const Tensor dy2 = grads[0].reshape(x2.sizes()).to(x2.scalar_type()).contiguous();
    const int64_t dw_type = ctx->saved_data["dw"].toInt(), db_type = ctx->saved_data["db"].toInt();
    Tensor dx = dense_like(x2), dw, db, ws;
    nb200_layer_norm_params p = norm_params(x2, s[1], ctx->saved_data["eps"].toDouble(), ctx->saved_data["out_scale"].toDouble());
    p.dy = dy2.data_ptr();
    p.dx = dx.data_ptr();
    p.mean = mean.data_ptr<float>();
    p.rstd = rstd.data_ptr<float>();
    if (dw_type >= 0) dw = at::empty({x2.size(1)}, x2.options());
    if (db_type >= 0) db = at::empty({x2.size(1)}, x2.options());
    if (dw.defined() || db.defined()) {
      size_t need = 0;
      check(lib.nb200_layer_norm_workspace_bytes(&p, &need), "nb200_layer_norm_workspace_bytes");
      ws = scratch(std::max<size_t>(need, 16), x2);
      p.workspace = ws.data_ptr();
      p.workspace_bytes = need;
      p.dweight = dw.defined() ? dw.data_ptr() : nullptr;
      p.dbias = db.defined() ? db.data_ptr() : nullptr;
    }
    check(lib.nb200_layer_norm_bwd(&p, stream_of(x2)), "nb200_layer_norm_bwd");
    if (dw.defined()) dw = dw.to(at::ScalarType(dw_type));
    if (db.defined()) db = db.to(at::ScalarType(db_type));
    return {dx.reshape(ctx->saved_data["shape"].toIntVector()), dw, db, Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, double out_scale) {
  const c10::cuda::CUDAGuard guard(x.device());
  refuse_tangents("layer_norm", x, weight, bias);
  return LayerNormRule::apply(x, weight, bias, eps, out_scale);
}

// ---- selective scan ------------------------------------------------------------------------------------------------------
nb200_selective_scan_params scan_params(const Tensor& x3, const Tensor& delta3, const Tensor& A, const Tensor& B3, const Tensor& C3,
                                        const Tensor& D) {
  nb200_selective_scan_params p{};
  p.struct_size = sizeof(p);
  p.batch = int32_t(x3.size(0)); p.length = int32_t(x3.size(1)); p.channels = int32_t(x3.size(2)); p.states = int32_t(A.size(1));
  p.dtype = dtype_code(x3.scalar_type());
  p.x = x3.data_ptr(); p.delta = delta3.data_ptr(); p.A = A.data_ptr(); p.B = B3.data_ptr(); p.C = C3.data_ptr();
  p.D = D.defined() ? D.data_ptr() : nullptr;
  return p;
}

// (..., l, n) broadcast over the leading axes of x and dense
Tensor broadcast_rows(const Tensor& t, const Tensor& x) {
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 2);
  shape.push_back(t.size(-2));
  shape.push_back(t.size(-1));
  return t.to(x.scalar_type()).expand(shape).reshape({-1, t.size(-2), t.size(-1)}).contiguous();
}
// gradient of an operand that was broadcast over the leading axes, in that operand's type
Tensor sum_to_operand(const Tensor& g3, at::IntArrayRef lead, at::IntArrayRef shape, int64_t type) {
  std::vector<int64_t> full(lead.begin(), lead.end());
  full.push_back(g3.size(-2));
  full.push_back(g3.size(-1));
  return at::sum_to(g3.reshape(full), shape).to(at::ScalarType(type));
}

// The backward's scratch comes from nitrix_b200.nn.ssm, which decides what a device without room for all of it gets.
PyObject* scan_allocator = nullptr;
// It gets the block with the bytes that are wanted and fills in the workspace.
Tensor scan_workspace(nb200_selective_scan_params& p, const Tensor& like) {
  check(lib.nb200_selective_scan_workspace_bytes(&p, &p.workspace_bytes), "nb200_selective_scan_workspace_bytes");
  py::gil_scoped_acquire gil;
  return py::reinterpret_borrow<py::object>(scan_allocator)(reinterpret_cast<uintptr_t>(&p), int(like.device().index())).cast<Tensor>();
}

// Saves the operands and the forward's checkpoints.
struct ScanRule : torch::autograd::Function<ScanRule> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                        const Tensor& C, const MaybeTensor& D, bool differentiate) {
    const auto dt = x.scalar_type();
    const Tensor x3 = x.reshape({-1, x.size(-2), x.size(-1)}).contiguous();
    const Tensor delta3 = delta.to(dt).reshape(x3.sizes()).contiguous();
    const Tensor B3 = broadcast_rows(B, x), C3 = broadcast_rows(C, x);
    const Tensor A2 = A.to(dt).contiguous(), D1 = D ? D->to(dt).contiguous() : Tensor();
    const Tensor y = dense_like(x3);
    nb200_selective_scan_params p = scan_params(x3, delta3, A2, B3, C3, D1);
    p.y = y.data_ptr();
    Tensor ck;
    if (differentiate) {
      size_t need = 0;
      check(lib.nb200_selective_scan_checkpoint_bytes(&p, &need), "nb200_selective_scan_checkpoint_bytes");
      ck = at::empty({std::max<int64_t>(int64_t(need) / 4, 1)}, x.options().dtype(at::kFloat));
      p.checkpoints = ck.data_ptr<float>();
    }
    check(lib.nb200_selective_scan_fwd(&p, stream_of(x)), "nb200_selective_scan_fwd");
    if (differentiate) {
      ctx->save_for_backward({x3, delta3, A2, B3, C3, D1, ck});
      ctx->saved_data["x"] = x.sizes().vec();
      ctx->saved_data["delta"] = delta.sizes().vec();
      ctx->saved_data["B"] = B.sizes().vec();
      ctx->saved_data["C"] = C.sizes().vec();
      ctx->saved_data["types"] = std::vector<int64_t>{int64_t(delta.scalar_type()), int64_t(A.scalar_type()), int64_t(B.scalar_type()),
                                                      int64_t(C.scalar_type()), D ? int64_t(D->scalar_type()) : int64_t(0)};
    }
    return y.reshape(x.sizes());
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor x3 = s[0], D1 = s[5];
    const c10::cuda::CUDAGuard guard(x3.device());
    const Tensor dy3 = grads[0].to(x3.scalar_type()).reshape(x3.sizes()).contiguous();
    const Tensor dx = dense_like(x3), ddelta = dense_like(x3), dA = dense_like(s[2]), dB = dense_like(s[3]), dC = dense_like(s[4]);
    const Tensor dD = D1.defined() ? dense_like(D1) : Tensor();
    nb200_selective_scan_params p = scan_params(x3, s[1], s[2], s[3], s[4], D1);
    p.checkpoints = s[6].data_ptr<float>();
    p.dy = dy3.data_ptr();
    p.dx = dx.data_ptr(); p.ddelta = ddelta.data_ptr(); p.dA = dA.data_ptr(); p.dB = dB.data_ptr(); p.dC = dC.data_ptr();
    p.dD = dD.defined() ? dD.data_ptr() : nullptr;
    const Tensor ws = scan_workspace(p, x3);
    check(lib.nb200_selective_scan_bwd(&p, stream_of(x3)), "nb200_selective_scan_bwd");
    const auto xs = ctx->saved_data["x"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
    const at::IntArrayRef lead(xs.data(), xs.size() - 2);
    return {dx.reshape(xs),
            ddelta.reshape(ctx->saved_data["delta"].toIntVector()).to(at::ScalarType(types[0])),
            dA.to(at::ScalarType(types[1])),
            sum_to_operand(dB, lead, ctx->saved_data["B"].toIntVector(), types[2]),
            sum_to_operand(dC, lead, ctx->saved_data["C"].toIntVector(), types[3]),
            dD.defined() ? dD.to(at::ScalarType(types[4])) : Tensor(),
            Tensor()};
  }
};

Tensor selective_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const MaybeTensor& D) {
  const c10::cuda::CUDAGuard guard(x.device());
  refuse_tangents("selective_scan", x, delta, A, B, C, D);
  bool differentiate = false;
  if (c10::GradMode::is_enabled()) {
    for (const Tensor* t : {&x, &delta, &A, &B, &C}) differentiate = differentiate || t->requires_grad();
    differentiate = differentiate || (D && D->requires_grad());
  }
  return ScanRule::apply(x, delta, A, B, C, D, differentiate);
}

// ---- checks that the operators of a decoder layer share --------------------------------------------------------------------
void check_float(const char* what, const char* name, const Tensor& t) {
  TORCH_CHECK_TYPE(t.is_cuda() && dtype_code(t.scalar_type()) >= 0, what, ": ", name, " must be a CUDA tensor of float32, bfloat16 or float16; got ",
                   t.scalar_type(), " on ", t.device());
}
// extents that the library takes as 32-bit numbers
void check_extents(const char* what, const Tensor& t) {
  for (int64_t n : t.sizes()) TORCH_CHECK_VALUE(n <= std::numeric_limits<int32_t>::max(), what, ": an axis of ", n, " elements does not fit 32 bits");
}
void check_ints(const char* what, const char* name, const Tensor& t, const Tensor& like, int64_t dims) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt && t.device() == like.device(), what, ": ", name, " must be int32 on ", like.device(), "; got ",
                   t.scalar_type(), " on ", t.device());
  TORCH_CHECK_VALUE(t.dim() == dims, what, ": ", name, " must have ", dims, " axes; got shape ", t.sizes());
  check_extents(what, t);
}
// rows along the last axis that begin on 16-byte boundaries, none of them shared
Tensor aligned_rows(const Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && !has_expanded_axis(t);
  for (int64_t a = 0; a + 1 < t.dim(); ++a) ok = ok && t.stride(a) * int64_t(t.element_size()) % 16 == 0;
  if (ok) return t;
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// ---- root-mean-square norm ----------------------------------------------------------------------------------------------------
// (rows, channels), dense; on a 16-byte boundary where the rows are of 16-byte words
Tensor dense_rows(const Tensor& t, int64_t channels) {
  const Tensor r = t.reshape({-1, channels}).contiguous();
  const bool words = channels * int64_t(r.element_size()) % 16 == 0;
  return words && reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 ? r.clone() : r;
}

nb200_rms_norm_params rms_params(const Tensor& x2, const Tensor& weight, double eps) {
  nb200_rms_norm_params p{};
  p.struct_size = sizeof(p);
  p.rows = x2.size(0);
  p.channels = int32_t(x2.size(1));
  p.dtype = dtype_code(x2.scalar_type());
  p.weight_dtype = weight.defined() ? dtype_code(weight.scalar_type()) : p.dtype;
  p.eps = float(eps);
  p.x = x2.data_ptr();
  p.weight = weight.defined() ? weight.data_ptr() : nullptr;
  return p;
}

// (y or codes, the sum of the streams, rstd, scales); rstd for a backward pass, scales with codes alone
struct RmsNorm {
  Tensor y, sum, rstd, scales;
};
RmsNorm rms_norm_forward(const Tensor& x, const MaybeTensor& residual, const Tensor& weight, double eps, bool with_rstd, bool eight, int64_t group) {
  const int64_t C = x.size(-1);
  const Tensor x2 = dense_rows(x, C), r2 = residual ? dense_rows(*residual, C) : Tensor();
  RmsNorm n;
  n.y = at::empty(x.sizes(), eight ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  if (residual) n.sum = at::empty(x.sizes(), x.options());
  if (with_rstd) n.rstd = at::empty({x2.size(0)}, x.options().dtype(at::kFloat));
  if (eight) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = group ? C / group : 1;
    n.scales = at::empty(shape, x.options().dtype(at::kFloat));
  }
  nb200_rms_norm_params p = rms_params(x2, weight, eps);
  p.residual = residual ? r2.data_ptr() : nullptr;
  p.y = n.y.data_ptr();
  p.sum = n.sum.defined() ? n.sum.data_ptr() : nullptr;
  p.rstd = n.rstd.defined() ? n.rstd.data_ptr<float>() : nullptr;
  p.scales = n.scales.defined() ? n.scales.data_ptr<float>() : nullptr;
  p.group = int32_t(group);
  check(lib.nb200_rms_norm_fwd(&p, stream_of(x)), "nb200_rms_norm_fwd");
  return n;
}

// Saves (h, weight, rstd), where h is x or the sum, returns (dx, dweight); the gradients of the two streams are one tensor.
struct RmsNormRule : torch::autograd::Function<RmsNormRule> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, double eps) {
    const Tensor w = weight ? aligned_rows(*weight) : Tensor();
    const RmsNorm n = rms_norm_forward(x, residual, w, eps, true, false, 0);
    ctx->save_for_backward({residual ? n.sum : x, w, n.rstd});
    ctx->saved_data["dw"] = weight && weight->requires_grad();
    ctx->set_materialize_grads(false);
    if (residual) return {n.y, n.sum};
    return {n.y};
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const Tensor gy = grads[0], gs = grads.size() > 1 ? grads[1] : Tensor();
    tensor_list d(4);
    if (!gy.defined() && !gs.defined()) return d;
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    const int64_t C = s[0].size(-1);
    const Tensor h2 = dense_rows(s[0], C), w = s[1].defined() ? aligned_rows(s[1]) : Tensor(), rstd = s[2].contiguous();
    const bool want_dw = ctx->saved_data["dw"].toBool();
    Tensor dx, dw;
    if (!gy.defined()) {      // (only the sum was used)
      dx = gs;
    } else {
      const Tensor dy = dense_rows(gy.to(h2.scalar_type()), C), ds = gs.defined() ? dense_rows(gs.to(h2.scalar_type()), C) : Tensor();
      dx = at::empty(s[0].sizes(), h2.options());
      nb200_rms_norm_params p = rms_params(h2, w, 0.0);
      p.dy = dy.data_ptr();
      p.dsum = ds.defined() ? ds.data_ptr() : nullptr;
      p.dx = dx.data_ptr();
      p.rstd = rstd.data_ptr<float>();
      Tensor ws;
      if (want_dw) {
        dw = at::empty({C}, w.options());
        check(lib.nb200_rms_norm_workspace_bytes(&p, &p.workspace_bytes), "nb200_rms_norm_workspace_bytes");
        ws = scratch(std::max<size_t>(p.workspace_bytes, 16), h2);
        p.workspace = ws.data_ptr();
        p.dweight = dw.data_ptr();
      }
      check(lib.nb200_rms_norm_bwd(&p, stream_of(h2)), "nb200_rms_norm_bwd");
    }
    d[0] = dx;
    if (grads.size() > 1) d[1] = dx;      // (a residual that is left out has no gradient)
    d[2] = dw;
    return d;
  }
};

void check_rms_operands(const char* what, const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight) {
  check_float(what, "x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, what, ": x must have a channel at least; got shape ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) <= int64_t(1) << 30, what, ": ", x.size(-1), " channels, at most 2^30");
  if (residual) {
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type() && residual->device() == x.device(), what, ": residual must be ", x.scalar_type(), " on ",
                     x.device(), "; got ", residual->scalar_type(), " on ", residual->device());
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), what, ": residual must have shape ", x.sizes(), "; got ", residual->sizes());
  }
  if (weight) {
    TORCH_CHECK_TYPE((weight->scalar_type() == x.scalar_type() || weight->scalar_type() == at::kFloat) && weight->device() == x.device(), what,
                     ": weight must be ", x.scalar_type(), " or Float on ", x.device(), "; got ", weight->scalar_type(), " on ", weight->device());
    TORCH_CHECK_VALUE(weight->dim() == 1 && weight->size(0) == x.size(-1), what, ": weight must have shape (", x.size(-1), ",); got ", weight->sizes());
  }
  refuse_tangents(what, x, residual, weight);
}

// (y, sum of the streams)
std::tuple<Tensor, MaybeTensor> rms_norm(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, double eps) {
  check_rms_operands("rms_norm", x, residual, weight);
  const c10::cuda::CUDAGuard guard(x.device());
  if (c10::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad()) || (weight && weight->requires_grad()))) {
    const tensor_list r = RmsNormRule::apply(x, residual, weight, eps);
    return {r[0], residual ? MaybeTensor(r[1]) : std::nullopt};
  }
  const RmsNorm n = rms_norm_forward(x, residual, weight ? aligned_rows(*weight) : Tensor(), eps, false, false, 0);
  return {n.y, residual ? MaybeTensor(n.sum) : std::nullopt};
}

// (codes, scales, sum of the streams); group 0: a scale per row
std::tuple<Tensor, Tensor, MaybeTensor> rms_norm_quantized(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, double eps, int64_t group) {
  const char* what = "rms_norm_quantized";
  check_rms_operands(what, x, residual, weight);
  TORCH_CHECK_VALUE(group == 0 || ((group == 32 || group == 64 || group == 128) && x.size(-1) % group == 0), what,
                    ": group_size must be 32, 64 or 128 and divide the ", x.size(-1), " channels; got ", group);
  TORCH_CHECK_NOT_IMPLEMENTED(!(c10::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad()) || (weight && weight->requires_grad()))),
                              what, " is not differentiable; rms_norm is");
  const c10::cuda::CUDAGuard guard(x.device());
  const RmsNorm n = rms_norm_forward(x, residual, weight ? aligned_rows(*weight) : Tensor(), eps, false, true, group);
  return {n.y, n.scales, residual ? MaybeTensor(n.sum) : std::nullopt};
}

// ---- rotary positions -------------------------------------------------------------------------------------------------------
// x (..., heads, D) as (B, S, heads, D); the result is dense
void rotary_operand(nb200_rotary_tensor& t, const Tensor& x4, const Tensor& y) {
  t.x = x4.data_ptr();
  t.y = y.data_ptr();
  for (int a = 0; a < 3; ++a) t.x_stride[a] = x4.stride(a);
  t.heads = int32_t(x4.size(2));
}
Tensor two_leading_axes(const Tensor& x) {
  const Tensor r = x.stride(-1) == 1 ? x : x.contiguous();
  if (r.dim() == 4) return r;
  if (r.dim() == 3) return r.unsqueeze(0);
  return r.reshape({1, -1, r.size(-2), r.size(-1)});
}

tensor_list rotate(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& frequencies, at::IntArrayRef sections,
                   bool interleaved, bool inverse) {
  const Tensor& any = q.defined() ? q : k;
  nb200_rotary_params p{};
  p.struct_size = sizeof(p);
  tensor_list out(2);
  Tensor held[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor& x = i ? k : q;
    if (!x.defined()) continue;
    held[i] = two_leading_axes(x);
    check_extents("rotary_embedding", held[i]);
    out[i] = at::empty(x.sizes(), x.options());
    rotary_operand(i ? p.k : p.q, held[i], out[i]);
    p.batch = int32_t(held[i].size(0));
    p.length = int32_t(held[i].size(1));
  }
  if (p.batch == 0 || p.length == 0) return out;
  p.positions = positions.data_ptr();
  p.frequencies = frequencies.data_ptr<float>();
  p.head_dim = int32_t(any.size(-1));
  p.axes = int32_t(sections.size());
  for (size_t a = 0; a < sections.size(); ++a) p.sections[a] = int32_t(sections[a]);
  p.position_dtype = positions.scalar_type() == at::kInt ? NB200_POS_I32 : positions.scalar_type() == at::kLong ? NB200_POS_I64 : NB200_POS_F32;
  p.dtype = dtype_code(any.scalar_type());
  p.interleaved = interleaved;
  p.inverse = inverse;
  check(lib.nb200_rotary(&p, stream_of(any)), "nb200_rotary");
  return out;
}

// Saves the positions and frequencies; the gradient turns back.
struct RotaryRule : torch::autograd::Function<RotaryRule> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k, const Tensor& positions, const Tensor& frequencies,
                             std::vector<int64_t> sections, bool interleaved) {
    tensor_list out = rotate(q, k.value_or(Tensor()), positions, frequencies, sections, interleaved, false);
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    if (!k) out.pop_back();
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const Tensor gq = grads[0], gk = grads.size() > 1 ? grads[1] : Tensor();
    tensor_list d(6);
    if (!gq.defined() && !gk.defined()) return d;
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    const tensor_list r = rotate(gq, gk, s[0].contiguous(), s[1].contiguous(), ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(), true);
    d[0] = r[0];
    d[1] = r[1];
    return d;
  }
};

std::tuple<Tensor, MaybeTensor> rotary(const Tensor& q, const MaybeTensor& k, const Tensor& positions, const Tensor& frequencies,
                                       std::vector<int64_t> sections, bool interleaved) {
  const char* what = "rotary_embedding";
  check_float(what, "q", q);
  TORCH_CHECK_VALUE(q.dim() >= 3, what, ": q must be (..., heads, head_dim); got shape ", q.sizes());
  check_extents(what, q);
  const c10::cuda::CUDAGuard guard(q.device());
  if (sections.empty()) sections.push_back(frequencies.numel());
  TORCH_CHECK_VALUE(sections.size() <= NB200_ROTARY_MAX_AXES, what, ": at most ", NB200_ROTARY_MAX_AXES, " axes; got ", sections.size());
  int64_t pairs = 0;
  for (int64_t n : sections) {
    TORCH_CHECK_VALUE(n >= 0, what, ": a section has ", n, " pairs");
    pairs += n;
  }
  const int64_t D = q.size(-1), axes = int64_t(sections.size());
  TORCH_CHECK_VALUE(2 * pairs <= D, what, ": ", pairs, " pairs do not fit head dim ", D);
  TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kFloat && frequencies.device() == q.device(), what, ": frequencies must be float32 on ",
                   q.device(), "; got ", frequencies.scalar_type(), " on ", frequencies.device());
  TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.size(0) == pairs, what, ": frequencies must have shape (", pairs, ",); got ", frequencies.sizes());
  const auto pt = positions.scalar_type();
  TORCH_CHECK_TYPE((pt == at::kInt || pt == at::kLong || pt == at::kFloat) && positions.device() == q.device(), what,
                   ": positions must be int32, int64 or float32 on ", q.device(), "; got ", pt, " on ", positions.device());
  const at::IntArrayRef lead = q.sizes().slice(0, q.dim() - 2);
  const bool with_axis = positions.dim() == int64_t(lead.size()) + 1 && positions.size(-1) == axes && positions.sizes().slice(0, lead.size()) == lead;
  TORCH_CHECK_VALUE(with_axis || (axes == 1 && positions.sizes() == lead), what, ": positions must have shape ", lead, " + (", axes, ",); got ", positions.sizes());
  if (k) {
    check_float(what, "k", *k);
    TORCH_CHECK_TYPE(k->scalar_type() == q.scalar_type() && k->device() == q.device(), what, ": k must be ", q.scalar_type(), " on ", q.device());
    TORCH_CHECK_VALUE(k->dim() == q.dim() && k->size(-1) == D && k->sizes().slice(0, lead.size()) == lead, what, ": k must be ", lead,
                      " + (heads, ", D, "); got ", k->sizes());
  }
  TORCH_CHECK_VALUE(!positions.requires_grad() && !frequencies.requires_grad(), what, ": positions and frequencies are not differentiable");
  refuse_tangents(what, q, k, positions, frequencies);
  const Tensor pos = positions.contiguous(), freq = frequencies.contiguous();
  if (c10::GradMode::is_enabled() && (q.requires_grad() || (k && k->requires_grad()))) {
    const tensor_list r = RotaryRule::apply(q, k, pos, freq, sections, interleaved);
    return {r[0], k ? MaybeTensor(r[1]) : std::nullopt};
  }
  const tensor_list r = rotate(q, k.value_or(Tensor()), pos, freq, sections, interleaved, false);
  return {r[0], k ? MaybeTensor(r[1]) : std::nullopt};
}

// ---- paged cache --------------------------------------------------------------------------------------------------------------
// `k_steps`: those of a cache in few bits, whose pages hold codes
void check_pool(const char* what, const Tensor& k_pages, const MaybeTensor& k_steps) {
  if (!k_steps) return check_float(what, "k_pages", k_pages);
  TORCH_CHECK_TYPE(k_pages.is_cuda() && k_pages.scalar_type() == at::kByte, what, ": k_codes must be a CUDA tensor of uint8; got ", k_pages.scalar_type(), " on ",
                   k_pages.device());
}

// The pages of a cache, or its codes and steps.
struct CachePages {
  nb200_cache_pages pages{};
  nb200_cache_steps steps{};

  bool coded() const { return steps.bits != 0; }
  CachePages(const char* what, const Tensor& k_pages, const Tensor& v_pages, const MaybeTensor& k_steps, const MaybeTensor& v_steps) {
    const char* names = k_steps ? "k_codes and v_codes" : "k_pages and v_pages";
    TORCH_CHECK_TYPE(v_pages.scalar_type() == k_pages.scalar_type() && v_pages.device() == k_pages.device(), what,
                     k_steps ? ": v_codes must be like k_codes" : ": v_pages must be like k_pages");
    TORCH_CHECK_VALUE(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes(), what, ": ", names, " must have one shape (pages, heads, page size, ",
                      k_steps ? "bytes" : "head dim", "); got ", k_pages.sizes(), " and ", v_pages.sizes());
    TORCH_CHECK_VALUE(k_pages.size(1) > 0 && k_pages.size(2) > 0 && k_pages.size(3) > 0, what, ": a page must hold a token at least; got shape ", k_pages.sizes());
    check_extents(what, k_pages);
    const Tensor* t[2] = {&k_pages, &v_pages};
    for (int i = 0; i < 2; ++i) {
      // (written in place: a copy in another layout would not do)
      TORCH_CHECK_VALUE(t[i]->stride(3) == 1 && !has_expanded_axis(*t[i]), what, ": pages must have unit stride along the ", k_steps ? "bytes of a row" : "head dim",
                        " and no expanded axis");
      for (int a = 0; a < 3; ++a) (i ? pages.v_stride : pages.k_stride)[a] = t[i]->stride(a);
    }
    pages.k = k_pages.data_ptr();
    pages.v = v_pages.data_ptr();
    pages.pages = int32_t(k_pages.size(0)); pages.heads = int32_t(k_pages.size(1));
    pages.page_size = int32_t(k_pages.size(2)); pages.head_dim = int32_t(k_pages.size(3));
    pages.dtype = dtype_code(k_pages.scalar_type());
    if (!k_steps) return;
    TORCH_CHECK_VALUE(bool(v_steps), what, ": k_steps without v_steps");
    for (const MaybeTensor* x : {&k_steps, &v_steps}) {
      TORCH_CHECK_TYPE((*x)->scalar_type() == at::kHalf && (*x)->device() == k_pages.device(), what, ": steps must be float16 on ", k_pages.device(), "; got ",
                       (*x)->scalar_type(), " on ", (*x)->device());
      TORCH_CHECK_VALUE((*x)->dim() == 4 && (*x)->sizes() == k_steps->sizes() && (*x)->sizes().slice(0, 3) == k_pages.sizes().slice(0, 3) && (*x)->size(3) > 0, what,
                        ": k_steps and v_steps must have one shape (", k_pages.size(0), ", ", k_pages.size(1), ", ", k_pages.size(2), ", groups); got ", (*x)->sizes());
      TORCH_CHECK_VALUE((*x)->stride(3) == 1 || (*x)->size(3) == 1, what, ": steps must have unit stride along the groups");
      TORCH_CHECK_VALUE(!has_expanded_axis(**x), what, ": steps must have no expanded axis");
    }
    const int64_t groups = k_steps->size(3), row = k_pages.size(3);
    steps.bits = row == 16 * groups ? 4 : row == 32 * groups ? 8 : 0;
    TORCH_CHECK_VALUE(steps.bits != 0, what, ": ", groups, " groups of 32 elements take ", 16 * groups, " bytes in 4 bits or ", 32 * groups, " in 8; the rows of codes have ", row);
    pages.head_dim = int32_t(32 * groups);
    steps.k = k_steps->data_ptr();
    steps.v = v_steps->data_ptr();
    for (int a = 0; a < 3; ++a) { steps.k_stride[a] = k_steps->stride(a); steps.v_stride[a] = v_steps->stride(a); }
  }
};

// Raises the version of what a call has written in place, by which autograd notices that a saved tensor is no longer what it was.
// (Inference tensors have none.)
template <typename... T>
void written(const T&... tensors) {
  for (const Tensor* t : {&tensors...})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

struct CacheCall {
  nb200_cache_quantized_params q{};      // p with what a cache in few bits has beside it
  nb200_cache_params& p = q.cache;
  Tensor lengths, free_pages, free_range;
  const char* what;

  CacheCall(const char* name, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths_in,
            const Tensor& free_pages_in, const Tensor& free_range_in, const MaybeTensor& k_steps, const MaybeTensor& v_steps)
      : what(name) {
    q.struct_size = sizeof(q);
    p.struct_size = sizeof(p);
    const CachePages c(what, k_pages, v_pages, k_steps, v_steps);
    p.pages = c.pages;
    if (c.coded()) p.pages.dtype = NB200_F16;      // (of the new tokens: append says which; else of no meaning)
    q.steps = c.steps;
    check_ints(what, "table", table, k_pages, 2);
    check_ints(what, "lengths", lengths_in, k_pages, 1);
    check_ints(what, "free_pages", free_pages_in, k_pages, 1);
    check_ints(what, "free_range", free_range_in, k_pages, 1);
    TORCH_CHECK_VALUE(table.is_contiguous(), what, ": table must be contiguous");
    TORCH_CHECK_VALUE(lengths_in.size(0) == table.size(0), what, ": ", table.size(0), " rows, but lengths of shape ", lengths_in.sizes());
    TORCH_CHECK_VALUE(table.size(1) > 0, what, ": the table's rows must hold a page at least");
    TORCH_CHECK_VALUE(free_pages_in.size(0) == k_pages.size(0) && free_range_in.size(0) == 2, what, ": free_pages must have shape (", k_pages.size(0),
                      ",) and free_range (2,)");
    lengths = lengths_in.contiguous();
    free_pages = free_pages_in.contiguous();
    free_range = free_range_in.contiguous();
    p.table = table.data_ptr<int32_t>();
    p.lengths = lengths.data_ptr<int32_t>();
    p.free_pages = free_pages.data_ptr<int32_t>();
    p.free_range = free_range.data_ptr<int32_t>();
    p.rows = int32_t(table.size(0));
    p.width = int32_t(table.size(1));
  }
  Tensor ints(int64_t n) const { return at::empty({n}, lengths.options()); }
  Tensor workspace() {
    size_t need = 0;
    check(lib.nb200_cache_workspace_bytes(&p, &need), "nb200_cache_workspace_bytes");
    Tensor ws = scratch(need, lengths);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
    return ws;
  }
  void run(int (*plain)(const nb200_cache_params*, void*), int (*quantized)(const nb200_cache_quantized_params*, void*), const Tensor& on) const {
    const std::string name = std::string("nb200_") + what;
    if (q.steps.bits) check(quantized(&q, stream_of(on)), (name + "_quantized").c_str());
    else check(plain(&p, stream_of(on)), name.c_str());
  }
};

// (lengths, free_range, shortfall)
std::tuple<Tensor, Tensor, Tensor> cache_append(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                                                const Tensor& free_pages, const Tensor& free_range, const Tensor& k, const Tensor& v,
                                                const Tensor& offsets, const MaybeTensor& k_steps, const MaybeTensor& v_steps) {
  const char* what = "cache_append";
  check_pool(what, k_pages, k_steps);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  CacheCall c(what, k_pages, v_pages, table, lengths, free_pages, free_range, k_steps, v_steps);
  if (k_steps) {      // (quantised from any of the three types)
    check_float(what, "k", k);
    c.p.pages.dtype = dtype_code(k.scalar_type());
  }
  const at::ScalarType type = k_steps ? k.scalar_type() : k_pages.scalar_type();
  for (const Tensor* t : {&k, &v}) {
    TORCH_CHECK_TYPE(t->scalar_type() == type && t->device() == k_pages.device(), what, ": k and v must be ", type, " on ", k_pages.device());
    TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == k.size(0) && t->size(1) == k_pages.size(1) && t->size(2) == c.p.pages.head_dim, what,
                      ": k and v must be (tokens, ", k_pages.size(1), ", ", c.p.pages.head_dim, "); got ", t->sizes());
  }
  check_ints(what, "offsets", offsets, k_pages, 1);
  TORCH_CHECK_VALUE(table.size(0) > 0 && offsets.size(0) == table.size(0) + 1, what, ": ", table.size(0), " rows, but offsets of shape ", offsets.sizes());
  refuse_tangents(what, k, v, k_pages, v_pages);
  const Tensor kr = aligned_rows(k), vr = aligned_rows(v), off = offsets.contiguous();
  const Tensor new_lengths = c.ints(table.size(0)), new_range = c.ints(2), shortfall = c.ints(1);
  c.p.new_k = kr.data_ptr();
  c.p.new_v = vr.data_ptr();
  for (int a = 0; a < 2; ++a) { c.p.new_k_stride[a] = kr.stride(a); c.p.new_v_stride[a] = vr.stride(a); }
  c.p.offsets = off.data_ptr<int32_t>();
  c.p.tokens = k.size(0);
  c.p.new_lengths = new_lengths.data_ptr<int32_t>();
  c.p.new_free_range = new_range.data_ptr<int32_t>();
  c.p.shortfall = shortfall.data_ptr<int32_t>();
  c.run(lib.nb200_cache_append, lib.nb200_cache_append_quantized, k_pages);
  if (k.size(0) > 0) {
    written(k_pages, v_pages, table);
    if (k_steps) written(*k_steps, *v_steps);
  }
  return {new_lengths, new_range, shortfall};
}

// (table, lengths, free_pages, free_range, shortfall); `rows`: parents (int32), or which rows are finished (bool)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> cache_fork(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                                                              const Tensor& free_pages, const Tensor& free_range, const Tensor& rows, bool finished,
                                                              const MaybeTensor& k_steps, const MaybeTensor& v_steps) {
  const char* what = finished ? "cache_free" : "cache_fork";
  check_pool(what, k_pages, k_steps);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  CacheCall c(what, k_pages, v_pages, table, lengths, free_pages, free_range, k_steps, v_steps);
  const Tensor r = rows.contiguous();
  if (finished) {
    TORCH_CHECK_TYPE(r.scalar_type() == at::kBool && r.device() == k_pages.device(), what, ": finished must be bool on ", k_pages.device());
    TORCH_CHECK_VALUE(r.dim() == 1 && r.size(0) == table.size(0), what, ": finished must have shape (", table.size(0), ",); got ", r.sizes());
    c.p.finished = static_cast<const uint8_t*>(r.data_ptr());
  } else {
    check_ints(what, "parents", r, k_pages, 1);
    c.p.parents = r.data_ptr<int32_t>();
  }
  const int64_t n = r.size(0);
  c.p.new_rows = int32_t(n);
  const Tensor new_table = at::empty({n, table.size(1)}, table.options()), new_lengths = c.ints(n), new_free = c.ints(k_pages.size(0)),
               new_range = c.ints(2), shortfall = c.ints(1);
  c.p.new_table = new_table.data_ptr<int32_t>();
  c.p.new_lengths = new_lengths.data_ptr<int32_t>();
  c.p.new_free_pages = new_free.data_ptr<int32_t>();
  c.p.new_free_range = new_range.data_ptr<int32_t>();
  c.p.shortfall = shortfall.data_ptr<int32_t>();
  const Tensor ws = c.workspace();
  c.run(lib.nb200_cache_fork, lib.nb200_cache_fork_quantized, k_pages);
  if (!finished) {      // (rows that stay, or become empty, copy nothing)
    written(k_pages, v_pages);
    if (k_steps) written(*k_steps, *v_steps);
  }
  return {new_table, new_lengths, new_free, new_range, shortfall};
}

// (table, free_pages, free_range, shortfall)
std::tuple<Tensor, Tensor, Tensor, Tensor> cache_compact(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths,
                                                         const Tensor& free_pages, const Tensor& free_range, const MaybeTensor& k_steps,
                                                         const MaybeTensor& v_steps) {
  const char* what = "cache_compact";
  check_pool(what, k_pages, k_steps);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  CacheCall c(what, k_pages, v_pages, table, lengths, free_pages, free_range, k_steps, v_steps);
  const Tensor new_table = at::empty(table.sizes(), table.options()), new_free = c.ints(k_pages.size(0)), new_range = c.ints(2),
               shortfall = c.ints(1);
  c.p.new_table = new_table.data_ptr<int32_t>();
  c.p.new_free_pages = new_free.data_ptr<int32_t>();
  c.p.new_free_range = new_range.data_ptr<int32_t>();
  c.p.shortfall = shortfall.data_ptr<int32_t>();
  const Tensor ws = c.workspace();
  c.run(lib.nb200_cache_compact, lib.nb200_cache_compact_quantized, k_pages);
  written(k_pages, v_pages);
  if (k_steps) written(*k_steps, *v_steps);
  return {new_table, new_free, new_range, shortfall};
}

Tensor decode_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths, double scale,
                        const MaybeTensor& k_steps, const MaybeTensor& v_steps) {
  const char* what = "decode_attention";
  check_pool(what, k_pages, k_steps);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  nb200_decode_quantized_params qp{};
  nb200_decode_params& p = qp.decode;
  qp.struct_size = sizeof(qp);
  p.struct_size = sizeof(p);
  const CachePages c(what, k_pages, v_pages, k_steps, v_steps);
  p.pages = c.pages;
  qp.steps = c.steps;
  if (c.coded()) {
    check_float(what, "q", q);
    p.pages.dtype = dtype_code(q.scalar_type());
  }
  const at::ScalarType type = c.coded() ? q.scalar_type() : k_pages.scalar_type();
  TORCH_CHECK_TYPE(q.scalar_type() == type && q.device() == k_pages.device(), what, ": q must be ", type, " on ", k_pages.device());
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == table.size(0) && q.size(2) == p.pages.head_dim && q.size(1) > 0 && q.size(1) % k_pages.size(1) == 0, what,
                    ": q must be (", table.size(0), ", a multiple of ", k_pages.size(1), ", ", p.pages.head_dim, "); got ", q.sizes());
  check_extents(what, q);
  check_ints(what, "table", table, k_pages, 2);
  check_ints(what, "lengths", lengths, k_pages, 1);
  TORCH_CHECK_VALUE(lengths.size(0) == table.size(0), what, ": ", table.size(0), " rows, but lengths of shape ", lengths.sizes());
  TORCH_CHECK_NOT_IMPLEMENTED(!(c10::GradMode::is_enabled() && (q.requires_grad() || k_pages.requires_grad() || v_pages.requires_grad() ||
                                                               (k_steps && (k_steps->requires_grad() || v_steps->requires_grad())))),
                              what, " is not differentiable; packed_attention is");
  refuse_tangents(what, q, k_pages, v_pages, k_steps, v_steps);
  const Tensor qr = aligned_rows(q), tab = table.contiguous(), len = lengths.contiguous();
  const Tensor out = at::empty(q.sizes(), q.options());
  p.table = tab.data_ptr<int32_t>();
  p.lengths = len.data_ptr<int32_t>();
  p.rows = int32_t(q.size(0));
  p.width = int32_t(table.size(1));
  p.q = qr.data_ptr();
  p.out = out.data_ptr();
  p.q_stride[0] = qr.stride(0);
  p.q_stride[1] = qr.stride(1);
  p.q_heads = int32_t(q.size(1));
  p.scale = float(scale);
  if (p.rows == 0) return out;
  if (c.coded()) check(lib.nb200_decode_quantized_workspace_bytes(&qp, &p.workspace_bytes), "nb200_decode_quantized_workspace_bytes");
  else check(lib.nb200_decode_workspace_bytes(&p, &p.workspace_bytes), "nb200_decode_workspace_bytes");
  const Tensor ws = scratch(p.workspace_bytes, q);
  p.workspace = ws.data_ptr();
  if (c.coded()) check(lib.nb200_decode_quantized(&qp, stream_of(q)), "nb200_decode_quantized");
  else check(lib.nb200_decode(&p, stream_of(q)), "nb200_decode");
  return out;
}

// (k, v) of `tokens` packed rows; codes become `type`, elements keep theirs
std::tuple<Tensor, Tensor> cache_read(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lengths, const Tensor& offsets,
                                      const MaybeTensor& starts, int64_t tokens, std::optional<at::ScalarType> type, const MaybeTensor& k_steps,
                                      const MaybeTensor& v_steps) {
  const char* what = "cache_read";
  check_pool(what, k_pages, k_steps);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  nb200_cache_read_params p{};
  p.struct_size = sizeof(p);
  const CachePages c(what, k_pages, v_pages, k_steps, v_steps);
  p.pages = c.pages;
  p.steps = c.steps;
  const at::ScalarType out = type ? *type : c.coded() ? at::kBFloat16 : k_pages.scalar_type();
  TORCH_CHECK_TYPE(dtype_code(out) >= 0 && (c.coded() || out == k_pages.scalar_type()), what, ": dtype must be ",
                   c.coded() ? "float32, bfloat16 or float16" : "that of the pages", "; got ", out);
  p.pages.dtype = dtype_code(out);
  check_ints(what, "table", table, k_pages, 2);
  check_ints(what, "lengths", lengths, k_pages, 1);
  check_ints(what, "offsets", offsets, k_pages, 1);
  TORCH_CHECK_VALUE(lengths.size(0) == table.size(0), what, ": ", table.size(0), " rows, but lengths of shape ", lengths.sizes());
  TORCH_CHECK_VALUE(offsets.size(0) == table.size(0) + 1, what, ": ", table.size(0), " rows, but offsets of shape ", offsets.sizes());
  if (starts) {
    check_ints(what, "starts", *starts, k_pages, 1);
    TORCH_CHECK_VALUE(starts->size(0) == table.size(0), what, ": ", table.size(0), " rows, but starts of shape ", starts->sizes());
  }
  TORCH_CHECK_VALUE(tokens >= 0 && tokens <= std::numeric_limits<int32_t>::max(), what, ": tokens must be a number of rows below 2^31; got ", tokens);
  TORCH_CHECK_NOT_IMPLEMENTED(!(c10::GradMode::is_enabled() && (k_pages.requires_grad() || v_pages.requires_grad() ||
                                                               (k_steps && (k_steps->requires_grad() || v_steps->requires_grad())))),
                              what, " is not differentiable");
  refuse_tangents(what, k_pages, v_pages, k_steps, v_steps);
  const Tensor tab = table.contiguous(), len = lengths.contiguous(), off = offsets.contiguous(), first = starts ? starts->contiguous() : Tensor();
  const Tensor k = at::empty({tokens, p.pages.heads, p.pages.head_dim}, k_pages.options().dtype(out)), v = at::empty(k.sizes(), k.options());
  p.table = tab.data_ptr<int32_t>();
  p.lengths = len.data_ptr<int32_t>();
  p.rows = int32_t(table.size(0));
  p.width = int32_t(table.size(1));
  p.offsets = off.data_ptr<int32_t>();
  p.starts = first.defined() ? first.data_ptr<int32_t>() : nullptr;
  p.out_k = k.data_ptr();
  p.out_v = v.data_ptr();
  p.tokens = tokens;
  check(lib.nb200_cache_read(&p, stream_of(k_pages)), "nb200_cache_read");
  return {k, v};
}

// ---- packed sequences ------------------------------------------------------------------------------------------------------
struct Packed {
  Tensor q, k, v, offsets_q, offsets_k;
  double scale;
  bool causal;
  int kernel;

  nb200_packed_params params() const {
    nb200_packed_params p{};
    p.struct_size = sizeof(p);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr();
    p.offsets_q = offsets_q.data_ptr<int32_t>();
    p.offsets_k = offsets_k.data_ptr<int32_t>();
    for (int a = 0; a < 2; ++a) { p.q_stride[a] = q.stride(a); p.k_stride[a] = k.stride(a); p.v_stride[a] = v.stride(a); }
    p.tokens_q = int32_t(q.size(0)); p.tokens_k = int32_t(k.size(0));
    p.sequences = int32_t(offsets_q.size(0) - 1);
    p.heads = int32_t(q.size(1)); p.kv_heads = int32_t(k.size(1)); p.head_dim = int32_t(q.size(2));
    p.dtype = dtype_code(q.scalar_type());
    p.causal = causal;
    p.scale = float(scale);
    p.kernel = kernel;
    return p;
  }
  int plan(int pass) const {
    nb200_packed_params p = params();
    p.dout_stride[0] = q.size(1) * q.size(2);      // (a cotangent is brought into rows that fit)
    p.dout_stride[1] = q.size(2);
    int chosen = 0;
    check(lib.nb200_packed_plan(&p, pass, &chosen), "nb200_packed_plan");
    return chosen;
  }
  Tensor workspace(nb200_packed_params& p, int pass) const {
    check(lib.nb200_packed_workspace_bytes(&p, pass, &p.workspace_bytes), "nb200_packed_workspace_bytes");
    Tensor ws;
    if (p.workspace_bytes) {
      ws = scratch(p.workspace_bytes, q);
      p.workspace = ws.data_ptr();
    }
    return ws;
  }
  std::pair<Tensor, Tensor> forward() const {
    const Tensor out = at::empty(q.sizes(), q.options());
    const Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    nb200_packed_params p = params();
    p.out = out.data_ptr();
    p.lse = lse.data_ptr<float>();
    const Tensor ws = workspace(p, NB200_PASS_FWD);
    check(lib.nb200_packed_fwd(&p, stream_of(q)), "nb200_packed_fwd");
    return {out, lse};
  }
  tensor_list backward(const Tensor& out, const Tensor& lse, const Tensor& grad) const {
    const Tensor dout = aligned_rows(grad);
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
    nb200_packed_params p = params();
    p.out = out.data_ptr();
    p.lse = lse.data_ptr<float>();
    p.dout = dout.data_ptr(); p.dq = dq.data_ptr(); p.dk = dk.data_ptr(); p.dv = dv.data_ptr();
    for (int a = 0; a < 2; ++a) p.dout_stride[a] = dout.stride(a);
    const Tensor ws = workspace(p, NB200_PASS_BWD);
    check(lib.nb200_packed_bwd(&p, stream_of(q)), "nb200_packed_bwd");
    return {dq, dk, dv};
  }
};

// Saves (q, k, v, offsets, out, lse), returns (dq, dk, dv).
struct PackedRule : torch::autograd::Function<PackedRule> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets_q, const Tensor& offsets_k,
                        double scale, bool causal, int64_t kernel) {
    auto [out, lse] = Packed{q, k, v, offsets_q, offsets_k, scale, causal, int(kernel)}.forward();
    ctx->save_for_backward({q, k, v, offsets_q, offsets_k, out, lse});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["flags"] = (kernel << 1) | int64_t(causal);
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, const tensor_list& grads) {
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    const int64_t flags = ctx->saved_data["flags"].toInt();
    // (a saved-tensor hook may hand the operands back in another layout)
    const Packed a{aligned_rows(s[0]), aligned_rows(s[1]), aligned_rows(s[2]), s[3].contiguous(), s[4].contiguous(),
                   ctx->saved_data["scale"].toDouble(), (flags & 1) != 0, int(flags >> 1)};
    tensor_list g = a.backward(s[5].contiguous(), s[6].contiguous(), grads[0].to(s[0].scalar_type()));
    g.resize(8);
    return g;
  }
};

// Without a tensor where the problem leaves the tensor-core family and the caller has not allowed that; whether it does so with its
// gradients only.
std::tuple<MaybeTensor, bool> packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, const MaybeTensor& offsets_k, double scale,
                             bool causal, int64_t kernel, bool any_family) {
  const char* what = "packed_attention";
  check_float(what, "q", q);
  const c10::cuda::CUDAGuard guard(q.device());
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK_TYPE(t->scalar_type() == q.scalar_type() && t->device() == q.device(), what, ": k and v must be ", q.scalar_type(), " on ", q.device());
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(2) == k.size(2), what,
                    ": q must be (tokens, heads, head dim), k and v (tokens, key heads, head dim); got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0, what, ": ", q.size(1), " query heads are no multiple of ", k.size(1), " key heads");
  check_extents(what, q);
  check_extents(what, k);
  check_ints(what, "offsets", offsets, q, 1);
  TORCH_CHECK_VALUE(offsets.size(0) >= 1, what, ": offsets must hold the number of sequences + 1 elements");
  if (offsets_k) {
    check_ints(what, "offsets_k", *offsets_k, q, 1);
    TORCH_CHECK_VALUE(offsets_k->sizes() == offsets.sizes(), what, ": offsets_k must have shape ", offsets.sizes(), "; got ", offsets_k->sizes());
  } else {
    TORCH_CHECK_VALUE(k.size(0) == q.size(0), what, ": ", q.size(0), " queries and ", k.size(0), " keys need offsets_k");
  }
  refuse_tangents(what, q, k, v);
  const Tensor oq = offsets.contiguous(), ok = offsets_k ? offsets_k->contiguous() : oq;
  const Packed a{aligned_rows(q), aligned_rows(k), aligned_rows(v), oq, ok, scale, causal, int(kernel)};
  const bool differentiate = c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  // (a batch without a query, a key or a sequence has nothing to compute in any family)
  if (kernel == NB200_KERNEL_AUTO && !any_family && q.size(0) > 0 && k.size(0) > 0 && offsets.size(0) > 1) {
    if (a.plan(NB200_PASS_FWD) != NB200_KERNEL_TCGEN05) return {std::nullopt, false};
    if (differentiate && a.plan(NB200_PASS_BWD) != NB200_KERNEL_TCGEN05) return {std::nullopt, true};
  }
  if (differentiate) return {PackedRule::apply(a.q, a.k, a.v, oq, ok, scale, causal, kernel), false};
  return {a.forward().first, false};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("entry_points", &entry_points);
  m.def("bind", &bind);
  // (torch's wrapper: its exception types, and no interpreter lock while the library is called)
  m.def("attention", torch::wrap_pybind_function_no_gil(attention));
  m.def("qk_norm_fits", torch::wrap_pybind_function(qk_norm_fits));
  m.def("qk_norm", torch::wrap_pybind_function_no_gil(qk_norm));
  m.def("layer_norm", torch::wrap_pybind_function_no_gil(layer_norm));
  m.def("set_scan_allocator", [](py::object allocator) { scan_allocator = allocator.release().ptr(); });   // (for good)
  m.def("selective_scan", torch::wrap_pybind_function_no_gil(selective_scan));
  m.def("rotary", torch::wrap_pybind_function_no_gil(rotary));
  m.def("cache_append", torch::wrap_pybind_function_no_gil(cache_append));
  m.def("cache_fork", torch::wrap_pybind_function_no_gil(cache_fork));
  m.def("cache_compact", torch::wrap_pybind_function_no_gil(cache_compact));
  m.def("decode_attention", torch::wrap_pybind_function_no_gil(decode_attention));
  m.def("cache_read", torch::wrap_pybind_function_no_gil(cache_read));
  m.def("rms_norm", torch::wrap_pybind_function_no_gil(rms_norm));
  m.def("rms_norm_quantized", torch::wrap_pybind_function_no_gil(rms_norm_quantized));
  m.def("packed_attention", torch::wrap_pybind_function_no_gil(packed_attention));
}
