// Attention of one new token per sequence over a paged cache in 4 or 8 bits, divided and joined as decode.cuh says.
//
//   s_t = scale q . k_t,  p = softmax(s),  out = sum_t p_t v_t,     k_t, v_t = step (code - 2^(b-1)) per group of 32 elements
//
// Bound by HBM: every code and step is read once, 72 bytes per 128 elements in 4 bits.
#include "cache_codes.cuh"
#include "decode.cuh"

namespace nb200 {
namespace {

struct QuantizedArgs : DecodeArgs {      // k, v: codes
  const uint16_t* k_steps;
  const uint16_t* v_steps;
  int kss[3], vss[3];      // head's rows of steps, over (page, head, slot)
  int groups;
};

__device__ __forceinline__ const uint16_t* steps_of(const uint16_t* base, const int (&stride)[3], int groups, int kv_head, Where w) {
  return base + (int64_t(w.page) * stride[0] + int64_t(kv_head) * stride[1] + int64_t(w.slot) * stride[2]) * groups;
}

// fp32 multiply-adds.  Eight lanes share a token, a part of its row of codes each; a warp's four groups take tokens of their own.
template <typename T, int kBits, int kGroups, int kNumHeads>
struct QuantizedFmaLoop {
  static constexpr const char* kName = "decode_kernel<quantized>";
  static constexpr int kHeads = kNumHeads;
  static constexpr int kSlots = 4;
  static constexpr int kMinCtas = 2;
  float o[kHeads][kGroups][4];
  float m[kHeads], l[kHeads];

  __device__ __forceinline__ void run(const QuantizedArgs& a, const int* row_table, int kv_head, const void* q_row, int heads, int t0, int t1,
                                      int wi, int wn) {
    const T* q = static_cast<const T*>(q_row);
    const int part = threadIdx.x & 7, first = wi * kSlots, mine = first + ((threadIdx.x & 31) >> 3), step = wn * kSlots;
    float qf[kHeads][kGroups][4];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qf[h][g][i] = h < heads && g < a.groups ? to_f32<T>(q[h * a.qs[1] + g * kGroup + part * 4 + i]) : 0.f;
          o[h][g][i] = 0.f;
        }
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
    const uint4* kbase = a.k + int64_t(kv_head) * a.ks[1];
    const uint4* vbase = a.v + int64_t(kv_head) * a.vs[1];
    // (all groups of a warp go round together: the shuffles are warp-wide; behind the last token that one's row is read again, with a
    // probability of zero)
    for (int b = t0; b + first < t1; b += step) {
      const Where at = where(a, row_table, min(b + mine, t1 - 1));
      const uint8_t* kr = reinterpret_cast<const uint8_t*>(row_of(kbase, a.ks, at));
      const uint8_t* vr = reinterpret_cast<const uint8_t*>(row_of(vbase, a.vs, at));
      const uint16_t* kt = steps_of(a.k_steps, a.kss, a.groups, kv_head, at);
      const uint16_t* vt = steps_of(a.v_steps, a.vss, a.groups, kv_head, at);
      float s[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) s[h] = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g >= a.groups) continue;
        float c[4];
        load_codes<kBits>(kr, a.groups, g, part, c);
        const float size = __half2float(__ushort_as_half(__ldg(kt + g)));
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) dot = fmaf(qf[h][g][i], c[i], dot);
          s[h] = fmaf(dot, size, s[h]);
        }
      }
      float p[kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], off);
        const float x = b + mine < t1 ? s[h] * a.mul : -INFINITY, m_new = fmaxf(m[h], x), shift = m_new == -INFINITY ? 0.f : m_new;
        const float old = ex2(m[h] - shift);
        p[h] = ex2(x - shift);
        l[h] = fmaf(l[h], old, p[h]);
        m[h] = m_new;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[h][g][i] *= old;
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g >= a.groups) continue;
        float c[4];
        load_codes<kBits>(vr, a.groups, g, part, c);
        const float size = __half2float(__ushort_as_half(__ldg(vt + g)));
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float w = p[h] * size;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[h][g][i] = fmaf(w, c[i], o[h][g][i]);
        }
      }
    }
  }

  __device__ __forceinline__ void store(const QuantizedArgs& a, float* dst) const {
    const int part = threadIdx.x & 7;
    float* slot = dst + (threadIdx.x >> 3) * kHeads * (a.D + 2);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float* row = slot + h * (a.D + 2);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (g < a.groups)
#pragma unroll
          for (int i = 0; i < 4; ++i) row[g * kGroup + part * 4 + i] = o[h][g][i];
      if (part == 0) {
        row[a.D] = m[h];
        row[a.D + 1] = l[h];
      }
    }
  }
};

struct Plan {
  int heads, side, chunks;      // query heads of a chunk, chunks side by side, times that a group is taken
  int unit, workers;
  size_t bytes;
};

int check(const nb200_decode_quantized_params* p, const char* what) {
  if (!p || p->struct_size != sizeof(nb200_decode_quantized_params) || p->decode.struct_size != sizeof(nb200_decode_params)) {
    set_error("%s: NULL params or wrong struct_size", what);
    return NB200_ERR_INVALID;
  }
  const nb200_decode_params& d = p->decode;
  const nb200_cache_pages& c = d.pages;
  if (c.dtype != NB200_F32 && c.dtype != NB200_BF16 && c.dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (c.pages < 0 || c.heads <= 0 || c.page_size <= 0 || c.head_dim <= 0 || d.rows < 0 || d.width < 0 || d.q_heads <= 0) {
    set_error("%s: bad extents", what);
    return NB200_ERR_INVALID;
  }
  if (d.q_heads % c.heads) { set_error("%s: %d query heads are no multiple of %d key heads", what, d.q_heads, c.heads); return NB200_ERR_INVALID; }
  if (c.head_dim > 256) { set_error("%s: head dim %d is more than 256", what, c.head_dim); return NB200_ERR_UNSUPPORTED; }
  if (d.rows > 65535) { set_error("%s: %d sequences, at most 65535", what, d.rows); return NB200_ERR_UNSUPPORTED; }
  return check_steps(c, p->steps, what);
}

Plan plan(const nb200_decode_params* p) {
  const nb200_cache_pages& c = p->pages;
  Plan pl{};
  const int group = p->q_heads / c.heads;
  pl.heads = c.head_dim > 128 ? 2 : 4;
  const int ctas = 2;      // resident per SM: the loops' kMinCtas
  const int chunks = (group + pl.heads - 1) / pl.heads;
  pl.side = chunks == 1 ? 1 : chunks == 2 ? 2 : 4;
  pl.chunks = (chunks + pl.side - 1) / pl.side;
  pl.unit = 64;
  const int64_t units = (int64_t(p->width) * c.page_size + pl.unit - 1) / pl.unit * p->rows * c.heads * pl.chunks;
  const int64_t most = int64_t(tc::sm_count()) * ctas;
  pl.workers = int(units < most ? (units > 0 ? units : 1) : most);
  pl.bytes = size_t(pl.workers) * 2 * pl.side * pl.heads * (c.head_dim + 4) * sizeof(float);
  return pl;
}

template <typename T, int kBits>
int launch_fma(const QuantizedArgs& a, int side, cudaStream_t st) {
  if (a.groups <= 2) return launch<T, QuantizedFmaLoop<T, kBits, 2, 4>, false>(a, side, st);
  if (a.groups <= 4) return launch<T, QuantizedFmaLoop<T, kBits, 4, 4>, false>(a, side, st);
  return launch<T, QuantizedFmaLoop<T, kBits, 8, 2>, false>(a, side, st);
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_decode_quantized_workspace_bytes(const nb200_decode_quantized_params* p, size_t* bytes) {
  if (!bytes) { set_error("bytes out-pointer is NULL"); return NB200_ERR_INVALID; }
  if (int rc = check(p, "decode_quantized_workspace_bytes")) return rc;
  *bytes = plan(&p->decode).bytes;
  return NB200_OK;
}

extern "C" NB200_API int nb200_decode_quantized(const nb200_decode_quantized_params* qp, void* cuda_stream) {
  const char* what = "decode_quantized";
  if (int rc = check(qp, what)) return rc;
  const nb200_decode_params* p = &qp->decode;
  if (p->rows == 0) return NB200_OK;
  const nb200_cache_pages& c = p->pages;
  if (!p->q || !p->out || !p->lengths || (p->width && !p->table) || (c.pages && (!c.k || !c.v))) { set_error("%s: NULL operand", what); return NB200_ERR_INVALID; }
  const int groups = c.head_dim / kGroup;
  bool ok = aligned16(c.k) && aligned16(c.v), near = true;
  auto fits = [&](int64_t stride) { near = near && stride <= 0x7fffffff && stride >= -0x7fffffff; return int(stride); };
  QuantizedArgs a{};
  for (int i = 0; i < 3; ++i) {
    ok = ok && c.k_stride[i] % 16 == 0 && c.v_stride[i] % 16 == 0;
    a.ks[i] = fits(c.k_stride[i] / 16);
    a.vs[i] = fits(c.v_stride[i] / 16);
    a.kss[i] = fits(qp->steps.k_stride[i] / groups);
    a.vss[i] = fits(qp->steps.v_stride[i] / groups);
  }
  if (!ok) { set_error("%s: the rows of the pages must begin on 16-byte boundaries", what); return NB200_ERR_ALIGNMENT; }
  if (!near) { set_error("%s: a stride of the pages is 2^31 words of 16 bytes, or rows of steps, or more", what); return NB200_ERR_UNSUPPORTED; }
  const Plan pl = plan(p);
  if (!p->workspace || p->workspace_bytes < pl.bytes) {
    set_error("%s: workspace of %zu bytes needed (nb200_decode_quantized_workspace_bytes), %zu given", what, pl.bytes, p->workspace_bytes);
    return NB200_ERR_WORKSPACE;
  }
  if (!aligned16(p->workspace)) { set_error("%s: the workspace must begin on a 16-byte boundary", what); return NB200_ERR_ALIGNMENT; }
  a.k = static_cast<const uint4*>(c.k);
  a.v = static_cast<const uint4*>(c.v);
  a.k_steps = static_cast<const uint16_t*>(qp->steps.k);
  a.v_steps = static_cast<const uint16_t*>(qp->steps.v);
  a.groups = groups;
  a.pages = c.pages; a.kv_heads = c.heads; a.page_size = c.page_size; a.D = c.head_dim;
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page_size == 1 << s) a.page_shift = s;
  a.table = p->table; a.lengths = p->lengths; a.rows = p->rows;
  a.width = c.pages ? p->width : 0;      // (without pages every sequence is empty)
  a.q = p->q; a.qs[0] = p->q_stride[0]; a.qs[1] = p->q_stride[1];
  a.out = p->out;
  a.q_heads = p->q_heads; a.group = p->q_heads / c.heads;
  a.chunks = pl.chunks;
  a.mul = p->scale * kLog2e;
  a.unit = pl.unit;
  a.part = static_cast<float*>(p->workspace);
  a.workers = pl.workers;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  const bool four = qp->steps.bits == 4;
  if (c.dtype == NB200_F32) return four ? launch_fma<float, 4>(a, pl.side, st) : launch_fma<float, 8>(a, pl.side, st);
  if (c.dtype == NB200_BF16) return four ? launch_fma<__nv_bfloat16, 4>(a, pl.side, st) : launch_fma<__nv_bfloat16, 8>(a, pl.side, st);
  return four ? launch_fma<__half, 4>(a, pl.side, st) : launch_fma<__half, 8>(a, pl.side, st);
}
