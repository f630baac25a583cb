// Tokens of a paged cache as packed rows, of the pages' own type or from codes of 4 or 8 bits.
//
// Bound by HBM: codes and steps (or elements) read once, the rows written once.  A warp takes a token at a time: its sequence by
// bisection of the offsets, its page from the table; then a lane eight elements at a time, which are two parts of a row of codes
// and one or two 16-byte words of the result.
#include <type_traits>

#include "cache_codes.cuh"
#include "sdpa_tc_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;

struct ReadArgs {
  const uint8_t* k;
  const uint8_t* v;
  int64_t ks[3], vs[3];            // bytes, over (page, head, slot)
  const uint16_t* k_steps;
  const uint16_t* v_steps;
  int64_t kss[3], vss[3];          // elements
  int pages, heads, page_size;
  int row;                         // units of a head's row: of 8 elements, or 16-byte words
  int unit_shift;                  // log2 of row, or -1
  const int* table;
  const int* lengths;
  int rows, width;
  const int* offsets;
  const int* starts;
  uint4* out_k;
  uint4* out_v;
  int64_t tokens;
};

template <typename T>
__device__ __forceinline__ void store8(uint4* p, const float2 (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    p[0] = make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
    p[1] = make_uint4(__float_as_uint(x[2].x), __float_as_uint(x[2].y), __float_as_uint(x[3].x), __float_as_uint(x[3].y));
  } else {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    p[0] = make_uint4(tc::pack2<kBf16>(x[0].x, x[0].y), tc::pack2<kBf16>(x[1].x, x[1].y), tc::pack2<kBf16>(x[2].x, x[2].y), tc::pack2<kBf16>(x[3].x, x[3].y));
  }
}

// kBits 0: words are copied; otherwise T is the type of the result.
template <int kBits, typename T>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const ReadArgs a) {
  constexpr int kWords = kBits == 0 ? 1 : int(sizeof(T)) / 2;      // 16-byte words of a unit of the result
  const int lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  // the first sequence that ends behind t
  int lo = 0, hi = a.rows;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (int64_t(__ldg(a.offsets + mid + 1)) <= t) lo = mid + 1;
    else hi = mid;
  }
  int page = -1, slot = 0;
  if (lo < a.rows) {
    const int64_t first = __ldg(a.offsets + lo), at = t - first + (a.starts ? __ldg(a.starts + lo) : 0);
    const int64_t held = min(int64_t(min(__ldg(a.lengths + lo), NB200_CACHE_MOST_TOKENS)), int64_t(a.width) * a.page_size);
    if (t >= first && at >= 0 && at < held) {
      const int column = int(at / a.page_size);
      slot = int(at - int64_t(column) * a.page_size);
      page = __ldg(a.table + int64_t(lo) * a.width + column);
    }
  }
  const int n = a.heads * a.row;
  uint4* ok = a.out_k + t * n * kWords;
  uint4* ov = a.out_v + t * n * kWords;
  if (page < 0 || page >= a.pages) {
    for (int i = lane; i < n * kWords; i += 32) ok[i] = ov[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint8_t* kp = a.k + page * a.ks[0] + slot * a.ks[2];
  const uint8_t* vp = a.v + page * a.vs[0] + slot * a.vs[2];
  if constexpr (kBits == 0) {
    for (int i = lane; i < n; i += 32) {
      const int h = i / a.row, c = i - h * a.row;
      const uint4 kw = __ldg(reinterpret_cast<const uint4*>(kp + h * a.ks[1]) + c), vw = __ldg(reinterpret_cast<const uint4*>(vp + h * a.vs[1]) + c);
      ok[i] = kw;
      ov[i] = vw;
    }
  } else {
    const int groups = a.row / 4;
    const uint16_t* kt = a.k_steps + page * a.kss[0] + slot * a.kss[2];
    const uint16_t* vt = a.v_steps + page * a.vss[0] + slot * a.vss[2];
    const int tail = groups % 2 == 0 ? 8 : 4;      // lanes that exchange words; n is a multiple
    // (whole warps go round together; lanes behind the end repeat its last group's work and store nothing)
#pragma unroll 2
    for (int w0 = 0; w0 < n; w0 += 32) {
      const int i = min(w0 + lane, n - tail + (lane & (tail - 1)));
      const int h = a.unit_shift >= 0 ? i >> a.unit_shift : i / a.row, c = i - h * a.row, group = c >> 2, u = c & 3;
      const uint2 kw = load_words<kBits>(kp + h * a.ks[1], groups, group, u), vw = load_words<kBits>(vp + h * a.vs[1], groups, group, u);
      const float k_step = __half2float(__ushort_as_half(__ldg(kt + h * a.kss[1] + group))), v_step = __half2float(__ushort_as_half(__ldg(vt + h * a.vss[1] + group)));
      float2 x[4];
      values_of<kBits>(kw, groups, group, k_step, x);
      if (w0 + lane < n) store8<T>(ok + int64_t(i) * kWords, x);
      values_of<kBits>(vw, groups, group, v_step, x);
      if (w0 + lane < n) store8<T>(ov + int64_t(i) * kWords, x);
    }
  }
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" NB200_API int nb200_cache_read(const nb200_cache_read_params* p, void* cuda_stream) {
  const char* what = "cache_read";
  if (!p || p->struct_size != sizeof(nb200_cache_read_params)) { set_error("%s: NULL params or wrong struct_size", what); return NB200_ERR_INVALID; }
  const nb200_cache_pages& c = p->pages;
  const bool coded = p->steps.bits != 0;
  if (c.dtype != NB200_F32 && c.dtype != NB200_BF16 && c.dtype != NB200_F16) { set_error("%s: bad dtype", what); return NB200_ERR_INVALID; }
  if (c.pages < 0 || c.heads <= 0 || c.page_size <= 0 || c.head_dim <= 0 || p->rows < 0 || p->width < 0 || p->tokens < 0 || p->tokens > 0x7fffffff) {
    set_error("%s: bad extents", what);
    return NB200_ERR_INVALID;
  }
  if (p->tokens == 0) return NB200_OK;
  if (!p->out_k || !p->out_v || (c.pages && (!c.k || !c.v)) || (p->rows && (!p->lengths || !p->offsets || (p->width && !p->table)))) {
    set_error("%s: NULL operand", what);
    return NB200_ERR_INVALID;
  }
  if (coded)
    if (int rc = check_steps(c, p->steps, what)) return rc;
  const int esz = coded ? 1 : dtype_size(c.dtype);
  const int row = coded ? c.head_dim / 8 * p->steps.bits : c.head_dim * esz;      // bytes
  bool ok = row % 16 == 0 && aligned16(c.k) && aligned16(c.v) && aligned16(p->out_k) && aligned16(p->out_v);
  for (int i = 0; i < 3; ++i) ok = ok && c.k_stride[i] * esz % 16 == 0 && c.v_stride[i] * esz % 16 == 0;
  if (!ok) { set_error("%s: rows must begin on 16-byte boundaries", what); return NB200_ERR_ALIGNMENT; }
  if (int64_t(c.heads) * c.head_dim > 0x3fffffff) { set_error("%s: rows too large", what); return NB200_ERR_UNSUPPORTED; }
  ReadArgs a{};
  a.k = static_cast<const uint8_t*>(c.k); a.v = static_cast<const uint8_t*>(c.v);
  a.k_steps = static_cast<const uint16_t*>(p->steps.k); a.v_steps = static_cast<const uint16_t*>(p->steps.v);
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = c.k_stride[i] * esz; a.vs[i] = c.v_stride[i] * esz;
    a.kss[i] = p->steps.k_stride[i]; a.vss[i] = p->steps.v_stride[i];
  }
  a.pages = c.pages; a.heads = c.heads; a.page_size = c.page_size;
  a.row = coded ? c.head_dim / 8 : row / 16;
  a.unit_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a.row == 1 << s) a.unit_shift = s;
  a.table = p->table; a.lengths = p->lengths; a.offsets = p->offsets; a.starts = p->starts;
  a.rows = p->rows; a.width = p->width;
  a.out_k = static_cast<uint4*>(p->out_k); a.out_v = static_cast<uint4*>(p->out_v);
  a.tokens = p->tokens;
  void (*kernel)(ReadArgs) = cache_read_kernel<0, uint4>;
  if (coded) {
    const bool four = p->steps.bits == 4;
    kernel = c.dtype == NB200_F32    ? four ? cache_read_kernel<4, float> : cache_read_kernel<8, float>
             : c.dtype == NB200_BF16 ? four ? cache_read_kernel<4, __nv_bfloat16> : cache_read_kernel<8, __nv_bfloat16>
             : four                  ? cache_read_kernel<4, __half> : cache_read_kernel<8, __half>;
  }
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  prof_call_begin(st);
  kernel<<<unsigned((p->tokens + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(a);
  count_launch();
  return check_launch("cache_read_kernel");
}
