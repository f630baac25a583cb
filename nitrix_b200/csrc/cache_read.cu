// Tokens of a paged cache as packed rows, of the pages' own type or from codes of 4 or 8 bits.
//
// Bound by HBM: codes and steps (or elements) read once, the rows written once.  A warp takes a token at a time: its sequence by
// bisection of the offsets, its page from the table; then a lane eight elements at a time, which are two parts of a row of codes
// and one or two 16-byte words of the result, of each group of a row of 64 or 128, whose codes lie side by side.
//
// 69 k tokens of 8 heads of 128 from 4 bits into bf16, 356 MB in all: 64 us (5.6 TB/s).  By single groups, with two loads of 16 bits for
// 8 codes, 90.
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
  const int* table;
  const int* lengths;
  int rows, width;
  const int* offsets;
  const int* starts;
  uint4* out_k;
  uint4* out_v;
  int64_t tokens;
  int tokens_per_warp;
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

struct TokenRows {
  const uint8_t* codes[2];
  const uint16_t* steps[2];
  int64_t codes_head[2], steps_head[2];      // from one head to the next
  uint4* to[2];
};

// A token's values, by a warp.  With kGroups, those of a head's row, a lane takes 8 elements of each of them, whose codes lie side by
// side; otherwise, for any number of groups, 8 elements.
template <int kBits, typename T, int kGroups>
__device__ __forceinline__ void read_token(const ReadArgs& a, const TokenRows& at) {
  constexpr int kWords = int(sizeof(T)) / 2, kEach = kGroups ? kGroups : 1;
  const int units = kGroups ? 4 : a.row, n = a.heads * units;
  for (int w = threadIdx.x & 31; w < n; w += 32) {
    const int h = w / units, c = w - h * units;
    const uint8_t* rows[2] = {at.codes[0] + h * at.codes_head[0], at.codes[1] + h * at.codes_head[1]};
    const uint16_t* steps[2] = {at.steps[0] + h * at.steps_head[0], at.steps[1] + h * at.steps_head[1]};
    const int64_t to = (int64_t(h) * a.row + c) * kWords;
    float2 x[4];
    if constexpr (kGroups > 0) {
      constexpr int nw = kGroups * kBits / 4;
      uint32_t codes[2][nw], s[2][kGroups / 2];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        load_words(codes[which], rows[which] + c * nw * 4);
        load_words(s[which], steps[which]);
      }
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int g = 0; g < kEach; ++g) {
          const float step = __half2float(__ushort_as_half(uint16_t(g % 2 ? s[which][g / 2] >> 16 : s[which][g / 2])));
          if constexpr (kBits == 4) values_of<4>(__byte_perm(codes[which][g / 2], codes[which][nw / 2 + g / 2], g % 2 ? 0x7632 : 0x5410), 0u, step, x);
          else values_of<8>(codes[which][g], codes[which][nw / 2 + g], step, x);
          store8<T>(at.to[which] + to + g * 4 * kWords, x);
        }
    } else {
      const int groups = a.row / 4, g = c >> 2, u = c & 3;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint32_t lo, hi = 0;
        if constexpr (kBits == 4) {
          const uint16_t* p = reinterpret_cast<const uint16_t*>(rows[which]) + 2 * u * groups + g;
          lo = __ldg(p) | uint32_t(__ldg(p + groups)) << 16;
        } else {
          const uint32_t* p = reinterpret_cast<const uint32_t*>(rows[which]) + 2 * u * groups + g;
          lo = __ldg(p);
          hi = __ldg(p + groups);
        }
        values_of<kBits>(lo, hi, __half2float(__ushort_as_half(__ldg(steps[which] + g))), x);
        store8<T>(at.to[which] + to, x);
      }
    }
  }
}

// The first sequence of lo .. hi that ends behind token t.
__device__ __forceinline__ int row_of(const ReadArgs& a, int64_t t, int lo, int hi) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (int64_t(__ldg(a.offsets + mid + 1)) <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
struct Slot {
  int page, slot;      // a page outside the pool: there is no such token
};
__device__ __forceinline__ Slot slot_of(const ReadArgs& a, int64_t t, int row) {
  if (row >= a.rows) return Slot{-1, 0};
  const int64_t first = __ldg(a.offsets + row), at = t - first + (a.starts ? __ldg(a.starts + row) : 0);
  const int64_t held = min(int64_t(min(__ldg(a.lengths + row), NB200_CACHE_MOST_TOKENS)), int64_t(a.width) * a.page_size);
  if (t < first || at < 0 || at >= held) return Slot{-1, 0};
  const int column = int(at) / a.page_size;
  return Slot{__ldg(a.table + int64_t(row) * a.width + column), int(at) - column * a.page_size};
}

// A token's rows from a slot of a page, or zeros.
template <int kBits, typename T>
__device__ __forceinline__ void read_slot(const ReadArgs& a, int64_t t, int page, int slot, int lane) {
  constexpr int kWords = kBits == 0 ? 1 : int(sizeof(T)) / 2;
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
    const TokenRows at{{kp, vp}, {a.k_steps + page * a.kss[0] + slot * a.kss[2], a.v_steps + page * a.vss[0] + slot * a.vss[2]},
                       {a.ks[1], a.vs[1]}, {a.kss[1], a.vss[1]}, {ok, ov}};
    if (a.row == 16) read_token<kBits, T, 4>(a, at);
    else if (a.row == 8) read_token<kBits, T, 2>(a, at);
    else read_token<kBits, T, 0>(a, at);
  }
}

// kBits 0: words are copied; otherwise T is the type of the result.
template <int kBits, typename T>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & 31;
  int64_t t = (int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * a.tokens_per_warp;
  const int64_t t_end = min(t + a.tokens_per_warp, a.tokens);
  if (t >= t_end) return;
  int row = row_of(a, t, 0, a.rows);
  Slot at = slot_of(a, t, row);
  for (; t < t_end; ++t) {
    const Slot here = at;
    if (t + 1 < t_end) {      // (the next token's place is on its way while this one's rows are)
      while (row < a.rows && int64_t(__ldg(a.offsets + row + 1)) <= t + 1) ++row;
      at = slot_of(a, t + 1, row);
    }
    read_slot<kBits, T>(a, t, here.page, here.slot, lane);
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
  // One token per warp while that does not fill the GPU's warps a few times over, then more, which share a search.
  a.tokens_per_warp = p->tokens < 148 * 128 ? 1 : p->tokens < 148 * 512 ? 2 : 4;
  const int64_t per_cta = int64_t(a.tokens_per_warp) * (kThreads / 32);
  kernel<<<unsigned((p->tokens + per_cta - 1) / per_cta), kThreads, 0, st>>>(a);
  count_launch();
  return check_launch("cache_read_kernel");
}
