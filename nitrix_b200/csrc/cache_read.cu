// Tokens of a paged cache as packed rows, of the pages' own type or from codes of 4 or 8 bits.
//
// Bound by HBM: codes and steps (or elements) read once, the rows written once.  A warp takes a token at a time: its sequence by
// bisection of the offsets, its page from the table; then a lane eight elements at a time, which are two parts of a row of codes
// and one or two 16-byte words of the result, of each group of a row of 64 or 128, whose codes lie side by side.
//
// 69 k tokens of 8 heads of 128 from 4 bits into bf16, 356 MB in all: 61 us (5.8 TB/s).  By single groups, with two loads of 16 bits for
// 8 codes, 90.  34 k tokens into fp32, 317 MB: 57 us (5.6 TB/s), of 8 bits 63; with two stores for a lane's 8 elements 96 and 114.
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
    // (a whole sector at once)
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0].x), "f"(x[0].y), "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y),
                 "f"(x[3].x), "f"(x[3].y)
                 : "memory");
  } else {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    p[0] = make_uint4(tc::pack2<kBf16>(x[0].x, x[0].y), tc::pack2<kBf16>(x[1].x, x[1].y), tc::pack2<kBf16>(x[2].x, x[2].y), tc::pack2<kBf16>(x[3].x, x[3].y));
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

// The rows of a token's slot.
struct Rows {
  const uint8_t* codes[2];
  const uint16_t* steps[2];
  __device__ __forceinline__ Rows(const ReadArgs& a, Slot at)
      : codes{a.k + at.page * a.ks[0] + at.slot * a.ks[2], a.v + at.page * a.vs[0] + at.slot * a.vs[2]},
        steps{a.k_steps + at.page * a.kss[0] + at.slot * a.kss[2], a.v_steps + at.page * a.vss[0] + at.slot * a.vss[2]} {}
};

// A token's values, by a warp.  With kGroups, those of a head's row, a lane takes 8 elements of each of them, whose codes lie side by
// side; otherwise, for any number of groups, 8 elements.  kBits 0: words are copied.
template <int kBits, typename T, int kGroups>
struct Token {
  static constexpr int kWords = kBits == 0 ? 1 : int(sizeof(T)) / 2, kEach = kGroups ? kGroups : 1;
  static constexpr int kCodeWords = kBits == 0 ? 4 : kGroups ? kGroups * kBits / 4 : kBits / 4, kStepWords = (kEach + 1) / 2;
  uint32_t codes[2][kCodeWords], steps[2][kStepWords];      // of the lane's place in a row

  __device__ __forceinline__ static int units(const ReadArgs& a) { return kGroups ? 4 : a.row; }
  __device__ __forceinline__ void load(const ReadArgs& a, const Rows& rows, int w) {
    const int h = w / units(a), c = w - h * units(a);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint8_t* row = rows.codes[which] + h * (which ? a.vs : a.ks)[1];
      if constexpr (kBits == 0) {
        load_words(codes[which], row + c * 16);
        continue;
      }
      const uint16_t* step = rows.steps[which] + h * (which ? a.vss : a.kss)[1];
      if constexpr (kGroups > 0) {
        load_words(codes[which], row + c * kCodeWords * 4);
        load_words(steps[which], step);
      } else {
        const int groups = a.row / 4, g = c >> 2, u = c & 3;
        if constexpr (kBits == 4) {
          const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + 2 * u * groups + g;
          codes[which][0] = __ldg(p) | uint32_t(__ldg(p + groups)) << 16;
        } else {
          const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + 2 * u * groups + g;
          codes[which][0] = __ldg(p);
          codes[which][kCodeWords - 1] = __ldg(p + groups);
        }
        steps[which][0] = __ldg(step + g);
      }
    }
  }
  __device__ __forceinline__ void store(const ReadArgs& a, int64_t t, int w) const {
    const int h = w / units(a), c = w - h * units(a);
    const int64_t to = ((t * a.heads + h) * a.row + c) * kWords;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint4* out = (which ? a.out_v : a.out_k) + to;
      if constexpr (kBits == 0) {
        out[0] = make_uint4(codes[which][0], codes[which][1], codes[which][2], codes[which][3]);
      } else {
#pragma unroll
        for (int g = 0; g < kEach; ++g) {
          constexpr int half = kCodeWords / 2;
          const float step = __half2float(__ushort_as_half(uint16_t(g % 2 ? steps[which][g / 2] >> 16 : steps[which][g / 2])));
          float2 x[4];
          if constexpr (kBits == 8) values_of<8>(codes[which][g], codes[which][half + g], step, x);
          else if constexpr (kGroups == 0) values_of<4>(codes[which][0], 0u, step, x);
          else values_of<4>(__byte_perm(codes[which][g / 2], codes[which][half + g / 2], g % 2 ? 0x7632 : 0x5410), 0u, step, x);
          store8<T>(out + g * 4 * kWords, x);
        }
      }
    }
  }
};

// Tokens t .. t_end, by a warp; the next one's place is on its way while this one's rows are.  (The next one's first words as well: 68
// us instead of 64 for 69 k tokens in 4 bits, bf16, 8 heads of 128.)
template <typename T>
__device__ __forceinline__ void read_tokens(const ReadArgs& a, int64_t t, int64_t t_end) {
  const int lane = threadIdx.x & 31, n = a.heads * T::units(a);
  int row = row_of(a, t, 0, a.rows);
  Slot at = slot_of(a, t, row);
  for (;; ++t) {
    const Slot here = at;
    const bool more = t + 1 < t_end;
    if (more) {
      while (row < a.rows && int64_t(__ldg(a.offsets + row + 1)) <= t + 1) ++row;
      at = slot_of(a, t + 1, row);
    }
    if (here.page < 0 || here.page >= a.pages) {
      const int words = a.heads * a.row * T::kWords;
      for (int i = lane; i < words; i += 32) a.out_k[t * words + i] = a.out_v[t * words + i] = make_uint4(0, 0, 0, 0);
    } else {
      const Rows rows(a, here);
      for (int w = lane; w < n; w += 32) {
        T token;
        token.load(a, rows, w);
        token.store(a, t, w);
      }
    }
    if (!more) return;
  }
}

// kBits 0: words are copied; otherwise T is the type of the result.
template <int kBits, typename T, int kGroups>
__global__ void __launch_bounds__(kThreads, kBits && sizeof(T) == 4 ? 3 : 4) cache_read_kernel(const ReadArgs a) {
  const int64_t t = (int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * a.tokens_per_warp;
  const int64_t t_end = min(t + a.tokens_per_warp, a.tokens);
  if (t < t_end) read_tokens<Token<kBits, T, kGroups>>(a, t, t_end);
}
using Kernel = void (*)(ReadArgs);
template <int kBits, typename T>
Kernel kernel_of(int groups) {
  return groups == 4 ? cache_read_kernel<kBits, T, 4> : groups == 2 ? cache_read_kernel<kBits, T, 2> : cache_read_kernel<kBits, T, 0>;
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
  if (coded && c.dtype == NB200_F32) ok = ok && (reinterpret_cast<uintptr_t>(p->out_k) | reinterpret_cast<uintptr_t>(p->out_v)) % 32 == 0;
  if (!ok) { set_error("%s: rows must begin on 16-byte boundaries (fp32 from codes: out_k and out_v on 32-byte ones)", what); return NB200_ERR_ALIGNMENT; }
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
  Kernel kernel = cache_read_kernel<0, uint4, 0>;
  if (coded) {
    const bool four = p->steps.bits == 4;
    const int groups = c.head_dim / kGroup;
    kernel = c.dtype == NB200_F32    ? four ? kernel_of<4, float>(groups) : kernel_of<8, float>(groups)
             : c.dtype == NB200_BF16 ? four ? kernel_of<4, __nv_bfloat16>(groups) : kernel_of<8, __nv_bfloat16>(groups)
             : four                  ? kernel_of<4, __half>(groups) : kernel_of<8, __half>(groups);
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
