// Forward attention over packed sequences with fp32 operands on the tcgen05 tensor cores: every fp32 number is three bf16
// numbers and every product the six bf16 products that matter (sdpa_fp32_tc.cu has the error bounds and the scheme of a tile).
//
// packed_planes_kernel writes the planes of q, k and v into the workspace as the tiles that the MMAs read, a sequence and key
// head at a time: 128 rows of queries (token after token, the query heads of the key head), 64 keys.  Rows behind the end of
// a sequence are zeros there, so nothing of a neighbouring sequence gets near a sum.  The tiles of sequence i begin at tile
// begin / tokens per tile + i: sequences that follow one another never share one, and nobody has to add up the lengths.
// packed_fwd_fp32_kernel then fetches whole tiles by untiled bulk copies; its blocks come from the list of packed_plan.cu.
//
// An infinity in a sequence's own operands becomes a NaN in its planes (x - x0), so that its scores are NaN where the fp32
// units may still give a number.
//
// Where these kernels run and where the fp32 units do: the rule and both sides are beside fp32_packed_supported.  Bound by the
// chain of a step (scores, soft-max, P V of a tile follow one another; two tiles per CTA at head dim 64, one at 128, where the
// planes of one fill the shared memory): 84 % and 64 % of the 275 TFLOP/s that six products at the bf16 rate leave, long sequences.
#include <math.h>

#include "dependent_launch.cuh"
#include "fp32_planes.cuh"
#include "packed_tc.cuh"

namespace nb200 {
namespace packed {

using namespace sm100;
using tc::wait_or_abort;

namespace {

constexpr int kKeys = 64;             // keys of a tile
constexpr int kRows = 128;            // rows of a query tile
constexpr int kRowBytes = 128;        // 64 bf16 of one plane

// ---- planes -----------------------------------------------------------------------------------------------------------------
struct PlaneOperand {
  const float* x;
  uint8_t* planes;
  const int* offsets;
  int64_t xs[2];        // element strides over (token, head)
  int total;            // tokens of the tensor
  int tokens, rows;     // of a tile
  int heads;            // rows per token
  uint32_t heads_magic; // ceil(2^16 / heads)
  int64_t tiles;        // that there is room for
};
struct PlaneArgs {
  PlaneOperand op[3];
  int sequences, kv_heads;
};

// First tile of a sequence's planes.
__device__ __forceinline__ int64_t first_tile(int begin, int tokens, int sequence) { return int64_t(begin / tokens) + sequence; }

// Grid (tiles, key heads, operands).  Bound by memory: 4 bytes in, 6 out per element.
template <int kCols>
__global__ void __launch_bounds__(128) packed_planes_kernel(const PlaneArgs a) {
  allow_dependents();
  const PlaneOperand& op = a.op[blockIdx.z];
  constexpr int kUnits = kCols / 8, kChunks = kCols / 64;
  const int64_t tile = blockIdx.x;
  // the last sequence whose tiles begin at this one or before it
  int lo = 0, hi = a.sequences - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first_tile(sequence_span(op.offsets, mid, op.total).x, op.tokens, mid) <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int2 span = sequence_span(op.offsets, lo, op.total);
  const int64_t index = tile - first_tile(span.x, op.tokens, lo);
  if (tile < op.tiles && index >= 0 && index * op.tokens < span.y) {
    const int first = span.x + int(index) * op.tokens, n = min(op.tokens, span.x + span.y - first);
    const float* x = op.x + int64_t(first) * op.xs[0] + int64_t(blockIdx.y) * op.heads * op.xs[1];
    const int chunk = op.rows * kRowBytes;
    uint8_t* dst_tile = op.planes + (tile * a.kv_heads + blockIdx.y) * (3 * kChunks * chunk);
    const bool vec = ((reinterpret_cast<uintptr_t>(op.x) & 15) == 0) && ((op.xs[0] | op.xs[1]) & 3) == 0;
#pragma unroll 4
    for (int u = threadIdx.x; u < op.rows * kUnits; u += 128) {
      const int r = u / kUnits, c = u - r * kUnits, token = int((uint32_t(r) * op.heads_magic) >> 16);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      if (token < n) {
        const float* src = x + token * op.xs[0] + (r - token * op.heads) * op.xs[1] + c * 8;
        if (vec) {
          *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
          *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(src + 4);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = src[i];
        }
      }
      uint4 w[3];
      split8(v, w);
      uint8_t* dst = dst_tile + (c / 8) * chunk + r * kRowBytes + (((c & 7) ^ (r & 7)) * 16);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(dst + p * kChunks * chunk) = w[p];
    }
  }
  wait_for_previous();      // (the list, which the kernel behind this one reads)
}

// ---- forward ----------------------------------------------------------------------------------------------------------------
struct Fp32Args {
  WorkList list;
  const uint8_t *q, *k, *v;     // planes
  int64_t q_tiles, k_tiles;     // that there is room for
  int kv_heads, group, heads;
  int tokens;                   // of a query tile
  uint32_t group_magic;
  int block;                    // tokens of a block
  int causal;
  float scale;
  float* out;                   // dense (tokens, heads, D)
  float* lse;
  int* status;
};

// The soft-max's reference lies kAbove over the last maximum taken, which a later score may outgrow by up to 2^kAbove: no
// probability is above 1.
constexpr float kAbove = 8.f;

template <int kCols>
struct Layout {
  static constexpr int kChunks = kCols / 64;
  static constexpr int kTiles = kCols == 64 ? 2 : 1;           // query tiles that a CTA has room for
  static constexpr int kStages = kCols == 64 ? 2 : 1;          // of K and of V
  static constexpr int kThreads = (5 * kTiles + 1) * 32;
  static constexpr int kPlane = kChunks * kKeys * kRowBytes;   // one plane of a tile of keys
  static constexpr int kKvBytes = 3 * kPlane;
  static constexpr int kQPlane = kChunks * kRows * kRowBytes;
  static constexpr int kQBytes = 3 * kQPlane;
  static constexpr int kQ = 0;
  static constexpr int kK = kTiles * kQBytes;
  static constexpr int kV = kK + kStages * kKvBytes;
  static constexpr int kBars = kV + kStages * kKvBytes;
  static constexpr int kBytes = kBars + 256;
  // TMEM columns of a query tile: scores, the three planes of P, output
  static constexpr int kTmS = 0, kTmP = 64, kTmO = 160, kTmTile = 256, kTmCols = 512;
};
enum Bar { K_FULL = 0, K_EMPTY = 2, V_FULL = 4, V_EMPTY = 6, Q_FULL = 8, S_FULL = 10, S_FREE = 12, P_FULL = 14, PV_DONE = 16, kBarCount = 18 };

// A CTA owns a block of one or two query tiles of a key head and streams the sequence's keys in steps of 64.  Warps 0-3 (4-7):
// a thread owns a row of the first (second) tile -- online soft-max, P into three planes in TMEM; the next warp fetches, the
// last one or two issue the MMAs of a tile each.  The scores are read into registers at once, so Q K^T of the next step runs
// under the soft-max of this one.  The tensor core truncates what it accumulates, so the output is taken out of TMEM into
// fp32 registers (round to nearest) every other step, and wherever a row's maximum has grown by more than 2^8.
template <int kCols>
__global__ void __launch_bounds__(Layout<kCols>::kThreads, 1) packed_fwd_fp32_kernel(const __grid_constant__ Fp32Args a) {
  using L = Layout<kCols>;
  constexpr int kSoftWarps = 4 * L::kTiles, kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  int* abort_flag = reinterpret_cast<int*>(smem + L::kBars + 192);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBars + 196);
  allow_dependents();
  wait_for_previous();
  if (sbase & 1023) {   // (the swizzled tiles need it; the shared-memory window starts on such a boundary)
    if (threadIdx.x == 0) atomicExch(a.status, 600);
    return;
  }
  const int place = int(blockIdx.x / unsigned(a.kv_heads)), head = int(blockIdx.x - unsigned(place) * unsigned(a.kv_heads));
  if (place >= *a.list.count) return;
  const WorkItem item = load_item(a.list.items + place);
  const int sequence = item.sequence;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_tiles = min((item.n + a.tokens - 1) / a.tokens, L::kTiles);
  // tokens of a tile, and the keys that token t of it sees
  auto tokens_of = [&](int g) { return min(item.n - g * a.tokens, a.tokens); };
  auto seen_by = [&](int g, int t) { return a.causal ? int(min(max(int64_t(item.seen) + g * a.tokens + t, int64_t(0)), int64_t(item.other_n))) : item.other_n; };
  auto steps_of = [&](int g) { return (seen_by(g, tokens_of(g) - 1) + kKeys - 1) / kKeys; };
  const int steps_max = steps_of(n_tiles - 1);
  auto bar = [&](int i) { return sbase + L::kBars + 8 * i; };
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kBarCount; ++i) {
      const bool rows = (i >= S_FREE && i < S_FREE + 2) || (i >= P_FULL && i < P_FULL + 2);
      const bool empty = (i >= K_EMPTY && i < K_EMPTY + 2) || (i >= V_EMPTY && i < V_EMPTY + 2);
      mbar_init(bar(i), rows ? 128 : (empty ? n_tiles : 1));
    }
    mbar_init_fence();
  }
  if (warp == kSoftWarps) {
    tmem_alloc(smem_u32(tmem_slot), L::kTmCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tm = *tmem_slot;

  if (warp == kSoftWarps) {
    const int begin = item.begin - item.index * a.block;     // of the sequence
    const int64_t q_tile = first_tile(begin, a.tokens, sequence) + int64_t(item.index) * (a.block / a.tokens);
    const int64_t k_tile = first_tile(item.other, kKeys, sequence);
    // (offsets that run backwards may list blocks whose tiles nobody wrote, or for which there is no room)
    const bool room = q_tile >= 0 && q_tile + n_tiles <= a.q_tiles && k_tile >= 0 && k_tile + steps_max <= a.k_tiles;
    if (elect_one()) {
      bool ok = true;
      for (int g = 0; g < n_tiles; ++g) {
        mbar_expect_tx(bar(Q_FULL + g), L::kQBytes);
        bulk_load(sbase + L::kQ + g * L::kQBytes, a.q + ((room ? q_tile + g : 0) * a.kv_heads + head) * L::kQBytes, L::kQBytes, bar(Q_FULL + g));
      }
      for (int j = 0; j < steps_max && ok; ++j) {
        const int st = j % kStages;
        const uint32_t ph = ((j / kStages) & 1) ^ 1;
        const int64_t at = ((room ? k_tile + j : 0) * a.kv_heads + head) * int64_t(L::kKvBytes);
        ok = wait_or_abort(bar(K_EMPTY + st), ph, abort_flag, a.status, 601);
        if (!ok) break;
        mbar_expect_tx(bar(K_FULL + st), L::kKvBytes);
        bulk_load(sbase + L::kK + st * L::kKvBytes, a.k + at, L::kKvBytes, bar(K_FULL + st));
        ok = wait_or_abort(bar(V_EMPTY + st), ph, abort_flag, a.status, 602);
        if (!ok) break;
        mbar_expect_tx(bar(V_FULL + st), L::kKvBytes);
        bulk_load(sbase + L::kV + st * L::kKvBytes, a.v + at, L::kKvBytes, bar(V_FULL + st));
      }
      // (a block without a step has nobody else who would wait for Q: the copies must not outlive the CTA)
      for (int g = 0; g < n_tiles && ok; ++g) ok = wait_or_abort(bar(Q_FULL + g), 0, abort_flag, a.status, 603);
      if (!ok) tc::drain_after_abort();
    }
  } else if (warp > kSoftWarps) {
    const int g = warp - kSoftWarps - 1;
    if (g < n_tiles && elect_one()) {
      constexpr uint32_t idesc_qk = make_idesc(true, kRows, kKeys, false, false);
      constexpr uint32_t idesc_pv = make_idesc(true, kRows, kCols, false, true);
      const uint64_t qd = make_smem_desc(sbase + L::kQ + g * L::kQBytes, 16, 1024), kd0 = make_smem_desc(sbase + L::kK, 16, 1024);
      const uint64_t vd0 = make_smem_desc(sbase + L::kV, kKeys * kRowBytes, 1024);
      const uint32_t tg = tm + g * L::kTmTile;
      const int steps = steps_of(g);
      bool ok = wait_or_abort(bar(Q_FULL + g), 0, abort_flag, a.status, 604);
      // (a tile that is done before the CTA's last one still hands every stage back: one arrival per tile and phase)
      for (int j = 0; j <= steps_max && ok; ++j) {
        if (j < steps_max) {
          const int st = j % kStages;
          ok = wait_or_abort(bar(K_FULL + st), (j / kStages) & 1, abort_flag, a.status, 605);
          if (!ok) break;
          if (j < steps) {
            ok = j == 0 || wait_or_abort(bar(S_FREE + g), (j - 1) & 1, abort_flag, a.status, 606);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t kd = kd0 + uint64_t((st * L::kKvBytes) >> 4);
#pragma unroll
            for (int i = 0; i < kProducts; ++i)
#pragma unroll
              for (int kk = 0; kk < kCols / 16; ++kk)
                mma_ss(tg + L::kTmS, qd + uint64_t((left_plane(i) * L::kQPlane + (kk / 4) * kRows * kRowBytes + (kk % 4) * 32) >> 4),
                       kd + uint64_t((right_plane(i) * L::kPlane + (kk / 4) * kKeys * kRowBytes + (kk % 4) * 32) >> 4), idesc_qk,
                       i + kk > 0 ? 1u : 0u);
            mma_commit(bar(S_FULL + g));
            mma_commit(bar(K_EMPTY + st));
          } else {
            mbar_arrive(bar(K_EMPTY + st));
          }
        }
        if (j > 0) {
          const int st = (j - 1) % kStages;
          ok = wait_or_abort(bar(V_FULL + st), ((j - 1) / kStages) & 1, abort_flag, a.status, 607);
          if (!ok) break;
          if (j - 1 < steps) {
            ok = wait_or_abort(bar(P_FULL + g), (j - 1) & 1, abort_flag, a.status, 608);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t vd = vd0 + uint64_t((st * L::kKvBytes) >> 4);
#pragma unroll
            for (int i = 0; i < kProducts; ++i)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ts(tg + L::kTmO, tg + L::kTmP + left_plane(i) * 32 + kk * 8,
                       vd + uint64_t((right_plane(i) * L::kPlane + kk * 2048) >> 4), idesc_pv, (j > 1 || i + kk > 0) ? 1u : 0u);
            mma_commit(bar(PV_DONE + g));
            mma_commit(bar(V_EMPTY + st));
          } else {
            mbar_arrive(bar(V_EMPTY + st));
          }
        }
      }
    }
  } else if ((warp >> 2) < n_tiles) {
    const int g = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int token = int((uint32_t(r) * a.group_magic) >> 16), member = r - token * a.group;
    const bool mine = token < tokens_of(g);
    const int seen = mine ? seen_by(g, token) : 0;
    const int steps = steps_of(g);
    const uint32_t tl = tm + g * L::kTmTile + (uint32_t(quad * 32) << 16);
    const float mul = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
    float o[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] = 0.f;
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const int keys = seen - j * kKeys;       // of this step's that the row sees
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(S_FULL + g), j & 1, abort_flag, a.status, 609));
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t s[2][32];
      tmem_ld32(tl + L::kTmS, s[0]);
      tmem_ld32(tl + L::kTmS + 32, s[1]);
      tmem_wait_ld();
      tc_fence_before_sync();
      mbar_arrive(bar(S_FREE + g));
      float mx = -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float x = half * 32 + c < keys ? __uint_as_float(s[half][c]) * mul : -INFINITY;
          s[half][c] = __float_as_uint(x);
          mx = fmaxf(mx, x);
        }
      // the reference maximum moves only when some row of the warp has outgrown it by 2^8
      const float m_new = fmaxf(m, mx);
      const bool move = __any_sync(0xffffffffu, m_new > m + kAbove);   // (true for the first key: m = -inf)
      float alpha = 1.f;
      if (move) {
        alpha = m_new == -INFINITY ? 1.f : tc::ex2(m - m_new);
        m = m_new;
        l *= alpha;
      }
      const float m_ref = m == -INFINITY ? 0.f : m + kAbove;           // no key so far: every p is 0
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float p = tc::ex2(__uint_as_float(s[half][c]) - m_ref);
          s[half][c] = __float_as_uint(p);
          sum[c & 3] += p;
        }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (j > 0) {
        ok = __all_sync(0xffffffffu, wait_or_abort(bar(PV_DONE + g), (j - 1) & 1, abort_flag, a.status, 610));
        if (!ok) break;
        tc_fence_after_sync();
        if (move || (j & 1) == 0) {
          uint32_t v[32];
#pragma unroll
          for (int c0 = 0; c0 < kCols; c0 += 32) {
            tmem_ld32(tl + L::kTmO + c0, v);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              o[c0 + c] = (o[c0 + c] + __uint_as_float(v[c])) * alpha;
              v[c] = 0u;
            }
            tmem_st32(tl + L::kTmO + c0, v);
          }
        }
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) w[c] = __byte_perm(s[half][2 * c], s[half][2 * c + 1], 0x7632);
          tmem_st16(tl + L::kTmP + p * 32 + half * 16, w);
          if (p < 2) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              s[half][c] = __float_as_uint(__uint_as_float(s[half][c]) - __uint_as_float(s[half][c] & 0xffff0000u));
          }
        }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(bar(P_FULL + g));
    }
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(PV_DONE + g), (steps - 1) & 1, abort_flag, a.status, 611));
      tc_fence_after_sync();
    }
    // out = o / l, zeros for a row without a key
    if (ok) {
      const float inv = 1.f / l;
      const int64_t row = (int64_t(item.begin) + g * a.tokens + token) * a.heads + head * a.group + member;
      float* op = a.out + row * kCols;
#pragma unroll
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tl + L::kTmO + c0, v);
        tmem_wait_ld();
        if (mine) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = seen > 0 ? __float_as_uint((o[c0 + c] + __uint_as_float(v[c])) * inv) : 0u;
#pragma unroll
          for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(op + c0 + c) = make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]);
        }
      }
      if (mine) a.lse[row] = seen > 0 ? m + kAbove + log2f(l) : -INFINITY;
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (*abort_flag) tc::drain_after_abort();
  if (warp == kSoftWarps) tmem_dealloc(tm, L::kTmCols);
}

int64_t query_tiles(const PackedArgs& a) { return most_blocks(a.tokens_q, a.sequences, tile_tokens(kRows, a.group)); }
int64_t key_tiles(const PackedArgs& a) { return most_blocks(a.tokens_k, a.sequences, kKeys); }
// two query tiles per CTA, which share the fetched keys, once one per CTA would be more than one wave
int block_tiles(const PackedArgs& a) { return a.D == 64 && query_tiles(a) * a.kv_heads > tc::sm_count() ? 2 : 1; }
size_t list_bytes(const PackedArgs& a) {
  return work_list_bytes(most_blocks(a.tokens_q, a.sequences, block_tiles(a) * tile_tokens(kRows, a.group)));
}
size_t query_bytes(const PackedArgs& a) { return size_t(query_tiles(a)) * a.kv_heads * (kRows * a.D * 6); }
size_t key_bytes(const PackedArgs& a) { return size_t(key_tiles(a)) * a.kv_heads * (kKeys * a.D * 6); }

template <int kCols>
int launch(const PackedArgs& p, void* ws, cudaStream_t st) {
  using L = Layout<kCols>;
  static_assert(L::kBytes <= 232448, "shared memory of a CTA");
  auto kernel = packed_fwd_fp32_kernel<kCols>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess) return check_launch("packed_fwd_fp32_kernel");
  Fp32Args a{};
  a.tokens = tile_tokens(kRows, p.group);
  a.block = block_tiles(p) * a.tokens;
  const int64_t blocks = most_blocks(p.tokens_q, p.sequences, a.block) * p.kv_heads;
  a.status = device_status_word();
  if (!a.status) { set_error("packed_fwd: no status word on this device"); return NB200_ERR_LAUNCH; }
  if (int rc = launch_plan(p, false, a.block, 1, ws, st, sizeof(float))) return rc;
  a.list.count = static_cast<const int*>(ws);
  a.list.items = reinterpret_cast<const WorkItem*>(static_cast<const char*>(ws) + 16);
  uint8_t* q = static_cast<uint8_t*>(ws) + list_bytes(p);
  uint8_t* k = q + query_bytes(p);
  uint8_t* v = k + key_bytes(p);
  a.q = q; a.k = k; a.v = v;
  a.q_tiles = query_tiles(p);
  a.k_tiles = key_tiles(p);
  a.kv_heads = p.kv_heads; a.group = p.group; a.heads = p.heads;
  a.group_magic = uint32_t((65536 + p.group - 1) / p.group);
  a.causal = p.causal;
  a.scale = p.scale;
  a.out = static_cast<float*>(p.out);
  a.lse = p.lse;
  PlaneArgs pa{};
  pa.sequences = p.sequences;
  pa.kv_heads = p.kv_heads;
  pa.op[0] = PlaneOperand{static_cast<const float*>(p.q), q, p.offsets_q, {p.qs[0], p.qs[1]}, p.tokens_q, a.tokens, kRows, p.group, a.group_magic, a.q_tiles};
  pa.op[1] = PlaneOperand{static_cast<const float*>(p.k), k, p.offsets_k, {p.ks[0], p.ks[1]}, p.tokens_k, kKeys, kKeys, 1, 65536u, a.k_tiles};
  pa.op[2] = PlaneOperand{static_cast<const float*>(p.v), v, p.offsets_k, {p.vs[0], p.vs[1]}, p.tokens_k, kKeys, kKeys, 1, 65536u, a.k_tiles};
  const int64_t tiles = a.q_tiles > a.k_tiles ? a.q_tiles : a.k_tiles;
  if (launch_dependent(packed_planes_kernel<kCols>, dim3(unsigned(tiles), unsigned(p.kv_heads), 3), dim3(128), 0, st, pa) != cudaSuccess)
    return check_launch("packed_planes_kernel");
  count_launch();
  if (int rc = check_launch("packed_planes_kernel")) return rc;
  if (launch_dependent(kernel, dim3(unsigned(blocks)), dim3(L::kThreads), L::kBytes, st, a) != cudaSuccess) return check_launch("packed_fwd_fp32_kernel");
  count_launch();
  return check_launch("packed_fwd_fp32_kernel");
}

}  // namespace

// Where these kernels win over the fp32 units: the lengths are known on the device only, so the rule is on their averages.
// Forward with equal lengths, causal, us, here / there (sequences x tokens, key heads x query heads of each):
//  D 64: 4 x 64, 2 x 4 12 / 10; 256 x 64, 1 x 1 35 / 16, 8 x 1 161 / 115, 8 x 8 453 / 762  <  the line  <  1 x 128, 2 x 4 13 / 15;
//   256 x 128, 1 x 1 43 / 37, 2 x 4 134 / 249; 4 x 256, 8 x 1 17 / 39; 8 x 512, 4 x 4 50 / 171; 4 x 2048, 4 x 4 179 / 1043; 1 x 8192,
//   8 x 8 2379 (231 TFLOP/s) / 14292
//  D 128: 32 x 64, 8 x 1 38 / 28; 4 x 64, 4 x 4 18 / 15  <  the line  <  4 x 128, 4 x 4 21 / 23; 256 x 128, 8 x 1 377 / 583; 64 x 512,
//   4 x 4 754 / 2394; 1 x 2048, 4 x 4 119 / 506; 1 x 8192, 8 x 8 6280 (175 TFLOP/s) / 28795
// The planes are 1.5 times the operands (and a tile per sequence): beyond 8 GiB of them a caller is more likely to miss the
// memory than the time.
bool fp32_packed_supported(const PackedArgs& a, int dtype) {
  if (dtype != NB200_F32 || (a.D != 64 && a.D != 128) || a.group > kRows || a.tokens_q <= 0 || a.tokens_k <= 0 || a.sequences <= 0) return false;
  if (reinterpret_cast<uintptr_t>(a.out) % 16) return false;
  const int64_t blocks = query_tiles(a) * a.kv_heads;
  if (blocks > 0x7fffffff || query_tiles(a) > 0x7fffffff) return false;
  if (int64_t(a.tokens_q) * a.group < 64 * int64_t(a.sequences) || a.tokens_k < 128 * int64_t(a.sequences)) return false;
  return fp32_packed_fwd_bytes(a) <= (size_t(8) << 30);
}

size_t fp32_packed_fwd_bytes(const PackedArgs& a) { return list_bytes(a) + query_bytes(a) + 2 * key_bytes(a); }

int fp32_packed_fwd(const PackedArgs& p, void* ws, cudaStream_t st) { return p.D == 64 ? launch<64>(p, ws, st) : launch<128>(p, ws, st); }

}  // namespace packed
}  // namespace nb200
