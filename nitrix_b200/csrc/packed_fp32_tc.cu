// Attention over packed sequences with fp32 operands on the tcgen05 tensor cores, forward at head dim 64 and 128, backward at
// head dim 64 (at 128 the planes of an owner's two operands alone are 192 KB of shared memory): every fp32 number is three
// bf16 numbers and every product the six bf16 products that matter (sdpa_fp32_tc.cu has the error bounds and the scheme of a
// tile).
//
// packed_planes_kernel writes the planes of q, k, v and dout into the workspace as the tiles that the MMAs read, a sequence and
// key head at a time: 128 rows of queries, or 64 (token after token, the query heads of the key head), 64 keys.  Rows behind
// the end of a sequence are zeros there, so nothing of a neighbouring sequence gets near a sum; so are, for the sums over queries,
// those of queries that see no key.  The tiles of sequence i begin
// at tile begin / tokens per tile + i: sequences that follow one another never share one, and nobody has to add up the lengths.
// The other kernels fetch whole tiles by untiled bulk copies; their blocks come from the lists of packed_plan.cu.
//
// An infinity in a sequence's own operands becomes a NaN in its planes (x - x0), so that its scores are NaN where the fp32
// units may still give a number.
//
// Where these kernels run and where the fp32 units do: the rules and both sides are beside fp32_packed_supported and
// fp32_packed_bwd_supported.  Forward: bound by the chain of a step (scores, soft-max, P V of a tile follow one another; two
// tiles per CTA at head dim 64, one at 128, where the planes of one fill the shared memory): 84 % and 64 % of the 275 TFLOP/s
// that six products at the bf16 rate leave, long sequences.  Backward: one step of a CTA at a time, 1.5 us each by keys, 45 % of
// that rate.
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
  const int* keys;      // offsets of the keys, where the first queries of a sequence with fewer keys are to be zeros
  int total_keys;
};
struct PlaneArgs {
  PlaneOperand op[4];
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
    const int blind = op.keys ? span.y - sequence_span(op.keys, lo, op.total_keys).y - int(index) * op.tokens : 0;      // tokens left out
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
      if (token >= blind && token < n) {
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

// ---- backward, head dim 64 --------------------------------------------------------------------------------------------------
struct Fp32BwdArgs {
  WorkList list;
  const uint8_t* y[2];          // planes of the operands that are streamed: k, v (query-major) or q, dout (key-major)
  const uint8_t* x[2];          // key-major: planes of k, v
  const float* rows[2];         // query-major: q, dout
  int64_t rs[2][2];             // their element strides over (token, head)
  int64_t x_tiles, y_tiles;     // that there is room for
  int kv_heads, group, heads;
  int tokens;                   // queries of an owner's 128 rows (query-major) or of a step's 64 (key-major)
  uint32_t group_magic;
  int causal;
  float scale;
  const float* lse;             // (tokens, heads), and delta
  const float* delta;
  float* dx[2];                 // dq, or dk and dv: dense
  int* status;
};
template <bool kKeyMajor>
struct BwdLayout {
  static constexpr int kPlane = kKeys * kRowBytes;
  static constexpr int kStages = kKeyMajor ? 2 : 4;
  static constexpr int kX = 0;                                           // key-major: [K, V][3][128 rows x 128 B]
  static constexpr int kY = kX + (kKeyMajor ? 2 * 3 * 2 * kPlane : 0);   // [kStages][Y0, Y1][3][64 rows x 128 B]
  static constexpr int kStageBytes = 2 * 3 * kPlane;
  static constexpr int kSide = kY + kStages * kStageBytes;               // key-major: lse and delta, [2 stages][2][64]
  static constexpr int kSumDk = kSide + 2 * 2 * 64 * 4;                  // key-major: the sums of dk, [32 columns][256 threads]
  static constexpr int kBars = kKeyMajor ? kSumDk + 32 * 256 * 4 : kSide;
  static constexpr int kBytes = kBars + 256;
  // TMEM: S, dP, planes of dS; then key-major: planes of P, accumulators, sum of dV; query-major: planes of q and dout,
  // accumulator
  static constexpr int kTmS = 0, kTmDP = 64, kTmDS = 128, kTmP = 224, kTmX = 224, kTmAcc = kKeyMajor ? 320 : 416;
  static constexpr int kTmAcc2 = 384, kTmSum2 = 448, kTmCols = 512;
};
enum BwdBar { Y_FULL = 0, Y_EMPTY = 4, LSE_FULL = 8, X_FULL = 10, SP_FULL, SP_FREE, PD_FULL, ACC_DONE, kBwdBars };

// One scheme, two owners, as for dense operands.  Query-major (dq): a CTA owns 128 rows of a key head -- token after token, its
// query heads -- and streams the sequence's keys; key-major (dk, dv): it owns 128 keys and streams the rows, 64 / G tokens a step,
// so that the sums over the group's heads are part of the product.  With X0, X1 the owner's (q, dout) or (k, v) and Y0, Y1 the
// other pair, per step
//     S = X0 Y0^T,  dP = X1 Y1^T,   P = exp2(S scale log2 e - lse),  dS = P (dP - delta),   dq += dS Y0   or   dk += dS Y0, dv += P Y1
// Warps 0-7: element-wise, warps 0-3 the first 32 columns of a step, 4-7 the other 32, a thread per row; warp 8 fetches, 9 issues
// the products, 10 the accumulates.  The accumulators are emptied every other step into fp32 sums: dq's in registers, dk's in
// shared memory, dv's in TMEM.  Every sum has one order.
template <bool kKeyMajor>
__global__ void __launch_bounds__(352, 1) packed_bwd_fp32_kernel(const __grid_constant__ Fp32BwdArgs a) {
  using L = BwdLayout<kKeyMajor>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  int* abort_flag = reinterpret_cast<int*>(smem + L::kBars + 192);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBars + 196);
  // The key-major kernel comes last and needs nothing of the query-major one, which has waited for all before it when it lets
  // this one start: it waits at its end.
  if constexpr (!kKeyMajor) wait_for_previous();
  allow_dependents();
  const int place = int(blockIdx.x / unsigned(a.kv_heads)), head = int(blockIdx.x - unsigned(place) * unsigned(a.kv_heads));
  if ((sbase & 1023) || place >= *a.list.count) {
    if ((sbase & 1023) && threadIdx.x == 0) atomicExch(a.status, 620);
    if constexpr (kKeyMajor) wait_for_previous();
    return;
  }
  const WorkItem item = load_item(a.list.items + place);
  const int sequence = item.sequence;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // query-major: keys that token t of the block sees
  auto seen_by = [&](int t) { return a.causal ? int(min(max(int64_t(item.seen) + t, int64_t(0)), int64_t(item.other_n))) : item.other_n; };
  const int j0 = kKeyMajor && a.causal ? min(max(item.seen, 0), item.other_n) / a.tokens : 0;
  const int j1 = kKeyMajor ? (item.other_n + a.tokens - 1) / a.tokens : (seen_by(item.n - 1) + kKeys - 1) / kKeys;
  const int steps = max(0, j1 - j0);
  auto bar = [&](int i) { return sbase + L::kBars + 8 * i; };
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kBwdBars; ++i)
      mbar_init(bar(i), i == SP_FREE || i == PD_FULL || (!kKeyMajor && i == X_FULL) ? 256 : (i == LSE_FULL || i == LSE_FULL + 1 ? 32 : 1));
    mbar_init_fence();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), L::kTmCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tm = *tmem_slot;

  if (warp == 8) {
    // (offsets that run backwards may list blocks whose tiles nobody wrote, or for which there is no room)
    const int n_x = (item.n + kKeys - 1) / kKeys;
    int64_t x_tile = kKeyMajor ? first_tile(item.begin - item.index * kRows, kKeys, sequence) + 2 * int64_t(item.index) : 0;
    int64_t y_tile = first_tile(item.other, kKeyMajor ? a.tokens : kKeys, sequence);
    const bool room = (!kKeyMajor || (x_tile >= 0 && x_tile + n_x <= a.x_tiles)) && y_tile >= 0 && y_tile + j1 <= a.y_tiles;
    bool ok = true;
    if (kKeyMajor && lane == 0 && steps > 0) {
      mbar_expect_tx(bar(X_FULL), n_x * 2 * 3 * L::kPlane);
      for (int w = 0; w < 2; ++w)
        for (int t = 0; t < n_x; ++t) {
          const uint8_t* src = a.x[w] + ((room ? x_tile + t : 0) * a.kv_heads + head) * (3 * L::kPlane);
          for (int i = 0; i < 3; ++i)
            bulk_load(sbase + L::kX + ((w * 3 + i) * 2 + t) * L::kPlane, src + i * L::kPlane, L::kPlane, bar(X_FULL));
        }
    }
    __syncwarp();
    for (int i = 0; i < steps && ok; ++i) {
      const int st = i % kStages, j = j0 + i;
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(Y_EMPTY + st), ((i / kStages) & 1) ^ 1, abort_flag, a.status, 621));
      if (!ok) break;
      if (lane == 0) {
        const int64_t at = ((room ? y_tile + j : 0) * a.kv_heads + head) * int64_t(3 * L::kPlane);
        mbar_expect_tx(bar(Y_FULL + st), L::kStageBytes);
        bulk_load(sbase + L::kY + st * L::kStageBytes, a.y[0] + at, 3 * L::kPlane, bar(Y_FULL + st));
        bulk_load(sbase + L::kY + st * L::kStageBytes + 3 * L::kPlane, a.y[1] + at, 3 * L::kPlane, bar(Y_FULL + st));
      }
      if constexpr (kKeyMajor) {
        // (zeros where there is no row: those of q and dout are zeros as well)
        float* side = reinterpret_cast<float*>(smem + L::kSide) + st * 128;
        for (int r = lane; r < kKeys; r += 32) {
          const int t = int((uint32_t(r) * a.group_magic) >> 16), token = j * a.tokens + t;
          const bool in = t < a.tokens && token < item.other_n;
          const int64_t at = (int64_t(item.other) + token) * a.heads + head * a.group + (r - t * a.group);
          side[r] = in ? a.lse[at] : 0.f;
          side[64 + r] = in ? a.delta[at] : 0.f;
        }
        mbar_arrive(bar(LSE_FULL + st));
      }
    }
    if (!ok) tc::drain_after_abort();
  } else if (warp == 9) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc(true, kRows, kKeys, false, false);
      const uint64_t x0 = make_smem_desc(sbase + L::kX, 16, 1024);
      const uint64_t y0 = make_smem_desc(sbase + L::kY, 16, 1024);
      bool ok = steps == 0 || wait_or_abort(bar(X_FULL), 0, abort_flag, a.status, 622);
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i % kStages;
        ok = wait_or_abort(bar(Y_FULL + st), (i / kStages) & 1, abort_flag, a.status, 623) &&
             (i == 0 || wait_or_abort(bar(SP_FREE), (i - 1) & 1, abort_flag, a.status, 624));
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t ys = y0 + uint64_t((st * L::kStageBytes) >> 4);
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int t = 0; t < kProducts; ++t)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t yd = ys + uint64_t(((w * 3 + right_plane(t)) * L::kPlane + kk * 32) >> 4);
              if constexpr (kKeyMajor)
                mma_ss(tm + (w ? L::kTmDP : L::kTmS), x0 + uint64_t(((w * 3 + left_plane(t)) * 2 * L::kPlane + kk * 32) >> 4), yd, idesc,
                       t + kk > 0 ? 1u : 0u);
              else
                mma_ts(tm + (w ? L::kTmDP : L::kTmS), tm + L::kTmX + (w * 3 + left_plane(t)) * 32 + kk * 8, yd, idesc, t + kk > 0 ? 1u : 0u);
            }
        mma_commit(bar(SP_FULL));
      }
    }
  } else if (warp == 10) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc(true, kRows, 64, false, true);
      const uint64_t y0 = make_smem_desc(sbase + L::kY, L::kPlane, 1024);
      bool ok = true;
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i % kStages;
        ok = wait_or_abort(bar(Y_FULL + st), (i / kStages) & 1, abort_flag, a.status, 625) &&
             wait_or_abort(bar(PD_FULL), i & 1, abort_flag, a.status, 626);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t ys = y0 + uint64_t((st * L::kStageBytes) >> 4);
#pragma unroll
        for (int w = 0; w < (kKeyMajor ? 2 : 1); ++w)      // dS Y0, then P Y1
#pragma unroll
          for (int t = 0; t < kProducts; ++t)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ts(tm + (w ? L::kTmAcc2 : L::kTmAcc), tm + (w ? L::kTmP : L::kTmDS) + left_plane(t) * 32 + kk * 8,
                     ys + uint64_t(((w * 3 + right_plane(t)) * L::kPlane + kk * 2048) >> 4), idesc, (i > 0 || t + kk > 0) ? 1u : 0u);
        mma_commit(bar(Y_EMPTY + st));
        mma_commit(bar(ACC_DONE));
      }
    }
  } else {
    const int half = warp >> 2, quad = warp & 3, r = quad * 32 + lane;      // this thread's row of the owner
    const uint32_t tl = tm + (uint32_t(quad * 32) << 16);
    const float mul = a.scale * kLog2e;
    // query-major
    const int token = int((uint32_t(r) * a.group_magic) >> 16), member = r - token * a.group;
    const bool mine = kKeyMajor ? r < item.n : token < item.n;
    const int64_t row = kKeyMajor ? (int64_t(item.begin) + r) * a.kv_heads + head
                                  : (int64_t(item.begin) + token) * a.heads + head * a.group + member;
    const int seen = !kKeyMajor && mine ? seen_by(token) : 0;
    float lse = 0.f, delta = 0.f;
    if constexpr (!kKeyMajor) {
      if (mine) {
        lse = a.lse[row];
        delta = a.delta[row];
      }
      // this thread's row of q (warps 0-3) or dout (4-7), split into TMEM
      const float* xp = a.rows[half];
      const int64_t s0 = a.rs[half][0], s1 = a.rs[half][1];
      const bool vec = ((reinterpret_cast<uintptr_t>(xp) & 15) == 0) && ((s0 | s1) & 3) == 0;
      xp += (int64_t(item.begin) + token) * s0 + (head * a.group + member) * s1;
      uint32_t x[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) x[c] = 0u;
      if (mine) {
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          if (vec) {
            const uint4 v = *reinterpret_cast<const uint4*>(xp + c);
            x[c] = v.x; x[c + 1] = v.y; x[c + 2] = v.z; x[c + 3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[c + e] = __float_as_uint(xp[c + e]);
          }
        }
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        uint32_t o[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = __byte_perm(x[2 * c], x[2 * c + 1], 0x7632);
        tmem_st32(tl + L::kTmX + (half * 3 + p) * 32, o);
        if (p < 2) {
#pragma unroll
          for (int c = 0; c < 64; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) - __uint_as_float(x[c] & 0xffff0000u));
        }
      }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(bar(X_FULL));
    }
    float sum[32];                                                              // of dq, this thread's row and 32 columns
    float* sum_dk = reinterpret_cast<float*>(smem + L::kSumDk) + threadIdx.x;   // of dk, a column every 256
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      if constexpr (kKeyMajor) sum_dk[c * 256] = 0.f;
      else sum[c] = 0.f;
    }
    bool ok = true;
    for (int i = 0; i < steps && ok; ++i) {
      const int j = j0 + i;
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(SP_FULL), i & 1, abort_flag, a.status, 627) &&
                                       (!kKeyMajor || wait_or_abort(bar(LSE_FULL + (i & 1)), (i >> 1) & 1, abort_flag, a.status, 628)));
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t s[32], d[32];
      tmem_ld32(tl + L::kTmS + half * 32, s);
      tmem_ld32(tl + L::kTmDP + half * 32, d);
      tmem_wait_ld();
      tc_fence_before_sync();
      mbar_arrive(bar(SP_FREE));
      const float* side = reinterpret_cast<const float*>(smem + L::kSide) + (i & 1) * 128 + half * 32;
      // columns kept: first <= c < end
      int first = 0, end = 0;
      if constexpr (kKeyMajor) {
        // (row y of a step is a query from token y / G on: at or behind token t where y >= t G)
        const int from = a.causal ? min(max(item.seen + r - j * a.tokens, 0), a.tokens) : 0;
        first = mine ? from * a.group - half * 32 : 64;
        end = min(item.other_n - j * a.tokens, a.tokens) * a.group - half * 32;
      } else {
        end = seen - j * kKeys - half * 32;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const bool in = (!kKeyMajor || c >= first) && c < end;
        const float ref = kKeyMajor ? side[c] : lse, dl = kKeyMajor ? side[64 + c] : delta;
        const float p = in ? tc::ex2(fmaf(__uint_as_float(s[c]), mul, -ref)) : 0.f;
        s[c] = __float_as_uint(p);
        d[c] = in ? __float_as_uint(p * (__uint_as_float(d[c]) - dl)) : 0u;
      }
      if (i > 0) {
        ok = __all_sync(0xffffffffu, wait_or_abort(bar(ACC_DONE), (i - 1) & 1, abort_flag, a.status, 629));
        if (!ok) break;
        tc_fence_after_sync();
        if ((i & 1) == 0) {
          uint32_t v[32];
          tmem_ld32(tl + L::kTmAcc + half * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if constexpr (kKeyMajor) sum_dk[c * 256] += __uint_as_float(v[c]);
            else sum[c] += __uint_as_float(v[c]);
            v[c] = 0u;
          }
          tmem_st32(tl + L::kTmAcc + half * 32, v);
        } else if (kKeyMajor && i > 1) {
          uint32_t v[32], w[32];
          tmem_ld32(tl + L::kTmAcc2 + half * 32, v);
          if (i > 3) tmem_ld32(tl + L::kTmSum2 + half * 32, w);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            w[c] = i > 3 ? __float_as_uint(__uint_as_float(w[c]) + __uint_as_float(v[c])) : v[c];
            v[c] = 0u;
          }
          tmem_st32(tl + L::kTmSum2 + half * 32, w);
          tmem_st32(tl + L::kTmAcc2 + half * 32, v);
        }
      }
#pragma unroll
      for (int w = 0; w < (kKeyMajor ? 2 : 1); ++w) {
        uint32_t(&v)[32] = w ? s : d;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          uint32_t o[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) o[c] = __byte_perm(v[2 * c], v[2 * c + 1], 0x7632);
          tmem_st16(tl + (w ? L::kTmP : L::kTmDS) + p * 32 + half * 16, o);
          if (p < 2) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) - __uint_as_float(v[c] & 0xffff0000u));
          }
        }
      }
      tmem_wait_st();
      tc_fence_before_sync();
      mbar_arrive(bar(PD_FULL));
    }
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(ACC_DONE), (steps - 1) & 1, abort_flag, a.status, 630));
      tc_fence_after_sync();
    }
    if (ok) {
#pragma unroll
      for (int w = 0; w < (kKeyMajor ? 2 : 1); ++w) {
        const float scale = w ? 1.f : a.scale;
        uint32_t o[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = 0u;
        if (steps > 0) {
          tmem_ld32(tl + (w ? L::kTmAcc2 : L::kTmAcc) + half * 32, o);
          tmem_wait_ld();
          if (w == 0) {
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint((kKeyMajor ? sum_dk[c * 256] : sum[c]) + __uint_as_float(o[c]));
          } else if (steps > 3) {
            uint32_t t[32];
            tmem_ld32(tl + L::kTmSum2 + half * 32, t);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(t[c]) + __uint_as_float(o[c]));
          }
        }
        if (mine) {
          float* op = a.dx[w] + row * 64 + half * 32;
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * scale);
#pragma unroll
          for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(op + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (*abort_flag) tc::drain_after_abort();
  if (warp == 9) tmem_dealloc(tm, L::kTmCols);
  if constexpr (kKeyMajor) wait_for_previous();
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

int64_t step_tiles(const PackedArgs& a) { return most_blocks(a.tokens_q, a.sequences, tile_tokens(kKeys, a.group)); }
size_t step_bytes(const PackedArgs& a) { return size_t(step_tiles(a)) * a.kv_heads * (kKeys * a.D * 6); }
size_t bwd_list_bytes(const PackedArgs& a, bool key_major) {
  return key_major ? work_list_bytes(most_blocks(a.tokens_k, a.sequences, kRows)) : work_list_bytes(query_tiles(a));
}

template <bool kKeyMajor>
int launch_bwd(const Fp32BwdArgs& a, int64_t blocks, cudaStream_t st) {
  using L = BwdLayout<kKeyMajor>;
  static_assert(L::kBytes <= 232448, "shared memory of a CTA");
  auto kernel = packed_bwd_fp32_kernel<kKeyMajor>;
  const char* name = kKeyMajor ? "packed_dkv_fp32_kernel" : "packed_dq_fp32_kernel";
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess) return check_launch(name);
  if (launch_dependent(kernel, dim3(unsigned(blocks)), dim3(352), L::kBytes, st, a) != cudaSuccess) return check_launch(name);
  count_launch();
  return check_launch(name);
}

PlaneOperand plane_operand(const void* x, uint8_t* planes, const int* offsets, const int64_t (&xs)[2], int total, int rows, int heads, int64_t tiles) {
  return PlaneOperand{static_cast<const float*>(x), planes, offsets, {xs[0], xs[1]}, total, tile_tokens(rows, heads), rows, heads,
                      uint32_t((65536 + heads - 1) / heads), tiles, nullptr, 0};
}
int launch_planes(const PlaneArgs& pa, int D, int operands, int64_t tiles, cudaStream_t st) {
  const dim3 grid(unsigned(tiles), unsigned(pa.kv_heads), unsigned(operands));
  if (launch_dependent(D == 64 ? packed_planes_kernel<64> : packed_planes_kernel<128>, grid, dim3(128), 0, st, pa) != cudaSuccess)
    return check_launch("packed_planes_kernel");
  count_launch();
  return check_launch("packed_planes_kernel");
}

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
  pa.op[0] = plane_operand(p.q, q, p.offsets_q, p.qs, p.tokens_q, kRows, p.group, a.q_tiles);
  pa.op[1] = plane_operand(p.k, k, p.offsets_k, p.ks, p.tokens_k, kKeys, 1, a.k_tiles);
  pa.op[2] = plane_operand(p.v, v, p.offsets_k, p.vs, p.tokens_k, kKeys, 1, a.k_tiles);
  if (int rc = launch_planes(pa, kCols, 3, a.q_tiles > a.k_tiles ? a.q_tiles : a.k_tiles, st)) return rc;
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

// Backward, us, here / there: a CTA of the key-major kernel walks over all rows of its 128 keys, G tokens' worth of the walk for
// a token, while the fp32 units cut the walk into parts where there are few keys.  Blocks of 128 keys, all key heads:
//  G 1 to 3: 1 block 22 / 39 (G 1), 29 / 39 (G 2); 8 blocks 39 / 39 (G 3)
//  G 4: 8 blocks 42 / 40, 109 / 106  <  the line  <  16 blocks 44 / 53, 203 / 364
//  G 8 to 64: 16 blocks 768 / 673, 70 / 90 (G 8), 1517 / 1308 (G 16), 950 / 888 (G 64)  <  the line  <  32 blocks 94 / 143, 1575 /
//   2165 (G 8), 1109 / 1572 (G 64)
//  4 x 2048 tokens, 4 x 4 heads 885 / 4122; 1 x 8192, 8 x 8 11084 / 58688
bool fp32_packed_bwd_supported(const PackedArgs& a, int dtype) {
  if (!fp32_packed_supported(a, dtype) || a.D != 64 || a.group > kKeys) return false;
  if (a.group > 3 && a.tokens_k / kRows * int64_t(a.kv_heads) < (a.group < 8 ? 16 : 32)) return false;
  if (reinterpret_cast<uintptr_t>(a.dq) % 16 || reinterpret_cast<uintptr_t>(a.dk) % 16 || reinterpret_cast<uintptr_t>(a.dv) % 16) return false;
  if (step_tiles(a) > 0x7fffffff || most_blocks(a.tokens_k, a.sequences, kRows) * a.kv_heads > 0x7fffffff) return false;
  return fp32_packed_bwd_bytes(a) <= (size_t(8) << 30);
}

size_t fp32_packed_bwd_bytes(const PackedArgs& a) {
  return bwd_list_bytes(a, false) + bwd_list_bytes(a, true) + 2 * step_bytes(a) + 2 * key_bytes(a);
}

// `p.delta` has been written.
int fp32_packed_bwd(const PackedArgs& p, void* ws, cudaStream_t st) {
  char* lists[2] = {static_cast<char*>(ws), static_cast<char*>(ws) + bwd_list_bytes(p, false)};
  uint8_t* q = reinterpret_cast<uint8_t*>(lists[1]) + bwd_list_bytes(p, true);
  uint8_t* planes[4] = {q, q + step_bytes(p), q + 2 * step_bytes(p), q + 2 * step_bytes(p) + key_bytes(p)};   // q, dout, k, v
  const int owner_tokens = tile_tokens(kRows, p.group), step_tokens = tile_tokens(kKeys, p.group);
  Fp32BwdArgs a{};
  a.status = device_status_word();
  if (!a.status) { set_error("packed_bwd: no status word on this device"); return NB200_ERR_LAUNCH; }
  if (int rc = launch_plan(p, true, kRows, step_tokens, lists[1], st, sizeof(float))) return rc;
  if (int rc = launch_plan(p, false, owner_tokens, 1, lists[0], st, 0)) return rc;
  PlaneArgs pa{};
  pa.sequences = p.sequences;
  pa.kv_heads = p.kv_heads;
  pa.op[0] = plane_operand(p.q, planes[0], p.offsets_q, p.qs, p.tokens_q, kKeys, p.group, step_tiles(p));
  pa.op[1] = plane_operand(p.dout, planes[1], p.offsets_q, p.dos, p.tokens_q, kKeys, p.group, step_tiles(p));
  if (p.causal) {
    for (int i = 0; i < 2; ++i) { pa.op[i].keys = p.offsets_k; pa.op[i].total_keys = p.tokens_k; }
  }
  pa.op[2] = plane_operand(p.k, planes[2], p.offsets_k, p.ks, p.tokens_k, kKeys, 1, key_tiles(p));
  pa.op[3] = plane_operand(p.v, planes[3], p.offsets_k, p.vs, p.tokens_k, kKeys, 1, key_tiles(p));
  if (int rc = launch_planes(pa, p.D, 4, step_tiles(p) > key_tiles(p) ? step_tiles(p) : key_tiles(p), st)) return rc;
  a.kv_heads = p.kv_heads; a.group = p.group; a.heads = p.heads;
  a.group_magic = pa.op[0].heads_magic;
  a.causal = p.causal;
  a.scale = p.scale;
  a.lse = p.lse;
  a.delta = p.delta;
  for (int key_major = 0; key_major < 2; ++key_major) {
    a.list.count = reinterpret_cast<const int*>(lists[key_major]);
    a.list.items = reinterpret_cast<const WorkItem*>(lists[key_major] + 16);
    if (!key_major) {
      a.tokens = owner_tokens;
      a.y[0] = planes[2]; a.y[1] = planes[3];
      a.y_tiles = key_tiles(p);
      a.rows[0] = static_cast<const float*>(p.q); a.rows[1] = static_cast<const float*>(p.dout);
      for (int i = 0; i < 2; ++i) { a.rs[0][i] = p.qs[i]; a.rs[1][i] = p.dos[i]; }
      a.dx[0] = static_cast<float*>(p.dq);
      if (int rc = launch_bwd<false>(a, query_tiles(p) * p.kv_heads, st)) return rc;
    } else {
      a.tokens = step_tokens;
      a.x[0] = planes[2]; a.x[1] = planes[3];
      a.y[0] = planes[0]; a.y[1] = planes[1];
      a.x_tiles = key_tiles(p);
      a.y_tiles = step_tiles(p);
      a.dx[0] = static_cast<float*>(p.dk); a.dx[1] = static_cast<float*>(p.dv);
      if (int rc = launch_bwd<true>(a, most_blocks(p.tokens_k, p.sequences, kRows) * p.kv_heads, st)) return rc;
    }
  }
  return NB200_OK;
}

}  // namespace packed
}  // namespace nb200
