// Forward attention over packed sequences for sm_100a: TMA -> shared memory -> tcgen05.mma with TMEM accumulators, fp32 online
// softmax in registers; bf16 and fp16, head dim 64 and 128, any group of up to 64 query heads per key head.
//
//   S = Q K^T, P = exp2(S scale log2 e - m), O = P V / sum P,  query i of a sequence sees keys up to i + lk - lq (causal)
//
// The rows of a query tile are, token after token, the query heads of one key head: 128 / G tokens fill 128 rows (some rows
// stay unused where G is no divisor), one TMA box brings them in that order, and a short sequence fills a tile G times as far
// as it would head by head; the keys are read once for the group.
//
// PERSISTENT: one CTA per SM takes blocks from a list (packed_plan.cu), the next one whenever it has loaded all of the last (the
// warp that loads takes it and hands its number on through a ring in shared memory);
// a block is two query tiles of one key head, for which the key tiles are streamed once.  Warps: 0 loads Q, K and V; 1 clears
// the rows of a sequence's last V tile that belong to its neighbour (their probabilities are zeros, but 0 * NaN is NaN; keys
// behind the end are masked by selection, and rows of Q behind the end stay in rows that nobody stores); 2 and 3 issue the
// MMAs of query tile 0 and 1; the others are the softmax, one thread per row at head dim 128, two at 64.  The scheme of the
// tiles -- halves of 64 keys whose P overwrites S at head dim 128, separate P at 64, a reference maximum that moves only past
// 2^8, every third pair of exponentials on the FMA units at head dim 128 -- is that of sdpa_tc_fwd.cu, which has the reasons.
// Head dim 128: bound by the tensor pipe with its operand fetch (busy 82 % of the time, 63 % of it multiplying: the MMAs of a half
// read 6 KB of operands for 32 cycles of products) at the clock that the power cap leaves; 8192 tokens, 16 heads on 4, 469 us (1170
// TFLOP/s), causal 232 (1180).  Key tiles taken whole, with N = 128 and the query tiles in turn, 606 -> 730 us.  Head dim 64: 398 and
// 207 us (690 and 660 TFLOP/s); what bounds it is not known: not the exponentials, of which every fourth on the FMA units changes nothing.
// All waits on mbarriers are bounded (sdpa_tc_common.cuh).
#include <type_traits>

#include "dependent_launch.cuh"
#include "packed_tc.cuh"

namespace nb200 {
namespace packed {

using namespace sm100;
using namespace tc;

namespace {

struct FwdArgs {
  WorkList list;
  int kv_heads, group, heads;
  int tokens;                // query tokens of a tile
  uint32_t group_magic;      // ceil(2^16 / group): row of a tile -> its token
  int causal;
  float scale;
  void* out;                 // dense (tokens, heads, D)
  float* lse;
  int* status;
  int out_v8;                // rows of out on 32-byte boundaries
  int smem_bytes;
};

template <int D>
struct Split {
  static constexpr int kHalves = D == 64 ? 2 : 1;       // threads per query row
  static constexpr int kThreads = 128 + 256 * kHalves;
  static constexpr int kLaunchRegs = kHalves == 1 ? 168 : 96;
  static constexpr int kProducerRegs = kHalves == 1 ? 56 : 64;
  static constexpr int kSoftmaxRegs = kHalves == 1 ? 216 : 104;
  static_assert((kLaunchRegs - kProducerRegs) * 128 >= (kSoftmaxRegs - kLaunchRegs) * 256 * kHalves,
                "softmax warps would wait forever for registers the producer warps never release");
};
// D = 128: one pair of exponentials in this many on the FMA units (every second 491 us, fourth 477, third 471 and 240 causal: 8192
// tokens, 16 heads on 4).  None at 64, where every fourth or eighth changes nothing and every sixteenth costs 8 %.
constexpr int kPolyPeriod = 3;

template <int D>
struct FwdSmem {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 64 ? 5 : 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kBars = kV + kStages * kTileBytes;
  static constexpr int kItems = 4;                        // numbers of blocks on their way to the other warps
  // q_full[2] q_empty[2] k_full[S] k_empty[S] v_full[S] v_empty[S] v_clear[S] s_full[4] p_ready[4] o_done[2] o_free[2] s_free[2]
  // pv_done[2] i_full[I] i_empty[I]
  static constexpr int kNumBars = 4 + 5 * kStages + 16 + 2 * kItems;
  static constexpr int kMisc = kBars + 8 * kNumBars;
  static constexpr int kItemRing = kMisc + 16;
  static constexpr int kExchange = kItemRing + 4 * kItems;   // one fp32 per query row of both tiles
  static constexpr int kTotal = kExchange + 2 * kTile * 4;
};

struct Item {
  int head;                 // key head
  int q0;                   // first query token
  int n;                    // query tokens of both tiles
  int k0, lk;
  int seen;                 // keys that the first query sees, before clamping (causal)
  int n0, n1;               // query tokens of the tiles
  int nt0, nt1, nt_max;     // key tiles
  bool tail;                // the block's last key tile is the sequence's last and not full
  __device__ __forceinline__ int nt(int g) const { return g ? nt1 : nt0; }
  __device__ __forceinline__ int tokens(int g) const { return g ? n1 : n0; }
};

// Piece of work `pos`: a block for one key head.
__device__ __forceinline__ void decode_item(const FwdArgs& a, int pos, Item* it) {
  const int entry = pos / a.kv_heads;
  const WorkItem w = load_item(a.list.items + entry);
  it->head = pos - entry * a.kv_heads;
  it->q0 = w.begin; it->n = w.n; it->k0 = w.other; it->lk = w.other_n; it->seen = w.seen;
  it->n0 = min(w.n, a.tokens);
  it->n1 = w.n - it->n0;
  auto tiles = [&](int end) {      // key tiles for the queries of the block before `end`
    const int keys = a.causal ? min(max(w.seen + end - 1, 0), w.other_n) : w.other_n;
    return (keys + kTile - 1) / kTile;
  };
  it->nt0 = tiles(it->n0);
  it->nt1 = it->n1 > 0 ? tiles(w.n) : 0;
  it->nt_max = max(it->nt0, it->nt1);
  it->tail = it->nt_max * kTile > w.other_n;
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(Split<D>::kThreads, 1)
packed_fwd_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const FwdArgs a) {
  using L = FwdSmem<D>;
  constexpr int kStages = L::kStages, kHalves = Split<D>::kHalves;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem + L::kTotal > smem_raw + a.smem_bytes) {   // never expected; refuse rather than overrun
    if (threadIdx.x == 0) atomicExch(a.status, 499);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  constexpr int Q_FULL = 0, Q_EMPTY = 2, K_FULL = 4, K_EMPTY = K_FULL + kStages, V_FULL = K_EMPTY + kStages,
                V_EMPTY = V_FULL + kStages, V_CLEAR = V_EMPTY + kStages, S_FULL = V_CLEAR + kStages, P_READY = S_FULL + 4,
                O_DONE = P_READY + 4, O_FREE = O_DONE + 2, S_FREE = O_FREE + 2, PV_DONE = S_FREE + 2, I_FULL = PV_DONE + 2,
                I_EMPTY = I_FULL + L::kItems;
  static_assert(I_EMPTY + L::kItems == L::kNumBars, "barrier count");
  constexpr bool kAlias = D == 128;      // P over S, key tiles in halves
  constexpr int kPoly = kAlias ? kPolyPeriod : 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kNumBars; ++i) {
      uint32_t count = 1;
      if (i >= P_READY && i < P_READY + 4) count = 4 * kHalves;                 // one lane per softmax warp of the tile
      if (i >= K_EMPTY && i < K_EMPTY + kStages) count = 2;                     // one arrival per MMA issuer
      if (i >= V_EMPTY && i < V_EMPTY + kStages) count = 3;                     // and one of the warp that clears tails
      if (i >= O_FREE && i < O_FREE + 2) count = 4 * kHalves;
      if (i >= S_FREE && i < S_FREE + 2) count = 4 * kHalves;
      if (i >= I_EMPTY && i < I_EMPTY + L::kItems) count = 3 + 8 * kHalves;      // warp 1, two issuers, the softmax warps
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 3) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  auto tm_S = [&](int g) { return tmem + g * 128; };
  auto tm_P = [&](int g) { return kAlias ? tmem + g * 128 : tmem + 256 + g * 64; };
  auto tm_O = [&](int g) { return kAlias ? tmem + 256 + g * D : tmem + 384 + g * D; };
  wait_for_previous();       // the work list is written by the launch before
  volatile int* const items = reinterpret_cast<volatile int*>(smem + L::kItemRing);
  // The `n`-th piece of work of this CTA, for every warp but the one that takes them: waits for its number (-1: no more, -2: the
  // wait was given up); give_back() once it has been read.
  auto next_item = [&](int n) {
    if (!wait_or_abort(bar(I_FULL + n % L::kItems), (n / L::kItems) & 1, abort_flag, a.status, 416)) return -2;
    return items[n % L::kItems];
  };
  auto give_back = [&](int n) { mbar_arrive(bar(I_EMPTY + n % L::kItems)); };

  // Phase bookkeeping across blocks (every role derives the same numbers from the same list):
  //   n    blocks that this CTA has taken so far
  //   kv   key tiles streamed so far            -> ring stage kv % kStages, phase (kv / kStages) & 1
  //   tc_g tiles query tile g has processed     -> phase of s_full / p_ready / s_free / pv_done
  //   oc_g blocks in which query tile g had any -> phase of q_full / q_empty / o_done / o_free
  //   clear: bit s is the phase of v_clear[s], which sees the tails only
  if (warp < 4) {
  Item it;
  reg_dealloc<Split<D>::kProducerRegs>();
  if (warp == 0) {
    // ---------------- Q / K / V ----------------
    if (elect_one()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int kv = 0, oc[2] = {0, 0};
      bool ok = true;
      const int total = *reinterpret_cast<const volatile int*>(a.list.count) * a.kv_heads;
      int pos = int(blockIdx.x) < total ? int(blockIdx.x) : -1;
      for (int n = 0;; ++n) {
        if (n >= L::kItems) ok = ok && wait_or_abort(bar(I_EMPTY + n % L::kItems), (n / L::kItems - 1) & 1, abort_flag, a.status, 417);
        if (!ok) break;
        items[n % L::kItems] = pos;
        mbar_arrive(bar(I_FULL + n % L::kItems));
        if (pos < 0) break;
        const int next = int(gridDim.x) + atomicAdd(a.list.taken, 1);      // (its latency runs under this block's loads)
        decode_item(a, pos, &it);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (it.nt(g) == 0) continue;
          if (oc[g] > 0) ok = ok && wait_or_abort(bar(Q_EMPTY + g), (oc[g] - 1) & 1, abort_flag, a.status, 400);
          if (!ok) break;
          mbar_expect_tx(bar(Q_FULL + g), uint32_t(a.tokens * a.group) * (D * 2));
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(sbase + L::kQ + g * L::kTileBytes + x * kBoxBytes, &tm_q, bar(Q_FULL + g), x * 64, it.head * a.group,
                        it.q0 + g * a.tokens, 0);
          ++oc[g];
        }
        for (int j = 0; j < it.nt_max && ok; ++j, ++kv) {
          const int st = kv % kStages;
          const uint32_t ph = (kv / kStages) & 1;
          if (!wait_or_abort(bar(K_EMPTY + st), ph ^ 1, abort_flag, a.status, 401)) { ok = false; break; }
          mbar_expect_tx(bar(K_FULL + st), L::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(sbase + L::kK + st * L::kTileBytes + x * kBoxBytes, &tm_k, bar(K_FULL + st), x * 64, it.head, it.k0 + j * kTile, 0);
          if (!wait_or_abort(bar(V_EMPTY + st), ph ^ 1, abort_flag, a.status, 402)) { ok = false; break; }
          mbar_expect_tx(bar(V_FULL + st), L::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(sbase + L::kV + st * L::kTileBytes + x * kBoxBytes, &tm_v, bar(V_FULL + st), x * 64, it.head, it.k0 + j * kTile, 0);
        }
        pos = next < total ? next : -1;
      }
    }
  } else if (warp == 1) {
    // ---------------- the neighbours' rows of a last V tile ----------------
    // (Every tile is waited for and given back, also those without a tail: a waiter that passes phases by would take an old one
    // of the same parity for its own, and one that holds nothing back could fall behind by two.)
    int kv = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int pos = next_item(n);
      if (!__all_sync(0xffffffffu, pos >= 0)) break;
      if (lane == 0) give_back(n);
      decode_item(a, pos, &it);
      for (int j = 0; j < it.nt_max; ++j, ++kv) {
        const int st = kv % kStages;
        ok = __all_sync(0xffffffffu, wait_or_abort(bar(V_FULL + st), (kv / kStages) & 1, abort_flag, a.status, 403));
        if (!ok) break;
        if (it.tail && j == it.nt_max - 1) {
          const int row0 = it.lk - j * kTile, words = (kTile - row0) * 8;      // of a box
          for (int i = lane; i < words * (D / 64); i += 32) {
            const int box = i / words, rem = i - box * words;
            st_shared_v4(sbase + L::kV + st * L::kTileBytes + box * kBoxBytes + row0 * 128 + rem * 16, make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();      // written by threads, read by the tensor core
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(V_CLEAR + st));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(V_EMPTY + st));
      }
    }
  } else {
    // ---------------- MMA issuers: warp 2 query tile 0, warp 3 query tile 1 ----------------
    const int g = warp - 2;
    if (elect_one()) {
      constexpr uint32_t idesc_qk = make_idesc(kBf16, kTile, kAlias ? kTile / 2 : kTile, false, false);
      constexpr uint32_t idesc_pv = make_idesc(kBf16, kTile, D, false, true);
      const uint64_t qdesc = make_smem_desc(sbase + L::kQ + g * L::kTileBytes, 16, 1024);
      const uint64_t kdesc0 = make_smem_desc(sbase + L::kK, 16, 1024);
      const uint64_t vdesc0 = make_smem_desc(sbase + L::kV, kBoxBytes, 1024);
      const uint32_t tSg = tm_S(g), tPg = tm_P(g), tOg = tm_O(g);
      bool ok = true;
      int kv = 0, tc = 0, oc = 0;
      uint32_t clear = 0;
      for (int n = 0; ok; ++n) {
        const int pos = next_item(n);
        if (pos < 0) break;
        give_back(n);
        decode_item(a, pos, &it);
        const int nt = it.nt(g);
        // V of tile j is in shared memory, its tail cleared; of a tail that this query tile skips only the phase is noted
        auto wait_v = [&](int j) {
          const int st = (kv + j) % kStages;
          bool good = wait_or_abort(bar(V_FULL + st), ((kv + j) / kStages) & 1, abort_flag, a.status, 406);
          if (it.tail && j == it.nt_max - 1) {
            if (good && j < nt) good = wait_or_abort(bar(V_CLEAR + st), (clear >> st) & 1u, abort_flag, a.status, 404);
            clear ^= 1u << st;
          }
          return good;
        };
        if constexpr (kAlias) {
          // round u = 2 j + hf: the scores of half u, then the output of half u - 1
          const int n_sub = 2 * it.nt_max;
          for (int u = 0; u <= n_sub && ok; ++u) {
            const int j = u >> 1, hf = u & 1;
            const int jp = (u - 1) >> 1, hp = (u - 1) & 1;
            const int st = (kv + j) % kStages, stp = (kv + jp) % kStages;
            if (u < n_sub && hf == 0) {
              ok = wait_or_abort(bar(K_FULL + st), ((kv + j) / kStages) & 1, abort_flag, a.status, 405);
              if (!ok) break;
              tc_fence_after_sync();
            }
            if (u < n_sub) {
              if (j < nt) {
                if (u == 0) {
                  ok = wait_or_abort(bar(Q_FULL + g), oc & 1, abort_flag, a.status, 407);
                  if (!ok) break;
                  tc_fence_after_sync();
                }
                const uint32_t tS = tSg + hf * 64;
                const uint64_t kdesc = kdesc0 + uint64_t(st * (L::kTileBytes >> 4) + ((hf * 64 * 128) >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint64_t off = uint64_t(((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4);
                  mma_ss(tS, qdesc + off, kdesc + off, idesc_qk, kk > 0 ? 1u : 0u);
                }
                mma_commit(bar(S_FULL + 2 * g + hf));
                if (u == 2 * nt - 1) mma_commit(bar(Q_EMPTY + g));
              }
              if (hf == 1) mma_commit(bar(K_EMPTY + st));
            }
            if (u >= 1) {
              if (hp == 0) {
                ok = wait_v(jp);
                if (!ok) break;
              }
              if (jp < nt) {
                ok = wait_or_abort(bar(P_READY + 2 * g + hp), (tc + jp) & 1, abort_flag, a.status, 408);
                if (ok && u == 1 && oc > 0) ok = wait_or_abort(bar(O_FREE + g), (oc - 1) & 1, abort_flag, a.status, 415);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t tP = tSg + hp * 64;
                const uint64_t vdesc = vdesc0 + uint64_t(stp * (L::kTileBytes >> 4) + ((hp * 4 * 2048) >> 4));
#pragma unroll
                for (int kk = 0; kk < kTile / 32; ++kk)
                  mma_ts(tOg, tP + kk * 8, vdesc + uint64_t((kk * 2048) >> 4), idesc_pv, (u > 1 || kk > 0) ? 1u : 0u);
                mma_commit(bar(PV_DONE + g));
                if (u == 2 * nt) mma_commit(bar(O_DONE + g));
              }
              if (hp == 1) mma_commit(bar(V_EMPTY + stp));
            }
          }
        } else {
          // round j: the scores of key tile j, then the output of key tile j - 1
          for (int j = 0; j <= it.nt_max && ok; ++j) {
            const int st = (kv + j) % kStages, stp = (kv + j + kStages - 1) % kStages;
            if (j < it.nt_max) ok = wait_or_abort(bar(K_FULL + st), ((kv + j) / kStages) & 1, abort_flag, a.status, 405);
            if (ok && j > 0) ok = wait_v(j - 1);
            if (!ok) break;
            tc_fence_after_sync();
            if (j < nt) {
              const int gt = tc + j;
              if (j == 0) ok = wait_or_abort(bar(Q_FULL + g), oc & 1, abort_flag, a.status, 407);
              if (ok && gt > 0) ok = wait_or_abort(bar(S_FREE + g), (gt - 1) & 1, abort_flag, a.status, 411);
              if (!ok) break;
              tc_fence_after_sync();
              const uint64_t kdesc = kdesc0 + uint64_t(st * (L::kTileBytes >> 4));
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint64_t off = uint64_t(((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4);
                mma_ss(tSg, qdesc + off, kdesc + off, idesc_qk, kk > 0 ? 1u : 0u);
              }
              mma_commit(bar(S_FULL + g));
              if (j == nt - 1) mma_commit(bar(Q_EMPTY + g));
            }
            const int jj = j - 1;
            if (j > 0 && jj < nt) {
              ok = wait_or_abort(bar(P_READY + g), (tc + jj) & 1, abort_flag, a.status, 408);
              if (ok && jj == 0 && oc > 0) ok = wait_or_abort(bar(O_FREE + g), (oc - 1) & 1, abort_flag, a.status, 415);
              if (!ok) break;
              tc_fence_after_sync();
              const uint64_t vdesc = vdesc0 + uint64_t(stp * (L::kTileBytes >> 4));
#pragma unroll
              for (int kk = 0; kk < kTile / 16; ++kk)
                mma_ts(tOg, tPg + kk * 8, vdesc + uint64_t((kk * 2048) >> 4), idesc_pv, (jj > 0 || kk > 0) ? 1u : 0u);
              mma_commit(bar(PV_DONE + g));
              if (jj == nt - 1) mma_commit(bar(O_DONE + g));
            }
            if (j < it.nt_max) mma_commit(bar(K_EMPTY + st));
            if (j > 0) mma_commit(bar(V_EMPTY + stp));
          }
        }
        kv += it.nt_max;
        tc += nt;
        oc += nt > 0 ? 1 : 0;
      }
    }
  }
  } else {
    reg_alloc<Split<D>::kSoftmaxRegs>();
    // ---------------- softmax (a query row, or half of a pass's keys of one, per thread) ----------------
    const int g = ((warp - 4) >> 2) & 1;
    const int half = kHalves == 1 ? 0 : (warp - 4) >> 3;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lane_addr = uint32_t(wq * 32) << 16;
    constexpr int kSub = kAlias ? kTile / 2 : kTile;   // keys per pass
    constexpr int kSubs = kTile / kSub;
    constexpr int kCols = kSub / kHalves;              // keys per pass and thread
    constexpr int kOutCols = D / kHalves;              // output columns per thread
    const uint32_t tS = tm_S(g) + half * kCols + lane_addr, tO = tm_O(g) + half * kOutCols + lane_addr;
    const uint32_t tP = tm_P(g) + half * (kCols / 2) + lane_addr;
    float* const xrow = reinterpret_cast<float*>(smem + L::kExchange) + g * kTile + r;
    const uint32_t pair_bar = 1 + g * 4 + wq;          // named barrier of the two warps that share these rows
    bool ok = true;
    const float mul = a.scale * kLog2e;                // exponent = (s - m) * mul, base 2
    const float thr = 8.f / mul;
    const float2 mul2 = make_float2(mul, mul);
    const int token = int((uint32_t(r) * a.group_magic) >> 16), in_group = r - token * a.group;   // of this row's tile
    int tc = 0, oc = 0;

    // A warp that gives up (`ok` false) waits no more and stores nothing, but walks on through its passes: its partner waits
    // for it at the pair's barrier, which has no time limit of its own.
    for (int n = 0;; ++n) {
      const int pos = ok ? next_item(n) : -2;
      // (two warps that share rows end together: one that has given up takes its partner along)
      const bool last = kHalves == 1 ? !__all_sync(0xffffffffu, pos >= 0) : named_barrier_or(pair_bar, 64, pos < 0);
      if (last) break;
      if (lane == 0) give_back(n);
      // of the block only what the passes and the epilogue need: a spilled register costs more than anything here (head dim 64)
      int my_nt, seen, row;
      {
        Item it;
        decode_item(a, pos, &it);
        const int local = g * a.tokens + token;            // query of the block
        my_nt = it.nt(g);
        seen = a.causal ? min(it.seen + local, it.lk) : it.lk;
        row = token < it.tokens(g) ? (it.q0 + local) * a.heads + it.head * a.group + in_group : -1;   // of out; -1: none
      }
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < my_nt; ++j) {
        const int gt = tc + j;
#pragma unroll 1
        for (int hf = 0; hf < kSubs; ++hf) {
          const int key0 = j * kTile + hf * kSub + half * kCols;
          const bool first = j == 0 && hf == 0;
          const int sbar = kAlias ? 2 * g + hf : g;
          const uint32_t tSh = tS + hf * kSub;
          const int n_keep = seen - key0;
          const bool need_mask = __any_sync(0xffffffffu, n_keep < kCols);

          ok = ok && wait_or_abort(bar(S_FULL + sbar), gt & 1, abort_flag, a.status, 409);
          tc_fence_after_sync();
          float2 t[kCols / 2];
          {
            uint32_t raw[kCols];
#pragma unroll
            for (int c = 0; c < kCols / 32; ++c) tmem_ld32(tSh + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[c * 32]));
            tmem_wait_ld();
            if constexpr (!kAlias) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(S_FREE + g));
            }
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) t[i] = make_float2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
          }
          if (need_mask) {
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) {
              if (2 * i >= n_keep) t[i].x = -INFINITY;
              if (2 * i + 1 >= n_keep) t[i].y = -INFINITY;
            }
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kCols / 2; ++i) mx4[i & 3] = max3(mx4[i & 3], t[i].x, t[i].y);
          const float mx = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3]));
          const bool bump = mx > m + thr;
          float m_use = m;
          bool moved = bump;
          if constexpr (kHalves == 1) {
            m_use = bump ? mx : m;
          } else if ((moved = named_barrier_or(pair_bar, 64, bump))) {
            m_use = bump ? mx : m;
            if (half == 0) *xrow = m_use;
            named_barrier_sync(pair_bar, 64);
            if (half == 1) { m_use = fmaxf(m_use, *xrow); *xrow = m_use; }
            named_barrier_sync(pair_bar, 64);
            if (half == 0) m_use = *xrow;
          }
          const float alpha = m_use > m ? ex2((m - m_use) * mul) : 1.f;
          const float neg = m_use == -INFINITY ? 0.f : -m_use * mul;
          const float2 neg2 = make_float2(neg, neg);
          float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t pk[kCols / 2];
#pragma unroll
          for (int i = 0; i < kCols / 2; ++i) {
            const float2 x = __ffma2_rn(t[i], mul2, neg2);
            const float2 p = (kPoly > 0 && i % (kPoly > 0 ? kPoly : 1) == 0) ? ex2_poly2(x) : make_float2(ex2(x.x), ex2(x.y));
            sum2[i & 1] = __fadd2_rn(sum2[i & 1], p);
            pk[i] = pack2<kBf16>(p.x, p.y);
          }
          l = l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
          const bool rescale = !first && (kHalves == 1 || moved) && __any_sync(0xffffffffu, m_use > m);
          if constexpr (!kAlias) {
            if (j > 0) ok = ok && wait_or_abort(bar(PV_DONE + g), (gt - 1) & 1, abort_flag, a.status, 412);
            tc_fence_after_sync();
          } else if (rescale) {
            ok = ok && wait_or_abort(bar(PV_DONE + g), (2 * gt + hf - 1) & 1, abort_flag, a.status, 412);
            tc_fence_after_sync();
          }
          if (rescale) {
#pragma unroll
            for (int c = 0; c < kOutCols / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(tO + c * 32, o);
            }
          }
          tmem_st32(tP + (kAlias ? hf * kSub : 0), pk);
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(P_READY + sbar));
          m = m_use;
        }
      }

      // ---------------- epilogue: out = O / l, lse = m mul + log2 l ----------------
      uint8_t* const orow = static_cast<uint8_t*>(a.out) + 2 * (int64_t(row) * D + half * kOutCols);
      if (my_nt > 0) {
        if constexpr (kHalves == 2) {
          if (half == 0) *xrow = l;
          named_barrier_sync(pair_bar, 64);
          if (half == 1) { l += *xrow; *xrow = l; }
          named_barrier_sync(pair_bar, 64);
          if (half == 0) l = *xrow;
        }
        ok = ok && wait_or_abort(bar(O_DONE + g), oc & 1, abort_flag, a.status, 410);
        if (ok) {
          tc_fence_after_sync();
          const float inv = 1.f / l;
#pragma unroll
          for (int c = 0; c < kOutCols / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
            if (c == kOutCols / 32 - 1) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(O_FREE + g));
            }
            if (row >= 0) {
              uint4 w[4];
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint4& x = w[i >> 3];
                x.x = pack2<kBf16>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                x.y = pack2<kBf16>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                x.z = pack2<kBf16>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                x.w = pack2<kBf16>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
              }
              if (a.out_v8) {
                st_global_v8(orow + c * 64, w[0], w[1]);
                st_global_v8(orow + c * 64 + 32, w[2], w[3]);
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(orow + c * 64 + i * 16) = w[i];
              }
            }
          }
          if (half == 0 && row >= 0) a.lse[row] = m * mul + log2f(l);
        }
      }
      if (ok && seen <= 0 && row >= 0) {      // no key: zeros
        for (int i = 0; i < kOutCols / 8; ++i) reinterpret_cast<uint4*>(orow)[i] = make_uint4(0, 0, 0, 0);
        if (half == 0) a.lse[row] = -INFINITY;
      }
      tc += my_nt;
      oc += my_nt > 0 ? 1 : 0;
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) drain_after_abort();
  if (warp == 3) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool kBf16>
int launch_one(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, FwdArgs a, int64_t most, cudaStream_t st) {
  auto kernel = packed_fwd_tc_kernel<D, kBf16>;
  using L = FwdSmem<D>;
  constexpr int smem = L::kTotal + 1024;
  static_assert(smem <= 232448, "shared memory of a CTA");
  a.smem_bytes = smem;
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev < 0 || !ready[dev]) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess || attr.numRegs != Split<D>::kLaunchRegs) {
      set_error("packed_fwd_tc_kernel was built with %d registers per thread, expected %d", attr.numRegs, Split<D>::kLaunchRegs);
      return NB200_ERR_LAUNCH;
    }
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute(packed_fwd_tc_kernel, %d): %s", smem, cudaGetErrorString(e));
      return NB200_ERR_LAUNCH;
    }
    if (dev >= 0) ready[dev] = true;
  }
  const int sms = sm_count();
  // (set up while the list is being written)
  if (launch_dependent(kernel, unsigned(most < sms ? most : sms), Split<D>::kThreads, smem, st, tq, tk, tv, a) != cudaSuccess)
    return check_launch("packed_fwd_tc_kernel");
  count_launch();
  return check_launch("packed_fwd_tc_kernel");
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool strides_fit(const void* base, const int64_t (&s)[2], int tokens, int heads) {
  return aligned16(base) && (tokens <= 1 || (s[0] > 0 && s[0] % 8 == 0)) && (heads <= 1 || (s[1] > 0 && s[1] % 8 == 0));
}

}  // namespace

// A group's heads of one token have to fit a tile (64 rows in the backward).  With a scale below 1e-30, 8 / scale (the forward's
// threshold) and lse / scale (the backward's addend) come near the end of fp32.
bool tc_packed_supported(const PackedArgs& a, int dtype) {
  return dtype != NB200_F32 && (a.D == 64 || a.D == 128) && a.group <= 64 && a.scale > 1e-30f && a.scale < 1e30f &&
         int64_t(a.tokens_q) * a.heads <= 0x7fffffff && int64_t(a.tokens_k) * a.kv_heads <= 0x7fffffff && a.tokens_q > 0 && a.tokens_k > 0 && a.sequences > 0 && strides_fit(a.q, a.qs, a.tokens_q, a.heads) &&
         strides_fit(a.k, a.ks, a.tokens_k, a.kv_heads) && strides_fit(a.v, a.vs, a.tokens_k, a.kv_heads) && aligned16(a.out);
}

bool tc_packed_bwd_supported(const PackedArgs& a, int dtype) {
  return tc_packed_supported(a, dtype) && strides_fit(a.dout, a.dos, a.tokens_q, a.heads) && aligned16(a.dq) && aligned16(a.dk) &&
         aligned16(a.dv);
}

size_t tc_packed_fwd_bytes(const PackedArgs& a) {
  return work_list_bytes(most_blocks(a.tokens_q, a.sequences, 2 * tile_tokens(kTile, a.group)));
}

int tc_packed_fwd(const PackedArgs& p, int dtype, void* ws, cudaStream_t st) {
  FwdArgs a{};
  a.tokens = tile_tokens(kTile, p.group);
  if (int rc = launch_plan(p, false, 2 * a.tokens, 1, ws, st)) return rc;
  CUtensorMap tq, tk, tv;
  if (!make_token_map(&tq, p.q, p.tokens_q, p.heads, p.D, p.qs[0], p.qs[1], a.tokens, p.group) ||
      !make_token_map(&tk, p.k, p.tokens_k, p.kv_heads, p.D, p.ks[0], p.ks[1], kTile, 1) ||
      !make_token_map(&tv, p.v, p.tokens_k, p.kv_heads, p.D, p.vs[0], p.vs[1], kTile, 1)) {
    set_error("packed_fwd: a tensor map was rejected");
    return NB200_ERR_LAUNCH;
  }
  a.list.count = static_cast<const int*>(ws);
  a.list.taken = static_cast<int*>(ws) + 1;
  a.list.items = reinterpret_cast<const WorkItem*>(static_cast<const char*>(ws) + 16);
  a.kv_heads = p.kv_heads; a.group = p.group; a.heads = p.heads;
  a.group_magic = uint32_t((65536 + p.group - 1) / p.group);
  a.causal = p.causal;
  a.scale = p.scale;
  a.out = p.out;
  a.lse = p.lse;
  a.status = device_status_word();
  if (!a.status) { set_error("packed_fwd: no status word on this device"); return NB200_ERR_LAUNCH; }
  a.out_v8 = reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
  const int64_t most = most_blocks(p.tokens_q, p.sequences, 2 * a.tokens) * p.kv_heads;
  const bool bf16 = dtype == NB200_BF16;
  if (p.D == 64) return bf16 ? launch_one<64, true>(tq, tk, tv, a, most, st) : launch_one<64, false>(tq, tk, tv, a, most, st);
  return bf16 ? launch_one<128, true>(tq, tk, tv, a, most, st) : launch_one<128, false>(tq, tk, tv, a, most, st);
}

}  // namespace packed
}  // namespace nb200
