// Backward of attention over packed sequences for sm_100a in ONE kernel: dq, dk and dv with S and dP computed once per tile
// pair; bf16 and fp16, head dim 64 and 128, any group of up to 64 query heads per key head.
//
//   P = exp2(S scale log2 e - lse), dV = P^T dO, dS = P (dO V^T - delta), dK = scale dS^T Q, dQ = scale dS K
//
// A CTA owns 128 keys of one sequence and key head and streams the sequence's rows -- token after token, the query heads of
// that key head -- in steps of 64 / G tokens, which fill 64 rows (some stay unused where G is no divisor).  dK and dV are sums
// over the rows, so that the sum over a group's heads costs nothing; dQ of a step goes to fp32 sums in global memory by
// 16-byte reductions, which is the one place where the order of a sum is not fixed.  The scheme of a step -- two issuing
// warps, two element-wise groups on alternate steps, lse and delta added by a K = 16 MMA step, dQ^T with d on the TMEM lanes --
// is that of sdpa_tc_bwd_d128.cu, which has the reasons and the measurements.  One thing is different: dS goes to TMEM as well,
// as the A operand of dK, which takes an eighth off what the MMAs read from shared memory (head dim 128: 4 % of the time).  At head
// dim 64 the tile of dQ^T has 128 lanes as well, of which the upper 64 (V in place of K: the tiles lie one after the other) are not
// read.
//
// P and dS are rounded to the operand type where they become operands (dS from the unrounded P); sums, lse and delta are fp32.
//
// What belongs to a neighbouring sequence must not get into a sum, not even as 0 * NaN: keys behind the end have P and dS
// selected to zero and their rows of K cleared in shared memory, queries behind the end have P and dS selected to zero and
// their rows of Q and dO cleared, as have queries that see no key.  Warp 3, which forms the addends of every step before its
// products may run, does that.
// Head dim 128: bound by the operands that the MMAs read from shared memory (about 1900 of a step's 2700 cycles) and by the sums
// of dq in L2 (without them, for timing: 744 -> 551 us when it was 744); 8192 tokens, 16 heads on 4, causal 720 to 731 us one at a
// time, 775 in a long loop under the power cap (fp16 743, 815).  Head dim 64: by the chain of a step; 518 to 524 us (fp16 528); two
// steps' products in TMEM took 522 to 508, two dS tiles as well 551.  All waits bounded.
#include <math.h>

#include <type_traits>

#include "dependent_launch.cuh"
#include "packed_tc.cuh"

namespace nb200 {
namespace packed {

using namespace sm100;
using namespace tc;

namespace {

constexpr int kThreads = 384;
constexpr int kStep = 64;                     // rows per step
constexpr int kYBoxBytes = kStep * 128;       // one 64-row x 128-byte box
constexpr int kProducerRegs = 88;
constexpr int kWorkerRegs = 208;
constexpr int kLaunchRegs = 168;              // what __launch_bounds__(384, 1) gives
static_assert((kLaunchRegs - kProducerRegs) * 128 >= (kWorkerRegs - kLaunchRegs) * 256,
              "worker warps would wait forever for registers the producer warps never release");

struct BwdArgs {
  WorkList list;
  int kv_heads, group, heads;
  int tokens;                // query tokens of a step
  int causal;
  float scale;
  const float* lse;          // (tokens_q, heads)
  const float* delta;
  float* dq_acc;             // [key head][step][row / 4][d][row % 4]
  int64_t all_steps;         // steps that the accumulator has room for, per key head
  const float* largest;      // fp16: what SequenceMost says, for every sequence
  void* dk;                  // dense (tokens_k, kv_heads, D)
  void* dv;
  int* status;
};

// fp16 has few exponents: with thousands of keys P and dS lie where it loses its digits.  P is taken times 2^10 (at most 1024), dS
// times the power of two that its bound allows: |dS| <= |dout row| |v row| + |delta| <= 2 max |dout row| max |v row|, since a row of
// out is a mean of rows of v.  Both factors leave with the results.  (Relative error of dq and dk over sequences of thousands of
// tokens: 4.1e-4 without, 3.1e-4 with them; the rounding of dS and that of the results are 2.1e-4 each.)  The bound is taken for each
// sequence by itself, over its queries that see a key: what stands elsewhere must not cost its gradients their digits.
__device__ __forceinline__ int ds_shift(const float* largest, int sequence) {
  const float bound = 2.f * sqrtf(largest[kMosts * sequence + kMostDout]) * sqrtf(largest[kMosts * sequence + kMostV]);
  if (!(bound < INFINITY)) return 0;
  const float room = floorf(log2f(60000.f / fmaxf(bound, 1e-30f)));
  return int(fminf(fmaxf(room, -14.f), 14.f));
}
// In a sequence with an addend that its fp16 numbers do not hold (scores or sums of out * dout of kRowAddendMost before the scale, or a
// scale below 1e-8) the addends of the MMA are zeros, and the element-wise warps take lse and delta off in fp32.

template <int D>
struct Smem {
  static constexpr int kXBytes = kTile * D * 2;                 // K or V tile
  static constexpr int kYBytes = kStep * D * 2;                 // Q or dO of a step
  static constexpr int kYStages = D == 64 ? 6 : 4;
  static constexpr int kYStageBytes = 2 * kYBytes;
  static constexpr int kX = 0;
  static constexpr int kY = kX + 2 * kXBytes;
  static constexpr int kDs = kY + kYStages * kYStageBytes;
  static constexpr int kWeightBytes = (kTile / 8) * 256;
  static constexpr int kAugTileBytes = (kStep / 8) * 256;
  static constexpr int kAugSlotBytes = 2 * kAugTileBytes;       // lse tile, delta tile
  static constexpr int kWeights = kDs + kBoxBytes;
  static constexpr int kAug = kWeights + kWeightBytes;          // two slots
  static constexpr int kBars = kAug + 2 * kAugSlotBytes;
  static constexpr int kNumBars = 26 + 2 * kYStages;
  static constexpr int kMisc = kBars + 8 * kNumBars;
  static constexpr int kTotal = kMisc + 16;
  static_assert(kY % 1024 == 0 && kDs % 1024 == 0, "swizzled tiles need 1024-byte alignment");
  static_assert(kTotal + 1024 <= 232448, "shared memory exceeds the per-CTA limit");
};

// Clears the rows of a step's Q and dO that lie outside [first, end), of `rows`; for a warp.  Out of line: few steps need it, and inside
// the loop of warp 3, which every step waits for, it costs all of them (8192 tokens, 16 heads on 4, causal: head dim 64 564 us for 518,
// 128 716 for 720).
template <int D>
__device__ __noinline__ void keep_rows(uint32_t stage, int first, int end, int rows) {
  for (int i = threadIdx.x & 31; i < rows * 8 * (2 * (D / 64)); i += 32) {
    const int box = i / (rows * 8), rem = i - box * (rows * 8);
    if (rem < first * 8 || rem >= end * 8) st_shared_v4(stage + box * kYBoxBytes + rem * 16, make_uint4(0, 0, 0, 0));
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
packed_bwd_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do, const BwdArgs a) {
  using L = Smem<D>;
  constexpr int NY = L::kYStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  constexpr int X_FULL = 0, Y_FULL = 1, Y_EMPTY = Y_FULL + NY, PROD_FULL = Y_EMPTY + NY, P_FREE = PROD_FULL + 4,
                E_READY = P_FREE + 4, E_FREE = E_READY + 2, DS_FREE = E_FREE + 2, DQ_FULL = DS_FREE + 2, DQ_FREE = DQ_FULL + 2,
                AUG_FULL = DQ_FREE + 2, AUG_FREE = AUG_FULL + 2, ACC_DONE = AUG_FREE + 2, P_READY = ACC_DONE + 1;
  static_assert(P_READY + 2 == L::kNumBars, "barrier count");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  wait_for_previous();       // the work list and delta are written by the launches before
  const int entry = blockIdx.x / a.kv_heads, head = blockIdx.x - entry * a.kv_heads;
  if (entry >= *reinterpret_cast<const volatile int*>(a.list.count)) return;
  const WorkItem it = load_item(a.list.items + entry);
  const int live_rows = a.tokens * a.group;                // rows of a step that hold a token
  const int s_begin = a.causal ? min(max(it.seen, 0), it.other_n) / a.tokens : 0, s_end = (it.other_n + a.tokens - 1) / a.tokens;
  const int n_steps = max(s_end - s_begin, 0);
  const bool wide = !kBf16 && !(a.largest[kMosts * it.sequence + kMostOfAddends] < kRowAddendMost);
  // The CTAs of one sequence and key head read the same rows and add into the same sums.  They walk from the sequence's end to
  // its front (and wrap around), each one step behind its neighbour: near enough to find the rows in L2, and not on the same
  // lines at the same moment.
  const int rot = n_steps > 0 ? int((uint32_t(it.index)) % uint32_t(n_steps)) : 0;
  auto step_of = [&](int n) {   // the n-th step this CTA visits, counted within the sequence
    int j = n + rot;
    if (j >= n_steps) j -= n_steps;
    return s_end - 1 - j;
  };

  if (threadIdx.x < L::kNumBars) {
    const int i = threadIdx.x;
    uint32_t count = 1;
    if (i >= P_FREE && i < P_FREE + 4) count = 4;      // one lane per warp of the group
    if (i >= E_READY && i < E_READY + 2) count = 4;
    if (i >= P_READY && i < P_READY + 2) count = 4;
    if (i >= DQ_FREE && i < DQ_FREE + 2) count = 4;
    mbar_init(bar(i), count);
    if (i == 0) *abort_flag = 0;
    mbar_init_fence();
  }
  __syncwarp();
  static_assert(L::kNumBars <= 64, "barrier initialisation assumes the first two warps cover all barriers");
  if (threadIdx.x < 64) asm volatile("bar.sync 1, 64;" ::: "memory");
  const uint32_t y_bytes = uint32_t(live_rows) * (D * 2);
  auto load_step = [&](int n) {       // into stage n % NY
    const int st = n % NY, token = it.other + step_of(n) * a.tokens;
    const uint32_t ybase = sbase + L::kY + st * L::kYStageBytes;
    mbar_expect_tx(bar(Y_FULL + st), 2 * y_bytes);
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
      tma_load_4d(ybase + x * kYBoxBytes, &tm_q, bar(Y_FULL + st), x * 64, head * a.group, token, 0);
      tma_load_4d(ybase + L::kYBytes + x * kYBoxBytes, &tm_do, bar(Y_FULL + st), x * 64, head * a.group, token, 0);
    }
  };
  if (threadIdx.x == 0 && n_steps > 0) {
    // the CTA's own tiles and the first ring stages: their latency runs under the rest of the start-up
    mbar_expect_tx(bar(X_FULL), 2 * L::kXBytes);
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
      tma_load_4d(sbase + L::kX + x * kBoxBytes, &tm_k, bar(X_FULL), x * 64, head, it.begin, 0);
      tma_load_4d(sbase + L::kX + L::kXBytes + x * kBoxBytes, &tm_v, bar(X_FULL), x * 64, head, it.begin, 0);
    }
    for (int n = 0; n < min(n_steps, NY); ++n) load_step(n);
  }
  {
    uint4* wt = reinterpret_cast<uint4*>(smem + L::kWeights);
    for (int idx = threadIdx.x; idx < L::kWeightBytes / 16; idx += kThreads)
      wt[idx] = (idx & 8) ? make_uint4(0, 0, 0, 0) : row_addend_weights<kBf16>();
    uint4* aug = reinterpret_cast<uint4*>(smem + L::kAug);
    for (int idx = threadIdx.x; idx < 2 * L::kAugSlotBytes / 16; idx += kThreads) aug[idx] = make_uint4(0, 0, 0, 0);
    // rows of the ring that no load fills (the group is no divisor of 64)
    const int words = (kStep - live_rows) * 8;
    for (int i = threadIdx.x; i < words * (NY * 2 * (D / 64)); i += kThreads) {
      const int box = i / words, rem = i - box * words;
      st_shared_v4(sbase + L::kY + box * kYBoxBytes + live_rows * 128 + rem * 16, make_uint4(0, 0, 0, 0));
    }
    fence_proxy_async_smem();   // written by threads, read by the tensor core
  }
  if (warp == 3) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // TMEM: dV, dK, the products P1 and P2 (at head dim 64 there is room for those of two steps), p and ds, dQ^T
  constexpr int kProds = D == 64 ? 2 : 1;
  const uint32_t tm_dv = tmem, tm_dk = tmem + D, tm_e = tmem + 384, tm_dq = tmem + 448;
  auto tm_p1 = [&](int n) { return tmem + 2 * D + (n & (kProds - 1)) * 64; };
  auto tm_p2 = [&](int n) { return tmem + 2 * D + kProds * 64 + (n & (kProds - 1)) * 64; };

  if (warp < 4) {
  reg_dealloc<kProducerRegs>();
  if (warp == 1) {
    // ---------------- Q / dO ring ----------------
    if (elect_one()) {
      for (int n = NY; n < n_steps; ++n) {
        if (!wait_or_abort(bar(Y_EMPTY + n % NY), ((n / NY) & 1) ^ 1, abort_flag, a.status, 502)) break;
        load_step(n);
      }
    }
  } else if (warp == 2) {
    // ---------------- MMA issuer 1: the products of every step ----------------
    if (elect_one() && n_steps > 0) {
      constexpr uint32_t idesc_prod = make_idesc(kBf16, kTile, kStep, false, false);
      bool ok = wait_or_abort(bar(X_FULL), 0, abort_flag, a.status, 503);
      const uint64_t kdesc = make_smem_desc(sbase + L::kX, 16, 1024);
      const uint64_t vdesc = make_smem_desc(sbase + L::kX + L::kXBytes, 16, 1024);
      const uint64_t wdesc = make_smem_desc_noswizzle(sbase + L::kWeights, 128, 256);
      for (int n = 0; n < n_steps && ok; ++n) {
        const int st = n % NY, s = n & 1;
        ok = wait_or_abort(bar(Y_FULL + st), (n / NY) & 1, abort_flag, a.status, 504);
        // a product may be overwritten once the warps of the step before on its columns hold it in registers
        if (ok && n >= kProds) ok = wait_or_abort(bar(P_FREE + ((n - kProds) & 1)), ((n - kProds) >> 1) & 1, abort_flag, a.status, 509);
        if (ok) ok = wait_or_abort(bar(AUG_FULL + s), (n >> 1) & 1, abort_flag, a.status, 512);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t ybase = sbase + L::kY + st * L::kYStageBytes;
        const uint64_t qdesc = make_smem_desc(ybase, 16, 1024), gdesc = make_smem_desc(ybase + L::kYBytes, 16, 1024);
        const uint32_t aslot = sbase + L::kAug + s * L::kAugSlotBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t xo = uint64_t(((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4);
          const uint64_t yo = uint64_t(((kk / 4) * kYBoxBytes + (kk % 4) * 32) >> 4);
          mma_ss(tm_p1(n), kdesc + xo, qdesc + yo, idesc_prod, kk > 0 ? 1u : 0u);
        }
        // P1 += W C1^T (C1: -lse / (scale log2e))
        mma_ss(tm_p1(n), wdesc, make_smem_desc_noswizzle(aslot, 128, 256), idesc_prod, 1u);
        mma_commit(bar(PROD_FULL + s));
        if (n >= kProds) ok = wait_or_abort(bar(P_FREE + 2 + ((n - kProds) & 1)), ((n - kProds) >> 1) & 1, abort_flag, a.status, 519);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t xo = uint64_t(((kk / 4) * kBoxBytes + (kk % 4) * 32) >> 4);
          const uint64_t yo = uint64_t(((kk / 4) * kYBoxBytes + (kk % 4) * 32) >> 4);
          mma_ss(tm_p2(n), vdesc + xo, gdesc + yo, idesc_prod, kk > 0 ? 1u : 0u);
        }
        // P2 += W C2^T (C2: -delta)
        mma_ss(tm_p2(n), wdesc, make_smem_desc_noswizzle(aslot + L::kAugTileBytes, 128, 256), idesc_prod, 1u);
        mma_commit(bar(AUG_FREE + s));
        mma_commit(bar(PROD_FULL + 2 + s));
      }
    }
  } else if (warp == 0) {
    // ---------------- MMA issuer 2: dV, dK and dQ^T of every step ----------------
    if (elect_one() && n_steps > 0) {
      constexpr uint32_t idesc_acc = make_idesc(kBf16, kTile, D, false, true);      // dV, dK: A (p, ds) from TMEM, B (dO, Q) MN-major
      constexpr uint32_t idesc_dq = make_idesc(kBf16, kTile, kStep, true, true);    // dQ^T: A = K MN-major, B = ds MN-major
      bool ok = wait_or_abort(bar(X_FULL), 0, abort_flag, a.status, 503);
      const uint64_t kmn = make_smem_desc(sbase + L::kX, kBoxBytes, 1024);          // K as [d x key], d contiguous
      const uint32_t dsbuf = sbase + L::kDs;
      const uint64_t ds_b = make_smem_desc(dsbuf, kBoxBytes, 1024);
      for (int m = 0; m < n_steps && ok; ++m) {
        const int st = m % NY, s = m & 1;
        const uint32_t ybase = sbase + L::kY + st * L::kYStageBytes;
        const uint64_t qmn = make_smem_desc(ybase, kYBoxBytes, 1024);                    // Q as [query x d], d contiguous
        const uint64_t gmn = make_smem_desc(ybase + L::kYBytes, kYBoxBytes, 1024);      // dO likewise
        const uint32_t e1 = tm_e, e2 = tm_e + 32;      // p, ds
        // dV += p^T dO as soon as p is there: it runs while the warps still form ds
        ok = wait_or_abort(bar(P_READY + s), (m >> 1) & 1, abort_flag, a.status, 519);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk)
          mma_ts(tm_dv, e1 + kk * 8, gmn + uint64_t((kk * 2048) >> 4), idesc_acc, (m > 0 || kk > 0) ? 1u : 0u);
        mma_commit(bar(E_FREE + s));             // p of this stage may be rewritten
        // dK += ds^T Q once the ds tile is in shared memory
        ok = wait_or_abort(bar(E_READY + s), (m >> 1) & 1, abort_flag, a.status, 505);
        if (!ok) break;
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk)
          mma_ts(tm_dk, e2 + kk * 8, qmn + uint64_t((kk * 2048) >> 4), idesc_acc, (m > 0 || kk > 0) ? 1u : 0u);
        mma_commit(bar(Y_EMPTY + st));           // the last readers of this Q / dO stage
        // dQ^T[d, row] = sum_key K[key, d] ds[key, row]; the previous tile must have been drained
        if (m >= 1) {
          ok = wait_or_abort(bar(DQ_FREE + ((m - 1) & 1)), ((m - 1) >> 1) & 1, abort_flag, a.status, 515);
          if (!ok) break;
          tc_fence_after_sync();
        }
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk)
          mma_ss(tm_dq, kmn + uint64_t((kk * 2048) >> 4), ds_b + uint64_t((kk * 2048) >> 4), idesc_dq, kk > 0 ? 1u : 0u);
        mma_commit(bar(DQ_FULL + (m & 1)));
        mma_commit(bar(DS_FREE + (m & 1)));      // the ds tile has been read by dK and dQ^T
        if (m == n_steps - 1) mma_commit(bar(ACC_DONE));
      }
    }
  } else {
    // ---------------- warp 3: the addends of every row as MMA operands, rows of other sequences cleared ----------------
    const float inv_mul = 1.f / (a.scale * kLog2e);
    // the sequence's first queries, which see no key; only its first block of keys comes near them
    const int blind = a.causal && it.index == 0 ? max(it.seen, 0) : 0;
    bool ok = true;
    // lse and delta of rows lane and lane + 32 of a step, fetched a step ahead; rows without a token or a key: zeros (P and
    // dS are selected there, the addends have to be finite)
    float next[2][2];
    auto fetch = [&](int n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = lane + 32 * e, t = row / a.group, token = step_of(n) * a.tokens + t;
        next[e][0] = next[e][1] = 0.f;
        if (row < live_rows && token < it.other_n) {
          const int64_t at = (int64_t(it.other) + token) * a.heads + head * a.group + (row - t * a.group);
          next[e][0] = a.lse[at];
          next[e][1] = a.delta[at];
        }
      }
    };
    if (n_steps > 0) fetch(0);
    for (int n = 0; n < n_steps && ok; ++n) {
      const int st = n % NY, s = n & 1;
      float c[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool keyless = next[e][0] == -INFINITY;
        c[e][0] = keyless || wide ? 0.f : -(next[e][0] - (kBf16 ? 0.f : float(kPShift))) * inv_mul;
        c[e][1] = keyless || wide ? 0.f : -next[e][1];
      }
      if (n + 1 < n_steps) fetch(n + 1);
      ok = wait_or_abort(bar(Y_FULL + st), (n / NY) & 1, abort_flag, a.status, 513);
      if (ok && n >= 2) ok = wait_or_abort(bar(AUG_FREE + s), ((n - 2) >> 1) & 1, abort_flag, a.status, 514);
      if (ok && n == 0) ok = wait_or_abort(bar(X_FULL), 0, abort_flag, a.status, 503);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (n == 0 && it.n < kTile) {
        const int words = (kTile - it.n) * 8;      // of a box of K
        for (int i = lane; i < words * (D / 64); i += 32) {
          const int box = i / words, rem = i - box * words;
          st_shared_v4(sbase + L::kX + box * kBoxBytes + it.n * 128 + rem * 16, make_uint4(0, 0, 0, 0));
        }
      }
      const int token0 = step_of(n) * a.tokens, end = min(it.other_n - token0, a.tokens) * a.group;      // end: of this sequence's rows
      if (end < live_rows || token0 < blind)
        keep_rows<D>(sbase + L::kY + st * L::kYStageBytes, min(max(blind - token0, 0), a.tokens) * a.group, end, live_rows);
      uint8_t* slot = smem + L::kAug + s * L::kAugSlotBytes;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int q = lane + 32 * e;
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          *reinterpret_cast<uint4*>(slot + tile * L::kAugTileBytes + (q >> 3) * 256 + (q & 7) * 16) = row_addend<kBf16>(c[e][tile]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(AUG_FULL + s));
    }
  }
  } else {
    reg_alloc<kWorkerRegs>();
    // ---------------- element-wise groups (one key per thread) ----------------
    const int grp = (warp - 4) >> 2;
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lane_addr = uint32_t(wq * 32) << 16;
    bool ok = true;
    const float mul = a.scale * kLog2e;
    const float2 mul2 = make_float2(mul, mul);
    const int shift = kBf16 ? 0 : ds_shift(a.largest, it.sequence);
    const float ds_mul = kBf16 ? 1.f : exp2f(float(shift - kPShift));      // (P is 2^10 times itself)
    const float2 ds_mul2 = make_float2(ds_mul, ds_mul);
    const bool dropped = r >= it.n;
    const int first_query = it.seen + r;      // that sees this key, counted within the sequence (causal)
    // The ds tile (16 KB, 128-byte swizzle) is [128 keys x 64 rows]: a thread writes its own 128-byte row as eight 16-byte
    // chunks, chunk i at position i ^ (r % 8).
    const uint32_t ds_thread = sbase + L::kDs + uint32_t(r) * 128 + (uint32_t(r & 7) << 4);
    float* const acc = a.dq_acc + (int64_t(head) * a.all_steps + it.steps) * (kStep * D) + r * 4;

    // wide: lse or delta of rows lane and lane + 32 of a step
    auto statistic = [&](const float* x, int n, float (&own)[2]) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = lane + 32 * e, t = row / a.group, token = step_of(n) * a.tokens + t;
        const bool in = row < live_rows && token < it.other_n;
        own[e] = in ? x[(int64_t(it.other) + token) * a.heads + head * a.group + (row - t * a.group)] : 0.f;
      }
    };

    // dQ^T of step j to the sums: [row / 4][d][row % 4] floats, so that a warp's reduction of four rows covers 512 bytes
    auto drain = [&](int j) -> bool {
      if (!wait_or_abort(bar(DQ_FULL + (j & 1)), (j >> 1) & 1, abort_flag, a.status, 516)) return false;
      tc_fence_after_sync();
      if (D == 128 || wq < 2) {      // (uniform over the warp)
        uint32_t v[kStep];
        tmem_ld32(tm_dq + lane_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(tm_dq + lane_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(DQ_FREE + (j & 1)));
        float* dst = acc + int64_t(step_of(j)) * (kStep * D);
#pragma unroll
        for (int c = 0; c < kStep / 4; ++c) red_add_v4(dst + c * (D * 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      } else if (lane == 0) {
        mbar_arrive(bar(DQ_FREE + (j & 1)));
      }
      return true;
    };

    // (a loop of its own for `wide`: as conditions inside one they cost the usual case 5 %)
    auto walk = [&](auto is_wide) {
    constexpr bool kWide = decltype(is_wide)::value;
    for (int n = grp; n < n_steps && ok; n += 2) {
      const int s = n & 1;
      // keep bits over the step's rows: row c needs a token of the sequence and (causal) one that sees the key
      uint32_t keep[2];
      {
        const int t0 = step_of(n) * a.tokens;
        const int hi = min(it.other_n - t0, a.tokens) * a.group;
        const int lo = a.causal ? min(max(first_query - t0, 0), kStep) * a.group : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int nh = hi - 32 * i, nl = lo - 32 * i;
          const uint32_t mh = nh >= 32 ? 0xffffffffu : (nh <= 0 ? 0u : ((1u << nh) - 1u));
          const uint32_t ml = nl <= 0 ? 0xffffffffu : (nl >= 32 ? 0u : ~((1u << nl) - 1u));
          keep[i] = dropped ? 0u : mh & ml;
        }
      }
      const bool need_mask = __any_sync(0xffffffffu, (keep[0] & keep[1]) != 0xffffffffu);

      ok = wait_or_abort(bar(PROD_FULL + s), (n >> 1) & 1, abort_flag, a.status, 506);
      if (!ok) break;
      tc_fence_after_sync();
      // the scores first: p = exp2(t log2e) (they arrive with -lse already added) while dP is still being computed
      float2 t[kStep / 2];
      {
        uint32_t raw[kStep];
        tmem_ld32(tm_p1(n) + lane_addr, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
        tmem_ld32(tm_p1(n) + lane_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FREE + s));
#pragma unroll
        for (int i = 0; i < kStep / 2; ++i) t[i] = make_float2(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
      }
      if constexpr (kWide) {
        // (p is 1 at most, where lse is so large that its own rounding would say otherwise)
        float lse[2];
        statistic(a.lse, n, lse);
        auto exponent = [&](float x, int row) {
          const float y = fmaf(x, mul, float(kPShift) - __shfl_sync(0xffffffffu, lse[row >> 5], row & 31));
          return y > float(kPShift) ? float(kPShift) : y;
        };
#pragma unroll
        for (int i = 0; i < kStep / 2; ++i) t[i] = make_float2(exponent(t[i].x, 2 * i), exponent(t[i].y, 2 * i + 1));
      }
      uint32_t e1[kStep / 2], e2[kStep / 2];
#pragma unroll
      for (int c = 0; c < kStep / 2; ++c) {
        float2 x = kWide ? t[c] : __fmul2_rn(t[c], mul2);
        if (need_mask) {
          if (!((keep[c >> 4] >> ((2 * c) & 31)) & 1u)) x.x = -INFINITY;
          if (!((keep[c >> 4] >> ((2 * c + 1) & 31)) & 1u)) x.y = -INFINITY;
        }
        t[c] = make_float2(ex2(x.x), ex2(x.y));
        e1[c] = pack2<kBf16>(t[c].x, t[c].y);
      }
      // p is still being read by dV of step n - 1
      if (n >= 1) {
        ok = wait_or_abort(bar(E_FREE + ((n - 1) & 1)), ((n - 1) >> 1) & 1, abort_flag, a.status, 510);
        if (!ok) break;
        tc_fence_after_sync();
      }
      tmem_st32(tm_e + lane_addr, e1);
      // ds = p dP (dP arrives with -delta already added)
      ok = wait_or_abort(bar(PROD_FULL + 2 + s), (n >> 1) & 1, abort_flag, a.status, 518);
      if (!ok) break;
      // p is in TMEM by now: dV += p^T dO may start while ds is formed
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(P_READY + s));
      tc_fence_after_sync();
      {
        uint32_t raw[kStep];
        tmem_ld32(tm_p2(n) + lane_addr, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
        tmem_ld32(tm_p2(n) + lane_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FREE + 2 + s));
        if constexpr (kWide) {
          float delta[2];
          statistic(a.delta, n, delta);
#pragma unroll
          for (int c = 0; c < kStep; ++c) raw[c] = __float_as_uint(__uint_as_float(raw[c]) - __shfl_sync(0xffffffffu, delta[c >> 5], c & 31));
        }
        if (need_mask) {
          // (a dropped key's row of V, or a masked score's dP, may be anything)
#pragma unroll
          for (int c = 0; c < kStep; ++c)
            if (!((keep[c >> 5] >> (c & 31)) & 1u)) raw[c] = 0u;
        }
#pragma unroll
        for (int c = 0; c < kStep / 2; ++c) {
          float2 ds = __fmul2_rn(t[c], make_float2(__uint_as_float(raw[2 * c]), __uint_as_float(raw[2 * c + 1])));
          if constexpr (!kBf16) ds = __fmul2_rn(ds, ds_mul2);
          e2[c] = pack2<kBf16>(ds.x, ds.y);
        }
      }
      // ds, in TMEM for dK and in shared memory for dQ, was last read by the MMAs of step n - 1
      if (n >= 1) {
        ok = wait_or_abort(bar(DS_FREE + ((n - 1) & 1)), ((n - 1) >> 1) & 1, abort_flag, a.status, 517);
        if (!ok) break;
        tc_fence_after_sync();
      }
      tmem_st32(tm_e + 32 + lane_addr, e2);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        st_shared_v4(ds_thread ^ (uint32_t(i) << 4), make_uint4(e2[4 * i], e2[4 * i + 1], e2[4 * i + 2], e2[4 * i + 3]));
      fence_proxy_async_smem();
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(E_READY + s));
      // dQ^T of the previous step (the other group's) is complete by now: add it to the sums
      if (n >= 1) ok = drain(n - 1);
    }
    };
    if constexpr (kBf16) {
      walk(std::false_type());
    } else {
      if (wide) walk(std::true_type());
      else walk(std::false_type());
    }
    // the last step's dQ^T is drained by the group that did not produce it
    if (ok && n_steps > 0 && grp == (n_steps & 1)) ok = drain(n_steps - 1);

    // ---------------- epilogue: group 0 writes dv, group 1 writes dk * scale ----------------
    if (ok && n_steps > 0) ok = wait_or_abort(bar(ACC_DONE), 0, abort_flag, a.status, 508);
    if (ok) {
      tc_fence_after_sync();
      const uint32_t tacc = (grp == 0 ? tm_dv : tm_dk) + lane_addr;
      const float omul = kBf16 ? (grp == 0 ? 1.f : a.scale) : grp == 0 ? exp2f(-float(kPShift)) : a.scale * exp2f(-float(shift));
      uint8_t* orow = static_cast<uint8_t*>(grp == 0 ? a.dv : a.dk) + 2 * ((int64_t(it.begin) + r) * a.kv_heads + head) * D;
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n_steps > 0) {
          tmem_ld32(tacc + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (!dropped) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            w.x = pack2<kBf16>(__uint_as_float(o[i]) * omul, __uint_as_float(o[i + 1]) * omul);
            w.y = pack2<kBf16>(__uint_as_float(o[i + 2]) * omul, __uint_as_float(o[i + 3]) * omul);
            w.z = pack2<kBf16>(__uint_as_float(o[i + 4]) * omul, __uint_as_float(o[i + 5]) * omul);
            w.w = pack2<kBf16>(__uint_as_float(o[i + 6]) * omul, __uint_as_float(o[i + 7]) * omul);
            *reinterpret_cast<uint4*>(orow + (c * 32 + i) * 2) = w;
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) drain_after_abort();
  if (warp == 3) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// delta[token][head] = sum_d out dout in fp32.  Bound by HBM: D / 8 lanes per row with 16 bytes of each tensor, four rows per
// lane whose loads are in flight together.  fp16: also the squared norms of the rows of dout, and, by the CTAs behind `delta_ctas`,
// of those of v; the launch that lists the blocks has their maxima.
constexpr int kDeltaThreads = 256, kDeltaRows = 4;

template <int D, bool kBf16>
__global__ void __launch_bounds__(kDeltaThreads) packed_delta_tc_kernel(const PackedArgs a, int delta_ctas) {
  constexpr int kLanes = D / 8, kGroups = kDeltaThreads / kLanes;
  const bool values = !kBf16 && int(blockIdx.x) >= delta_ctas;
  const int heads = values ? a.kv_heads : a.heads, rows = values ? a.tokens_k * a.kv_heads : a.tokens_q * a.heads;      // (below 2^31: checked on the host)
  const int row0 = (int(blockIdx.x) - (values ? delta_ctas : 0)) * (kGroups * kDeltaRows) + int(threadIdx.x) / kLanes, c = threadIdx.x % kLanes;
  uint4 o[kDeltaRows], g[kDeltaRows];
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const int row = row0 + i * kGroups;
    o[i] = g[i] = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      const int token = row / heads, head = row - token * heads;
      const int64_t at = values ? token * a.vs[0] + head * a.vs[1] : token * a.dos[0] + head * a.dos[1];
      if (!values) o[i] = ldg_no_allocate(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.out) + int64_t(row) * D) + c);
      g[i] = ldg_no_allocate(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(values ? a.v : a.dout) + at) + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const uint32_t ow[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, gw[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
    float sum = 0.f, squares = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = unpack2<kBf16>(ow[j]), y = unpack2<kBf16>(gw[j]);
      sum = fmaf(x.x, y.x, fmaf(x.y, y.y, sum));
      if constexpr (!kBf16) squares = fmaf(y.x, y.x, fmaf(y.y, y.y, squares));
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if constexpr (!kBf16) squares += __shfl_xor_sync(0xffffffffu, squares, off);
    }
    const int row = row0 + i * kGroups;
    if (!values && row < rows && c == 0) a.delta[row] = sum;
    if (!kBf16 && row < rows && c == 0) a.squares[(values ? int64_t(a.tokens_q) * a.heads : 0) + row] = squares;
  }
}

// dq = scale * (fp32 sums) in the operand type: one CTA per step and key head; a thread takes four rows x eight d (eight
// 16-byte loads, four 16-byte stores).
template <int D, bool kBf16>
__global__ void __launch_bounds__(kStep / 4 * (D / 8)) packed_dq_finish_kernel(const PackedArgs a, const float* __restrict__ acc,
                                                                                int64_t all_steps, int tokens, const float* largest) {
  const int head = blockIdx.y, dchunk = threadIdx.x % (D / 8), rg = threadIdx.x / (D / 8);
  const float* src = acc + (int64_t(head) * all_steps + blockIdx.x) * (kStep * D) + rg * (D * 4) + dchunk * 32;
  float4 v[8];      // in flight while the step's sequence is looked for
#pragma unroll
  for (int d = 0; d < 8; ++d) v[d] = __ldcs(reinterpret_cast<const float4*>(src) + d);
  const Place place = find_place(int(blockIdx.x), a.sequences, [&](int i) { return (sequence_span(a.offsets_q, i, a.tokens_q).y + tokens - 1) / tokens; });
  if (place.index < 0) return;
  const int2 q = sequence_span(a.offsets_q, place.sequence, a.tokens_q);
  const float scale = kBf16 ? a.scale : a.scale * exp2f(-float(ds_shift(largest, place.sequence)));
#pragma unroll
  for (int rr = 0; rr < 4; ++rr) {
    const int row = rg * 4 + rr, t = row / a.group, token = place.index * tokens + t;
    if (t >= tokens || token >= q.y) break;
    float x[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) x[d] = (rr == 0 ? v[d].x : rr == 1 ? v[d].y : rr == 2 ? v[d].z : v[d].w) * scale;
    uint4 w;
    w.x = pack2<kBf16>(x[0], x[1]);
    w.y = pack2<kBf16>(x[2], x[3]);
    w.z = pack2<kBf16>(x[4], x[5]);
    w.w = pack2<kBf16>(x[6], x[7]);
    const int64_t at = (int64_t(q.x) + token) * a.heads + head * a.group + (row - t * a.group);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dq) + at * D + dchunk * 8) = w;
  }
}

int64_t most_steps(const PackedArgs& a) { return most_blocks(a.tokens_q, a.sequences, tile_tokens(kStep, a.group)); }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t delta_bytes(const PackedArgs& a) { return up256(size_t(a.tokens_q) * a.heads * sizeof(float)); }
size_t squares_bytes(const PackedArgs& a, bool bf16) {
  return bf16 ? 0 : up256((size_t(a.tokens_q) * a.heads + size_t(a.tokens_k) * a.kv_heads) * sizeof(float));
}
size_t list_bytes(const PackedArgs& a) { return work_list_bytes(most_blocks(a.tokens_k, a.sequences, kTile)); }
size_t largest_bytes(const PackedArgs& a, bool bf16) { return bf16 ? 0 : up256(size_t(a.sequences) * kMosts * sizeof(float)); }      // in front of the sums, cleared with them
size_t acc_bytes(const PackedArgs& a) { return size_t(a.kv_heads) * size_t(most_steps(a)) * kStep * a.D * sizeof(float); }

template <int D, bool kBf16>
int launch_all(PackedArgs p, void* ws, cudaStream_t st) {
  auto kernel = packed_bwd_tc_kernel<D, kBf16>;
  using L = Smem<D>;
  constexpr int smem = L::kTotal + 1024;
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev < 0 || !ready[dev]) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess || attr.numRegs != kLaunchRegs) {
      set_error("packed_bwd_tc_kernel was built with %d registers per thread, expected %d", attr.numRegs, kLaunchRegs);
      return NB200_ERR_LAUNCH;
    }
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute(packed_bwd_tc_kernel, %d): %s", smem, cudaGetErrorString(e));
      return NB200_ERR_LAUNCH;
    }
    if (dev >= 0) ready[dev] = true;
  }
  char* base = static_cast<char*>(ws);
  p.delta = reinterpret_cast<float*>(base);
  void* list = base + delta_bytes(p);
  char* rest = base + delta_bytes(p) + list_bytes(p);
  if (!kBf16) p.squares = reinterpret_cast<float*>(rest);
  rest += squares_bytes(p, kBf16);
  if (!kBf16) p.largest = reinterpret_cast<unsigned*>(rest);
  float* acc = reinterpret_cast<float*>(rest + largest_bytes(p, kBf16));
  BwdArgs a{};
  a.tokens = tile_tokens(kStep, p.group);
  constexpr int kDeltaCta = kDeltaThreads / (D / 8) * kDeltaRows;      // rows
  const int64_t delta_grid = (int64_t(p.tokens_q) * p.heads + kDeltaCta - 1) / kDeltaCta;
  const int64_t value_grid = kBf16 ? 0 : (int64_t(p.tokens_k) * p.kv_heads + kDeltaCta - 1) / kDeltaCta;
  if (cudaMemsetAsync(rest, 0, largest_bytes(p, kBf16) + acc_bytes(p), st) != cudaSuccess) return check_launch("packed_bwd: clearing the sums of dq");
  packed_delta_tc_kernel<D, kBf16><<<unsigned(delta_grid + value_grid), kDeltaThreads, 0, st>>>(p, int(delta_grid));
  count_launch();
  if (int rc = check_launch("packed_delta_tc_kernel")) return rc;
  if (int rc = launch_plan(p, true, kTile, a.tokens, list, st)) return rc;
  CUtensorMap tk, tv, tq, tdo;
  if (!make_token_map(&tk, p.k, p.tokens_k, p.kv_heads, D, p.ks[0], p.ks[1], kTile, 1) ||
      !make_token_map(&tv, p.v, p.tokens_k, p.kv_heads, D, p.vs[0], p.vs[1], kTile, 1) ||
      !make_token_map(&tq, p.q, p.tokens_q, p.heads, D, p.qs[0], p.qs[1], a.tokens, p.group) ||
      !make_token_map(&tdo, p.dout, p.tokens_q, p.heads, D, p.dos[0], p.dos[1], a.tokens, p.group)) {
    set_error("packed_bwd: a tensor map was rejected");
    return NB200_ERR_LAUNCH;
  }
  a.list.count = static_cast<const int*>(list);
  a.list.items = reinterpret_cast<const WorkItem*>(static_cast<const char*>(list) + 16);
  a.kv_heads = p.kv_heads; a.group = p.group; a.heads = p.heads;
  a.causal = p.causal;
  a.scale = p.scale;
  a.lse = p.lse;
  a.delta = p.delta;
  a.dq_acc = acc;
  a.largest = reinterpret_cast<const float*>(p.largest);
  a.all_steps = most_steps(p);
  a.dk = p.dk;
  a.dv = p.dv;
  a.status = device_status_word();
  if (!a.status) { set_error("packed_bwd: no status word on this device"); return NB200_ERR_LAUNCH; }
  const int64_t grid = most_blocks(p.tokens_k, p.sequences, kTile) * p.kv_heads;
  if (launch_dependent(kernel, unsigned(grid), kThreads, smem, st, tk, tv, tq, tdo, a) != cudaSuccess) return check_launch("packed_bwd_tc_kernel");
  count_launch();
  if (int rc = check_launch("packed_bwd_tc_kernel")) return rc;
  packed_dq_finish_kernel<D, kBf16><<<dim3(unsigned(a.all_steps), unsigned(p.kv_heads)), kStep / 4 * (D / 8), 0, st>>>(p, acc, a.all_steps, a.tokens, a.largest);
  count_launch();
  return check_launch("packed_dq_finish_kernel");
}

}  // namespace

size_t tc_packed_bwd_bytes(const PackedArgs& a, int dtype) {
  const bool bf16 = dtype == NB200_BF16;
  return delta_bytes(a) + list_bytes(a) + squares_bytes(a, bf16) + largest_bytes(a, bf16) + acc_bytes(a);
}

int tc_packed_bwd(const PackedArgs& p, int dtype, void* ws, cudaStream_t st) {
  const bool bf16 = dtype == NB200_BF16;
  if (p.D == 64) return bf16 ? launch_all<64, true>(p, ws, st) : launch_all<64, false>(p, ws, st);
  return bf16 ? launch_all<128, true>(p, ws, st) : launch_all<128, false>(p, ws, st);
}

}  // namespace packed
}  // namespace nb200
