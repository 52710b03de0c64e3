// Attention weight sums of a prompt (tcgen05, tensor memory, TMA): how much weight its queries gave to every key.
//
//   sums[b, h, t] (+)= sum over the query heads g of kv head h and the counted queries i of
//                      e^(scale * q[b,g,i] . k[b,h,t] - lse[b,g,i])            (t <= q_start + i when causal)
//
// lse is the forward's log-sum-exp, so each term is a probability of the forward's softmax.  Keys t >= len take no part
// (len = seq_lens[b], or Skv).  Every query counts, unless the mask is causal and lengths are given: then row i, at position
// q_start + i, is a query of the same sequence and counts when that position is < len.  A window > 0 counts only the last
// `window` of them: positions >= len - window, or the last rows of q where there are no positions to go by.
//
// The product is formed transposed, S^T = K Q^T: keys are the 128 rows of the accumulator and queries its columns, so a
// thread that reads its tensor-memory lane holds one key, and the sum over queries is a sum over its own registers -- no
// reduction across threads, no second product.  Per element that leaves one fused multiply-add (scale and lse), one
// exponential and one addition.
//
// Work decomposition.  A unit is (sequence, kv head, 256 keys): two key tiles that share every query tile.  Its steps are
// the (head of the group, 128 queries) pairs that the mask lets it see; under a causal mask the first keys have the
// most.  Where no more than 64 (32) queries of a head can count -- a window, a short prompt -- a step takes the queries
// of two (four) heads: a step costs much the same however many of its columns count (4 prompts of 8192 tokens, window 64,
// groups of 4: 54 us with one head a step, 40 with two).  The steps of all units (plus kUnitCost cells each for what a unit
// costs by itself) form one index space that the persistent blocks share evenly; the lengths live on the device, so every
// block works out its share for itself, in closed form per sequence.  A unit cut between blocks leaves one fp32 partial per
// key and block; the last block to arrive adds them up in block order.
//
// Measured, per call, calls back to back: all queries of 8192 tokens, 32/4 heads: 339 us under the power cap, 820 TFLOP/s (305 us
// in short runs); bound by the exponentials (1.07 G of them are 240 us at the special-function units' rate, 0.83 busy).  The last 64
// queries of 4 prompts of 4307 to 8030 tokens, 32/8 heads: 31 us; bound by what a unit of two steps costs besides them.
//
// Rounding: scores, terms and sums are fp32, the exponential is the hardware's approximation (2^-22 relative); a key's terms go into
// four running sums per step, these into one over the unit's steps, and those of a cut unit are added in block order.  Over all
// queries of 8192 tokens, groups of 8: 8.9e-8 rms from 64 bits (an fp32 product, exponential and sum: 4.9e-8).
//
// Warps: 0-15 the exponentials, one key per thread -- warpgroups 0 and 2 key tile 0, 1 and 3 key tile 1, taking its
// steps in turn: four warps per scheduler, so that one's tensor-memory load hides behind the others' exponentials -- 16 Q
// producer, 17 MMA issuer, 18 lse loader, 19 K producer.  (A second MMA issuer, one per key tile: 350 us instead of 308.)
// Tensor memory: two 128-column accumulators per key tile.  Shared memory: K 3 x 32 KB (the next unit's first keys arrive
// during this one's steps), Q 3 x 32 KB (with two the copies' latency showed), lse 16 x 512 B (eight steps on their way).
#pragma once

#include "gqa_prefill.cuh"
#include "kv8_decode.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace sums {

constexpr int kD = 128;
constexpr int kKeys = 128, kTiles = 2, kPair = kKeys * kTiles;  // keys per tile and unit
constexpr int kQ = 128;                                          // queries per step
constexpr int kTurns = 2;                                        // warpgroups per key tile: they take its steps in turn
constexpr int kEpiWarps = kTiles * kTurns * 4;
constexpr int kThreads = (kEpiWarps + 4) * 32;
// What a unit costs by itself, in steps.  At least one: a unit that no query sees has a cell, whose holder clears its sums.  With 1, 2,
// 3 and 4: all queries of 8192 tokens 305, 305, 305 and 306 us; a window of 64 of 4 prompts of 4096 to 8192 tokens (groups of 4)
// 37.3, 35.5, 35.3, 35.3; of 16 of 1024 to 2048 (groups of 8) 33.9, 33.5, 35.1, 35.2; all queries of 8 of 512 to 1024 44.3, 46.7,
// 47.3, 47.6.
constexpr int kUnitCost = 2;
constexpr int kSlabBytes = 128 * 128;         // [128 rows][64 dims] bf16, one swizzled slab
constexpr int kTileBytes = 2 * kSlabBytes;
constexpr int kKStages = 3, kQStages = 3, kLseStages = 16, kLseAhead = 8;
constexpr int kSmemK = 0;
constexpr int kSmemQ = kKStages * kTileBytes;
constexpr int kSmemLse = kSmemQ + kQStages * kTileBytes;
constexpr int kSmemDead = kSmemLse + kLseStages * kQ * 4;  // one bit per column: its row's lse is -inf, it adds nothing
constexpr int kSmemBar = kSmemDead + kLseStages * (kQ / 8);
constexpr int kNumBars = 2 * kKStages + 2 * kQStages + 2 * kLseStages + 4 * kTiles + 1;
constexpr int kSmemHalf = kSmemBar + kNumBars * 8;  // the second warpgroup's sum of every key
constexpr int kSmemMisc = kSmemHalf + kPair * 4;
constexpr int kSmemWalk = (kSmemMisc + 32 + 7) / 8 * 8;  // the block's first unit, found by one warp
constexpr int kSmemBytes = kSmemWalk + 128 + 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kEpiThreads = kEpiWarps * 32;

enum : int {
    SITE_SUMS_K = 90, SITE_SUMS_Q = 91, SITE_SUMS_LSE = 92, SITE_SUMS_D = 93, SITE_SUMS_DRAIN = 94,
};

struct Params {
    const float* lse;
    const int* seq_lens;  // nullable
    float* out;
    float* slots;         // [W][2][kPair]
    unsigned* counters;
    float scale_log2;
    int B, Sq, Skv, Hq, Hkv, G, q_start, window, causal, accumulate, n_pairs;
    int head_shift;       // log2 of the columns that a head has in a query tile: 7, or 6 or 5 where that takes all its queries
    int groups;           // heads of a kv head's group, or those pairs or fours of them

};

// a / b for non-negative values; most of them fit 32 bits, where a division costs a quarter
__device__ __forceinline__ long long div_nonneg(long long a, long long b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}
// the cells [worker_lo(w), worker_lo(w + 1)) of block w, and the block that holds cell c
__device__ __forceinline__ long long worker_lo(long long w, long long T, long long W) { return div_nonneg(w * T, W); }
__device__ __forceinline__ long long worker_of_cell(long long c, long long T, long long W) {
    return div_nonneg((c + 1) * W - 1, T);
}

// The part of a sequence's work that does not depend on the kv head: which queries count, and how many steps a pair of key
// tiles takes per head.
struct Seq {
    int len;           // keys that take part
    int i_lo, i_hi;    // counted query rows
    int np;            // pairs that hold keys; of these
    int p1, n0, m;     // pairs p < p1 see n0 query tiles per head, later ones max(0, m - 2 p)
    long long cells;   // of all pairs of one kv head

    __device__ __forceinline__ int tiles(int p) const {
        if (p < p1) return n0;
        return p < np && m > 2 * p ? m - 2 * p : 0;
    }
    // cells of the pairs before p
    __device__ __forceinline__ long long before(const Params& prm, int p) const {
        const int a = p < p1 ? p : p1;
        long long n = static_cast<long long>(n0) * a;
        // pairs [p1, e) have m - 2 p > 0 tiles
        int e = (m + 1) / 2;
        if (e > np) e = np;
        if (e > p) e = p;
        if (e > p1) n += static_cast<long long>(m) * (e - p1) - (static_cast<long long>(e) * (e - 1) - static_cast<long long>(p1) * (p1 - 1));
        return static_cast<long long>(kUnitCost) * p + prm.groups * n;
    }
};

__device__ __forceinline__ Seq describe(const Params& p, int b) {
    Seq s;
    s.len = p.seq_lens ? kv8::clamp_len(__ldg(p.seq_lens + b), p.Skv) : p.Skv;
    const bool positions = p.causal && p.seq_lens;
    const long long end = positions ? static_cast<long long>(s.len) - p.q_start : p.Sq;
    const long long start = p.window > 0 ? end - p.window : 0;
    s.i_hi = static_cast<int>(end < 0 ? 0 : (end > p.Sq ? p.Sq : end));
    s.i_lo = static_cast<int>(start < 0 ? 0 : (start > p.Sq ? p.Sq : start));
    s.np = (s.len + kPair - 1) / kPair;
    if (s.i_lo >= s.i_hi || s.len == 0) {
        s.p1 = s.n0 = s.m = 0;
    } else if (p.causal) {
        s.n0 = (s.i_hi - s.i_lo + kQ - 1) / kQ;
        // no query before position t sees key t: later pairs start at their own first key
        s.p1 = (s.i_lo + p.q_start) / kPair + 1;
        s.m = (s.i_hi + p.q_start + kQ - 1) / kQ;
        if (s.p1 > s.np) s.p1 = s.np;
    } else {
        s.n0 = (s.i_hi - s.i_lo + kQ - 1) / kQ;
        s.p1 = s.np;
        s.m = 0;
    }
    s.cells = s.before(p, p.n_pairs);
    return s;
}

// Walks over the units of a block's share.  Every role of the block walks for itself.
struct Walk {
    long long T, W, lo, hi;
    long long unit_lo;  // first cell of the current unit
    int b, kvh, p;
    Seq seq;
    // of the current unit
    int n, steps;       // query tiles per head (or heads that share one), steps in all
    int s_lo, s_hi;     // this block's steps
    bool first;         // the block's first unit

    __device__ __forceinline__ void enter(const Params& prm) {
        n = seq.tiles(p);
        steps = prm.groups * n;
        const long long base = unit_lo + kUnitCost;
        s_lo = lo > base ? static_cast<int>(lo - base) : 0;
        s_hi = hi < base + steps ? static_cast<int>(hi - base) : steps;
    }
    __device__ __forceinline__ bool done() const { return unit_lo >= hi; }
    __device__ __forceinline__ bool active() const { return s_lo < s_hi; }
    __device__ __forceinline__ void next(const Params& prm) {
        first = false;
        unit_lo += kUnitCost + steps;
        if (++p == prm.n_pairs) {
            p = 0;
            if (++kvh == prm.Hkv) {
                kvh = 0;
                if (++b == prm.B) {
                    unit_lo = hi;
                    return;
                }
                seq = describe(prm, b);
            }
        }
        if (unit_lo < hi) enter(prm);
    }
    // first query row of the unit's tile j, and the number of its columns that count
    __device__ __forceinline__ int row0(const Params& prm, int j) const {
        const int own = prm.causal ? p * kPair - prm.q_start : 0;
        return (own > seq.i_lo ? own : seq.i_lo) + j * kQ;
    }
    // heads whose queries the tiles of group g hold
    __device__ __forceinline__ int heads(const Params& prm, int g, int head_shift) const {
        const int most = kQ >> head_shift, left = prm.G - g * most;
        return left < most ? left : most;
    }
    // key tiles of the unit that hold keys: a second one without any is not loaded
    __device__ __forceinline__ int key_tiles() const { return p * kPair + kKeys < seq.len ? 2 : 1; }
};

__device__ __forceinline__ Walk start_walk(const Params& p, int lane) {
    Walk w;
    long long sum = 0;
    for (int i = lane; i < p.B; i += 32) sum += describe(p, i).cells;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w.T = sum * p.Hkv;
    w.W = gridDim.x < w.T ? gridDim.x : w.T;
    w.lo = w.hi = w.unit_lo = 0;
    w.b = w.kvh = w.p = 0;
    w.first = true;
    if (blockIdx.x >= w.W) return w;
    const long long edge = worker_lo(blockIdx.x + (lane & 1), w.T, w.W);  // both ends at once
    w.lo = __shfl_sync(0xffffffffu, edge, 0);
    w.hi = __shfl_sync(0xffffffffu, edge, 1);
    long long seq_lo = 0;
    for (int i0 = 0; i0 < p.B; i0 += 32) {
        const int i = i0 + lane;
        const long long n = i < p.B ? describe(p, i).cells * p.Hkv : 0;
        long long end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += u;
        }
        end += seq_lo;
        const unsigned holds = __ballot_sync(0xffffffffu, w.lo < end);
        if (holds) {
            const int at = __ffs(holds) - 1;
            w.b = i0 + at;
            seq_lo = __shfl_sync(0xffffffffu, end - n, at);
            break;
        }
        seq_lo = __shfl_sync(0xffffffffu, end, 31);
    }
    w.seq = describe(p, w.b);
    w.kvh = static_cast<int>(div_nonneg(w.lo - seq_lo, w.seq.cells));
    const long long head_lo = seq_lo + w.kvh * w.seq.cells;
    const long long off = w.lo - head_lo;
    int a = 0, z = p.n_pairs;  // the last pair whose first cell is <= off lies in [a, z); 32 places are looked at at once
    while (z - a > 1) {
        const int step = (z - a + 31) / 32, at = a + lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, at < z && w.seq.before(p, at) <= off);  // lane 0 among them
        const int last = 31 - __clz(static_cast<int>(below));
        z = a + (last + 1) * step < z ? a + (last + 1) * step : z;
        a += last * step;
    }
    w.p = a;
    w.unit_lo = head_lo + w.seq.before(p, a);
    w.enter(p);
    return w;
}

// kShared: heads share a query tile
template <bool kShared>
__global__ void __launch_bounds__(kThreads, 1)
weight_sums_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const Params p) {
    using namespace prefill;
    const int head_shift = kShared ? p.head_shift : 7;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
    float* lse_buf = reinterpret_cast<float*>(gen_base + sums::kSmemLse);
    uint32_t* dead_buf = reinterpret_cast<uint32_t*>(gen_base + sums::kSmemDead);
    const uint32_t bar0 = base + sums::kSmemBar;
    auto k_full = [&](int s) { return bar0 + 8 * s; };
    auto k_empty = [&](int s) { return bar0 + 8 * (kKStages + s); };
    auto q_full = [&](int s) { return bar0 + 8 * (2 * kKStages + s); };
    auto q_empty = [&](int s) { return bar0 + 8 * (2 * kKStages + kQStages + s); };
    constexpr int kLseBar = 2 * kKStages + 2 * kQStages;
    auto lse_full = [&](int s) { return bar0 + 8 * (kLseBar + s); };
    auto lse_empty = [&](int s) { return bar0 + 8 * (kLseBar + kLseStages + s); };
    constexpr int kDBar = kLseBar + 2 * kLseStages;
    auto d_full = [&](int t, int s) { return bar0 + 8 * (kDBar + t * 2 + s); };
    auto d_empty = [&](int t, int s) { return bar0 + 8 * (kDBar + 2 * sums::kTiles + t * 2 + s); };
    const uint32_t drain_bar = bar0 + 8 * (sums::kNumBars - 1);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen_base + sums::kSmemMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + sums::kSmemMisc + 8);
    volatile int* misc = abort_flag + 1;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kKStages; ++s) {
            mbar_init(k_full(s), 1);
            mbar_init(k_empty(s), 1);
        }
        for (int s = 0; s < kQStages; ++s) {
            mbar_init(q_full(s), 1);
            mbar_init(q_empty(s), 1);
        }
        for (int s = 0; s < kLseStages; ++s) {
            mbar_init(lse_full(s), 32);
            mbar_init(lse_empty(s), kEpiWarps);
        }
        for (int t = 0; t < sums::kTiles; ++t)
            for (int s = 0; s < 2; ++s) {
                mbar_init(d_full(t, s), 1);
                mbar_init(d_empty(t, s), 4);
            }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kEpiWarps + 1) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    Walk* first_walk = reinterpret_cast<Walk*>(gen_base + sums::kSmemWalk);
    static_assert(sizeof(Walk) <= 128, "the walk's place in shared memory");
    if (warp == 1) {  // all 20 warps finding it at once were in one another's way: 6000 cycles instead of 3900
        const Walk found = start_walk(p, lane);
        if (lane == 0) *first_walk = found;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    Walk w = *first_walk;
    const uint32_t tmem_base = *tmem_slot;

    if (warp == kEpiWarps) {
        // ------------------------------- Q producer -------------------------------
        if (lane == 0) {
            tma_prefetch_desc(&tm_q);
            int qs = 0;
            uint32_t qp = 0;
            for (; !w.done(); w.next(p)) {
                if (!w.active()) continue;
                int g = w.s_lo / w.n, j = w.s_lo - g * w.n;
                for (int s = w.s_lo; s < w.s_hi; ++s) {
                    mbar_wait_idle(q_empty(qs), qp ^ 1u, abort_flag, SITE_SUMS_Q, qs);
                    const int heads = w.heads(p, g, head_shift), i0 = w.row0(p, j);
                    const int head0 = w.kvh * p.G + g * (kQ >> head_shift);
                    const uint32_t dst = base + sums::kSmemQ + qs * sums::kTileBytes;
                    mbar_arrive_expect_tx(q_full(qs), heads * (sums::kTileBytes >> (7 - head_shift)));
                    for (int u = 0; u < heads; ++u)
                        for (int d = 0; d < 2; ++d)
                            tma_load_4d(dst + d * kSlabBytes + (u << head_shift) * 128, &tm_q, q_full(qs), d * 64, i0, head0 + u, w.b);
                    if (++qs == kQStages) {
                        qs = 0;
                        qp ^= 1u;
                    }
                    if (++j == w.n) {
                        j = 0;
                        ++g;
                    }
                }
            }
            if (*abort_flag) {
                // a wait gave up somewhere: let the copies already issued land before the block retires
                const long long t0 = clock64();
                for (int s = 0; s < kQStages; ++s)
                    while (!mbar_try_wait(q_full(s), s < qs ? qp : qp ^ 1u) && clock64() - t0 < kWaitLimitCycles / 64) {
                    }
            }
        }
    } else if (warp == kEpiWarps + 3) {
        // ------------- K producer: on its own, so that the next unit's keys are under way during this one's steps -------------
        if (lane == 0) {
            tma_prefetch_desc(&tm_k);
            int ks = 0;
            uint32_t kp = 0;
            for (; !w.done(); w.next(p)) {
                if (!w.active()) continue;
                for (int t = 0; t < w.key_tiles(); ++t) {
                    mbar_wait_idle(k_empty(ks), kp ^ 1u, abort_flag, SITE_SUMS_K, ks);
                    mbar_arrive_expect_tx(k_full(ks), sums::kTileBytes);
                    for (int d = 0; d < 2; ++d)
                        tma_load_4d(base + sums::kSmemK + ks * sums::kTileBytes + d * kSlabBytes, &tm_k, k_full(ks), d * 64,
                                    w.p * kPair + t * kKeys, w.kvh, w.b);
                    if (++ks == kKStages) {
                        ks = 0;
                        kp ^= 1u;
                    }
                }
            }
            if (*abort_flag) {
                const long long t0 = clock64();
                for (int s = 0; s < kKStages; ++s)
                    while (!mbar_try_wait(k_full(s), s < ks ? kp : kp ^ 1u) && clock64() - t0 < kWaitLimitCycles / 64) {
                    }
            }
        }
    } else if (warp == kEpiWarps + 1) {
        // -------------------------------- MMA issuer --------------------------------
        // The whole warp runs the loop and the leader lane's predicate guards the MMAs (see tc_mma_ss_lo_if).  What the operands
        // and the control flow depend on goes through a broadcast: only then does the compiler know that it is the same in all
        // lanes, and keeps it in uniform registers.
        const uint32_t leader = lane == 0 ? 1u : 0u;
        const uint32_t hi = smem_desc_hi(1024);
        auto same = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
        const uint32_t acc0 = static_cast<uint32_t>(same(static_cast<int>(tmem_base)));
        int ks = 0, qs = 0, ds[sums::kTiles] = {0, 0};
        uint32_t kp = 0, qp = 0, dp[sums::kTiles] = {0, 0};
        for (; same(!w.done()); w.next(p)) {
            const int n_steps = same(w.s_hi - w.s_lo);
            if (n_steps <= 0) continue;
            int k_stage[sums::kTiles] = {0, 0};
            const int n_tiles = same(w.key_tiles());
#pragma unroll
            for (int t = 0; t < sums::kTiles; ++t) {
                if (t >= n_tiles) continue;
                mbar_wait_idle(k_full(ks), kp, abort_flag, SITE_SUMS_K, ks);
                k_stage[t] = ks;
                if (++ks == kKStages) {
                    ks = 0;
                    kp ^= 1u;
                }
            }
            // tile j of the unit's n is seen by key tile t from j_sees on (as the exponentials have it)
            const int n = same(w.n), r0 = w.row0(p, 0), key0 = w.p * kPair;
            int j = same(w.s_lo % w.n), j_sees[sums::kTiles];
#pragma unroll
            for (int t = 0; t < sums::kTiles; ++t) {
                const int ahead = p.causal ? key0 + t * kKeys - p.q_start - r0 : 0;
                j_sees[t] = same(t >= n_tiles ? 0x7fffffff : (ahead > 0 ? ahead / kQ : 0));
            }
            for (int left = n_steps; left > 0; --left) {
                mbar_wait_idle(q_full(qs), qp, abort_flag, SITE_SUMS_Q, qs);
                const uint32_t bq = smem_desc_lo(base + sums::kSmemQ + qs * sums::kTileBytes, 16);
#pragma unroll
                for (int t = 0; t < sums::kTiles; ++t) {
                    if (j < j_sees[t]) continue;
                    mbar_wait_idle(d_empty(t, ds[t]), dp[t] ^ 1u, abort_flag, SITE_SUMS_D, t);
                    __syncwarp();
                    tc_fence_after();
                    const uint32_t a = smem_desc_lo(base + sums::kSmemK + k_stage[t] * sums::kTileBytes, 16);
                    const uint32_t d = acc0 + (t * 2 + ds[t]) * kQ;
                    tc_mma_ss_lo_if<false>(leader, d, a, bq, hi, kIdescQK);
#pragma unroll
                    for (int k = 1; k < 8; ++k) {
                        const uint32_t off = ((k >> 2) * kSlabBytes + (k & 3) * 32) >> 4;
                        tc_mma_ss_lo_if<true>(leader, d, a + off, bq + off, hi, kIdescQK);
                    }
                    tc_commit_if(leader, d_full(t, ds[t]));
                    if ((ds[t] ^= 1) == 0) dp[t] ^= 1u;
                }
                tc_commit_if(leader, q_empty(qs));
                if (++qs == kQStages) {
                    qs = 0;
                    qp ^= 1u;
                }
                if (++j == n) j = 0;
            }
            for (int t = 0; t < n_tiles; ++t) tc_commit_if(leader, k_empty(k_stage[t]));
        }
        __syncwarp();
        if (lane == 0) {
            // everything issued must have retired before tensor memory is released
            tc_commit(drain_bar);
            mbar_wait_idle(drain_bar, 0, abort_flag, SITE_SUMS_DRAIN, 0);
            if (*abort_flag) {
                const long long t0 = clock64();
                while (!mbar_try_wait(drain_bar, 0) && clock64() - t0 < kWaitLimitCycles / 64) {
                }
            }
        }
        __syncwarp();
    } else if (warp == kEpiWarps + 2) {
        // -------------------------------- lse loader --------------------------------
        // Copies the steps' lse values (four per lane) eight steps ahead, and turns each lane's own four into
        // -lse * log2(e) once they have landed.  A row with lse = -inf saw no key and adds nothing, whatever its query holds: its
        // column's bit has the exponentials leave it out.  Values behind the last counted row are never looked at.
        int put = 0, got = 0;  // steps issued, steps handed over
        auto hand_over = [&]() {
            const int slot = got % kLseStages;
            unsigned dead = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float* x = lse_buf + slot * kQ + e * 32 + lane;
                const unsigned word = __ballot_sync(0xffffffffu, *x == -INFINITY);
                if (lane == e) dead = word;
                *x = -*x * sums::kLog2e;
            }
            if (lane < 4) dead_buf[slot * 4 + lane] = dead;
            mbar_arrive(lse_full(slot));
            ++got;
        };
        for (; !w.done(); w.next(p)) {
            if (!w.active()) continue;
            int g = w.s_lo / w.n, j = w.s_lo - g * w.n;
            for (int s = w.s_lo; s < w.s_hi; ++s) {
                const int i0 = w.row0(p, j), slot = put % kLseStages;
                const int heads = w.heads(p, g, head_shift);
                const float* src = p.lse + (static_cast<long long>(w.b) * p.Hq + w.kvh * p.G + g * (kQ >> head_shift)) * p.Sq;
                mbar_wait_idle(lse_empty(slot), (static_cast<uint32_t>(put / kLseStages) & 1u) ^ 1u, abort_flag, SITE_SUMS_LSE, slot);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int c = e * 32 + lane, u = c >> head_shift, i = i0 + (c & ((1 << head_shift) - 1));
                    kv8::cp_async_4(smem_u32(lse_buf + slot * kQ + c),
                                    src + static_cast<long long>(u < heads ? u : 0) * p.Sq + (i < w.seq.i_hi ? i : i0));
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++put > kLseAhead) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kLseAhead) : "memory");
                    hand_over();
                }
                if (++j == w.n) {
                    j = 0;
                    ++g;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        while (got < put) hand_over();
    } else if (warp < kEpiWarps) {
        // ------------------------- exponentials and sums (one key per thread) -------------------------
        // warpgroup 2 * turn + t: key tile t, those of its steps whose product lands in accumulator `turn`
        const int t = (warp >> 2) & 1, turn = warp >> 3;
        const int key_in_pair = threadIdx.x & (kPair - 1);
        float* other = reinterpret_cast<float*>(gen_base + sums::kSmemHalf);
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t acc = tmem_base + lane_base + (t * 2 + turn) * kQ;
        int ls = 0, next_turn = 0;
        uint32_t lp = 0, dph = 0;
        for (; !w.done(); w.next(p)) {
            const int key = w.p * kPair + key_in_pair;
            float* out = p.out + (static_cast<long long>(w.b) * p.Hkv + w.kvh) * p.Skv + key;
            if (!w.active()) {
                // a unit without steps: whoever holds its first cell clears its sums
                if (turn == 0 && w.steps == 0 && w.unit_lo >= w.lo && key < p.Skv && !p.accumulate) *out = 0.f;
                continue;
            }
            float total = 0.f;
            // In the unit's own terms: query tile j starts at row r0 + 128 j, and the key tile sees tiles j >= j_sees (none if
            // it holds no keys).
            const int key0 = w.p * kPair + t * kKeys, r0 = w.row0(p, 0);
            const int ahead = p.causal ? key0 - p.q_start - r0 : 0;  // rows between r0 and the key tile's own first query
            const int j_sees = key0 >= w.seq.len ? 0x7fffffff : (ahead > 0 ? ahead / kQ : 0);
            const int rows = w.seq.i_hi - r0;
            // the first column of tile 0 that this key sees; without a causal mask every one, for all keys of a warp alike
            const int own = p.causal ? ahead + static_cast<int>(threadIdx.x & (kKeys - 1)) : lane - 31;
            const float scale = p.scale_log2;
            int j = w.s_lo % w.n, g = w.s_lo / w.n;
#pragma unroll 1
            for (int left = w.s_hi - w.s_lo; left > 0; --left) {
                mbar_wait_idle(lse_full(ls), lp, abort_flag, SITE_SUMS_LSE, ls);
                const bool mine = j >= j_sees && next_turn == turn;
                if (j >= j_sees) next_turn ^= 1;
                if (mine) {
                    mbar_wait_idle(d_full(t, turn), dph, abort_flag, SITE_SUMS_D, t);
                    dph ^= 1u;
                    __syncwarp();
                    tc_fence_after();
                    const float* nl = lse_buf + ls * kQ;
                    const uint4 dead4 = *reinterpret_cast<const uint4*>(dead_buf + ls * 4);
                    const bool dead = (dead4.x | dead4.y | dead4.z | dead4.w) != 0u;  // for all threads alike
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    // columns that count: from the warp's keys' own first ones up to i_hi
                    const int lo = own - j * kQ, hi = rows - j * kQ;
                    const int lo_first = lo - lane, lo_last = lo_first + 31;  // of the warp's lowest and highest key
                    auto add_chunk = [&](const float (&x)[32], const float* l) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 l4 = *reinterpret_cast<const float4*>(l + e);
                            sum[0] += fast_exp2(fmaf(x[e], scale, l4.x));
                            sum[1] += fast_exp2(fmaf(x[e + 1], scale, l4.y));
                            sum[2] += fast_exp2(fmaf(x[e + 2], scale, l4.z));
                            sum[3] += fast_exp2(fmaf(x[e + 3], scale, l4.w));
                        }
                    };
                    const int cols = 1 << head_shift, end = w.heads(p, g, head_shift) << head_shift;  // of a head, of all heads
                    if (lo_last <= 0 && hi >= cols && end == kQ && !dead) {
#pragma unroll
                        for (int c = 0; c < kQ; c += 32) {
                            float x[32];
                            tmem_ld32_wait(acc + c, x);
                            add_chunk(x, nl + c);
                        }
                    } else {
#pragma unroll 1
                        for (int at = 0; at < end; at += 32) {
                            const int c = at & (cols - 1);  // within the head
                            if (c >= hi || lo_first >= c + 32) continue;  // nothing for any key of the warp
                            float x[32];
                            tmem_ld32_wait(acc + at, x);
                            if (lo_last <= c && hi >= c + 32 && !dead) {
                                add_chunk(x, nl + at);
                                continue;
                            }
                            // bit e: the chunk's column e counts for this key.  What does not count may be anything, NaN too
                            const uint32_t seen = (lo <= c ? 0xffffffffu : lo < c + 32 ? 0xffffffffu << (lo - c) : 0u) &
                                                  (hi >= c + 32 ? 0xffffffffu : (1u << (hi - c)) - 1u) &
                                                  ~dead_buf[ls * 4 + at / 32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float y = fmaf(x[e], scale, nl[at + e]);
                                sum[e & 3] += fast_exp2(seen >> e & 1u ? y : -INFINITY);
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(d_empty(t, turn));
                    total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(lse_empty(ls));
                if (++ls == kLseStages) {
                    ls = 0;
                    lp ^= 1u;
                }
                if (++j == w.n) {
                    j = 0;
                    ++g;
                }
            }
            if (key >= w.seq.len) total = 0.f;  // whatever lies behind the sequence
            // the two warpgroups' sums of a key meet; the barrier also keeps the next unit's value out until this one has been read
            if (turn == 1) other[key_in_pair] = total;
            named_bar_sync(1, kEpiThreads);
            if (turn == 0) total += other[key_in_pair];
            named_bar_sync(1, kEpiThreads);
            if (w.s_lo == 0 && w.s_hi == w.steps) {
                if (turn == 0 && key < p.Skv) *out = p.accumulate ? *out + total : total;
                continue;
            }
            // this block's part of the unit goes to the workspace; the last block to arrive adds the parts up
            if (turn == 0) p.slots[(static_cast<long long>(blockIdx.x) * 2 + (w.first ? 0 : 1)) * kPair + key_in_pair] = total;
            const long long w_first = worker_of_cell(w.unit_lo + kUnitCost, w.T, w.W);
            const long long w_last = worker_of_cell(w.unit_lo + kUnitCost + w.steps - 1, w.T, w.W);
            const int n_pieces = static_cast<int>(w_last - w_first) + 1;
            named_bar_sync(1, kEpiThreads);
            if (threadIdx.x == 0) {
                unsigned* counter = p.counters + w_first;
                __threadfence();
                const bool last = atomicAdd(counter, 1u) == static_cast<unsigned>(n_pieces - 1);
                __threadfence();
                if (last) *counter = 0u;  // the counters are zero again when the kernel ends
                *misc = last ? 1 : 0;
            }
            named_bar_sync(1, kEpiThreads);
            if (*misc != 0 && turn == 0) {
                const int which_first = worker_lo(w_first, w.T, w.W) >= w.unit_lo ? 0 : 1;
                float sum = 0.f;
                for (int i = 0; i < n_pieces; ++i)
                    sum += __ldcg(p.slots + ((w_first + i) * 2 + (i == 0 ? which_first : 0)) * kPair + key_in_pair);
                if (key < p.Skv) *out = p.accumulate ? *out + sum : sum;
            }
        }
        tc_fence_before();
    }

    __syncthreads();
    if (warp == kEpiWarps + 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
static int encode_map(CUtensorMap* map, const void* basep, int B, int H, int S, uint32_t rows) {
    const uint64_t row = static_cast<uint64_t>(kD) * 2;
    const uint64_t dims[4] = {static_cast<uint64_t>(kD), static_cast<uint64_t>(S), static_cast<uint64_t>(H),
                              static_cast<uint64_t>(B)};
    const uint64_t strides[3] = {row, row * S, row * S * H};
    const uint32_t box[4] = {64, rows, 1, 1};
    return encode_bf16_4d(map, basep, dims, strides, box);
}

static int blocks_for(int sm_count) {
    return sm_count < decode::kFixedCounters ? sm_count : decode::kFixedCounters;
}
static size_t workspace_bytes(int sm_count) {
    return decode::kSlotOffsetBytes + static_cast<size_t>(blocks_for(sm_count)) * 2 * kPair * sizeof(float);
}

static int launch(const void* q, const void* k, const float* lse, const int* seq_lens, float scale, int causal, int q_start,
                  int window, int flags, float* out, void* workspace, size_t ws_bytes, int B, int Sq, int Skv, int Hq,
                  int Hkv, int D, cudaStream_t st) {
    if (!q || !k || !lse || !out) return CLLO_E_BAD_ARG;
    if (B <= 0 || Sq <= 0 || Skv <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return CLLO_E_BAD_ARG;
    if (q_start < 0 || window < 0 || !isfinite(scale) || (flags & ~(CLLO_SUMS_ACCUMULATE | CLLO_WS_COUNTERS_ZERO)))
        return CLLO_E_BAD_ARG;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(lse, 4) || !aligned_to(out, 4) || !aligned_to(seq_lens, 4))
        return CLLO_E_BAD_ARG;
    const int most = 1 << 30;
    if (D != kD || Sq > most || Skv > most || q_start > most / 2) return CLLO_E_UNSUPPORTED;
    const long long tiles = static_cast<long long>(Hq / Hkv) * ((Sq + kQ - 1) / kQ);
    if (tiles > most) return CLLO_E_UNSUPPORTED;  // a unit's steps are counted in 32 bits
    DeviceInfo* di = nullptr;
    int rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    if (!workspace || ws_bytes < workspace_bytes(di->sm_count) || !aligned_to(workspace, 256)) return CLLO_E_WORKSPACE;
    Params p;
    p.lse = lse;
    p.seq_lens = seq_lens;
    p.out = out;
    p.counters = static_cast<unsigned*>(workspace);
    p.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + decode::kSlotOffsetBytes);
    p.scale_log2 = scale * kLog2e;
    p.B = B;
    p.Sq = Sq;
    p.Skv = Skv;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.q_start = q_start;
    p.window = window;
    p.causal = causal ? 1 : 0;
    p.accumulate = flags & CLLO_SUMS_ACCUMULATE ? 1 : 0;
    p.n_pairs = (Skv + kPair - 1) / kPair;
    const int most_rows = window > 0 && window < Sq ? window : Sq;  // queries of a head that count at most
    p.head_shift = most_rows <= 32 ? 5 : most_rows <= 64 ? 6 : 7;
    p.groups = (p.G + (kQ >> p.head_shift) - 1) / (kQ >> p.head_shift);
    CUtensorMap tm_q, tm_k;
    if ((rc = encode_map(&tm_q, q, B, Hq, Sq, 1u << p.head_shift)) != CLLO_OK) return rc;
    if ((rc = encode_map(&tm_k, k, B, Hkv, Skv, kKeys)) != CLLO_OK) return rc;
    if (!di->sums_attr_set) {
        CLLO_CUDA_TRY(cudaFuncSetAttribute(weight_sums_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        CLLO_CUDA_TRY(cudaFuncSetAttribute(weight_sums_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        di->sums_attr_set = true;
    }
    const int blocks = blocks_for(di->sm_count);
    if (!(flags & CLLO_WS_COUNTERS_ZERO)) CLLO_CUDA_TRY(cudaMemsetAsync(workspace, 0, blocks * sizeof(unsigned), st));
    if (p.head_shift < 7)
        weight_sums_kernel<true><<<blocks, kThreads, kSmemBytes, st>>>(tm_q, tm_k, p);
    else
        weight_sums_kernel<false><<<blocks, kThreads, kSmemBytes, st>>>(tm_q, tm_k, p);
    CLLO_CUDA_TRY(cudaGetLastError());
    return CLLO_OK;
}

}  // namespace sums
}  // namespace cllo
