// Single-token GQA attention over an 8-bit KV cache.
//
//   s_t = scale * q . (kscale_blk(t) * k8_t),  o = sum_t softmax(s)_t * vscale_blk(t) * v8_t,  lse = log sum_t e^(s_t)
//
// over the seq_lens[b] tokens that the cache holds of sequence b; with `weights`, the probabilities of the step are
// added to weights[b, kv head, t], summed over the query heads of the group in a fixed order.
//
// Measured, per call, calls back to back: 60 x 4096 tokens, 128/8 heads, e4m3, tokens before heads: 103 us, 4.9 TB/s (0.75 of a
// copy; 99 us in a graph), bound by the memory system (the same copies without arithmetic, in a graph: 97 us; heads before
// tokens 91 and 83); 1,048,576 tokens, 64/8 heads, int8: 414 us, 0.79 of a copy, under the power cap (ten calls in a row 333 us);
// 17 sequences of 0 to 16384 tokens, 40/8 heads, with weights: 58 us, 4.1 TB/s, bound by issue and by what short units cost;
// one sequence of 1024 tokens: 15 us (13 in a graph), a chain of latencies.  Groups above 16 heads are several units, each of which
// copies and converts the cache for itself: 16 x 16384 tokens, 8 kv heads, e4m3: 91 us with groups of 16, 163 with 20 or 32.
//
// Work decomposition, as in the bf16 decode kernel (gqa_decode.cuh): a unit is one (sequence, kv head, block of <= 16
// query heads), cut into tiles of 64 tokens (at least one, so that an empty sequence writes its zeros); the tiles of all
// units form one index space that W persistent blocks share evenly.  The lengths live on the device, so every block adds
// them up for itself and finds its own range.  Four producer warps stream the tiles by TMA (8 KB of K, 8 KB of V, 128-byte
// swizzle, one box each) into a ring of eight stages; eight consumer warps in four groups take the tiles in turn, 32 tokens
// per warp, with a private online softmax state; states are merged through shared memory at the end of a unit, pieces of
// a cut unit through the workspace by the last block to arrive.  All SMs take part: at 8 stages (128 KB) the bytes in
// flight stay below what slows the memory system (12 stages: 5 % slower on 148 SMs), and it is the arithmetic that bounds.
//
// Arithmetic on codes.  The codes become f16, which holds every e4m3 and int8 value exactly, and feed mma.sync m16n8k16 with
// fp32 accumulation; the scales never touch the codes.  (mma.sync on e4m3 operands is carried out as two f16 products on
// this part: with the query split into two e4m3 terms the scores cost 16 more of them per 16 tokens, 121 us instead of 105.)
//   * a query row is brought to [2^14, 2^15) by a power of two before it becomes f16: exact for every bf16 value within
//     2^28 of the row's largest, and below 2^-39 of it otherwise;
//   * the factor of the query row and the K scale multiply the fp32 scores: 16 tokens of a warp lie in one block of the
//     cache (blocks are multiples of 16);
//   * the V codes become f16 for m16n8k16, and the V scale goes into the exponent: with lv = log2 vscale,
//     p'_t = 2^(s_t + lv_t - m + 11), m = max(s_t + lv_t), so that O = sum p' v8 needs no scaling and
//     l = sum p'_t / vscale_t.  p' is rounded to f16 for the product (half a step: 2^-11 relative, 2^-25 absolute below f16's
//     normal range), l is summed in fp32 before rounding; three more bits than the bf16 that the output is rounded to, whose
//     rounding is all that shows against 64 bits (1.7e-3 rms, as with fp32 probabilities; some outputs land a bf16 step
//     from where fp32 probabilities put them, 5e-4 rms).  The reference m may lag behind the true maximum by 2^4 (kLazy),
//     so the largest p' lies in [2^11, 2^15] and the absolute part is at most 2^-36 of it.  Below 2^-126 a p' is 0: with V
//     scales 2^120 apart that takes a probability below 2^-16 of the other token's.
//
// Layout without transposes.  K: a lane reads 32 consecutive bytes of its token's row as the B operand; the k index may be
// permuted freely as long as Q uses the same permutation.  V: the transposing 8-bit load hands a lane four tokens of one
// dim, two B operand registers once they are f16.  The tokens of the score columns are ordered so that a lane's
// probabilities are of those same four tokens.
#pragma once

#include "gqa_decode.cuh"
#include "host_util.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

constexpr int kTok = 64;  // tokens per stage
constexpr int kStages = 8;
constexpr int kGroups = 4;
constexpr int kWarpsPerGroup = 2;
constexpr int kSubTok = kTok / kWarpsPerGroup;  // tokens per warp and stage
constexpr int kParts = kSubTok / 16;            // 16 tokens each: one k-step of P V
constexpr int kConsumerWarps = kGroups * kWarpsPerGroup;
// Two consumer warpgroups and one of producers.  The consumers hold a unit's Q and O fragments, 96 registers, and the codes
// and scores of their tokens beside them; at the 168 registers that 384 threads get they would spill.  The pool is what
// the block was launched with; asking for more in total would never return.
constexpr int kDecodeThreads = (kConsumerWarps + 4) * 32;
constexpr int kLaunchRegs = 168, kConsumerRegs = 232, kProducerRegs = 40;
static_assert(2 * kConsumerRegs + kProducerRegs <= 3 * kLaunchRegs, "setmaxnreg budget exceeds the block's register pool");
static_assert(kConsumerWarps == 8 && kDecodeThreads == 384, "the register budget is for three warpgroups");
constexpr int kTileBytes = kTok * kD;           // K or V of one stage
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kRows = 16;
constexpr int kPW = kD + 2;                   // {O[128], m (log2 units), l}
constexpr int kSlotFloats = kRows * kPW;
constexpr int kQuarters = kTok / 16;
constexpr int kQPitch = kD * 2 + 16;          // a query row in shared memory; the padding spreads the rows over the banks
constexpr int kQBytes = kRows * kQPitch;      // two of them: the next unit's rows arrive while this one's are in use
// shared memory: ring | exchange of the eight states | their (m, l) | Q x 2 | barriers | block scales per stage | misc
constexpr int kSmemXchg = kStages * kStageBytes;
constexpr int kSmemStat = kSmemXchg + kConsumerWarps * 16 * 32 * 4;
constexpr int kSmemQ = kSmemStat + kConsumerWarps * 4 * 32 * 4;
constexpr int kSmemBar = kSmemQ + 2 * kQBytes;
constexpr int kNumBars = 2 * kStages + 4;
constexpr int kSmemScale = kSmemBar + kNumBars * 8;
constexpr int kSmemMisc = kSmemScale + kStages * 2 * kQuarters * 4;
constexpr int kSmemShare = kSmemMisc + 32;
constexpr int kDecodeSmemBytes = kSmemShare + 64 + 1024;
static_assert(kDecodeSmemBytes <= 227 * 1024, "shared memory of a block");
// What a unit costs beyond its tiles (its query rows, the merge of the eight states, the output), in tiles.  The shares of
// the blocks are cut in these units, so that a block that gets many short sequences is not the last one to finish: 17 sequences
// of 0 to 16384 tokens, 8 kv heads, groups of 5: 57.5 us at 0, 48.9 at 4, 47.1 at 8, 46.9 at 10, 46.8 at 12, 46.9 at 14, 47.1 at 16
// (groups of 4, 8 and 16 likewise, 8 to 14 within 2 %); 64 of 0 to 2048, 4 kv heads, groups of 8: 37.7, 31.1, 26.9, 26.9, 26.9, 27.1,
// 28.5; 33 of 0 to 8192, 2 kv heads, groups of 16: 26.9, 24.8, 23.7, then 22.8.  No effect on full batches.
// Held to the tiles that a block gets on average: where there are fewer than that, spreading the tiles comes first.
constexpr int kUnitCost = 10;
// A unit that many blocks share (one long sequence, few kv heads) is merged in two steps, kFan pieces each: one block that
// reads 148 pieces of 16 rows takes longer than the attention (16384 tokens of one kv head, 148 blocks: 41.7 us in one
// step, 22.3 in two; with 4, 8, 16 or 24 pieces each 24.5, 21.7, 22.5, 20.6; two kv heads, 74 blocks each: 24.7 in one step, 18.4 in
// two of any of these).  Up to kFlatPieces one step is as fast (24 pieces 16.3 us either way).
constexpr int kFlatPieces = 24, kFan = 12;
constexpr int kMaxWorkers = 512;  // two sets of arrival counters in the first 4 KB of the workspace
static_assert(2 * kMaxWorkers <= decode::kFixedCounters, "the counters' place in the workspace");
constexpr float kLazy = 4.f;                 // a reference may lag behind the true maximum by this much (log2)
constexpr float kPShift = 15.f - kLazy;      // p' <= 2^15
// A V scale of 0 (a block that nothing was written to, all codes 0) has no logarithm and no reciprocal; 2^-80 keeps the sum of
// 2^30 tokens' p' / vscale inside fp32.
constexpr float kMinVScale = 8.271806e-25f;
constexpr float kMinFactor = 7.888609e-31f;  // 2^-100: a score is at most 2^31 times its factor, so this much is nothing
static_assert(kStages % kGroups == 0, "a stage buffer must always belong to the same consumer group");

enum : int { SITE_KV8_FULL = 80, SITE_KV8_EMPTY = 81, SITE_KV8_DRAIN = 82, SITE_KV8_Q_FULL = 83, SITE_KV8_Q_EMPTY = 84 };

struct DecodeParams {
    const __nv_bfloat16* q;
    const float* k_scale;
    const float* v_scale;
    const int* seq_lens;
    __nv_bfloat16* o;
    float* lse;       // nullable
    float* scores;    // nullable: [B, Hq, score_pitch] scaled scores in log2 units, for the weights
    float* lse2;      // with scores: [B, Hq] log2 of the normaliser
    float* slots;     // [W][2][16][kPW]
    unsigned* counters;
    long long score_pitch;  // capacity rounded up to whole tiles
    float scale_log2;
    int B, Hq, Hkv, G, n_gblk, capacity, n_blocks, block_shift, kv_layout;
};

// tiles of a sequence; an empty one has one, so that its output is written
__device__ __forceinline__ int tiles_of(int len) { return len <= 0 ? 1 : (len + kTok - 1) / kTok; }

// The cells [cell_lo(w), cell_lo(w + 1)) of block w, cell_lo(w) = floor(w T / W), and the block that holds cell c.  T is below
// 2^31 and W at most kMaxWorkers, so that all but the second's product fits 32 bits.
__device__ __forceinline__ int cell_lo(int w, int T, int W) { return w * (T / W) + w * (T % W) / W; }
__device__ __forceinline__ int block_of_cell(int c, int T, int W) {
    const unsigned long long x = (c + 1ull) * W - 1;
    return static_cast<int>(x >> 32 == 0 ? static_cast<uint32_t>(x) / T : x / T);
}

// counts an arrival: what this block wrote before is visible to whoever counts later, what the others wrote to this block
__device__ __forceinline__ unsigned atomic_inc_acq_rel(unsigned* p) {
    unsigned old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
    return old;
}

// The index space that the blocks share: per unit `cost` cells without a tile, then one cell per tile.
struct Share {
    int T, W, lo, hi;  // all cells, blocks that take part, this block's range
    int cost;
    int b, len;        // the sequence that holds cell lo, and its tokens
    int unit, unit_lo; // the unit of that sequence that does, and the index of its first cell
};

// One warp finds the block's share: two passes over the lengths, the second from registers or L1.
__device__ __forceinline__ Share find_share(const DecodeParams& p, int lane) {
    const int U = p.Hkv * p.n_gblk, grid = static_cast<int>(gridDim.x);
    const int len0 = lane < p.B ? clamp_len(__ldg(p.seq_lens + lane), p.capacity) : 0;  // of the first 32 sequences
    auto len_of = [&](int i) { return i < 32 ? len0 : clamp_len(__ldg(p.seq_lens + i), p.capacity); };
    Share s;
    int tiles = 0;
    for (int i = lane; i < p.B; i += 32) tiles += tiles_of(len_of(i));
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    s.cost = tiles * U >= kUnitCost * grid ? kUnitCost : tiles * U / grid;
    s.T = (tiles + s.cost * p.B) * U;
    // no more blocks than cells: every block between the first and the last tile of a unit then holds some of its tiles,
    // which the count of pieces relies on
    s.W = grid < s.T ? grid : s.T;
    s.lo = s.hi = 0;
    s.b = s.len = s.unit = s.unit_lo = 0;
    const int w = static_cast<int>(blockIdx.x);
    if (w >= s.W) return s;
    const int edge = cell_lo(w + (lane & 1), s.T, s.W);  // both ends at once
    s.lo = __shfl_sync(0xffffffffu, edge, 0);
    s.hi = __shfl_sync(0xffffffffu, edge, 1);
    if (s.lo >= s.hi) return s;
    int before = 0;
    for (int i0 = 0; i0 < p.B; i0 += 32) {
        const int i = i0 + lane;
        const int len = i < p.B ? len_of(i) : 0;
        const int n = i < p.B ? (s.cost + tiles_of(len)) * U : 0;
        int end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += u;
        }
        end += before;
        const unsigned holds = __ballot_sync(0xffffffffu, s.lo < end);
        if (holds) {
            const int at = __ffs(holds) - 1;
            s.b = i0 + at;
            s.len = __shfl_sync(0xffffffffu, len, at);
            const int seq_lo = __shfl_sync(0xffffffffu, end - n, at), n_cells = s.cost + tiles_of(s.len);
            s.unit = (s.lo - seq_lo) / n_cells;
            s.unit_lo = seq_lo + s.unit * n_cells;
            break;
        }
        before = __shfl_sync(0xffffffffu, end, 31);
    }
    return s;
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two 16 x 16 byte matrices, transposed: of the first, r0 holds rows 4 (lane % 4) .. + 3 of column lane / 4 and r1 the same
// rows of column lane / 4 + 8; r2 and r3 of the second.  Lanes 0-15 give the rows of the first, 16-31 of the second.
__device__ __forceinline__ void ldmatrix_b8_x2_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
    return r;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
    float x;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr));
    return x;
}
// an arrival on a barrier once this thread's earlier asynchronous copies have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// untiled asynchronous copy, 16-byte aligned, size a multiple of 16
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// log2 of a normal positive x, exact for powers of two: the exponent apart, the approximation sees [1, 2) only
__device__ __forceinline__ float log2_approx(float x) {
    const uint32_t bits = __float_as_uint(x);
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u)));
    return y + static_cast<float>(static_cast<int>(bits >> 23) - 127);
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// log2 of the softmax's normaliser, m - kPShift + log2(l).  Small V scales make m small and l large: l's exponent is added to m
// first, which leaves no rounding at the size of either.
__device__ __forceinline__ float log2_of_sum(float m, float l) {
    if (l == 0.f) return -INFINITY;
    const uint32_t bits = __float_as_uint(l);
    const int e = static_cast<int>(bits >> 23 & 0xffu) - 127;
    if (e == 128) return l;  // infinite or NaN
    return (m + (static_cast<float>(e) - kPShift)) + log2f(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u));
}

// log-sum-exp merge of the pieces of one unit, 8 columns of one row per thread; pieces in worker order
template <int kBatch, typename RowPtr>
__device__ __forceinline__ void merge_pieces(int n, int c8, RowPtr row_ptr, float (&acc)[8], float& m_out, float& l_out) {
    float mrun = -INFINITY, lrun = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += kBatch) {
        float2 ml[kBatch], d[kBatch][4];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float* row = row_ptr(i0 + i < n ? i0 + i : n - 1);
            ml[i] = __ldcg(reinterpret_cast<const float2*>(row + kD));
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = __ldcg(reinterpret_cast<const float2*>(row + c8 + 2 * e));
            if (i0 + i >= n) ml[i] = make_float2(-INFINITY, 0.f);
        }
        float mnew = mrun;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) mnew = fmaxf(mnew, ml[i].x);
        const float keep = mrun == -INFINITY ? (lrun == 0.f ? 0.f : 1.f) : fast_exp2(mrun - mnew);
        lrun *= keep;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (ml[i].y == 0.f) continue;  // no token; a NaN passes
            const float wgt = fast_exp2(ml[i].x - (mnew == -INFINITY ? 0.f : mnew));
            lrun += wgt * ml[i].y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[2 * e] += wgt * d[i][e].x;
                acc[2 * e + 1] += wgt * d[i][e].y;
            }
        }
        mrun = mnew;
    }
    m_out = mrun;
    l_out = lrun;
}

template <int kFmt, bool kScores>
__global__ void __launch_bounds__(kDecodeThreads, 1)
decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const DecodeParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
    float* stat = reinterpret_cast<float*>(gen_base + kSmemStat);
    float* xchg = reinterpret_cast<float*>(gen_base + kSmemXchg);
    const uint32_t bar_base = base + kSmemBar;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + kSmemMisc);
    volatile int* misc = abort_flag + 1;
    volatile int* pieces = misc + 1;  // of a cut unit: the first block that holds some, their number, the first one's slot
    auto full_bar = [&](int s) { return bar_base + s * 8; };
    auto empty_bar = [&](int s) { return bar_base + (kStages + s) * 8; };
    auto q_full_bar = [&](int s) { return bar_base + (2 * kStages + s) * 8; };
    auto q_empty_bar = [&](int s) { return bar_base + (2 * kStages + 2 + s) * 8; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (kScores) pdl_launch_dependents();  // the weights kernel's blocks may take their places; they wait for this grid's end

    // found once and kept in shared memory: what only the merge of a cut unit needs takes no registers in between
    volatile Share& share = *reinterpret_cast<volatile Share*>(gen_base + kSmemShare);
    const int U = p.Hkv * p.n_gblk;

    if (warp >= kConsumerWarps) {
        // The registers are given away, and the tensor maps fetched, while the consumers' first warps set up the barriers and find
        // the share (2700 cycles from the launch, 1300 of them the latency of the lengths).
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
        if (warp == kConsumerWarps && lane == 0) {
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
        named_bar_sync(2, kDecodeThreads);
        const int lo = share.lo, hi = share.hi, cost = share.cost;
        if (lo >= hi) return;
        // ------------------------------ producers ------------------------------
        // One warp per consumer group, each with the group's own two stages: a wait, two tile copies and the scale copies
        // take the issuing thread about as long as a block at full bandwidth has for two tiles, so one producer for all
        // groups was what bounded the kernel.  Lane 0 copies the tiles, lanes 0-7 one block scale each (a quarter's K or V
        // scale); their arrivals are part of the stage's full barrier.  The last producer also brings the query rows, its lanes
        // in turn: on the way to the first tile they would be as long as the tile's own copies.
        const int grp = warp - kConsumerWarps;
        if (lane < 2 * kQuarters) {
            int b = share.b;
            int n_cells = cost + tiles_of(share.len);
            int cell = lo - share.unit_lo;  // of the unit, next to look at
            int kvh = share.unit / p.n_gblk, gblk = share.unit - kvh * p.n_gblk;
            int slot = grp, q_slot = 0;
            uint32_t phase = 0, q_phase = 0;
            int turn = 0;  // the group whose turn the next tile is
            const bool bshd = p.kv_layout == CLLO_KV_BSHD;
            const float* scales = lane < kQuarters ? p.k_scale : p.v_scale;
            const int quarter = lane % kQuarters;
            const uint32_t scale_dst = base + kSmemScale + lane * 4;
            int left = hi - lo;  // cells of this block's range still ahead
#pragma unroll 1
            while (left > 0) {
                const int here = left < n_cells - cell ? left : n_cells - cell;  // of this unit
                int tile = cell - cost;
                const int tile_end = tile + here;
                if (tile < 0) tile = 0;
                if (tile < tile_end) {
                    const int n_here = tile_end - tile;
                    if (grp == kGroups - 1) {
                        const int rows = (p.G - gblk * kRows) < kRows ? (p.G - gblk * kRows) : kRows;
                        const long long head0 = static_cast<long long>(b) * p.Hq + static_cast<long long>(kvh) * p.G + gblk * kRows;
                        mbar_wait_idle(q_empty_bar(q_slot), q_phase ^ 1u, abort_flag, SITE_KV8_Q_EMPTY, q_slot);
                        if (lane == 0) mbar_arrive_expect_tx(q_full_bar(q_slot), rows * kD * 2);
                        for (int r = lane; r < rows; r += 2 * kQuarters)
                            bulk_load(base + kSmemQ + q_slot * kQBytes + r * kQPitch, p.q + (head0 + r) * kD, kD * 2, q_full_bar(q_slot));
                    }
                    if ((q_slot ^= 1) == 0) q_phase ^= 1u;
                    const float* row = scales + (static_cast<long long>(b) * p.Hkv + kvh) * p.n_blocks;
#pragma unroll 1
                    for (tile += (grp - turn + kGroups) % kGroups; tile < tile_end; tile += kGroups) {
                        mbar_wait_idle(empty_bar(slot), phase ^ 1u, abort_flag, SITE_KV8_EMPTY, slot);
                        const int s0 = tile * kTok;
                        int blk = (s0 + quarter * 16) >> p.block_shift;
                        blk = blk < p.n_blocks ? blk : p.n_blocks - 1;  // a quarter behind the cache: any scale, nobody uses it
                        cp_async_4(scale_dst + slot * (2 * kQuarters * 4), row + blk);
                        cp_async_arrive(full_bar(slot));
                        if (lane == 0) {
                            const int c1 = bshd ? kvh : s0, c2 = bshd ? s0 : kvh;
                            const uint32_t dst = base + slot * kStageBytes;
                            mbar_arrive_expect_tx(full_bar(slot), kStageBytes);
                            tma_load_4d(dst, &tm_k, full_bar(slot), 0, c1, c2, b);
                            tma_load_4d(dst + kTileBytes, &tm_v, full_bar(slot), 0, c1, c2, b);
                        }
                        if ((slot += kGroups) >= kStages) {
                            slot -= kStages;
                            phase ^= 1u;
                        }
                    }
                    turn = (turn + n_here) % kGroups;
                }
                left -= here;
                cell = 0;
                if (++gblk == p.n_gblk) {
                    gblk = 0;
                    if (++kvh == p.Hkv) {
                        kvh = 0;
                        if (++b < p.B) n_cells = cost + tiles_of(clamp_len(__ldg(p.seq_lens + b), p.capacity));
                    }
                }
            }
            if (lane == 0 && *abort_flag) {
                // a wait gave up somewhere: make sure no copy of this warp is still landing when the block retires.  A stage
                // that was filled n times is in phase n - 1; (slot, phase) say how often each one was.
                const long long t0 = clock64();
                auto drain = [&](uint32_t bar, uint32_t parity) {
                    while (!mbar_try_wait(bar, parity)) {
                        if (clock64() - t0 > kWaitLimitCycles / 64) {
                            record_timeout(SITE_KV8_DRAIN, grp);
                            break;
                        }
                    }
                };
                for (int st = grp; st < kStages; st += kGroups) drain(full_bar(st), st < slot ? phase : phase ^ 1u);
                if (grp == kGroups - 1)
                    for (int st = 0; st < 2; ++st) drain(q_full_bar(st), st < q_slot ? q_phase : q_phase ^ 1u);
            }
        }
        return;
    }

    // -------------------------------- consumers --------------------------------
    if (warp == 0) {
        const Share found = find_share(p, lane);
        if (lane == 0) *reinterpret_cast<Share*>(gen_base + kSmemShare) = found;
    } else if (threadIdx.x == 32) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1 + 2 * kQuarters);  // the tile copy and the eight scale copies
            mbar_init(empty_bar(s), kWarpsPerGroup);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(q_full_bar(s), 1);
            mbar_init(q_empty_bar(s), kConsumerWarps);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    named_bar_sync(2, kDecodeThreads);
    const int lo = share.lo, hi = share.hi, cost = share.cost;
    if (lo >= hi) return;
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
    const int g = lane >> 2, tig = lane & 3;
    const int grp = warp / kWarpsPerGroup, sub = warp % kWarpsPerGroup;
    // Tokens of a 16-token part: column n of score n-block nt is token 4 (n >> 1) + 2 nt + (n & 1), so that a lane's four score
    // columns are the tokens 4 tig .. 4 tig + 3, which is also what the transposing load of V hands it.
    // Byte offsets in a tile: K row of n-block nt, 16-byte chunk 2 tig (chunk 2 tig + 1 differs in bit 4; the lanes of a quarter
    // warp touch all eight chunks of the swizzled rows), and the V row this lane addresses, its chunk 0 or 1.
    uint32_t k_off[2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
        const uint32_t row = static_cast<uint32_t>(sub * kSubTok + 4 * (g >> 1) + 2 * nt + (g & 1));
        k_off[nt] = row * 128u + ((static_cast<uint32_t>(2 * tig) ^ (row & 7u)) << 4);
    }
    const uint32_t v_row = static_cast<uint32_t>(sub * kSubTok + (lane & 15));
    const uint32_t v_off = v_row * 128u, v_swz = (v_row & 7u) ^ static_cast<uint32_t>(lane >> 4);

    int b = share.b;
    int len = share.len;
    int n_cells = cost + tiles_of(len);
    int unit = share.unit;  // within the sequence
    int unit_lo = share.unit_lo;
    bool first_unit = true;
    int turn = 0;    // the group whose turn the next tile is
    int slot = grp;  // the next stage of this warp's group
    uint32_t phase = 0;
    int q_slot = 0;
    uint32_t q_phase = 0;

#pragma unroll 1
    while (unit_lo < hi) {
        const int n_t = n_cells - cost;
        // this block's tiles of the unit
        int tile = lo > unit_lo + cost ? lo - unit_lo - cost : 0;
        const int tile_end = hi < unit_lo + n_cells ? hi - unit_lo - cost : n_t;
        const bool whole = tile == 0 && tile_end == n_t;
        if (tile < tile_end) {
        const int kvh = unit / p.n_gblk, gblk = unit - kvh * p.n_gblk;
        const int rows = (p.G - gblk * kRows) < kRows ? (p.G - gblk * kRows) : kRows;
        const long long head0 = static_cast<long long>(b) * p.Hq + static_cast<long long>(kvh) * p.G + gblk * kRows;

        if (!whole && threadIdx.x == 0) {
            // the blocks that hold pieces of the unit, worked out while the first copies are on their way
            const int T = share.T, W = share.W;
            const int w_first = block_of_cell(unit_lo + cost, T, W);
            pieces[0] = w_first;
            pieces[1] = block_of_cell(unit_lo + n_cells - 1, T, W) - w_first + 1;
            pieces[2] = cell_lo(w_first, T, W) >= unit_lo ? 0 : 1;  // the first one's slot for it
        }

        // Q fragments: a lane's K codes of a token are dims 32 tig .. 32 tig + 31, and so are its dims of a query row; four dims
        // make a k-step
        uint32_t qf[8][4];
        float mul0, mul1;  // |scale| * log2(e) / the rows' factors
        mbar_wait_idle(q_full_bar(q_slot), q_phase, abort_flag, SITE_KV8_Q_FULL, q_slot);
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            uint4 raw[4];
            float amax = 0.f;
            const bool ok = g + 8 * r < rows;
            const uint32_t src = base + kSmemQ + q_slot * kQBytes + (g + 8 * r) * kQPitch + tig * 64;
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = ok ? lds128(src + i * 16) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(finite_abs(bf16_lo(w[e])), finite_abs(bf16_hi(w[e]))));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
            e -= 14;  // the row's largest magnitude goes to [2^14, 2^15)
            e = e < -100 ? -100 : e;  // rows below 2^-100 or so (zero among them): their scores vanish either way
            const float f = copysignf(exp2_int(-e), p.scale_log2);  // the sign of the scale goes with the query
            (r ? mul1 : mul0) = fabsf(p.scale_log2) * exp2_int(e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    qf[2 * i + (c >> 1)][(c & 1) * 2 + r] = pack_f16x2(bf16_lo(w[c]) * f, bf16_hi(w[c]) * f);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty_bar(q_slot));
        if ((q_slot ^= 1) == 0) q_phase ^= 1u;

        float o[16][4];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

        // the groups take the block's tiles in turn, across units, so that a stage always belongs to the same group
        const int n_here = tile_end - tile;
#pragma unroll 1
        for (tile += (grp - turn + kGroups) % kGroups; tile < tile_end; tile += kGroups) {
            mbar_wait_idle(full_bar(slot), phase, abort_flag, SITE_KV8_FULL, slot);
            __syncwarp();
            const uint32_t kb = base + slot * kStageBytes, vb = kb + kTileBytes;
            const int tok0 = tile * kTok + sub * kSubTok;
            const int valid = len - tok0;  // of this warp's tokens; the rest holds whatever the cache holds
            if (valid > 0) {
                float ksc[kParts], vsc[kParts];  // of this warp's 16-token parts
#pragma unroll
                for (int u = 0; u < kParts; ++u) {
                    const uint32_t at = base + kSmemScale + slot * (2 * kQuarters * 4) + (sub * kParts + u) * 4;
                    ksc[u] = lds32(at);
                    vsc[u] = fmaxf(lds32(at + kQuarters * 4), kMinVScale);
                }
                // ---- scores: 16 heads x 16 tokens a part; two accumulators per n-block make independent chains ----
                float s[kParts][2][4];
#pragma unroll
                for (int u = 0; u < kParts; ++u) {
                    uint32_t kw[2][8];
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const uint4 x = lds128(kb + u * 2048 + k_off[nt]), y = lds128(kb + u * 2048 + (k_off[nt] ^ 16u));
                        kw[nt][0] = x.x;
                        kw[nt][1] = x.y;
                        kw[nt][2] = x.z;
                        kw[nt][3] = x.w;
                        kw[nt][4] = y.x;
                        kw[nt][5] = y.y;
                        kw[nt][6] = y.z;
                        kw[nt][7] = y.w;
                    }
                    float s2[2][4];
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[u][nt][e] = s2[nt][e] = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            uint32_t b0, b1;
                            decode4_f16<kFmt>(kw[nt][i], b0, b1);
                            mma_f16_16816((i & 1) ? s2[nt] : s[u][nt], qf[i], b0, b1);
                        }
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[u][nt][e] += s2[nt][e];
                }
                if (valid < kSubTok) {
                    // tokens behind the sequence have no score, a part without tokens no scales that anybody wrote
                    if (valid <= 16) ksc[kParts - 1] = vsc[kParts - 1] = 1.f;
#pragma unroll
                    for (int u = 0; u < kParts; ++u)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            const int c = u * 16 + 4 * tig + 2 * nt;
                            if (c >= valid) s[u][nt][0] = s[u][nt][2] = -INFINITY;
                            if (c + 1 >= valid) s[u][nt][1] = s[u][nt][3] = -INFINITY;
                        }
                }
                // ---- online softmax on the raw scores: y = s * f, V scale in the exponent ----
                float f0[kParts], f1[kParts], lv[kParts];
                float mn0 = -INFINITY, mn1 = -INFINITY;
#pragma unroll
                for (int u = 0; u < kParts; ++u) {
                    f0[u] = fmaxf(mul0 * ksc[u], kMinFactor);
                    f1[u] = fmaxf(mul1 * ksc[u], kMinFactor);
                    lv[u] = log2_approx(vsc[u]);
                    mn0 = fmaxf(mn0, fmaf(fmaxf(fmaxf(s[u][0][0], s[u][0][1]), fmaxf(s[u][1][0], s[u][1][1])), f0[u], lv[u]));
                    mn1 = fmaxf(mn1, fmaf(fmaxf(fmaxf(s[u][0][2], s[u][0][3]), fmaxf(s[u][1][2], s[u][1][3])), f1[u], lv[u]));
                }
                if (kScores) {
                    // the pitch has room for whole tiles; what is written behind the sequence is never read
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if (g + 8 * r < rows) {
                            float* dst = p.scores + (head0 + g + 8 * r) * p.score_pitch + tok0 + 4 * tig;
#pragma unroll
                            for (int u = 0; u < kParts; ++u) {
                                const float f = r ? f1[u] : f0[u];
                                *reinterpret_cast<float4*>(dst + u * 16) =
                                    make_float4(s[u][0][2 * r] * f, s[u][0][2 * r + 1] * f, s[u][1][2 * r] * f, s[u][1][2 * r + 1] * f);
                            }
                        }
                    }
                }
                // the reference is raised only when a p' would pass 2^15
                if (__any_sync(0xffffffffu, (mn0 > m0 + kLazy) || (mn1 > m1 + kLazy))) {
                    mn0 = fmaxf(mn0, __shfl_xor_sync(0xffffffffu, mn0, 1));
                    mn1 = fmaxf(mn1, __shfl_xor_sync(0xffffffffu, mn1, 1));
                    mn0 = fmaxf(mn0, __shfl_xor_sync(0xffffffffu, mn0, 2));
                    mn1 = fmaxf(mn1, __shfl_xor_sync(0xffffffffu, mn1, 2));
                    const float r0 = fmaxf(m0, mn0), r1 = fmaxf(m1, mn1);
                    const float a0 = fast_exp2(m0 - r0), a1 = fast_exp2(m1 - r1);
                    l0 *= a0;
                    l1 *= a1;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        o[i][0] *= a0;
                        o[i][1] *= a0;
                        o[i][2] *= a1;
                        o[i][3] *= a1;
                    }
                    m0 = r0;
                    m1 = r1;
                }
#pragma unroll
                for (int u = 0; u < kParts; ++u) {
                    // V codes: word i of a load is dim 32 cp + 8 i + g of the tokens 4 tig .. 4 tig + 3
                    uint32_t vw[4][4];
#pragma unroll
                    for (int cp = 0; cp < 4; ++cp)
                        ldmatrix_b8_x2_trans(vb + u * 2048 + v_off + ((v_swz ^ static_cast<uint32_t>(cp * 2)) << 4), vw[cp]);
                    if (valid < kSubTok) {
                        // values of tokens behind the sequence may be NaN codes, which a zero probability does not silence
                        const int n = valid - (u * 16 + 4 * tig);
                        const uint32_t keep = n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
#pragma unroll
                        for (int cp = 0; cp < 4; ++cp)
#pragma unroll
                            for (int i = 0; i < 4; ++i) vw[cp][i] &= keep;
                    }
                    const float iv = rcp_approx(vsc[u]);
                    const float c0 = lv[u] + kPShift - m0, c1 = lv[u] + kPShift - m1;
                    const float p00 = fast_exp2(fmaf(s[u][0][0], f0[u], c0)), p01 = fast_exp2(fmaf(s[u][0][1], f0[u], c0));
                    const float p02 = fast_exp2(fmaf(s[u][0][2], f1[u], c1)), p03 = fast_exp2(fmaf(s[u][0][3], f1[u], c1));
                    const float p10 = fast_exp2(fmaf(s[u][1][0], f0[u], c0)), p11 = fast_exp2(fmaf(s[u][1][1], f0[u], c0));
                    const float p12 = fast_exp2(fmaf(s[u][1][2], f1[u], c1)), p13 = fast_exp2(fmaf(s[u][1][3], f1[u], c1));
                    l0 = fmaf((p00 + p01) + (p10 + p11), iv, l0);
                    l1 = fmaf((p02 + p03) + (p12 + p13), iv, l1);
                    uint32_t pa[4];
                    pa[0] = pack_f16x2(p00, p01);
                    pa[1] = pack_f16x2(p02, p03);
                    pa[2] = pack_f16x2(p10, p11);
                    pa[3] = pack_f16x2(p12, p13);
                    // ---- O += P V ----
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        uint32_t b0, b1;
                        decode4_f16<kFmt>(vw[c >> 2][c & 3], b0, b1);
                        mma_f16_16816(o[c], pa, b0, b1);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty_bar(slot));
            if ((slot += kGroups) >= kStages) {
                slot -= kStages;
                phase ^= 1u;
            }
        }
        turn = (turn + n_here) % kGroups;

        // ---- merge the private states: every warp posts its (m, l) and, four 8-dim n-blocks at a time, its O; a warp sums two
        // values per lane and round over the warps, in fixed order and with each one's factor: n-block 4 rd + (warp >> 1), row
        // half warp & 1 ----
        *reinterpret_cast<float4*>(stat + (warp * 32 + lane) * 4) = make_float4(m0, m1, l0, l1);
        float2* post = reinterpret_cast<float2*>(xchg);
        const int half = warp & 1;
        float f[kConsumerWarps], ms = -INFINITY, lt = 0.f, acc[4][2];
#pragma unroll
        for (int rd = 0; rd < 4; ++rd) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    post[((warp * 4 + c) * 2 + r) * 32 + lane] = make_float2(o[4 * rd + c][2 * r], o[4 * rd + c][2 * r + 1]);
            named_bar_sync(1, kConsumerWarps * 32);
            if (rd == 0) {
#pragma unroll
                for (int sw = 0; sw < kConsumerWarps; ++sw) ms = fmaxf(ms, stat[(sw * 32 + lane) * 4 + half]);
#pragma unroll
                for (int sw = 0; sw < kConsumerWarps; ++sw) {
                    // a state without tokens has m = -inf and l = 0; one whose scores are all NaN has m = -inf and l = NaN,
                    // and its NaN must survive
                    const float m = stat[(sw * 32 + lane) * 4 + half], l = stat[(sw * 32 + lane) * 4 + 2 + half];
                    f[sw] = m == -INFINITY && l == 0.f ? 0.f : fast_exp2(m - (ms == -INFINITY ? 0.f : ms));
                    lt += l * f[sw];
                }
                lt += __shfl_xor_sync(0xffffffffu, lt, 1);
                lt += __shfl_xor_sync(0xffffffffu, lt, 2);
            }
            float a0 = 0.f, a1 = 0.f;
#pragma unroll
            for (int sw = 0; sw < kConsumerWarps; ++sw) {
                const float2 x = post[((sw * 4 + (warp >> 1)) * 2 + half) * 32 + lane];
                a0 += x.x * f[sw];
                a1 += x.y * f[sw];
            }
            acc[rd][0] = a0;
            acc[rd][1] = a1;
            named_bar_sync(1, kConsumerWarps * 32);
        }

        // ---- every warp writes its share: dims 32 rd + 8 (warp >> 1) + 2 tig + {0, 1} of row g + 8 half ----
        const int col0 = (warp >> 1) * 8 + 2 * tig, row = g + 8 * half;
        if (row < rows) {
            if (whole) {
                const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
                for (int rd = 0; rd < 4; ++rd)
                    *reinterpret_cast<uint32_t*>(p.o + (head0 + row) * kD + rd * 32 + col0) =
                        pack_bf16x2(acc[rd][0] * inv, acc[rd][1] * inv);
                if (col0 == 0) {
                    const float l2 = log2_of_sum(ms, lt);
                    if (p.lse) p.lse[head0 + row] = l2 * kLn2;
                    if (kScores) p.lse2[head0 + row] = l2;
                }
            } else {
                float* dst = p.slots + (static_cast<long long>(blockIdx.x) * 2 + (first_unit ? 0 : 1)) * kSlotFloats + row * kPW;
#pragma unroll
                for (int rd = 0; rd < 4; ++rd)
                    *reinterpret_cast<float2*>(dst + rd * 32 + col0) = make_float2(acc[rd][0], acc[rd][1]);
                if (col0 == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(ms, lt);
            }
        }

        if (!whole) {
            // this block's piece of the unit is in the workspace: count it in; the last one to arrive merges
            const int w_first = pieces[0], n_pieces = pieces[1], which_first = pieces[2];
            auto piece = [&](int i) { return p.slots + static_cast<long long>((w_first + i) * 2 + (i == 0 ? which_first : 0)) * kSlotFloats; };
            // kFan neighbours first, their sum in the first one's slot, then those sums; few pieces go straight to the second step
            const int mine = static_cast<int>(blockIdx.x) - w_first;
            const bool flat = n_pieces <= kFlatPieces;
            const int mrow = threadIdx.x >> 4, c8 = (threadIdx.x & 15) * 8;
#pragma unroll 1
            for (int step = flat ? 1 : 0; step < 2; ++step) {
                const int at = step == 0 ? mine / kFan * kFan : 0;                    // first of the pieces to be merged
                const int stride = step == 0 || flat ? 1 : kFan;
                int n = step == 1 ? (n_pieces + stride - 1) / stride : n_pieces - at;  // their number
                if (step == 0 && n > kFan) n = kFan;
                if (step == 0 && n == 1) continue;
                named_bar_sync(1, kConsumerWarps * 32);
                if (threadIdx.x == 0) {
                    unsigned* counter = p.counters + step * kMaxWorkers + w_first + at;
                    const bool last = atomic_inc_acq_rel(counter) == static_cast<unsigned>(n - 1);
                    if (last) *counter = 0u;  // the counters are zero again when the kernel ends
                    misc[0] = last ? 1 : 0;
                }
                named_bar_sync(1, kConsumerWarps * 32);
                if (misc[0] == 0) break;
                float mg[8], mm = 0.f, ll = 0.f;
                if (mrow < rows) {
                    auto row_of = [&](int i) { return piece(at + i * stride) + mrow * kPW; };
                    if (n <= 4)
                        merge_pieces<4>(n, c8, row_of, mg, mm, ll);
                    else
                        merge_pieces<8>(n, c8, row_of, mg, mm, ll);
                }
                if (step == 0) {
                    named_bar_sync(1, kConsumerWarps * 32);  // the first one's (m, l) have been read by all that need them
                    if (mrow < rows) {
                        float* dst = piece(at) + mrow * kPW;
#pragma unroll
                        for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(dst + c8 + e) = make_float2(mg[e], mg[e + 1]);
                        if (c8 == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(mm, ll);
                    }
                } else if (mrow < rows) {
                    const float inv = ll == 0.f ? 0.f : 1.f / ll;
                    uint4 pk;
                    pk.x = pack_bf16x2(mg[0] * inv, mg[1] * inv);
                    pk.y = pack_bf16x2(mg[2] * inv, mg[3] * inv);
                    pk.z = pack_bf16x2(mg[4] * inv, mg[5] * inv);
                    pk.w = pack_bf16x2(mg[6] * inv, mg[7] * inv);
                    *reinterpret_cast<uint4*>(p.o + (head0 + mrow) * kD + c8) = pk;
                    if (c8 == 0) {
                        const float l2 = log2_of_sum(mm, ll);
                        if (p.lse) p.lse[head0 + mrow] = l2 * kLn2;
                        if (kScores) p.lse2[head0 + mrow] = l2;
                    }
                }
            }
        }

        }
        // next unit of this block's range
        first_unit = false;
        unit_lo += n_cells;
        if (++unit == U) {
            unit = 0;
            if (++b >= p.B) break;
            len = clamp_len(__ldg(p.seq_lens + b), p.capacity);
            n_cells = cost + tiles_of(len);
        }
    }
}

// weights[b, h, t] += sum over the group's heads, in order, of 2^(score - lse2); one thread per token.  A kernel of its own since
// a probability needs the normaliser of the whole sequence; the scores are 4 B per query head and token, mostly still in L2
// (17 sequences of 0 to 16384 tokens, 40 heads: 47 us without weights, 59 with).
constexpr int kWeightThreads = 256, kWeightTok = 1024;
__global__ void __launch_bounds__(kWeightThreads) decode_weights_kernel(const DecodeParams p, float* weights, int n_chunks) {
    pdl_wait_prior_grid();  // scores and normalisers; by every block, so that this grid never ends before the decode's
    const int chunk = blockIdx.x % n_chunks, row = blockIdx.x / n_chunks;  // row = (b, h)
    const int b = row / p.Hkv, h = row - b * p.Hkv;
    const int len = clamp_len(__ldg(p.seq_lens + b), p.capacity);
    const int t0 = chunk * kWeightTok;
    if (t0 >= len) return;
    constexpr int kPer = kWeightTok / kWeightThreads;
    float sum[kPer] = {};
    const long long head0 = static_cast<long long>(b) * p.Hq + static_cast<long long>(h) * p.G;
    for (int g = 0; g < p.G; ++g) {
        const float l2 = __ldg(p.lse2 + head0 + g);
        const float* src = p.scores + (head0 + g) * p.score_pitch;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int t = t0 + i * kWeightThreads + threadIdx.x;
            if (t < len) sum[i] += fast_exp2(__ldcg(src + t) - l2);
        }
    }
    float* dst = weights + static_cast<long long>(row) * p.capacity;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = t0 + i * kWeightThreads + threadIdx.x;
        if (t < len) dst[t] += sum[i];
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// Workspace: arrival counters at the start (4 KB, as in the bf16 decode), partial slots, then -- with weights -- the
// log2 normalisers and the scores of every (query head, token).
struct DecodePlan {
    int W, n_gblk;
    size_t slot_offset, lse2_offset, score_offset, bytes;
};

static long long score_pitch(int capacity) { return (static_cast<long long>(capacity) + kTok - 1) / kTok * kTok; }

static int make_decode_plan(int B, int capacity, int Hq, int Hkv, int D, bool with_weights, int num_workers, int sm_count,
                            DecodePlan* plan) {
    if (B <= 0 || capacity <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || num_workers < 0 || Hq % Hkv != 0) return CLLO_E_BAD_ARG;
    if (D != kD || capacity > kMaxCapacity) return CLLO_E_UNSUPPORTED;
    plan->n_gblk = (Hq / Hkv + kRows - 1) / kRows;
    const long long units = static_cast<long long>(B) * Hkv * plan->n_gblk;
    if (units * kRows > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;
    const long long most = units * ((capacity + kTok - 1) / kTok);  // tiles if every sequence filled the cache
    if (most + units * kUnitCost > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;  // cells are counted in 32 bits
    long long W = num_workers > 0 ? num_workers : sm_count;
    if (W > kMaxWorkers) W = kMaxWorkers;
    if (W > most) W = most;
    if (W < 1) W = 1;
    plan->W = static_cast<int>(W);
    plan->slot_offset = decode::kSlotOffsetBytes;
    plan->lse2_offset = plan->slot_offset + static_cast<size_t>(W) * 2 * kSlotFloats * sizeof(float);
    const size_t rows = static_cast<size_t>(B) * Hq;
    plan->score_offset = plan->lse2_offset + (with_weights ? (rows * sizeof(float) + 255) / 256 * 256 : 0);
    plan->bytes = plan->score_offset + (with_weights ? rows * score_pitch(capacity) * sizeof(float) : 0);
    return CLLO_OK;
}

static int encode_cache_map(CUtensorMap* map, const void* base, int B, int capacity, int Hkv, int kv_layout) {
    EncodeTiledFn fn;
    int rc = get_encode_fn(&fn);
    if (rc != CLLO_OK) return rc;
    const bool bshd = kv_layout == CLLO_KV_BSHD;
    const cuuint64_t S = static_cast<cuuint64_t>(capacity), H = static_cast<cuuint64_t>(Hkv);
    cuuint64_t dims[4] = {kD, bshd ? H : S, bshd ? S : H, static_cast<cuuint64_t>(B)};
    cuuint64_t strides[3] = {kD, bshd ? kD * H : kD * S, kD * H * S};
    cuuint32_t box[4] = {kD, bshd ? 1u : kTok, bshd ? kTok : 1u, 1u};
    cuuint32_t es[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, es,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        t_last_cuda_error = static_cast<int>(cudaErrorInvalidValue);
        return CLLO_E_CUDA;
    }
    return CLLO_OK;
}

template <int kFmt, bool kScores>
static int decode_launch_kernel(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const DecodeParams& p, int W,
                                std::atomic<bool>* attr_set, cudaStream_t st) {
    if (!*attr_set) {
        // refuse to launch, rather than wait inside setmaxnreg, should the compiler have given the kernel a smaller pool
        cudaFuncAttributes fa;
        CLLO_CUDA_TRY(cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(decode_kernel<kFmt, kScores>)));
        if (fa.numRegs < kLaunchRegs) return CLLO_E_UNSUPPORTED;
        CLLO_CUDA_TRY(cudaFuncSetAttribute(decode_kernel<kFmt, kScores>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kDecodeSmemBytes));
        *attr_set = true;
    }
    decode_kernel<kFmt, kScores><<<W, kDecodeThreads, kDecodeSmemBytes, st>>>(tm_k, tm_v, p);
    CLLO_CUDA_TRY(cudaGetLastError());
    return CLLO_OK;
}

static int decode_launch(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                         const int* seq_lens, float scale, void* o, float* lse, float* weights, void* workspace,
                         size_t workspace_bytes, int B, int capacity, int Hq, int Hkv, int D, int kv_layout, int block,
                         int format, int num_workers, cudaStream_t st) {
    if (!q || !k || !v || !k_scale || !v_scale || !seq_lens || !o) return CLLO_E_BAD_ARG;
    const bool counters_zero = (kv_layout & CLLO_WS_COUNTERS_ZERO) != 0;
    kv_layout &= ~CLLO_WS_COUNTERS_ZERO;
    if (kv_layout != CLLO_KV_BSHD && kv_layout != CLLO_KV_BHSD) return CLLO_E_BAD_ARG;
    if (!valid_format(format) || !valid_block(block)) return CLLO_E_BAD_ARG;
    if (!isfinite(scale)) return CLLO_E_BAD_ARG;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(o, 16) || !aligned_to(k_scale, 4) ||
        !aligned_to(v_scale, 4) || !aligned_to(seq_lens, 4) || !aligned_to(lse, 4) || !aligned_to(weights, 4))
        return CLLO_E_BAD_ARG;
    DecodePlan plan;
    int rc = make_decode_plan(B, capacity, Hq, Hkv, D, weights != nullptr, num_workers, 1, &plan);  // arguments only
    if (rc != CLLO_OK) return rc;
    DeviceInfo* di = nullptr;
    rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    rc = make_decode_plan(B, capacity, Hq, Hkv, D, weights != nullptr, num_workers, di->sm_count, &plan);
    if (rc != CLLO_OK) return rc;
    if (!workspace || workspace_bytes < plan.bytes || !aligned_to(workspace, 256)) return CLLO_E_WORKSPACE;
    const int n_chunks = (capacity + kWeightTok - 1) / kWeightTok;
    const long long weight_blocks = static_cast<long long>(B) * Hkv * n_chunks;
    if (weights && weight_blocks > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;
    char* ws = static_cast<char*>(workspace);
    DecodeParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.seq_lens = seq_lens;
    p.o = static_cast<__nv_bfloat16*>(o);
    p.lse = lse;
    p.scores = weights ? reinterpret_cast<float*>(ws + plan.score_offset) : nullptr;
    p.score_pitch = score_pitch(capacity);
    p.lse2 = reinterpret_cast<float*>(ws + plan.lse2_offset);
    p.slots = reinterpret_cast<float*>(ws + plan.slot_offset);
    p.counters = reinterpret_cast<unsigned*>(ws);
    p.scale_log2 = scale * kLog2e;
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.n_gblk = plan.n_gblk;
    p.capacity = capacity;
    p.n_blocks = (capacity + block - 1) / block;
    p.block_shift = block_shift_of(block);
    p.kv_layout = kv_layout;
    CUtensorMap tm_k, tm_v;
    if ((rc = encode_cache_map(&tm_k, k, B, capacity, Hkv, kv_layout)) != CLLO_OK) return rc;
    if ((rc = encode_cache_map(&tm_v, v, B, capacity, Hkv, kv_layout)) != CLLO_OK) return rc;
    if (!counters_zero && plan.W > 1) CLLO_CUDA_TRY(cudaMemsetAsync(ws, 0, 2 * kMaxWorkers * sizeof(unsigned), st));
    std::atomic<bool>* attr = di->kv8_decode_attr_set;
    if (format == CLLO_FMT_E4M3)
        rc = weights ? decode_launch_kernel<CLLO_FMT_E4M3, true>(tm_k, tm_v, p, plan.W, attr + 0, st)
                     : decode_launch_kernel<CLLO_FMT_E4M3, false>(tm_k, tm_v, p, plan.W, attr + 1, st);
    else
        rc = weights ? decode_launch_kernel<CLLO_FMT_INT8, true>(tm_k, tm_v, p, plan.W, attr + 2, st)
                     : decode_launch_kernel<CLLO_FMT_INT8, false>(tm_k, tm_v, p, plan.W, attr + 3, st);
    if (rc != CLLO_OK || !weights) return rc;
    cudaLaunchAttribute dependent;
    const cudaLaunchConfig_t cfg = dependent_launch(&dependent, static_cast<unsigned>(weight_blocks), kWeightThreads, st);
    CLLO_CUDA_TRY(cudaLaunchKernelEx(&cfg, decode_weights_kernel, p, weights, n_chunks));
    return CLLO_OK;
}

}  // namespace kv8
}  // namespace cllo
