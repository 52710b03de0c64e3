// Eviction from the 8-bit KV cache by accumulated attention weight.
//
// Per (batch, kv head) row of len > budget tokens: the first `sink` and the last `recent` tokens stay, and of those
// between them the budget - sink - recent with the largest weight (of equal weights the one that comes first; a NaN counts as
// larger than any number).  What stays keeps its order and moves to another cache; a row within its budget moves whole.
//
// select_kernel finds the threshold weight by radix selection (three passes over order-preserving integers) and writes the
// kept positions in order; gather_kernel moves the rows: codes -> values (exact: a product with a power of two) -> amax of
// the new block -> codes in the new scale.
#pragma once

#include "host_util.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace kv8 {

struct EvictParams {
    const float* weights;  // [B, Hkv, capacity]
    const int* seq_lens;
    int* new_lens;
    int* indices;  // [B, Hkv, budget]
    const uint8_t* from[2];
    uint8_t* to[2];
    const float* scale_from[2];
    float* scale_to[2];
    float* weights_to;  // nullable, [B, Hkv, capacity_to]
    RowStrides stride_from, stride_to;
    int Hkv, capacity, capacity_to, n_blocks_from, n_blocks_to, budget, sink, recent, block_shift;
};

// fp32 -> uint32 in the same order; -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Threads of a selecting block: 1024, or 512 where its chunk of a row is small (8 rows of 4096 tokens in two blocks each, with
// the moving kernel: 12.7 us with 1024, 11.7 with 512) and where there are more rows than SMs, so that two blocks share one (512
// rows of 2048: 66 and 47 us; 160 rows of 2304: 35 and 27).  Else 1024 (144 rows of 2752: 23.6 and 24.2 us, of 8192 44 and 47).
constexpr int kSelectThreads = 1024, kSelectThreadsHalf = 512;
constexpr int kSmallChunk = 2048;
constexpr int kHalfMaxTokens = 16384;                          // what two blocks hold in shared memory beside each other
constexpr int kDigitBits = 11, kBins = 1 << kDigitBits;      // three passes: 11, 11 and 10 bits
constexpr int kMaxCluster = 8;
constexpr int kKeysInSmem = 48 * 1024;                         // of a block's chunk; what is longer is read again in each pass
constexpr int kSelectUnroll = 8;
// Keys that a chunk of n tokens takes in shared memory: whole groups of four, since they are counted four at a time.
__host__ __device__ constexpr int keys_in_smem(int n) { return ((n < kKeysInSmem ? n : kKeysInSmem) + 3) & ~3; }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
// a word of another block's shared memory, at the address it has in this block's
__device__ __forceinline__ int cluster_load(const int* p, uint32_t rank) {
    uint32_t remote;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

__device__ __forceinline__ void cluster_load2(const int* p, uint32_t rank, int& x, int& y) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(remote) : "memory");
}

// One cluster of blocks per (batch, kv head) row, each block a contiguous chunk of the row.  The chunk's weights are read
// once and stay in shared memory as integers; a pass counts the digits of the keys that share the prefix found so far
// (equal digits of a warp are added together first: weights cluster in few exponents, and ties share every digit), the
// blocks add up each other's counts over distributed shared memory, and every block finds the same digit.  Bound by the
// latency of its passes, 5 cluster barriers and 9 block barriers: 32 rows of 32768 tokens 16 us, 264 of up to 2304 14 us.
template <int kThreads>
__global__ void __launch_bounds__(kThreads, kSelectThreads / kThreads) select_kernel(const EvictParams p) {
    constexpr int kWarps = kThreads / 32;
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ __align__(8) int hist[3][kBins];  // one per pass
    __shared__ int group_sum[3][32];             // of kBins / 32 bins each
    __shared__ int s_digit, s_need;
    __shared__ int s_counts[2];  // this block's tokens that stay whatever the others hold, and those at the threshold
    pdl_launch_dependents();  // the moving blocks may take their places; they wait for this grid's end
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < 3 * kBins; i += kThreads) hist[0][i] = 0;
    const int C = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
    const int row = blockIdx.x / C;
    const int h = row % p.Hkv, b = row / p.Hkv;
    {  // the row's weights set out for L2 while the length is on its way
        const int part = (p.capacity + C - 1) / C, end = part * (rank + 1) < p.capacity ? part * (rank + 1) : p.capacity;
        const float* all = p.weights + static_cast<long long>(row) * p.capacity;
        for (int i = part * rank + tid * 32; i < end; i += kThreads * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(all + i));
    }
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    int* idx = p.indices + static_cast<long long>(row) * p.budget;
    const int kept = len < p.budget ? len : p.budget;
    if (h == 0 && tid == 0 && rank == 0) p.new_lens[b] = kept;
    for (int j = kept + rank * kThreads + tid; j < p.budget; j += C * kThreads) idx[j] = -1;
    if (len <= p.budget) {  // the whole cluster alike
        for (int j = rank * kThreads + tid; j < len; j += C * kThreads) idx[j] = j;
        return;
    }
    const int chunk = (len + C - 1) / C;
    const int t0 = chunk * rank < len ? chunk * rank : len;
    const int n = t0 + chunk < len ? chunk : len - t0;
    const float* w = p.weights + static_cast<long long>(row) * p.capacity + t0;
    const int lo = p.sink - t0, hi = len - p.recent - t0;  // candidates [lo, hi) in the chunk's own terms
    const int n_smem = n < kKeysInSmem ? n : kKeysInSmem;
    // The key of a token that is no candidate is 0, which no weight has: order_key is at least that of -infinity.
    auto candidate_key = [&](int i, float x) { return i >= lo && i < hi ? order_key(x) : 0u; };
    const int n_pad = keys_in_smem(n);
    for (int i0 = tid; i0 < n_pad; i0 += kThreads * kSelectUnroll) {
        float x[kSelectUnroll];
#pragma unroll
        for (int u = 0; u < kSelectUnroll; ++u) {
            const int i = i0 + u * kThreads;
            x[u] = i < n_smem ? __ldg(w + i) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kSelectUnroll; ++u) {
            const int i = i0 + u * kThreads;
            if (i < n_pad) keys[i] = i < n_smem ? candidate_key(i, x[u]) : 0u;
        }
    }
    auto key_at = [&](int i) { return i < n_smem ? keys[i] : candidate_key(i, __ldg(w + i)); };
    __syncthreads();

    const bool any = p.budget > p.sink + p.recent;
    uint32_t prefix = 0u, mask = 0u;
    int need = p.budget - p.sink - p.recent;  // how many of the keys that share the prefix are kept
    if (any) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t digits = pass == 2 ? 0x3ffu : 0x7ffu;
            int* counts = hist[pass];
            auto count = [&](uint32_t key) {  // by all lanes of a warp together
                const bool in = (key & mask) == prefix;
                const unsigned active = __ballot_sync(0xffffffffu, in);
                if (active == 0u) return;
                const int first = __ffs(active) - 1;
                const int d = static_cast<int>((key >> shift) & digits), d0 = __shfl_sync(0xffffffffu, d, first);
                if (__all_sync(0xffffffffu, !in || d == d0)) {
                    if (lane == first) atomicAdd(&counts[d0], __popc(active));  // ties, or one exponent for all
                } else if (in) {
                    atomicAdd(&counts[d], 1);
                }
            };
            const int quads = n_pad / 4;
#pragma unroll 2
            for (int q0 = 0; q0 < quads; q0 += kThreads) {
                const uint4 k4 = q0 + tid < quads ? reinterpret_cast<const uint4*>(keys)[q0 + tid] : make_uint4(0u, 0u, 0u, 0u);
                count(k4.x);
                count(k4.y);
                count(k4.z);
                count(k4.w);
            }
#pragma unroll 1
            for (int i0 = n_smem; i0 < n; i0 += kThreads) count(i0 + tid < n ? key_at(i0 + tid) : 0u);
            // The largest digit at which the count from the top reaches `need`, over the whole cluster: first its group of 64
            // bins by the groups' sums, then the bin; few words cross between the blocks (all 2048 bins of every other block: 1000
            // cycles more a pass).
            __syncthreads();
#pragma unroll
            for (int g = warp; g < 32; g += kWarps) {
                const int2 x = *reinterpret_cast<const int2*>(&counts[64 * g + 2 * lane]);
                const int sum = __reduce_add_sync(0xffffffffu, x.x + x.y);
                if (lane == 0) group_sum[pass][g] = sum;
            }
            cluster_sync();
            if (warp == 0) {
                auto from_top = [&](int v) {  // inclusive sum over the lanes
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int u = __shfl_up_sync(0xffffffffu, v, o);
                        if (lane >= o) v += u;
                    }
                    return v;
                };
                int part[kMaxCluster][2], c[2] = {0, 0};
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) part[r][0] = r < C ? cluster_load(&group_sum[pass][31 - lane], r) : 0;
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) c[0] += part[r][0];
                int v = from_top(c[0]);
                const int at = __ffs(__ballot_sync(0xffffffffu, v - c[0] < need && need <= v)) - 1;
                int before = __shfl_sync(0xffffffffu, v - c[0], at);  // keys in higher groups
                const int top = 64 * (31 - at) + 63 - 2 * lane;       // this lane's higher bin of the group
                c[0] = c[1] = 0;
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {
                    part[r][0] = part[r][1] = 0;
                    if (r < C) cluster_load2(&counts[top - 1], r, part[r][1], part[r][0]);
                }
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {
                    c[0] += part[r][0];
                    c[1] += part[r][1];
                }
                before += from_top(c[0] + c[1]) - c[0] - c[1];  // keys in higher bins
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (before < need && need <= before + c[u]) {
                        s_digit = top - u;
                        s_need = need - before;
                    }
                    before += c[u];
                }
            }
            __syncthreads();
            prefix |= static_cast<uint32_t>(s_digit) << shift;
            mask |= digits << shift;
            need = s_need;
        }
    }

    // positions in order: how many stay and how many sit at the threshold before each token
    auto classify = [&](int i, bool& above, bool& equal) {
        above = equal = false;
        if (i >= n) return;
        if (i < lo || i >= hi) {
            above = true;  // sink or recent
        } else if (any) {
            const uint32_t key = key_at(i);
            above = key > prefix;
            equal = key == prefix;
        }
    };
    // a warp owns a contiguous stretch of the chunk, so that only the warps' totals have to meet
    const int per_warp = ((n + kWarps - 1) / (kWarps) + 31) / 32 * 32;
    const int w_lo = warp * per_warp, w_hi = w_lo + per_warp < n ? w_lo + per_warp : n;
    int n_above = 0, n_equal = 0;
    unsigned kept_above = 0u, kept_equal = 0u;  // lane k: the warp's answers of its k-th step
#pragma unroll 4
    for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
        bool above, equal;
        classify(i0 + lane, above, equal);
        const unsigned ba = __ballot_sync(0xffffffffu, above), be = __ballot_sync(0xffffffffu, equal);
        n_above += __popc(ba);
        n_equal += __popc(be);
        if (i0 - w_lo == lane * 32) {
            kept_above = ba;
            kept_equal = be;
        }
    }
    int* totals = hist[0];  // two ints per warp; the others read the first pass's counts before they came to the second's barrier
    if (lane == 0) {
        totals[2 * warp] = n_above;
        totals[2 * warp + 1] = n_equal;
    }
    __syncthreads();
    if (warp == 0) {
        int a = lane < kWarps ? totals[2 * lane] : 0, e = lane < kWarps ? totals[2 * lane + 1] : 0;
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            e += __shfl_xor_sync(0xffffffffu, e, o);
        }
        if (lane == 0) {
            s_counts[0] = a;
            s_counts[1] = e;
        }
    }
    cluster_sync();
    int a_before = 0, e_before = 0;
    for (int r = 0; r < rank; ++r) {
        a_before += cluster_load(&s_counts[0], r);
        e_before += cluster_load(&s_counts[1], r);
    }
    {
        int a = lane < warp ? totals[2 * lane] : 0, e = lane < warp ? totals[2 * lane + 1] : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            e += __shfl_xor_sync(0xffffffffu, e, o);
        }
        a_before += a;
        e_before += e;
    }
    cluster_arrive();  // this block has read what it reads of the others
    const unsigned below = (1u << lane) - 1u;
#pragma unroll 2
    for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
        unsigned ba, be;
        if (const int k = (i0 - w_lo) / 32; k < 32) {
            ba = __shfl_sync(0xffffffffu, kept_above, k);
            be = __shfl_sync(0xffffffffu, kept_equal, k);
        } else {
            bool above, equal;
            classify(i0 + lane, above, equal);
            ba = __ballot_sync(0xffffffffu, above);
            be = __ballot_sync(0xffffffffu, equal);
        }
        const bool above = ba >> lane & 1u, equal = be >> lane & 1u;
        const int a = a_before + __popc(ba & below), e = e_before + __popc(be & below);
        // of the tokens at the threshold the first `need` stay
        if (above || (equal && e < need)) idx[a + (e < need ? e : need)] = t0 + i0 + lane;
        a_before += __popc(ba);
        e_before += __popc(be);
    }
    cluster_wait();  // no block leaves while another may still read its counts
}

// four lanes per row, 32 bytes of K and of V per lane
__host__ __device__ constexpr int gather_threads(int block) { return block * 4; }

// One thread block per block of the second cache, one row per four lanes: all loads in flight before the first is looked at;
// values -> amax -> new scale -> codes.  Bound by the latency of its gathers (position, then 128-byte rows) and by issue: what
// a row costs besides its values (addresses, scales) is as much as the values cost, so a lane takes 32 bytes of each (33 x 1152
// to 2304 int8 tokens: 46 us, 5.1 TB/s; with 16 bytes of each of two rows per lane 60).
template <int kFmt, int kBlock>
__global__ void __launch_bounds__(gather_threads(kBlock)) gather_kernel(const EvictParams p) {
    constexpr int kThreads = gather_threads(kBlock);
    __shared__ float warp_amax[2][kThreads / 32];
    pdl_wait_prior_grid();  // the positions; by every block, so that this grid never ends before the one that writes them
    // kv heads next to each other: with tokens before heads in memory they share DRAM pages
    const int h = blockIdx.x % p.Hkv, at = blockIdx.x / p.Hkv;
    const int b = at / p.n_blocks_to, blk = at % p.n_blocks_to, row = b * p.Hkv + h;
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    const int kept = len < p.budget ? len : p.budget;
    const int j0 = blk * kBlock;
    if (j0 >= kept) return;
    const int j = j0 + (threadIdx.x >> 2), c32 = (threadIdx.x & 3) * 32;
    const bool live = j < kept;
    uint4 c[2][2];
    float s[2] = {0.f, 0.f};
    c[0][0] = c[0][1] = c[1][0] = c[1][1] = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
        const int t = __ldcg(p.indices + static_cast<long long>(row) * p.budget + j);
        const long long from = b * p.stride_from.batch + h * p.stride_from.head + t * p.stride_from.token + c32;
        const long long scale_at = static_cast<long long>(row) * p.n_blocks_from + (t >> p.block_shift);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint4* src = reinterpret_cast<const uint4*>(p.from[which] + from);
            c[which][0] = __ldg(src);
            c[which][1] = __ldg(src + 1);
            s[which] = __ldg(p.scale_from[which] + scale_at);
        }
        if (p.weights_to && (threadIdx.x & 3) == 0)
            p.weights_to[static_cast<long long>(row) * p.capacity_to + j] =
                __ldg(p.weights + static_cast<long long>(row) * p.capacity + t);
    }
    // codes -> f16 pairs, which hold them exactly; the rows' largest magnitudes times their scales give the block's
    uint32_t f[2][16];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const uint32_t w[8] = {c[which][0].x, c[which][0].y, c[which][0].z, c[which][0].w,
                               c[which][1].x, c[which][1].y, c[which][1].z, c[which][1].w};
        uint32_t top = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            decode4_f16<kFmt>(w[k], f[which][2 * k], f[which][2 * k + 1]);
            top = max_f16x2(top, max_f16x2(f[which][2 * k] & 0x7fff7fffu, f[which][2 * k + 1] & 0x7fff7fffu));
        }
        float amax = finite_abs(f16_max_of_pair(top) * s[which]);  // a NaN does not take part
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) warp_amax[which][threadIdx.x >> 5] = amax;
    }
    __syncthreads();
    const long long to = b * p.stride_to.batch + h * p.stride_to.head + j * p.stride_to.token + c32;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) amax = fmaxf(amax, warp_amax[which][i]);
        const int e_new = scale_exp<kFmt>(amax);
        const float inv = exp2_int(-e_new);
        if (threadIdx.x == 0) p.scale_to[which][static_cast<long long>(row) * p.n_blocks_to + blk] = exp2_int(e_new);
        if (!live) continue;
        uint32_t d[8];
        // Scales are powers of two: the code times their ratio is exact in f16 where it can still round to a code other than
        // zero, so one rounding, to the new code, is all there is.  A ratio beyond f16 (a block of nothing but codes at the
        // very bottom of e4m3) or scales that are no powers of two go through fp32.
        const float ratio = s[which] * inv;
        if ((__float_as_uint(ratio) & 0x7fffffu) == 0u && fabsf(ratio) <= 32768.f) {
            const uint32_t r = pack_f16x2(ratio, ratio);
#pragma unroll
            for (int k = 0; k < 8; ++k) d[k] = requant4<kFmt>(f[which][2 * k], f[which][2 * k + 1], r);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float v[4];
                f16x2_to_f32(f[which][2 * k], v[0], v[1]);
                f16x2_to_f32(f[which][2 * k + 1], v[2], v[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = v[e] * s[which] * inv;
                d[k] = encode4<kFmt>(v[0], v[1], v[2], v[3]);
            }
        }
        uint4* dst = reinterpret_cast<uint4*>(p.to[which] + to);
        dst[0] = make_uint4(d[0], d[1], d[2], d[3]);
        dst[1] = make_uint4(d[4], d[5], d[6], d[7]);
    }
}

template <int kFmt>
static cudaError_t gather_dispatch(const EvictParams& p, int block, unsigned grid, cudaStream_t st) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = dependent_launch(&attr, grid, static_cast<unsigned>(gather_threads(block)), st);
    switch (block) {
        case 16: return cudaLaunchKernelEx(&cfg, gather_kernel<kFmt, 16>, p);
        case 32: return cudaLaunchKernelEx(&cfg, gather_kernel<kFmt, 32>, p);
        case 64: return cudaLaunchKernelEx(&cfg, gather_kernel<kFmt, 64>, p);
        default: return cudaLaunchKernelEx(&cfg, gather_kernel<kFmt, 128>, p);
    }
}

static bool ranges_overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

static int evict_launch(const void* k, const void* v, const float* k_scale, const float* v_scale, const float* weights,
                        const int* seq_lens, void* k_to, void* v_to, float* k_scale_to, float* v_scale_to,
                        float* weights_to, int* new_lens, int* indices, int B, int capacity, int capacity_to, int Hkv,
                        int D, int budget, int sink, int recent, int kv_layout, int block, int format, cudaStream_t st) {
    if (!k || !v || !k_scale || !v_scale || !weights || !seq_lens || !k_to || !v_to || !k_scale_to || !v_scale_to ||
        !new_lens || !indices)
        return CLLO_E_BAD_ARG;
    if (B <= 0 || capacity <= 0 || capacity_to <= 0 || Hkv <= 0 || D <= 0) return CLLO_E_BAD_ARG;
    if (budget <= 0 || sink < 0 || recent < 0 || static_cast<long long>(sink) + recent > budget) return CLLO_E_BAD_ARG;
    if ((budget < capacity ? budget : capacity) > capacity_to) return CLLO_E_BAD_ARG;
    if (kv_layout != CLLO_KV_BSHD && kv_layout != CLLO_KV_BHSD) return CLLO_E_BAD_ARG;
    if (!valid_format(format) || !valid_block(block)) return CLLO_E_BAD_ARG;
    if (D != kD) return CLLO_E_UNSUPPORTED;
    if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(k_to, 16) || !aligned_to(v_to, 16)) return CLLO_E_BAD_ARG;
    if (!aligned_to(k_scale, 4) || !aligned_to(v_scale, 4) || !aligned_to(weights, 4) || !aligned_to(seq_lens, 4) ||
        !aligned_to(k_scale_to, 4) || !aligned_to(v_scale_to, 4) || !aligned_to(weights_to, 4) || !aligned_to(new_lens, 4) ||
        !aligned_to(indices, 4))
        return CLLO_E_BAD_ARG;
    if (capacity > kMaxCapacity || capacity_to > kMaxCapacity || budget > kMaxCapacity) return CLLO_E_UNSUPPORTED;
    const size_t rows = static_cast<size_t>(B) * Hkv;
    const size_t n = rows * capacity * kD, n_to = rows * capacity_to * kD;
    const size_t n_scale = rows * ((capacity + block - 1) / block) * 4, n_scale_to = rows * ((capacity_to + block - 1) / block) * 4;
    // Blocks read while others write: no tensor written to may share memory with one that is read, or with another one written to.
    struct Range {
        const void* at;
        size_t bytes;
    };
    const Range written[] = {{k_to, n_to}, {v_to, n_to}, {k_scale_to, n_scale_to}, {v_scale_to, n_scale_to},
                             {new_lens, static_cast<size_t>(B) * 4}, {indices, rows * budget * 4},
                             {weights_to, weights_to ? rows * capacity_to * 4 : 0}};
    const Range read[] = {{k, n}, {v, n}, {k_scale, n_scale}, {v_scale, n_scale}, {weights, rows * capacity * 4},
                          {seq_lens, static_cast<size_t>(B) * 4}};
    for (const Range* w = written; w != written + 7; ++w) {
        if (w->bytes == 0) continue;
        for (const Range& r : read)
            if (ranges_overlap(w->at, w->bytes, r.at, r.bytes)) return CLLO_E_BAD_ARG;
        for (const Range* o = written; o != w; ++o)
            if (ranges_overlap(w->at, w->bytes, o->at, o->bytes)) return CLLO_E_BAD_ARG;
    }
    DeviceInfo* di = nullptr;
    int rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    EvictParams p;
    p.weights = weights;
    p.seq_lens = seq_lens;
    p.new_lens = new_lens;
    p.indices = indices;
    p.from[0] = static_cast<const uint8_t*>(k);
    p.from[1] = static_cast<const uint8_t*>(v);
    p.to[0] = static_cast<uint8_t*>(k_to);
    p.to[1] = static_cast<uint8_t*>(v_to);
    p.scale_from[0] = k_scale;
    p.scale_from[1] = v_scale;
    p.scale_to[0] = k_scale_to;
    p.scale_to[1] = v_scale_to;
    p.weights_to = weights_to;
    p.stride_from = cache_strides(kv_layout, capacity, Hkv);
    p.stride_to = cache_strides(kv_layout, capacity_to, Hkv);
    p.Hkv = Hkv;
    p.capacity = capacity;
    p.capacity_to = capacity_to;
    p.n_blocks_from = (capacity + block - 1) / block;
    p.n_blocks_to = (capacity_to + block - 1) / block;
    p.budget = budget;
    p.sink = sink;
    p.recent = recent;
    p.block_shift = block_shift_of(block);
    const long long blocks = static_cast<long long>(rows) * p.n_blocks_to;
    if (blocks > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;
    // blocks per row: enough to fill the GPU, chunks of at least 2048 tokens (both kernels of 32 rows of 32768 tokens: 31 us with
    // four, 52 with one; 8 rows of 131072: 34 us with eight, 42 with as few as hold the keys)
    int cluster = 1;
    while (cluster < kMaxCluster && rows * cluster * 2 <= static_cast<size_t>(di->sm_count) && capacity / (cluster * 2) >= 2048) cluster *= 2;
    // rows longer than what one block holds in shared memory are shared out even on a full GPU
    while (cluster < kMaxCluster && capacity / cluster > kKeysInSmem) cluster *= 2;
    const int chunk = (capacity + cluster - 1) / cluster;
    const int smem = keys_in_smem(chunk) * 4;
    if (rows * cluster > 0x7fffffffULL) return CLLO_E_UNSUPPORTED;
    if (!di->kv8_select_attr_set) {
        CLLO_CUDA_TRY(cudaFuncSetAttribute(select_kernel<kSelectThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeysInSmem * 4));
        CLLO_CUDA_TRY(cudaFuncSetAttribute(select_kernel<kSelectThreadsHalf>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kHalfMaxTokens * 4));
        di->kv8_select_attr_set = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
    const bool half = chunk <= kSmallChunk || (rows > static_cast<size_t>(di->sm_count) && chunk <= kHalfMaxTokens);
    cfg.blockDim = dim3(half ? kSelectThreadsHalf : kSelectThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CLLO_CUDA_TRY(cudaLaunchKernelEx(&cfg, half ? select_kernel<kSelectThreadsHalf> : select_kernel<kSelectThreads>, p));
    const unsigned grid = static_cast<unsigned>(blocks);
    CLLO_CUDA_TRY((format == CLLO_FMT_E4M3 ? gather_dispatch<CLLO_FMT_E4M3> : gather_dispatch<CLLO_FMT_INT8>)(p, block, grid, st));
    return CLLO_OK;
}

}  // namespace kv8
}  // namespace cllo
