// Eviction from the 8-bit KV cache by accumulated attention weight.
//
// Per (batch, kv head) row of len > budget tokens: the first `sink` and the last `recent` tokens stay, and of those
// between them the budget - sink - recent with the largest weight (of equal weights the one that comes first; a NaN counts as
// larger than any number).  What stays keeps its order and moves to another cache; a row within its budget moves whole.
//
// select_kernel finds the threshold weight by radix selection (four passes of 8 bits over order-preserving integers) and
// writes the kept positions in order; gather_kernel moves the rows: codes -> values (exact: a product with a power of
// two) -> amax of the new block -> codes in the new scale.
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

constexpr int kSelectThreads = 1024;

__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictParams p) {
    __shared__ int hist[256];
    __shared__ int warp_sum[kSelectThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_total;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    int* idx = p.indices + static_cast<long long>(blockIdx.x) * p.budget;
    const int kept = len < p.budget ? len : p.budget;
    if (h == 0 && tid == 0) p.new_lens[b] = kept;
    if (len <= p.budget) {
        for (int j = tid; j < p.budget; j += kSelectThreads) idx[j] = j < len ? j : -1;
        return;
    }
    const float* w = p.weights + static_cast<long long>(blockIdx.x) * p.capacity;
    const int lo = p.sink, hi = len - p.recent;
    if (tid == 0) {
        s_prefix = 0u;
        s_need = p.budget - p.sink - p.recent;  // how many of the keys that share the prefix are kept
    }
    // a row within a budget of forced tokens alone keeps nothing between them: the threshold is never looked at
    uint32_t mask = 0u;
    for (int shift = 24; shift >= 0 && p.budget > p.sink + p.recent; shift -= 8) {
        for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int t = lo + tid; t < hi; t += kSelectThreads) {
            const uint32_t key = order_key(w[t]);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int need = s_need, d = 255;
            while (d > 0 && hist[d] < need) need -= hist[d--];
            s_need = need;
            s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
        }
        mask |= 255u << shift;
        __syncthreads();
    }
    __syncthreads();
    const uint32_t thr = s_prefix;
    const int quota = s_need;  // keys equal to the threshold that are kept, the first ones
    const bool any = p.budget > p.sink + p.recent;
    int above_before = 0, equal_before = 0;
    for (int t0 = 0; t0 < len; t0 += kSelectThreads) {
        const int t = t0 + tid;
        bool above = false, equal = false;
        if (t < len) {
            if (t < lo || t >= hi)
                above = true;
            else if (any) {
                const uint32_t key = order_key(w[t]);
                above = key > thr;
                equal = key == thr;
            }
        }
        const unsigned ba = __ballot_sync(0xffffffffu, above), be = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) warp_sum[warp] = __popc(ba) | (__popc(be) << 16);
        __syncthreads();
        if (warp == 0) {
            const int mine = warp_sum[lane];
            int v = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            warp_sum[lane] = v - mine;
            if (lane == 31) s_total = v;
        }
        __syncthreads();
        const unsigned below = (1u << lane) - 1u;
        const int a = above_before + (warp_sum[warp] & 0xffff) + __popc(ba & below);
        const int e = equal_before + (warp_sum[warp] >> 16) + __popc(be & below);
        if (above || (equal && e < quota)) idx[a + (e < quota ? e : quota)] = t;
        above_before += s_total & 0xffff;
        equal_before += s_total >> 16;
        __syncthreads();
    }
}

constexpr int kGatherThreads = 128;

template <int kFmt, int kBlock>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const EvictParams p) {
    __shared__ float warp_amax[kGatherThreads / 32];
    const int which = blockIdx.y;
    const int row = blockIdx.x / p.n_blocks_to, blk = blockIdx.x % p.n_blocks_to;
    const int h = row % p.Hkv, b = row / p.Hkv;
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    const int kept = len < p.budget ? len : p.budget;
    const int j0 = blk * kBlock;
    if (j0 >= kept) return;
    const int* idx = p.indices + static_cast<long long>(row) * p.budget;
    const uint8_t* from = p.from[which] + b * p.stride_from.batch + h * p.stride_from.head;
    uint8_t* to = p.to[which] + b * p.stride_to.batch + h * p.stride_to.head;
    const float* scale_from = p.scale_from[which] + static_cast<long long>(row) * p.n_blocks_from;
    constexpr int kRows = kGatherThreads / 16, kPasses = kBlock / kRows;
    const int r_in = threadIdx.x >> 4, c8 = (threadIdx.x & 15) * 8;
    uint2 c[kPasses];
    float s[kPasses], amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int j = j0 + i * kRows + r_in;
        c[i] = make_uint2(0u, 0u);
        s[i] = 0.f;
        if (j < kept) {
            const int t = idx[j];
            c[i] = __ldg(reinterpret_cast<const uint2*>(from + t * p.stride_from.token + c8));
            s[i] = scale_from[t >> p.block_shift];
            if (which == 0 && p.weights_to && (threadIdx.x & 15) == 0)
                p.weights_to[static_cast<long long>(row) * p.capacity_to + j] =
                    p.weights[static_cast<long long>(row) * p.capacity + t];
        }
    }
    auto values = [&](int i, float (&v)[8]) {
        decode4<kFmt>(c[i].x, *reinterpret_cast<float(*)[4]>(v));
        decode4<kFmt>(c[i].y, *reinterpret_cast<float(*)[4]>(v + 4));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= s[i];
    };
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        float v[8];
        values(i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) warp_amax[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kGatherThreads / 32; ++i) amax = fmaxf(amax, warp_amax[i]);
    const int e_new = scale_exp<kFmt>(amax);
    const float inv = exp2_int(-e_new);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int j = j0 + i * kRows + r_in;
        if (j >= kept) continue;
        float v[8];
        values(i, v);
        uint2 d;
        d.x = encode4<kFmt>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        d.y = encode4<kFmt>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint2*>(to + j * p.stride_to.token + c8) = d;
    }
    if (threadIdx.x == 0) p.scale_to[which][static_cast<long long>(row) * p.n_blocks_to + blk] = exp2_int(e_new);
}

template <int kFmt>
static void gather_dispatch(const EvictParams& p, int block, dim3 grid, cudaStream_t st) {
    switch (block) {
        case 16: gather_kernel<kFmt, 16><<<grid, kGatherThreads, 0, st>>>(p); break;
        case 32: gather_kernel<kFmt, 32><<<grid, kGatherThreads, 0, st>>>(p); break;
        case 64: gather_kernel<kFmt, 64><<<grid, kGatherThreads, 0, st>>>(p); break;
        default: gather_kernel<kFmt, 128><<<grid, kGatherThreads, 0, st>>>(p); break;
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
    if (capacity > kMaxCapacity || capacity_to > kMaxCapacity) return CLLO_E_UNSUPPORTED;
    const size_t rows = static_cast<size_t>(B) * Hkv;
    const size_t n = rows * capacity * kD, n_to = rows * capacity_to * kD;
    const size_t n_scale = rows * ((capacity + block - 1) / block) * 4, n_scale_to = rows * ((capacity_to + block - 1) / block) * 4;
    // rows move while others are still being read: the caches (and the weights) may not share memory
    if (ranges_overlap(k, n, k_to, n_to) || ranges_overlap(k, n, v_to, n_to) || ranges_overlap(v, n, k_to, n_to) ||
        ranges_overlap(v, n, v_to, n_to) ||
        ranges_overlap(k_scale, n_scale, k_scale_to, n_scale_to) || ranges_overlap(k_scale, n_scale, v_scale_to, n_scale_to) ||
        ranges_overlap(v_scale, n_scale, k_scale_to, n_scale_to) || ranges_overlap(v_scale, n_scale, v_scale_to, n_scale_to) ||
        (weights_to && ranges_overlap(weights, rows * capacity * 4, weights_to, rows * capacity_to * 4)))
        return CLLO_E_BAD_ARG;
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
    select_kernel<<<static_cast<unsigned>(rows), kSelectThreads, 0, st>>>(p);
    CLLO_CUDA_TRY(cudaGetLastError());
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    if (format == CLLO_FMT_E4M3)
        gather_dispatch<CLLO_FMT_E4M3>(p, block, grid, st);
    else
        gather_dispatch<CLLO_FMT_INT8>(p, block, grid, st);
    CLLO_CUDA_TRY(cudaGetLastError());
    return CLLO_OK;
}

}  // namespace kv8
}  // namespace cllo
