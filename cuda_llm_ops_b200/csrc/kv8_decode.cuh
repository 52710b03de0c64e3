// Single-token GQA attention over an 8-bit KV cache.
//
//   s_t = scale * q . (kscale_blk(t) * k8_t),  o = sum_t softmax(s)_t * vscale_blk(t) * v8_t,  lse = log sum_t e^(s_t)
//
// over the sequence_lens[b] tokens that the cache holds of sequence b; with `weights`, the probabilities of the step are
// added to weights[b, kv head, t], summed over the query heads of the group in a fixed order.
//
// Plain form: one block per (sequence, query head), eight warps that take tokens in turn, 4 dims per lane, private online
// softmax states merged at the end; the weights in a second kernel that forms the scores again.
#pragma once

#include "host_util.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace kv8 {

constexpr int kDecodeWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeParams {
    const __nv_bfloat16* q;
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    const int* seq_lens;
    __nv_bfloat16* o;
    float* lse;
    float* weights;  // nullable
    RowStrides stride;
    float scale_log2;
    int Hq, Hkv, G, capacity, n_blocks, block_shift;
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <int kFmt>
__device__ __forceinline__ float score_log2(const DecodeParams& p, const float (&q)[4], const uint8_t* k_row,
                                            float k_scale, int lane) {
    float x[4];
    decode4<kFmt>(__ldg(reinterpret_cast<const uint32_t*>(k_row) + lane), x);
    const float d = warp_sum(q[0] * x[0] + q[1] * x[1] + q[2] * x[2] + q[3] * x[3]);
    return d * (k_scale * p.scale_log2);
}

__device__ __forceinline__ void load_q4(const __nv_bfloat16* q, int lane, float (&x)[4]) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(q) + lane);
    x[0] = bf16_lo(w.x);
    x[1] = bf16_hi(w.x);
    x[2] = bf16_lo(w.y);
    x[3] = bf16_hi(w.y);
}

template <int kFmt>
__global__ void __launch_bounds__(kDecodeWarps * 32) decode_kernel(const DecodeParams p) {
    __shared__ float sm[kDecodeWarps], sl[kDecodeWarps], so[kDecodeWarps][kD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hq = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, h = hq / p.G;
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    const long long base = b * p.stride.batch + h * p.stride.head;
    const float* ks = p.k_scale + (static_cast<long long>(b) * p.Hkv + h) * p.n_blocks;
    const float* vs = p.v_scale + (static_cast<long long>(b) * p.Hkv + h) * p.n_blocks;
    float q[4];
    load_q4(p.q + (static_cast<long long>(b) * p.Hq + hq) * kD, lane, q);
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = warp; t < len; t += kDecodeWarps) {
        const float s = score_log2<kFmt>(p, q, p.k + base + t * p.stride.token, ks[t >> p.block_shift], lane);
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.f : mn;  // a NaN score passes through the exponential
        const float keep = fast_exp2(m - ref), e = fast_exp2(s - ref);
        float x[4];
        decode4<kFmt>(__ldg(reinterpret_cast<const uint32_t*>(p.v + base + t * p.stride.token) + lane), x);
        const float w = e * vs[t >> p.block_shift];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = acc[i] * keep + w * x[i];
        l = l * keep + e;
        m = mn;
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) so[warp][lane * 4 + i] = acc[i];
    __syncthreads();
    if (threadIdx.x >= kD) return;
    float mm = -INFINITY, ll = 0.f, o = 0.f;
    for (int w = 0; w < kDecodeWarps; ++w) mm = fmaxf(mm, sm[w]);
    for (int w = 0; w < kDecodeWarps; ++w) {
        const float f = sl[w] == 0.f ? 0.f : fast_exp2(sm[w] - mm);
        ll += f * sl[w];
        o += f * so[w][threadIdx.x];
    }
    const long long row = static_cast<long long>(b) * p.Hq + hq;
    p.o[row * kD + threadIdx.x] = __float2bfloat16(ll == 0.f ? 0.f : o / ll);
    if (p.lse && threadIdx.x == 0) p.lse[row] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
}

// weights[b, h, t] += sum over the group's heads of e^(s_t - lse); one warp per token
template <int kFmt>
__global__ void __launch_bounds__(256) decode_weights_kernel(const DecodeParams p, int B) {
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
    const int len = clamp_len(p.seq_lens[b], p.capacity);
    const float* ks = p.k_scale + (static_cast<long long>(b) * p.Hkv + h) * p.n_blocks;
    for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < len; t += gridDim.x * 8) {
        float sum = 0.f;
        for (int g = 0; g < p.G; ++g) {
            const long long row = static_cast<long long>(b) * p.Hq + h * p.G + g;
            float q[4];
            load_q4(p.q + row * kD, lane, q);
            const float s = score_log2<kFmt>(p, q, p.k + b * p.stride.batch + h * p.stride.head + t * p.stride.token,
                                             ks[t >> p.block_shift], lane);
            sum += fast_exp2(s - p.lse[row] * kLog2e);
        }
        if (lane == 0) p.weights[(static_cast<long long>(b) * p.Hkv + h) * p.capacity + t] += sum;
    }
}

static size_t decode_workspace_bytes(int B, int capacity, int Hq, int Hkv, int D, int with_weights) {
    if (B <= 0 || capacity <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D != kD) return 0;
    return with_weights ? static_cast<size_t>(B) * Hq * sizeof(float) : 256;
}

static int decode_launch(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale,
                         const int* seq_lens, float scale, void* o, float* lse, float* weights, void* workspace,
                         size_t workspace_bytes, int B, int capacity, int Hq, int Hkv, int D, int kv_layout, int block,
                         int format, int num_workers, cudaStream_t st) {
    if (!q || !k || !v || !k_scale || !v_scale || !seq_lens || !o) return CLLO_E_BAD_ARG;
    if (B <= 0 || capacity <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return CLLO_E_BAD_ARG;
    if (kv_layout != CLLO_KV_BSHD && kv_layout != CLLO_KV_BHSD) return CLLO_E_BAD_ARG;
    if (!valid_format(format) || !valid_block(block)) return CLLO_E_BAD_ARG;
    if (!isfinite(scale) || num_workers < 0) return CLLO_E_BAD_ARG;
    if (D != kD || capacity > kMaxCapacity) return CLLO_E_UNSUPPORTED;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(o, 16)) return CLLO_E_BAD_ARG;
    const size_t need = decode_workspace_bytes(B, capacity, Hq, Hkv, D, weights != nullptr);
    if (!workspace || workspace_bytes < need || !aligned_to(workspace, 256)) return CLLO_E_WORKSPACE;
    if (static_cast<long long>(B) * Hq > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;
    DeviceInfo* di = nullptr;
    int rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    DecodeParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const uint8_t*>(k);
    p.v = static_cast<const uint8_t*>(v);
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.seq_lens = seq_lens;
    p.o = static_cast<__nv_bfloat16*>(o);
    p.lse = lse ? lse : (weights ? static_cast<float*>(workspace) : nullptr);
    p.weights = weights;
    p.stride = cache_strides(kv_layout, capacity, Hkv);
    p.scale_log2 = scale * kLog2e;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.capacity = capacity;
    p.n_blocks = (capacity + block - 1) / block;
    p.block_shift = block_shift_of(block);
    const bool fp8 = format == CLLO_FMT_E4M3;
    (fp8 ? decode_kernel<CLLO_FMT_E4M3> : decode_kernel<CLLO_FMT_INT8>)<<<B * Hq, kDecodeWarps * 32, 0, st>>>(p);
    CLLO_CUDA_TRY(cudaGetLastError());
    if (weights) {
        if (static_cast<long long>(B) * Hkv > 65535) return CLLO_E_UNSUPPORTED;
        const int gx = (capacity + 7) / 8 < 512 ? (capacity + 7) / 8 : 512;
        (fp8 ? decode_weights_kernel<CLLO_FMT_E4M3> : decode_weights_kernel<CLLO_FMT_INT8>)<<<dim3(gx, B * Hkv), 256, 0, st>>>(p, B);
        CLLO_CUDA_TRY(cudaGetLastError());
    }
    return CLLO_OK;
}

}  // namespace kv8
}  // namespace cllo
