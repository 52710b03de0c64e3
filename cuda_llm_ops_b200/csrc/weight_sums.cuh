// Attention weight sums of a prompt: how much weight its queries gave to every key.
//
//   sums[b, h, t] (+)= sum over the query heads g of kv head h and the counted queries i of
//                      e^(scale * q[b,g,i] . k[b,h,t] - lse[b,g,i])            (t <= q_start + i when causal)
//
// lse is the forward's log-sum-exp, so each term is a probability of the forward's softmax.  Keys t >= len take no part
// (len = seq_lens[b], or Skv).  Every query counts, unless the mask is causal and lengths are given: then row i, at position
// q_start + i, is a query of the same sequence and counts when that position is < len.  A window > 0 counts only the last
// `window` of them: positions >= len - window, or the last rows of q where there are no positions to go by.
//
// Plain form: a block of 256 threads owns 64 keys and walks over 64-query tiles in shared memory, 4 x 4 products a thread.
#pragma once

#include "host_util.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace sums {

constexpr int kD = 128;
constexpr int kTile = 64;
constexpr int kPitch = kD + 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSmemBytes = 2 * kTile * kPitch * 4 + kTile * 4;

struct Params {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const float* lse;
    const int* seq_lens;  // nullable
    float* out;
    float scale_log2;
    int Sq, Skv, Hq, Hkv, G, q_start, window, causal, accumulate;
};

__device__ __forceinline__ void load_tile(float* dst, const __nv_bfloat16* src, int rows) {
    for (int i = threadIdx.x; i < kTile * (kD / 2); i += blockDim.x) {
        const int r = i / (kD / 2), c = i % (kD / 2);
        const uint32_t w = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + static_cast<long long>(r) * kD) + c) : 0u;
        dst[r * kPitch + 2 * c] = kv8::bf16_lo(w);
        dst[r * kPitch + 2 * c + 1] = kv8::bf16_hi(w);
    }
}

__global__ void __launch_bounds__(256) weight_sums_kernel(const Params p) {
    extern __shared__ float sm[];
    float* sk = sm;
    float* sq = sm + kTile * kPitch;
    float* sl = sq + kTile * kPitch;
    const int h = blockIdx.y % p.Hkv, b = blockIdx.y / p.Hkv;
    const int t0 = blockIdx.x * kTile;
    int len = p.seq_lens ? kv8::clamp_len(p.seq_lens[b], p.Skv) : p.Skv;
    // counted queries: rows [i_lo, i_hi)
    long long i_hi = p.causal && p.seq_lens ? static_cast<long long>(len) - p.q_start : p.Sq;
    long long i_lo = p.window > 0 ? i_hi - p.window : 0;
    if (i_hi > p.Sq) i_hi = p.Sq;
    if (i_lo < 0) i_lo = 0;
    if (p.causal && i_lo < t0 - p.q_start) i_lo = t0 - p.q_start;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;  // keys ty*4.., queries tx*4..
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (t0 < len && i_lo < i_hi) {
        load_tile(sk, p.k + ((static_cast<long long>(b) * p.Hkv + h) * p.Skv + t0) * kD, p.Skv - t0);
        for (int g = 0; g < p.G; ++g) {
            const long long head = static_cast<long long>(b) * p.Hq + h * p.G + g;
            for (int i0 = static_cast<int>(i_lo); i0 < i_hi; i0 += kTile) {
                __syncthreads();
                load_tile(sq, p.q + (head * p.Sq + i0) * kD, static_cast<int>(i_hi) - i0);
                if (threadIdx.x < kTile)
                    sl[threadIdx.x] = i0 + static_cast<int>(threadIdx.x) < i_hi ? p.lse[head * p.Sq + i0 + threadIdx.x] * kLog2e : INFINITY;
                __syncthreads();
                float acc[4][4] = {};
                for (int d = 0; d < kD; ++d) {
                    float a[4], c[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = sk[(ty * 4 + e) * kPitch + d];
                        c[e] = sq[(tx * 4 + e) * kPitch + d];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int f = 0; f < 4; ++f) acc[e][f] += a[e] * c[f];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        const int i = i0 + tx * 4 + f;
                        const bool counts = i < i_hi && sl[tx * 4 + f] != -INFINITY &&
                                            (!p.causal || t0 + ty * 4 + e <= p.q_start + i);
                        if (counts) sum[e] += fast_exp2(acc[e][f] * p.scale_log2 - sl[tx * 4 + f]);
                    }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        for (int o = 8; o; o >>= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
        const int t = t0 + ty * 4 + e;
        if (tx == 0 && t < p.Skv) {
            float* out = p.out + (static_cast<long long>(b) * p.Hkv + h) * p.Skv + t;
            const float add = t < len ? sum[e] : 0.f;
            *out = p.accumulate ? *out + add : add;
        }
    }
}

static int launch(const void* q, const void* k, const float* lse, const int* seq_lens, float scale, int causal, int q_start,
                  int window, int accumulate, float* out, int B, int Sq, int Skv, int Hq, int Hkv, int D, cudaStream_t st) {
    if (!q || !k || !lse || !out) return CLLO_E_BAD_ARG;
    if (B <= 0 || Sq <= 0 || Skv <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || Hq % Hkv != 0) return CLLO_E_BAD_ARG;
    if (q_start < 0 || window < 0 || !isfinite(scale)) return CLLO_E_BAD_ARG;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(lse, 4) || !aligned_to(out, 4) || !aligned_to(seq_lens, 4))
        return CLLO_E_BAD_ARG;
    if (D != kD) return CLLO_E_UNSUPPORTED;
    if (static_cast<long long>(B) * Hkv > 65535 || Sq > (1 << 30) || Skv > (1 << 30) || q_start > (1 << 30))
        return CLLO_E_UNSUPPORTED;
    DeviceInfo* di = nullptr;
    int rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.lse = lse;
    p.seq_lens = seq_lens;
    p.out = out;
    p.scale_log2 = scale * kLog2e;
    p.Sq = Sq;
    p.Skv = Skv;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.q_start = q_start;
    p.window = window;
    p.causal = causal ? 1 : 0;
    p.accumulate = accumulate ? 1 : 0;
    if (!di->sums_attr_set) {
        CLLO_CUDA_TRY(cudaFuncSetAttribute(weight_sums_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        di->sums_attr_set = true;
    }
    weight_sums_kernel<<<dim3((Skv + kTile - 1) / kTile, B * Hkv), 256, kSmemBytes, st>>>(p);
    CLLO_CUDA_TRY(cudaGetLastError());
    return CLLO_OK;
}

}  // namespace sums
}  // namespace cllo
