// Append to the 8-bit KV cache: bf16 K/V rows -> codes and block scales.
//
// One thread block handles consecutive cache blocks of one (batch, kv head, K or V).  Of a cache block's rows some may be
// old (the sequence ended inside it), some are new, the rest lie behind the sequence and are left alone:
//     scale' = max(scale of the old rows, 2^e(amax of the new rows)),   code = rne(x / scale'),
// and the old rows are re-rounded to scale' only if it grew.  The scale is that of format kv8_format.cuh: powers of two,
// so x / scale' is a product and exact.
//
// Bound by memory: 2 B read and 1 B written per value.  The new rows are loaded once, 16 bytes per lane (half a warp per
// row), and wait in registers for the block's amax, while the next cache block's rows are already on their way: 4 prompts of
// 16384 tokens, 8 kv heads, e4m3: 74 us per call, 5.5 TB/s (0.83 of a copy); 69 us in a graph.  int8 81 us in a graph, 0.75: a
// code takes a conversion, two bounds and its place in the word, where e4m3 has one instruction for two; lengths that
// differ cost nothing (16 sequences of 0 to 8192 tokens 85 us, of 4096 each 85).  One token each for 60 sequences: 5 us in a graph,
// the latency of lengths, rows and two barriers; 11 per call, the host.
#pragma once

#include "host_util.cuh"
#include "kv8_format.cuh"

namespace cllo {
namespace kv8 {

constexpr int kAppendThreads = 128;
constexpr int kRowsPerPass = kAppendThreads / 16;  // half a warp per row

struct AppendParams {
    const __nv_bfloat16* src[2];  // K rows, V rows
    RowStrides src_stride[2];
    uint8_t* cache[2];
    float* scale[2];  // [B, Hkv, n_blocks]
    RowStrides stride;
    const int* seq_lens;
    const int* new_lens;  // nullable
    int T, capacity, Hkv, n_blocks, blocks_touched, per_cta;
};

template <int kFmt, int kBlock>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
    __shared__ float warp_amax[2][kAppendThreads / 32];
    const int which = blockIdx.y;
    const int ctas = (p.blocks_touched + p.per_cta - 1) / p.per_cta;  // of a (batch, kv head)
    // kv heads next to each other: with tokens before heads in memory they share DRAM pages
    const int h = blockIdx.x % p.Hkv, at = blockIdx.x / p.Hkv;
    const int b = at / ctas, first = (at % ctas) * p.per_cta, row = b * p.Hkv + h;
    const int held = clamp_len(__ldg(p.seq_lens + b), p.capacity);
    int n = p.new_lens ? clamp_len(__ldg(p.new_lens + b), p.T) : p.T;
    if (n > p.capacity - held) n = p.capacity - held;
    if (n <= 0) return;
    const int end = held + n;
    int blk = held / kBlock + first;
    const int blk_end = first + p.per_cta < p.blocks_touched ? blk + p.per_cta : blk + p.blocks_touched - first;

    const int r_in = threadIdx.x >> 4, c8 = (threadIdx.x & 15) * 8;
    const long long src_token = p.src_stride[which].token;
    const __nv_bfloat16* src = p.src[which] + b * p.src_stride[which].batch + h * p.src_stride[which].head + c8;
    uint8_t* dst = p.cache[which] + b * p.stride.batch + h * p.stride.head + c8;
    float* scales = p.scale[which] + static_cast<long long>(row) * p.n_blocks;

    constexpr int kPasses = kBlock / kRowsPerPass;
    // the next block's rows are on their way while this one's are turned into codes
    uint4 next[kPasses];
    auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int pos = at * kBlock + i * kRowsPerPass + r_in;
            next[i] = make_uint4(0u, 0u, 0u, 0u);
            if (pos >= held && pos < end) next[i] = __ldg(reinterpret_cast<const uint4*>(src + (pos - held) * src_token));
        }
    };
    if (blk * kBlock < end) fetch(blk);
#pragma unroll 1
    for (; blk < blk_end && blk * kBlock < end; ++blk) {
        const int row0 = blk * kBlock, buf = blk & 1;
        uint4 x[kPasses];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) x[i] = next[i];
        const bool has_old = row0 < held;
        const float old_scale = has_old ? scales[blk] : 0.f;
        if (blk + 1 < blk_end && row0 + kBlock < end) fetch(blk + 1);
        // the largest magnitude of the new rows, as bf16 bits; infinities and NaN, which do not take part, lie above all numbers
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
            top = max_u16x2(max_u16x2(top, max_u16x2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu)),
                            max_u16x2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
        float amax = fmaxf(finite_abs(bf16_lo(top)), finite_abs(bf16_hi(top)));
        if ((top & 0x7fffu) >= 0x7f80u || (top >> 16) >= 0x7f80u) {
            amax = 0.f;
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(finite_abs(bf16_lo(w[e])), finite_abs(bf16_hi(w[e]))));
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) warp_amax[buf][threadIdx.x >> 5] = amax;
        __syncthreads();  // also: every thread has read the old scale before one of them writes the new one
#pragma unroll
        for (int i = 0; i < kAppendThreads / 32; ++i) amax = fmaxf(amax, warp_amax[buf][i]);
        const int e_new = scale_exp<kFmt>(amax);
        float s = exp2_int(e_new), inv = exp2_int(-e_new);
        if (has_old && old_scale >= s) {
            s = old_scale;
            inv = 1.f / old_scale;
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int pos = row0 + i * kRowsPerPass + r_in;
            uint2* at = reinterpret_cast<uint2*>(dst + pos * p.stride.token);
            if (pos >= held && pos < end) {
                const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint2 c;
                c.x = encode4<kFmt>(bf16_lo(w[0]) * inv, bf16_hi(w[0]) * inv, bf16_lo(w[1]) * inv, bf16_hi(w[1]) * inv);
                c.y = encode4<kFmt>(bf16_lo(w[2]) * inv, bf16_hi(w[2]) * inv, bf16_lo(w[3]) * inv, bf16_hi(w[3]) * inv);
                *at = c;
            } else if (has_old && pos < held && s != old_scale) {
                const uint2 c = *at;
                const float ratio = old_scale * inv;
                float v[8];
                decode4<kFmt>(c.x, *reinterpret_cast<float(*)[4]>(v));
                decode4<kFmt>(c.y, *reinterpret_cast<float(*)[4]>(v + 4));
                uint2 d;
                d.x = encode4<kFmt>(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
                d.y = encode4<kFmt>(v[4] * ratio, v[5] * ratio, v[6] * ratio, v[7] * ratio);
                *at = d;
            }
        }
        if (threadIdx.x == 0) scales[blk] = s;
    }
}

template <int kFmt>
static void append_dispatch(const AppendParams& p, int block, dim3 grid, cudaStream_t st) {
    switch (block) {
        case 16: append_kernel<kFmt, 16><<<grid, kAppendThreads, 0, st>>>(p); break;
        case 32: append_kernel<kFmt, 32><<<grid, kAppendThreads, 0, st>>>(p); break;
        case 64: append_kernel<kFmt, 64><<<grid, kAppendThreads, 0, st>>>(p); break;
        default: append_kernel<kFmt, 128><<<grid, kAppendThreads, 0, st>>>(p); break;
    }
}

static int append_launch(const void* k_new, const long long* k_strides, const void* v_new, const long long* v_strides,
                         const int* seq_lens, const int* new_lens, void* k_cache, void* v_cache, float* k_scale,
                         float* v_scale, int B, int T, int capacity, int Hkv, int D, int kv_layout, int block, int format,
                         cudaStream_t st) {
    if (!k_new || !v_new || !k_strides || !v_strides || !seq_lens || !k_cache || !v_cache || !k_scale || !v_scale)
        return CLLO_E_BAD_ARG;
    if (B <= 0 || T <= 0 || capacity <= 0 || Hkv <= 0 || D <= 0) return CLLO_E_BAD_ARG;
    if (kv_layout != CLLO_KV_BSHD && kv_layout != CLLO_KV_BHSD) return CLLO_E_BAD_ARG;
    if (!valid_format(format) || !valid_block(block)) return CLLO_E_BAD_ARG;
    if (D != kD || T > kMaxCapacity || capacity > kMaxCapacity) return CLLO_E_UNSUPPORTED;
    if (!aligned_to(k_new, 16) || !aligned_to(v_new, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) ||
        !aligned_to(seq_lens, 4) || !aligned_to(new_lens, 4) || !aligned_to(k_scale, 4) || !aligned_to(v_scale, 4))
        return CLLO_E_BAD_ARG;
    for (int i = 0; i < 3; ++i)
        if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return CLLO_E_BAD_ARG;  // 16-byte loads of whole rows
    DeviceInfo* di = nullptr;
    int rc = current_device_info(&di);
    if (rc != CLLO_OK) return rc;
    if (di->cc_major != 10) return CLLO_E_UNSUPPORTED;
    AppendParams p;
    p.src[0] = static_cast<const __nv_bfloat16*>(k_new);
    p.src[1] = static_cast<const __nv_bfloat16*>(v_new);
    p.src_stride[0] = {k_strides[0], k_strides[1], k_strides[2]};
    p.src_stride[1] = {v_strides[0], v_strides[1], v_strides[2]};
    p.cache[0] = static_cast<uint8_t*>(k_cache);
    p.cache[1] = static_cast<uint8_t*>(v_cache);
    p.scale[0] = k_scale;
    p.scale[1] = v_scale;
    p.stride = cache_strides(kv_layout, capacity, Hkv);
    p.seq_lens = seq_lens;
    p.new_lens = new_lens;
    p.T = T;
    p.capacity = capacity;
    p.Hkv = Hkv;
    p.n_blocks = (capacity + block - 1) / block;
    // T tokens starting anywhere inside a block reach this many blocks at most
    const int touched = (T - 1 + block - 1) / block + 1;
    p.blocks_touched = touched < p.n_blocks ? touched : p.n_blocks;
    // Cache blocks per thread block: several, one loading while the one before it is turned into codes, where there are enough
    // to fill the GPU all the same (4 prompts of 16384 tokens, in a graph: 68.4 us with up to 8, 72.9 with one each; smaller calls get
    // one).
    const long long per_cta = static_cast<long long>(B) * Hkv * p.blocks_touched * 2 / (static_cast<long long>(di->sm_count) * 16);
    p.per_cta = static_cast<int>(per_cta < 1 ? 1 : (per_cta > 8 ? 8 : per_cta));
    const long long blocks = static_cast<long long>(B) * Hkv * ((p.blocks_touched + p.per_cta - 1) / p.per_cta);
    if (blocks > 0x7fffffffLL) return CLLO_E_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    if (format == CLLO_FMT_E4M3)
        append_dispatch<CLLO_FMT_E4M3>(p, block, grid, st);
    else
        append_dispatch<CLLO_FMT_INT8>(p, block, grid, st);
    CLLO_CUDA_TRY(cudaGetLastError());
    return CLLO_OK;
}

}  // namespace kv8
}  // namespace cllo
