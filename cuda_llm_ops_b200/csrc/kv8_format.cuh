// The 8-bit KV cache format: one byte per K or V value (e4m3 or a signed integer) and one fp32 scale per (batch, kv
// head, block of tokens) for K and for V.  A value is code * scale.
//
// Scales are powers of two.  For a block whose largest finite magnitude is amax the scale is the smallest 2^e with
// amax <= qmax * 2^e (qmax = 448 or 127), e held to [-60, 60].  A power of two costs an e4m3 code nothing (its three
// mantissa bits do not depend on the scale) and an integer code at most one bit, and in return
//   * x / scale is exact, so the only rounding of a stored value is the one to the code (half a step: 2^-4 relative for
//     e4m3, 1/2 scale for int8), and the code can be computed with a product instead of a quotient;
//   * when a block's scale has to grow later (an appended token, a row moved to another block) an e4m3 code moves to the
//     new scale unchanged unless it falls below the format's normal range.
// The bounds of e keep every product code * scale and every ratio of two scales inside fp32's normal range.
#pragma once

#include "common.cuh"

namespace cllo {
namespace kv8 {

constexpr int kD = 128;
constexpr int kMinScaleExp = -60, kMaxScaleExp = 60;

__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }  // 2^e, -126 <= e <= 127

// |x| of a finite x, 0 for infinities and NaN: what is not finite does not take part in a block's amax
__device__ __forceinline__ float finite_abs(float x) {
    const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
    return a < 0x7f800000u ? __uint_as_float(a) : 0.f;
}

// exponent of the block scale for a largest magnitude of amax (finite, >= 0)
template <int kFmt>
__device__ __forceinline__ int scale_exp(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = static_cast<int>(bits >> 23) - 127;  // amax = 1.f * 2^e
    const uint32_t frac = bits & 0x7fffffu;
    // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const int s = kFmt == CLLO_FMT_E4M3 ? e - 8 + (frac > 0x600000u) : e - 6 + (frac > 0x7e0000u);
    return s < kMinScaleExp ? kMinScaleExp : (s > kMaxScaleExp ? kMaxScaleExp : s);
}

// four values in units of the scale -> four codes (round to nearest even, saturating; NaN: the NaN code, or 0 as integer)
template <int kFmt>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if (kFmt == CLLO_FMT_E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    }
    auto one = [](float x) {
        const int i = __float2int_rn(x);  // saturating; 0 for NaN
        return static_cast<uint32_t>(max(-127, min(127, i))) & 0xffu;
    };
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
}

// two codes (the low or the high half of a word) -> packed f16 pair, exactly
template <int kFmt>
__device__ __forceinline__ void decode4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (kFmt == CLLO_FMT_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        // byte u = x + 128 under the exponent of 1024: 1024 + u, then minus 1152 (both exact in f16)
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    }
}

__device__ __forceinline__ void f16x2_to_f32(uint32_t h, float& lo, float& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(h));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// the larger of each half; of a number and a NaN the number
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float f16_max_of_pair(uint32_t h) {
    float lo, hi;
    f16x2_to_f32(h, lo, hi);
    return fmaxf(lo, hi);
}

template <int kFmt>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    uint32_t h[2];
    decode4_f16<kFmt>(w, h[0], h[1]);
    f16x2_to_f32(h[0], x[0], x[1]);
    f16x2_to_f32(h[1], x[2], x[3]);
}

// two f16 pairs times the f16 pair r -> four codes (round to nearest even).  The products must not pass the largest code.
template <int kFmt>
__device__ __forceinline__ uint32_t requant4(uint32_t lo, uint32_t hi, uint32_t r) {
    uint32_t d;
    if (kFmt == CLLO_FMT_E4M3) {
        asm("{\n\t.reg .b32 x, y;\n\t.reg .b16 a, b;\n\t"
            "mul.rn.f16x2 x, %1, %3;\n\tmul.rn.f16x2 y, %2, %3;\n\t"
            "cvt.rn.satfinite.e4m3x2.f16x2 a, x;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, y;\n\t"
            "mov.b32 %0, {a, b};\n\t}"
            : "=r"(d)
            : "r"(lo), "r"(hi), "r"(r));
    } else {
        // x r + 1536 in f16, whose step there is 1: rounded to an integer, which the low byte holds
        uint32_t x, y;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x) : "r"(lo), "r"(r), "r"(0x66006600u));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(hi), "r"(r), "r"(0x66006600u));
        d = __byte_perm(x, y, 0x6420);
    }
    return d;
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// asynchronous copy of one thread, global -> shared
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// element strides of a cache row (b, t, h) and its start
struct RowStrides {
    long long batch, token, head;
};
static inline RowStrides cache_strides(int kv_layout, long long capacity, long long Hkv) {
    RowStrides s;
    s.batch = capacity * Hkv * kD;
    s.token = kv_layout == CLLO_KV_BSHD ? Hkv * kD : kD;
    s.head = kv_layout == CLLO_KV_BSHD ? kD : capacity * kD;
    return s;
}

static inline bool valid_format(int format) { return format == CLLO_FMT_E4M3 || format == CLLO_FMT_INT8; }
static inline bool valid_block(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }

static inline int block_shift_of(int block) { return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7; }
constexpr int kMaxCapacity = 1 << 30;  // positions and block counts stay clear of 32-bit overflow

// a length read from device memory, held to what the cache has room for
__device__ __forceinline__ int clamp_len(int n, int capacity) { return n < 0 ? 0 : (n > capacity ? capacity : n); }

}  // namespace kv8
}  // namespace cllo
