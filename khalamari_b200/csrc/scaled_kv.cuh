// The scaled 8-bit cache formats: codes of one byte and one scale byte per (token, KV head) row, behind the codes of
// their page:
//   code of (plane, head, row, d):  page + ((plane * Hkv + head) * P + row) * D + d          plane 0 = K, 1 = V
//   scale byte of the same row:     page + 2 * Hkv * P * D + (head * 2 + plane) * P + row
// A row stands for code * 2^(b - 127). Powers of two, so that scaling a value into the codes' range, and a code back,
// rounds nothing: the only rounding is the one to the code, and int8 or E4M3 codes times 2^e are exact in bf16 as far as
// its range goes (a row of its largest value stands for 2^128, one of f16's for 2^16). b = 0:
// a row of zeros. b = 255: a row with a NaN or an infinity; its codes are zeros, and 0 * inf = NaN on the way back.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace kh {

enum CodeKind : int { kCodeInt8 = 0, kCodeE4M3 = 1 };

// 2^(b - 127); 0 for b = 0, infinity for b = 255.
__device__ __forceinline__ float scale_of_byte(uint32_t b) { return __uint_as_float(b << 23); }

// Scale byte of a row whose largest finite magnitude is `top`: the smallest exponent, -126 at least, for which
// top * 2^-e rounds into the codes' range. With top = m * 2^k, m in [1, 2): int8 needs m * 2^(k - e) < 127.5 =
// 1.9921875 * 2^6, E4M3 needs m * 2^(k - e) <= 448 = 1.75 * 2^8.
template <int CODE>
__device__ __forceinline__ uint32_t scale_byte_of(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int exponent = int(bits >> 23);  // k + 127 (0 for an f32 subnormal, which is far below 2^-126 codes anyway)
    const uint32_t mantissa = bits & 0x7fffffu;
    const int b = CODE == kCodeInt8 ? exponent - 6 + (mantissa >= 0x7f0000u ? 1 : 0)
                                    : exponent - 8 + (mantissa > 0x600000u ? 1 : 0);
    return top > 0.0f ? uint32_t(max(b, 1)) : 0u;
}

// Eight values to eight code bytes; `inverse` = 2^-e (the products are exact).
template <int CODE>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inverse) {
    uint32_t word[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if constexpr (CODE == kCodeInt8) {
            // 1.5 * 2^23 has a unit in its last place: the sum is rounded to the nearest integer, ties to even, and its low
            // byte is the integer's
            const float magic = 12582912.0f;
            const uint32_t c0 = __float_as_uint(fmaf(x[4 * w], inverse, magic)), c1 = __float_as_uint(fmaf(x[4 * w + 1], inverse, magic));
            const uint32_t c2 = __float_as_uint(fmaf(x[4 * w + 2], inverse, magic)), c3 = __float_as_uint(fmaf(x[4 * w + 3], inverse, magic));
            word[w] = __byte_perm(__byte_perm(c0, c1, 0x0040), __byte_perm(c2, c3, 0x0040), 0x5410);
        } else {
            uint16_t lo, hi;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * w + 1] * inverse), "f"(x[4 * w] * inverse));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * w + 3] * inverse), "f"(x[4 * w + 2] * inverse));
            word[w] = uint32_t(lo) | (uint32_t(hi) << 16);
        }
    }
    return make_uint2(word[0], word[1]);
}

// Four code bytes to four f16 elements, exactly: element i of the word in lane i & 1 of (i < 2 ? lo : hi).
template <int CODE>
__device__ __forceinline__ void codes4_to_half(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if constexpr (CODE == kCodeInt8) {
        // c + 128 placed in the low byte of an f16 1024 + (c + 128); minus 1152. Integers below 2048: exact.
        const uint32_t biased = word ^ 0x80808080u;
        const __half2 offset = __floats2half2_rn(1152.0f, 1152.0f);
        uint32_t a = __byte_perm(biased, 0x64646464u, 0x4140), b = __byte_perm(biased, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), offset), y = __hsub2(*reinterpret_cast<__half2*>(&b), offset);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
            : "=r"(lo), "=r"(hi) : "r"(word));
    }
}

// 2^(b - 127) as packed pairs of T, in two factors: f16 scales may lie below its smallest normal number, and the product
// of a code with the first factor is exact. Where V's byte marks a row that is not finite its codes count as zeros (the
// row's K is NaN, which is what reaches the queries that see it).
template <typename T>
__device__ __forceinline__ void scaled_factors(uint32_t b, bool v, uint32_t& first, uint32_t& second);
template <>
__device__ __forceinline__ void scaled_factors<__nv_bfloat16>(uint32_t b, bool v, uint32_t& first, uint32_t& second) {
    if (v && b == 255) b = 0;
    first = (b << 7) * 0x00010001u;
    second = 0;
}
template <>
__device__ __forceinline__ void scaled_factors<__half>(uint32_t b, bool v, uint32_t& first, uint32_t& second) {
    if (b == 255 || b == 0) {
        first = b == 0 || v ? 0u : 0x7c007c00u;
        second = 0x3c003c00u;
        return;
    }
    const int e = int(b) - 127;
    const int high = max(min(e, 15), -14), rest = max(min(e - high, 15), -24);
    first = uint32_t((high + 15) << 10) * 0x00010001u;
    // (below 2^-14 a subnormal power; scales below 2^-38 leave nothing of a code either way)
    second = (rest >= -14 ? uint32_t((rest + 15) << 10) : 1u << (rest + 24)) * 0x00010001u;
}

// The same for operands of a product (sdpa_scaled_tc.cuh): bf16 rows are taken 2^-kOperandShift times their size, so that a row
// of bf16's largest value (2^128 in codes) is finite. Rows below 2^-116 lose bits to that (their factor is subnormal).
template <typename T>
constexpr int kOperandShift = std::is_same<T, __nv_bfloat16>::value ? 10 : 0;
template <typename T>
__device__ __forceinline__ void operand_factors(uint32_t b, bool v, uint32_t& first, uint32_t& second) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        if (v && b == 255) b = 0;
        // (the upper half of an f32 power is the bf16 one)
        first = __byte_perm(__float_as_uint(__uint_as_float(b << 23) * (1.0f / (1 << kOperandShift<T>))), 0u, 0x3232);
        second = 0;
    } else {
        scaled_factors<T>(b, v, first, second);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <>
__device__ __forceinline__ uint32_t mul2<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Four codes to four elements of T, exactly, unscaled.
template <typename T, int CODE>
__device__ __forceinline__ void codes4_to(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if constexpr (std::is_same<T, __half>::value) {
        codes4_to_half<CODE>(word, lo, hi);
    } else if constexpr (CODE == kCodeInt8) {
        // bf16 has 8 significant bits: 128 + (c & 127) minus 128 (c >= 0) or 256 (c < 0), whose patterns are 0x4300 with
        // the code's low seven bits and 0x4300 with its sign bit
        const uint32_t a = __byte_perm(word, 0x43434343u, 0x4140), b = __byte_perm(word, 0x43434343u, 0x4342);
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a & 0xff7fff7fu), "r"(a & 0xff80ff80u));
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(b & 0xff7fff7fu), "r"(b & 0xff80ff80u));
    } else {
        // sign and the seven magnitude bits placed so that the code's exponent sits at the bottom of bf16's, times 2^120:
        // subnormal codes come out right too (the NaN codes as +-480: a page's codes are finite, others are masked)
        const uint32_t a = __byte_perm(word, 0u, 0x1404), b = __byte_perm(word, 0u, 0x3424);
        lo = mul2<__nv_bfloat16>((a & 0x80008000u) | ((a >> 4) & 0x07f007f0u), 0x7b807b80u);
        hi = mul2<__nv_bfloat16>((b & 0x80008000u) | ((b >> 4) & 0x07f007f0u), 0x7b807b80u);
    }
}

// Values c * 2^e of four codes as packed pairs of T, rounded once; beyond f16's largest value they become infinities.
template <typename T, int CODE>
__device__ __forceinline__ void decode4(uint32_t word, uint32_t first, uint32_t second, uint32_t& lo, uint32_t& hi) {
    codes4_to<T, CODE>(word, lo, hi);
    lo = mul2<T>(lo, first);
    hi = mul2<T>(hi, first);
    if constexpr (std::is_same<T, __half>::value) {
        lo = mul2<T>(lo, second);
        hi = mul2<T>(hi, second);
    }
}

// Infinities to the largest finite value; NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t saturate2(uint32_t v);
template <>
__device__ __forceinline__ uint32_t saturate2<__half>(uint32_t v) {
    const __half2 most = __halves2half2(__ushort_as_half(0x7bff), __ushort_as_half(0x7bff)), least = __hneg2(most);
    const __half2 cut = __hmin2_nan(__hmax2_nan(*reinterpret_cast<__half2*>(&v), least), most);
    return *reinterpret_cast<const uint32_t*>(&cut);
}
template <>
__device__ __forceinline__ uint32_t saturate2<__nv_bfloat16>(uint32_t v) {
    const __nv_bfloat162 most = __halves2bfloat162(__ushort_as_bfloat16(0x7f7f), __ushort_as_bfloat16(0x7f7f)), least = __hneg2(most);
    const __nv_bfloat162 cut = __hmin2_nan(__hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&v), least), most);
    return *reinterpret_cast<const uint32_t*>(&cut);
}
// The same in f32, at the largest value of T.
template <typename T>
__device__ __forceinline__ float saturate(float x) {
    const float most = std::is_same<T, __half>::value ? 65504.0f : __uint_as_float(0x7f7f0000u);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(most));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-most));
    return x;
}
// Statistics of a published partial: a sum of 1 under the logarithm of the whole sum (0 and -inf of a row that sees nothing),
// so that it weighs at most 1 in the merge and outputs near the type's largest value leave room for their sum. A NaN sum
// needs a finite maximum to reach the merged output, whatever its own is. `m` and the sum in the natural-log domain.
__device__ __forceinline__ void publish_partial_stats(float* partial_sum, float* partial_max, uint64_t index, float m, float sum) {
    partial_sum[index] = sum != sum ? sum : sum == 0.0f ? 0.0f : 1.0f;
    partial_max[index] = sum != sum ? 0.0f : sum == 0.0f ? -INFINITY : m + logf(sum);
}
// Scale bytes from which a code can leave T's range (codes are below 2^9).
template <typename T>
__device__ __forceinline__ constexpr uint32_t first_large_byte() { return std::is_same<T, __half>::value ? 134u : 246u; }

}  // namespace kh
