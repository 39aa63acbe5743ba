// The scaled 8-bit cache formats: codes of one byte and one scale byte per (token, KV head) row, behind the codes of
// their page:
//   code of (plane, head, row, d):  page + ((plane * Hkv + head) * P + row) * D + d          plane 0 = K, 1 = V
//   scale byte of the same row:     page + 2 * Hkv * P * D + (head * 2 + plane) * P + row
// A row stands for code * 2^(b - 127). Powers of two, so that scaling a value into the codes' range, and a code back,
// rounds nothing: the only rounding is the one to the code, and int8 or E4M3 codes times 2^e are exact in bf16. b = 0:
// a row of zeros. b = 255: a row with a NaN or an infinity; its codes are zeros, and 0 * inf = NaN on the way back.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

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
            const uint32_t c0 = uint32_t(__float2int_rn(x[4 * w] * inverse)), c1 = uint32_t(__float2int_rn(x[4 * w + 1] * inverse));
            const uint32_t c2 = uint32_t(__float2int_rn(x[4 * w + 2] * inverse)), c3 = uint32_t(__float2int_rn(x[4 * w + 3] * inverse));
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

}  // namespace kh
