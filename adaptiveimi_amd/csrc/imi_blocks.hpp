// Rows in 8 and 4 bits: codes and, for every 32 dims, a power of two.
//
// value = code * 2^(e - 127), e one byte per block, 255: NaN.  A block's power
// is the smallest with max |x| <= M 2^k (M the format's largest number), at
// least 2^-117, and code = x 2^-k to the nearest, ties to even: the scaling is
// exact, so a block is rounded once.  Powers of two, because gfx950 converts
// such codes to bf16 and fp16 in one instruction for two of them, subnormals,
// infinities and NaN included (every code with every exponent was compared);
// in bf16 the result is exact (8 significant bits at most, and 2^-117 keeps
// it normal), so reading such rows rounds nothing.
#pragma once

#include "imi_common.hpp"

namespace imi {

constexpr int kBlock = 32;      // dims that share a power

typedef __attribute__((ext_vector_type(4))) unsigned int blk_u32x4;

// 2^(e - 127), NaN for 255
__device__ __forceinline__ float block_power(uint32_t e) {
    return e == 255 ? __uint_as_float(0x7FC00000u) : __builtin_ldexpf(1.0f, static_cast<int>(e) - 127);
}

template <bool HALF>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (HALF) {
        typedef __attribute__((ext_vector_type(2))) _Float16 h2;
        return __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
    } else {
        typedef __attribute__((ext_vector_type(2))) float f2;
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
    }
}

// The formats.  kBits: of a code (16: no codes, the rows are bf16 or fp16);
// kWords: 32-bit words of 8 codes; decode: 8 codes to bf16 (fp16: HALF);
// encode: 8 scaled values to codes.  The largest number is m 2^kExp, m in
// [0.5, 1) with kLead its fraction bits in fp32; kSafe is the largest under
// 2^kSafeExp, see block_exponent.
struct Raw16 {
    static constexpr int kFormat = IMI_ROWS, kBits = 16, kWords = 4;
};
struct Fp8 {   // e4m3
    static constexpr int kFormat = IMI_FP8, kBits = 8, kWords = 2;
    static constexpr uint32_t kLead = 0x600000;   // 448 = 0.875 * 2^9
    static constexpr int kExp = 9;
    static constexpr int kSafeExp = 8;            // codes from 2^8 on
    static constexpr float kSafe = 240.0f;
    template <bool HALF>
    static __device__ __forceinline__ blk_u32x4 decode(const uint32_t (&w)[2], uint32_t e) {
        const float s = __uint_as_float(e << 23);
        blk_u32x4 r;
        if constexpr (HALF) {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], s, false));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], s, true));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], s, false));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], s, true));
        } else {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, false));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, true));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, false));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, true));
        }
        return r;
    }
    static __device__ __forceinline__ void encode(const float (&y)[8], uint32_t (&w)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int x = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
            w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], x, true);
        }
    }
};
struct Int8 {
    static constexpr int kFormat = IMI_INT8, kBits = 8, kWords = 2;
    static constexpr uint32_t kLead = 0x7E0000;   // 127 = 0.9921875 * 2^7
    static constexpr int kExp = 7;
    static constexpr int kSafeExp = 6;
    static constexpr float kSafe = 63.0f;
    template <bool HALF>
    static __device__ __forceinline__ blk_u32x4 decode(const uint32_t (&w)[2], uint32_t e) {
        const float s = block_power(e);
        blk_u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = w[i >> 1] >> (16 * (i & 1));
            r[i] = pack_pair<HALF>(static_cast<float>(static_cast<int8_t>(x)) * s,
                                   static_cast<float>(static_cast<int8_t>(x >> 8)) * s);
        }
        return r;
    }
    static __device__ __forceinline__ void encode(const float (&y)[8], uint32_t (&w)[2]) {
        // next to 1.5 * 2^23 fp32 has steps of 1: the sum is rounded as wanted and
        // its low byte is the code
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(y[i] + 12582912.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0C0C0400u), 0x05040100u);
    }
};
struct Fp4 {   // e2m1, two in a byte, the lower half first
    static constexpr int kFormat = IMI_FP4, kBits = 4, kWords = 1;
    static constexpr uint32_t kLead = 0x400000;   // 6 = 0.75 * 2^3
    static constexpr int kExp = 3;
    static constexpr int kSafeExp = 2;
    static constexpr float kSafe = 3.0f;
    template <bool HALF>
    static __device__ __forceinline__ blk_u32x4 decode(const uint32_t (&w)[1], uint32_t e) {
        const float s = __uint_as_float(e << 23);
        blk_u32x4 r;
        if constexpr (HALF) {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 0));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 1));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 2));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 3));
        } else {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 0));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 1));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 2));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 3));
        }
        return r;
    }
    static __device__ __forceinline__ void encode(const float (&y)[8], uint32_t (&w)[1]) {
        uint32_t x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], 1.0f, 0);
        x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, y[2], y[3], 1.0f, 1);
        x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, y[4], y[5], 1.0f, 2);
        w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(x, y[6], y[7], 1.0f, 3);
    }
};

// A block's exponent byte from the bits of its largest magnitude (fp32):
// 2^(x - 127) <= top < 2^(x - 126) with fraction f, and M 2^k >= top is
// k = x - 126 - kExp, or one more where f is past M's.  A block never reads
// back as an infinity: k is at most the power at which codes from 2^kSafeExp on
// are past the range of bf16 (fp16: HALF), and there codes stay at kSafe (65504
// in fp16 is 255.9 * 2^8, which would round to 256 * 2^8).
template <typename C, bool HALF>
constexpr int kTopPower = (HALF ? 16 : 128) - C::kSafeExp;
template <typename C, bool HALF>
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
    if (top >= 0x7F800000u) return 255;
    const int k = static_cast<int>(top >> 23) - 126 - C::kExp + ((top & 0x7FFFFFu) > C::kLead ? 1 : 0);
    return static_cast<uint32_t>(min(max(k, -117), kTopPower<C, HALF>) + 127);
}

// 8 values to codes, given the exponent of their block.
template <typename C, bool HALF>
__device__ __forceinline__ void block_encode(const float (&y)[8], uint32_t e, uint32_t (&w)[C::kWords]) {
    float x[8];
    const float s = __uint_as_float((254 - e) << 23);   // 2^-k (255: left out below)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i] * s;
    const bool top = e >= 127 + kTopPower<C, HALF>;   // rare, 255 among them
    if (__ballot(top)) {
        const float lim = top ? C::kSafe : 1024.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = e == 255 ? 0.0f : __builtin_amdgcn_fmed3f(x[i], -lim, lim);
    }
    C::encode(x, w);
}

}  // namespace imi
