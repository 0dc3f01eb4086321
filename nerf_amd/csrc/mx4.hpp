// Microscaled 4-bit numbers: blocks of 32 values that share one power of two.
//
// A block of x has the exponent e = floor(log2 max |x|) - 2, clamped to [-127, 127], and each value is
// rounded to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times 2^e, ties to the even code, larger ones to 6.
// Stored: the code (sign, two exponent bits, one mantissa bit; the first value of a pair in the low half of a
// byte), and e + 127 in a byte; 255 stands for NaN and is what a block with an infinity or a NaN gets.
// A row of k values is ceil(k / 32) blocks, the last one filled with zeros: 16 bytes of codes and
// one of scales each.  gfx950 rounds to these codes (v_cvt_scalef32_pk_fp4_*: nearest even, saturating, a
// scale of 2^-127 included) and multiplies them with their scales on the matrix pipes.
#pragma once
#include "common.hpp"

namespace nerfx {

constexpr int MX4_BLOCK = 32;
constexpr int MX4_BLOCK_BYTES = 16;

__host__ __device__ inline int mx4_blocks(int k) { return (k + MX4_BLOCK - 1) / MX4_BLOCK; }

#ifdef __HIPCC__
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Sixteen bytes of a row of floats, which begins wherever it begins.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// N consecutive values of one block in one lane, as they are in memory (16-bit types two to a word).
template <int DT, int N>
struct Mx4Raw {
    static constexpr int WORDS = DT == NERFX_TYPE_F32 ? N : N / 2;
    uint32_t w[WORDS];

    // The exponent field a fp32 number of the largest magnitude has (0 for a subnormal one or zero; 255: inf or NaN).
    // Magnitudes are compared as integers, which also puts a NaN above all others.
    __device__ __forceinline__ uint32_t top_bits() const {
        uint32_t top = 0;
        if constexpr (DT == NERFX_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) top = max(top, w[i] & 0x7fffffffu);
        } else {
            u16x2_t t = {0, 0};
#pragma unroll
            for (int i = 0; i < WORDS; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
            top = max(t[0], t[1]);
        }
        return top;                                           // comparable between lanes of one type
    }
    // The stored scale for a block whose largest magnitude has these bits.
    static __device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
        uint32_t e;
        if constexpr (DT == NERFX_TYPE_F32) e = top >> 23;
        else if constexpr (DT == NERFX_TYPE_BF16) e = top >> 7;
        else e = top >= 0x7c00u ? 255u : __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)top)) >> 23;
        return e == 255u ? 255u : (uint32_t)max((int)e - 2, 0);
    }
    // The scale byte as the float the conversions divide by; a NaN block's codes are zeros times the sign.
    static __device__ __forceinline__ float scale_value(uint32_t byte) {
        return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255u ? 0x7f000000u : byte << 23);
    }
    // Codes of values 8 i .. 8 i + 7.
    __device__ __forceinline__ uint32_t codes(int i, float scale) const {
        uint32_t r = 0;
        if constexpr (DT == NERFX_TYPE_F32) {
#define NERFX_PAIR(s) r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __builtin_bit_cast(float, w[8 * i + 2 * s]), \
                                                                   __builtin_bit_cast(float, w[8 * i + 2 * s + 1]), scale, s)
            NERFX_PAIR(0); NERFX_PAIR(1); NERFX_PAIR(2); NERFX_PAIR(3);
#undef NERFX_PAIR
        } else if constexpr (DT == NERFX_TYPE_BF16) {
#define NERFX_PAIR(s) r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w[4 * i + s]), scale, s)
            NERFX_PAIR(0); NERFX_PAIR(1); NERFX_PAIR(2); NERFX_PAIR(3);
#undef NERFX_PAIR
        } else {
#define NERFX_PAIR(s) r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, w[4 * i + s]), scale, s)
            NERFX_PAIR(0); NERFX_PAIR(1); NERFX_PAIR(2); NERFX_PAIR(3);
#undef NERFX_PAIR
        }
        return r;
    }
};
#endif

}  // namespace nerfx
