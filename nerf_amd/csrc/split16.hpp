// fp32 numbers as pairs of f16 halves, and the matrix layout the orthogonalisation's products read.
//
// v = hi + lo with hi = f16(v) and lo = f16(v - hi): 22 significand bits as long as |v| is far above
// f16's smallest step (2^-24), which the callers see to by a power-of-two scale.  A product of two such
// numbers is hi hi + hi lo + lo hi; what is left out (lo lo) and what the halves round off are both
// below 2^-22 of the product.  Three f16 matrix instructions do the work of one fp32 one at a fifth of
// its time (f16 runs at 16 times fp32's rate).
//
// Layout of an R x K matrix (K a multiple of 32): row after row, each row K / 32 blocks of 128 bytes,
// each block 32 hi halves and then 32 lo halves.
#pragma once
#include "common.hpp"

namespace nerfx {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float16_t_ __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int SPLIT_BLOCK = 32;                 // values in one block of a row
constexpr int SPLIT_BLOCK_BYTES = 128;

#ifdef __HIPCC__
__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}
// Byte address of the hi half of element (r, k); its lo half is 64 bytes on.
__device__ __forceinline__ char* split_at(char* base, int64_t r, int k, int n_cols) {
    return base + (r * (n_cols / SPLIT_BLOCK) + k / SPLIT_BLOCK) * SPLIT_BLOCK_BYTES + (k % SPLIT_BLOCK) * 2;
}
// Four values that follow each other along a row (k a multiple of 4).
__device__ __forceinline__ void split_store4(char* base, int64_t r, int k, int n_cols, const float (&v)[4]) {
    half4_t hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) { _Float16 h, l; split16(v[i], h, l); hi[i] = h; lo[i] = l; }
    char* p = split_at(base, r, k, n_cols);
    *(half4_t*)p = hi;
    *(half4_t*)(p + 64) = lo;
}
struct Split4 { half4_t hi, lo; };
#endif

}  // namespace nerfx
