// Microscaled 4-bit numbers (mx4.hpp): to them, back, and the product of two matrices of them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "lds_dma.hpp"
#include "mx4.hpp"
#include "split16.hpp"

namespace nerfx {

// ---- to and from -----------------------------------------------------------------------------------------------------
// Four lanes make a block, eight values each: every load and store of a wave is one run of memory, 16 bytes a lane wherever the
// row begins: the memory pipes take any address (100,000 x 300 bf16 by 301, both ways: 194 us value by value, 76 so).  Bound by memory
// (524,288 x 256 bf16: 56 us either way, 6.1 TB/s), as long as nothing but the conversion instructions touches the values: where
// rows are whole blocks the matrix is one run, and no division finds the row.

// Part `q`, N values, begins at `at` of its row; -> its place in memory, row * k + at.  RUN: k is a multiple of 32, every part
// is whole and the row is of no interest.
template <bool RUN, int N>
__device__ __forceinline__ int64_t mx4_place(uint64_t q, int k, int& at) {
    at = 0;
    if constexpr (RUN) return (int64_t)q * N;
    const uint32_t nb = mx4_blocks(k), parts = MX4_BLOCK / N;
    const uint64_t block = q / parts, row = block >> 32 ? block / nb : (uint32_t)block / nb;
    at = (int)(block - row * nb) * MX4_BLOCK + (int)(q % parts) * N;
    return (int64_t)row * k + at;
}

// N values (a multiple of 8, at most 32) from `row + at` on: all there, or zeros behind k.  ODD: 16-bit rows may begin in the middle
// of a word, where the pipes are half as fast (260,000 x 3 bf16 by 295: 51 us); read are then the words that hold a value, one more
// of them if the first begins with half of one, and moved.
template <int DT, int N, bool ODD>
__device__ __forceinline__ Mx4Raw<DT, N> mx4_load_whole(const char* row, int at) {
    constexpr int WORDS = Mx4Raw<DT, N>::WORDS;
    const char* from = row + (int64_t)at * (DT == NERFX_TYPE_F32 ? 4 : 2);
    const uint32_t half = ODD ? (uint32_t)(uintptr_t)from & 2 : 0;
    from -= half;
    Mx4Raw<DT, N> v;
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
        const u32x4_t w = *(const u32x4_any_t*)(from + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v.w[4 * i + j] = w[j];
    }
    if constexpr (ODD) {
        const uint32_t last = *(const uint32_t*)(from + 4 * WORDS - (half ? 0 : 4));
#pragma unroll
        for (int i = 0; i < WORDS; ++i) v.w[i] = __builtin_amdgcn_alignbit(i + 1 < WORDS ? v.w[i + 1] : last, v.w[i], 8 * half);
    }
    return v;
}
static bool mx4_odd(const void* x, int k, int dtype) { return dtype != NERFX_TYPE_F32 && ((k & 1) || ((uintptr_t)x & 3)); }

// A row's last values, fewer than N, are read as its last N and moved down: one by one each would be waited for.
template <int DT, int N, bool ODD>
__device__ __forceinline__ Mx4Raw<DT, N> mx4_load(const char* row, int at, int k) {
    using Raw = Mx4Raw<DT, N>;
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2;
    Raw v;
    if (at + N <= k) {
        v = mx4_load_whole<DT, N, ODD>(row, at);
    } else if (at >= k) {
#pragma unroll
        for (int i = 0; i < Raw::WORDS; ++i) v.w[i] = 0u;
    } else if (k >= N) {
        v = mx4_load_whole<DT, N, ODD>(row, k - N);
        const int down = N - k % N;                            // the same for every lane
        if (SIZE == 2 && (down & 1)) {
#pragma unroll
            for (int i = 0; i < Raw::WORDS; ++i) v.w[i] = v.w[i] >> 16 | (i + 1 < Raw::WORDS ? v.w[i + 1] << 16 : 0u);
        }
        const int words = SIZE == 2 ? down / 2 : down;
#pragma unroll
        for (int bit = 1; bit < Raw::WORDS; bit *= 2) {
            if (words & bit) {
#pragma unroll
                for (int i = 0; i < Raw::WORDS; ++i) v.w[i] = i + bit < Raw::WORDS ? v.w[i + bit] : 0u;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < Raw::WORDS; ++i) {
            if constexpr (SIZE == 4) {
                v.w[i] = at + i < k ? *(const uint32_t*)(row + (int64_t)(at + i) * 4) : 0u;
            } else {
                const uint32_t lo = at + 2 * i < k ? *(const uint16_t*)(row + (int64_t)(at + 2 * i) * 2) : 0u;
                const uint32_t hi = at + 2 * i + 1 < k ? *(const uint16_t*)(row + (int64_t)(at + 2 * i + 1) * 2) : 0u;
                v.w[i] = lo | hi << 16;
            }
        }
    }
    return v;
}

// Rows of whole blocks, one run of memory; others; others that may begin in the middle of a word.
enum { MX4_RUN, MX4_ANY, MX4_ODD };

// Part q's codes are stored, `scale(byte)` stores its block's scale.
template <int DT, int ROWS, class Scale>
__device__ __forceinline__ void mx4_quantize_part(const void* x, int64_t q, int k, uint32_t* codes, Scale scale) {
    using Raw = Mx4Raw<DT, 8>;
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2;
    int at;
    const int64_t place = mx4_place<ROWS == MX4_RUN, 8>(q, k, at);
    Raw v;
    if constexpr (ROWS == MX4_RUN) v = mx4_load_whole<DT, 8, false>((const char*)x + place * SIZE, 0);
    else v = mx4_load<DT, 8, ROWS == MX4_ODD>((const char*)x + (place - at) * SIZE, at, k);
    uint32_t top = v.top_bits();
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    const uint32_t byte = Raw::scale_byte(top);
    codes[q] = byte == 255u ? 0u : v.codes(0, Raw::scale_value(byte));
    if ((q & 3) == 0) scale((uint8_t)byte);
}

template <int DT, int ROWS>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* __restrict__ x, int64_t parts, int k,
                                                           uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < parts; q += (int64_t)gridDim.x * 256)
        mx4_quantize_part<DT, ROWS>(x, q, k, codes, [&](uint8_t byte) { scales[q >> 2] = byte; });
}

// Sixteen bytes of the result a lane: with eight fp32 values to a lane a store is half of every line it touches (400,000 x 256: 176 us).
template <int DT> constexpr int MX4_OUT = DT == NERFX_TYPE_F32 ? 4 : 8;
template <int DT, bool RUN>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const void* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             int64_t parts, int k, void* __restrict__ out) {
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2, N = MX4_OUT<DT>;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < parts; q += (int64_t)gridDim.x * 256) {
        int at;
        char* dst = (char*)out + mx4_place<RUN, N>(q, k, at) * SIZE;
        if (!RUN && at >= k) continue;
        const uint32_t byte = scales[q / (MX4_BLOCK / N)];
        const float scale = Mx4Raw<DT, 8>::scale_value(byte);
        u32x4_any_t w;
        if constexpr (DT == NERFX_TYPE_F32) {
            const uint32_t c = ((const uint16_t*)codes)[q];
            const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
            const float v[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
        } else {
            const uint32_t c = ((const uint32_t*)codes)[q];
#define NERFX_PAIR(s)                                                                                                                  \
            if constexpr (DT == NERFX_TYPE_BF16) w[s] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, s)); \
            else w[s] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, s));
            NERFX_PAIR(0) NERFX_PAIR(1) NERFX_PAIR(2) NERFX_PAIR(3)
#undef NERFX_PAIR
        }
        if (byte == 255u) w = DT == NERFX_TYPE_F32 ? 0x7fc00000u : DT == NERFX_TYPE_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
        if constexpr (RUN) {
            __builtin_nontemporal_store(w, (u32x4_any_t*)dst);
        } else if (at + N <= k) {
            *(u32x4_any_t*)dst = w;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (at + i >= k) continue;
                if constexpr (SIZE == 4) *(uint32_t*)(dst + 4 * i) = w[i];
                else *(uint16_t*)(dst + 2 * i) = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
}

// ---- the product -----------------------------------------------------------------------------------------------------
struct Mx4LinearArgs {
    const uint8_t *w, *w_scales, *x, *x_scales;
    const float* bias;
    void* y;
    uint8_t* y_scales;
    int64_t m;
    int32_t n, k, activ, y_dtype;
};

__device__ __forceinline__ float mx4_activate(float v, int activ) {
    if (activ == NERFX_ACT_RELU) return v < 0.f ? 0.f : v;
    if (activ == NERFX_ACT_LEAKY_RELU) return v < 0.f ? 0.01f * v : v;
    if (activ == NERFX_ACT_SILU) return v / (1.0f + expf(-v));
    return v;
}

typedef int i32x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8_t mx4_operand(u32x4_t c) { return {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0}; }

// One activation for 16 values: the choice is made once, not in front of each of them.
__device__ __forceinline__ void mx4_activate16(float (&v)[16], int activ) {
    auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = f(v[e]);
    };
    if (activ == NERFX_ACT_RELU) each([](float x) { return mx4_activate(x, NERFX_ACT_RELU); });
    else if (activ == NERFX_ACT_LEAKY_RELU) each([](float x) { return mx4_activate(x, NERFX_ACT_LEAKY_RELU); });
    else if (activ == NERFX_ACT_SILU) each([](float x) { return mx4_activate(x, NERFX_ACT_SILU); });
}

__device__ __forceinline__ void mx4_store(const Mx4LinearArgs& a, int64_t at, float v) {
    if (a.y_dtype == NERFX_TYPE_F32) ((float*)a.y)[at] = v;
    else if (a.y_dtype == NERFX_TYPE_BF16) ((__bf16*)a.y)[at] = (__bf16)v;
    else ((_Float16*)a.y)[at] = (_Float16)v;
}

// y from 32 x 32 accumulators (bias included) of rows m0 .. of x and, tile after tile, of neighbouring columns.  A lane holds row
// m0 + lane % 32 and, with h = lane / 32, columns n0 + 8 q + 4 h + i of it in element 4 q + i: written from there, a store would
// touch 32 rows with 32 bytes each.  So a wave collects 128 bytes of each of its rows in LDS (one tile of fp32, two of 16 bits,
// eight of blocks) and writes them as lines (524,288 x 256 by 256 x 256, bf16: 138 us without, 114 with).  Rows lie 144 bytes apart
// there: a phase's sixteen on different banks.
struct Mx4Lines {
    static constexpr int PITCH = 144, BYTES = 32 * PITCH;      // of LDS, for one wave
    // Columns that are stored from the registers (1M x 128 in blocks by 3, fp32: 16 us, 23 by way of LDS; by 8: 24 and 18).
    static constexpr int FEW = 4;
    char* lds;
    int begin = 0, end = 0;                                    // bytes of y's rows that are collected

    __device__ __forceinline__ void add(const Mx4LinearArgs& a, const float16_t_& acc, int64_t m0, int n0) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        const int64_t m = m0 + (lane & 31);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[e];
        mx4_activate16(v, a.activ);
        char* row = lds + (lane & 31) * PITCH;
        int to, row_bytes;                                     // bytes of a row that are there with this tile, and of all of it
        if (a.n <= FEW && a.y_dtype != NERFX_TYPE_MX4) {       // heads: next to nothing to write
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + 8 * (e >> 2) + 4 * h + (e & 3);
                if (8 * (e >> 2) < FEW && m < a.m && n < a.n) mx4_store(a, m * a.n + n, v[e]);
            }
            return;
        } else if (a.y_dtype == NERFX_TYPE_MX4) {                     // the tile's 32 columns are a block of y
            using Raw = Mx4Raw<NERFX_TYPE_F32, 16>;
            Raw raw;
#pragma unroll
            for (int e = 0; e < 16; ++e) raw.w[e] = n0 + 8 * (e >> 2) + 4 * h + (e & 3) < a.n ? __builtin_bit_cast(uint32_t, v[e]) : 0u;
            uint32_t top = raw.top_bits();
            const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            const uint32_t byte = Raw::scale_byte(max(both[0], both[1]));
            const float scale = Raw::scale_value(byte);
            // this lane's codes are the lower (h = 0) or upper halves of the block's four words: after the exchange the lower
            // lane has all of the first two, the upper lane of the other two
            const auto half = __builtin_amdgcn_permlane32_swap(raw.codes(0, scale), raw.codes(1, scale), false, false);
            u32x2_t w = {__builtin_amdgcn_perm(half[1], half[0], 0x05040100u), __builtin_amdgcn_perm(half[1], half[0], 0x07060302u)};
            if (byte == 255u) w = {0, 0};
            if (h == 0 && m < a.m) a.y_scales[m * mx4_blocks(a.n) + n0 / MX4_BLOCK] = (uint8_t)byte;
            open(n0 / 2);
            *(u32x2_t*)(row + n0 / 2 - begin + 8 * h) = w;
            to = n0 / 2 + 16;
            row_bytes = mx4_blocks(a.n) * 16;
        } else if (a.y_dtype == NERFX_TYPE_F32) {
            open(4 * n0);
#pragma unroll
            for (int q = 0; q < 4; ++q) *(f32x4_t*)(row + 32 * q + 16 * h) = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            to = 4 * n0 + 128;
            row_bytes = 4 * a.n;
        } else {
            // two 16-bit values a word; word 2 q + p holds columns 8 q + 4 h + 2 p, + 1
            uint32_t w[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) w[p] = __builtin_bit_cast(uint32_t, (bf16x2_t){(__bf16)v[2 * p], (__bf16)v[2 * p + 1]});
            if (a.y_dtype == NERFX_TYPE_F16) {
#pragma unroll
                for (int p = 0; p < 8; ++p) w[p] = __builtin_bit_cast(uint32_t, (f16x2_t){(_Float16)v[2 * p], (_Float16)v[2 * p + 1]});
            }
            // exchange halves between lanes l and l + 32, so that one lane has 16 columns in a row: the lower lane
            // q = 0, 1 (columns 0 .. 15), the upper one q = 2, 3
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const auto r = __builtin_amdgcn_permlane32_swap(w[p], w[p + 4], false, false);
                w[p] = r[0];
                w[p + 4] = r[1];
            }
            open(2 * n0);
            *(u32x4_t*)(row + 2 * n0 - begin + 32 * h) = {w[0], w[1], w[4], w[5]};
            *(u32x4_t*)(row + 2 * n0 - begin + 32 * h + 16) = {w[2], w[3], w[6], w[7]};
            to = 2 * n0 + 64;
            row_bytes = 2 * a.n;
        }
        end = to;
        if (end - begin == 128 || end >= row_bytes) flush(a, m0, row_bytes);   // lines are there, or the rows end
    }

private:
    __device__ __forceinline__ void open(int at) { if (end == 0) begin = at; }
public:
    // Also needed behind the last tile of some columns, where they end in the middle of a row's line.
    __device__ __forceinline__ void flush(const Mx4LinearArgs& a, int64_t m0, int row_bytes) {
        const int lane = threadIdx.x & 63, at = begin + 16 * (lane & 7);
        const int there = min(end, row_bytes) - at;            // bytes of this lane's piece
        wave_lds_in_order();                                   // written by other lanes
        u32x4_t piece[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) piece[i] = *(const u32x4_t*)(lds + (8 * i + (lane >> 3)) * PITCH + 16 * (lane & 7));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + 8 * i + (lane >> 3);
            if (m < a.m && there >= 16) *(u32x4_any_t*)((char*)a.y + m * row_bytes + at) = piece[i];
        }
        if ((min(end, row_bytes) - begin) % 16 != 0) {         // rows that end in the middle of one
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                const int64_t m = m0 + 8 * i + (lane >> 3);
                const char* left = lds + (8 * i + (lane >> 3)) * PITCH + 16 * (lane & 7);
                if (m < a.m && there < 16)
                    for (int c = 0; c < there; c += 2) *(uint16_t*)((char*)a.y + m * row_bytes + at + c) = *(const uint16_t*)(left + c);
            }
        }
        wave_lds_in_order();                                   // the next tile is written there
        end = 0;
    }
    __device__ __forceinline__ void rest(const Mx4LinearArgs& a, int64_t m0) {
        if (end) flush(a, m0, a.y_dtype == NERFX_TYPE_MX4 ? mx4_blocks(a.n) * 16 : a.n * (a.y_dtype == NERFX_TYPE_F32 ? 4 : 2));
    }
};

// Scales in the order in which tiles need them: of eight blocks at a time, all rows.  Behind a row's end 127, a number.
constexpr int MX4_STAGE = 8;                                   // blocks
__host__ __device__ inline int mx4_stages(int nb) { return (nb + MX4_STAGE - 1) / MX4_STAGE; }
__host__ __device__ inline int64_t mx4_ordered_bytes(int64_t rows) { return (rows + 1) / 2 * 2 * MX4_STAGE; }    // of one stage

__device__ __forceinline__ void mx4_order_scales(const uint8_t* __restrict__ from, int64_t rows, int nb, uint8_t* __restrict__ to,
                                                 int64_t first, int64_t step) {
    const int stages = mx4_stages(nb);
    for (int64_t i = first; i < rows * stages; i += step) {
        const int64_t row = i / stages;
        const int st = (int)(i - row * stages), there = nb - st * MX4_STAGE;
        const uint8_t* src = from + row * nb + st * MX4_STAGE;
        u32x2_t v = {0x7f7f7f7fu, 0x7f7f7f7fu};
        if (there >= MX4_STAGE) {
            __builtin_memcpy(&v, src, 8);
        } else {
#pragma unroll
            for (int b = 0; b < MX4_STAGE; ++b)
                if (b < there) v[b / 4] = (v[b / 4] & ~(255u << (8 * (b % 4)))) | (uint32_t)src[b] << (8 * (b % 4));
        }
        *(u32x2_t*)(to + st * mx4_ordered_bytes(rows) + row * MX4_STAGE) = v;
    }
}

// What a product in tiles needs beforehand, in one launch: the first `w_groups` workgroups order W's scales, the others quantise x
// with its scales in order (or, if x is quantised, order those).
struct Mx4PrepareArgs {
    const void* x;
    const uint8_t *x_scales, *w_scales;
    uint32_t* codes;
    uint8_t *x_ordered, *w_ordered;
    int64_t m;
    int32_t n, k, w_groups;
};
template <int DT, int ROWS>
__global__ __launch_bounds__(256) void mx4_prepare_kernel(const Mx4PrepareArgs a) {
    const int nb = mx4_blocks(a.k);
    if ((int)blockIdx.x < a.w_groups) {
        mx4_order_scales(a.w_scales, a.n, nb, a.w_ordered, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)a.w_groups * 256);
        return;
    }
    const int64_t first = (int64_t)(blockIdx.x - a.w_groups) * 256 + threadIdx.x, step = (int64_t)(gridDim.x - a.w_groups) * 256;
    if constexpr (DT == NERFX_TYPE_MX4) {
        mx4_order_scales(a.x_scales, a.m, nb, a.x_ordered, first, step);
    } else {
        const int64_t parts = a.m * nb * 4, stage_bytes = mx4_ordered_bytes(a.m);
        for (int64_t q = first; q < parts; q += step)
            mx4_quantize_part<DT, ROWS>(a.x, q, a.k, a.codes, [&](uint8_t byte) {
                const uint64_t block = (uint64_t)q >> 2, row = block >> 32 ? block / nb : (uint32_t)block / nb;
                const int b = (int)(block - row * nb);
                uint8_t* to = a.x_ordered + b / MX4_STAGE * stage_bytes + row * MX4_STAGE;
                to[b % MX4_STAGE] = byte;
                if (b == nb - 1)
                    for (int i = b % MX4_STAGE + 1; i < MX4_STAGE; ++i) to[i] = 127;
            });
    }
}

// A (32 FP WP) x (32 FQ WQ) tile of W x^T per workgroup of WP x WQ waves.  A stage is eight blocks (256 values) of every
// row of both operands, 128 bytes a row, brought by LDS-DMA while the S - 1 stages before are worked on; block c of row r lies
// at place c ^ (r / 2 % 8), so that the sixteen rows of a read phase touch different banks.  The stage's scales, eight bytes a row,
// come the same way, from scales put in order beforehand: as they are given every row's few bytes are a request of their own
// (4096 x 4096 by 8192, x in blocks: 93 us by way of registers, 85 so, 3 of them for the order).  Fragments are read one step (64
// values) ahead of their use.  Rows behind the last one and blocks behind a row's end are read from the last ones: the results of
// the former are not stored, the codes of the latter are cleared on one side.
// Bound by its loads: for 4096 x 4096 results 4,096 more of K take 34 us in tiles of 256; 22 of these are the products (6.2 PFLOP/s,
// all that the instructions do by themselves), without loads it is 25.  LDS holds two stages of that tile; four of 128 x 128 in
// their place change nothing.
template <int FP, int WP, int FQ, int WQ, int S>
struct Mx4Tile {
    static constexpr int WAVES = WP * WQ, TP = 32 * FP * WP, TQ = 32 * FQ * WQ, STAGES = S;
    static constexpr int ROW_BYTES = MX4_STAGE * MX4_BLOCK_BYTES, STAGE_BYTES = (TP + TQ) * ROW_BYTES, SCALE_BYTES = (TP + TQ) * MX4_STAGE;
    static constexpr int SCALES_AT = STAGES * STAGE_BYTES, BIAS_AT = SCALES_AT + STAGES * SCALE_BYTES, LDS_BYTES = BIAS_AT + 4 * TP;
    static constexpr int LOADS_P = TP / (8 * WAVES), LOADS_Q = TQ / (8 * WAVES), LOADS = LOADS_P + LOADS_Q;    // of a wave and stage
    static constexpr int SCALE_WAVES = SCALE_BYTES / 1024;     // waves that have one more, for scales
    static_assert(TP % (8 * WAVES) == 0 && TQ % (8 * WAVES) == 0 && WAVES % 2 == 0 && SCALE_BYTES % 1024 == 0 && SCALE_WAVES <= WAVES &&
                  LDS_BYTES <= 160 * 1024, "whole loads per wave");

    struct Frags { u32x4_t p[FP], q[FQ]; };
    // step s of the stage in `buf`
    static __device__ __forceinline__ void read(Frags& f, const char* buf, int s, int p_row, int q_row, int h) {
        auto frag = [&](int row) { return *(const u32x4_t*)(buf + row * ROW_BYTES + (((2 * s + h) ^ (row >> 1 & 7)) * 16)); };
#pragma unroll
        for (int i = 0; i < FP; ++i) f.p[i] = frag(p_row + 32 * i);
#pragma unroll
        for (int j = 0; j < FQ; ++j) f.q[j] = frag(q_row + 32 * j);
        __builtin_amdgcn_sched_barrier(0);                     // in front of the products of the step before, not behind them
    }
    // Of a row in a stage: those of blocks 2 s + h, one a byte.
    static __device__ __forceinline__ uint32_t scales(const char* stage, int row, int h) {
        const u32x2_t v = *(const u32x2_t*)(stage + row * MX4_STAGE);
        return __builtin_amdgcn_perm(v[1], v[0], h ? 0x07050301u : 0x06040200u);
    }
};

template <int FP, int WP, int FQ, int WQ, int S>
__global__ __launch_bounds__(64 * WP * WQ) void mx4_tile_kernel(const Mx4LinearArgs a) {
    using T = Mx4Tile<FP, WP, FQ, WQ, S>;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int nb = mx4_blocks(a.k), stages = mx4_stages(nb);
    int m_tile, n_tile;
    band_at(xcd_place(), (int)((a.m + T::TQ - 1) / T::TQ), (a.n + T::TP - 1) / T::TP, m_tile, n_tile);
    const int n0 = n_tile * T::TP;
    const int64_t m0 = (int64_t)m_tile * T::TQ;
    const int wp = wave / WQ * 32 * FP, wq = wave % WQ * 32 * FQ;
    const uint32_t pitch = (uint32_t)nb * MX4_BLOCK_BYTES, lds0 = lds_address(lds);
    const char *P = (const char*)a.w + (int64_t)n0 * pitch, *Q = (const char*)a.x + m0 * pitch;
    const int p_last = a.n - 1 - n0, q_last = (int)min((int64_t)T::TQ, a.m - m0) - 1;     // last row that is there
    // this lane's part of a stage: one block of some rows
    const int my_row = 8 * wave + (lane >> 3), my_block = (lane & 7) ^ (my_row >> 1 & 7);
    uint32_t p_at[T::LOADS_P], q_at[T::LOADS_Q];
#pragma unroll
    for (int i = 0; i < T::LOADS_P; ++i) p_at[i] = (uint32_t)min(my_row + 8 * T::WAVES * i, p_last) * pitch;
#pragma unroll
    for (int i = 0; i < T::LOADS_Q; ++i) q_at[i] = (uint32_t)min(my_row + 8 * T::WAVES * i, q_last) * pitch;
    // and two rows' scales, of the stage that is fetched next
    const int scale_row = 128 * wave + 2 * lane;
    const int64_t scale_step = mx4_ordered_bytes(scale_row < T::TP ? a.n : a.m);
    const char* scale_from = scale_row < T::TP ? (const char*)a.w_scales + (int64_t)(n0 + min(scale_row, p_last & ~1)) * MX4_STAGE
                                               : (const char*)a.x_scales + (m0 + min(scale_row - T::TP, q_last & ~1)) * MX4_STAGE;
    auto fetch = [&](int st) {
        if (wave < T::SCALE_WAVES) dma16(lds0 + T::SCALES_AT + (uint32_t)(st % T::STAGES) * T::SCALE_BYTES + wave * 1024, scale_from);
        scale_from += scale_step;
        const uint32_t to = lds0 + (uint32_t)(st % T::STAGES) * T::STAGE_BYTES + wave * 1024;
        const uint32_t block = (uint32_t)min(st * 8 + my_block, nb - 1) * MX4_BLOCK_BYTES;
#pragma unroll
        for (int i = 0; i < T::LOADS_P; ++i) dma16(to + i * T::WAVES * 1024, P, p_at[i] + block);
#pragma unroll
        for (int i = 0; i < T::LOADS_Q; ++i) dma16(to + T::TP * T::ROW_BYTES + i * T::WAVES * 1024, Q, q_at[i] + block);
    };
    const int p_row = wp + (lane & 31), q_row = T::TP + wq + (lane & 31);
    uint32_t sp[FP], sq[FQ];
    auto take_scales = [&](int st) {
        const char* stage = lds + T::SCALES_AT + st % T::STAGES * T::SCALE_BYTES;
#pragma unroll
        for (int i = 0; i < FP; ++i) sp[i] = T::scales(stage, p_row + 32 * i, h);
#pragma unroll
        for (int j = 0; j < FQ; ++j) sq[j] = T::scales(stage, q_row + 32 * j, h);
    };
    float16_t_ acc[FP][FQ];
    auto multiply = [&](const typename T::Frags& f, auto step) {
        constexpr int s = decltype(step)::value;
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(f.p[i]), mx4_operand(f.q[j]), acc[i][j], 4, 4,
                                                                           s, (int)sp[i], s, (int)sq[j]);
    };
    using S0 = std::integral_constant<int, 0>; using S1 = std::integral_constant<int, 1>;
    using S2 = std::integral_constant<int, 2>; using S3 = std::integral_constant<int, 3>;
    typename T::Frags f0, f1;
    float* bias_lds = (float*)(lds + T::BIAS_AT);
    for (int c = threadIdx.x; c < T::TP; c += 64 * T::WAVES) bias_lds[c] = a.bias && c <= p_last ? a.bias[n0 + c] : 0.f;
    for (int st = 0; st < min(S, stages); ++st) fetch(st);
    landed<0>();
#pragma unroll
    for (int i = 0; i < FP; ++i)                               // sums begin as the bias, in the other kernel as here: the same results
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4_t b = *(const f32x4_t*)(bias_lds + wp + 32 * i + 8 * q + 4 * h);
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = b[e];
        }
    take_scales(0);
    T::read(f0, lds, 0, p_row, q_row, h);
    for (int st = 0; st < stages - 1; ++st) {
        const char* buf = lds + (st % T::STAGES) * T::STAGE_BYTES;
        T::read(f1, buf, 1, p_row, q_row, h);
        multiply(f0, S0{});
        T::read(f0, buf, 2, p_row, q_row, h);
        multiply(f1, S1{});
        T::read(f1, buf, 3, p_row, q_row, h);
        multiply(f0, S2{});
        // the next stage is there, and every wave has read all of this one
        if (S == 2 || st + S > stages) landed<0>();
        else if (wave < T::SCALE_WAVES) landed<(S - 2) * (T::LOADS + 1)>();
        else landed<(S - 2) * T::LOADS>();
        if (st + S < stages) fetch(st + S);
        T::read(f0, lds + ((st + 1) % T::STAGES) * T::STAGE_BYTES, 0, p_row, q_row, h);
        multiply(f1, S3{});
        take_scales(st + 1);
    }
    const char* buf = lds + ((stages - 1) % T::STAGES) * T::STAGE_BYTES;
    const int left = nb - 8 * (stages - 1);                    // blocks of the last stage
    auto clear = [&](typename T::Frags& f, int s) {
        if (2 * s + h >= left)
#pragma unroll
            for (int i = 0; i < FP; ++i) f.p[i] = {0, 0, 0, 0};
    };
    clear(f0, 0);
    T::read(f1, buf, 1, p_row, q_row, h);
    multiply(f0, S0{});
    if (left > 2) {
        clear(f1, 1);
        multiply(f1, S1{});
    }
    if (left > 4) {
        T::read(f0, buf, 2, p_row, q_row, h);
        T::read(f1, buf, 3, p_row, q_row, h);
        clear(f0, 2);
        multiply(f0, S2{});
        if (left > 6) {
            clear(f1, 3);
            multiply(f1, S3{});
        }
    }
    __syncthreads();                                           // the stages have been read: their place is the waves' own now
    Mx4Lines lines{lds + wave * Mx4Lines::BYTES};
    static_assert(T::WAVES * Mx4Lines::BYTES <= T::LDS_BYTES, "a place for each wave");
#pragma unroll
    for (int j = 0; j < FQ; ++j) {
#pragma unroll
        for (int i = 0; i < FP; ++i) {
            const int n = n0 + wp + 32 * i;
            if (n >= a.n) break;
            lines.add(a, acc[i][j], m0 + wq + 32 * j, n);
        }
        lines.rest(a, m0 + wq + 32 * j);
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------------------
// Up to 64 rows of x: the weight is read once and nothing else counts.  A workgroup takes 16 rows of W, its waves parts
// of K; each lane's 16-byte load is a block of W, which is an operand of the matrix instruction as it
// is (16 x 16 x 128).  Rows of x in a float type are quantised by the workgroup into LDS, a block a thread, while the first
// loads of W are on their way (one row by 4096 x 4096: 5.2 us a call in a captured graph; a launch
// behind another is 1.5 of it and 9 MB at 5 TB/s are 2).
constexpr int SKINNY_ROWS = 64, SKINNY_WAVES = 8, SKINNY_AHEAD = 4, SKINNY_LDS = 64 * 1024, SKINNY_FLOATS = 128 * 1024;

__device__ __forceinline__ void mx4_store_one(const Mx4LinearArgs& a, int64_t m, int n, float acc) {
    mx4_store(a, m * a.n + n, mx4_activate(acc + (a.bias ? a.bias[n] : 0.f), a.activ));
}

template <int DT, int MT>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void mx4_skinny_kernel(const Mx4LinearArgs a) {
    extern __shared__ __align__(16) char lds[];
    constexpr bool FLOAT = DT != NERFX_TYPE_MX4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const int nb = mx4_blocks(a.k), m = (int)a.m;
    const int n0 = blockIdx.x * 16, row = min(n0 + l16, a.n - 1);
    const int steps = (nb + 3) / 4, per = (steps + SKINNY_WAVES - 1) / SKINNY_WAVES;
    const int first = min(wave * per, steps), last = min(first + per, steps);
    const u32x4_t* w = (const u32x4_t*)a.w + (int64_t)row * nb;
    const uint8_t* ws = a.w_scales + (int64_t)row * nb;
    u32x4_t wc[SKINNY_AHEAD];
    uint32_t wsc[SKINNY_AHEAD];
    auto fetch = [&](int step, u32x4_t& c, uint32_t& s) {
        const int b = min(4 * step + g, nb - 1);               // behind the last block x has zeros
        c = __builtin_nontemporal_load(w + b);
        s = ws[b];
    };
#pragma unroll
    for (int u = 0; u < SKINNY_AHEAD; ++u)
        if (first + u < last) fetch(first + u, wc[u], wsc[u]);
    if constexpr (FLOAT) {
        using Raw = Mx4Raw<DT, 32>;
        for (int q = threadIdx.x; q < m * nb; q += 64 * SKINNY_WAVES) {
            const int r = q / nb, b = q - r * nb;
            const Raw v = mx4_load<DT, 32, false>((const char*)a.x + (int64_t)r * a.k * (DT == NERFX_TYPE_F32 ? 4 : 2), b * 32, a.k);
            const uint32_t byte = Raw::scale_byte(v.top_bits());
            const float scale = Raw::scale_value(byte);
            *(u32x4_t*)(lds + q * 16) = {v.codes(0, scale), v.codes(1, scale), v.codes(2, scale), v.codes(3, scale)};
            *(uint8_t*)(lds + m * nb * 16 + q) = (uint8_t)byte;
        }
        __syncthreads();
    }
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = {0.f, 0.f, 0.f, 0.f};
    for (int base = first; base < last; base += SKINNY_AHEAD) {
#pragma unroll
        for (int u = 0; u < SKINNY_AHEAD; ++u) {
            const int step = base + u;
            if (step >= last) break;
            const u32x4_t c = wc[u];
            const uint32_t s = wsc[u];
            if (step + SKINNY_AHEAD < last) fetch(step + SKINNY_AHEAD, wc[u], wsc[u]);
            const int b = 4 * step + g;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int r = 16 * t + l16;
                u32x4_t xc = {0, 0, 0, 0};
                uint32_t xs = 127u;
                if (r < m && b < nb) {
                    const int q = r * nb + b;
                    if constexpr (FLOAT) {
                        xc = *(const u32x4_t*)(lds + q * 16);
                        xs = *(const uint8_t*)(lds + m * nb * 16 + q);
                    } else {
                        xc = *((const u32x4_t*)a.x + q);
                        xs = a.x_scales[q];
                    }
                }
                acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(c), mx4_operand(xc), acc[t], 4, 4, 0, (int)s, 0, (int)xs);
            }
        }
    }
    // sums of the waves' parts of K, in their order; element i of a lane: row m = lane % 16, column n = 4 (lane / 16) + i
    __syncthreads();
    f32x4_t* part = (f32x4_t*)lds;
#pragma unroll
    for (int t = 0; t < MT; ++t) part[(wave * MT + t) * 64 + lane] = acc[t];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * 64; o += 64 * SKINNY_WAVES) {
        f32x4_t sum = part[o];
#pragma unroll
        for (int v = 1; v < SKINNY_WAVES; ++v) sum += part[v * MT * 64 + o];
        const int r = 16 * (o >> 6) + (o & 15), n = n0 + 4 * ((o & 63) >> 4);
        if (r >= m) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.n) mx4_store_one(a, r, n + i, sum[i]);
    }
}

// ---- many rows, few columns ------------------------------------------------------------------------------------------
// Up to 256 columns and 512 values a row: a layer of a field for a batch of samples.  Bound by memory: x is read once, in
// whatever type it has, and y written once.  W stays in LDS (its rows (2 KS + 1) * 16 bytes apart: sixteen rows of a read on
// sixteen different banks); a wave takes 32 rows of x, a lane two blocks of every 64 values of its row, quantises them in
// registers, where they are operands of the matrix instruction as they are, and goes over W's columns (524,288 x 256 bf16 by 256:
// 112 us, 4.8 TB/s).
constexpr int STREAM_WAVES = 8;                                // at most

__host__ __device__ inline int stream_row_bytes(int ks) { return (2 * ks + 1) * 16; }
__host__ __device__ inline int stream_scale_bytes(int ks) { return ks > 4 ? 16 : 8; }      // both halves of a row
__host__ __device__ inline int stream_lds(int ks, int columns, int waves) {
    return columns * (stream_row_bytes(ks) + stream_scale_bytes(ks) + 4) + waves * Mx4Lines::BYTES;
}

template <int DT, int KS, bool ODD>
__global__ __launch_bounds__(64 * STREAM_WAVES) void mx4_stream_kernel(const Mx4LinearArgs a, int columns) {
    extern __shared__ __align__(16) char lds[];
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2, SB = KS > 4 ? 8 : 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int nb = mx4_blocks(a.k), c0 = blockIdx.y * columns;
    char* scale_lds = lds + columns * stream_row_bytes(KS);
    float* bias_lds = (float*)(scale_lds + columns * stream_scale_bytes(KS));
    char* line_lds = (char*)(bias_lds + columns) + wave * Mx4Lines::BYTES;
    const int threads = blockDim.x;
    for (int c = threadIdx.x; c < columns; c += threads) bias_lds[c] = a.bias && c0 + c < a.n ? a.bias[c0 + c] : 0.f;
    constexpr int W_AT_ONCE = 4;
    for (int first = threadIdx.x; first < columns * 2 * KS; first += W_AT_ONCE * threads) {
        u32x4_t v[W_AT_ONCE];
        uint32_t s[W_AT_ONCE];
#pragma unroll
        for (int i = 0; i < W_AT_ONCE; ++i) {
            const int c = first + i * threads, r = c / (2 * KS), b = c - r * 2 * KS;
            v[i] = {0, 0, 0, 0};
            s[i] = 127u;
            if (r < columns && c0 + r < a.n && b < nb) {
                v[i] = *((const u32x4_t*)a.w + (int64_t)(c0 + r) * nb + b);
                s[i] = a.w_scales[(int64_t)(c0 + r) * nb + b];
            }
        }
#pragma unroll
        for (int i = 0; i < W_AT_ONCE; ++i) {
            const int c = first + i * threads, r = c / (2 * KS), b = c - r * 2 * KS;
            if (r >= columns) break;
            *(u32x4_t*)(lds + r * stream_row_bytes(KS) + b * 16) = v[i];
            scale_lds[r * 2 * SB + (b & 1) * SB + (b >> 1)] = (char)s[i];
        }
    }
    __syncthreads();
    const int rows = threads >> 1;                             // 32 a wave
    for (int64_t m0 = (int64_t)blockIdx.x * rows + 32 * wave; m0 < a.m; m0 += (int64_t)gridDim.x * rows) {
        const int64_t m = min(m0 + (lane & 31), a.m - 1);
        u32x4_t xc[KS];
        uint32_t xs[(KS + 3) / 4] = {};
        if constexpr (DT == NERFX_TYPE_MX4) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                xc[s] = {0, 0, 0, 0};
                uint32_t byte = 127u;
                if (2 * s + h < nb) {
                    xc[s] = *((const u32x4_t*)a.x + m * nb + 2 * s + h);
                    byte = a.x_scales[m * nb + 2 * s + h];
                }
                xs[s / 4] |= byte << (8 * (s & 3));
            }
        } else {
            using Raw = Mx4Raw<DT, 32>;
            constexpr int AT_ONCE = DT == NERFX_TYPE_F32 ? 2 : 4;          // as many loads in flight as registers allow
            const char* row = (const char*)a.x + m * a.k * SIZE;
            const int whole = a.k / MX4_BLOCK;                             // blocks
            auto take = [&](const Raw& raw, int s) {
                const uint32_t byte = Raw::scale_byte(raw.top_bits());
                const float scale = Raw::scale_value(byte);
                xc[s] = {raw.codes(0, scale), raw.codes(1, scale), raw.codes(2, scale), raw.codes(3, scale)};
                xs[s / 4] |= byte << (8 * (s & 3));
            };
            if (whole > 0) {
#pragma unroll
                for (int s0 = 0; s0 < KS; s0 += AT_ONCE) {
                    Raw raw[AT_ONCE];
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u)                      // behind the row's last whole block: that one again
                        if (s0 + u < KS) raw[u] = mx4_load_whole<DT, 32, ODD>(row, min(2 * (s0 + u) + h, whole - 1) * MX4_BLOCK);
#pragma unroll
                    for (int u = 0; u < AT_ONCE; ++u) {
                        if (s0 + u < KS) take(raw[u], s0 + u);
                    }
                    if (KS > AT_ONCE) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (nb != 2 * KS || whole != nb) {                             // rows that end earlier: a part of a block, and zeros
                Raw tail = mx4_load<DT, 32, ODD>(row, whole * MX4_BLOCK, a.k);
                const uint32_t byte = Raw::scale_byte(tail.top_bits());
                const float scale = Raw::scale_value(byte);
                const u32x4_t codes = {tail.codes(0, scale), tail.codes(1, scale), tail.codes(2, scale), tail.codes(3, scale)};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int b = 2 * s + h;
                    if (b < whole) continue;
                    const bool part = b == whole && whole < nb;
                    xc[s] = part ? codes : (u32x4_t){0, 0, 0, 0};
                    xs[s / 4] = (xs[s / 4] & ~(255u << (8 * (s & 3)))) | (part ? byte : 127u) << (8 * (s & 3));
                }
            }
        }
        Mx4Lines lines{line_lds};
        for (int n = 0; n < columns && c0 + n < a.n; n += 32) {
            const int r = n + (lane & 31);
            const char* wr = lds + r * stream_row_bytes(KS) + h * 16;
            uint32_t ws[SB / 4];
            ws[0] = *(const uint32_t*)(scale_lds + r * 2 * SB + h * SB);
            if constexpr (SB == 8) ws[1] = *(const uint32_t*)(scale_lds + r * 2 * SB + h * SB + 4);
            float16_t_ acc;                                        // begins as the bias
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_t b = *(const f32x4_t*)(bias_lds + n + 8 * q + 4 * h);
                acc[4 * q] = b[0]; acc[4 * q + 1] = b[1]; acc[4 * q + 2] = b[2]; acc[4 * q + 3] = b[3];
            }
#define NERFX_STEP(s)                                                                                                                  \
            if constexpr (s < KS)                                                                                                      \
                acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(*(const u32x4_t*)(wr + s * 32)), mx4_operand(xc[s < KS ? s : 0]), acc, \
                                                                      4, 4, s & 3, (int)ws[s / 4 < SB / 4 ? s / 4 : 0], s & 3, (int)xs[s / 4 < (KS + 3) / 4 ? s / 4 : 0]);
            NERFX_STEP(0) NERFX_STEP(1) NERFX_STEP(2) NERFX_STEP(3) NERFX_STEP(4) NERFX_STEP(5) NERFX_STEP(6) NERFX_STEP(7)
#undef NERFX_STEP
            lines.add(a, acc, m0, c0 + n);
        }
        lines.rest(a, m0);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static dim3 mx4_grid(int64_t parts) { return dim3((unsigned)std::min<int64_t>((parts + 255) / 256, 256 * 32)); }

// f(type, rows) for a float type and how its rows lie.
template <class F>
static int mx4_by_rows(const void* x, int k, int dtype, F f) {
    using F32 = std::integral_constant<int, NERFX_TYPE_F32>; using BF16 = std::integral_constant<int, NERFX_TYPE_BF16>;
    using F16 = std::integral_constant<int, NERFX_TYPE_F16>;
    using Run = std::integral_constant<int, MX4_RUN>; using Any = std::integral_constant<int, MX4_ANY>; using Odd = std::integral_constant<int, MX4_ODD>;
    const bool odd = mx4_odd(x, k, dtype);
    if (k % MX4_BLOCK == 0) return dtype == NERFX_TYPE_F32 ? f(F32{}, Run{}) : dtype == NERFX_TYPE_BF16 ? f(BF16{}, Run{}) : f(F16{}, Run{});
    if (dtype == NERFX_TYPE_F32) return f(F32{}, Any{});
    if (dtype == NERFX_TYPE_BF16) return odd ? f(BF16{}, Odd{}) : f(BF16{}, Any{});
    return odd ? f(F16{}, Odd{}) : f(F16{}, Any{});
}

static int quantize_launch(const void* x, int dtype, int64_t rows, int k, uint8_t* codes, uint8_t* scales, hipStream_t stream) {
    const int64_t parts = rows * mx4_blocks(k) * 4;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, mx4_grid(parts), dim3(256), 0, stream, x, parts, k, (uint32_t*)codes, scales);
        return launch_status("mx4_quantize_kernel");
    };
    return mx4_by_rows(x, k, dtype, [&](auto type, auto rows) { return go(mx4_quantize_kernel<decltype(type)::value, decltype(rows)::value>); });
}

static int prepare_launch(Mx4PrepareArgs& a, int dtype, hipStream_t stream) {
    const int64_t nb = mx4_blocks(a.k), parts = dtype == NERFX_TYPE_MX4 ? a.m * mx4_stages(nb) : a.m * nb * 4;
    a.w_groups = (int)std::min<int64_t>(((int64_t)a.n * mx4_stages(nb) + 255) / 256, 256);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.w_groups + mx4_grid(parts).x), dim3(256), 0, stream, a);
        return launch_status("mx4_prepare_kernel");
    };
    if (dtype == NERFX_TYPE_MX4) return go(mx4_prepare_kernel<NERFX_TYPE_MX4, MX4_RUN>);
    return mx4_by_rows(a.x, a.k, dtype, [&](auto type, auto rows) { return go(mx4_prepare_kernel<decltype(type)::value, decltype(rows)::value>); });
}

template <int FP, int WP, int FQ, int WQ, int S>
static int tile_launch(const Mx4LinearArgs& a, hipStream_t stream) {
    using T = Mx4Tile<FP, WP, FQ, WQ, S>;
    const int64_t tiles = ((a.n + T::TP - 1) / T::TP) * ((a.m + T::TQ - 1) / T::TQ);
    NERFX_REQUIRE(tiles <= 1 << 22, "%lld x %d results are too many for one launch", (long long)a.m, a.n);
    NERFX_OPT_IN_LDS((mx4_tile_kernel<FP, WP, FQ, WQ, S>), T::LDS_BYTES);
    hipLaunchKernelGGL((mx4_tile_kernel<FP, WP, FQ, WQ, S>), dim3((unsigned)tiles), dim3(64 * T::WAVES), T::LDS_BYTES, stream, a);
    return launch_status("mx4_tile_kernel");
}

// How a product is done, by its sizes:
//  skinny  up to 64 rows of x: W is read once, by as many workgroups as it has 16 rows (one row by 4096 x 4096: 5.2 us, 10.2 with
//          tiles).  Each of them quantises float rows for itself, up to 128 KB of them (64 x 1000 fp32 by 1000: 15 us, 6.9 with
//          tiles; 32 x 2048 bf16 by 256: 6.7 and 7.8), or 16 rows: by way of the workspace, if their codes do not fit in LDS.
//          Not for a result in blocks, which are of 32 columns;
//  stream  otherwise up to 256 values a row (of floats, up to 512 bytes), or 512 and up to 256 columns: float rows are quantised in
//          registers, once for every 256 columns (16,384 x 4096 bf16 by 128: 31 us, 42 with tiles; by 512: 80, and 57 with tiles);
//  tile    everything else, float rows by way of the workspace: a tile of x is read by every tile of columns.  256 x 256 where
//          that makes 192 tiles or more; 64 x 64 where there are no more than 512 (two a compute unit): a small product lasts as
//          long as one tile does (256 x 4096 by 4096: 13 us, 19 with 128 x 128; 1024 x 4096 by 4096, 1024 tiles: 27 and 24);
//          else 128 x 128.
enum { MX4_SKINNY, MX4_STREAM, MX4_TILE };
// Steps of 64 values that a row is worked on in; the stream kernel is made for each number of them.
static int stream_steps(int k) { return (k + 63) / 64; }
struct Mx4Plan {
    int kind;
    int64_t w_ordered, x_ordered, codes;                       // bytes of the workspace, in this order; all multiples of 16
    int64_t scales;                                            // or, without tiles: scales in rows, behind the codes
};
static Mx4Plan mx4_plan(int64_t m, int n, int k, int x_dtype, int y_dtype) {
    const bool is_float = x_dtype != NERFX_TYPE_MX4, blocks_out = y_dtype == NERFX_TYPE_MX4;
    const int64_t nb = mx4_blocks(k);
    Mx4Plan plan{};
    const int row_bytes = !is_float ? 0 : x_dtype == NERFX_TYPE_F32 ? 4 * k : 2 * k;       // to be quantised
    if (!blocks_out && m <= (m * row_bytes <= SKINNY_FLOATS ? SKINNY_ROWS : 16)) {
        plan.kind = MX4_SKINNY;
        if (is_float && m * nb * 17 > SKINNY_LDS) { plan.codes = m * nb * 16; plan.scales = (m * nb + 15) / 16 * 16; }
    } else if (k <= (n <= 256 ? 512 : 256) && n <= 1 << 20 && (row_bytes <= 512 || n <= 256)) {
        plan.kind = MX4_STREAM;
    } else {
        plan.kind = MX4_TILE;
        plan.w_ordered = mx4_stages(nb) * mx4_ordered_bytes(n);
        plan.x_ordered = mx4_stages(nb) * mx4_ordered_bytes(m);
        if (is_float) plan.codes = m * nb * 16;
    }
    return plan;
}

template <int DT>
static int skinny_launch(const Mx4LinearArgs& a, hipStream_t stream) {
    const int mt = (int)(a.m + 15) / 16, nb = mx4_blocks(a.k);
    const size_t codes = DT == NERFX_TYPE_MX4 ? 0 : (size_t)a.m * nb * 17, sums = (size_t)SKINNY_WAVES * mt * 1024;
    const size_t lds = std::max(codes, sums);
    const dim3 grid((unsigned)((a.n + 15) / 16)), block(64 * SKINNY_WAVES);
    auto go = [&](auto kernel) {
        NERFX_OPT_IN_LDS(kernel, std::max<size_t>(SKINNY_LDS, SKINNY_WAVES * 4 * 1024));       // of any call
        hipLaunchKernelGGL(kernel, grid, block, lds, stream, a);
        return launch_status("mx4_skinny_kernel");
    };
    switch (mt) {
        case 1: return go(mx4_skinny_kernel<DT, 1>);
        case 2: return go(mx4_skinny_kernel<DT, 2>);
        case 3: return go(mx4_skinny_kernel<DT, 3>);
        default: return go(mx4_skinny_kernel<DT, 4>);
    }
}

template <int DT>
static int stream_launch(const Mx4LinearArgs& a, hipStream_t stream) {
    // Few rows: smaller workgroups and fewer columns in each until the device is full.  A lane's row is a line of its own, so that
    // the loads of eight waves take a CU 3.5 us for every 256 bytes a row (1000 x 128 fp32 by 295: 6.9 us with one wave, 11.6 with
    // eight, in a captured graph); and a wave brings 256 blocks of W at a time, for which it may wait twice.  Half of the device is
    // enough below eight waves (16,000 x 256 bf16 by 256: 9.2 us with 125 workgroups of four, 10.3 with 250 of two), not with them
    // (32,000 x 128 fp32 by 256: 17.6 us with 125 of eight, 12.9 with 250 of four).
    const int tiles = (a.n + 31) / 32, ks = stream_steps(a.k);
    int waves = 2 * STREAM_WAVES, groups;
    int64_t row_tiles;
    do {
        waves /= 2;
        row_tiles = (a.m + 32 * waves - 1) / (32 * waves);
        const int most = std::min(8, std::max(1, 8 * waves / ks));             // tiles of columns
        groups = (tiles + most - 1) / most;
    } while (waves > 1 && row_tiles * groups < (waves == STREAM_WAVES ? 192 : 120));
    groups = (int)std::min<int64_t>(tiles, std::max<int64_t>(groups, 256 / row_tiles));
    const int per = (tiles + groups - 1) / groups;
    const int columns = 32 * per;
    const dim3 grid((unsigned)std::min<int64_t>(row_tiles, 512), (unsigned)((tiles + per - 1) / per)), block(64 * waves);
    auto go = [&](auto kernel, int ks) {
        const size_t lds = stream_lds(ks, columns, waves);
        NERFX_OPT_IN_LDS(kernel, stream_lds(ks, 256, STREAM_WAVES));           // of any call
        hipLaunchKernelGGL(kernel, grid, block, lds, stream, a, columns);
        return launch_status("mx4_stream_kernel");
    };
    auto by_steps = [&](auto odd) {
        constexpr bool ODD = decltype(odd)::value;
        switch (stream_steps(a.k)) {
            case 1: return go(mx4_stream_kernel<DT, 1, ODD>, 1);
            case 2: return go(mx4_stream_kernel<DT, 2, ODD>, 2);
            case 3: return go(mx4_stream_kernel<DT, 3, ODD>, 3);
            case 4: return go(mx4_stream_kernel<DT, 4, ODD>, 4);
            case 5: return go(mx4_stream_kernel<DT, 5, ODD>, 5);
            case 6: return go(mx4_stream_kernel<DT, 6, ODD>, 6);
            case 7: return go(mx4_stream_kernel<DT, 7, ODD>, 7);
            default: return go(mx4_stream_kernel<DT, 8, ODD>, 8);
        }
    };
    if constexpr (DT == NERFX_TYPE_BF16 || DT == NERFX_TYPE_F16)
        if (mx4_odd(a.x, a.k, DT)) return by_steps(std::true_type{});
    return by_steps(std::false_type{});
}

static int check_mx4(int64_t rows, int k) {
    NERFX_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31, "rows %lld out of range [0, 2^31)", (long long)rows);
    NERFX_REQUIRE(k >= 1 && k <= 1 << 20, "k %d out of range [1, 2^20]", k);
    return 0;
}
static bool float_type(int dtype) { return dtype == NERFX_TYPE_F32 || dtype == NERFX_TYPE_BF16 || dtype == NERFX_TYPE_F16; }

}  // namespace nerfx

using namespace nerfx;

extern "C" int nerfx_mx4_quantize(const void* x, int dtype, int64_t rows, int k, uint8_t* codes, uint8_t* scales, void* stream) {
    if (int rc = check_mx4(rows, k)) return rc;
    NERFX_REQUIRE(float_type(dtype), "unknown type %d", dtype);
    if (rows == 0) return 0;
    NERFX_REQUIRE(x && codes && scales, "x / codes / scales is NULL");
    NERFX_REQUIRE(((uintptr_t)codes & 3) == 0, "codes are not aligned to 4 bytes");
    return quantize_launch(x, dtype, rows, k, codes, scales, (hipStream_t)stream);
}

extern "C" int nerfx_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int k, int dtype, void* out, void* stream) {
    if (int rc = check_mx4(rows, k)) return rc;
    NERFX_REQUIRE(float_type(dtype), "unknown type %d", dtype);
    if (rows == 0) return 0;
    NERFX_REQUIRE(codes && scales && out, "codes / scales / out is NULL");
    NERFX_REQUIRE(((uintptr_t)codes & 3) == 0, "codes are not aligned to 4 bytes");
    const int64_t parts = rows * mx4_blocks(k) * (MX4_BLOCK / (dtype == NERFX_TYPE_F32 ? MX4_OUT<NERFX_TYPE_F32> : MX4_OUT<NERFX_TYPE_BF16>));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, mx4_grid(parts), dim3(256), 0, (hipStream_t)stream, codes, scales, parts, k, out);
        return launch_status("mx4_dequantize_kernel");
    };
    if (k % MX4_BLOCK == 0) {
        return dtype == NERFX_TYPE_F32 ? go(mx4_dequantize_kernel<NERFX_TYPE_F32, true>)
             : dtype == NERFX_TYPE_BF16 ? go(mx4_dequantize_kernel<NERFX_TYPE_BF16, true>) : go(mx4_dequantize_kernel<NERFX_TYPE_F16, true>);
    }
    return dtype == NERFX_TYPE_F32 ? go(mx4_dequantize_kernel<NERFX_TYPE_F32, false>)
         : dtype == NERFX_TYPE_BF16 ? go(mx4_dequantize_kernel<NERFX_TYPE_BF16, false>) : go(mx4_dequantize_kernel<NERFX_TYPE_F16, false>);
}

static bool mx4_type(int dtype) { return float_type(dtype) || dtype == NERFX_TYPE_MX4; }
// Columns of a result: one in blocks is a matrix that the other calls take.
static int check_columns(int n, int y_dtype) {
    NERFX_REQUIRE(n >= 0 && n <= 1 << 24, "n %d out of range [0, 2^24]", n);
    NERFX_REQUIRE(y_dtype != NERFX_TYPE_MX4 || (n >= 1 && n <= 1 << 20), "n %d of a result in blocks out of range [1, 2^20]", n);
    return 0;
}

extern "C" int64_t nerfx_mx4_linear_workspace_bytes(int64_t m, int n, int k, int x_dtype, int y_dtype) {
    if (check_mx4(m, k) || !mx4_type(x_dtype) || !mx4_type(y_dtype) || check_columns(n, y_dtype)) return -1;
    const Mx4Plan plan = mx4_plan(m, n, k, x_dtype, y_dtype);
    return plan.w_ordered + plan.x_ordered + plan.codes + plan.scales;
}

extern "C" int nerfx_mx4_linear(const void* x, int x_dtype, const uint8_t* x_scales, int64_t m, int k, const uint8_t* w_codes,
                                const uint8_t* w_scales, int n, const float* bias, int activ, void* y, int y_dtype,
                                uint8_t* y_scales, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_mx4(m, k)) return rc;
    NERFX_REQUIRE(mx4_type(x_dtype), "unknown type %d of x", x_dtype);
    NERFX_REQUIRE(mx4_type(y_dtype), "unknown type %d of y", y_dtype);
    if (int rc = check_columns(n, y_dtype)) return rc;
    NERFX_REQUIRE(activ >= NERFX_ACT_NONE && activ <= NERFX_ACT_SILU, "unknown activation %d", activ);
    if (m == 0 || n == 0) return 0;
    NERFX_REQUIRE(x && w_codes && w_scales && y && (x_dtype != NERFX_TYPE_MX4 || x_scales) && (y_dtype != NERFX_TYPE_MX4 || y_scales),
                  "a required pointer is NULL");
    NERFX_REQUIRE(y_dtype != NERFX_TYPE_MX4 || aligned16(y), "y's codes are not aligned to 16 bytes");
    NERFX_REQUIRE(aligned16(w_codes) && (x_dtype != NERFX_TYPE_MX4 || aligned16(x)), "codes are not aligned to 16 bytes");
    const int64_t need = nerfx_mx4_linear_workspace_bytes(m, n, k, x_dtype, y_dtype);
    NERFX_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
                  "workspace NULL, not aligned to 16 bytes, or of %lld bytes with %lld needed", (long long)workspace_bytes, (long long)need);
    Mx4LinearArgs a{};
    a.w = w_codes; a.w_scales = w_scales; a.bias = bias; a.y = y; a.y_scales = y_scales;
    a.m = m; a.n = n; a.k = k; a.activ = activ; a.y_dtype = y_dtype;
    a.x = (const uint8_t*)x; a.x_scales = x_scales;
    const hipStream_t st = (hipStream_t)stream;
    const Mx4Plan plan = mx4_plan(m, n, k, x_dtype, y_dtype);
    if (plan.kind == MX4_TILE) {
        Mx4PrepareArgs p{};
        p.x = x; p.x_scales = x_scales; p.w_scales = w_scales; p.m = m; p.n = n; p.k = k;
        p.w_ordered = (uint8_t*)workspace;
        p.x_ordered = p.w_ordered + plan.w_ordered;
        p.codes = (uint32_t*)(p.x_ordered + plan.x_ordered);
        if (int rc = prepare_launch(p, x_dtype, st)) return rc;
        a.w_scales = p.w_ordered; a.x_scales = p.x_ordered;
        if (x_dtype != NERFX_TYPE_MX4) a.x = (const uint8_t*)p.codes;
        const int64_t big = ((a.m + 255) / 256) * ((a.n + 255) / 256), small = ((a.m + 63) / 64) * ((a.n + 63) / 64);
        if (small <= 512) return tile_launch<1, 2, 1, 2, 3>(a, st);
        return big >= 192 ? tile_launch<4, 2, 2, 4, 2>(a, st) : tile_launch<2, 2, 2, 2, 2>(a, st);
    }
    if (plan.codes) {
        uint8_t *codes = (uint8_t*)workspace, *scales = codes + plan.codes;
        if (int rc = quantize_launch(x, x_dtype, m, k, codes, scales, st)) return rc;
        a.x = codes; a.x_scales = scales;
        x_dtype = NERFX_TYPE_MX4;
    }
    auto by_type = [&](auto skinny, auto str) { return plan.kind == MX4_SKINNY ? skinny(a, st) : str(a, st); };
    switch (x_dtype) {
        case NERFX_TYPE_F32: return by_type(skinny_launch<NERFX_TYPE_F32>, stream_launch<NERFX_TYPE_F32>);
        case NERFX_TYPE_BF16: return by_type(skinny_launch<NERFX_TYPE_BF16>, stream_launch<NERFX_TYPE_BF16>);
        case NERFX_TYPE_F16: return by_type(skinny_launch<NERFX_TYPE_F16>, stream_launch<NERFX_TYPE_F16>);
        default: return by_type(skinny_launch<NERFX_TYPE_MX4>, stream_launch<NERFX_TYPE_MX4>);
    }
}
