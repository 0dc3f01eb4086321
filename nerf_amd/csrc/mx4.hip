// Microscaled 4-bit numbers (mx4.hpp): to them, back, and the product of two matrices of them.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "mx4.hpp"
#include "split16.hpp"

namespace nerfx {

// ---- to and from -----------------------------------------------------------------------------------------------------
// Four lanes make a block, eight values each: every load and store of a wave is one run of memory.  Bound by
// memory: x is read once, 4.25 bits a value are written.
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* __restrict__ x, int64_t rows, int k, int whole,
                                                           uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    using Raw = Mx4Raw<DT, 8>;
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2;
    const int nb = mx4_blocks(k);
    const int64_t total = rows * nb * 4;
    const int part = threadIdx.x & 3;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t block = q >> 2, row = block / nb;
        const int at = (int)(block - row * nb) * MX4_BLOCK + part * 8;
        Raw v;
        const char* src = (const char*)x + (row * k + at) * SIZE;
        if (whole && at + 8 <= k) {                            // 16-byte pieces; k is a multiple of 8
#pragma unroll
            for (int i = 0; i < Raw::WORDS / 4; ++i) {
                const u32x4_t p = *(const u32x4_t*)(src + 16 * i);
                v.w[4 * i] = p[0]; v.w[4 * i + 1] = p[1]; v.w[4 * i + 2] = p[2]; v.w[4 * i + 3] = p[3];
            }
        } else {
#pragma unroll
            for (int i = 0; i < Raw::WORDS; ++i) {
                if constexpr (DT == NERFX_TYPE_F32) {
                    v.w[i] = at + i < k ? *(const uint32_t*)(src + 4 * i) : 0u;
                } else {
                    const uint32_t lo = at + 2 * i < k ? *(const uint16_t*)(src + 4 * i) : 0u;
                    const uint32_t hi = at + 2 * i + 1 < k ? *(const uint16_t*)(src + 4 * i + 2) : 0u;
                    v.w[i] = lo | hi << 16;
                }
            }
        }
        uint32_t top = v.top_bits();
        top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
        const uint32_t byte = Raw::scale_byte(top);
        codes[q] = byte == 255u ? 0u : v.codes(0, Raw::scale_value(byte));
        if (part == 0) scales[block] = (uint8_t)byte;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             int64_t rows, int k, int whole, void* __restrict__ out) {
    constexpr int SIZE = DT == NERFX_TYPE_F32 ? 4 : 2;
    const int nb = mx4_blocks(k);
    const int64_t total = rows * nb * 4;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t block = q >> 2, row = block / nb;
        const int at = (int)(block - row * nb) * MX4_BLOCK + (int)(q & 3) * 8;
        if (at >= k) continue;
        const uint32_t c = codes[q], byte = scales[block];
        uint32_t w[8 * SIZE / 4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t code = c >> (4 * i) & 15u, m = code & 7u;
            // 0, 0.5 apart, code m is (2 + m % 2) 2^(m / 2 - 3) ... as a float; then times 2^(byte - 127)
            const float grid = m < 2 ? 0.5f * (float)m : __builtin_bit_cast(float, (126u + (m >> 1)) << 23 | (m & 1u) << 22);
            float v = byte == 255u ? __builtin_nanf("") : ldexpf(grid, (int)byte - 127);
            v = code & 8u ? -v : v;
            if constexpr (DT == NERFX_TYPE_F32) {
                w[i] = __builtin_bit_cast(uint32_t, v);
            } else {
                const uint32_t h = DT == NERFX_TYPE_F16 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v)
                                                        : (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);
                if (i & 1) w[i / 2] |= h << 16; else w[i / 2] = h;
            }
        }
        char* dst = (char*)out + (row * k + at) * SIZE;
        if (whole && at + 8 <= k) {
#pragma unroll
            for (int i = 0; i < SIZE / 2; ++i) *(u32x4_t*)(dst + 16 * i) = {w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
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
    int32_t n, k, activ, y_dtype, y_whole;     // y_whole: 16-byte stores are possible
};

__device__ __forceinline__ float mx4_activate(float v, int activ) {
    if (activ == NERFX_ACT_RELU) return v < 0.f ? 0.f : v;
    if (activ == NERFX_ACT_LEAKY_RELU) return v < 0.f ? 0.01f * v : v;
    if (activ == NERFX_ACT_SILU) return v / (1.0f + expf(-v));
    return v;
}

typedef int i32x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8_t mx4_operand(u32x4_t c) { return {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0}; }

// y for the 32 x 32 accumulator of rows n0 .. of W and rows m0 .. of x: a lane holds row m = m0 + lane % 32 and, with
// h = lane / 32, columns n0 + 8 q + 4 h + i in element 4 q + i.
__device__ __forceinline__ void mx4_store(const Mx4LinearArgs& a, const float16_t_& acc, int64_t m0, int n0) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int64_t m = m0 + (lane & 31);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int n = n0 + 8 * (e >> 2) + 4 * h + (e & 3);
        v[e] = mx4_activate(acc[e] + (a.bias && n < a.n ? a.bias[n] : 0.f), a.activ);
    }
    if (a.y_dtype == NERFX_TYPE_F32) {
        if (m >= a.m) return;
        float* y = (float*)a.y + m * a.n;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + 8 * q + 4 * h;
            if (a.y_whole) {
                if (n < a.n) *(u32x4_t*)(y + n) = __builtin_bit_cast(u32x4_t, (float __attribute__((ext_vector_type(4)))){v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < a.n) y[n + i] = v[4 * q + i];
            }
        }
        return;
    }
    // two 16-bit values a word; word 2 q + p holds columns 8 q + 4 h + 2 p, + 1
    uint32_t w[8];
#pragma unroll
    for (int p = 0; p < 8; ++p)
        w[p] = a.y_dtype == NERFX_TYPE_BF16 ? __builtin_bit_cast(uint32_t, (bf16x2_t){(__bf16)v[2 * p], (__bf16)v[2 * p + 1]})
                                            : __builtin_bit_cast(uint32_t, (f16x2_t){(_Float16)v[2 * p], (_Float16)v[2 * p + 1]});
    if (!a.y_whole) {
        if (m >= a.m) return;
        uint16_t* y = (uint16_t*)a.y + m * a.n;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int n = n0 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (n < a.n) y[n] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
        return;
    }
    // exchange halves between lanes l and l + 32, so that one lane has 16 columns in a row: the lower lane
    // q = 0, 1 (columns 0 .. 15), the upper one q = 2, 3
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const auto r = __builtin_amdgcn_permlane32_swap(w[p], w[p + 4], false, false);
        w[p] = r[0];
        w[p + 4] = r[1];
    }
    if (m >= a.m) return;
    uint16_t* y = (uint16_t*)a.y + m * a.n;
    const int n = n0 + 16 * h;
    if (n < a.n) *(u32x4_t*)(y + n) = {w[0], w[1], w[4], w[5]};
    if (n + 8 < a.n) *(u32x4_t*)(y + n + 8) = {w[2], w[3], w[6], w[7]};
}

// A (32 FP WP) x (32 FQ WQ) tile of W x^T per workgroup of WP x WQ waves.  A stage is eight blocks (256 values) of every
// row of both operands, 128 bytes a row, brought by LDS-DMA; block c of row r lies at place c ^ (r / 2 % 8), as in the
// split16 products.  The scales, one byte a block, go straight into registers one stage ahead.
template <int FP, int WP, int FQ, int WQ, int STAGES>
struct Mx4Tile {
    static constexpr int WAVES = WP * WQ, TP = 32 * FP * WP, TQ = 32 * FQ * WQ;
    static constexpr int STAGE_BLOCKS = 8, ROW_BYTES = STAGE_BLOCKS * MX4_BLOCK_BYTES;
    static constexpr int STAGE_BYTES = (TP + TQ) * ROW_BYTES, LDS_BYTES = STAGES * STAGE_BYTES;
    static constexpr int LOADS_P = TP / (8 * WAVES), LOADS_Q = TQ / (8 * WAVES);
    static_assert(TP % (8 * WAVES) == 0 && TQ % (8 * WAVES) == 0 && LDS_BYTES <= 160 * 1024, "whole loads per wave");
};

template <int FP, int WP, int FQ, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void mx4_tile_kernel(const Mx4LinearArgs a) {
    using T = Mx4Tile<FP, WP, FQ, WQ, 1>;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int nb = mx4_blocks(a.k), stages = (nb + 7) / 8;
    const int n_tiles = (a.n + T::TP - 1) / T::TP;
    const int n0 = (int)(blockIdx.x % n_tiles) * T::TP;
    const int64_t m0 = (int64_t)(blockIdx.x / n_tiles) * T::TQ;
    const int wp = wave / WQ * 32 * FP, wq = wave % WQ * 32 * FQ;
    float16_t_ acc[FP][FQ];
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    for (int st = 0; st < stages; ++st) {
        __syncthreads();
        for (int c = threadIdx.x; c < (T::TP + T::TQ) * 8; c += 64 * T::WAVES) {
            const int r = c >> 3, b = st * 8 + (c & 7);
            u32x4_t v = {0, 0, 0, 0};
            if (b < nb) {
                if (r < T::TP) { if (n0 + r < a.n) v = *(const u32x4_t*)(a.w + ((int64_t)(n0 + r) * nb + b) * 16); }
                else if (m0 + r - T::TP < a.m) v = *(const u32x4_t*)(a.x + ((m0 + r - T::TP) * nb + b) * 16);
            }
            *(u32x4_t*)(lds + r * T::ROW_BYTES + (((c & 7) ^ (r >> 1 & 7)) * 16)) = v;
        }
        __syncthreads();
        uint32_t sp[FP][4], sq[FQ][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int b = st * 8 + 2 * s + h;
#pragma unroll
            for (int i = 0; i < FP; ++i) {
                const int r = n0 + wp + 32 * i + (lane & 31);
                sp[i][s] = b < nb && r < a.n ? a.w_scales[(int64_t)r * nb + b] : 127u;
            }
#pragma unroll
            for (int j = 0; j < FQ; ++j) {
                const int64_t r = m0 + wq + 32 * j + (lane & 31);
                sq[j][s] = b < nb && r < a.m ? a.x_scales[r * nb + b] : 127u;
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (st * 8 + 2 * s >= nb) break;
            u32x4_t fp[FP], fq[FQ];
#pragma unroll
            for (int i = 0; i < FP; ++i) {
                const int r = wp + 32 * i + (lane & 31);
                fp[i] = *(const u32x4_t*)(lds + r * T::ROW_BYTES + (((2 * s + h) ^ (r >> 1 & 7)) * 16));
            }
#pragma unroll
            for (int j = 0; j < FQ; ++j) {
                const int r = T::TP + wq + 32 * j + (lane & 31);
                fq[j] = *(const u32x4_t*)(lds + r * T::ROW_BYTES + (((2 * s + h) ^ (r >> 1 & 7)) * 16));
            }
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(fp[i]), mx4_operand(fq[j]), acc[i][j], 4, 4,
                                                                               0, (int)sp[i][s], 0, (int)sq[j][s]);
        }
    }
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j)
            if (n0 + wp + 32 * i < a.n) mx4_store(a, acc[i][j], m0 + wq + 32 * j, n0 + wp + 32 * i);
}

// ---- host side -------------------------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int quantize_launch(const void* x, int dtype, int64_t rows, int k, uint8_t* codes, uint8_t* scales, hipStream_t stream) {
    const int64_t threads = rows * mx4_blocks(k) * 4;
    const dim3 grid((unsigned)std::min<int64_t>((threads + 255) / 256, 256 * 32));
    const int whole = k % 8 == 0 && aligned16(x);
    uint32_t* c = (uint32_t*)codes;
    if (dtype == NERFX_TYPE_F32) hipLaunchKernelGGL(mx4_quantize_kernel<NERFX_TYPE_F32>, grid, dim3(256), 0, stream, x, rows, k, whole, c, scales);
    else if (dtype == NERFX_TYPE_BF16) hipLaunchKernelGGL(mx4_quantize_kernel<NERFX_TYPE_BF16>, grid, dim3(256), 0, stream, x, rows, k, whole, c, scales);
    else hipLaunchKernelGGL(mx4_quantize_kernel<NERFX_TYPE_F16>, grid, dim3(256), 0, stream, x, rows, k, whole, c, scales);
    return launch_status("mx4_quantize_kernel");
}

template <int FP, int WP, int FQ, int WQ>
static int tile_launch(const Mx4LinearArgs& a, hipStream_t stream) {
    using T = Mx4Tile<FP, WP, FQ, WQ, 1>;
    const int64_t tiles = ((a.n + T::TP - 1) / T::TP) * ((a.m + T::TQ - 1) / T::TQ);
    NERFX_REQUIRE(tiles <= 1 << 22, "%lld x %d results are too many for one launch", (long long)a.m, a.n);
    NERFX_OPT_IN_LDS((mx4_tile_kernel<FP, WP, FQ, WQ>), T::LDS_BYTES);
    hipLaunchKernelGGL((mx4_tile_kernel<FP, WP, FQ, WQ>), dim3((unsigned)tiles), dim3(64 * T::WAVES), T::LDS_BYTES, stream, a);
    return launch_status("mx4_tile_kernel");
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
    const int64_t threads = rows * mx4_blocks(k) * 4;
    const dim3 grid((unsigned)std::min<int64_t>((threads + 255) / 256, 256 * 32));
    const int whole = k % 8 == 0 && aligned16(out);
    const uint32_t* c = (const uint32_t*)codes;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == NERFX_TYPE_F32) hipLaunchKernelGGL(mx4_dequantize_kernel<NERFX_TYPE_F32>, grid, dim3(256), 0, s, c, scales, rows, k, whole, out);
    else if (dtype == NERFX_TYPE_BF16) hipLaunchKernelGGL(mx4_dequantize_kernel<NERFX_TYPE_BF16>, grid, dim3(256), 0, s, c, scales, rows, k, whole, out);
    else hipLaunchKernelGGL(mx4_dequantize_kernel<NERFX_TYPE_F16>, grid, dim3(256), 0, s, c, scales, rows, k, whole, out);
    return launch_status("mx4_dequantize_kernel");
}

extern "C" int64_t nerfx_mx4_linear_workspace_bytes(int64_t m, int n, int k, int x_dtype) {
    if (check_mx4(m, k) || check_mx4(n, k) || !(float_type(x_dtype) || x_dtype == NERFX_TYPE_MX4)) return -1;
    if (x_dtype == NERFX_TYPE_MX4) return 0;
    return (m * mx4_blocks(k) * 17 + 15) / 16 * 16;
}

extern "C" int nerfx_mx4_linear(const void* x, int x_dtype, const uint8_t* x_scales, int64_t m, int k, const uint8_t* w_codes,
                                const uint8_t* w_scales, int n, const float* bias, int activ, void* y, int y_dtype,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_mx4(m, k)) return rc;
    if (int rc = check_mx4(n, k)) return rc;
    NERFX_REQUIRE(float_type(x_dtype) || x_dtype == NERFX_TYPE_MX4, "unknown type %d of x", x_dtype);
    NERFX_REQUIRE(float_type(y_dtype), "unknown type %d of y", y_dtype);
    NERFX_REQUIRE(activ >= NERFX_ACT_NONE && activ <= NERFX_ACT_SILU, "unknown activation %d", activ);
    if (m == 0 || n == 0) return 0;
    NERFX_REQUIRE(x && w_codes && w_scales && y && (x_dtype != NERFX_TYPE_MX4 || x_scales), "a required pointer is NULL");
    NERFX_REQUIRE(aligned16(w_codes) && (x_dtype != NERFX_TYPE_MX4 || aligned16(x)), "codes are not aligned to 16 bytes");
    const int64_t need = nerfx_mx4_linear_workspace_bytes(m, n, k, x_dtype);
    NERFX_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
                  "workspace NULL, not aligned to 16 bytes, or of %lld bytes with %lld needed", (long long)workspace_bytes, (long long)need);
    Mx4LinearArgs a{};
    a.w = w_codes; a.w_scales = w_scales; a.bias = bias; a.y = y;
    a.m = m; a.n = n; a.k = k; a.activ = activ; a.y_dtype = y_dtype;
    a.y_whole = aligned16(y) && n % (y_dtype == NERFX_TYPE_F32 ? 4 : 8) == 0;
    a.x = (const uint8_t*)x; a.x_scales = x_scales;
    if (x_dtype != NERFX_TYPE_MX4) {
        uint8_t* codes = (uint8_t*)workspace;
        uint8_t* scales = codes + m * mx4_blocks(k) * 16;
        if (int rc = quantize_launch(x, x_dtype, m, k, codes, scales, (hipStream_t)stream)) return rc;
        a.x = codes; a.x_scales = scales;
    }
    return tile_launch<2, 2, 2, 2>(a, (hipStream_t)stream);
}
