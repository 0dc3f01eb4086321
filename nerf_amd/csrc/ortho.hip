// Orthogonalised updates: Newton-Schulz steps on a group of matrices, and the optimiser step around them.
//
// For a matrix G (rows x cols), X = G / max(|G|_F, eps), transposed if it is taller than wide (m <= n), then
// per step   A = X X^T,   B = b A + c A A,   X <- a X + B X
// which takes every singular value s to a s + b s^3 + c s^5 and leaves the singular vectors.  The result goes
// back in G's own orientation.  A whole group of matrices of any shapes shares every launch: a launch's grid
// is the concatenation of the matrices' tiles, and a workgroup finds its matrix by walking the (short) table
// in the kernel's arguments, so nothing is copied to the device and the call can be captured.
#include <algorithm>
#include <cmath>

#include "lds_dma.hpp"
#include "split16.hpp"

namespace nerfx {

constexpr int ORTHO_GROUP = 32;                 // matrices per launch: the table has to fit the kernel arguments
constexpr int ORTHO_MAX_SIDE = 32768;
constexpr int ORTHO_MAX_STEPS = 32;
constexpr int NORM_PARTS = 512;                 // partial sums of squares per matrix
constexpr int PREP_TILE = 64;

struct OrthoMat {
    const void* grad;
    float* momentum;                            // optimiser step only
    float* param;
    void* out;                                  // orthogonalize only
    int64_t base;                               // byte offset of this matrix's part of the workspace
    int32_t rows, cols;                         // as the caller has it
    int32_t m, n;                               // smaller and larger side, padded to whole tiles
    float lr;                                   // optimiser step: learning rate with its shape factor
    int32_t tall;                               // rows > cols: X is the transpose
};
struct OrthoArgs {
    OrthoMat mat[ORTHO_GROUP];
    int32_t first[ORTHO_GROUP];                 // first block of each matrix in this launch; INT_MAX behind the last
    char* work;
    const float* grad_scale;
    const float* found_inf;
    float momentum, rest, decay;                // rest: 1 - momentum, decay: 1 - lr * weight_decay
    int32_t growth;                             // the steps together grow a singular value by at most 2^growth
    float eps, alpha, beta, x_scale;            // alpha, beta: factors of the epilogue's element and accumulator
    int32_t count, nesterov, dtype, muon;
    int32_t from, to;                           // which of the two X^T copies is read and written
};
static_assert(sizeof(OrthoArgs) <= 4096, "the group's table has to fit the kernel arguments");

// Parts of a matrix's workspace: X (m x n), two copies of X^T (n x m), A and B (m x m), partial sums.
__host__ __device__ inline int64_t ortho_x_bytes(const OrthoMat& q) { return (int64_t)q.m * q.n * 4; }
__host__ __device__ inline int64_t ortho_a_bytes(const OrthoMat& q) { return (int64_t)q.m * q.m * 4; }
__host__ __device__ inline int64_t ortho_xt_at(const OrthoMat& q, int which) { return q.base + ortho_x_bytes(q) * (1 + which); }
__host__ __device__ inline int64_t ortho_a_at(const OrthoMat& q) { return q.base + 3 * ortho_x_bytes(q); }
__host__ __device__ inline int64_t ortho_b_at(const OrthoMat& q) { return ortho_a_at(q) + ortho_a_bytes(q); }
__host__ __device__ inline int64_t ortho_sums_at(const OrthoMat& q) { return ortho_b_at(q) + ortho_a_bytes(q); }
__host__ __device__ inline int64_t ortho_bytes(const OrthoMat& q) {
    return 3 * ortho_x_bytes(q) + 2 * ortho_a_bytes(q) + NORM_PARTS * 8 + 16;
}
__host__ __device__ inline int64_t ortho_lift_at(const OrthoMat& q) { return ortho_sums_at(q) + NORM_PARTS * 8; }
__host__ __device__ inline int norm_parts(const OrthoMat& q) {
    const int64_t parts = ((int64_t)q.rows * q.cols + 4095) / 4096;
    return parts < NORM_PARTS ? (int)parts : NORM_PARTS;
}

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == NERFX_TYPE_F32) return ((const float*)p)[i];
    if (dtype == NERFX_TYPE_F16) return (float)((const _Float16*)p)[i];
    return (float)((const __bf16*)p)[i];
}
__device__ __forceinline__ void store_from_float(void* p, int64_t i, float v, int dtype) {
    if (dtype == NERFX_TYPE_F32) ((float*)p)[i] = v;
    else if (dtype == NERFX_TYPE_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}
// What is orthogonalised, at flat index i: the gradient, or the optimiser's mix of it and the (new) momentum.
__device__ __forceinline__ float update_at(const OrthoArgs& a, const OrthoMat& q, int64_t i, float unscale) {
    const float g = load_as_float(q.grad, i, a.dtype);
    if (!a.muon) return g;
    const float mom = q.momentum[i];
    return a.nesterov ? fmaf(a.momentum, mom, a.rest * (g * unscale)) : mom;
}

// The matrix that this block works on, and the block's number within it.  (All of the table is read at once:
// walking it would wait for each entry in turn.)
__device__ __forceinline__ int which_matrix(const OrthoArgs& a, int& block) {
    const int b = blockIdx.x;
    int k = 0, start = 0;
#pragma unroll
    for (int i = 1; i < ORTHO_GROUP; ++i) {
        const int f = a.first[i];
        if (b >= f) { k = i; start = f; }
    }
    block = b - start;
    return k;
}
enum { ORTHO_GRAM, ORTHO_POLY, ORTHO_APPLY, ORTHO_LAST };

// Momentum, and partial sums of squares of what is orthogonalised.  In double: a fp32 gradient's square
// neither overflows nor vanishes there, and a sum of 2^30 of them keeps fp32's precision.
__global__ __launch_bounds__(256) void ortho_norm_kernel(const OrthoArgs a) {
    int b;
    const OrthoMat q = a.mat[which_matrix(a, b)];
    const int64_t total = (int64_t)q.rows * q.cols;
    const int parts = norm_parts(q);
    const bool skip = a.found_inf && *a.found_inf != 0.f;
    const float unscale = a.grad_scale ? 1.0f / *a.grad_scale : 1.0f;
    double acc = 0;
    for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < total; i += (int64_t)parts * 256) {
        if (a.muon && !skip)
            q.momentum[i] = fmaf(a.momentum, q.momentum[i], a.rest * (((const float*)q.grad)[i] * unscale));
        const double u = update_at(a, q, i, unscale);
        acc = fma(u, u, acc);
    }
    __shared__ double part[4];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)(a.work + ortho_sums_at(q)))[b] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X and X^T from what is orthogonalised: one 64 x 64 tile of X per block, through LDS, zeros in the padding.
__global__ __launch_bounds__(256) void ortho_prep_kernel(const OrthoArgs a) {
    int b;
    const OrthoMat q = a.mat[which_matrix(a, b)];
    __shared__ float tile[PREP_TILE][PREP_TILE + 1];
    const double* sums = (const double*)(a.work + ortho_sums_at(q));
    __shared__ double part[4];
    double total = 0;
    for (int k = threadIdx.x; k < norm_parts(q); k += 256) total += sums[k];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
    __syncthreads();
    const double norm = sqrt((part[0] + part[1]) + (part[2] + part[3]));
    double factor = (double)a.x_scale / (norm < (double)a.eps ? (double)a.eps : norm);                 // NaN stays NaN
    // A norm far below eps leaves X tiny, and f16 has few small numbers: X is then kept 2^lift larger, with room for
    // the growth of all steps.  (A, far smaller than 1 there, is stored as it is: X X^T / 4^lift.)
    int lift = 0;
    if (norm < (double)a.eps) lift = max(0, min(120, norm > 0 ? ilogb((double)a.eps / norm) - a.growth : 0));
    factor = ldexp(factor, lift);
    if (b == 0 && threadIdx.x == 0) *(int*)(a.work + ortho_lift_at(q)) = lift;
    const float unscale = a.grad_scale ? 1.0f / *a.grad_scale : 1.0f;
    const int x0 = b / (q.n / PREP_TILE) * PREP_TILE, y0 = b % (q.n / PREP_TILE) * PREP_TILE;   // of X
    // G's rows run along X's columns, or, if G is tall, along X's rows
    const int r0 = q.tall ? y0 : x0, c0 = q.tall ? x0 : y0;
    for (int e = threadIdx.x; e < PREP_TILE * PREP_TILE; e += 256) {
        const int r = e / PREP_TILE, c = e % PREP_TILE;
        float v = 0.f;
        if (r0 + r < q.rows && c0 + c < q.cols) v = (float)(update_at(a, q, (int64_t)(r0 + r) * q.cols + c0 + c, unscale) * factor);
        if (q.tall) tile[c][r] = v; else tile[r][c] = v;
    }
    __syncthreads();
    char* x = a.work + q.base;
    char* xt = a.work + ortho_xt_at(q, 0);
    for (int e = threadIdx.x; e < PREP_TILE * PREP_TILE / 4; e += 256) {
        const int r = e / (PREP_TILE / 4), k = (e % (PREP_TILE / 4)) * 4;
        const float row[4] = {tile[r][k], tile[r][k + 1], tile[r][k + 2], tile[r][k + 3]};
        const float col[4] = {tile[k][r], tile[k + 1][r], tile[k + 2][r], tile[k + 3][r]};
        split_store4(x, x0 + r, y0 + k, q.n, row);
        split_store4(xt, y0 + r, x0 + k, q.m, col);
    }
}

// ---- the products ---------------------------------------------------------------------------------------------------
// One T x T tile of P Q^T for two row-major split matrices with rows along K: 2 x WAVES / 2 waves, each its part of
// the tile.  A stage is one 32-wide block of K of both operands; STAGES of them lie in LDS, all but one of them on
// their way while one is worked on (LDS-DMA: no registers hold them).  16-byte chunk c of row r lies at place
// c ^ (r / 2 % 8), so that the sixteen rows a ds_read_b128 phase touches (256 bytes of banks) lie apart; LDS-DMA
// writes lane after lane, so it is the source address that is permuted.
template <int T, int WAVES, int STAGES>
struct SplitTile {
    static constexpr int FP = T / 64, FQ = T / (16 * WAVES); // 32 x 32 fragments per wave and side
    static constexpr int LOADS = T / (8 * WAVES);            // per wave, stage and operand
    static constexpr int STAGE_BYTES = 2 * T * SPLIT_BLOCK_BYTES;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
    static_assert(STAGES >= 2 && STAGES <= 8 && 2 * LOADS * (STAGES - 1) < 64, "waits of landed()");
    float16_t_ acc[FP][FQ];

    // Until all stages but the newest `later` have landed.
    static __device__ __forceinline__ void wait(int later) {
        switch (later < STAGES - 1 ? later : STAGES - 1) {
            case 0: landed<0>(); break;
            case 1: landed<2 * LOADS>(); break;
            case 2: landed<2 * LOADS * (STAGES > 2 ? 2 : 0)>(); break;
            case 3: landed<2 * LOADS * (STAGES > 3 ? 3 : 0)>(); break;
            case 4: landed<2 * LOADS * (STAGES > 4 ? 4 : 0)>(); break;
            case 5: landed<2 * LOADS * (STAGES > 5 ? 5 : 0)>(); break;
            case 6: landed<2 * LOADS * (STAGES > 6 ? 6 : 0)>(); break;
            default: landed<2 * LOADS * (STAGES > 7 ? 7 : 0)>(); break;
        }
    }
    struct Frags { half8_t ph[FP], pl[FP], qh[FQ], ql[FQ]; };
    // half s of stage buffer `buf`: 16 of its 32 columns
    static __device__ __forceinline__ void read(Frags& f, const char* buf, int s, int wave, int lane) {
        auto frag = [&](int row, int chunk) {
            return *(const half8_t*)(buf + row * SPLIT_BLOCK_BYTES + ((chunk ^ (row >> 1 & 7)) * 16));
        };
        const int p_row = row_of(wave) + (lane & 31), q_row = T + col_of(wave) + (lane & 31), c = 2 * s + (lane >> 5);
#pragma unroll
        for (int i = 0; i < FP; ++i) { f.ph[i] = frag(p_row + 32 * i, c); f.pl[i] = frag(p_row + 32 * i, c + 4); }
#pragma unroll
        for (int j = 0; j < FQ; ++j) { f.qh[j] = frag(q_row + 32 * j, c); f.ql[j] = frag(q_row + 32 * j, c + 4); }
    }
    // the three products of a fragment lie apart, so that no instruction waits for the one before
    __device__ __forceinline__ void multiply(const Frags& f) {
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(t == 1 ? f.pl[i] : f.ph[i], t == 0 ? f.ql[j] : f.qh[j],
                                                                       acc[i][j], 0, 0, 0);
    }

    __device__ __forceinline__ void run(char* lds, const char* P, const char* Q, int K) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t pitch = (uint32_t)K / SPLIT_BLOCK * SPLIT_BLOCK_BYTES;
        const int steps = K / SPLIT_BLOCK;
        const uint32_t lds0 = lds_address(lds);
        // this lane's 16 bytes of the first of the rows that the wave's loads bring; the others lie 8 WAVES rows apart
        const int row = 8 * wave + (lane >> 3);
        const uint32_t offset = (uint32_t)row * pitch + ((lane & 7) ^ (row >> 1 & 7)) * 16;
        auto fetch = [&](int kb) {
            const uint32_t to = lds0 + (uint32_t)(kb % STAGES) * STAGE_BYTES + wave * 1024;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const uint32_t at = to + i * WAVES * 1024, from = offset + i * 8 * WAVES * pitch;
                dma16(at, P + (int64_t)kb * SPLIT_BLOCK_BYTES, from);
                dma16(at + T * SPLIT_BLOCK_BYTES, Q + (int64_t)kb * SPLIT_BLOCK_BYTES, from);
            }
        };
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
#pragma unroll
        for (int kb = 0; kb < STAGES; ++kb)
            if (kb < steps) fetch(kb);
        Frags f0, f1;
        wait(steps - 1);
        read(f0, lds, 0, wave, lane);
        for (int kb = 0; kb < steps - 1; ++kb) {             // fragments are read one half stage ahead of their use
            read(f1, lds + (kb % STAGES) * STAGE_BYTES, 1, wave, lane);
            multiply(f0);
            wait(min(STAGES - 2, steps - 2 - kb));           // stage kb + 1 is there, and every wave has read all of stage kb,
            if (kb + STAGES < steps) fetch(kb + STAGES);     // whose place this one takes
            read(f0, lds + ((kb + 1) % STAGES) * STAGE_BYTES, 0, wave, lane);
            multiply(f1);
        }
        read(f1, lds + ((steps - 1) % STAGES) * STAGE_BYTES, 1, wave, lane);
        multiply(f0);
        multiply(f1);
    }
    // where in the tile a wave's part begins
    static __device__ __forceinline__ int row_of(int wave) { return wave / (WAVES / 2) * (T / 2); }
    static __device__ __forceinline__ int col_of(int wave) { return wave % (WAVES / 2) * (2 * T / WAVES); }
};

// Number t of a lower triangle's tiles, row after row -> (row, column).
__device__ __forceinline__ void triangle_at(int64_t t, int& i, int& j) {
    i = (int)((sqrt(8.0 * (double)t + 1.0) - 1.0) * 0.5);
    while ((int64_t)i * (i + 1) / 2 > t) --i;
    while ((int64_t)(i + 1) * (i + 2) / 2 <= t) ++i;
    j = (int)(t - (int64_t)i * (i + 1) / 2);
}

template <int T, int WAVES, int STAGES, int KIND>
__global__ __launch_bounds__(64 * WAVES) void ortho_product_kernel(const OrthoArgs a) {
    extern __shared__ __align__(16) char lds[];
    constexpr bool SYM = KIND == ORTHO_GRAM || KIND == ORTHO_POLY;       // the result is symmetric: half of the tiles
    int b;
    const OrthoMat q = a.mat[which_matrix(a, b)];
    int ti, tj;
    if constexpr (SYM) {
        triangle_at(b, ti, tj);
    } else {
        ti = b % (q.m / T);
        tj = b / (q.m / T);
    }
    char* X = a.work + q.base;
    char* A = a.work + ortho_a_at(q);
    char* B = a.work + ortho_b_at(q);
    const char* P = KIND == ORTHO_GRAM ? X : KIND == ORTHO_POLY ? A : B;
    const char* Q = KIND == ORTHO_GRAM ? X : KIND == ORTHO_POLY ? A : a.work + ortho_xt_at(q, a.from);
    const int K = KIND == ORTHO_GRAM ? q.n : q.m;
    using Tile = SplitTile<T, WAVES, STAGES>;
    Tile tile;
    // element (row, col) of a 32 x 32 accumulator: col = lane % 32, row = 8 (e / 4) + 4 (lane / 32) + e % 4
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // the element itself, A[row][col] = A[col][row] or X[row][col] = X^T[col][row], is on its way from the start
    Split4 own[Tile::FP][Tile::FQ][4];
    if constexpr (KIND != ORTHO_GRAM) {
#pragma unroll
        for (int i = 0; i < Tile::FP; ++i)
#pragma unroll
            for (int j = 0; j < Tile::FQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    own[i][j][e] = split_load4(Q, tj * T + Tile::col_of(wave) + 32 * j + (lane & 31),
                                               ti * T + Tile::row_of(wave) + 32 * i + 4 * (lane >> 5) + 8 * e, q.m);
    }
    tile.run(lds, P + (int64_t)ti * T * K * 4, Q + (int64_t)tj * T * K * 4, K);
    float alpha = a.alpha, beta = a.beta;
    if constexpr (KIND == ORTHO_GRAM || KIND == ORTHO_LAST) {            // see the kernel that made X
        const int lift = *(const int*)(a.work + ortho_lift_at(q));
        beta = ldexpf(beta, KIND == ORTHO_GRAM ? -2 * lift : -lift);
        alpha = ldexpf(alpha, -lift);
    }
    const bool skip = KIND == ORTHO_LAST && a.found_inf && *a.found_inf != 0.f;
#pragma unroll
    for (int i = 0; i < Tile::FP; ++i)
#pragma unroll
        for (int j = 0; j < Tile::FQ; ++j) {
            const int row0 = ti * T + Tile::row_of(wave) + 32 * i + 4 * (lane >> 5);
            const int col = tj * T + Tile::col_of(wave) + 32 * j + (lane & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + 8 * e;
                float v[4];
                if constexpr (KIND == ORTHO_GRAM) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = beta * tile.acc[i][j][4 * e + k];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[k] = fmaf(beta, tile.acc[i][j][4 * e + k], alpha * ((float)own[i][j][e].hi[k] + (float)own[i][j][e].lo[k]));
                }
                if constexpr (SYM) {
                    char* dst = KIND == ORTHO_GRAM ? A : B;
                    if (ti != tj) split_store4(dst, col, row, q.m, v);             // the mirrored tile
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        _Float16 hi, lo;
                        split16(v[k], hi, lo);
                        char* p = split_at(dst, row + k, col, q.m);
                        *(_Float16*)p = hi;
                        *(_Float16*)(p + 64) = lo;
                    }
                } else if constexpr (KIND == ORTHO_APPLY) {
                    split_store4(a.work + ortho_xt_at(q, a.to), col, row, q.m, v);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        _Float16 hi, lo;
                        split16(v[k], hi, lo);
                        char* p = split_at(X, row + k, col, q.n);
                        *(_Float16*)p = hi;
                        *(_Float16*)(p + 64) = lo;
                    }
                } else if (!skip) {                                                // into the caller's matrix
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = q.tall ? col : row + k, c = q.tall ? row + k : col;
                        if (r >= q.rows || c >= q.cols) continue;
                        const int64_t at = (int64_t)r * q.cols + c;
                        if (a.muon) q.param[at] = fmaf(-q.lr, v[k], q.param[at] * a.decay);
                        else store_from_float(q.out, at, v[k], a.dtype);
                    }
                }
            }
        }
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Sides are padded to whole tiles: of 128 where there is enough work for them somewhere, else of 64.
static int tile_side(const nerfx_matrix_t* mats, int count) {
    int64_t big = 0;
    for (int k = 0; k < count; ++k) {
        const int64_t r = (mats[k].rows + 127) / 128, c = (mats[k].cols + 127) / 128;
        big += r * c;
    }
    return big >= 192 ? 128 : 64;
}

static int64_t fill_group(const nerfx_matrix_t* mats, int count, int tile, OrthoArgs& a) {
    int64_t at = 0;
    a.count = 0;
    for (int k = 0; k < count; ++k) {
        if (mats[k].rows == 0 || mats[k].cols == 0) continue;
        OrthoMat& q = a.mat[a.count++];
        q = OrthoMat{};
        q.grad = mats[k].grad; q.momentum = mats[k].momentum; q.param = mats[k].param; q.out = mats[k].out;
        q.rows = mats[k].rows; q.cols = mats[k].cols;
        q.tall = q.rows > q.cols;
        auto up = [&](int v) { return (v + tile - 1) / tile * tile; };
        q.m = up(std::min(q.rows, q.cols));
        q.n = up(std::max(q.rows, q.cols));
        q.base = at;
        at += (ortho_bytes(q) + 255) / 256 * 256;
    }
    return at;
}

static int check_sizes(const nerfx_matrix_t* mats, int count) {
    NERFX_REQUIRE(count >= 0 && (count == 0 || mats), "bad matrix table");
    for (int k = 0; k < count; ++k)
        NERFX_REQUIRE(mats[k].rows >= 0 && mats[k].rows <= ORTHO_MAX_SIDE && mats[k].cols >= 0 && mats[k].cols <= ORTHO_MAX_SIDE,
                      "matrix %d is %d x %d: sides up to %d", k, mats[k].rows, mats[k].cols, ORTHO_MAX_SIDE);
    return 0;
}

// Largest singular value after each step, for start values up to 1: the maximum of |a s + b s^3 + c s^5| over
// [0, top] by sampling (the polynomial's own maximum lies within the margin of a sample).  It says which
// power-of-two scales keep X, A and B inside f16.
struct OrthoScales { float x, a, b; int growth; };
static int scales_for(const float* coef, int steps, OrthoScales& s) {
    double top = 1.001, x = top, ga = 0, gb = 0, all = 1;
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        NERFX_REQUIRE(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), "coefficient %d is not finite", k);
        double next = 0, gain = 1;
        for (int i = 0; i <= 1024; ++i) {
            const double v = top * i / 1024, l = v * v;
            next = std::max(next, std::fabs(v * (a + l * (b + l * c))));
            gain = std::max(gain, std::fabs(a + l * (b + l * c)));
            gb = std::max(gb, std::fabs(l * (b + l * c)));
        }
        ga = std::max(ga, top * top);
        x = std::max(x, top);
        top = next * 1.01;
        all *= gain * 1.01;
        NERFX_REQUIRE(top <= 64, "step %d lets singular values grow to %.3g: coefficients out of range", k, top);
    }
    auto scale = [](double bound) { return (float)std::exp2(std::floor(std::log2(32768 / std::max(bound * 1.02, 1e-3)))); };
    s = {scale(x), scale(ga), scale(gb), (int)std::ceil(std::log2(all))};
    return 0;
}

// A launch's grid is the matrices' blocks one after the other.
template <class F>
static int64_t lay_out(OrthoArgs& a, F blocks_of) {
    int64_t at = 0;
    for (int k = 0; k < ORTHO_GROUP; ++k) {
        a.first[k] = k < a.count ? (int32_t)at : INT32_MAX;
        if (k < a.count) at += blocks_of(a.mat[k]);
    }
    return at;
}

template <int KIND>
static int64_t product_blocks(OrthoArgs& a, int tile) {
    return lay_out(a, [tile](const OrthoMat& q) {
        const int64_t mt = q.m / tile;
        return KIND == ORTHO_GRAM || KIND == ORTHO_POLY ? mt * (mt + 1) / 2 : mt * (q.n / tile);
    });
}

template <int T, int WAVES, int STAGES, int KIND>
static int product_as(const OrthoArgs& a, int64_t blocks, hipStream_t stream) {
    constexpr size_t lds = SplitTile<T, WAVES, STAGES>::LDS_BYTES;
    NERFX_OPT_IN_LDS((ortho_product_kernel<T, WAVES, STAGES, KIND>), lds);
    hipLaunchKernelGGL((ortho_product_kernel<T, WAVES, STAGES, KIND>), dim3((unsigned)blocks), dim3(64 * WAVES), lds, stream, a);
    return 0;
}

// The tile a product takes, by how many of them there are:
//  128  where whole rounds of them fill at least four fifths of the 256 CUs: half of the operand traffic of 64
//       (2048 x 2048 by 2048: 50 us; 55 in tiles of 64);
//  64   with two stages, five workgroups to a CU, where they would not: of a symmetric result 136 tiles of 128 take as long as
//       all 256 (50 us), 528 of 64 take 41; three and four stages hold fewer workgroups and take 44 and 50;
//  64   with eight stages where there is at most one to a CU: all of a K of 256 is on its way at once.
template <int KIND>
static int product(OrthoArgs& a, int pad, hipStream_t stream) {
    if (pad == 128) {
        const int64_t blocks = product_blocks<KIND>(a, 128), rounds = (blocks + 255) / 256;
        if (blocks * 5 >= rounds * 256 * 4) return product_as<128, 8, 4, KIND>(a, blocks, stream);
    }
    const int64_t blocks = product_blocks<KIND>(a, 64);
    return blocks <= 256 ? product_as<64, 4, 8, KIND>(a, blocks, stream) : product_as<64, 4, 2, KIND>(a, blocks, stream);
}

static int ortho_run(OrthoArgs& a, int pad, const float* coef, int steps, const OrthoScales& s, hipStream_t stream) {
    a.x_scale = s.x;
    a.growth = s.growth;
    int64_t blocks = lay_out(a, [](const OrthoMat& q) { return (int64_t)norm_parts(q); });
    hipLaunchKernelGGL(ortho_norm_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    blocks = lay_out(a, [](const OrthoMat& q) { return (int64_t)(q.m / PREP_TILE) * (q.n / PREP_TILE); });
    hipLaunchKernelGGL(ortho_prep_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    for (int k = 0; k < steps; ++k) {
        const float ca = coef[3 * k], cb = coef[3 * k + 1], cc = coef[3 * k + 2];
        a.beta = s.a / (s.x * s.x);
        if (int rc = product<ORTHO_GRAM>(a, pad, stream)) return rc;
        a.alpha = cb * (s.b / s.a);
        a.beta = cc * (s.b / s.a / s.a);
        if (int rc = product<ORTHO_POLY>(a, pad, stream)) return rc;
        a.from = k & 1; a.to = a.from ^ 1;
        const bool last = k == steps - 1;
        a.alpha = last ? ca / s.x : ca;                       // the last step leaves the scale
        a.beta = last ? 1.0f / (s.b * s.x) : 1.0f / s.b;
        if (int rc = last ? product<ORTHO_LAST>(a, pad, stream) : product<ORTHO_APPLY>(a, pad, stream)) return rc;
    }
    return launch_status("orthogonalisation kernels");
}

// Groups of at most ORTHO_GROUP matrices, one after the other in the same workspace (same stream: in order).
static int64_t group_bytes(const nerfx_matrix_t* mats, int count) {
    int64_t most = 0;
    OrthoArgs a;
    for (int k = 0; k < count; k += ORTHO_GROUP) {
        const int c = std::min(ORTHO_GROUP, count - k);
        most = std::max(most, fill_group(mats + k, c, tile_side(mats + k, c), a));
    }
    return most;
}

static int ortho_groups(const nerfx_matrix_t* mats, int count, OrthoArgs& a, const float* coef, int steps, void* workspace,
                        int64_t workspace_bytes, double lr, int adjust, hipStream_t stream) {
    NERFX_REQUIRE(steps >= 1 && steps <= ORTHO_MAX_STEPS && coef, "steps %d outside 1..%d, or no coefficients", steps, ORTHO_MAX_STEPS);
    NERFX_REQUIRE(a.eps > 0.f && std::isfinite(a.eps), "eps must be positive and finite");
    OrthoScales s;
    if (int rc = scales_for(coef, steps, s)) return rc;
    const int64_t need = group_bytes(mats, count);
    NERFX_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0), "workspace is NULL or not aligned to 16 bytes");
    NERFX_REQUIRE(workspace_bytes >= need, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    a.work = (char*)workspace;
    for (int k = 0; k < count; k += ORTHO_GROUP) {
        const int c = std::min(ORTHO_GROUP, count - k), tile = tile_side(mats + k, c);
        fill_group(mats + k, c, tile, a);
        if (a.count == 0) continue;
        for (int i = 0; i < a.count; ++i) {
            const double r = a.mat[i].rows, l = a.mat[i].cols;
            a.mat[i].lr = (float)(lr * (adjust == NERFX_LR_MATCH_RMS ? 0.2 * std::sqrt(std::max(r, l)) : std::sqrt(std::max(1.0, r / l))));
        }
        if (int rc = ortho_run(a, tile, coef, steps, s, stream)) return rc;
    }
    return 0;
}

}  // namespace nerfx

using namespace nerfx;

extern "C" int64_t nerfx_orthogonalize_workspace_bytes(const nerfx_matrix_t* mats, int count) {
    if (check_sizes(mats, count)) return -1;
    return group_bytes(mats, count);
}

extern "C" int nerfx_orthogonalize(const nerfx_matrix_t* mats, int count, int dtype, const float* coefficients, int steps,
                                   float eps, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_sizes(mats, count)) return rc;
    NERFX_REQUIRE(dtype == NERFX_TYPE_F32 || dtype == NERFX_TYPE_BF16 || dtype == NERFX_TYPE_F16, "unknown type %d", dtype);
    for (int k = 0; k < count; ++k)
        NERFX_REQUIRE(mats[k].rows == 0 || mats[k].cols == 0 || (mats[k].grad && mats[k].out), "matrix %d: grad / out is NULL", k);
    OrthoArgs a{};
    a.dtype = dtype; a.eps = eps;
    return ortho_groups(mats, count, a, coefficients, steps, workspace, workspace_bytes, 0, 0, (hipStream_t)stream);
}

extern "C" int nerfx_muon_step(const nerfx_matrix_t* mats, int count, double lr, double momentum, int nesterov, double weight_decay,
                               int adjust_lr, const float* coefficients, int steps, float eps, const float* grad_scale,
                               const float* found_inf, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_sizes(mats, count)) return rc;
    NERFX_REQUIRE(momentum >= 0 && momentum < 1, "momentum outside [0, 1)");
    NERFX_REQUIRE(lr >= 0 && std::isfinite(lr) && weight_decay >= 0 && std::isfinite(weight_decay), "lr / weight_decay negative or not finite");
    NERFX_REQUIRE(adjust_lr == NERFX_LR_ORIGINAL || adjust_lr == NERFX_LR_MATCH_RMS, "unknown learning-rate rule %d", adjust_lr);
    for (int k = 0; k < count; ++k)
        NERFX_REQUIRE(mats[k].rows == 0 || mats[k].cols == 0 || (mats[k].grad && mats[k].momentum && mats[k].param),
                      "matrix %d: grad / momentum / param is NULL", k);
    OrthoArgs a{};
    a.muon = 1; a.nesterov = nesterov != 0; a.momentum = (float)momentum; a.rest = (float)(1 - momentum);
    a.decay = (float)(1 - lr * weight_decay); a.eps = eps;
    a.grad_scale = grad_scale; a.found_inf = found_inf;
    return ortho_groups(mats, count, a, coefficients, steps, workspace, workspace_bytes, lr, adjust_lr, (hipStream_t)stream);
}
