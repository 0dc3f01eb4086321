// Orthogonalised updates: Newton-Schulz steps on a group of matrices, and the optimiser step around them.
//
// For a matrix G (rows x cols), X = G / max(|G|_F, eps), transposed if it is taller than wide (m <= n), then
// per step   A = X X^T,   B = b A + c A A,   X <- a X + B X
// which takes every singular value s to a s + b s^3 + c s^5 and leaves the singular vectors.  The result goes
// back in G's own orientation.  A whole group of matrices of any shapes shares every launch: a launch's grid
// is the concatenation of the matrices' tiles, and a workgroup finds its matrix in a table.  The first launch has the
// table in its arguments and leaves it in the workspace, so nothing is copied to the device and the call can be captured;
// the others read it there.
//
// Groups of small matrices (sides up to 64 and 256) take one launch altogether: see ortho_small_kernel.
#include <algorithm>
#include <cmath>

#include "lds_dma.hpp"
#include "split16.hpp"

namespace nerfx {

// Four values of a row of the caller's, which begins wherever it begins.
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

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
struct OrthoCall {
    const float* grad_scale;
    const float* found_inf;
    float momentum, rest, decay;                // rest: 1 - momentum, decay: 1 - lr * weight_decay
    float eps, x_scale;
    int32_t growth;                             // the steps together grow a singular value by at most 2^growth
    int32_t count, nesterov, dtype, muon;
};
enum { ORTHO_NORM_GRID, ORTHO_PREP_GRID, ORTHO_SYM_GRID, ORTHO_FULL_GRID, ORTHO_GRIDS };
struct OrthoTable {
    OrthoMat mat[ORTHO_GROUP];
    int32_t first[ORTHO_GRIDS][ORTHO_GROUP];    // first block of each matrix in a launch; INT_MAX behind the last
    OrthoCall call;
};
static_assert(sizeof(OrthoTable) <= 3584, "the table has to fit the kernel arguments");
constexpr int64_t ORTHO_TABLE_BYTES = 3584;     // at the start of the workspace

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
// What is orthogonalised: the gradient, or the optimiser's mix of it and the (new) momentum.
__device__ __forceinline__ float update_of(const OrthoCall& a, float g, float mom, float unscale) {
    if (!a.muon) return g;
    return a.nesterov ? fmaf(a.momentum, mom, a.rest * (g * unscale)) : mom;
}
__device__ __forceinline__ float update_at(const OrthoCall& a, const OrthoMat& q, int64_t i, float unscale) {
    return update_of(a, load_as_float(q.grad, i, a.dtype), a.muon ? q.momentum[i] : 0.f, unscale);
}

// The matrix that this block works on, and the block's number within it.  (All of a row of the table is read at
// once: walking it would wait for each entry in turn.)
__device__ __forceinline__ int which_matrix(const OrthoTable& t, int grid, int b, int& block) {
    int k = 0, start = 0;
#pragma unroll
    for (int i = 1; i < ORTHO_GROUP; ++i) {
        const int f = t.first[grid][i];
        if (b >= f) { k = i; start = f; }
    }
    block = b - start;
    return k;
}
enum { ORTHO_GRAM, ORTHO_POLY, ORTHO_APPLY, ORTHO_LAST };

// Matrices with a side of up to 16 are kept and multiplied in fp32: sums of so few terms leave nothing for the 2^-23 of two halves to
// average out in (8 x 60: 6e-7 off float64, in halves 1.0e-6), and there is next to nothing to compute.  X and X^T, A and B take
// the same places, an element its 4 bytes.
__host__ __device__ inline bool ortho_tiny(const OrthoMat& q) { return (q.rows < q.cols ? q.rows : q.cols) <= 16; }

// 16 rows of P times 16 rows of Q, over values k0, k0 + 1 .. + 15, then step values on, up to K (a multiple of 16): element i of the
// result is that of P's row 4 (lane / 16) + i and Q's row lane % 16.
__device__ __forceinline__ f32x4_t tiny_product(const float* P, int64_t p_pitch, const float* Q, int64_t q_pitch, int k0, int step, int K) {
    const int lane = threadIdx.x & 63;
    P += (lane & 15) * p_pitch + 4 * (lane >> 4);
    Q += (lane & 15) * q_pitch + 4 * (lane >> 4);
    f32x4_t sum[4] = {};
    for (int k = k0; k < K; k += step) {
        const f32x4_t a = *(const f32x4_t*)(P + k), b = *(const f32x4_t*)(Q + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], sum[j], 0, 0, 0);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
// The parts of a sum that a workgroup's waves have, added up: in the first wave.
template <int WAVES>
__device__ __forceinline__ f32x4_t tiny_sum(f32x4_t v, float* lds) {
    *(f32x4_t*)(lds + 4 * threadIdx.x) = v;
    __syncthreads();
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
    if (threadIdx.x < 64)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += *(const f32x4_t*)(lds + 4 * (threadIdx.x + 64 * w));
    return sum;
}

// Momentum, and partial sums of squares of what is orthogonalised.  In double: a fp32 gradient's square
// neither overflows nor vanishes there, and a sum of 2^30 of them keeps fp32's precision.
__global__ __launch_bounds__(256) void ortho_norm_kernel(const OrthoTable t, char* work) {
    int b;
    const OrthoMat q = t.mat[which_matrix(t, ORTHO_NORM_GRID, blockIdx.x, b)];
    const OrthoCall& a = t.call;
    if (blockIdx.x == 0)                                       // for the launches behind this one
        for (int i = threadIdx.x; i < (int)(sizeof(OrthoTable) / 4); i += 256) ((uint32_t*)work)[i] = ((const uint32_t*)&t)[i];
    const int64_t total = (int64_t)q.rows * q.cols;
    const int parts = norm_parts(q);
    const bool skip = a.found_inf && *a.found_inf != 0.f;
    const float unscale = a.grad_scale ? 1.0f / *a.grad_scale : 1.0f;
    double acc = 0;
    const int64_t step = (int64_t)parts * 256;
    constexpr int AT_ONCE = 8;                                 // loads in flight: a momentum's store would end the next one's
    for (int64_t i0 = (int64_t)b * 256 + threadIdx.x; i0 < total; i0 += AT_ONCE * step) {
        float g[AT_ONCE], mom[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int64_t i = min(i0 + j * step, total - 1);
            g[j] = load_as_float(q.grad, i, a.dtype);
            mom[j] = a.muon ? q.momentum[i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            if (i0 + j * step >= total) break;
            float u = g[j];
            if (a.muon) {
                if (!skip) q.momentum[i0 + j * step] = mom[j] = fmaf(a.momentum, mom[j], a.rest * (g[j] * unscale));
                u = update_of(a, g[j], mom[j], unscale);
            }
            acc = fma((double)u, (double)u, acc);
        }
    }
    __shared__ double part[4];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)(work + ortho_sums_at(q)))[b] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X and X^T from what is orthogonalised: one 64 x 64 tile of X per block, through LDS, zeros in the padding.
__global__ __launch_bounds__(256) void ortho_prep_kernel(const OrthoTable* __restrict__ t, char* __restrict__ work) {
    int b;
    const OrthoMat q = t->mat[which_matrix(*t, ORTHO_PREP_GRID, blockIdx.x, b)];
    const OrthoCall a = t->call;
    __shared__ float tile[PREP_TILE][PREP_TILE + 1];
    const float unscale = a.grad_scale ? 1.0f / *a.grad_scale : 1.0f;
    const int x0 = b / (q.n / PREP_TILE) * PREP_TILE, y0 = b % (q.n / PREP_TILE) * PREP_TILE;   // of X
    // G's rows run along X's columns, or, if G is tall, along X's rows
    const int r0 = q.tall ? y0 : x0, c0 = q.tall ? x0 : y0;
    float own[PREP_TILE * PREP_TILE / 256];                    // on its way while the norm is put together
#pragma unroll
    for (int j = 0; j < PREP_TILE * PREP_TILE / 256; ++j) {
        const int e = threadIdx.x + 256 * j, r = min(r0 + e / PREP_TILE, q.rows - 1), c = min(c0 + e % PREP_TILE, q.cols - 1);
        own[j] = update_at(a, q, (int64_t)r * q.cols + c, unscale);
    }
    const double* sums = (const double*)(work + ortho_sums_at(q));
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
    if (b == 0 && threadIdx.x == 0) *(int*)(work + ortho_lift_at(q)) = lift;
#pragma unroll
    for (int j = 0; j < PREP_TILE * PREP_TILE / 256; ++j) {
        const int e = threadIdx.x + 256 * j, r = e / PREP_TILE, c = e % PREP_TILE;
        const float v = r0 + r < q.rows && c0 + c < q.cols ? (float)(own[j] * factor) : 0.f;
        if (q.tall) tile[c][r] = v; else tile[r][c] = v;
    }
    __syncthreads();
    char* x = work + q.base;
    char* xt = work + ortho_xt_at(q, 0);
    for (int e = threadIdx.x; e < PREP_TILE * PREP_TILE / 4; e += 256) {
        const int r = e / (PREP_TILE / 4), k = (e % (PREP_TILE / 4)) * 4;
        const float row[4] = {tile[r][k], tile[r][k + 1], tile[r][k + 2], tile[r][k + 3]};
        const float col[4] = {tile[k][r], tile[k + 1][r], tile[k + 2][r], tile[k + 3][r]};
        if (ortho_tiny(q)) {
            *(f32x4_t*)((float*)x + (int64_t)(x0 + r) * q.n + y0 + k) = (f32x4_t){row[0], row[1], row[2], row[3]};
            *(f32x4_t*)((float*)xt + (int64_t)(y0 + r) * q.m + x0 + k) = (f32x4_t){col[0], col[1], col[2], col[3]};
        } else {
            split_store4(x, x0 + r, y0 + k, q.n, row);
            split_store4(xt, y0 + r, x0 + k, q.m, col);
        }
    }
}

// ---- the products ---------------------------------------------------------------------------------------------------
// One T x T tile of P Q^T for two row-major split matrices with rows along K: 2 x WAVES / 2 waves, each its part of
// the tile.  A stage is one 32-wide block of K of both operands; STAGES of them lie in LDS, all but one of them on
// their way while one is worked on (LDS-DMA: no registers hold them).  16-byte chunk c of row r lies at place
// c ^ (r / 2 % 8), so that the sixteen rows a ds_read_b128 phase touches (256 bytes of banks) lie apart; LDS-DMA
// writes lane after lane, so it is the source address that is permuted.
// Bound by LDS reads where there are many tiles: a stage of a tile of 64 is 32 KB of fragments for its four waves and 192 cycles of
// matrix instructions, of a tile of 128 96 KB and 768 cycles; LDS gives a CU at most 128 bytes a cycle.  (2048 x 2048 by 2048: 49.9 us, 50.2
// without loads of stages, 41.6 without products.)  Rows of X are not divided over workgroups: a matrix with a side of up to 64 has one for
// its Gram matrix, which goes over the other side by itself (64 x 32768: 1.4 ms, 16 x 32768: 0.8).
template <int T, int WAVES, int STAGES>
struct SplitTile {
    static constexpr int FP = T / 64, FQ = T / (16 * WAVES); // 32 x 32 fragments per wave and side
    static constexpr int LOADS = T / (8 * WAVES);            // per wave, stage and operand
    static constexpr int STAGE_BYTES = 2 * T * SPLIT_BLOCK_BYTES;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
    static_assert(STAGES >= 2 && STAGES <= 8 && 2 * LOADS * (STAGES - 1) < 64, "waits of landed()");
    float16_t_ acc[FP][FQ], cross[FP][FQ];

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
    // hi hi goes into sums of its own: what rounds each time is then K / 16 additions at the result's size, and the two thirds
    // that the cross terms are round at theirs, 2^-11 of it.  (In one sum a Gram matrix of rows of 1,500 was 1e-6 off.)
    __device__ __forceinline__ void multiply(const Frags& f) {
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j) {
                    if (t == 1) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[i], f.qh[j], acc[i][j], 0, 0, 0);
                    else cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(t == 2 ? f.pl[i] : f.ph[i], t == 0 ? f.ql[j] : f.qh[j],
                                                                              cross[i][j], 0, 0, 0);
                }
    }

    // `seen(kb, stage)` is called once per stage, while it is in LDS.
    template <class Seen>
    __device__ __forceinline__ void run(char* lds, const char* P, const char* Q, int K, Seen seen) {
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
                for (int e = 0; e < 16; ++e) acc[i][j][e] = cross[i][j][e] = 0.f;
#pragma unroll
        for (int kb = 0; kb < STAGES; ++kb)
            if (kb < steps) fetch(kb);
        Frags f0, f1;
        if (whole(K)) {                                      // all there is, in LDS at once: no waits between the stages
            landed<0>();
            read(f0, lds, 0, wave, lane);
            read(f1, lds, 1, wave, lane);
            for (int kb = 0; kb < steps - 1; ++kb) {
                seen(kb, lds + kb * STAGE_BYTES);
                Frags g0, g1;
                read(g0, lds + (kb + 1) * STAGE_BYTES, 0, wave, lane);
                read(g1, lds + (kb + 1) * STAGE_BYTES, 1, wave, lane);
                multiply(f0);
                multiply(f1);
                f0 = g0;
                f1 = g1;
            }
            seen(steps - 1, lds + (steps - 1) * STAGE_BYTES);
            multiply(f0);
            multiply(f1);
            add_cross();
            return;
        }
        wait(steps - 1);
        read(f0, lds, 0, wave, lane);
        for (int kb = 0; kb < steps - 1; ++kb) {             // fragments are read one half stage ahead of their use
            read(f1, lds + (kb % STAGES) * STAGE_BYTES, 1, wave, lane);
            seen(kb, lds + (kb % STAGES) * STAGE_BYTES);
            multiply(f0);
            wait(min(STAGES - 2, steps - 2 - kb));           // stage kb + 1 is there, and every wave has read all of stage kb,
            if (kb + STAGES < steps) fetch(kb + STAGES);     // whose place this one takes
            read(f0, lds + ((kb + 1) % STAGES) * STAGE_BYTES, 0, wave, lane);
            multiply(f1);
        }
        read(f1, lds + ((steps - 1) % STAGES) * STAGE_BYTES, 1, wave, lane);
        seen(steps - 1, lds + ((steps - 1) % STAGES) * STAGE_BYTES);
        multiply(f0);
        multiply(f1);
        add_cross();
    }
    // Whether rows of K values lie in LDS altogether.
    static __device__ __forceinline__ bool whole(int K) { return STAGES == 8 && K <= STAGES * SPLIT_BLOCK; }
    // In a stage: its values k .. k + 3 of Q's row r (of the tile).
    static __device__ __forceinline__ Split4 here(const char* stage, int r, int k) {
        const char* row = stage + (T + r) * SPLIT_BLOCK_BYTES + 2 * (k & 4);
        const int turn = (T + r) >> 1 & 7;
        return {*(const half4_t*)(row + (k / 8 ^ turn) * 16), *(const half4_t*)(row + (k / 8 + 4 ^ turn) * 16)};
    }
    __device__ __forceinline__ void add_cross() {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] += cross[i][j];
    }
    // where in the tile a wave's part begins
    static __device__ __forceinline__ int row_of(int wave) { return wave / (WAVES / 2) * (T / 2); }
    static __device__ __forceinline__ int col_of(int wave) { return wave % (WAVES / 2) * (2 * T / WAVES); }
};

// The result for X's row and column, into the caller's matrix.
__device__ __forceinline__ void ortho_out(const OrthoCall& a, const OrthoMat& q, int row, int col, float v) {
    const int r = q.tall ? col : row, c = q.tall ? row : col;
    if (r >= q.rows || c >= q.cols) return;
    const int64_t at = (int64_t)r * q.cols + c;
    if (a.muon) q.param[at] = fmaf(-q.lr, v, q.param[at] * a.decay);
    else store_from_float(q.out, at, v, a.dtype);
}
// Those for four neighbours in the caller's row r: 16 bytes, wherever the row begins.
__device__ __forceinline__ void ortho_out4(const OrthoCall& a, const OrthoMat& q, int r, int c, f32x4_t v) {
    const int64_t at = (int64_t)r * q.cols + c;
    if (c + 4 > q.cols) {
        for (int i = 0; c + i < q.cols; ++i) {
            if (a.muon) q.param[at + i] = fmaf(-q.lr, v[i], q.param[at + i] * a.decay);
            else store_from_float(q.out, at + i, v[i], a.dtype);
        }
    } else if (a.muon) {
        f32x4_any_t* p = (f32x4_any_t*)(q.param + at);
        f32x4_any_t w = *p;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fmaf(-q.lr, v[i], w[i] * a.decay);
        *p = w;
    } else if (a.dtype == NERFX_TYPE_F32) {
        *(f32x4_any_t*)((float*)q.out + at) = v;
    } else if (a.dtype == NERFX_TYPE_F16) {
        *(f16x4_any_t*)((_Float16*)q.out + at) = (f16x4_any_t){(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
        *(bf16x4_any_t*)((__bf16*)q.out + at) = (bf16x4_any_t){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
}

// A wave's 32 x 32 results on their way to a split matrix and to its transpose.  They go through LDS, one orientation after the
// other, and leave as whole lines of 128 bytes: stored from the registers, in pieces of 2 and 8 bytes, they were a quarter of a
// small matrix's time (a field's six: 129 us, 122 so).
struct SplitLines {
    static constexpr int PITCH = SPLIT_BLOCK_BYTES + 16, BYTES = 32 * PITCH;
    char* lds;
    half4_t hi[4], lo[4];

    // Rows 8 e + 4 (lane / 32) .. + 3 of column lane % 32.
    __device__ __forceinline__ void take(int e, const float (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            _Float16 h, l;
            split16(v[k], h, l);
            hi[e][k] = h;
            lo[e][k] = l;
        }
    }
    __device__ __forceinline__ void store(char* dst, int row, int col, int width) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                char* p = lds + (8 * e + 4 * (lane >> 5) + k) * PITCH + 2 * (lane & 31);
                *(_Float16*)p = hi[e][k];
                *(_Float16*)(p + 64) = lo[e][k];
            }
        leave(dst, row, col, width);
    }
    __device__ __forceinline__ void store_transposed(char* dst, int row, int col, int width) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            char* p = lds + (lane & 31) * PITCH + 2 * (8 * e + 4 * (lane >> 5));
            *(half4_t*)p = hi[e];
            *(half4_t*)(p + 64) = lo[e];
        }
        leave(dst, row, col, width);
    }

    // The same for the caller's matrix, in fp32 and as that lies.
    __device__ __forceinline__ void take_out(int e, const float (&v)[4], bool tall) {
        const int lane = threadIdx.x & 63, row = 8 * e + 4 * (lane >> 5);
        if (tall) {
            *(f32x4_t*)(lds + (lane & 31) * PITCH + 4 * row) = (f32x4_t){v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) *(float*)(lds + (row + k) * PITCH + 4 * (lane & 31)) = v[k];
        }
    }
    // row, col: of X.
    __device__ __forceinline__ void leave_out(const OrthoCall& a, const OrthoMat& q, int row, int col) const {
        const int lane = threadIdx.x & 63, c = (q.tall ? row : col) + 4 * (lane & 7);
        wave_lds_in_order();
        if (c < q.cols) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 8 * i + (lane >> 3), r = (q.tall ? col : row) + at;
                if (r < q.rows) ortho_out4(a, q, r, c, *(const f32x4_t*)(lds + at * PITCH + 16 * (lane & 7)));
            }
        }
        wave_lds_in_order();
    }

private:
    __device__ __forceinline__ void leave(char* dst, int row, int col, int width) const {
        const int lane = threadIdx.x & 63;
        wave_lds_in_order();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 3), piece = 16 * (lane & 7);
            *(u32x4_t*)(split_at(dst, row + r, col, width) + piece) = *(const u32x4_t*)(lds + r * PITCH + piece);
        }
        wave_lds_in_order();
    }
};

// Number t of a lower triangle's tiles, row after row -> (row, column).
__device__ __forceinline__ void triangle_at(int t, int& i, int& j) {
    i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    j = t - i * (i + 1) / 2;
}

// A tile of ortho_product_kernel for a matrix in fp32: the first 16 rows are all there are.
template <int T, int WAVES, int KIND>
__device__ __forceinline__ void ortho_tiny_product(const OrthoTable& t, const OrthoMat& q, char* work, char* lds, int ti, int tj, float alpha,
                                                   float beta, int from) {
    static_assert(T == 16 * WAVES, "a wave has 16 columns");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = 4 * (lane >> 4);
    float *X = (float*)(work + q.base), *A = (float*)(work + ortho_a_at(q)), *B = (float*)(work + ortho_b_at(q));
    if (ti != 0 || ((KIND == ORTHO_GRAM || KIND == ORTHO_POLY) && tj != 0)) return;
    const int lift = *(const int*)(work + ortho_lift_at(q));
    if constexpr (KIND == ORTHO_GRAM) {
        const f32x4_t v = tiny_sum<WAVES>(tiny_product(X, q.n, X, q.n, 16 * wave, 16 * WAVES, q.n), (float*)lds);
        if (wave == 0)                                         // symmetric: a row for a column
            *(f32x4_t*)(A + (lane & 15) * q.m + row) = v * ldexpf(beta, -2 * lift);
    } else if constexpr (KIND == ORTHO_POLY) {
        if (wave != 0) return;
        const f32x4_t v = tiny_product(A, q.m, A, q.m, 0, 16, 16), own = *(const f32x4_t*)(A + (lane & 15) * q.m + row);
        f32x4_t b;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = fmaf(beta, v[i], alpha * own[i]);
        *(f32x4_t*)(B + (lane & 15) * q.m + row) = b;
    } else {
        const int col = tj * T + 16 * wave + (lane & 15);
        const float* XT = (const float*)(work + ortho_xt_at(q, from));
        const f32x4_t v = tiny_product(B, q.m, XT + (int64_t)(tj * T + 16 * wave) * q.m, q.m, 0, 16, 16);
        const f32x4_t own = *(const f32x4_t*)(XT + (int64_t)col * q.m + row);
        const float xa = KIND == ORTHO_LAST ? ldexpf(alpha, -lift) : alpha, xb = KIND == ORTHO_LAST ? ldexpf(beta, -lift) : beta;
        f32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaf(xb, v[i], xa * own[i]);
        if constexpr (KIND == ORTHO_APPLY) {
            *(f32x4_t*)((float*)(work + ortho_xt_at(q, from ^ 1)) + (int64_t)col * q.m + row) = x;
#pragma unroll
            for (int i = 0; i < 4; ++i) X[(int64_t)(row + i) * q.n + col] = x[i];
        } else {
            if (t.call.found_inf && *t.call.found_inf != 0.f) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) ortho_out(t.call, q, row + i, col, x[i]);
        }
    }
}

template <int T, int WAVES, int STAGES, int KIND>
__global__ __launch_bounds__(64 * WAVES) void ortho_product_kernel(const OrthoTable* __restrict__ t, char* __restrict__ work, float alpha,
                                                                float beta, int from) {
    extern __shared__ __align__(16) char lds[];
    constexpr bool SYM = KIND == ORTHO_GRAM || KIND == ORTHO_POLY;       // the result is symmetric: half of the tiles
    int b;
    const OrthoMat q = t->mat[which_matrix(*t, SYM ? ORTHO_SYM_GRID : ORTHO_FULL_GRID, xcd_place(), b)];
    int ti, tj;
    if constexpr (SYM) {
        triangle_at(b, ti, tj);
    } else {
        ti = b % (q.m / T);
        tj = b / (q.m / T);
    }
    char* X = work + q.base;
    char* A = work + ortho_a_at(q);
    char* B = work + ortho_b_at(q);
    if (ortho_tiny(q)) {
        ortho_tiny_product<T, WAVES, KIND>(*t, q, work, lds, ti, tj, alpha, beta, from);
        return;
    }
    const char* P = KIND == ORTHO_GRAM ? X : KIND == ORTHO_POLY ? A : B;
    const char* Q = KIND == ORTHO_GRAM ? X : KIND == ORTHO_POLY ? A : work + ortho_xt_at(q, from);
    const int K = KIND == ORTHO_GRAM ? q.n : q.m;
    using Tile = SplitTile<T, WAVES, STAGES>;
    Tile tile;
    // element (row, col) of a 32 x 32 accumulator: col = lane % 32, row = 8 (e / 4) + 4 (lane / 32) + e % 4
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the element itself, A[row][col] = A[col][row] or X[row][col] = X^T[col][row], comes by in one of the stages
    Split4 own[Tile::FP][Tile::FQ][4];
    auto keep_own = [&](int kb, const char* stage) {
        if constexpr (KIND != ORTHO_GRAM) {
#pragma unroll
            for (int i = 0; i < Tile::FP; ++i) {
                if (kb != (ti * T + Tile::row_of(wave)) / SPLIT_BLOCK + i) continue;
#pragma unroll
                for (int j = 0; j < Tile::FQ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        own[i][j][e] = Tile::here(stage, Tile::col_of(wave) + 32 * j + (lane & 31), 4 * (lane >> 5) + 8 * e);
            }
        }
    };
    int lift = 0;                                                        // see the kernel that made X
    if constexpr (KIND == ORTHO_GRAM || KIND == ORTHO_LAST) lift = *(const int*)(work + ortho_lift_at(q));
    tile.run(lds, P + (int64_t)ti * T * K * 4, Q + (int64_t)tj * T * K * 4, K, keep_own);
    if constexpr (KIND == ORTHO_GRAM || KIND == ORTHO_LAST) {
        beta = ldexpf(beta, KIND == ORTHO_GRAM ? -2 * lift : -lift);
        alpha = ldexpf(alpha, -lift);
    }
    const OrthoCall a = t->call;
    const bool skip = KIND == ORTHO_LAST && a.found_inf && *a.found_inf != 0.f;
    __syncthreads();                                                     // the stages have been read: their place is the waves' own now
    SplitLines lines{lds + wave * SplitLines::BYTES};
    static_assert(WAVES * SplitLines::BYTES <= Tile::LDS_BYTES, "a place for each wave");
#pragma unroll
    for (int i = 0; i < Tile::FP; ++i)
#pragma unroll
        for (int j = 0; j < Tile::FQ; ++j) {
            const int row0 = ti * T + Tile::row_of(wave) + 32 * i + 4 * (lane >> 5);
            const int col = tj * T + Tile::col_of(wave) + 32 * j + (lane & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v[4];
                if constexpr (KIND == ORTHO_GRAM) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = beta * tile.acc[i][j][4 * e + k];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[k] = fmaf(beta, tile.acc[i][j][4 * e + k], alpha * ((float)own[i][j][e].hi[k] + (float)own[i][j][e].lo[k]));
                }
                if constexpr (KIND != ORTHO_LAST) lines.take(e, v);
                else lines.take_out(e, v, q.tall);
            }
            if constexpr (KIND == ORTHO_LAST) {                // into the caller's matrix
                if (!skip) lines.leave_out(a, q, row0 - 4 * (lane >> 5), col - (lane & 31));
            }
            if constexpr (KIND != ORTHO_LAST) {
                const int r = row0 - 4 * (lane >> 5), c = col - (lane & 31);
                char* dst = KIND == ORTHO_GRAM ? A : KIND == ORTHO_POLY ? B : X;
                lines.store(dst, r, c, SYM ? q.m : q.n);
                if (!SYM || ti != tj) lines.store_transposed(SYM ? dst : work + ortho_xt_at(q, from ^ 1), c, r, q.m);
            }
        }
}

// ---- small matrices: one launch ---------------------------------------------------------------------------------------
// A matrix whose smaller side is at most 64 and whose larger one is at most 256 fits in LDS with everything that the steps
// need (X, X^T, A and B: 160 KB), so that a workgroup takes all of its steps by itself.  What bounds the other way there is
// the number of launches: 17 of 6 us each.  Only for groups of nothing but such matrices; in a group with a larger one they
// ride along in its launches.
//
// A row takes 128 bytes for every 32 of its columns, as in memory; 16-byte chunk c (of a pair of blocks: 0 .. 15) of row r lies at
// place c ^ (r % 16), so that the sixteen rows of a read phase touch different banks.  Every matrix and row begins at a multiple
// of 256 bytes, so that an address is a per-lane one with a constant's bits flipped.
constexpr int SMALL_M = 64, SMALL_N = 256, SMALL_WAVES = 8;

__device__ __forceinline__ int small_at(int r, int k, int pitch) {             // of the hi half; the lo half: ^ 64
    return r * pitch + (k >> 6) * 256 + ((((k >> 5 & 1) * 8 + (k >> 3 & 3)) ^ (r & 15)) * 16) + (k & 7) * 2;
}
__device__ __forceinline__ void small_put(char* m, int at, float v) {
    _Float16 hi, lo;
    split16(v, hi, lo);
    *(_Float16*)(m + at) = hi;
    *(_Float16*)(m + (at ^ 64)) = lo;
}
// 32 x 32 of P Q^T from rows p0 .. of P and q0 .. of Q; K a multiple of 64.
__device__ __forceinline__ float16_t_ small_product(const char* P, int p0, int p_pitch, const char* Q, int q0, int q_pitch, int K) {
    const int lane = threadIdx.x & 63, p = p0 + (lane & 31), q = q0 + (lane & 31), h = lane >> 5;
    const int pv = p * p_pitch + ((h ^ (p & 15)) * 16), qv = q * q_pitch + ((h ^ (q & 15)) * 16);
    float16_t_ main, cross, low;
#pragma unroll
    for (int e = 0; e < 16; ++e) main[e] = cross[e] = low[e] = 0.f;
    for (int kb = 0; kb < K / 64; ++kb) {
        half8_t ph[4], pl[4], qh[4], ql[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int c = (s >> 1) * 128 + (s & 1) * 32;
            ph[s] = *(const half8_t*)(P + kb * 256 + (pv ^ c)); pl[s] = *(const half8_t*)(P + kb * 256 + (pv ^ (c + 64)));
            qh[s] = *(const half8_t*)(Q + kb * 256 + (qv ^ c)); ql[s] = *(const half8_t*)(Q + kb * 256 + (qv ^ (c + 64)));
        }
#pragma unroll
        // Here lo lo is not left out: it costs nothing (latency bounds these products), and with a few elements to a sum there
        // is little for its 2^-24 to average out in.
        for (int s = 0; s < 4; ++s) {
            cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[s], ql[s], cross, 0, 0, 0);
            main = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[s], qh[s], main, 0, 0, 0);
            cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[s], qh[s], cross, 0, 0, 0);
            low = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[s], ql[s], low, 0, 0, 0);
        }
    }
    return main + (cross + low);
}

struct OrthoSteps { float coef[3 * ORTHO_MAX_STEPS]; int32_t steps; float sx, sa, sb; };

// What ortho_small_kernel does from there on, for a matrix in fp32.  In LDS: X (16 x n), X^T (n x 16), A and B, rows four values
// further apart than they are long; and a place for sums.  All of it is zeros.
__device__ __forceinline__ void ortho_tiny_steps(const OrthoTable& t, const OrthoSteps& c, const OrthoMat& q, char* lds, int lift,
                                                 double factor, float unscale, bool skip) {
    constexpr int PITCH = 20;
    const OrthoCall& a = t.call;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = 64 * SMALL_WAVES, total = q.rows * q.cols;
    const int xp = q.n + 4, row = 4 * (lane >> 4);
    float *X = (float*)lds, *XT = X + 16 * xp, *A = XT + q.n * PITCH, *B = A + 16 * PITCH, *sums = B + 16 * PITCH;
    __syncthreads();                                           // what the norm was put together in is cleared
    for (int i = tid; i < total; i += threads) {
        const int r = i / q.cols, k = i - r * q.cols;
        const float v = (float)(update_at(a, q, i, unscale) * factor);
        X[(q.tall ? k : r) * xp + (q.tall ? r : k)] = v;
        XT[(q.tall ? r : k) * PITCH + (q.tall ? k : r)] = v;
    }
    __syncthreads();
    for (int step = 0; step < c.steps; ++step) {
        const bool last = step == c.steps - 1;
        const f32x4_t gram = tiny_sum<SMALL_WAVES>(tiny_product(X, xp, X, xp, 16 * wave, 16 * SMALL_WAVES, q.n), sums);
        if (wave == 0) {                                       // LDS of one wave: no barrier between A and what reads it
            *(f32x4_t*)(A + (lane & 15) * PITCH + row) = gram * ldexpf(c.sa / (c.sx * c.sx), -2 * lift);
            wave_lds_in_order();
            const f32x4_t v = tiny_product(A, PITCH, A, PITCH, 0, 16, 16), own = *(const f32x4_t*)(A + (lane & 15) * PITCH + row);
            const float pa = c.coef[3 * step + 1] * (c.sb / c.sa), pb = c.coef[3 * step + 2] * (c.sb / c.sa / c.sa);
            f32x4_t b;
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = fmaf(pb, v[i], pa * own[i]);
            *(f32x4_t*)(B + (lane & 15) * PITCH + row) = b;
        }
        __syncthreads();
        const float xa = last ? ldexpf(c.coef[3 * step] / c.sx, -lift) : c.coef[3 * step];
        const float xb = last ? ldexpf(1.0f / (c.sb * c.sx), -lift) : 1.0f / c.sb;
        for (int c0 = 16 * wave; c0 < q.n; c0 += 16 * SMALL_WAVES) {               // a wave's own rows of X^T and columns of X
            float* at = XT + (c0 + (lane & 15)) * PITCH + row;
            const f32x4_t v = tiny_product(B, PITCH, XT + c0 * PITCH, PITCH, 0, 16, 16), own = *(const f32x4_t*)at;
            f32x4_t x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(xb, v[i], xa * own[i]);
            wave_lds_in_order();
            *(f32x4_t*)at = x;
#pragma unroll
            for (int i = 0; i < 4; ++i) X[(row + i) * xp + c0 + (lane & 15)] = x[i];
        }
        __syncthreads();
    }
    if (skip) return;
    for (int i = tid; i < total; i += threads) {
        const int r = i / q.cols, k = i - r * q.cols;
        ortho_out(a, q, q.tall ? k : r, q.tall ? r : k, X[(q.tall ? k : r) * xp + (q.tall ? r : k)]);
    }
}

__global__ __launch_bounds__(64 * SMALL_WAVES) void ortho_small_kernel(const OrthoTable t, const OrthoSteps c) {
    extern __shared__ __align__(256) char lds[];
    const OrthoMat q = t.mat[blockIdx.x];
    const OrthoCall& a = t.call;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total = q.rows * q.cols, threads = 64 * SMALL_WAVES, xp = q.n * 4, side = min(q.rows, q.cols);
    char *A = lds, *B = lds + SMALL_M * 256, *XT = lds + 2 * SMALL_M * 256, *X = XT + q.n * 256;
    const bool skip = a.found_inf && *a.found_inf != 0.f;
    const float unscale = a.grad_scale ? 1.0f / *a.grad_scale : 1.0f;
    // zeros: what lies behind the matrix's sides stays as it is
    for (int i = tid; i < (2 * SMALL_M * 256 + q.n * 512) / 16; i += threads) *(u32x4_t*)(lds + 16 * i) = (u32x4_t){0, 0, 0, 0};
    // momentum and norm, as in the kernels above
    double acc = 0;
    for (int i = tid; i < total; i += threads) {
        if (a.muon && !skip)
            q.momentum[i] = fmaf(a.momentum, q.momentum[i], a.rest * (((const float*)q.grad)[i] * unscale));
        const double u = update_at(a, q, i, unscale);
        acc = fma(u, u, acc);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    __syncthreads();
    double* part = (double*)B;
    if (lane == 0) part[wave] = acc;
    __syncthreads();
    double sum = 0;
#pragma unroll
    for (int w = 0; w < SMALL_WAVES; ++w) sum += part[w];
    const double norm = sqrt(sum);
    double factor = (double)a.x_scale / (norm < (double)a.eps ? (double)a.eps : norm);
    int lift = 0;
    if (norm < (double)a.eps) lift = max(0, min(120, norm > 0 ? ilogb((double)a.eps / norm) - a.growth : 0));
    factor = ldexp(factor, lift);
    __syncthreads();
    if (tid < SMALL_WAVES) part[tid] = 0;
    if (side <= 16) {
        ortho_tiny_steps(t, c, q, lds, lift, factor, unscale, skip);
        return;
    }
    for (int i = tid; i < total; i += threads) {
        const int r = i / q.cols, k = i - r * q.cols;
        const float v = (float)(update_at(a, q, i, unscale) * factor);
        small_put(X, small_at(q.tall ? k : r, q.tall ? r : k, xp), v);
        small_put(XT, small_at(q.tall ? r : k, q.tall ? k : r, 256), v);
    }
    __syncthreads();
    // a wave's 32 x 32 part of A and B: four waves have one, those behind the matrix's side none
    const int row0 = 32 * (wave >> 1 & 1), col0 = 32 * (wave & 1);
    const bool square = wave < 4 && row0 < side && col0 < side;
    const float gram = ldexpf(c.sa / (c.sx * c.sx), -2 * lift);
    // elements row .. row + 3 of column `col`, as a run of a symmetric matrix's row or of X^T's: 8 (e / 4) + 4 h rows on
    auto run_at = [&](int col, int row) { return ((col * 256 + (col & 15) * 16) ^ (row / 32 * 128)) + 8 * h; };
    auto put4 = [&](char* at, int e, const float (&v)[4]) {
        half4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) { _Float16 f, l; split16(v[i], f, l); hi[i] = f; lo[i] = l; }
        *(half4_t*)(lds + ((int)(at - lds) ^ (e / 4 * 16))) = hi;
        *(half4_t*)(lds + ((int)(at - lds) ^ (e / 4 * 16 + 64))) = lo;
        return Split4{hi, lo};
    };
    auto get4 = [&](const char* at, int e) {
        return Split4{*(const half4_t*)(lds + ((int)(at - lds) ^ (e / 4 * 16))), *(const half4_t*)(lds + ((int)(at - lds) ^ (e / 4 * 16 + 64)))};
    };
    const int tiles = q.n / 32 * 2;                                            // of X: 64 rows
    for (int step = 0; step < c.steps; ++step) {
        const float ca = c.coef[3 * step], cb = c.coef[3 * step + 1], cc = c.coef[3 * step + 2];
        const bool last = step == c.steps - 1;
        const int run = run_at(col0 + (lane & 31), row0);
        if (square) {
            const float16_t_ v = small_product(X, row0, xp, X, col0, xp, q.n);
#pragma unroll
            for (int e = 0; e < 16; e += 4) put4(A + run, e, {gram * v[e], gram * v[e + 1], gram * v[e + 2], gram * v[e + 3]});
        }
        __syncthreads();
        if (square) {
            const float16_t_ v = small_product(A, row0, 256, A, col0, 256, SMALL_M);
            const float pa = cb * (c.sb / c.sa), pb = cc * (c.sb / c.sa / c.sa);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const Split4 own = get4(A + run, e);
                float w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = fmaf(pb, v[e + k], pa * ((float)own.hi[k] + (float)own.lo[k]));
                put4(B + run, e, w);
            }
        }
        __syncthreads();
        constexpr int MOST = SMALL_N / 32 * 2 / SMALL_WAVES;
        float16_t_ x[MOST];
        const float xa = last ? ldexpf(ca / c.sx, -lift) : ca, xb = last ? ldexpf(1.0f / (c.sb * c.sx), -lift) : 1.0f / c.sb;
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const int tile = wave + SMALL_WAVES * i, r0 = 32 * (tile & 1), n0 = 32 * (tile >> 1);
            if (tile >= tiles || r0 >= side) continue;
            x[i] = small_product(B, r0, 256, XT, n0, 256, SMALL_M);
            const char* at = XT + run_at(n0 + (lane & 31), r0);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const Split4 own = get4(at, e);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i][e + k] = fmaf(xb, x[i][e + k], xa * ((float)own.hi[k] + (float)own.lo[k]));
            }
        }
        __syncthreads();                                                       // X^T has been read
        float* out = (float*)X;                                                // X as well: the last step's result goes there
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const int tile = wave + SMALL_WAVES * i, r0 = 32 * (tile & 1), n0 = 32 * (tile >> 1), k = n0 + (lane & 31);
            if (tile >= tiles || r0 >= side) continue;
            if (last) {
#pragma unroll
                for (int e = 0; e < 16; ++e) out[(r0 + 4 * h + 8 * (e / 4) + e % 4) * q.n + k] = x[i][e];
                continue;
            }
            char* at = XT + run_at(k, r0);
            const int xv = (r0 + 4 * h) * xp + (k >> 6) * 256 + ((((k >> 5 & 1) * 8 + (k >> 3 & 3)) ^ 4 * h) * 16) + (k & 7) * 2;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const Split4 v = put4(at, e, {x[i][e], x[i][e + 1], x[i][e + 2], x[i][e + 3]});
#pragma unroll
                for (int j = 0; j < 4; ++j) {                                  // row r0 + 4 h + 2 e + j of X
                    char* to = X + (2 * e + j) * xp;
                    *(_Float16*)(to + (xv ^ ((2 * e & 8) + j) * 16)) = v.hi[j];
                    *(_Float16*)(to + (xv ^ (((2 * e & 8) + j) * 16 + 64))) = v.lo[j];
                }
            }
        }
        __syncthreads();
    }
    if (skip) return;
    for (int i = tid; i < total; i += threads) {
        const int r = i / q.cols, k = i - r * q.cols;
        const float v = ((const float*)X)[q.tall ? k * q.n + r : r * q.n + k];
        if (a.muon) q.param[i] = fmaf(-q.lr, v, q.param[i] * a.decay);
        else store_from_float(q.out, i, v, a.dtype);
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

static int64_t fill_group(const nerfx_matrix_t* mats, int count, int tile, OrthoTable& a) {
    int64_t at = ORTHO_TABLE_BYTES;
    a.call.count = 0;
    for (int k = 0; k < count; ++k) {
        if (mats[k].rows == 0 || mats[k].cols == 0) continue;
        OrthoMat& q = a.mat[a.call.count++];
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
// power-of-two scales keep X, A and B inside f16, from above.  From below: small singular values go with the product of the a's.
// Where X shrinks to less than a 64th of its largest before the last step, its halves run out of f16's small numbers (a = 0.03 five
// times: 3e-4 off, 0.01: 2.6e-2), and the coefficients are refused.
struct OrthoScales { float x, a, b; int growth; };
static int scales_for(const float* coef, int steps, OrthoScales& s) {
    double top = 1.001, x = top, ga = 0, gb = 0, all = 1, small = 1, least = 1;
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
        least = std::min(least, small);
        small *= std::fabs(a);
        top = next * 1.01;
        all *= gain * 1.01;
        NERFX_REQUIRE(top <= 64, "step %d lets singular values grow to %.3g: coefficients out of range", k, top);
    }
    NERFX_REQUIRE(least * 64 >= x, "coefficients out of range: they shrink small singular values to %.3g before the last step, with %.3g for the largest",
                  least, x);
    auto scale = [](double bound) { return (float)std::exp2(std::floor(std::log2(32768 / std::max(bound * 1.02, 1e-3)))); };
    s = {scale(x), scale(ga), scale(gb), (int)std::ceil(std::log2(all))};
    return 0;
}

// A launch's grid is the matrices' blocks one after the other.
template <class F>
static int64_t lay_out(OrthoTable& t, int grid, F blocks_of) {
    int64_t at = 0;
    for (int k = 0; k < ORTHO_GROUP; ++k) {
        t.first[grid][k] = k < t.call.count ? (int32_t)at : INT32_MAX;
        if (k < t.call.count) at += blocks_of(t.mat[k]);
    }
    return at;
}

// The tile a product takes, by how many of them there are:
//  128  where whole rounds of them fill at least four fifths of the 256 CUs: half of the operand traffic of 64
//       (2048 x 2048 by 2048: 57 us; 67 in tiles of 64);
//  64   with two stages, four workgroups to a CU, where they would not: a symmetric result's 136 tiles of 128 take 46 us, 528 of
//       64 take 39; three stages hold fewer workgroups and take 43;
//  64   with four stages where there are at most two to a CU, which is what LDS holds then: nothing but stages ahead hides
//       the way of a load there (408 tiles, K up to 2048: 32 us, 38 with two);
//  64   with eight stages where there is at most one to a CU: all of a K of 256 is on its way at once (a field's six matrices in
//       all: 112 us, 119 with two).
enum { ORTHO_TILE_128, ORTHO_TILE_64, ORTHO_TILE_64_MORE, ORTHO_TILE_64_DEEP };
struct OrthoShape { int kind; int64_t blocks; };
static OrthoShape choose(OrthoTable& t, int grid, int pad) {
    auto blocks = [&](int tile) {
        return lay_out(t, grid, [=](const OrthoMat& q) {
            const int64_t mt = q.m / tile;
            return grid == ORTHO_SYM_GRID ? mt * (mt + 1) / 2 : mt * (q.n / tile);
        });
    };
    if (pad == 128) {
        const int64_t big = blocks(128);
        if (big * 5 >= (big + 255) / 256 * 256 * 4) return {ORTHO_TILE_128, big};
    }
    const int64_t small = blocks(64);
    return {small <= 256 ? ORTHO_TILE_64_DEEP : small <= 512 ? ORTHO_TILE_64_MORE : ORTHO_TILE_64, small};
}

template <int T, int WAVES, int STAGES, int KIND>
static int product_as(int64_t blocks, char* work, float alpha, float beta, int from, hipStream_t stream) {
    constexpr size_t lds = SplitTile<T, WAVES, STAGES>::LDS_BYTES;
    NERFX_OPT_IN_LDS((ortho_product_kernel<T, WAVES, STAGES, KIND>), lds);
    hipLaunchKernelGGL((ortho_product_kernel<T, WAVES, STAGES, KIND>), dim3((unsigned)blocks), dim3(64 * WAVES), lds, stream,
                       (const OrthoTable*)work, work, alpha, beta, from);
    return 0;
}
template <int KIND>
static int product(const OrthoShape& s, char* work, float alpha, float beta, int from, hipStream_t stream) {
    if (s.kind == ORTHO_TILE_128) return product_as<128, 8, 4, KIND>(s.blocks, work, alpha, beta, from, stream);
    if (s.kind == ORTHO_TILE_64) return product_as<64, 4, 2, KIND>(s.blocks, work, alpha, beta, from, stream);
    if (s.kind == ORTHO_TILE_64_MORE) return product_as<64, 4, 4, KIND>(s.blocks, work, alpha, beta, from, stream);
    return product_as<64, 4, 8, KIND>(s.blocks, work, alpha, beta, from, stream);
}

static bool all_small(const OrthoTable& t) {
    for (int k = 0; k < t.call.count; ++k)
        if (t.mat[k].m > SMALL_M || t.mat[k].n > SMALL_N) return false;
    return true;
}

static int small_run(OrthoTable& t, const float* coef, int steps, const OrthoScales& s, hipStream_t stream) {
    t.call.x_scale = s.x;
    t.call.growth = s.growth;
    OrthoSteps c{};
    std::copy(coef, coef + 3 * steps, c.coef);
    c.steps = steps; c.sx = s.x; c.sa = s.a; c.sb = s.b;
    int n = 0;
    for (int k = 0; k < t.call.count; ++k) n = std::max(n, t.mat[k].n);
    const size_t lds = 2 * SMALL_M * 256 + (size_t)n * 512;
    NERFX_OPT_IN_LDS(ortho_small_kernel, 2 * SMALL_M * 256 + SMALL_N * 512);       // of any call
    hipLaunchKernelGGL(ortho_small_kernel, dim3((unsigned)t.call.count), dim3(64 * SMALL_WAVES), lds, stream, t, c);
    return launch_status("ortho_small_kernel");
}

static int ortho_run(OrthoTable& t, char* work, int pad, const float* coef, int steps, const OrthoScales& s, hipStream_t stream) {
    t.call.x_scale = s.x;
    t.call.growth = s.growth;
    const int64_t norm = lay_out(t, ORTHO_NORM_GRID, [](const OrthoMat& q) { return (int64_t)norm_parts(q); });
    const int64_t prep = lay_out(t, ORTHO_PREP_GRID, [](const OrthoMat& q) { return (int64_t)(q.m / PREP_TILE) * (q.n / PREP_TILE); });
    const OrthoShape sym = choose(t, ORTHO_SYM_GRID, pad), full = choose(t, ORTHO_FULL_GRID, pad);
    hipLaunchKernelGGL(ortho_norm_kernel, dim3((unsigned)norm), dim3(256), 0, stream, t, work);
    hipLaunchKernelGGL(ortho_prep_kernel, dim3((unsigned)prep), dim3(256), 0, stream, (const OrthoTable*)work, work);
    for (int k = 0; k < steps; ++k) {
        const float ca = coef[3 * k], cb = coef[3 * k + 1], cc = coef[3 * k + 2];
        if (int rc = product<ORTHO_GRAM>(sym, work, 0.f, s.a / (s.x * s.x), 0, stream)) return rc;
        if (int rc = product<ORTHO_POLY>(sym, work, cb * (s.b / s.a), cc * (s.b / s.a / s.a), 0, stream)) return rc;
        // the last step leaves the scales
        if (int rc = k == steps - 1 ? product<ORTHO_LAST>(full, work, ca / s.x, 1.0f / (s.b * s.x), k & 1, stream)
                                    : product<ORTHO_APPLY>(full, work, ca, 1.0f / s.b, k & 1, stream)) return rc;
    }
    return launch_status("orthogonalisation kernels");
}

static_assert(sizeof(OrthoTable) + sizeof(OrthoSteps) <= 4096, "kernel arguments");
// Groups of at most ORTHO_GROUP matrices, one after the other in the same workspace (same stream: in order).
static int64_t group_bytes(const nerfx_matrix_t* mats, int count) {
    int64_t most = 0;
    OrthoTable a;
    for (int k = 0; k < count; k += ORTHO_GROUP) {
        const int c = std::min(ORTHO_GROUP, count - k);
        const int64_t bytes = fill_group(mats + k, c, tile_side(mats + k, c), a);
        if (a.call.count && !all_small(a)) most = std::max(most, bytes);
    }
    return most;
}

static int ortho_groups(const nerfx_matrix_t* mats, int count, OrthoTable& a, const float* coef, int steps, void* workspace,
                        int64_t workspace_bytes, double lr, int adjust, hipStream_t stream) {
    NERFX_REQUIRE(steps >= 1 && steps <= ORTHO_MAX_STEPS && coef, "steps %d outside 1..%d, or no coefficients", steps, ORTHO_MAX_STEPS);
    NERFX_REQUIRE(a.call.eps > 0.f && std::isfinite(a.call.eps), "eps must be positive and finite");
    OrthoScales s;
    if (int rc = scales_for(coef, steps, s)) return rc;
    const int64_t need = group_bytes(mats, count);
    NERFX_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0), "workspace is NULL or not aligned to 16 bytes");
    NERFX_REQUIRE(workspace_bytes >= need, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    for (int k = 0; k < count; k += ORTHO_GROUP) {
        const int c = std::min(ORTHO_GROUP, count - k), tile = tile_side(mats + k, c);
        fill_group(mats + k, c, tile, a);
        if (a.call.count == 0) continue;
        for (int i = 0; i < a.call.count; ++i) {
            const double r = a.mat[i].rows, l = a.mat[i].cols;
            a.mat[i].lr = (float)(lr * (adjust == NERFX_LR_MATCH_RMS ? 0.2 * std::sqrt(std::max(r, l)) : std::sqrt(std::max(1.0, r / l))));
        }
        if (all_small(a)) {
            if (int rc = small_run(a, coef, steps, s, stream)) return rc;
            continue;
        }
        if (int rc = ortho_run(a, (char*)workspace, tile, coef, steps, s, stream)) return rc;
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
    OrthoTable a{};
    a.call.dtype = dtype; a.call.eps = eps;
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
    OrthoTable a{};
    OrthoCall& c = a.call;
    c.muon = 1; c.nesterov = nesterov != 0; c.momentum = (float)momentum; c.rest = (float)(1 - momentum);
    c.decay = (float)(1 - lr * weight_decay); c.eps = eps;
    c.grad_scale = grad_scale; c.found_inf = found_inf;
    return ortho_groups(mats, count, a, coefficients, steps, workspace, workspace_bytes, lr, adjust_lr, (hipStream_t)stream);
}
