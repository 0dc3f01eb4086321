// What kernels that bring tiles into LDS share: loads from memory straight into it, the wait for them, and the order of tiles.
#pragma once
#include "common.hpp"

namespace nerfx {

#ifdef __HIPCC__
// Workgroups go to the eight XCDs in turn, each XCD with an L2 of its own.  -> this one's place in an order where an XCD's are
// neighbours: what neighbouring tiles share is then read into one L2, not into all of them (the orthogonalisation of a field's six
// matrices takes 129 us so, 138 in turn).
__device__ __forceinline__ int xcd_place() {
    const int x = blockIdx.x & 7, each = gridDim.x >> 3, more = gridDim.x & 7;
    return x * each + min(x, more) + (blockIdx.x >> 3);
}
// Place t of a rows x cols field of tiles -> (row, column): bands of as many rows as make an XCD's part about square, which
// shares the most (microscaled product, 512 x 4096 by 4096: 16 us, 19 row by row; 100,000 x 300 by 301: 63 and 70).
__device__ __forceinline__ void band_at(int t, int rows, int cols, int& row, int& col) {
    const int band = min(rows, max(1, (int)sqrtf((float)gridDim.x * 0.125f)));
    const int first = t / (band * cols) * band, in = t - first * cols, high = min(band, rows - first);
    col = in / high;
    row = first + in - col * high;
}
__device__ __forceinline__ uint32_t lds_address(const char* lds) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds;
}
// 64 lanes x 16 bytes from base + offset (per lane) to LDS at `lds` + 16 * lane.  The compiler does not know of the
// load: whoever reads the LDS waits with landed().
__device__ __forceinline__ void dma16(uint32_t lds, const char* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// The same from an address of each lane's own.
__device__ __forceinline__ void dma16(uint32_t lds, const char* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}
// All but the newest N of this wave's loads are done, and so are its LDS reads: then, behind the barrier, so are every wave's.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// Between lanes of one wave that hand values on by way of LDS, behind the writes and behind the reads.  The hardware keeps a wave's LDS
// accesses in order by itself; the compiler, to which each lane is a thread, need not.  No instruction comes of it.
__device__ __forceinline__ void wave_lds_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
#endif

}  // namespace nerfx
