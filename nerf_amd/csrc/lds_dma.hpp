// Loads from memory straight into LDS, and the wait that goes with them.
#pragma once
#include "common.hpp"

namespace nerfx {

#ifdef __HIPCC__
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
#endif

}  // namespace nerfx
