// dcq_lds_load.h — loads from global memory straight into LDS: lane l's 4 (dma4) or 16 (dma16) bytes go to lds_base + 4 l
// (16 l), no registers held while they are on their way. lds_base is uniform over the wave and goes to M0, which has no
// other use in the kernels that call these; addresses are aligned to the load's size.
//
// The ISA asks for one wait state between a scalar write of M0 and a load that takes its LDS base from there, and the
// compiler inserts it only for loads that it knows: hence the s_nop, which tests/test_isa_hazards.py looks for.
//
// Inline asm, because the builtin form makes the compiler wait for every earlier direct load (it cannot tell the
// destinations apart) before the next one, or before ordinary loads and LDS reads. The compiler does not count these loads:
// where ordinary loads are issued beside them these come first (loads retire in order, so the compiler's own waits stay
// conservative), and an explicit wait stands before what they bring is read, and before the barrier that publishes it.
// PRIVATE: to room that only the issuing wave reads, after its own wait, so that the load may stay on its way across a
// barrier; the asm's comment says so to the assembly scan.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#pragma clang diagnostic ignored "-Winline-asm"  // M0 in the clobber list

namespace dcq {

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    typedef __attribute__((address_space(3))) const void* LdsPtr;
    return (uint32_t)(uintptr_t)(LdsPtr)p;
}

// an address per lane
template <bool PRIVATE = false>
__device__ __forceinline__ void dma4(const void* g, const void* lds_base) {
    const uint32_t m0 = lds_address(lds_base);
    if constexpr (PRIVATE)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off ; wave-private" ::"v"(g), "s"(m0) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "s"(m0) : "memory", "m0");
}
template <bool PRIVATE = false>
__device__ __forceinline__ void dma16(const void* g, const void* lds_base) {
    const uint32_t m0 = lds_address(lds_base);
    if constexpr (PRIVATE)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off ; wave-private" ::"v"(g), "s"(m0) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(m0) : "memory", "m0");
}

// a uniform base (in scalar registers) and 32 bits of unsigned byte offset per lane: a step of the base costs scalar adds only
template <bool PRIVATE = false>
__device__ __forceinline__ void dma4(const void* base, uint32_t off, const void* lds_base) {
    const uint32_t m0 = lds_address(lds_base);
    if constexpr (PRIVATE)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1 ; wave-private" ::"v"(off), "s"(base), "s"(m0)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(m0) : "memory", "m0");
}
template <bool PRIVATE = false>
__device__ __forceinline__ void dma16(const void* base, uint32_t off, const void* lds_base) {
    const uint32_t m0 = lds_address(lds_base);
    if constexpr (PRIVATE)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 ; wave-private" ::"v"(off), "s"(base), "s"(m0)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m0) : "memory", "m0");
}

}  // namespace dcq
