// Asynchronous copies from global memory into LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace si {

// One asynchronous 16-byte copy per lane from global memory into LDS at
// lds_base + 16 x lane.  The wave-uniform LDS base goes in M0 (the compiler
// writes it there as the operand's register); the s_nop is the wait state an
// LDS-bound load needs after an M0 write.
__device__ __forceinline__ void copy16_to_lds(const void* src, uint32_t lds_base)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds_base) : "memory");
}

// The same from a wave-uniform base and a byte offset of each lane.
__device__ __forceinline__ void copy16_to_lds(uint32_t offset, const void* base, uint32_t lds_base)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(lds_base) : "memory");
}

// Waits until at most N of this wave's memory loads (copies included) are in
// flight.
template <int N>
__device__ __forceinline__ void wait_copies()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace si
