// Global -> LDS loads without registers, and the barrier that goes with them.
#pragma once
#include <hip/hip_runtime.h>

namespace mcmc {
namespace {

typedef __attribute__((address_space(3))) char lds_char;
// One LDS-DMA load (global_load_lds_dwordx4: lane i's 16 bytes land at the wave-uniform LDS byte address lds_dst + 16 i), as an
// asm statement so that hipcc does not count it: with the builtin every LDS read that follows waits vmcnt(0) for it (the
// compiler cannot tell that the read does not alias the destination), which would expose the load in the very next phase.
// Completion is counted by hand: s_waitcnt vmcnt(0) in the issuing wave, then a barrier, then the reads.  M0 is written in the
// statement that uses it and restored.
__device__ __forceinline__ void glds16(const void* gsrc, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(gsrc), "s"(lds_dst)
                 : "memory");
}
// the same with four bytes a lane
__device__ __forceinline__ void glds4(const void* gsrc, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(gsrc), "s"(lds_dst)
                 : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) { return (unsigned)(size_t)(const lds_char*)reinterpret_cast<const char*>(p); }

// Workgroup barrier that leaves VMEM in flight: __syncthreads() drains vmcnt while an LDS-DMA load is outstanding;
// LDS traffic is retired by the lgkmcnt wait.
__device__ __forceinline__ void barrier_lds_only() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

}  // namespace
}  // namespace mcmc
