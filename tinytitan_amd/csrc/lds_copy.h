// Copies from memory straight into LDS, whose completion the kernels track by hand.
#pragma once
#include <hip/hip_runtime.h>

namespace tt {

// 16 bytes per lane, global -> LDS without passing through registers: lane l's 16 bytes land at
// lds_addr + 16 l.  Issued as inline assembly on purpose: the compiler, when it sees an LDS DMA,
// guards every later LDS read with a full vmcnt(0) wait (it cannot tell the stages apart),
// which would turn a multi-stage prefetch into none.  Completion is tracked by hand instead:
// TT_WAIT_VMCNT before the barrier that publishes a stage.
__device__ __forceinline__ void copy16_global_to_lds(const void *base, unsigned lane_offset, unsigned lds_addr) {
    // base and lds_addr are wave-uniform by construction; say so, in case the compiler lost track
    const unsigned long long b = (unsigned long long)base;
    const unsigned b_hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(b >> 32));
    const unsigned b_lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b);  // (the builtin returns a signed int)
    base = (const void *)(((unsigned long long)b_hi << 32) | (unsigned long long)b_lo);
    lds_addr = (unsigned)__builtin_amdgcn_readfirstlane((int)lds_addr);
    // m0 carries the LDS address of the copy.  The compiler owns m0 (it is a reserved register: naming it as a clobber is not honoured), but has
    // no use for it in the kernels that copy by this (tests/test_wait_states.py looks), so it is not put back.  Between a scalar write of m0 and a
    // copy into LDS belongs one wait state, which is nobody's to add but the block's own.
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" : : "s"(base), "v"(lane_offset), "s"(lds_addr) : "memory");
}

// vmcnt(n) only: leaves the LDS/scalar and export counters alone.
#define TT_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (((n) >> 4) << 14) | (0x7 << 4) | (0xF << 8))

}  // namespace tt
