// fq_dma.h -- copies from global memory straight into LDS, counted by hand.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fq {

// Global memory straight into LDS: 16 bytes per lane, from base + off (base
// wave-uniform, off a 32-bit per-lane byte offset, so that a loop that moves base
// keeps the per-lane part in one register and its address arithmetic on the
// scalar unit) to lds + 16 lane (lds wave-uniform, in M0).  Issued as inline
// assembly on purpose: the compiler cannot tell which LDS bytes the builtin's copy
// writes, so it waits for every outstanding load (vmcnt(0)) before the next
// LDS read, which would serialise a kernel's loads with its compute.  The
// kernel counts the copies itself (wait_vm) before it reads what they wrote.  The
// compiler does not see these copies either when it counts its own loads, so its
// waits for register loads issued before a copy only ever wait longer than
// needed.
//
// Base and M0 pass through scalar moves within the block: a vector instruction may
// have written either just before (as a spilled scalar register's return does), and
// a load must not read such a register within five states, which the compiler
// sees to for its own loads only.  A scalar move waits for it, what the move
// wrote may be read at once, and M0 after one state, the second move.
__device__ __forceinline__ void dma16s(uint32_t off, const uint8_t* base, uint32_t lds) {
    uint64_t at;
    uint32_t m0;
    asm volatile("s_mov_b32 m0, %4\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
                 : "=&s"(at), "=&{m0}"(m0)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}

// The same of 4 bytes per lane, from an address of each lane's own, to lds + 4 lane.
__device__ __forceinline__ void dma4(const void* at, uint32_t lds) {
    uint32_t m0;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 : "=&{m0}"(m0)
                 : "v"(at), "s"(lds)
                 : "memory");
}

// Wait until at most N vector-memory loads of this wave are outstanding.
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// The LDS address of p as the 32-bit value M0 takes.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p;
}

}  // namespace fq
