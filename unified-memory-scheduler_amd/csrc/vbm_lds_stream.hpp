// Streams of weights through rings in LDS: loads straight from memory to LDS, and the waits that count them.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

namespace vbm {
namespace {

// Loads from memory to LDS (lane l's bytes land at m0 + l * size), in inline assembly so that the compiler does not wait for
// all of them before every LDS read; the kernel waits itself before each barrier. The compiler knows of no other use of
// M0 here, and the wait state between a scalar write of M0 and the load that reads it is written out. A scalar base needs five wait states
// behind a vector instruction that wrote it, which is the caller's business: bases are sums by scalar instructions, or wait themselves. A test looks back from each load in
// the compiled code along every way to it. (Waits here, for all: FP8 and integers 4096 x 4096 x 4096 each 1 % slower.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds_16(const void * src, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds_16(const void * base, uint32_t offset, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(base), "v"(offset), "s"(m0) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds_4(const void * src, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(m0) : "memory", "m0");
}
// By all lanes (`all` -1) or by lane 0 alone (0), which the waits count alike; all lanes are active where it is called.
__device__ __forceinline__ void load_to_lds_4(const void * src, uint32_t m0, int all) {
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dword %0, off\n\ts_mov_b64 exec, -1" ::"v"(src), "s"(m0), "s"(all | 1), "s"(all) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until all but the wave's newest N loads have landed and its LDS reads are done, then for the workgroup's other waves.
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// All but the wave's newest N loads have landed, and its LDS reads are done.
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// The last steps of a ring, at most LEFT + 1 of them, with P loads each on their way.
template <int LEFT, int P, class F>
__device__ __forceinline__ void drain(int i, int n, const F & compute) {
    if (n - i > LEFT) {
        landed<LEFT * P>();
        compute(i);
        ++i;
    }
    if constexpr (LEFT > 0) drain<LEFT - 1, P>(i, n, compute);
}

}  // namespace
}  // namespace vbm
