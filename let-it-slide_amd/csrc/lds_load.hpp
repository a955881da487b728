// Loads from global memory straight into LDS, and the waits they need.
#pragma once

#include "rptc_common.hpp"

namespace rptc {

#ifdef __HIPCC__
typedef int int4_t __attribute__((ext_vector_type(4)));

// A value every lane of the wave holds, as one the compiler knows to be such (scalar registers, scalar branches).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// 16 bytes a lane from `offset` of the buffer to LDS at `to` + 16 lane (no register receives anything: the request may
// stay in flight behind the statement).  As assembly because the compiler, which cannot tell the two buffers in LDS
// apart, waits for such a request in front of the next transposing LDS read, which reads the other buffer.  (m0 is
// reserved for such single uses: the compiler sets it in front of each of its own.)
__device__ __forceinline__ void load_to_lds(uint32_t offset, int4_t resource, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(resource), "s"(to) : "memory");
}
__device__ __forceinline__ void wait_for_lds_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// all but the N requests made last
template <int N>
__device__ __forceinline__ void wait_for_lds_loads_but()
{
    static_assert(N < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// what was read from LDS is in registers: its place may be written over
__device__ __forceinline__ void wait_for_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}
// The descriptor of `bytes` bytes from base on, in scalar registers; what lies at or past their end reads as zero.
__device__ __forceinline__ int4_t buffer_resource(const void *base, int bytes)
{
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    const int4_t r = {uniform((int)p), uniform((int)(p >> 32) & 0xFFFF), uniform(bytes), 0x00027000};
    return r;
}
#endif

}  // namespace rptc
