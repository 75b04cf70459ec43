// What the attention kernels share: lanes' halves, copies from global memory straight to LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace kea {

typedef __attribute__((address_space(3))) void *lptr_t;

// A lane's value and that of the lane 32 away, the lower half's first. (The components are read before they are cast:
// hipcc's __builtin_bit_cast of a component access gives component 0.)
__device__ __forceinline__ float2 halves(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t lower = s[0], upper = s[1];
    return make_float2(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper));
}
__device__ __forceinline__ float other_half_max(float v) {
    const float2 s = halves(v);
    return fmaxf(s.x, s.y);
}
__device__ __forceinline__ float both_halves(float v) {
    const float2 s = halves(v);
    return s.x + s.y;
}

// 16 bytes a lane from global memory straight to LDS, at the wave's base address plus 16 a lane; done when vmcnt says so. In
// place of the builtin, after which the compiler waits for all of a wave's copies before its next transposing read, those for
// the tile ahead among them. (Nothing else in the kernels that use it uses m0.) The second form reads at a uniform address plus an
// offset.
__device__ __forceinline__ void copy16(const void *src, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(src) : "memory");
}
__device__ __forceinline__ void copy16(const void *src, uint32_t offset, uint32_t base) {
    const uint64_t at = (uint64_t)(uintptr_t)src;
    const uint64_t uniform = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(offset), "s"(uniform) : "memory");
}
// Four bytes a lane, at the base address plus four a lane.
__device__ __forceinline__ void copy4(const void *src, uint32_t base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(base)), "v"(src) : "memory");
}

}  // namespace kea
