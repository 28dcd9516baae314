// dg_lanes.hpp -- sums and maxima over neighbouring lanes, and order between a wave's LDS accesses.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dg {

__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ uint32_t as_bits(float x) { return __builtin_bit_cast(uint32_t, x); }

// What one lane of a wave wrote to LDS may be read by the others.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Calls step(other) for each halving of `n` neighbouring lanes (a power of two, the same for the wave;
// all lanes active), where other(x) is x of the lane across: the same combination in each lane, in
// a fixed order.
template <typename F>
__device__ __forceinline__ void over_lanes(int n, F&& step)
{
    if (n > 1) step([](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true); });   // lanes 1 0 3 2
    if (n > 2) step([](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true); });   // 2 3 0 1
    if (n > 4) step([](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true); });  // mirrored in 8
    if (n > 8) step([](uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true); });  // in 16
    // (the swap of a value with itself holds, in each lane, its own and the other's: what is not its own)
    if (n > 16) step([](uint32_t x) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); return r[0] ^ r[1] ^ x; });
    if (n > 32) step([](uint32_t x) { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); return r[0] ^ r[1] ^ x; });
}
__device__ __forceinline__ float sum_lanes(float x, int n)
{
    over_lanes(n, [&](auto&& other) { x += as_float(other(as_bits(x))); });
    return x;
}
__device__ __forceinline__ double sum_lanes(double x, int n)
{
    over_lanes(n, [&](auto&& other) {
        const uint64_t b = __builtin_bit_cast(uint64_t, x);
        x += __builtin_bit_cast(double, (uint64_t)other((uint32_t)(b >> 32)) << 32 | other((uint32_t)b));
    });
    return x;
}

inline int power_of_two(int x)  // the first from x on
{
    int p = 1;
    while (p < x) p *= 2;
    return p;
}

}  // namespace dg
