// dg_grid.hpp -- launches of any number of workgroups.
//
// A launch holds less than 2^32 threads along an axis, and one of more runs without an error on what
// is left of its number modulo 2^32. So workgroups beyond a row of 2^20 lie along a second axis; the
// last row's surplus has numbers past the end, which the kernel returns for.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace dg {

inline dim3 workgroups(int64_t n)
{
    const int64_t across = std::max<int64_t>(1, std::min<int64_t>(n, 1 << 20));
    return dim3((unsigned)across, (unsigned)((n + across - 1) / across));
}
__device__ __forceinline__ int64_t workgroup() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

}  // namespace dg
