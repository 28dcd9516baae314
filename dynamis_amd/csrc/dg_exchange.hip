// dg_exchange.hip -- rows into the order of the experts that they are routed to, and back.
//
//   dispatch   out[places[i, j]] = x[i], and zeros behind the last choice that was taken
//   combine    out[i] = residual[i] + sum_j weights[i, j] y[places[i, j]]     (without weights: ones)
//   backward   dy[places[i, j]] = weights[i, j] g[i],   dweights[i, j] = <g[i], y[places[i, j]]>
//
// The gradient of a dispatch is a combine without weights.  A place p < 0 is a choice of none: -1 - p
// is its place behind the last, which gets zeros and is not read.  places is a permutation, so every
// row of the experts' order is written by one owner (a place past the last row is left out); a row's sum is
// taken over j in order, in 32 bits.
//
// Bound by memory: rows are read and written whole, 16 bytes a lane, a power of two of lanes to a row
// as far as its width goes (an x row is read once for all of its places; a sum's k rows are in flight
// together).  Rows whose chunks are not whole and aligned go element by element.
//
// 300,007 sums of 6 rows of 128 and a residual in bfloat16: 129 us, 4.9 TB/s, what a copy reaches; 100,000 rows of 256 to
// two places each: 27 us, 5.6 TB/s (the caches hold a part); 32,000 rows of 256 floats, two places, backward: 27
// us, 5.7 TB/s.  Element by element a request carries less: 32,000 rows of 333, two places, dispatched and combined: in
// float 26 and 35 us (25 at a copy's rate), in bfloat16 23 and 40 (12); of 100 and 130 bfloat16 10 to 20 us (4 to 5).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <string>

#include "../../include/dynamis_graph.h"
#include "dg_grid.hpp"
#include "dg_lanes.hpp"

namespace dg {
dg_status fail(dg_status st, const std::string& msg);  // dg_graph.hip
}

namespace {

using namespace dg;

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f32x4 = __attribute__((ext_vector_type(4))) float;

constexpr int kThreads = 256;
constexpr int kInFlight = 4;  // rows of a sum

struct Args {
    const void *x, *y, *residual, *grad;  // x, residual and grad: rows `ld` apart
    const int32_t* places;
    const float* weights;
    void* out;
    float* dweights;
    int64_t rows, ld;
    int k, width, lanes;
};

// C elements of a row at a time: 16 bytes, or one.
template <typename T, bool WHOLE>
struct Chunk {
    static constexpr int C = WHOLE ? 16 / (int)sizeof(T) : 1;
    static __device__ __forceinline__ void load(const T* p, float (&v)[C])
    {
        if constexpr (!WHOLE) {
            v[0] = (float)*p;
        } else if constexpr (sizeof(T) == 4) {
            const f32x4 f = *(const f32x4*)p;
            for (int i = 0; i < 4; ++i) v[i] = f[i];
        } else {
            const u32x4 r = *(const u32x4*)p;
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = r[i];
                v[2 * i] = __builtin_bit_cast(float, w << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ void store(T* p, const float (&v)[C])
    {
        if constexpr (!WHOLE) {
            *p = (T)v[0];
        } else if constexpr (sizeof(T) == 4) {
            f32x4 f;
            for (int i = 0; i < 4; ++i) f[i] = v[i];
            *(f32x4*)p = f;
        } else {
            __attribute__((ext_vector_type(8))) __bf16 f;
            for (int i = 0; i < 8; ++i) f[i] = (__bf16)v[i];
            *(decltype(f)*)p = f;
        }
    }
};

// This thread's row and first chunk (in elements).
template <int C>
__device__ __forceinline__ int64_t my_row(const Args& a, int& c0)
{
    c0 = (int)(threadIdx.x & (a.lanes - 1)) * C;
    return workgroup() * (kThreads / a.lanes) + threadIdx.x / a.lanes;
}

// Where a place points to, and whether that row is of a choice; false: there is no such row.
__device__ __forceinline__ bool place_of(const Args& a, int32_t p, int64_t& at, bool& taken)
{
    taken = p >= 0;
    at = taken ? p : -1 - p;
    return at < a.rows * a.k;
}

// (Bits as they are: W is a chunk of 16 bytes, or an element.)
template <typename W>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(Args a)
{
    int c0;
    const int64_t row = my_row<1>(a, c0);
    if (row >= a.rows) return;
    const int32_t* places = a.places + row * a.k;
    for (int c = c0; c < a.width; c += a.lanes) {
        const W v = ((const W*)a.x)[row * a.ld + c], zero = {};
        for (int j = 0; j < a.k; ++j) {
            int64_t at;
            bool taken;
            if (place_of(a, places[j], at, taken)) ((W*)a.out)[at * a.width + c] = taken ? v : zero;
        }
    }
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void combine_kernel(Args a)
{
    using Ch = Chunk<T, WHOLE>;
    int c0;
    const int64_t row = my_row<Ch::C>(a, c0);
    if (row >= a.rows) return;
    const int32_t* places = a.places + row * a.k;
    for (int c = c0; c < a.width; c += a.lanes * Ch::C) {
        float sum[Ch::C] = {};
        for (int j0 = 0; j0 < a.k; j0 += kInFlight) {
            float y[kInFlight][Ch::C], w[kInFlight];
            bool there[kInFlight];
#pragma unroll
            for (int j = 0; j < kInFlight; ++j) {
                int64_t at;
                there[j] = j0 + j < a.k;
                if (there[j]) {
                    bool taken;
                    there[j] = place_of(a, places[j0 + j], at, taken) && taken;
                }
                w[j] = 1.0f;
                if (there[j]) {
                    Ch::load((const T*)a.y + at * a.width + c, y[j]);
                    if (a.weights) w[j] = a.weights[row * a.k + j0 + j];
                }
            }
#pragma unroll
            for (int j = 0; j < kInFlight; ++j)
                if (there[j])
                    for (int i = 0; i < Ch::C; ++i) sum[i] = fmaf(w[j], y[j][i], sum[i]);
        }
        if (a.residual) {
            float r[Ch::C];
            Ch::load((const T*)a.residual + row * a.ld + c, r);
            for (int i = 0; i < Ch::C; ++i) sum[i] += r[i];
        }
        Ch::store((T*)a.out + row * a.width + c, sum);
    }
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(Args a)
{
    using Ch = Chunk<T, WHOLE>;
    int c0;
    const int64_t row = my_row<Ch::C>(a, c0);
    const bool live = row < a.rows;  // (the wave stays whole for its sums)
    for (int j = 0; j < a.k; ++j) {
        int64_t at = 0;
        bool taken = false;
        const bool there = live && place_of(a, a.places[row * a.k + j], at, taken);
        taken = taken && there;
        const float w = taken ? a.weights[row * a.k + j] : 0.0f;
        at *= a.width;
        float dot = 0.0f;
        if (there)
            for (int c = c0; c < a.width; c += a.lanes * Ch::C) {
                float d[Ch::C] = {};
                if (taken) {
                    float g[Ch::C], y[Ch::C];
                    Ch::load((const T*)a.grad + row * a.ld + c, g);
                    if (a.dweights) {
                        Ch::load((const T*)a.y + at + c, y);
                        for (int i = 0; i < Ch::C; ++i) dot = fmaf(g[i], y[i], dot);
                    }
                    for (int i = 0; i < Ch::C; ++i) d[i] = w * g[i];
                }
                if (a.out) Ch::store((T*)a.out + at + c, d);
            }
        if (a.dweights) {
            dot = sum_lanes(dot, a.lanes);
            if (live && c0 == 0) a.dweights[row * a.k + j] = dot;
        }
    }
}

// ---------------------------------------------------------------- host
dg_status check(const dg_exchange_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->dtype != DG_F32 && d->dtype != DG_BF16) return fail(DG_ERR_INVALID, "rows must be float32 or bfloat16");
    if (d->k < 1 || d->k > 64) return fail(DG_ERR_INVALID, "k must be in [1, 64]");
    if (d->n_rows < 0 || d->n_rows > 0x7fffffffll / d->k) return fail(DG_ERR_INVALID, "rows times k must be below 2^31");
    if (d->width < 1 || d->width > (1 << 20)) return fail(DG_ERR_INVALID, "the width must be in [1, 2^20]");
    if (d->ld < 0 || d->ld > (1ll << 31)) return fail(DG_ERR_INVALID, "rows must lie 0 to 2^31 elements apart");
    return DG_OK;
}

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

Args make_args(const dg_exchange_desc* d, const int32_t* places)
{
    Args a = {};
    a.rows = d->n_rows;
    a.ld = d->ld;
    a.k = d->k;
    a.width = d->width;
    a.places = places;
    return a;
}

// Whole chunks of 16 bytes: of every row that is read or written.
bool whole(const dg_exchange_desc* d, std::initializer_list<const void*> p)
{
    const int c = d->dtype == DG_F32 ? 4 : 8;
    bool ok = d->width % c == 0 && d->ld % c == 0;
    for (const void* x : p) ok = ok && ((uintptr_t)x & 15) == 0;
    return ok;
}

// Lanes of a row of chunks of c elements, and the workgroups.
dim3 grid_of(Args& a, int c)
{
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes * c < a.width) a.lanes *= 2;
    const int64_t rows = kThreads / a.lanes;
    return workgroups((a.rows + rows - 1) / rows);
}
template <typename F>
void run(const dg_exchange_desc* d, Args& a, bool whole, F&& launch)
{
    launch(grid_of(a, !whole ? 1 : d->dtype == DG_F32 ? 4 : 8));
}

}  // namespace

#define DG_LAUNCH(kernel)                                                                                              \
    run(d, a, all, [&](dim3 grid) {                                                                                    \
        if (d->dtype == DG_BF16) {                                                                                     \
            if (all) hipLaunchKernelGGL((kernel<__bf16, true>), grid, dim3(kThreads), 0, s, a);                        \
            else hipLaunchKernelGGL((kernel<__bf16, false>), grid, dim3(kThreads), 0, s, a);                           \
        } else {                                                                                                       \
            if (all) hipLaunchKernelGGL((kernel<float, true>), grid, dim3(kThreads), 0, s, a);                         \
            else hipLaunchKernelGGL((kernel<float, false>), grid, dim3(kThreads), 0, s, a);                            \
        }                                                                                                              \
    })

extern "C" {

dg_status dg_exchange_dispatch(const dg_exchange_desc* d, const void* x, const int32_t* places, void* out, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_rows == 0) return DG_OK;
    if (!x || !places || !out) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    Args a = make_args(d, places);
    a.x = x;
    a.out = out;
    const int c = d->dtype == DG_F32 ? 4 : 8;
    const bool all = whole(d, {x, out});
    if (all) {
        a.width /= c;
        a.ld /= c;
    }
    const dim3 grid = grid_of(a, 1), block(kThreads);
    if (all) hipLaunchKernelGGL(dispatch_kernel<u32x4>, grid, block, 0, s, a);
    else if (c == 4) hipLaunchKernelGGL(dispatch_kernel<uint32_t>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(dispatch_kernel<uint16_t>, grid, block, 0, s, a);
    return launched("dg_exchange_dispatch");
}

dg_status dg_exchange_combine(const dg_exchange_desc* d, const void* y, const int32_t* places, const float* weights,
                              const void* residual, void* out, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_rows == 0) return DG_OK;
    if (!y || !places || !out) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    Args a = make_args(d, places);
    a.y = y;
    a.weights = weights;
    a.residual = residual;
    a.out = out;
    const bool all = whole(d, {y, residual, out});
    DG_LAUNCH(combine_kernel);
    return launched("dg_exchange_combine");
}

dg_status dg_exchange_combine_backward(const dg_exchange_desc* d, const void* y, const int32_t* places, const float* weights,
                                       const void* grad, void* dy, float* dweights, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_rows == 0 || (!dy && !dweights)) return DG_OK;
    if (!y || !places || !weights || !grad) return fail(DG_ERR_INVALID, "inputs are NULL");
    Args a = make_args(d, places);
    a.y = y;
    a.weights = weights;
    a.grad = grad;
    a.out = dy;
    a.dweights = dweights;
    const bool all = whole(d, {y, grad, dy});
    DG_LAUNCH(combine_backward_kernel);
    return launched("dg_exchange_combine_backward");
}

}  // extern "C"
