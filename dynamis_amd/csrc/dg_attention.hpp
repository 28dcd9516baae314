// dg_attention.hpp -- what the attention kernels over neighbour lists share.
//
// Per edge e of target t with source j, head h, kv head c = h / per (base-2 logits):
//   s = scale log2e <q[t,h], k[j,c]> + log2e table[bucket(e),h]
//   p = 2^(s - m[t,h]) / l[t,h],  m = max_e s,  l = sum_e 2^(s - m),  out[t,h] = sum_e p v[j,c]
// and backward, with g = d out and delta = <g[t,h], out[t,h]>:
//   ds = p (<g[t,h], v[j,c]> - delta)
//   dq[t,h] = scale sum_e ds k[j,c]      dtable[b,h] = sum_{e in b} ds
//   dk[j,c] = scale sum_e sum_h ds q[t,h]    dv[j,c] = sum_e sum_h p g[t,h]
// An entry of minus infinity in the table takes the edge out for that head, whatever the
// tensors hold there; a row without an edge gives zeros and a log-sum of -inf.  (m, 1 / l) are
// kept for the backward pass as they are: in the log-sum m + log2 l the second term would be
// lost to rows whose logits all sit at a lowest value.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/dynamis_graph.h"

namespace dg {

dg_status fail(dg_status st, const std::string& msg);  // dg_graph.hip

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kXcds = 8;
constexpr int kMaxTable = 4096;  // buckets * heads

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;

// The lists of one direction (dg_neighbor_lists, see the C header).
struct Lists {
    int64_t n_rows, n_items;  // rows: of the pass (the targets' are the first ones)
    const int32_t* order;
    const int32_t* ptr;
    const int32_t* idx;
    const uint8_t* bucket;
    const int4* items;
    const int32_t* item_first;
    const int32_t* long_slot;
    int64_t n_long;
};

struct AttnArgs {
    Lists L;
    const void* q;
    const void* k;
    const void* v;
    const void* g;  // d out
    int64_t ldq, ldk, ldv, ldg;  // row strides, in elements
    const float* table;  // [n_buckets, heads] or null
    int n_buckets;
    int64_t n_targets, n_nodes;
    int heads, kv_heads, dim, per;
    float scale;
    // forward
    void* out;     // [n_targets, heads * dim]
    float* out32;  // the same unrounded, for the backward pass, or null
    float* lse;    // natural log, [n_targets, heads], or null
    float2* norm;  // (m, 1 / l), [n_targets, heads]; null: not kept
    // backward
    void* dq;
    void* dk;
    void* dv;
    float4* stats;    // [n_targets, heads]: m, 1 / l, delta, 0
    float* dtab;      // [workgroups, n_buckets * heads] partial sums, or null
    // long rows: [items, ...] partial results
    float* part_m;
    float* part_l;
    float* part_acc;
    float* part_acc2;
};

// A wave's piece of work: the entries [begin, end) of a row, and where the result goes.
struct Piece {
    int begin, end;
    int node;      // -1: nothing to do
    int64_t item;  // >= 0: the item's partial result, else the row's own
};

// Units of an XCD's waves (workgroups go to the XCDs in turn): its share of the parts of long
// rows, then of the rows, so that its waves read neighbouring rows through one L2.
struct Walk {
    int64_t at, end, step;               // this wave's units
    int64_t items, item0, row0;          // the XCD's parts, its first one, its first row
    __device__ __forceinline__ bool is_item(int64_t u) const { return u < items; }
    __device__ __forceinline__ int64_t item(int64_t u) const { return item0 + u; }
    __device__ __forceinline__ int64_t slot(int64_t u) const { return row0 + (u - items); }
};
__device__ __forceinline__ Walk walk_of(const Lists& L, int waves_per_group)
{
    const int xcds = min((int)gridDim.x, kXcds);
    const int x = blockIdx.x % xcds, j = blockIdx.x / xcds;
    const int64_t groups = ((int)gridDim.x - x + xcds - 1) / xcds;  // of this XCD
    Walk w;
    w.item0 = L.n_items * x / xcds;
    w.items = L.n_items * (x + 1) / xcds - w.item0;
    w.row0 = L.n_rows * x / xcds;
    w.end = w.items + L.n_rows * (x + 1) / xcds - w.row0;
    w.step = groups * waves_per_group;
    w.at = (int64_t)j * waves_per_group + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    return w;
}

__device__ __forceinline__ Piece piece_of(const Lists& L, const Walk& w, int64_t u)
{
    Piece p;
    if (w.is_item(u)) {
        p.item = w.item(u);
        const int4 i = L.items[p.item];
        p.begin = i.x;
        p.end = i.y;
        p.node = i.z;
    } else {
        const int64_t slot = w.slot(u);
        p.begin = L.ptr[slot];
        p.end = L.ptr[slot + 1];
        p.node = L.order[slot];
        p.item = -1;
        if (L.n_items && p.end - p.begin > DG_NEIGHBOR_SPLIT) p.node = -1;
    }
    if (p.node < 0) p.end = p.begin;
    return p;
}

// A table entry in base 2: the type's lowest and highest values stay finite.
__device__ __forceinline__ float entry_base2(float x)
{
    const float y = x * kLog2e;
    return isinf(y) && !isinf(x) ? copysignf(3.402823466e+38f, x) : y;
}

// A row's results that are not its weighted sum.
__device__ __forceinline__ void store_norm(const AttnArgs& a, int64_t row, float m, float l)
{
    if (a.lse) a.lse[row] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
    if (a.norm) a.norm[row] = make_float2(m, l == 0.0f ? 0.0f : 1.0f / l);
}

// Sum over groups of W neighbouring lanes (a power of two).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x)
{
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int W>
__device__ __forceinline__ float sum_lanes(float x)
{
    if constexpr (W >= 2) x = dpp_add<0xB1>(x);   // quad_perm 1,0,3,2
    if constexpr (W >= 4) x = dpp_add<0x4E>(x);   // quad_perm 2,3,0,1
    if constexpr (W >= 8) x = dpp_add<0x141>(x);  // row_half_mirror
    if constexpr (W >= 16) x = dpp_add<0x140>(x); // row_mirror
    if constexpr (W >= 32) x += __shfl_xor(x, 16, 64);
    if constexpr (W >= 64) x += __shfl_xor(x, 32, 64);
    return x;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float bf16_up(uint32_t bits16) { return __builtin_bit_cast(float, bits16 << 16); }

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&x)[4])
{
    const float4 f = *(const float4*)p;
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
}
template <>
__device__ __forceinline__ void load4<__bf16>(const __bf16* p, float (&x)[4])
{
    const uint2 u = *(const uint2*)p;
    x[0] = bf16_up(u.x & 0xffff);
    x[1] = __builtin_bit_cast(float, u.x & 0xffff0000u);
    x[2] = bf16_up(u.y & 0xffff);
    x[3] = __builtin_bit_cast(float, u.y & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, const float (&x)[4])
{
    *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
}
template <>
__device__ __forceinline__ void store4<__bf16>(__bf16* p, const float (&x)[4])
{
    bf16x4 y;
    for (int i = 0; i < 4; ++i) y[i] = (__bf16)x[i];
    *(bf16x4*)p = y;
}

}  // namespace dg
