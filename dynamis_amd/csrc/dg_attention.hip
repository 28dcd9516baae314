// dg_attention.hip -- attention of every target over its neighbour list, forward and backward,
// for any head width: the kernels on the vector units, the joins of long rows, the entry
// points.
//
// A lane holds four channels of one head; the lanes of a head reduce its dot products among
// themselves, the heads of an edge sit side by side in the wave, and where they fill less than
// the wave it takes several edges at once, each with a running maximum and sum of its own that
// are merged at the row's end.  One pass over a row's edges: logits, running softmax and the
// weighted sum of v in registers, nothing per edge written.  The backward pass recomputes the
// probabilities from the saved maxima and sums: one pass by target (dq, and the table's gradient from
// private rows in LDS, in a fixed order), one by source (dk, dv).  No atomics: every sum has
// one owner and one order, so results repeat bit for bit.
//
// All arithmetic is in 32 bits, whatever the tensors' type; outputs are rounded once.
//
// Bound by the vector units' instructions (a logit of 32 channels is four multiply-adds and three
// exchanges a lane, of which half the lanes' work is the reduction's) next to the gathered rows:
// 360,000 edges of 4 heads of 32 floats take 29 us, 13 TB/s of rows out of the caches, at 65 % of the
// vector units; 26.5M edges of 8 heads of 16 1630 us, 17 TB/s.  Few rows are
// bound by the wait for a row's loads in turn: 864 rows of 86 edges take 18 us forward, 21 us by
// target and 20 us by source.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "../../include/dynamis_graph.h"
#include "dg_attention.hpp"
#include "dg_attention_mfma.hpp"
#include "dg_grid.hpp"

namespace {

using namespace dg;

inline size_t al(size_t x) { return (x + 255) & ~(size_t)255; }
inline unsigned nblk(int64_t n, int b = 256) { return (unsigned)((n + b - 1) / b); }

constexpr int kWaves = 4;

// How lanes map to heads (of q in the target passes, of k in the source pass).
struct Lanes {
    int heads, per_wave;  // heads of a wave; lanes of an edge = slots * LPH
    int slots;            // per_wave rounded up to a power of two
    int groups;           // head groups of a row
};

template <int LPH>
__host__ __device__ inline Lanes lanes_of(int heads)
{
    Lanes m;
    m.heads = heads;
    const int most = 64 / LPH;
    m.per_wave = heads < most ? heads : most;
    m.slots = 1;
    while (m.slots < m.per_wave) m.slots *= 2;
    m.groups = (heads + m.per_wave - 1) / m.per_wave;
    return m;
}

// The table in base 2 in LDS; returns (to all threads) whether it holds an entry of -inf.
__device__ __forceinline__ bool stage_table(const AttnArgs& a, float* s_tab)
{
    __shared__ int s_any;
    if (threadIdx.x == 0) s_any = 0;
    __syncthreads();
    if (a.table) {
        const int n = a.n_buckets * a.heads;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const float x = a.table[i];
            s_tab[i] = entry_base2(x);
            if (x == -INFINITY) s_any = 1;  // (every writer writes the same value)
        }
    }
    __syncthreads();
    return s_any != 0;
}

constexpr int kUnroll = 4;  // (600,000 edges of 8 heads of 32 floats: 140 us, eight edges a step 148 us)

// The entries of a lane's next edges, under way while the ones before are worked on: of few rows a
// wave else waits twice for each of its steps, for the entries and for the rows that they name.
// (1000 rows of 60 edges, 8 heads of 32 floats: 34 us, without 47 us; 100,000 rows: 1697 and 1644 us.)
template <int N>
struct Entries {
    int node[N], bucket[N];
    __device__ __forceinline__ void load(const AttnArgs& a, const Piece& p, int e0, int span)
    {
#pragma unroll
        for (int r = 0; r < N; ++r) {
            const int at = max(min(e0 + r * span, p.end - 1), 0);  // (an empty row reads some entry)
            node[r] = a.L.idx[at];
            bucket[r] = a.table ? (int)a.L.bucket[at] : 0;
        }
    }
};

template <typename T, int LPH>
__global__ __launch_bounds__(64 * kWaves) void forward_kernel(AttnArgs a)
{
    extern __shared__ float s_tab[];
    const bool takes_out = stage_table(a, s_tab);
    const Lanes m = lanes_of<LPH>(a.heads);
    const int lane = threadIdx.x & 63;
    const int part = lane % LPH, hl = (lane / LPH) % m.slots, es = lane / (LPH * m.slots);
    const int span = 64 / (LPH * m.slots);  // edges at once
    const bool wide = part * 4 < a.dim;     // (the last lanes of a head whose width is no power of two idle)
    const int ch = wide ? part * 4 : 0;
    const float scale2 = a.scale * kLog2e;
    const Walk w = walk_of(a.L, kWaves);
    for (int64_t u = w.at; u < w.end; u += w.step) {
        const Piece p = piece_of(a.L, w, u);
        if (p.node < 0) continue;
        const int h_raw = (int)blockIdx.y * m.per_wave + hl;
        const bool mine = hl < m.per_wave && h_raw < a.heads;
        const int h = mine ? h_raw : 0;
        const int64_t kch = (int64_t)(h / a.per) * a.dim + ch;
        float q[4], acc[4] = {0, 0, 0, 0};
        load4((const T*)a.q + p.node * a.ldq + (int64_t)h * a.dim + ch, q);
        if (!wide)
            for (int i = 0; i < 4; ++i) q[i] = 0;
        float mx = -INFINITY, l = 0;
        Entries<kUnroll> entry;
        entry.load(a, p, p.begin + es, span);
        for (int e0 = p.begin; e0 < p.end; e0 += kUnroll * span) {
            float k[kUnroll][4], v[kUnroll][4], s[kUnroll];
            bool there[kUnroll];
#pragma unroll
            for (int r = 0; r < kUnroll; ++r) {
                const int64_t j = entry.node[r];
                load4((const T*)a.k + j * a.ldk + kch, k[r]);
                load4((const T*)a.v + j * a.ldv + kch, v[r]);
                s[r] = e0 + r * span + es < p.end ? 0.0f : -INFINITY;
                if (a.table) s[r] += s_tab[entry.bucket[r] * a.heads + h];
                there[r] = s[r] != -INFINITY;
            }
            // (lanes past the row's end hold its last edge: a weight of zero must not meet an infinity)
            const bool hides = takes_out || p.end - e0 < kUnroll * span;
            entry.load(a, p, e0 + kUnroll * span + es, span);
            float top = mx;
#pragma unroll
            for (int r = 0; r < kUnroll; ++r) {
                if (!wide)
                    for (int i = 0; i < 4; ++i) k[r][i] = 0;
                float d = q[0] * k[r][0];
                d = fmaf(q[1], k[r][1], d);
                d = fmaf(q[2], k[r][2], d);
                d = fmaf(q[3], k[r][3], d);
                d = sum_lanes<LPH>(d);
                // an edge that is not there stays at -inf whatever its product is
                s[r] = there[r] ? fmaf(d, scale2, s[r]) : s[r];
                top = fmaxf(top, s[r]);
            }
            const float base = top == -INFINITY ? 0.0f : top;
            const float shrink = exp2_fast(mx - base);
            l *= shrink;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= shrink;
#pragma unroll
            for (int r = 0; r < kUnroll; ++r) {
                const float pr = exp2_fast(s[r] - base);
                if (hides && !there[r])
                    for (int i = 0; i < 4; ++i) v[r][i] = 0;
                l += pr;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = fmaf(pr, v[r][i], acc[i]);
            }
            mx = top;
        }
        // the edges that the wave took side by side
        for (int o = LPH * m.slots; o < 64; o *= 2) {
            const float m2 = __shfl_xor(mx, o, 64), l2 = __shfl_xor(l, o, 64);
            const float top = fmaxf(mx, m2), base = top == -INFINITY ? 0.0f : top;
            const float f1 = exp2_fast(mx - base), f2 = exp2_fast(m2 - base);
            l = l * f1 + l2 * f2;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = acc[i] * f1 + __shfl_xor(acc[i], o, 64) * f2;
            mx = top;
        }
        if (es != 0 || !mine) continue;
        if (p.item >= 0) {
            if (part == 0) {
                a.part_m[p.item * a.heads + h] = mx;
                a.part_l[p.item * a.heads + h] = l;
            }
            if (wide) store4(a.part_acc + (p.item * a.heads + h) * a.dim + ch, acc);
            continue;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = l == 0.0f ? 0.0f : acc[i] * inv;
        const int64_t at = ((int64_t)p.node * a.heads + h) * a.dim + ch;
        if (wide) {
            store4((T*)a.out + at, acc);
            if (a.out32) store4(a.out32 + at, acc);
        }
        if (part == 0) store_norm(a, (int64_t)p.node * a.heads + h, mx, l);
    }
}

// A workgroup joins the parts of one long row for 64 channels: sixteen lanes of four channels times
// STRANDS over the parts (four to a wave), first for the maximum, then for the sums against it,
// so that a strand's loads do not wait for each other.

__device__ __forceinline__ float strand_sum(float x)
{
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

template <typename T, int STRANDS>
__global__ __launch_bounds__(16 * STRANDS) void forward_join_kernel(AttnArgs a, int slices)
{
    const int64_t unit = workgroup(), rank = unit / slices;
    const int slot = rank < a.L.n_long ? a.L.long_slot[rank] : -1, slice = (int)(unit % slices);
    if (slot < 0) return;  // (fewer long rows than said)
    const int first = a.L.item_first[slot], n = a.L.item_first[slot + 1] - first, node = a.L.order[slot];
    constexpr int kJoinWaves = STRANDS / 4;
    __shared__ float s_m[kJoinWaves][16], s_l[kJoinWaves][16], s_acc[kJoinWaves][4][16];
    const int x = threadIdx.x % 16, y = threadIdx.x / 16, wave = threadIdx.x / 64;
    const int wide = a.heads * a.dim, ch = slice * 64 + x * 4;
    const int h = min(ch, wide - 4) / a.dim;
    float mx = -INFINITY;
#pragma unroll 4
    for (int i = y; i < n; i += STRANDS) mx = fmaxf(mx, a.part_m[(int64_t)(first + i) * a.heads + h]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    s_m[wave][x] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinWaves; ++i) mx = fmaxf(mx, s_m[i][x]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    float l = 0, acc[4] = {0, 0, 0, 0};
    if (ch < wide)
#pragma unroll 4
        for (int i = y; i < n; i += STRANDS) {
            const int64_t it = first + i;
            const float f = exp2_fast(a.part_m[it * a.heads + h] - base);
            float b[4];
            load4(a.part_acc + it * wide + ch, b);
            l = fmaf(a.part_l[it * a.heads + h], f, l);
            for (int c = 0; c < 4; ++c) acc[c] = fmaf(b[c], f, acc[c]);
        }
    s_l[wave][x] = strand_sum(l);
    for (int c = 0; c < 4; ++c) s_acc[wave][c][x] = strand_sum(acc[c]);
    __syncthreads();
    if (y != 0 || ch >= wide) return;
    l = 0;
    for (int c = 0; c < 4; ++c) acc[c] = 0;
#pragma unroll
    for (int i = 0; i < kJoinWaves; ++i) {
        l += s_l[i][x];
        for (int c = 0; c < 4; ++c) acc[c] += s_acc[i][c][x];
    }
    for (int c = 0; c < 4; ++c) acc[c] = l == 0.0f ? 0.0f : acc[c] / l;
    const int64_t at = (int64_t)node * wide + ch;
    store4((T*)a.out + at, acc);
    if (a.out32) store4(a.out32 + at, acc);
    if (ch % a.dim == 0) store_norm(a, (int64_t)node * a.heads + h, mx, l);
}

// By target: dq, the table's gradient, and what the pass by source needs of a row.
template <typename T, int LPH>
__global__ __launch_bounds__(64 * kWaves) void backward_q_kernel(AttnArgs a)
{
    extern __shared__ float s_tab[];
    const bool takes_out = stage_table(a, s_tab);
    const Lanes m = lanes_of<LPH>(a.heads);
    const int lane = threadIdx.x & 63;
    const int part = lane % LPH, hl = (lane / LPH) % m.slots, es = lane / (LPH * m.slots);
    const int span = 64 / (LPH * m.slots);
    const bool wide = part * 4 < a.dim;
    const int ch = wide ? part * 4 : 0;
    const float scale2 = a.scale * kLog2e;
    // each wave's, and each edge's of those side by side, own copy of the table's gradient
    const int cells = a.n_buckets * a.heads;
    float* s_dtab = s_tab + cells;
    if (a.dtab)
        for (int i = threadIdx.x; i < kWaves * span * cells; i += blockDim.x) s_dtab[i] = 0;
    __syncthreads();
    float* my_dtab = s_dtab + ((threadIdx.x / 64) * span + es) * cells;
    const Walk w = walk_of(a.L, kWaves);
    for (int64_t u = w.at; u < w.end; u += w.step) {
        const Piece p = piece_of(a.L, w, u);
        if (p.node < 0) continue;
        const int h_raw = (int)blockIdx.y * m.per_wave + hl;
        const bool mine = hl < m.per_wave && h_raw < a.heads;
        const int h = mine ? h_raw : 0;
        const int64_t kch = (int64_t)(h / a.per) * a.dim + ch;
        const int64_t row = ((int64_t)p.node * a.heads + h) * a.dim + ch;
        float q[4], g[4], o[4], dq[4] = {0, 0, 0, 0};
        load4((const T*)a.q + p.node * a.ldq + (int64_t)h * a.dim + ch, q);
        load4((const T*)a.g + p.node * a.ldg + (int64_t)h * a.dim + ch, g);
        load4(a.out32 + row, o);
        if (!wide)
            for (int i = 0; i < 4; ++i) q[i] = g[i] = o[i] = 0;
        float delta = g[0] * o[0];
        for (int i = 1; i < 4; ++i) delta = fmaf(g[i], o[i], delta);
        delta = sum_lanes<LPH>(delta);
        const float2 norm = a.norm[(int64_t)p.node * a.heads + h];
        if (part == 0 && es == 0 && mine)
            a.stats[(int64_t)p.node * a.heads + h] = make_float4(norm.x, norm.y, delta, 0.0f);
        Entries<kUnroll> entry;
        entry.load(a, p, p.begin + es, span);
        for (int e0 = p.begin; e0 < p.end; e0 += kUnroll * span) {
            float k[kUnroll][4], v[kUnroll][4], s[kUnroll];
            int b[kUnroll];
#pragma unroll
            for (int r = 0; r < kUnroll; ++r) {
                const int64_t j = entry.node[r];
                load4((const T*)a.k + j * a.ldk + kch, k[r]);
                load4((const T*)a.v + j * a.ldv + kch, v[r]);
                s[r] = e0 + r * span + es < p.end ? 0.0f : -INFINITY;
                b[r] = entry.bucket[r] * a.heads + h;
                if (a.table) s[r] += s_tab[b[r]];
            }
            entry.load(a, p, e0 + kUnroll * span + es, span);
#pragma unroll
            for (int r = 0; r < kUnroll; ++r) {
                if (!wide)
                    for (int i = 0; i < 4; ++i) k[r][i] = v[r][i] = 0;
                float d = q[0] * k[r][0], dp = g[0] * v[r][0];
                for (int i = 1; i < 4; ++i) {
                    d = fmaf(q[i], k[r][i], d);
                    dp = fmaf(g[i], v[r][i], dp);
                }
                d = sum_lanes<LPH>(d);
                dp = sum_lanes<LPH>(dp);
                const bool there = s[r] != -INFINITY;
                const float pr = exp2_fast(fmaf(d, scale2, s[r]) - norm.x) * norm.y;
                const float ds = there ? pr * (dp - delta) : 0.0f;
                if (takes_out && !there)
                    for (int i = 0; i < 4; ++i) k[r][i] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) dq[i] = fmaf(ds, k[r][i], dq[i]);
                if (a.dtab && part == 0 && mine && there) my_dtab[b[r]] += ds;
            }
        }
        for (int o2 = LPH * m.slots; o2 < 64; o2 *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) dq[i] += __shfl_xor(dq[i], o2, 64);
        if (es != 0 || !mine || !wide) continue;
        if (p.item >= 0) {
            store4(a.part_acc + (p.item * a.heads + h) * a.dim + ch, dq);
        } else {
            for (int i = 0; i < 4; ++i) dq[i] *= a.scale;
            store4((T*)a.dq + row, dq);
        }
    }
    if (!a.dtab) return;
    __syncthreads();
    for (int i = threadIdx.x; i < cells; i += blockDim.x) {
        float x = 0;
        for (int c = 0; c < kWaves * span; ++c) x += s_dtab[c * cells + i];
        a.dtab[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * cells + i] = x;
    }
}

// By source: dk and dv.  Lanes sit on k's heads; the q heads that share one follow each other.
template <typename T, int LPH>
__global__ __launch_bounds__(64 * kWaves) void backward_kv_kernel(AttnArgs a)
{
    extern __shared__ float s_tab[];
    const bool takes_out = stage_table(a, s_tab);
    const Lanes m = lanes_of<LPH>(a.kv_heads);
    const int lane = threadIdx.x & 63;
    const int part = lane % LPH, hl = (lane / LPH) % m.slots, es = lane / (LPH * m.slots);
    const int span = 64 / (LPH * m.slots);
    const bool wide = part * 4 < a.dim;
    const int ch = wide ? part * 4 : 0;
    const float scale2 = a.scale * kLog2e;
    constexpr int kTwo = 2;
    const Walk w = walk_of(a.L, kWaves);
    for (int64_t u = w.at; u < w.end; u += w.step) {
        const Piece p = piece_of(a.L, w, u);
        if (p.node < 0) continue;
        const int c_raw = (int)blockIdx.y * m.per_wave + hl;
        const bool mine = hl < m.per_wave && c_raw < a.kv_heads;
        const int c = mine ? c_raw : 0;
        float k[4], v[4], dk[4] = {0, 0, 0, 0}, dv[4] = {0, 0, 0, 0};
        load4((const T*)a.k + p.node * a.ldk + (int64_t)c * a.dim + ch, k);
        load4((const T*)a.v + p.node * a.ldv + (int64_t)c * a.dim + ch, v);
        if (!wide)
            for (int i = 0; i < 4; ++i) k[i] = v[i] = 0;
        Entries<kTwo> entry;
        entry.load(a, p, p.begin + es, span);
        for (int e0 = p.begin; e0 < p.end; e0 += kTwo * span) {
            int64_t t[kTwo];
            int b[kTwo];
            bool in[kTwo];
#pragma unroll
            for (int r = 0; r < kTwo; ++r) {
                t[r] = entry.node[r];
                b[r] = entry.bucket[r] * a.heads;
                in[r] = e0 + r * span + es < p.end;
            }
            entry.load(a, p, e0 + kTwo * span + es, span);
            for (int x = 0; x < a.per; ++x) {
                const int h = c * a.per + x;
                float q[kTwo][4], g[kTwo][4], s[kTwo];
                float4 st[kTwo];
#pragma unroll
                for (int r = 0; r < kTwo; ++r) {
                    load4((const T*)a.q + t[r] * a.ldq + (int64_t)h * a.dim + ch, q[r]);
                    load4((const T*)a.g + t[r] * a.ldg + (int64_t)h * a.dim + ch, g[r]);
                    st[r] = a.stats[t[r] * a.heads + h];
                    s[r] = in[r] ? 0.0f : -INFINITY;
                    if (a.table) s[r] += s_tab[b[r] + h];
                }
#pragma unroll
                for (int r = 0; r < kTwo; ++r) {
                    if (!wide)
                        for (int i = 0; i < 4; ++i) q[r][i] = g[r][i] = 0;
                    float d = q[r][0] * k[0], dp = g[r][0] * v[0];
                    for (int i = 1; i < 4; ++i) {
                        d = fmaf(q[r][i], k[i], d);
                        dp = fmaf(g[r][i], v[i], dp);
                    }
                    d = sum_lanes<LPH>(d);
                    dp = sum_lanes<LPH>(dp);
                    const bool there = s[r] != -INFINITY;
                    const float pr = there ? exp2_fast(fmaf(d, scale2, s[r]) - st[r].x) * st[r].y : 0.0f;
                    const float ds = there ? pr * (dp - st[r].z) : 0.0f;
                    if (!there && (takes_out || !in[r]))
                        for (int i = 0; i < 4; ++i) q[r][i] = g[r][i] = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        dk[i] = fmaf(ds, q[r][i], dk[i]);
                        dv[i] = fmaf(pr, g[r][i], dv[i]);
                    }
                }
            }
        }
        for (int o2 = LPH * m.slots; o2 < 64; o2 *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dk[i] += __shfl_xor(dk[i], o2, 64);
                dv[i] += __shfl_xor(dv[i], o2, 64);
            }
        if (es != 0 || !mine || !wide) continue;
        if (p.item >= 0) {
            const int64_t at = (p.item * a.kv_heads + c) * a.dim + ch;
            store4(a.part_acc + at, dk);
            store4(a.part_acc2 + at, dv);
        } else {
            const int64_t at = ((int64_t)p.node * a.kv_heads + c) * a.dim + ch;
            for (int i = 0; i < 4; ++i) dk[i] *= a.scale;
            store4((T*)a.dk + at, dk);
            store4((T*)a.dv + at, dv);
        }
    }
}

// The sum of the parts of one long row, as forward_join_kernel lays it out.
template <typename T, int STRANDS>
__global__ __launch_bounds__(16 * STRANDS) void sum_join_kernel(Lists L, const float* __restrict__ part, int wide,
                                                                 int slices, float factor, T* __restrict__ out)
{
    const int64_t unit = workgroup(), rank = unit / slices;
    const int slot = rank < L.n_long ? L.long_slot[rank] : -1, slice = (int)(unit % slices);
    if (slot < 0) return;
    const int first = L.item_first[slot], n = L.item_first[slot + 1] - first, node = L.order[slot];
    constexpr int kJoinWaves = STRANDS / 4;
    __shared__ float s_acc[kJoinWaves][4][16];
    const int x = threadIdx.x % 16, y = threadIdx.x / 16, wave = threadIdx.x / 64;
    const int ch = slice * 64 + x * 4;
    float acc[4] = {0, 0, 0, 0};
    if (ch < wide)
#pragma unroll 4
        for (int i = y; i < n; i += STRANDS) {
            float b[4];
            load4(part + (int64_t)(first + i) * wide + ch, b);
            for (int c = 0; c < 4; ++c) acc[c] += b[c];
        }
    for (int c = 0; c < 4; ++c) s_acc[wave][c][x] = strand_sum(acc[c]);
    __syncthreads();
    if (y != 0 || ch >= wide) return;
    for (int c = 0; c < 4; ++c) acc[c] = 0;
#pragma unroll
    for (int i = 0; i < kJoinWaves; ++i)
        for (int c = 0; c < 4; ++c) acc[c] += s_acc[i][c][x];
    for (int c = 0; c < 4; ++c) acc[c] *= factor;
    store4(out + (int64_t)node * wide + ch, acc);
}

// The table's gradient from the workgroups' sums: 16 columns and 64 strands a workgroup.
__global__ __launch_bounds__(1024) void table_join_kernel(const float* __restrict__ part, int groups, int cells,
                                                          float* __restrict__ out)
{
    __shared__ float s_x[64][17];
    const int x = threadIdx.x % 16, y = threadIdx.x / 16;
    const int cell = blockIdx.x * 16 + x;
    float sum = 0;
    if (cell < cells)
        for (int i = y; i < groups; i += 64) sum += part[(int64_t)i * cells + cell];
    s_x[y][x] = sum;
    __syncthreads();
    if (y != 0 || cell >= cells) return;
    for (int i = 1; i < 64; ++i) sum += s_x[i][x];
    out[cell] = sum;
}

// ---------------------------------------------------------------- host
constexpr int64_t kMaxNodes = 0x7fffff00LL;  // as of the lists

// Lanes of a head: a lane's four channels, rounded up to a power of two.
int lanes_per_head(int dim)
{
    int l = 2;
    while (4 * l < dim) l *= 2;
    return l;
}

// A wave for each row (or part) of each group of heads, up to what fills every CU; the kernels
// walk what is left over.
dim3 grid_of(const Lists& L, int head_groups, int per_cu)
{
    const int64_t most = std::max(1, 256 * per_cu / head_groups);
    const int64_t need = (L.n_items + L.n_rows + kWaves - 1) / kWaves;
    return dim3((unsigned)std::max<int64_t>(1, std::min(most, need)), (unsigned)head_groups);
}

// (600,000 edges of 8 heads of 32 floats: 144 us with 4, 137 us with 6, 138 us with 8)
constexpr int kGroupsPerCu = 6;

struct Layout {
    size_t o_stats, o_dtab, o_m, o_l, o_acc, o_acc2, total;
};

Layout layout(const dg_attention_desc* d, const dg_neighbor_lists* t, const dg_neighbor_lists* s)
{
    Layout L;
    size_t o = 0;
    auto take = [&](size_t b) { size_t r = o; o = al(o + (b ? b : 1)); return r; };
    const size_t q = (size_t)d->heads * d->dim, kv = (size_t)d->kv_heads * d->dim;
    const size_t ti = (size_t)t->n_items, si = s ? (size_t)s->n_items : 0;
    L.o_stats = take(s ? 16 * (size_t)d->n_targets * d->heads : 0);
    L.o_dtab = take(s ? 4 * (size_t)std::max({256 * kGroupsPerCu, kMfmaTableParts, d->heads}) * d->n_buckets * d->heads : 0);
    L.o_m = take(s ? 0 : 4 * ti * d->heads);
    L.o_l = take(s ? 0 : 4 * ti * d->heads);
    L.o_acc = take(4 * std::max(ti * q, si * kv));
    L.o_acc2 = take(4 * si * kv);
    L.total = o;
    return L;
}

dg_status check(const dg_attention_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->dtype != DG_F32 && d->dtype != DG_BF16)
        return fail(DG_ERR_INVALID, "q, k and v must be float32 or bfloat16");
    if (d->n_nodes < 0 || d->n_nodes > kMaxNodes) return fail(DG_ERR_INVALID, "n_nodes must be in [0, 2^31 - 256]");
    if (d->n_targets < 0 || d->n_nodes < d->n_targets)
        return fail(DG_ERR_INVALID, "n_targets must be in [0, n_nodes]");
    if (d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads || d->heads > 1024)
        return fail(DG_ERR_INVALID, "heads must be a multiple of kv_heads, 1 to 1024");
    if (d->dim < 8 || d->dim > 256 || d->dim % 8)
        return fail(DG_ERR_INVALID, "the head width must be a multiple of 8, 8 to 256, got " + std::to_string(d->dim));
    if (d->n_buckets < 0 || d->n_buckets > 128 || (int64_t)d->n_buckets * d->heads > kMaxTable)
        return fail(DG_ERR_INVALID, "at most 128 buckets, and 4096 buckets times heads");
    const int64_t a = d->dtype == DG_F32 ? 4 : 8;  // rows start at 16 bytes
    const int64_t ld[4] = {d->ld_q, d->ld_k, d->ld_v, d->ld_g};
    for (int64_t x : ld)
        if (x % a || x < 0 || x > (1ll << 60) / (d->n_nodes + 1))  // (offsets in bytes stay below 2^63)
            return fail(DG_ERR_INVALID, "row strides must be multiples of 16 bytes, and all rows below 2^60 elements");
    if (!isfinite(d->scale)) return fail(DG_ERR_INVALID, "scale must be finite");
    return DG_OK;
}

dg_status check_lists(const dg_attention_desc* d, const dg_neighbor_lists* l)
{
    if (!l) return fail(DG_ERR_INVALID, "lists are NULL");
    if (l->n_rows != d->n_nodes) return fail(DG_ERR_INVALID, "the lists are of another number of nodes");
    if (l->n_rows > 0 && (!l->order || !l->ptr || !l->idx)) return fail(DG_ERR_INVALID, "lists are NULL");
    if (d->n_buckets > 0 && !l->bucket) return fail(DG_ERR_INVALID, "a table, but the lists hold no buckets");
    if (l->n_items > kMaxNodes || l->n_long > kMaxNodes)
        return fail(DG_ERR_INVALID, "lists hold less than 2^31 parts");
    if (l->n_items < 0 || (l->n_items > 0 && (!l->items || !l->item_first || !l->long_slot || l->n_long < 1)))
        return fail(DG_ERR_INVALID, "the parts of long rows are NULL");
    return DG_OK;
}

Lists lists_of(const dg_neighbor_lists* l, int64_t rows)
{
    Lists r;
    r.n_rows = rows;
    r.n_items = l->n_items;
    r.order = l->order;
    r.ptr = l->ptr;
    r.idx = l->idx;
    r.bucket = l->bucket;
    r.items = (const int4*)l->items;
    r.item_first = l->item_first;
    r.long_slot = l->long_slot;
    r.n_long = l->n_long;
    return r;
}

AttnArgs args_of(const dg_attention_desc* d, const void* q, const void* k, const void* v, const float* table)
{
    AttnArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = d->ld_q;
    a.ldk = d->ld_k;
    a.ldv = d->ld_v;
    a.ldg = d->ld_g;
    a.table = d->n_buckets > 0 ? table : nullptr;
    a.n_buckets = a.table ? d->n_buckets : 0;
    a.n_targets = d->n_targets;
    a.n_nodes = d->n_nodes;
    a.heads = d->heads;
    a.kv_heads = d->kv_heads;
    a.dim = d->dim;
    a.per = d->heads / d->kv_heads;
    a.scale = d->scale;
    return a;
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

template <int LPH>
struct Width {
    static constexpr int lph = LPH;
};

// f(Width<LPH>) for the head width
template <typename T, typename F>
void by_width(int dim, F&& f)
{
    if constexpr (sizeof(T) == 2) {  // (heads of up to kMfmaDim channels go to the matrix units)
        f(Width<64>{});
        return;
    }
    switch (lanes_per_head(dim)) {
    case 2: f(Width<2>{}); break;
    case 4: f(Width<4>{}); break;
    case 8: f(Width<8>{}); break;
    case 16: f(Width<16>{}); break;
    case 32: f(Width<32>{}); break;
    default: f(Width<64>{}); break;
    }
}

// f(strands of the joins): 64 where the long rows have many parts, one wave where there are few (the
// whole forward pass, 8 heads of 32: 4 rows of 348 parts 67 us with 64 strands, 81 us with 4; 1000
// rows of 2 parts 152 us with 64, 125 us with 4).
template <typename F>
void by_parts(const Lists& L, F&& f)
{
    if (L.n_items > 16 * L.n_long) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 4>{});
}

template <typename T>
void run_forward(const AttnArgs& a, hipStream_t s)
{
    // (bfloat16 on the matrix units: 26.5M edges of 8 heads of 16 take 840 us there, 2016 us here; the
    // registers of a wave hold heads of up to kMfmaDim channels)
    if (sizeof(T) == 2 && a.dim <= kMfmaDim) {
        forward_mfma(a, s);
    } else {
        const size_t lds = 4 * (size_t)a.n_buckets * a.heads;
        by_width<T>(a.dim, [&](auto w) {
            constexpr int LPH = decltype(w)::lph;
            hipLaunchKernelGGL((forward_kernel<T, LPH>), grid_of(a.L, lanes_of<LPH>(a.heads).groups, kGroupsPerCu),
                               dim3(64 * kWaves), lds, s, a);
        });
    }
    if (a.L.n_items > 0) {
        const int slices = (a.heads * a.dim + 63) / 64;
        by_parts(a.L, [&](auto strands) {
            hipLaunchKernelGGL((forward_join_kernel<T, strands()>), workgroups(a.L.n_long * slices),
                               dim3(16 * strands()), 0, s, a, slices);
        });
    }
}

template <typename T>
void run_backward(AttnArgs a, const Lists& by_target, const Lists& by_source, float* dtable, hipStream_t s)
{
    // (the matrix kernels' rows without entries read some target's row: there has to be one)
    const bool matrix = sizeof(T) == 2 && a.dim <= kMfmaDim && a.n_targets > 0;
    const size_t cells = (size_t)a.n_buckets * a.heads;
    a.L = by_target;
    unsigned groups = 1;
    if (matrix) {
        groups = backward_q_mfma(a, s);
    } else {
        by_width<T>(a.dim, [&](auto w) {
            constexpr int LPH = decltype(w)::lph;
            const Lanes m = lanes_of<LPH>(a.heads);
            const int span = 64 / (LPH * m.slots);
            const dim3 grid = grid_of(a.L, m.groups, kGroupsPerCu);
            groups = grid.x * grid.y;
            const size_t lds = 4 * cells * (1 + (a.dtab ? kWaves * span : 0));
            hipLaunchKernelGGL((backward_q_kernel<T, LPH>), grid, dim3(64 * kWaves), lds, s, a);
        });
    }
    if (a.dtab)
        hipLaunchKernelGGL(table_join_kernel, dim3(nblk((int64_t)cells, 16)), dim3(1024), 0, s, (const float*)a.dtab,
                           (int)groups, (int)cells, dtable);
    if (a.L.n_items > 0) {
        const int wide = a.heads * a.dim, slices = (wide + 63) / 64;
        by_parts(a.L, [&](auto strands) {
            hipLaunchKernelGGL((sum_join_kernel<T, strands()>), workgroups(a.L.n_long * slices),
                               dim3(16 * strands()), 0, s, a.L, (const float*)a.part_acc, wide, slices, a.scale,
                               (T*)a.dq);
        });
    }
    a.L = by_source;
    if (matrix) {
        backward_kv_mfma(a, s);
    } else {
        by_width<T>(a.dim, [&](auto w) {
            constexpr int LPH = decltype(w)::lph;
            hipLaunchKernelGGL((backward_kv_kernel<T, LPH>), grid_of(a.L, lanes_of<LPH>(a.kv_heads).groups, kGroupsPerCu),
                               dim3(64 * kWaves), 4 * cells, s, a);
        });
    }
    if (a.L.n_items > 0) {
        const int wide = a.kv_heads * a.dim, slices = (wide + 63) / 64;
        by_parts(a.L, [&](auto strands) {
            const dim3 grid = workgroups(a.L.n_long * slices), block(16 * strands());
            hipLaunchKernelGGL((sum_join_kernel<T, strands()>), grid, block, 0, s, a.L, (const float*)a.part_acc, wide,
                               slices, a.scale, (T*)a.dk);
            hipLaunchKernelGGL((sum_join_kernel<T, strands()>), grid, block, 0, s, a.L, (const float*)a.part_acc2, wide,
                               slices, 1.0f, (T*)a.dv);
        });
    }
}

}  // namespace

extern "C" {

size_t dg_attention_workspace_size(const dg_attention_desc* d, const dg_neighbor_lists* by_target,
                                   const dg_neighbor_lists* by_source)
{
    if (check(d) != DG_OK || check_lists(d, by_target) != DG_OK) return 0;
    if (by_source && check_lists(d, by_source) != DG_OK) return 0;
    return layout(d, by_target, by_source).total;
}

dg_status dg_attention_forward(const dg_attention_desc* d, const dg_neighbor_lists* by_target, const void* q,
                               const void* k, const void* v, const float* table, void* out, float* out32, float* norm,
                               float* lse, void* ws, size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st == DG_OK) st = check_lists(d, by_target);
    if (st != DG_OK) return st;
    const Layout L = layout(d, by_target, nullptr);
    if (by_target->n_items > 0 && (!ws || ws_bytes < L.total)) return fail(DG_ERR_WORKSPACE, "workspace too small");
    if (d->n_targets == 0) return DG_OK;
    if (!q || !k || !v || !out || (d->n_buckets > 0 && !table))
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out) || !aligned(out32))
        return fail(DG_ERR_INVALID, "tensors must be aligned to 16 bytes");
    char* w = (char*)ws;
    AttnArgs a = args_of(d, q, k, v, table);
    a.L = lists_of(by_target, d->n_targets);
    a.out = out;
    a.out32 = out32;
    a.norm = (float2*)norm;
    a.lse = lse;
    a.part_m = (float*)(w + L.o_m);
    a.part_l = (float*)(w + L.o_l);
    a.part_acc = (float*)(w + L.o_acc);
    if (d->dtype == DG_BF16) run_forward<__bf16>(a, s);
    else run_forward<float>(a, s);
    return launched("dg_attention_forward");
}

dg_status dg_attention_backward(const dg_attention_desc* d, const dg_neighbor_lists* by_target,
                                const dg_neighbor_lists* by_source, const void* q, const void* k, const void* v,
                                const float* table, const float* out32, const float* norm, const void* grad_out,
                                void* dq, void* dk, void* dv, float* dtable, void* ws, size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st == DG_OK) st = check_lists(d, by_target);
    if (st == DG_OK) st = check_lists(d, by_source);
    if (st != DG_OK) return st;
    const Layout L = layout(d, by_target, by_source);
    if (!ws || ws_bytes < L.total) return fail(DG_ERR_WORKSPACE, "workspace too small");
    if (d->n_nodes == 0) {  // (no terms: the table's gradient is zeros, the others are empty)
        const int cells = d->n_buckets * d->heads;
        if (cells == 0) return DG_OK;
        if (!dtable) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
        hipLaunchKernelGGL(table_join_kernel, dim3(nblk(cells, 16)), dim3(1024), 0, s, (const float*)nullptr, 0, cells,
                           dtable);
        return launched("dg_attention_backward");
    }
    if (!k || !v || !dk || !dv || (d->n_targets > 0 && (!q || !out32 || !norm || !grad_out || !dq)) ||
        (d->n_buckets > 0 && (!table || !dtable)))
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(grad_out) || !aligned(out32) || !aligned(dq) ||
        !aligned(dk) || !aligned(dv))
        return fail(DG_ERR_INVALID, "tensors must be aligned to 16 bytes");
    char* w = (char*)ws;
    AttnArgs a = args_of(d, q, k, v, table);
    a.g = grad_out;
    a.out32 = const_cast<float*>(out32);
    a.norm = (float2*)const_cast<float*>(norm);
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.stats = (float4*)(w + L.o_stats);
    a.dtab = a.table ? (float*)(w + L.o_dtab) : nullptr;
    a.part_acc = (float*)(w + L.o_acc);
    a.part_acc2 = (float*)(w + L.o_acc2);
    const Lists to = lists_of(by_target, d->n_targets), fro = lists_of(by_source, d->n_nodes);
    if (d->dtype == DG_BF16) run_backward<__bf16>(a, to, fro, dtable, s);
    else run_backward<float>(a, to, fro, dtable, s);
    return launched("dg_attention_backward");
}

}  // extern "C"
