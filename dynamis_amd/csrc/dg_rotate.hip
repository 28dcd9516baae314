// dg_rotate.hip -- heads of queries and keys, normalised and rotated by their atoms' positions:
// forward and backward.
//
//   n[c]     = x[c] / sqrt(mean_c x[c]^2 + eps) * w[c]              (or n = x)
//   theta[j] = position[i, axis(j)] * frequency[j]                  pair j = channels (j, j + P) or (2j, 2j + 1)
//   y_a = n_a cos - n_b sin,   y_b = n_a sin + n_b cos              channels from 2 P on: y = n
//
//   g' = the gradient of y turned back by theta;  xhat = x / rms;  t = g' w
//   dx = (t - xhat mean(t xhat)) / rms,   dw = sum g' xhat,
//   dtheta[j] = sum_heads n_a g'_b - n_b g'_a,   dposition[i, a] = sum_{j of axis a} frequency[j] dtheta[j]
//
// Every element is read and written once, with some twenty operations: bound by memory.  A lane
// holds 16 bytes of a head, a power of two of lanes the head, and a group of lanes all heads of one
// atom, as many at once as there are lanes; waves share nothing, so there is no barrier.  The
// angles' sines are made once for an atom and serve all of its heads from LDS.  An angle is
// worked out in turns in 64 bits and brought into half a turn before it is rounded: positions are
// as far away as they like.  Where pairs lie P channels apart a channel's partner, at any P,
// comes through LDS, in 32 bits.  All sums have one owner and one order.  The gradient of positions that have
// 64 bits is worked out in them from the inputs on, sines and mean squares included.
//
// 8 + 8 heads of 32 in bfloat16, 1M atoms: 396 us, 5.2 TB/s, what a copy reaches.  16 + 4 heads of 64, 32,000
// atoms: forward 37 us (4.4 TB/s), backward 74 (3.3 TB/s), which its instructions bound (some 250 for a lane's
// 8 channels, at three waves a SIMD).  864 atoms: 5.8 us, the latency of a position, its angle and a row in turn.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "../../include/dynamis_graph.h"
#include "dg_lanes.hpp"

namespace dg {
dg_status fail(dg_status st, const std::string& msg);  // dg_graph.hip
}

namespace {

using namespace dg;

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f32x4 = __attribute__((ext_vector_type(4))) float;

constexpr int kWaves = 4;
constexpr int kMaxAxes = 8;
// Workgroups: each takes as many atoms as the others, so a second round of them would leave most of the card idle.
// Measured in bfloat16: 1M atoms forward, interleaved, 404 us with 1536, 451 with 2048; backward of 32,000, pairs
// apart, three waves a SIMD, 73 us with 768, 89 with 1024.  The other instances have the same or, backward,
// as many as their registers let reside (float three to five waves a SIMD; wide two, in float three); 32,000 atoms,
// 16 + 4 heads of 64, pairs apart and interleaved: forward 31 and 29 us, in float 62 and 62 (328 MB, a copy's rate);
// backward 66 and 56, in float 103 and 102 (492 MB, 95 at a copy's rate), wide 114 and 103, in float 139 and 133 (with as many as without
// 145 and 131, 173 and 163).  The norms' weights' gradients are summed by workgroup, so above 512 of them their last bits go
// with whether float64 positions want a gradient.
constexpr int kForwardBlocks = 1536;
constexpr int kMaxBlocks = 1024;
inline int backward_blocks(int32_t dtype, bool wide) { return dtype == DG_BF16 ? (wide ? 512 : 768) : wide ? 768 : kMaxBlocks; }

template <typename T>
constexpr int kC = 16 / (int)sizeof(T);  // channels of a lane

struct Args {
    const void *q, *k, *pos, *gq, *gk, *qw, *kw;
    const float* freq;
    void *oq, *ok;    // results, or (backward) dq and dk
    void* dpos;
    float* part;      // [blocks, 2, dim] sums of dw
    int64_t targets, nodes, ldq, ldk, ldgq, ldgk;
    int heads, kv, dim, pairs, axes, pos_dtype;
    int norm, w_own;  // w_own: the weights are of the heads' type (else float)
    float eps, inv_dim;
    int per, at_once;  // lanes of a head; heads at once (powers of two, their product up to 64)
    int count, batch;  // atoms of a wave's step; atoms whose angles it makes at once, a multiple of those
    int q_steps, steps;  // of an atom's heads of q, and of all
    int ends[kMaxAxes];  // pairs up to and with an axis
};

template <typename T>
__device__ __forceinline__ void unpack(u32x4 r, float (&v)[kC<T>])
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 f = __builtin_bit_cast(f32x4, r);
        for (int i = 0; i < 4; ++i) v[i] = f[i];
    } else {
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __builtin_bit_cast(float, r[i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
        }
    }
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&v)[kC<T>])
{
    u32x4 r;
    if constexpr (sizeof(T) == 4) {
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, v[i]);
    } else {
        using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * i], (__bf16)v[2 * i + 1]});
    }
    return r;
}

__device__ __forceinline__ double position(const Args& a, int64_t i)
{
    return a.pos_dtype == DG_F32   ? (double)((const float*)a.pos)[i]
           : a.pos_dtype == DG_F64 ? ((const double*)a.pos)[i]
                                   : (double)((const int64_t*)a.pos)[i];
}

__device__ __forceinline__ int axis_of(const Args& a, int j)
{
    int x = 0;
    for (int i = 0; i + 1 < a.axes; ++i) x += j >= a.ends[i];
    return x;
}

// LDS of a wave: its atoms' cosines and sines (at most 32 C of them, whatever the head; WIDE: in 64 bits too), and
// a word for each channel in flight.  One word in nine is spare, so that lanes eight apart do not meet.
template <typename T, bool WIDE>
struct Shared {
    double2 turn64[WIDE ? 32 * kC<T> : 1];
    float2 turn[32 * kC<T>];
    float row[64 * kC<T> + 64 * kC<T> / 8];
};
__device__ __forceinline__ int spread(int i) { return i + (i >> 3); }

// The norms' weights (ones without), [2][dim].
template <typename T>
__device__ __forceinline__ void load_weights(const Args& a, float* s_w)
{
    for (int i = threadIdx.x; i < 2 * a.dim; i += 64 * kWaves) {
        const void* w = i < a.dim ? a.qw : a.kw;
        const int c = i < a.dim ? i : i - a.dim;
        s_w[i] = !w ? 1.0f : a.w_own ? (float)((const T*)w)[c] : ((const float*)w)[c];
    }
    __syncthreads();
}

// Angles in turns.  A wave takes `batch` atoms at a time; where their pairs are no more than its lanes, a lane
// has its pair for good, and the next batch's position under way.
struct Angles {
    static constexpr double kInverse = 0.15915494309189533577;  // 1 / (2 pi)
    int t, axis;
    double freq, next;
};
__device__ __forceinline__ void prefetch(const Args& a, Angles& g, int64_t first)
{
    g.next = g.t < a.batch && first + g.t < a.nodes ? position(a, (first + g.t) * a.axes + g.axis) : 0.0;
}
__device__ __forceinline__ Angles make_angles(const Args& a, int lane, int64_t first)
{
    Angles g;
    g.t = lane / a.pairs;
    const int j = lane - g.t * a.pairs;
    g.axis = axis_of(a, j);
    g.freq = (double)a.freq[j] * Angles::kInverse;
    if (a.batch * a.pairs <= 64) prefetch(a, g, first);
    return g;
}
__device__ __forceinline__ float2 cos_sin(double turns)
{
    float sine, cosine;
    sincospif(2.0f * (float)(turns - rint(turns)), &sine, &cosine);
    return make_float2(cosine, sine);
}
template <typename T, bool WIDE>
__device__ __forceinline__ void make_turns(const Args& a, Angles& g, int64_t first, int64_t after, int lane, Shared<T, WIDE>& s)
{
    auto put = [&](int i, double turns) {
        s.turn[i] = cos_sin(turns);
        if constexpr (WIDE) {
            double sine, cosine;
            sincospi(2.0 * (turns - rint(turns)), &sine, &cosine);
            s.turn64[i] = make_double2(cosine, sine);
        }
    };
    if (a.batch * a.pairs <= 64) {
        const double at = g.next;
        prefetch(a, g, after);
        if (g.t < a.batch) put(lane, at * g.freq);
    } else {
        for (int i = lane; i < a.batch * a.pairs; i += 64) {
            const int t = i / a.pairs, j = i - t * a.pairs;
            const double at = first + t < a.nodes ? position(a, (first + t) * a.axes + axis_of(a, j)) : 0.0;
            put(i, at * ((double)a.freq[j] * Angles::kInverse));
        }
    }
    wave_sync();
}

// Where a lane works: chunk `c0` of head `slot` (plus a multiple of at_once) of atom `t` of the wave's.
// HALVES: where each channel's partner and its angle lie (bytes from Shared::row and from the atom's turns).
template <typename T, bool HALVES>
struct Seat {
    int c0, slot, t;
    int row;  // of the lane's channels in Shared::row
    uint32_t partner[HALVES ? kC<T> : 1];
    __device__ __forceinline__ Seat(const Args& a, int lane)
    {
        const int group = a.per * a.at_once;
        c0 = (lane & (a.per - 1)) * kC<T>;
        slot = (lane & (group - 1)) / a.per;
        t = lane / group;
        const int base = (lane & ~(a.per - 1)) * kC<T>;
        row = base + c0;
        if constexpr (HALVES)
            for (int i = 0; i < kC<T>; ++i) {
                const int c = c0 + i, j = c < a.pairs ? c : c - a.pairs;
                const int other = c < a.pairs ? c + a.pairs : j;
                partner[i] = c < 2 * a.pairs ? (uint32_t)spread(base + other) * 4 | (uint32_t)j << 19 : 0;
            }
    }
};

// The lane's channels v turned by the angles (BACK: by their opposites), with HALVES through LDS.  BACK: `across`
// is what a channel's n is multiplied by in the angle's gradient, g'_b for a pair's first and -g'_a for its
// second (a lane makes its partner's g' itself, and needs not its n).
template <typename T, bool HALVES, bool BACK, bool WIDE>
__device__ __forceinline__ void turn(const Args& a, const Seat<T, HALVES>& at, const float2* turns, Shared<T, WIDE>& s,
                                     const float (&v)[kC<T>], float (&y)[kC<T>], float (&across)[kC<T>])
{
    constexpr int C = kC<T>;
    if constexpr (HALVES) {
#pragma unroll
        for (int i = 0; i < C; ++i) s.row[spread(at.row + i)] = v[i];
        wave_sync();
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = at.c0 + i;
            const float other = *(const float*)((const char*)s.row + (at.partner[i] & 0xffff));
            const float2 z = *(const float2*)((const char*)turns + (at.partner[i] >> 16));
            const float sine = (c >= a.pairs) != BACK ? z.y : -z.y;
            const bool turned = c < 2 * a.pairs;
            y[i] = turned ? fmaf(v[i], z.x, other * sine) : v[i];
            // (the partner's: its own by cos, ours by the other sine)
            if constexpr (BACK) {
                const float theirs = fmaf(other, z.x, -(v[i] * sine));
                across[i] = !turned ? 0.0f : c < a.pairs ? theirs : -theirs;
            }
        }
        wave_sync();
    } else {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            const bool turned = at.c0 + i < 2 * a.pairs;
            const float2 z = turned ? turns[(at.c0 + i) / 2] : make_float2(1.0f, 0.0f);
            const float sine = BACK ? -z.y : z.y;
            y[i] = turned ? fmaf(v[i], z.x, -(v[i + 1] * sine)) : v[i];
            y[i + 1] = turned ? fmaf(v[i + 1], z.x, v[i] * sine) : v[i + 1];
            if constexpr (BACK) {
                across[i] = turned ? y[i + 1] : 0.0f;
                across[i + 1] = turned ? -y[i] : 0.0f;
            }
        }
    }
}

// What turn<BACK> calls `across`, times n, in 64 bits, added to `sum`: of gradients g and inputs x, r = 1 / rms.  The
// partners' g are where turn left them.
template <typename T, bool HALVES>
__device__ __forceinline__ void add_slopes(const Args& a, const Seat<T, HALVES>& at, const double2* turns, const Shared<T, true>& s,
                                           const float (&g)[kC<T>], const float (&x)[kC<T>], double r, const float* wt,
                                           double (&sum)[kC<T>])
{
#pragma unroll
    for (int i = 0; i < kC<T>; ++i) {
        const int c = at.c0 + i;
        if (c >= 2 * a.pairs) continue;
        const double2 z = HALVES ? turns[at.partner[HALVES ? i : 0] >> 19] : turns[c / 2];
        const double other = HALVES ? *(const float*)((const char*)s.row + (at.partner[HALVES ? i : 0] & 0xffff)) : g[i ^ 1];
        const bool second = HALVES ? c >= a.pairs : i & 1;
        const double theirs = fma(other, z.x, second ? g[i] * z.y : -(g[i] * z.y));
        sum[i] = fma((double)x[i] * r * (double)wt[i], second ? -theirs : theirs, sum[i]);
    }
}

template <typename T>
__device__ __forceinline__ double inverse_rms64(const Args& a, const float (&x)[kC<T>])
{
    double ss = 0;
    for (int i = 0; i < kC<T>; ++i) ss = fma((double)x[i], (double)x[i], ss);
    return 1.0 / sqrt(sum_lanes(ss, a.per) / a.dim + (double)a.eps);
}
template <typename T>
__device__ __forceinline__ float inverse_rms(const Args& a, const float (&x)[kC<T>])
{
    float ss = 0;
    for (int i = 0; i < kC<T>; ++i) ss = fmaf(x[i], x[i], ss);
    return __builtin_amdgcn_rsqf(fmaf(sum_lanes(ss, a.per), a.inv_dim, a.eps));
}

// Where a wave is: a step of an atom's heads, of the `sub`-th `count` atoms of its batch at `first`.
struct Cursor {
    int64_t first;
    int sub, step;
    __device__ __forceinline__ void next(const Args& a, int64_t stride)
    {
        if (++step < a.steps) return;
        step = 0;
        sub += a.count;
        if (sub < a.batch) return;
        sub = 0;
        first += stride;
    }
};

// A lane's part in a step: `at_once` heads of q, or of k after those.
struct Part {
    int64_t node;
    int head;
    bool is_q, live;
};
template <typename T, bool HALVES>
__device__ __forceinline__ Part part_of(const Args& a, const Seat<T, HALVES>& at, const Cursor& c)
{
    Part p;
    p.is_q = c.step < a.q_steps;
    p.head = (p.is_q ? c.step : c.step - a.q_steps) * a.at_once + at.slot;
    p.node = c.first + c.sub + at.t;
    p.live = at.c0 < a.dim && p.node < (p.is_q ? a.targets : a.nodes) && p.head < (p.is_q ? a.heads : a.kv);
    return p;
}

template <typename T, bool HALVES>
__global__ __launch_bounds__(64 * kWaves) void forward_kernel(Args a)
{
    __shared__ Shared<T, false> shared[kWaves];
    __shared__ __attribute__((aligned(16))) float s_w[2 * 256];
    constexpr int C = kC<T>;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Shared<T, false>& s = shared[w];
    load_weights<T>(a, s_w);
    const Seat<T, HALVES> at(a, lane);
    const int64_t stride = (int64_t)gridDim.x * kWaves * a.batch;
    int64_t first = ((int64_t)blockIdx.x * kWaves + w) * a.batch;
    if (first >= a.nodes) return;
    auto load = [&](const Part& p) {
        u32x4 r = {0, 0, 0, 0};
        if (p.live) r = *(const u32x4*)((const T*)(p.is_q ? a.q : a.k) + p.node * (p.is_q ? a.ldq : a.ldk) + p.head * a.dim + at.c0);
        return r;
    };
    Cursor cursor{first, 0, 0};
    Part next = part_of(a, at, cursor);
    u32x4 next_x = load(next);
    Angles angles = make_angles(a, lane, first);
    for (; first < a.nodes; first += stride) {
        make_turns(a, angles, first, first + stride, lane, s);
        while (cursor.first == first) {
            const float2* turns = s.turn + (cursor.sub + at.t) * a.pairs;
            const Part p = next;
            float x[C], y[C], unused[C];
            unpack<T>(next_x, x);
            cursor.next(a, stride);
            next = part_of(a, at, cursor);
            next_x = load(next);
            if (a.norm) {
                const float r = inverse_rms<T>(a, x);
                const float* wt = s_w + (p.is_q ? 0 : a.dim) + (at.c0 < a.dim ? at.c0 : 0);
                for (int i = 0; i < C; ++i) x[i] = x[i] * r * wt[i];
            }
            turn<T, HALVES, false>(a, at, turns, s, x, y, unused);
            if (p.live)
                *(u32x4*)((T*)(p.is_q ? a.oq : a.ok) + (p.node * (p.is_q ? a.heads : a.kv) + p.head) * a.dim + at.c0) = pack<T>(y);
        }
        wave_sync();
    }
}

// WIDE: the positions' gradient in 64 bits, that of positions which have them.
template <typename T, bool HALVES, bool WIDE>
__global__ __launch_bounds__(64 * kWaves) void backward_kernel(Args a)
{
    __shared__ Shared<T, WIDE> shared[kWaves];
    __shared__ __attribute__((aligned(16))) float s_w[2 * 256];
    __shared__ float s_sum[64 * kWaves * kC<T>];
    constexpr int C = kC<T>;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Shared<T, WIDE>& s = shared[w];
    load_weights<T>(a, s_w);
    const Seat<T, HALVES> at(a, lane);
    const int group = a.per * a.at_once;
    const int64_t stride = (int64_t)gridDim.x * kWaves * a.batch;
    int64_t first = ((int64_t)blockIdx.x * kWaves + w) * a.batch;
    auto load = [&](const Part& p, u32x4& x, u32x4& g) {
        x = g = u32x4{0, 0, 0, 0};
        if (p.live) {
            const int64_t in = p.head * a.dim + at.c0;
            x = *(const u32x4*)((const T*)(p.is_q ? a.q : a.k) + p.node * (p.is_q ? a.ldq : a.ldk) + in);
            g = *(const u32x4*)((const T*)(p.is_q ? a.gq : a.gk) + p.node * (p.is_q ? a.ldgq : a.ldgk) + in);
        }
    };
    // (the lane's channels' axes, four bits each)
    auto pair_of = [&](int i) {
        const int c = at.c0 + i;
        return c >= 2 * a.pairs ? 0 : HALVES ? (c < a.pairs ? c : c - a.pairs) : c / 2;
    };
    uint32_t axes = 0;
    for (int i = 0; i < C; ++i) axes |= (uint32_t)(at.c0 + i < 2 * a.pairs ? axis_of(a, pair_of(i)) : 15) << 4 * i;
    using F = typename std::conditional<WIDE, double, float>::type;
    float sum_q[C] = {}, sum_k[C] = {};
    F dtheta[C] = {};
    Cursor cursor{first, 0, 0};
    Part next = part_of(a, at, cursor);
    u32x4 next_x, next_g;
    load(next, next_x, next_g);
    Angles angles = make_angles(a, lane, first);
    for (; first < a.nodes; first += stride) {
        make_turns(a, angles, first, first + stride, lane, s);
        while (cursor.first == first) {
            const float2* turns = s.turn + (cursor.sub + at.t) * a.pairs;
            const bool last = cursor.step + 1 == a.steps;  // of the atoms' heads
            const Part p = next;
            float x[C], g[C], back[C], across[C];
            unpack<T>(next_x, x);
            unpack<T>(next_g, g);
            cursor.next(a, stride);
            next = part_of(a, at, cursor);
            load(next, next_x, next_g);
            turn<T, HALVES, true>(a, at, turns, s, g, back, across);
            // (a lane without a head adds nothing: an angle or a scale that is not finite would make a NaN of its zeros)
            const float* wt = s_w + (p.is_q ? 0 : a.dim) + (at.c0 < a.dim ? at.c0 : 0);
            if constexpr (WIDE) {
                const double r = a.norm ? inverse_rms64<T>(a, x) : 1.0;
                if (p.live) add_slopes<T, HALVES>(a, at, s.turn64 + (turns - s.turn), s, g, x, r, wt, dtheta);
                wave_sync();
            }
            float r = 1.0f;
            if (a.norm) {
                r = inverse_rms<T>(a, x);
                for (int i = 0; i < C; ++i) x[i] *= r;
            }
            if constexpr (!WIDE)
                if (a.dpos && p.live)
                    for (int i = 0; i < C; ++i) dtheta[i] = fmaf(x[i] * wt[i], across[i], dtheta[i]);
            if (a.norm) {
                if (a.part && p.live) {
                    if (p.is_q)
                        for (int i = 0; i < C; ++i) sum_q[i] = fmaf(back[i], x[i], sum_q[i]);
                    else
                        for (int i = 0; i < C; ++i) sum_k[i] = fmaf(back[i], x[i], sum_k[i]);
                }
                float dot = 0;
                for (int i = 0; i < C; ++i) {
                    back[i] *= wt[i];
                    dot = fmaf(back[i], x[i], dot);
                }
                dot = sum_lanes(dot, a.per) * a.inv_dim;
                for (int i = 0; i < C; ++i) back[i] = r * (back[i] - x[i] * dot);
            }
            if (p.live)
                *(u32x4*)((T*)(p.is_q ? a.oq : a.ok) + (p.node * (p.is_q ? a.heads : a.kv) + p.head) * a.dim + at.c0) = pack<T>(back);
            if (a.dpos && last) {
                for (int i = 0; i < C; ++i) dtheta[i] *= (F)a.freq[pair_of(i)];
                for (int axis = 0; axis < a.axes; ++axis) {
                    F sum = 0;
                    for (int i = 0; i < C; ++i) sum += (axes >> 4 * i & 15) == (uint32_t)axis ? dtheta[i] : (F)0;
                    sum = sum_lanes(sum, group);
                    if ((lane & (group - 1)) == 0 && p.node < a.nodes) ((F*)a.dpos)[p.node * a.axes + axis] = sum;
                }
                for (int i = 0; i < C; ++i) dtheta[i] = 0;
            }
        }
        wave_sync();
    }
    if (!a.part) return;
    // the workgroup's sums of each channel, in the lanes' order
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        for (int i = 0; i < C; ++i) s_sum[threadIdx.x * C + i] = which ? sum_k[i] : sum_q[i];
        __syncthreads();
        if ((int)threadIdx.x < a.dim) {
            const int c = threadIdx.x;
            float x = 0;
            for (int l = c / C; l < 64 * kWaves; l += a.per) x += s_sum[l * C + c % C];
            a.part[((int64_t)blockIdx.x * 2 + which) * a.dim + c] = x;
        }
    }
}

// dw: the workgroups' sums of 16 channels, 64 strands of them in turn.
template <typename T>
__global__ __launch_bounds__(1024) void join_kernel(const float* part, int blocks, int dim, void* dqw, void* dkw, int w_own)
{
    __shared__ float s[16][16];
    const int strand = threadIdx.x >> 4, which = blockIdx.y, c = blockIdx.x * 16 + (threadIdx.x & 15);
    float x = 0;
    if (c < dim)
#pragma unroll 8
        for (int b = strand; b < blocks; b += 64) x += part[((int64_t)b * 2 + which) * dim + c];
    x += __shfl_xor(x, 16, 64);
    x += __shfl_xor(x, 32, 64);
    if (threadIdx.x % 64 < 16) s[threadIdx.x >> 6][threadIdx.x & 15] = x;
    __syncthreads();
    void* out = which ? dkw : dqw;
    if (threadIdx.x >= 16 || c >= dim || !out) return;
    x = 0;
    for (int i = 0; i < 16; ++i) x += s[i][threadIdx.x];
    if (w_own) ((T*)out)[c] = (T)x;
    else ((float*)out)[c] = x;
}

// ---------------------------------------------------------------- host
dg_status check(const dg_rotate_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->dtype != DG_F32 && d->dtype != DG_BF16) return fail(DG_ERR_INVALID, "q and k must be float32 or bfloat16");
    if (d->weight_dtype != DG_F32 && d->weight_dtype != d->dtype)
        return fail(DG_ERR_INVALID, "the weights must be float32 or of q's type");
    if (d->pos_dtype != DG_F32 && d->pos_dtype != DG_F64 && d->pos_dtype != DG_I64)
        return fail(DG_ERR_INVALID, "positions must be float32, float64 or int64");
    if (d->n_nodes < 0 || d->n_nodes > (1ll << 40) || d->n_targets < 0 || d->n_targets > d->n_nodes)
        return fail(DG_ERR_INVALID, "nodes must be in [0, 2^40] and targets among them");
    if (d->heads < 1 || d->heads > 1024 || d->kv_heads < 1 || d->kv_heads > 1024)
        return fail(DG_ERR_INVALID, "heads must be in [1, 1024]");
    if (d->dim < 8 || d->dim > 256 || d->dim % 8) return fail(DG_ERR_INVALID, "dim must be a multiple of 8 in [8, 256]");
    if (d->axes < 1 || d->axes > kMaxAxes) return fail(DG_ERR_INVALID, "axes must be in [1, 8]");
    int64_t pairs = 0;
    for (int i = 0; i < d->axes; ++i) {
        if (d->sections[i] < 0) return fail(DG_ERR_INVALID, "sections must not be negative");
        pairs += d->sections[i];
    }
    if (pairs < 1 || pairs > d->dim / 2) return fail(DG_ERR_INVALID, "sections must add up to 1 to dim / 2 pairs");
    if (d->norm && !(d->eps >= 0.0f && d->eps <= 3e38f)) return fail(DG_ERR_INVALID, "eps must be finite and not negative");
    const int64_t most = 1ll << 40;
    for (int64_t ld : {d->ld_q, d->ld_k, d->ld_gq, d->ld_gk}) {
        if (ld < 0 || ld > most || ld % (d->dtype == DG_F32 ? 4 : 8))
            return fail(DG_ERR_INVALID, "rows must lie a multiple of 16 bytes apart");
        if (d->n_nodes > 0 && ld > (1ll << 60) / d->n_nodes) return fail(DG_ERR_INVALID, "rows reach past 2^60 elements");
    }
    return DG_OK;
}

// Heads of an atom at once: as many as there are lanes for, but fewer where that leaves lanes without a head
// (16 and 4 heads on 8 places: a sixth of them) and there are atoms for them instead.
int heads_at_once(const dg_rotate_desc* d, int most)
{
    auto places = [&](int n) { return ((d->heads + n - 1) / n + (d->kv_heads + n - 1) / n) * n; };
    most = std::min(most, power_of_two(std::max(d->heads, d->kv_heads)));
    int best = most;
    if (d->n_nodes >= kMaxBlocks * kWaves * 4)
        for (int n = most / 2; n >= 1; n /= 2)
            if (places(n) < places(best)) best = n;
    return best;
}

Args make_args(const dg_rotate_desc* d)
{
    Args a = {};
    a.targets = d->n_targets;
    a.nodes = d->n_nodes;
    a.ldq = d->ld_q;
    a.ldk = d->ld_k;
    a.ldgq = d->ld_gq;
    a.ldgk = d->ld_gk;
    a.heads = d->heads;
    a.kv = d->kv_heads;
    a.dim = d->dim;
    a.inv_dim = 1.0f / (float)d->dim;
    a.axes = d->axes;
    a.pos_dtype = d->pos_dtype;
    a.norm = d->norm != 0;
    a.w_own = d->weight_dtype == d->dtype && d->dtype != DG_F32;
    a.eps = d->eps;
    for (int i = 0; i < d->axes; ++i) {
        a.pairs += d->sections[i];
        a.ends[i] = a.pairs;
    }
    const int c = d->dtype == DG_F32 ? 4 : 8;
    a.per = power_of_two(d->dim / c);
    a.at_once = heads_at_once(d, 64 / a.per);
    a.count = 64 / (a.per * a.at_once);
    a.batch = a.count * std::max(1, 64 / (a.count * a.pairs));
    // (few atoms: rather a wave for each step's)
    while (a.batch > a.count && a.nodes < (int64_t)a.batch * kWaves * kMaxBlocks) a.batch -= a.count;
    a.q_steps = (d->heads + a.at_once - 1) / a.at_once;
    a.steps = a.q_steps + (d->kv_heads + a.at_once - 1) / a.at_once;
    return a;
}

// Workgroups: as many as are resident, a wave then takes its atoms batch after batch.
int64_t blocks_of(const Args& a, int most)
{
    const int64_t pass = (int64_t)kWaves * a.batch;
    return std::max<int64_t>(1, std::min<int64_t>((a.nodes + pass - 1) / pass, most));
}

bool misaligned(std::initializer_list<const void*> p)
{
    for (const void* x : p)
        if ((uintptr_t)x & 15) return true;
    return false;
}

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

template <typename T>
void run_forward(const Args& a, bool interleaved, hipStream_t s)
{
    const dim3 grid((unsigned)blocks_of(a, kForwardBlocks));
    if (interleaved) hipLaunchKernelGGL((forward_kernel<T, false>), grid, dim3(64 * kWaves), 0, s, a);
    else hipLaunchKernelGGL((forward_kernel<T, true>), grid, dim3(64 * kWaves), 0, s, a);
}

template <typename T>
void run_backward(const Args& a, bool interleaved, void* dqw, void* dkw, hipStream_t s)
{
    const bool wide = a.dpos && a.pos_dtype == DG_F64;
    const int64_t blocks = a.nodes ? blocks_of(a, backward_blocks(sizeof(T) == 2 ? DG_BF16 : DG_F32, wide)) : 0;
    if (blocks) {
        const dim3 grid((unsigned)blocks);
        if (interleaved && wide) hipLaunchKernelGGL((backward_kernel<T, false, true>), grid, dim3(64 * kWaves), 0, s, a);
        else if (interleaved) hipLaunchKernelGGL((backward_kernel<T, false, false>), grid, dim3(64 * kWaves), 0, s, a);
        else if (wide) hipLaunchKernelGGL((backward_kernel<T, true, true>), grid, dim3(64 * kWaves), 0, s, a);
        else hipLaunchKernelGGL((backward_kernel<T, true, false>), grid, dim3(64 * kWaves), 0, s, a);
    }
    if (a.part)
        hipLaunchKernelGGL(join_kernel<T>, dim3((a.dim + 15) / 16, 2), dim3(1024), 0, s, a.part, (int)blocks, a.dim, dqw, dkw,
                           a.w_own);
}

}  // namespace

extern "C" {

dg_status dg_rotate_forward(const dg_rotate_desc* d, const void* q, const void* k, const void* positions,
                            const float* frequencies, const void* q_weight, const void* k_weight, void* q_out, void* k_out,
                            hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_nodes == 0) return DG_OK;
    if ((d->n_targets > 0 && (!q || !q_out)) || !k || !positions || !frequencies || !k_out)
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    if (misaligned({q, k, q_out, k_out})) return fail(DG_ERR_INVALID, "q, k and the results must be aligned to 16 bytes");
    if (!d->norm && (q_weight || k_weight)) return fail(DG_ERR_INVALID, "weights come with norm");
    Args a = make_args(d);
    a.q = q;
    a.k = k;
    a.pos = positions;
    a.freq = frequencies;
    a.qw = q_weight;
    a.kw = k_weight;
    a.oq = q_out;
    a.ok = k_out;
    if (d->dtype == DG_BF16) run_forward<__bf16>(a, d->interleaved != 0, s);
    else run_forward<float>(a, d->interleaved != 0, s);
    return launched("dg_rotate_forward");
}

size_t dg_rotate_workspace_size(const dg_rotate_desc* d)
{
    if (check(d) != DG_OK) return 0;
    const Args a = make_args(d);
    return (size_t)blocks_of(a, backward_blocks(d->dtype, false)) * 2 * a.dim * sizeof(float);  // (wide: no more)
}

dg_status dg_rotate_backward(const dg_rotate_desc* d, const void* q, const void* k, const void* positions,
                             const float* frequencies, const void* q_weight, const void* k_weight, const void* grad_q,
                             const void* grad_k, void* dq, void* dk, void* dpositions, void* dq_weight, void* dk_weight,
                             void* ws, size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_nodes > 0 && ((d->n_targets > 0 && (!q || !grad_q || !dq)) || !k || !positions || !frequencies || !grad_k || !dk))
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    if (misaligned({q, k, grad_q, grad_k, dq, dk}))
        return fail(DG_ERR_INVALID, "q, k, their gradients and the results must be aligned to 16 bytes");
    if (!d->norm && (q_weight || k_weight || dq_weight || dk_weight)) return fail(DG_ERR_INVALID, "weights come with norm");
    if ((dq_weight && !q_weight) || (dk_weight && !k_weight)) return fail(DG_ERR_INVALID, "a weight's gradient comes with it");
    if (dpositions && d->pos_dtype == DG_I64) return fail(DG_ERR_INVALID, "whole positions have no gradient");
    Args a = make_args(d);
    a.q = q;
    a.k = k;
    a.pos = positions;
    a.freq = frequencies;
    a.qw = q_weight;
    a.kw = k_weight;
    a.gq = grad_q;
    a.gk = grad_k;
    a.oq = dq;
    a.ok = dk;
    a.dpos = dpositions;
    if (dq_weight || dk_weight) {
        if (!ws || ws_bytes < dg_rotate_workspace_size(d)) return fail(DG_ERR_WORKSPACE, "workspace too small");
        a.part = (float*)ws;
    }
    if (d->dtype == DG_BF16) run_backward<__bf16>(a, d->interleaved != 0, dq_weight, dk_weight, s);
    else run_backward<float>(a, d->interleaved != 0, dq_weight, dk_weight, s);
    return launched("dg_rotate_backward");
}

}  // extern "C"
