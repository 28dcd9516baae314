// dg_route.hip -- rows routed to experts: each row's choices, their weights, their gradient.
//
//   s = softmax(x) or 1 / (1 + exp(-x)) of a row's logits x, one an expert
//   v = x (no bias), or s + bias: what is chosen by.  A logit or a bias of -inf is never chosen
//   groups: neighbouring experts; a group's worth is its largest v, or the sum of its two largest s (+ bias);
//           only the experts of the top_groups worthiest are chosen from
//   experts[i] = the k largest v, NaN above all, ties to the lowest index;  -1 where none is left
//   weights[i, j] = scale s[chosen] (/ sum over the chosen s)
//   sizes[e] = rows that chose e;  places[i, j] = place of the choice in the order by expert, then row
//   dx[j] = scale u_j (g_j - sum g u) (1 - s_j: sigmoid) for renormalised weights u, else
//   dx[j] = scale p_j (g_j [chosen] - sum_chosen g p) (softmax), scale g_j s_j (1 - s_j) (sigmoid)
//
// A power of two of lanes, W, holds a row, V neighbouring experts each; k rounds take the largest left
// out, each a maximum over the lanes and a ballot for its first holder.  Sums of scores are compared as 64
// bits have them, so that what a rounding of 32 would merge or swap is chosen as the definition has it.
// The places are a stable counting sort in three launches: each workgroup's counts of its rows' choices, a
// scan of them for each expert, and the ranks within a workgroup by matching lanes; nothing depends
// on the order of atomics (counts alone are added up by them).
//
// Instructions bound it, not the bytes: 300,007 rows over 64 experts in 8 groups, 6 chosen with a bias, in float: 60 us
// for the choices and 18 for the rows done again (98 MB: 19 us at a copy's rate), scan and places 5 and 11.  32,000
// rows over 128 experts, 8 chosen, in bfloat16 (8 MB): 14, 5 and 4 us, backward 9: rounds of maxima over 16
// lanes, one after the other, and launches.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "../../include/dynamis_graph.h"
#include "dg_grid.hpp"
#include "dg_lanes.hpp"

namespace dg {
dg_status fail(dg_status st, const std::string& msg);  // dg_graph.hip
}

namespace {

using namespace dg;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 64;
constexpr int kBlockRows = 256;  // of a workgroup, at most

struct Args {
    const void* logits;
    const float* bias;
    float* weights;
    int32_t* experts;
    int64_t* sizes;
    int32_t* places;
    uint32_t* counts;  // [experts + 1][blocks]: of each workgroup's rows, the last of choices of none
    uint32_t* totals;  // [experts + 1]
    uint32_t* close;   // [blocks][kBlockRows / 32]: rows that are done in 64 bits
    int64_t rows, ld;
    int n, k, groups, top_groups, group_best;
    int sigmoid, renormalize;
    float scale;
    int lanes;        // W
    int group_lanes;  // of a group, where a power of two of lanes hold it whole (else 0)
    int64_t block_rows, blocks;
    const float* grad;
    void* dlogits;
};

__device__ __forceinline__ uint32_t max_lanes(uint32_t x, int n)
{
    over_lanes(n, [&](auto&& other) { x = max(x, other(x)); });
    return x;
}
__device__ __forceinline__ uint64_t max_lanes(uint64_t x, int n)
{
    over_lanes(n, [&](auto&& other) {
        const uint64_t y = (uint64_t)other((uint32_t)(x >> 32)) << 32 | other((uint32_t)x);
        x = max(x, y);
    });
    return x;
}
// Whole numbers in the order of the floating ones: 0 is nothing, NaN the largest; -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = as_bits(x + 0.0f);
    if (x != x) return 0xffffffffu;
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    if (x != x) return ~0ull;
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}

__device__ __forceinline__ float number_of(uint32_t key) { return as_float(key >> 31 ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ double number_of(uint64_t key)
{
    return __builtin_bit_cast(double, key >> 63 ? key ^ 0x8000000000000000ull : ~key);
}

template <typename T>
__device__ __forceinline__ float logit(const Args& a, int64_t row, int e)
{
    return (float)((const T*)a.logits)[row * a.ld + e];
}

// V neighbouring logits of a lane; experts past the last are -inf.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const Args& a, int64_t row, int e0, bool live, float (&x)[V])
{
    const T* p = (const T*)a.logits + row * a.ld + e0;
    if (live && e0 + V <= a.n) {  // (in one load of the element's alignment: gfx950 reads any)
        struct __attribute__((packed, aligned(2))) U { T v[V]; } u = *(const U*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float)u.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = live && e0 + i < a.n ? (float)p[i] : -INFINITY;
    }
}

// A row's choices: k rounds of the largest key, first holder first, into `picks` (-1: none left) with what
// the key's low half stands for (where keys have 32 bits, the value).
struct Pick {
    int e;
    float x;
};
template <int V, typename K>
__device__ __forceinline__ void choose(const Args& a, K (&key)[V], int lane, int e0, uint64_t of_row, Pick* picks)
{
    for (int j = 0; j < a.k; ++j) {
        K best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        const K top = max_lanes(best, a.lanes);
        const uint64_t holders = __ballot(best == top) & of_row;
        if (lane == __builtin_ctzll(holders)) {
            int at = V - 1;
#pragma unroll
            for (int i = V - 2; i >= 0; --i) at = key[i] == top ? i : at;
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = i == at ? 0 : key[i];
            picks[j] = Pick{top ? e0 + at : -1, number_of((uint32_t)top)};
        }
    }
}

// Keys whose low bits may go hold their place among the lane's in them (the first the largest), in falling order:
// then a round looks at each lane's first alone, and the winner's others move up.  The low bits may go where they say
// nothing (a bfloat16's), or no more than `apart` allows for.  (300,007 rows over 64 experts, 8 a lane, 6 rounds: 60
// us; when it came, 64, and 70 where each round looked through all.)
template <int V>
__device__ __forceinline__ void sort_packed(uint32_t (&key)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = key[i] ? (key[i] & ~(uint32_t)(V - 1)) | (uint32_t)(V - 1 - i) : 0;
    // (merges of odd and even places, with the larger first)
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = key[i + j], b = key[i + j + k];
                        key[i + j] = max(a, b);
                        key[i + j + k] = min(a, b);
                    }
}
// Returns, with LEFT, the largest key left.
template <int V, bool LEFT>
__device__ __forceinline__ uint32_t choose_packed(const Args& a, uint32_t (&key)[V], int lane, int e0, uint64_t of_row, Pick* picks)
{
    constexpr uint32_t kPlace = V - 1;
    for (int j = 0;; ++j) {
        if (!LEFT && j == a.k) return 0;
        // (between lanes their order decides equals, not the places in them)
        const uint32_t mine = key[0] & ~kPlace, top = max_lanes(mine, a.lanes);
        if (LEFT && j == a.k) return top;
        const uint64_t holders = __ballot(mine == top) & of_row;
        if (lane == __builtin_ctzll(holders)) {
            // (below zero a key's bits are turned: those that were given up are ones)
            picks[j] = Pick{top ? e0 + V - 1 - (int)(key[0] & kPlace) : -1, number_of(top >> 31 ? top : top | kPlace)};
#pragma unroll
            for (int i = 0; i + 1 < V; ++i) key[i] = key[i + 1];
            key[V - 1] = 0;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void choose_logits(const Args& a, uint32_t (&key)[V], int lane, int e0, uint64_t of_row, Pick* picks)
{
    if constexpr (sizeof(T) == 2) {
        sort_packed<V>(key);
        choose_packed<V, false>(a, key, lane, e0, of_row, picks);
    } else {
        choose<V>(a, key, lane, e0, of_row, picks);
    }
}

// Whether a lane's experts are in one of the worthiest groups, for groups of whole lanes (a.group_lanes, a power of two, to a group).
template <int V>
__device__ __forceinline__ bool mine_is_worthy(const Args& a, const uint32_t (&key)[V], int lane, int e0, uint32_t* s_worth)
{
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) best = max(best, key[i]);
    best = max_lanes(best, a.group_lanes);
    const int own = (lane & (a.lanes - 1)) / a.group_lanes;
    if (e0 < a.n) s_worth[own] = best;
    wave_sync();
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
        const uint32_t x = s_worth[g];
        rank += x > best || (x == best && g < own);
    }
    wave_sync();
    return rank < a.top_groups;
}
// A group's worth in 32 bits, the sum of its two largest where there are two; past: whether it is no 32-bit number though
// the group has members (infinities lie nowhere apart, and 64 bits may tell two such sums from each other).
__device__ __forceinline__ float worth_of(const Args& a, float best, float second, bool& past)
{
    const float worth = a.group_best == 2 && second > -INFINITY ? best + second : best;
    past = best > -INFINITY && !(fabsf(worth) < INFINITY);
    return worth;
}
// By sums in 32 bits; near: whether another group's lies nearer than `apart`, or the group's is past 32 bits.
template <int V>
__device__ __forceinline__ bool mine_is_worthy(const Args& a, const float (&v)[V], int lane, int e0, float* s_worth, float apart,
                                               bool& near)
{
    float best = v[0], second = -INFINITY;
#pragma unroll
    for (int i = 1; i < V; ++i) {
        second = __builtin_amdgcn_fmed3f(best, second, v[i]);
        best = fmaxf(best, v[i]);
    }
    over_lanes(a.group_lanes, [&](auto&& other) {
        const float b = as_float(other(as_bits(best))), t = as_float(other(as_bits(second)));
        second = fmaxf(fminf(best, b), fmaxf(second, t));
        best = fmaxf(best, b);
    });
    bool past;
    const float worth = worth_of(a, best, second, past);
    if (e0 < a.n) s_worth[(lane & (a.lanes - 1)) / a.group_lanes] = worth;
    wave_sync();
    int rank = 0, around = 0;
    for (int g = 0; g < a.groups; ++g) {
        const float x = s_worth[g];
        rank += x > worth;
        around += fabsf(x - worth) <= apart;  // (its own among them)
    }
    wave_sync();
    near = past || around > 1;
    return rank < a.top_groups;
}

// Which groups of a row are the worthiest, as a mask, for groups of any size.  `worth`: the keys that a group's
// worth sums, 0 for what is never chosen.
template <int V, typename K>
__device__ __forceinline__ uint64_t worthiest(const Args& a, const K (&worth)[V], int lane, int e0, K* s_key, K* s_worth)
{
    const int l = lane & (a.lanes - 1), per = a.n / a.groups;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (e0 + i < a.n) s_key[e0 + i] = worth[i];
    wave_sync();
    K mine = 0;
    if (l < a.groups) {
        K best = 0, second = 0;
        for (int i = l * per; i < (l + 1) * per; ++i) {
            const K x = s_key[i];
            second = max(second, min(best, x));
            best = max(best, x);
        }
        mine = a.group_best == 2 && second ? key_of(number_of(best) + number_of(second)) : best;
        s_worth[l] = mine;
    }
    wave_sync();
    int rank = 0;
    if (l < a.groups)
        for (int g = 0; g < a.groups; ++g) {
            const K x = s_worth[g];
            rank += x > mine || (x == mine && g < l);
        }
    wave_sync();
    return __ballot(l < a.groups && mine && rank < a.top_groups) >> (lane & ~(a.lanes - 1));
}
// The same by sums in 32 bits; near: whether the lane's group and another lie nearer than `apart`, or its own is past them.
template <int V>
__device__ __forceinline__ uint64_t worthiest(const Args& a, const float (&v)[V], int lane, int e0, float* s_value, float* s_worth,
                                              float apart, bool& near)
{
    const int l = lane & (a.lanes - 1), per = a.n / a.groups;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (e0 + i < a.n) s_value[e0 + i] = v[i];
    wave_sync();
    float worth = -INFINITY;
    bool past = false;
    if (l < a.groups) {
        float best = -INFINITY, second = -INFINITY;
        for (int i = l * per; i < (l + 1) * per; ++i) {
            const float x = s_value[i];
            second = __builtin_amdgcn_fmed3f(best, second, x);
            best = fmaxf(best, x);
        }
        worth = worth_of(a, best, second, past);
        s_worth[l] = worth;
    }
    wave_sync();
    int rank = 0, around = 0;
    if (l < a.groups)
        for (int g = 0; g < a.groups; ++g) {
            const float x = s_worth[g];
            rank += x > worth;
            around += fabsf(x - worth) <= apart;  // (its own among them)
        }
    wave_sync();
    near = past || around > 1;
    return __ballot(l < a.groups && rank < a.top_groups) >> (lane & ~(a.lanes - 1));
}

// The groups of a lane's experts, a byte each.
template <int V>
struct Groups {
    uint32_t of[(V + 3) / 4] = {};
    __device__ __forceinline__ Groups(const Args& a, int e0)
    {
        const int per = a.n / a.groups;
        if (a.groups > 1)
            for (int i = 0; i < V; ++i) of[i / 4] |= (uint32_t)(min(e0 + i, a.n - 1) / per) << 8 * (i % 4);
    }
    template <typename K>
    __device__ __forceinline__ void keep(uint64_t groups, K (&key)[V]) const
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!(groups >> (of[i / 4] >> 8 * (i % 4) & 255) & 1)) key[i] = 0;
    }
};

// For what is chosen by: exp, from that of 2 (its argument's rounding is |x| 2^-24 of it, and beneath 2^-126 it is 0),
// and the sigmoid from exp(-|x|), which overflows nowhere.  A row whose choice hangs on either's error is done again.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(1.44269504f * x); }
__device__ __forceinline__ float sigmoid(float x)
{
    const float e = exp_of(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return x < 0.0f ? e * r : r;
}

// For what is returned: exp(x - y), the difference in two parts (exact together, so that a weight's digits do not go
// with its logit's distance from the largest), and the sigmoid, which is 0 where it is in 32 bits.
__device__ __forceinline__ float exp_between(float x, float y)
{
    const float d = x - y, b = d - x, e = expf(d);
    return d > -200.0f ? fmaf(e, (x - (d - b)) - (y + b), e) : e;
}
__device__ __forceinline__ float exact_sigmoid(float x)
{
    const float e = expf(-fabsf(x));
    return (x < 0.0f ? e : 1.0f) / (1.0f + e);
}
// A weight of logit c up to a factor that is the row's: 1 for the largest chosen, m, or above 1/2 (a sigmoid's, whose
// exponential is taken relative to the largest's: far below zero all of them would vanish).
__device__ __forceinline__ float share_of(const Args& a, float c, float m)
{
    return a.sigmoid ? exp_between(fminf(c, 0.0f), fminf(m, 0.0f)) / (1.0f + expf(-fabsf(c))) : exp_between(c, m);
}

// s of a row's logits, in 32 bits or 64.
template <int V, typename F>
__device__ __forceinline__ void scores(const Args& a, const float (&x)[V], float top, F (&s)[V])
{
    F sum = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(F) == 8) {
            s[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top);
        } else {
            s[i] = a.sigmoid ? sigmoid(x[i]) : exp_of(x[i] - top);
        }
        sum += s[i];
    }
    if (!a.sigmoid) {
        sum = sum_lanes(sum, a.lanes);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] /= sum;
    }
}

// kLogits: the logits are what is chosen by.  kScores: a bias, or groups worth a sum of scores.  What is chosen by
// is then worked out in 32 bits; a row where two values that a choice or a group hangs on lie nearer than the
// rounding, or are no numbers, is left to a second launch, kWide, which takes it in 64.  That is one of some hundred to
// thousand while the biases are small; what counts as near goes by the largest |bias| of all, so that one large entry
// sends more there.  300,007 rows over 64 experts in groups, biases of some 0.1: 60 and 18 us, a call 89; with one entry of
// -10 93, -100 101, -1e3 164, -1e4 (every row) 192 (a bias of -inf takes an expert out at no cost).  In one
// launch, where the wide part's registers leave the other three waves a SIMD, 92.  What bounds kScores is
// instructions, some thousand for a wave's eight rows; five waves a SIMD are worth the registers that spill (57 us, four 72).
enum { kLogits, kScores, kWide };

template <typename T, int V, int HOW>
__global__ __launch_bounds__(kThreads, HOW == kScores && V <= 8 ? 5 : 1) void route_kernel(Args a)
{
    constexpr bool SCORED = HOW != kLogits;
    using K = typename std::conditional<HOW == kWide, uint64_t, uint32_t>::type;
    __shared__ uint32_t s_close[kBlockRows / 32], s_rows;
    __shared__ uint8_t s_list[kBlockRows];
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint32_t* s_count = (uint32_t*)smem;  // [n + 1]
    const int lane = threadIdx.x & 63, in_block = threadIdx.x / a.lanes, at_once = kThreads / a.lanes;
    const int l = lane & (a.lanes - 1), e0 = l * V;
    Pick* s_picks = (Pick*)(s_count + ((a.n + 4) & ~3));
    Pick* picks = s_picks + in_block * a.k;
    // (with groups: a row's keys, and its groups' worths)
    K* s_key = (K*)(s_picks + ((at_once * a.k + 1) & ~1)) + in_block * a.n;
    K* s_worth = (K*)(s_picks + ((at_once * a.k + 1) & ~1)) + at_once * a.n + in_block * a.groups;
    const int64_t block = workgroup();
    if (block >= a.blocks) return;
    for (int i = threadIdx.x; i <= a.n; i += kThreads) s_count[i] = 0;
    if (threadIdx.x < kBlockRows / 32) s_close[threadIdx.x] = HOW == kWide ? a.close[block * (kBlockRows / 32) + threadIdx.x] : 0;
    if (threadIdx.x == 0) s_rows = 0;
    __syncthreads();
    const int64_t r0 = block * a.block_rows;
    int rows = (int)min(a.block_rows, a.rows - r0);
    if constexpr (HOW == kWide) {  // (in any order: each is by itself)
        if (threadIdx.x < kBlockRows && s_close[threadIdx.x / 32] >> threadIdx.x % 32 & 1) s_list[atomicAdd(&s_rows, 1u)] = threadIdx.x;
        __syncthreads();
        rows = (int)s_rows;
        if (!rows) return;
    }
    const uint64_t of_row = a.lanes == 64 ? ~0ull : ((1ull << a.lanes) - 1) << (lane & ~(a.lanes - 1));
    float bias[V];
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = SCORED && a.bias && e0 + i < a.n ? a.bias[e0 + i] : 0.0f;
    const Groups<V> groups(a, e0);
    uint32_t never = 0;  // the lane's experts that no row takes
    float most = 0.0f;   // of the biases
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool none = e0 + i >= a.n || bias[i] == -INFINITY;
        never |= (uint32_t)none << i;
        most = none ? most : fmaxf(most, fabsf(bias[i]));
    }
    over_lanes(a.lanes, [&](auto&& other) { most = fmaxf(most, as_float(other(as_bits(most)))); });
    most += 1.0f;  // of a value
    // How near two values may lie before 32 bits do not tell them apart: a sigmoid is within 6 2^-24, a softmax, whose
    // sum has n terms, within 32 2^-24, their sum with the bias within another 2^-24 of itself; two values,
    // each of them a sum of two; and the packed places.
    const float apart = (a.sigmoid ? 2e-6f : 8e-6f) * (1.0f + most) + 2.4e-7f * V * most;
    for (int base = 0; base < rows; base += at_once) {
        const int at = base + in_block;
        bool live = at < rows;
        const int64_t row = r0 + (HOW == kWide ? (live ? s_list[at] : 0) : at);
        float x[V];
        load_logits<T, V>(a, row, e0, live, x);
        // the row's maximum and sum, where a weight or a choice needs them
        float top = -INFINITY, total = 1.0f;
        const bool softmax_all = !a.sigmoid && (SCORED || !a.renormalize);
        if (softmax_all) {
#pragma unroll
            for (int i = 0; i < V; ++i) top = x[i] > top ? x[i] : top;  // (a NaN makes the sum one)
            over_lanes(a.lanes, [&](auto&& other) { top = fmaxf(top, as_float(other(as_bits(top)))); });
            if (top == -INFINITY) top = 0.0f;
        }
        if (!a.sigmoid && !a.renormalize) {
            float sum = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += exp_of(x[i] - top);
            total = sum_lanes(sum, a.lanes);
        }
        // (a row's keys: of its logits, where those are chosen by)
        uint32_t plain[V];
        auto gone = [&](int i) { return x[i] == -INFINITY || (never >> i & 1); };
        if (HOW != kScores || !a.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i) plain[i] = gone(i) ? 0 : key_of(x[i]);
        }
        bool poisoned = false;  // a softmax with a NaN or an infinity: every weight is one, whichever are chosen
        if constexpr (HOW == kScores) {
            float v[V], all = 0.0f;
            uint32_t key[V];
            scores<V>(a, x, top, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = gone(i) ? -INFINITY : v[i] + bias[i];
                all += v[i];
                key[i] = a.bias ? (gone(i) ? 0 : key_of(v[i])) : plain[i];
            }
            bool close = all != all;  // (a NaN, or infinities of both signs)
            if (a.groups > 1) {
                bool near;
                if (a.group_lanes) {
                    const bool worthy = mine_is_worthy<V>(a, v, lane, e0, (float*)s_worth, apart, near);
#pragma unroll
                    for (int i = 0; i < V; ++i) key[i] = worthy ? key[i] : 0;
                } else {
                    groups.keep(worthiest<V>(a, v, lane, e0, (float*)s_key, (float*)s_worth, apart, near), key);
                }
                close = close || near;
            }
            if (a.bias) {
                sort_packed<V>(key);
                const uint32_t left = choose_packed<V, true>(a, key, lane, e0, of_row, picks);
                wave_sync();
                if (l < a.k && picks[l].e >= 0) {  // (a value and the next one; none: no matter)
                    const bool last = l + 1 == a.k, none = last ? !left : picks[l + 1].e < 0;
                    const float next = last ? number_of(left) : picks[l + 1].x;
                    close = close || (!none && !(picks[l].x - next > apart));
                }
            } else {  // (the keys are the logits, and exact)
                choose_logits<T, V>(a, key, lane, e0, of_row, picks);
            }
            if (__ballot(live && close) & of_row) {
                live = false;
                if (l == 0) atomicOr(&s_close[at / 32], 1u << at % 32);
            }
        } else if constexpr (HOW == kWide) {
            double d[V];
            scores<V>(a, x, top, d);
            K key[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                key[i] = plain[i] ? key_of(d[i] + (double)bias[i]) : 0;
                poisoned = poisoned || (!a.sigmoid && d[i] != d[i]);
            }
            poisoned = __ballot(poisoned) & of_row;
            const uint64_t kept = a.groups > 1 ? worthiest<V>(a, key, lane, e0, s_key, s_worth) : ~0ull;
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = a.bias ? key[i] : plain[i];
            if (a.groups > 1) groups.keep(kept, key);
            choose<V>(a, key, lane, e0, of_row, picks);
        } else {
            if (a.groups > 1 && a.group_lanes) {
                const bool worthy = mine_is_worthy<V>(a, plain, lane, e0, s_worth);
#pragma unroll
                for (int i = 0; i < V; ++i) plain[i] = worthy ? plain[i] : 0;
            } else if (a.groups > 1) {
                groups.keep(worthiest<V>(a, plain, lane, e0, s_key, s_worth), plain);
            }
            choose_logits<T, V>(a, plain, lane, e0, of_row, picks);
        }
        wave_sync();
        // a lane for each choice
        const bool mine = live && l < a.k;
        const Pick pick = l < a.k ? picks[l] : Pick{-1, 0.0f};
        const int e = pick.e;
        const float c = !mine || e < 0 ? -INFINITY : SCORED && a.bias ? logit<T>(a, row, e) : pick.x;
        float w = 0.0f;
        if (a.renormalize) {
            // (relative to the largest chosen: a sum that vanishes in 32 bits has no ratio)
            float m = c;
            over_lanes(a.lanes, [&](auto&& other) {
                const float y = as_float(other(as_bits(m)));
                m = y > m || y != y ? y : m;
            });
            if (e >= 0) w = share_of(a, c, m);
            const float sum = sum_lanes(w, a.lanes);
            if (e >= 0) w = w / sum;
        } else if (e >= 0) {
            w = a.sigmoid ? exact_sigmoid(c) : exp_between(c, top) / total;
        }
        if (mine) {
            a.experts[row * a.k + l] = e;
            a.weights[row * a.k + l] = poisoned && e >= 0 ? NAN : w * a.scale;
            atomicAdd(&s_count[e < 0 ? a.n : e], 1u);
        }
        wave_sync();
    }
    __syncthreads();
    if (HOW == kScores && threadIdx.x < kBlockRows / 32) a.close[block * (kBlockRows / 32) + threadIdx.x] = s_close[threadIdx.x];
    for (int i = threadIdx.x; i <= a.n; i += kThreads) {
        uint32_t* c = a.counts + i * a.blocks + block;
        *c = HOW == kWide ? *c + s_count[i] : s_count[i];
    }
}

// The counts of an expert become those of the workgroups before; a workgroup for each.
__global__ __launch_bounds__(1024) void scan_kernel(Args a)
{
    __shared__ uint32_t s_wave[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = blockIdx.x;
    uint32_t* c = a.counts + e * a.blocks;
    uint32_t before = 0;
    for (int64_t i0 = 0; i0 < a.blocks; i0 += 1024) {
        const int64_t i = i0 + threadIdx.x;
        const uint32_t x = i < a.blocks ? c[i] : 0;
        uint32_t in = x;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(in, o, 64);
            if (lane >= o) in += y;
        }
        if (lane == 63) s_wave[w] = in;
        __syncthreads();
        uint32_t all = 0, mine = before + in - x;
        for (int j = 0; j < 16; ++j) {
            if (j < w) mine += s_wave[j];
            all += s_wave[j];
        }
        if (i < a.blocks) c[i] = mine;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        a.totals[e] = before;
        if (e < a.n) a.sizes[e] = before;
    }
}

// The places of a workgroup's choices: where its experts' choices begin, and a rank within the
// workgroup in the choices' order (a quarter of them to a wave).  SUMS: adds up the counts itself, which
// saves the scan's launch (864 rows: 22.6 to 18.7 us a call) but has each workgroup read them all.
constexpr int kFewBlocks = 32;
template <bool SUMS>
__global__ __launch_bounds__(kThreads) void place_kernel(Args a)
{
    __shared__ uint32_t s_at[kWaves][kMaxExperts + 1];
    __shared__ uint32_t s_wave[kWaves];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t block = workgroup();
    if (block >= a.blocks) return;
    for (int i = threadIdx.x; i < kWaves * (a.n + 1); i += kThreads) s_at[i / (a.n + 1)][i % (a.n + 1)] = 0;
    __syncthreads();
    const int64_t first = block * a.block_rows * a.k, last = min((block + 1) * a.block_rows, a.rows) * a.k;
    const int64_t share = ((last - first + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int64_t from = min(first + w * share, last), to = min(from + share, last);
    for (int64_t i = from + lane; i < to; i += 64) {
        const int e = a.experts[i];
        atomicAdd(&s_at[w][e < 0 ? a.n : e], 1u);
    }
    __syncthreads();
    // each wave's first place of each expert
    uint32_t before = 0;
    for (int e0 = 0; e0 <= a.n; e0 += kThreads) {
        const int e = e0 + threadIdx.x;
        uint32_t x = 0, earlier = 0;
        if (e <= a.n) {
            if constexpr (SUMS) {
#pragma unroll 8
                for (int b = 0; b < a.blocks; ++b) {
                    const uint32_t n = a.counts[e * a.blocks + b];
                    x += n;
                    earlier += b < block ? n : 0;
                }
                if (block == 0 && e < a.n) a.sizes[e] = x;
            } else {
                x = a.totals[e];
                earlier = a.counts[e * a.blocks + block];
            }
        }
        uint32_t in = x;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(in, o, 64);
            if (lane >= o) in += y;
        }
        if (lane == 63) s_wave[w] = in;
        __syncthreads();
        uint32_t at = before + in - x;
        for (int j = 0; j < kWaves; ++j) {
            if (j < w) at += s_wave[j];
            before += s_wave[j];
        }
        if (e <= a.n) {
            at += earlier;
            for (int j = 0; j < kWaves; ++j) {
                const uint32_t n = s_at[j][e];
                s_at[j][e] = at;
                at += n;
            }
        }
        __syncthreads();
    }
    int bits = 1;
    while (a.n >> bits) ++bits;
    for (int64_t i0 = from; i0 < to; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool mine = i < to;
        const int e = mine ? a.experts[i] : 0, bin = e < 0 ? a.n : e;
        uint64_t same = __ballot(mine);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(bin >> b & 1);
            same &= bin >> b & 1 ? set : ~set;
        }
        const uint64_t below = same & ((1ull << lane) - 1);
        uint32_t at = 0;
        if (mine) at = s_at[w][bin];
        wave_sync();
        if (mine && !below) s_at[w][bin] = at + __popcll(same);
        if (mine) {
            const int32_t p = (int32_t)(at + __popcll(below));
            a.places[i] = e < 0 ? -1 - p : p;
        }
        wave_sync();
    }
}

// The logits' gradient: a row's choices' terms through LDS into the whole row.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void backward_kernel(Args a)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, in_block = threadIdx.x / a.lanes, at_once = kThreads / a.lanes;
    const int l = lane & (a.lanes - 1), e0 = l * V;
    float* s_row = (float*)smem + in_block * a.lanes * V;
    const int64_t row = workgroup() * at_once + in_block;
    const bool live = row < a.rows;
    const bool softmax_all = !a.sigmoid && !a.renormalize;
    float x[V], top = -INFINITY, total = 1.0f;
    if (softmax_all) {
        load_logits<T, V>(a, row, e0, live, x);
#pragma unroll
        for (int i = 0; i < V; ++i) top = x[i] > top ? x[i] : top;
        over_lanes(a.lanes, [&](auto&& other) { top = fmaxf(top, as_float(other(as_bits(top)))); });
        if (top == -INFINITY) top = 0.0f;
        float sum = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum += exp_of(x[i] - top);  // (as the forward pass has it)
            x[i] = expf(x[i] - top);
        }
        total = sum_lanes(sum, a.lanes);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_row[e0 + i] = 0.0f;
    wave_sync();
    const int e = live && l < a.k ? a.experts[row * a.k + l] : -1;
    const bool taken = e >= 0 && e < a.n;
    const float c = taken ? logit<T>(a, row, e) : -INFINITY, g = taken ? a.grad[row * a.k + l] * a.scale : 0.0f;
    float d = 0.0f, dot = 0.0f;
    if (a.renormalize) {
        float m = c;
        over_lanes(a.lanes, [&](auto&& other) {
            const float y = as_float(other(as_bits(m)));
            m = y > m || y != y ? y : m;
        });
        float u = 0.0f;
        if (taken) u = share_of(a, c, m);
        const float sum = sum_lanes(u, a.lanes);
        if (taken) u = u / sum;
        dot = sum_lanes(u * g, a.lanes);
        d = u * (g - dot);
        if (a.sigmoid) d = d * exact_sigmoid(-c);  // 1 - s
    } else if (a.sigmoid) {
        // s (1 - s), from the smaller of the two sides' exponentials
        const float z = expf(-fabsf(c));
        d = g * z / ((1.0f + z) * (1.0f + z));
    } else {
        d = taken ? g * (exp_between(c, top) / total) : 0.0f;
        dot = sum_lanes(d, a.lanes);
    }
    if (taken) s_row[e] = d;
    wave_sync();
    if (!live) return;
    T* out = (T*)a.dlogits + row * a.n + e0;
    T y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float v = s_row[e0 + i];
        if (softmax_all && dot != 0.0f) v -= x[i] / total * dot;
        y[i] = (T)v;
    }
    if (e0 + V <= a.n) {
        struct __attribute__((packed, aligned(2))) U { T v[V]; } u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.v[i] = y[i];
        *(U*)out = u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i < a.n) out[i] = y[i];
    }
}

// ---------------------------------------------------------------- host
inline size_t al(size_t x) { return (x + 255) & ~(size_t)255; }

dg_status check(const dg_route_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->dtype != DG_F32 && d->dtype != DG_BF16) return fail(DG_ERR_INVALID, "logits must be float32 or bfloat16");
    if (d->n_experts < 1 || d->n_experts > kMaxExperts) return fail(DG_ERR_INVALID, "experts must be in [1, 1024]");
    if (d->k < 1 || d->k > kMaxChoices || d->k > d->n_experts)
        return fail(DG_ERR_INVALID, "k must be in [1, 64] and at most the experts");
    if (d->n_rows < 0 || d->n_rows > 0x7fffffffll / d->k) return fail(DG_ERR_INVALID, "rows times k must be below 2^31");
    if (d->groups < 1 || d->groups > 64 || d->n_experts % d->groups)
        return fail(DG_ERR_INVALID, "groups must be in [1, 64] and divide the experts");
    if (d->top_groups < 1 || d->top_groups > d->groups) return fail(DG_ERR_INVALID, "top_groups must be in [1, groups]");
    if (d->group_best != 1 && d->group_best != 2) return fail(DG_ERR_INVALID, "group_best must be 1 or 2");
    if (d->ld < 0 || d->ld > (1ll << 31)) return fail(DG_ERR_INVALID, "logits' rows must lie 0 to 2^31 elements apart");
    if (!(d->scale >= -3e38f && d->scale <= 3e38f)) return fail(DG_ERR_INVALID, "scale must be finite");
    return DG_OK;
}

// Lanes of a row and experts of a lane.
void share(const dg_route_desc* d, int* lanes, int* each)
{
    *lanes = std::min(64, std::max({power_of_two((d->n_experts + 7) / 8), power_of_two(d->k), power_of_two(d->groups)}));
    *each = power_of_two((d->n_experts + *lanes - 1) / *lanes);
}

// Rows of a workgroup.
int64_t rows_of_block(const dg_route_desc* d)
{
    int64_t n = 32;
    while (n < kBlockRows && n * 2048 < d->n_rows) n *= 2;
    return n;
}

struct Layout {
    int64_t blocks;
    size_t o_totals, o_close, total;
};
Layout layout(const dg_route_desc* d)
{
    Layout L;
    L.blocks = (d->n_rows + rows_of_block(d) - 1) / rows_of_block(d);
    L.o_totals = al(4 * (size_t)(L.blocks * (d->n_experts + 1)));
    L.o_close = L.o_totals + al(4 * (size_t)(d->n_experts + 1));
    L.total = L.o_close + al((size_t)L.blocks * (kBlockRows / 8));
    return L;
}

Args make_args(const dg_route_desc* d, int* each)
{
    Args a = {};
    a.rows = d->n_rows;
    a.ld = d->ld;
    a.n = d->n_experts;
    a.k = d->k;
    a.groups = d->groups;
    a.top_groups = d->top_groups;
    a.group_best = d->group_best;
    a.sigmoid = d->sigmoid != 0;
    a.renormalize = d->renormalize != 0;
    a.scale = d->scale;
    share(d, &a.lanes, each);
    const int per = a.n / a.groups, whole = per / *each;
    a.group_lanes = per % *each == 0 && whole == power_of_two(whole) ? whole : 0;
    return a;
}

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

template <typename T, int V>
void run_route(const Args& a, hipStream_t s)
{
    const bool scored = a.bias || (a.groups > 1 && a.group_best == 2);
    const int at_once = kThreads / a.lanes;
    const size_t lds = 4 * (size_t)((a.n + 4) & ~3) + 8 * (size_t)((at_once * a.k + 1) & ~1);
    const size_t keys = a.groups > 1 ? (size_t)at_once * (a.n + a.groups) : 0;
    const dim3 grid = workgroups(a.blocks), block(kThreads);
    if (!scored) {
        hipLaunchKernelGGL((route_kernel<T, V, kLogits>), grid, block, lds + 4 * keys, s, a);
    } else {
        hipLaunchKernelGGL((route_kernel<T, V, kScores>), grid, block, lds + 4 * keys, s, a);
        hipLaunchKernelGGL((route_kernel<T, V, kWide>), grid, block, lds + 8 * keys, s, a);
    }
}

template <typename T>
void run_route(const Args& a, int each, hipStream_t s)
{
    switch (each) {
        case 1: return run_route<T, 1>(a, s);
        case 2: return run_route<T, 2>(a, s);
        case 4: return run_route<T, 4>(a, s);
        case 8: return run_route<T, 8>(a, s);
        default: return run_route<T, 16>(a, s);
    }
}

template <typename T>
void run_backward(const Args& a, int each, hipStream_t s)
{
    const int at_once = kThreads / a.lanes;
    const dim3 grid = workgroups((a.rows + at_once - 1) / at_once), block(kThreads);
    const size_t lds = 4 * (size_t)kThreads * each;
    switch (each) {
        case 1: hipLaunchKernelGGL((backward_kernel<T, 1>), grid, block, lds, s, a); break;
        case 2: hipLaunchKernelGGL((backward_kernel<T, 2>), grid, block, lds, s, a); break;
        case 4: hipLaunchKernelGGL((backward_kernel<T, 4>), grid, block, lds, s, a); break;
        case 8: hipLaunchKernelGGL((backward_kernel<T, 8>), grid, block, lds, s, a); break;
        default: hipLaunchKernelGGL((backward_kernel<T, 16>), grid, block, lds, s, a);
    }
}

}  // namespace

extern "C" {

size_t dg_route_workspace_size(const dg_route_desc* d)
{
    if (check(d) != DG_OK) return 0;
    return layout(d).total;
}

dg_status dg_route_forward(const dg_route_desc* d, const void* logits, const float* bias, float* weights, int32_t* experts,
                           int64_t* sizes, int32_t* places, void* ws, size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (!sizes || (d->n_rows > 0 && (!logits || !weights || !experts || !places)))
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    const Layout L = layout(d);
    if (!ws || ws_bytes < L.total) return fail(DG_ERR_WORKSPACE, "workspace too small");
    int each;
    Args a = make_args(d, &each);
    a.logits = logits;
    a.bias = bias;
    a.weights = weights;
    a.experts = experts;
    a.sizes = sizes;
    a.places = places;
    a.block_rows = rows_of_block(d);
    a.blocks = L.blocks;
    a.counts = (uint32_t*)ws;
    a.totals = (uint32_t*)((char*)ws + L.o_totals);
    a.close = (uint32_t*)((char*)ws + L.o_close);
    if (d->n_rows > 0) {
        if (d->dtype == DG_BF16) run_route<__bf16>(a, each, s);
        else run_route<float>(a, each, s);
    }
    if (a.blocks > 0 && a.blocks <= kFewBlocks) {
        hipLaunchKernelGGL(place_kernel<true>, dim3((unsigned)a.blocks), dim3(kThreads), 0, s, a);
        return launched("dg_route_forward");
    }
    hipLaunchKernelGGL(scan_kernel, dim3(a.n + 1), dim3(1024), 0, s, a);
    if (d->n_rows > 0) hipLaunchKernelGGL(place_kernel<false>, workgroups(a.blocks), dim3(kThreads), 0, s, a);
    return launched("dg_route_forward");
}

dg_status dg_route_backward(const dg_route_desc* d, const void* logits, const int32_t* experts, const float* grad_weights,
                            void* grad_logits, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_rows == 0) return DG_OK;
    if (!logits || !experts || !grad_weights || !grad_logits) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    int each;
    Args a = make_args(d, &each);
    a.logits = logits;
    a.experts = const_cast<int32_t*>(experts);
    a.grad = grad_weights;
    a.dlogits = grad_logits;
    if (d->dtype == DG_BF16) run_backward<__bf16>(a, each, s);
    else run_backward<float>(a, each, s);
    return launched("dg_route_backward");
}

}  // extern "C"
