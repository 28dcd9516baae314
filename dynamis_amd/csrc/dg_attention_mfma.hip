// dg_attention_mfma.hip -- attention over neighbour lists on the matrix units, bfloat16.
//
// A wave takes up to eight heads of a row, 32 edges a step.  The gathered rows of k are the
// matrix operand as they lie in memory: 16 edges by 32 channels, a lane holding 16 bytes of one
// edge.  The other operand is q spread out block-diagonally, 32 channels by 16 columns, column h
// holding head h's channels and zeros, so that the products over all channels of all heads add
// up in one accumulator of 16 edges by heads: no reduction across lanes, the logits of an edge
// sit in the registers of the softmax.  v enters the second product turned (channels by edges)
// by byte permutes of the loaded registers: a lane loads four channels of the eight edges whose
// probabilities it holds, so neither the probabilities nor v pass through LDS.
//
// Columns 8 .. 15 repeat the heads: the first eight carry the probability rounded to bfloat16,
// the others what the rounding left, also in bfloat16, and the two results are added at the
// row's end.  The weighted sum so has 16 bits of the probability at no further product; the
// forward pass adds a third part.
//
// The zeros of the block diagonal would spread a NaN or an infinity of one head of k over the
// others (0 * inf), and a weight's parts, some of them zero or negative, make a NaN of an infinity in
// v: a row whose sums are not finite is done again with products formed head by head, and with v's
// infinities taken apart from its numbers.
// Where the table holds entries of -inf, v of edges that these take out for all heads of the
// group is zeroed; a row that meets values that are not finite and hidden from some heads only
// is done again on the vector units.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/dynamis_graph.h"
#include "dg_attention.hpp"
#include "dg_attention_mfma.hpp"

#include <algorithm>
#include <type_traits>

namespace dg {
namespace {

// Heads that a wave takes together: at most eight (the columns of an operand, twice), with at
// most 128 channels of k between them.  (Groups of 256 channels need 256 registers and more, two
// waves a SIMD: 452 us against 226 us for two groups of 128, 2.9M edges of 8 heads of 32.)
struct HeadGroups {
    int heads, groups;
    int tiles;       // 64-channel tiles of the accumulators: 1 or 2
    uint32_t per_m;  // x / per = x per_m >> 20 for x < 1024 (per <= 1024), exact: off by less than x 2^-20
};

HeadGroups head_groups(int heads, int per, int dim)
{
    HeadGroups r{};
    for (int h = std::min(heads, 8); h >= 1; --h) {
        const int groups = (heads + h - 1) / h;
        int widest = 0;
        for (int g = 0; g < groups; ++g) {
            const int a = g * h, b = std::min(heads, a + h) - 1;
            widest = std::max(widest, (b / per - a / per + 1) * dim);
        }
        if (widest > 128 && h > 1) continue;
        // as few heads a group as the number of groups takes, so that the last is no smaller
        const int even = (heads + groups - 1) / groups;
        if (even < h) {
            h = even + 1;
            continue;
        }
        r.heads = h;
        r.groups = groups;
        r.tiles = widest <= 64 ? 1 : 2;
        r.per_m = ((1 << 20) + per - 1) / per;
        return r;
    }
    return r;
}

// The same for the pass by source: `heads` of k, and of the q heads that share each, `shared` a
// pass over the row's edges.
struct KvGroups {
    int heads, groups, shared, passes, tiles;
};

KvGroups kv_groups(int kv_heads, int per, int dim)
{
    KvGroups r{};
    r.shared = 1;
    for (int s = 2; s <= std::min(per, 8); ++s)
        if (per % s == 0 && s * dim <= 128) r.shared = s;
    r.passes = per / r.shared;
    r.heads = 1;
    if (r.passes == 1) {
        r.heads = std::max(1, std::min({kv_heads, 8 / r.shared, 128 / (r.shared * dim)}));
        const int groups = (kv_heads + r.heads - 1) / r.heads;
        r.heads = (kv_heads + groups - 1) / groups;
    }
    r.groups = (kv_heads + r.heads - 1) / r.heads;
    r.tiles = r.heads * r.shared * dim <= 64 ? 1 : 2;
    return r;
}

using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kWaves = 4;
constexpr float kSlack = 8.0f;  // the running maximum is renewed when a logit passes it by 2^8

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// x and its value in the lane 16 (32) over, in an order of their own.
template <int APART>
__device__ __forceinline__ float2 with_lane(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = APART == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                               : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];  // (a bit cast of r[1] itself would read r[0])
    return make_float2(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
// Maximum and sum over the four lanes of a column (16 apart), to all of them.
__device__ __forceinline__ float column_max(float x)
{
    const float2 a = with_lane<16>(x);
    const float2 b = with_lane<32>(fmaxf(a.x, a.y));
    return fmaxf(b.x, b.y);
}
__device__ __forceinline__ float column_sum(float x)
{
    const float2 a = with_lane<16>(x);
    const float2 b = with_lane<32>(a.x + a.y);
    return b.x + b.y;
}
// x of the lane eight columns over (row_ror:8), added
__device__ __forceinline__ float add_twin(float x)
{
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
}

// What a lane is in a group of heads: column n, quarter g of the summed index.
struct Lane {
    int n, g, head;  // head: of its column, in the tensors
    bool real;       // that head exists
    int kv0;         // the group's first head of k
    int source;      // the head whose channels stand in its column of the spread row
    int base;        // first channel of its rows of the gathered heads, from the group's first
    int wide;        // channels of the group's gathered heads
};

__device__ __forceinline__ int over_per(const HeadGroups& hg, int x) { return (int)(x * hg.per_m >> 20); }

// Keeps the compiler from doing both sides of a branch that is hardly ever taken.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// The same value, computed anew: keeps what depends on it out of the registers of a row's loop.
__device__ __forceinline__ int anew(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ Lane lane_of(const AttnArgs& a, const HeadGroups& hg, int group)
{
    Lane l;
    const int lane = threadIdx.x & 63;
    l.n = lane & 15;
    l.g = lane >> 4;
    const int h0 = group * hg.heads, hn = min(hg.heads, a.heads - h0);
    l.real = (l.n & 7) < hn;
    l.head = h0 + min(l.n & 7, hn - 1);
    l.kv0 = over_per(hg, h0);
    l.source = l.head;
    l.base = (over_per(hg, l.head) - l.kv0) * a.dim;
    l.wide = (over_per(hg, h0 + hn - 1) - l.kv0 + 1) * a.dim;
    return l;
}

// Byte offset of row j: 32 bits where tensor and nodes allow it (a multiply-add of 24 bits and a
// register less a row than 64).
template <bool FAR>
using Offset = std::conditional_t<FAR, uint64_t, uint32_t>;
template <bool FAR>
__device__ __forceinline__ Offset<FAR> row_at(int j, int64_t ld_bytes)
{
    if constexpr (FAR) return (uint64_t)j * (uint64_t)ld_bytes;
    else return __umul24((uint32_t)j, (uint32_t)ld_bytes);
}

// A row's channels of one tensor as the block-diagonal operand: step s, column n; kept in LDS, each
// lane its own 16 bytes a step.  Loaded through a descriptor of the row, where what lies off the
// diagonal is out of range and so reads as zero, without a branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* p, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
template <int NT>
struct Spread {
    u32x4 v[2 * NT];
    __device__ __forceinline__ void load(const __bf16* row, int heads, const Lane& l, int dim)
    {
        const __amdgpu_buffer_rsrc_t b = row_buffer(row, 2 * heads * dim);
        const int at = 8 * l.g - l.base;  // channel of step 0 in the column's head
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) {
            const bool in = l.real && (uint32_t)(at + 32 * s) < (uint32_t)dim;
            v[s] = __builtin_amdgcn_raw_buffer_load_b128(b, in ? 2 * (l.source * dim + at + 32 * s) : 0x7ffffff0, 0, 0);
        }
    }
    __device__ __forceinline__ void put(u32x4* s_x) const
    {
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) s_x[64 * s] = v[s];
    }
};

// A lane's channels of an edge in memory: eight (16 bytes) where the group has 128 channels or
// more, so that four lanes make a whole 64-byte access; the sixteen lanes of a quarter side by
// side.  (Loaded as the matrix operand wants them, a row of k a lane, every access would fetch 16
// bytes of 64: 1245 us instead of 618 for 26.5M edges of 128 channels.)
template <int NT>
constexpr int kV = NT == 1 ? 4 : 8;
template <int NT>
using VChunk = std::conditional_t<NT == 1, u32x2, u32x4>;
// `at`: the lane's first byte in a row, at most the group's last chunk (where the group has fewer
// channels the chunk is read again; its products meet zeros and its sums are not stored).
template <int NT>
__device__ __forceinline__ uint32_t lane_bytes(const Lane& l)
{
    return 2 * min(kV<NT> * l.n, l.wide - kV<NT>);
}
template <int NT, bool FAR>
__device__ __forceinline__ VChunk<NT> load_edge(const char* base, uint32_t node, int64_t ld, uint32_t at)
{
    return *(const VChunk<NT>*)(base + (row_at<FAR>(node, 2 * ld) + at));
}

// Sixteen edges' rows in LDS, a wave's own, in chunks of 16 bytes swapped within the row so that
// neither a row's writes nor sixteen rows' reads of one chunk meet on a bank.
template <int NT>
constexpr int kRowBytes = 128 * NT;
template <int NT>
__device__ __forceinline__ int chunk_at(int row, int chunk)
{
    return row * kRowBytes<NT> + (chunk ^ (NT == 1 ? (row >> 1) & 7 : row)) * 16;
}
template <int NT>
__device__ __forceinline__ void put_edge(char* s_k, int row, const Lane& l, VChunk<NT> x)
{
    if constexpr (NT == 1) *(u32x2*)(s_k + chunk_at<NT>(row, l.n / 2) + l.n % 2 * 8) = x;
    else *(u32x4*)(s_k + chunk_at<NT>(row, l.n)) = x;
}

// Products of sixteen edges with the spread row.
template <int NT>
__device__ __forceinline__ f32x4 products_at_once(const char* s_k, const Lane& l, const u32x4* spread)
{
    f32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s)
        c = mfma(__builtin_bit_cast(bf16x8, *(const u32x4*)(s_k + chunk_at<NT>(l.n, 4 * s + l.g))),
                 __builtin_bit_cast(bf16x8, spread[64 * s]), c);
    return c;
}

// The same head of k by head of k, for rows that hold what is not finite: a column sees its own
// head's channels only.  The same products in the same places, so the same bits.
template <int NT>
__device__ __forceinline__ f32x4 products_apart(const char* s_k, const Lane& l, int dim, const u32x4* spread)
{
    f32x4 c = {0, 0, 0, 0};
#pragma unroll 1
    for (int first = 0; first < l.wide; first += dim) {
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 2 * NT; ++s) {
            u32x4 v = {0, 0, 0, 0};
            if ((uint32_t)(32 * s + 8 * l.g - first) < (uint32_t)dim) v = *(const u32x4*)(s_k + chunk_at<NT>(l.n, 4 * s + l.g));
            x = mfma(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, spread[64 * s]), x);
        }
        if (l.base == first) c = x;
    }
    return c;
}

// Edges 4 i .. 4 i + 3 of a lane's eight (sixteen of the step) through LDS: their products with
// the spread row.
template <int NT, bool APART>
__device__ __forceinline__ f32x4 products(char* s_k, const Lane& l, int dim, const u32x4* spread, const VChunk<NT> (&k)[8],
                                          int i)
{
#pragma unroll
    for (int x = 0; x < 4; ++x) put_edge<NT>(s_k, 4 * l.g + x, l, k[4 * i + x]);
    if constexpr (APART) return products_apart<NT>(s_k, l, dim, spread);
    return products_at_once<NT>(s_k, l, spread);
}

// The channels of each of a lane's eight edges -> for channel i of them, the eight edges.
template <typename C>
__device__ __forceinline__ bf16x8 turned(const C (&v)[8], int i)
{
    u32x4 r;
#pragma unroll
    for (int d = 0; d < 4; ++d)
        r[d] = __builtin_amdgcn_perm(v[2 * d + 1][i / 2], v[2 * d][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(bf16x8, r);
}

// Those of eight values that are infinite, the others as zeros (or, FINITE, the other way round).
template <bool FINITE>
__device__ __forceinline__ bf16x8 only(bf16x8 v)
{
    const u32x4 u = __builtin_bit_cast(u32x4, v);
    u32x4 r;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t mask = ((u[d] & 0x7fffu) == 0x7f80u ? 0xffffu : 0) | ((u[d] & 0x7fff0000u) == 0x7f800000u ? 0xffff0000u : 0);
        r[d] = u[d] & (FINITE ? ~mask : mask);
    }
    return __builtin_bit_cast(bf16x8, r);
}

// Whether any of the values is a NaN or an infinity.
template <typename C>
__device__ __forceinline__ bool unbounded(C v)
{
    bool r = false;
#pragma unroll
    for (int d = 0; d < (int)sizeof(C) / 4; ++d) r |= (v[d] & 0x7f80u) == 0x7f80u || (v[d] & 0x7f800000u) == 0x7f800000u;
    return r;
}

// Whether the logit of an edge of the lane is -inf in every column (the sixteen lanes of its quarter).
__device__ __forceinline__ bool of_no_head(const Lane& l, float s)
{
    return ((__ballot(s == -INFINITY) >> (16 * l.g)) & 0xffffu) == 0xffffu;
}

// Where the table holds entries of -inf: values of edges that these take out for every head become
// zeros; true where values that are not finite remain.
template <int NT>
__device__ __forceinline__ bool hide(const Lane& l, const float (&s)[8], VChunk<NT> (&v)[8])
{
    bool bad = false;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        if (of_no_head(l, s[x])) v[x] = VChunk<NT>{};
        bad |= unbounded(v[x]);
    }
    return bad;
}

// One row for heads [h0, h0 + hn), an edge and a head at a time: four channels a lane.  For rows
// that hold what is not finite.
__device__ void forward_apart(const AttnArgs& a, const Piece& p, int h0, int hn, const float* tab)
{
    const int lane = anew(threadIdx.x & 63), ch = 4 * lane;
    const bool wide = ch < a.dim;
    for (int h = h0; h < min(h0 + hn, a.heads); ++h) {
        const int64_t at = (int64_t)(h / a.per) * a.dim + ch;
        float q[4] = {0, 0, 0, 0}, acc[4] = {0, 0, 0, 0}, m = -INFINITY, sum = 0;
        if (wide) load4((const __bf16*)a.q + p.node * a.ldq + (int64_t)h * a.dim + ch, q);
        for (int e = p.begin; e < p.end; ++e) {
            const float b = tab ? tab[(int)a.L.bucket[e] * a.heads + h] : 0.0f;
            if (b == -INFINITY) continue;
            const int64_t j = a.L.idx[e];
            float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
            if (wide) {
                load4((const __bf16*)a.k + j * a.ldk + at, k);
                load4((const __bf16*)a.v + j * a.ldv + at, v);
            }
            float d = 0;
            for (int i = 0; i < 4; ++i) d = fmaf(q[i], k[i], d);
            const float s = fmaf(sum_lanes<64>(d), a.scale * kLog2e, b);
            const float to = fmaxf(m, s), base = to == -INFINITY ? 0.0f : to;
            const float shrink = exp2_fast(m - base), pr = exp2_fast(s - base);
            sum = sum * shrink + pr;
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(pr, v[i], acc[i] * shrink);
            m = to;
        }
        if (p.item >= 0) {
            if (lane == 0) {
                a.part_m[p.item * a.heads + h] = m;
                a.part_l[p.item * a.heads + h] = sum;
            }
            if (wide) store4(a.part_acc + (p.item * a.heads + h) * a.dim + ch, acc);
            continue;
        }
        const int64_t row = (int64_t)p.node * a.heads + h;
        for (int i = 0; i < 4; ++i) acc[i] = sum == 0.0f ? 0.0f : acc[i] / sum;
        if (wide) {
            store4((__bf16*)a.out + row * a.dim + ch, acc);
            if (a.out32) store4(a.out32 + row * a.dim + ch, acc);
        }
        if (lane == 0) store_norm(a, row, m, sum);
    }
}

// Weights of a lane's eight edges as the operand: rounded in columns 0 .. 7, the rest in 8 .. 15.
// (`minus`: 0 in the former, -1 in the latter)
__device__ __forceinline__ bf16x8 two_parts(const float (&p)[8], float minus)
{
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)fmaf((float)(__bf16)p[i], minus, p[i]);
    return r;
}

// One where a weight is not zero: what an infinity is to be multiplied with (and a NaN, as the weights are).
__device__ __forceinline__ bf16x8 above_zero(const float (&p)[8])
{
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)(p[i] > 0.0f ? 1.0f : p[i]);
    return r;
}

// What two_parts leave out, in columns 0 .. 7.  (That is 2^-18 of a weight at most; but the backward
// pass takes <g, out> from the sums, which is summed over a bucket's edges where it cancels: with two
// parts the table's gradient was 1.0e-6 off the 64-bit one, with three it is 2e-7.  27M edges of 8
// heads of 16: 851 us with two, 887 us with three, 904 us with `v` turned anew for the third.)
__device__ __forceinline__ bf16x8 third_part(const float (&p)[8], bool first)
{
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float rest = p[i] - (float)(__bf16)p[i];
        r[i] = (__bf16)(first ? rest - (float)(__bf16)rest : 0.0f);
    }
    return r;
}

// Whether all sums of a lane are numbers.
template <int NT>
__device__ __forceinline__ bool finite(const f32x4 (&acc)[kV<NT>])
{
    float x = 0;
#pragma unroll
    for (int i = 0; i < kV<NT>; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) x = fmaf(0.0f, acc[i][r], x);
    return x == 0.0f;
}

// 32 entries of a row, one a lane: the node, with the bucket in the upper eight bits where nodes
// take 24 (!FAR).  A lane past the row's end holds the row's last entry.  The lanes of a step
// then fetch the entries that they need from each other: one access a list where loads by those
// lanes would be eight, and accesses to the cache are what these kernels run out of.
template <bool FAR>
struct Block {
    uint32_t node;
    uint32_t bucket;  // FAR only
};

template <bool BUCKETS, bool FAR>
__device__ __forceinline__ Block<FAR> block_at(const Lists& L, int e0, int end)
{
    // (an empty row reads some entry)
    const int e = min(e0 + (int)(threadIdx.x & 31), max(end - 1, 0));
    Block<FAR> b;
    b.node = L.idx[e];
    b.bucket = 0;
    if (BUCKETS) {
        const uint32_t x = L.bucket[e];
        if (FAR) b.bucket = x;
        else b.node |= x << 24;
    }
    return b;
}

// The eight edges of a step's 32 that a lane loads, and holds in the softmax.
__device__ __forceinline__ int edge_of(const Lane& l, int x) { return (x < 4 ? 0 : 12) + 4 * l.g + x; }

__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane)
{
    return __builtin_amdgcn_ds_bpermute(4 * lane, x);
}

template <bool FAR>
struct Step {
    Block<FAR> edge[8];
};

template <bool BUCKETS, bool FAR>
__device__ __forceinline__ Step<FAR> step_of(const Block<FAR>& b, const Lane& l)
{
    Step<FAR> s;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        s.edge[x].node = from_lane(b.node, edge_of(l, x));
        s.edge[x].bucket = BUCKETS && FAR ? from_lane(b.bucket, edge_of(l, x)) : 0;
    }
    return s;
}

// The bounds of a unit, under way in vector registers.
struct Bounds {
    int begin, end, node;
};
__device__ __forceinline__ Bounds bounds_at(const Lists& L, const Walk& w, int64_t u)
{
    u = min(u, w.end - 1);
    const int* item = (const int*)(L.items + w.item(u));
    const bool is = w.is_item(u);
    const int* begin = is ? item : L.ptr + w.slot(u);
    const int* node = is ? item + 2 : L.order + w.slot(u);
    return Bounds{begin[0], begin[1], *node};
}
__device__ __forceinline__ Piece piece_from(const Lists& L, const Walk& w, int64_t u, const Bounds& b)
{
    Piece p;
    p.begin = __builtin_amdgcn_readfirstlane(b.begin);
    p.end = __builtin_amdgcn_readfirstlane(b.end);
    p.node = __builtin_amdgcn_readfirstlane(b.node);
    p.item = w.is_item(u) ? w.item(u) : -1;
    if (!w.is_item(u) && L.n_items && p.end - p.begin > DG_NEIGHBOR_SPLIT) p.node = -1;
    if (p.node < 0) p.end = p.begin;
    return p;
}

template <bool FAR>
__device__ __forceinline__ uint32_t bucket_of(const Block<FAR>& b)
{
    return FAR ? b.bucket : b.node >> 24;
}

// A row's sums of both parts: f(x, ch) for each chunk of eight channels that a lane holds of its
// column's head, ch its first channel there.  The lanes of the first eight columns add their twins'.
template <int NT, typename F>
__device__ __forceinline__ void each_chunk(const Lane& l, int dim, const f32x4 (&acc)[kV<NT>], F&& f)
{
    constexpr int VW = kV<NT>;
    const int first = anew(4 * VW * l.g - l.base);
#pragma unroll
    for (int k = 0; k < VW / 2; ++k) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = add_twin(VW == 8 ? acc[i][k] : acc[i % 4][2 * k + i / 4]);
        const int ch = first + 8 * k;
        if (l.real && l.n < 8 && (uint32_t)ch < (uint32_t)dim) f(x, ch);
    }
}

__device__ __forceinline__ void store8(float* p, const float (&x)[8])
{
    *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__bf16* p, const float (&x)[8])
{
    bf16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (__bf16)x[i];
    *(bf16x8*)p = y;
}

template <int NT>
__device__ __forceinline__ void finish_row(const AttnArgs& a, const Piece& p, const Lane& l, const f32x4 (&acc)[kV<NT>],
                                           float m, float sum)
{
    sum = column_sum(sum);
    const int64_t row = (int64_t)p.node * a.heads + l.head;
    const float inv = sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum);
    each_chunk<NT>(l, a.dim, acc, [&](float (&x)[8], int ch) {
        if (p.item >= 0) {
            store8(a.part_acc + (p.item * a.heads + l.head) * a.dim + ch, x);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        store8((__bf16*)a.out + row * a.dim + ch, x);
        if (a.out32) store8(a.out32 + row * a.dim + ch, x);
    });
    if (l.real && l.g == 0 && l.n < 8) {
        if (p.item >= 0) {
            a.part_m[p.item * a.heads + l.head] = m;
            a.part_l[p.item * a.heads + l.head] = sum;
        } else {
            store_norm(a, row, m, sum);
        }
    }
}

// The table in base 2 in LDS; whether it holds an entry of -inf.
template <bool BUCKETS>
__device__ __forceinline__ bool stage_table(const AttnArgs& a, float* s_tab, int* s_any)
{
    if (!BUCKETS) return false;
    if (threadIdx.x == 0) *s_any = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_buckets * a.heads; i += 64 * kWaves) {
        const float x = a.table[i];
        s_tab[i] = entry_base2(x);
        if (x == -INFINITY) *s_any = 1;  // (every writer writes the same value)
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*s_any) != 0;
}

// Base-2 logits of the lane's eight edges for its column's head: -inf where there is none.
template <bool BUCKETS, bool FAR>
__device__ __forceinline__ void logits(const AttnArgs& a, const Lane& l, const Step<FAR>& st, const f32x4 (&products)[2], int n,
                                       float scale2, bool takes_out, const float* s_tab, float (&s)[8])
{
    float b[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        b[x] = BUCKETS ? s_tab[__umul24(bucket_of(st.edge[x]), a.heads) + l.head] : 0.0f;
        s[x] = fmaf(products[x / 4][x % 4], scale2, b[x]);
    }
    if (BUCKETS && takes_out) {
        keep_branch();
#pragma unroll
        for (int x = 0; x < 8; ++x) s[x] = b[x] == -INFINITY ? b[x] : s[x];
    }
    if (n < 32) {
        keep_branch();
#pragma unroll
        for (int x = 0; x < 8; ++x) s[x] = edge_of(l, x) < n ? s[x] : -INFINITY;
    }
}

// Waves a SIMD, by tiles of 64 channels: as many as the loads of a step in flight leave registers
// for.  (2.9M edges, 8 heads of 32: 200 us with 2, 183 with 3, 378 with 4, which spills; 4 heads of
// 16: 75 us with 3, 70 with 4, 83 with 5.)  What bounds it there: the gathered rows, 64 bytes a clock
// and CU into registers (80 us), the vector units' instructions (90 us), and the wait for one step's
// rows, of which a wave has no more than one under way: 26.5M edges of 8 heads of 16 take 840 us, at 63 %
// of the vector units' cycles and 58 % of the L1's.
constexpr int waves_of(int NT) { return NT == 2 ? 3 : 4; }

template <int NT, bool BUCKETS, bool FAR>
__global__ __launch_bounds__(64 * kWaves, waves_of(NT)) void forward_mfma_kernel(AttnArgs a, HeadGroups hg)
{
    extern __shared__ float s_tab[];
    __shared__ u32x4 s_q[kWaves][2 * NT * 64];
    __shared__ __attribute__((aligned(16))) char s_k[kWaves][16 * kRowBytes<NT>];
    __shared__ int s_any;
    const bool takes_out = stage_table<BUCKETS>(a, s_tab, &s_any);
    const float scale2 = a.scale * kLog2e;
    const Walk w = walk_of(a.L, kWaves);
    if (w.at >= w.end) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    u32x4* my_q = s_q[wave] + (threadIdx.x & 63);
    char* my_k = s_k[wave];
    const Lane l = lane_of(a, hg, blockIdx.y);
    const uint32_t lane_at = lane_bytes<NT>(l);
    const char* kb = (const char*)a.k + 2 * l.kv0 * a.dim;
    const char* vb = (const char*)a.v + 2 * l.kv0 * a.dim;
    // The entries of the next step, and the bounds of the row after the next, are under way while
    // a step is worked on: they come from memory for the first time.  Every step issues the same
    // loads in the same order (the tail's lanes load the last edge again), so that the waits
    // between them can be counted.  A row without entries has a step too, whose sums are dropped.
    // The next row's q is under way while a row's result is stored.
    Piece p = piece_from(a.L, w, w.at, bounds_at(a.L, w, w.at));
    Piece next = piece_from(a.L, w, w.at + w.step, bounds_at(a.L, w, w.at + w.step));
    Block<FAR> block = block_at<BUCKETS, FAR>(a.L, p.begin, p.end);
    Spread<NT> q;
    q.load((const __bf16*)a.q + max(p.node, 0) * a.ldq, a.heads, l, a.dim);
    q.put(my_q);
    for (int64_t u = w.at; u < w.end; u += w.step) {
        Bounds later;
        f32x4 acc[kV<NT>];
        float m, sum;
        bool redo;
        auto row = [&](auto apart) {
            constexpr bool APART = decltype(apart)::value;
#pragma unroll
            for (int i = 0; i < kV<NT>; ++i) acc[i] = f32x4{0, 0, 0, 0};
            m = -INFINITY;
            sum = 0;
            redo = false;
            int e0 = p.begin;
            do {
                const int n = p.end - e0;
                const Step<FAR> st = step_of<BUCKETS, FAR>(block, l);
                VChunk<NT> k[8], v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) k[x] = load_edge<NT, FAR>(kb, st.edge[x].node, a.ldk, lane_at);
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = load_edge<NT, FAR>(vb, st.edge[x].node, a.ldv, lane_at);
                __builtin_amdgcn_sched_barrier(0);  // (all in flight before the first is waited for)
                block = block_at<BUCKETS, FAR>(a.L, n > 32 ? e0 + 32 : next.begin, n > 32 ? p.end : next.end);
                later = bounds_at(a.L, w, u + 2 * w.step);
                __builtin_amdgcn_sched_barrier(0);
                const f32x4 qk[2] = {products<NT, APART>(my_k, l, a.dim, my_q, k, 0), products<NT, APART>(my_k, l, a.dim, my_q, k, 1)};
                float s[8];
                logits<BUCKETS>(a, l, st, qk, n, scale2, takes_out, s_tab, s);
                const float top = column_max(fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                                                   fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))));
                if (e0 == p.begin) {
                    m = top;
                } else if (__any(top > m + kSlack)) {
                    const float to = fmaxf(m, top);
                    const float shrink = to == -INFINITY ? 1.0f : exp2_fast(m - to);
                    m = to;
                    sum *= shrink;
#pragma unroll
                    for (int i = 0; i < kV<NT>; ++i) acc[i] *= shrink;
                }
                const float base = m == -INFINITY ? 0.0f : m;
                float pr[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    pr[x] = exp2_fast(s[x] - base);
                    sum += pr[x];
                }
                const bf16x8 weight = two_parts(pr, l.n >= 8 ? -1.0f : 0.0f), last = third_part(pr, l.n < 8);
                if (BUCKETS && takes_out) {
                    keep_branch();
                    redo |= hide<NT>(l, s, v);
                }
                if constexpr (APART) {  // (lanes past the row's end hold its last edge)
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if (edge_of(l, x) >= n) v[x] = VChunk<NT>{};
                }
#pragma unroll
                for (int i = 0; i < kV<NT>; ++i) {
                    const bf16x8 vi = turned(v, i);
                    if constexpr (APART) {  // an infinity meets a weight that is whole
                        const bf16x8 finite = only<true>(vi);
                        acc[i] = mfma(finite, last, mfma(finite, weight, acc[i]));
                        acc[i] = mfma(only<false>(vi), above_zero(pr), acc[i]);
                    } else {
                        acc[i] = mfma(vi, last, mfma(vi, weight, acc[i]));
                    }
                }
                e0 += 32;
            } while (e0 < p.end);
        };
        row(std::false_type{});
        // (said to be rare: else what this branch needs spills registers of the loop, 962 us against 850 for
        // 27M edges of 8 heads of 16)
        if (__builtin_expect(__any(isnan(sum) || !finite<NT>(acc)), 0)) {
            keep_branch();
            block = block_at<BUCKETS, FAR>(a.L, p.begin, p.end);
            row(std::true_type{});
        }
        q.load((const __bf16*)a.q + max(next.node, 0) * a.ldq, a.heads, l, a.dim);
        if (p.begin == p.end) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < kV<NT>; ++i) acc[i] = f32x4{0, 0, 0, 0};
        }
        if (__any(redo) && p.node >= 0) forward_apart(a, p, (int)blockIdx.y * hg.heads, hg.heads, s_tab);
        else if (p.node >= 0) finish_row<NT>(a, p, l, acc, m, sum);
        q.put(my_q);
        p = next;
        next = piece_from(a.L, w, u + 2 * w.step, later);
    }
}

// ---------------------------------------------------------------- backward, by target
// (as waves_of; the whole backward pass, 8 heads of 32: 743 us with 1, 601 with 2, 985 with 3; 4
// heads of 16: 238 us with 2, 222 with 3, 240 with 4)
constexpr int waves_of_q(int NT) { return NT == 2 ? 2 : 3; }

// delta = <g, out> of a column's head: eight channels a lane, whose sums the head's lanes add up.
__device__ __forceinline__ float delta_of(const AttnArgs& a, const HeadGroups& hg, int node, const Lane& l, float* s_x)
{
    const int h0 = (int)blockIdx.y * hg.heads, chunks = min(hg.heads, a.heads - h0) * a.dim / 8;
    const __bf16* g = (const __bf16*)a.g + node * a.ldg + h0 * a.dim;
    const float* o = a.out32 + ((int64_t)node * a.heads + h0) * a.dim;
    for (int c = anew(threadIdx.x & 63); c < chunks; c += 64) {
        float x[4], y[4];
        load4(g + 8 * c, x);
        load4(g + 8 * c + 4, y);
        const float4 u = *(const float4*)(o + 8 * c), v = *(const float4*)(o + 8 * c + 4);
        float d = x[0] * u.x;
        d = fmaf(x[1], u.y, d);
        d = fmaf(x[2], u.z, d);
        d = fmaf(x[3], u.w, d);
        d = fmaf(y[0], v.x, d);
        d = fmaf(y[1], v.y, d);
        d = fmaf(y[2], v.z, d);
        s_x[c] = fmaf(y[3], v.w, d);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float d = 0;
    const float* mine = s_x + (l.head - h0) * (a.dim / 8);
    for (int i = 0; i < a.dim / 8; ++i) d += mine[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return d;
}

// dq of one row for heads [h0, h0 + hn), as forward_apart.
__device__ void backward_q_apart(const AttnArgs& a, const Piece& p, int h0, int hn, const float* tab)
{
    const int lane = anew(threadIdx.x & 63), ch = 4 * lane;
    const bool wide = ch < a.dim;
    for (int h = h0; h < min(h0 + hn, a.heads); ++h) {
        const int64_t at = (int64_t)(h / a.per) * a.dim + ch, row = (int64_t)p.node * a.heads + h;
        const float4 st = a.stats[row];
        float q[4] = {0, 0, 0, 0}, g[4] = {0, 0, 0, 0}, dq[4] = {0, 0, 0, 0};
        if (wide) {
            load4((const __bf16*)a.q + p.node * a.ldq + (int64_t)h * a.dim + ch, q);
            load4((const __bf16*)a.g + p.node * a.ldg + (int64_t)h * a.dim + ch, g);
        }
        for (int e = p.begin; e < p.end; ++e) {
            const float b = tab[(int)a.L.bucket[e] * a.heads + h];
            if (b == -INFINITY) continue;
            const int64_t j = a.L.idx[e];
            float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
            if (wide) {
                load4((const __bf16*)a.k + j * a.ldk + at, k);
                load4((const __bf16*)a.v + j * a.ldv + at, v);
            }
            float s = 0, dp = 0;
            for (int i = 0; i < 4; ++i) {
                s = fmaf(q[i], k[i], s);
                dp = fmaf(g[i], v[i], dp);
            }
            s = fmaf(sum_lanes<64>(s), a.scale * kLog2e, b);
            const float ds = exp2_fast(s - st.x) * st.y * (sum_lanes<64>(dp) - st.z);
            for (int i = 0; i < 4; ++i) dq[i] = fmaf(ds, k[i], dq[i]);
        }
        if (!wide) continue;
        if (p.item >= 0) {
            store4(a.part_acc + (p.item * a.heads + h) * a.dim + ch, dq);
        } else {
            for (int i = 0; i < 4; ++i) dq[i] *= a.scale;
            store4((__bf16*)a.dq + row * a.dim + ch, dq);
        }
    }
}

// dq, stats, and with BT > 0 the table's gradient: its sums over the edges of a bucket are products
// with the buckets' indicators, 16 buckets by 4 edges a step in full float (one bit of each
// indicator is set, so every term is exact), and stay in BT accumulators for all of a wave's rows.
// What is not finite would meet the indicators' zeros: it goes to LDS by itself.  3.0M edges of 8
// heads of 32, 32 buckets: 348 us, at 38 % of the vector units and 33 % of the L1's cycles, waiting for
// rows as in the forward pass; 7.8M edges of 8 heads over 2: 341 us.
template <int NT, int BT, bool FAR>
__global__ __launch_bounds__(64 * kWaves, waves_of_q(NT)) void backward_q_mfma_kernel(AttnArgs a, HeadGroups hg)
{
    constexpr bool BUCKETS = BT > 0;
    extern __shared__ float s_tab[];
    __shared__ u32x4 s_q[kWaves][2 * NT * 64], s_g[kWaves][2 * NT * 64];
    __shared__ __attribute__((aligned(16))) char s_k[kWaves][16 * kRowBytes<NT>];
    __shared__ int s_any;
    const int cells = a.n_buckets * a.heads;
    float* s_odd = s_tab + cells;  // [cells], then [kWaves][16 BT][8]
    float* s_sum = s_odd + cells;
    const bool takes_out = stage_table<BUCKETS>(a, s_tab, &s_any);
    if (BUCKETS) {
        for (int i = threadIdx.x; i < cells; i += 64 * kWaves) s_odd[i] = 0;
        __syncthreads();
    }
    const float scale2 = a.scale * kLog2e;
    const Walk w = walk_of(a.L, kWaves);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    u32x4* my_q = s_q[wave] + (threadIdx.x & 63);
    u32x4* my_g = s_g[wave] + (threadIdx.x & 63);
    char* my_k = s_k[wave];
    const Lane l = lane_of(a, hg, blockIdx.y);
    const uint32_t lane_at = lane_bytes<NT>(l);
    const char* kb = (const char*)a.k + 2 * l.kv0 * a.dim;
    const char* vb = (const char*)a.v + 2 * l.kv0 * a.dim;
    f32x4 tab[BUCKETS ? BT : 1] = {};
    if (w.at < w.end) {
        // (what runs ahead: as in forward_mfma_kernel)
        Piece p = piece_from(a.L, w, w.at, bounds_at(a.L, w, w.at));
        Piece next = piece_from(a.L, w, w.at + w.step, bounds_at(a.L, w, w.at + w.step));
        Block<FAR> block = block_at<BUCKETS, FAR>(a.L, p.begin, p.end);
        Spread<NT> q, g;
        float2 norm;
        float delta;
        auto load_row = [&](int node) {
            q.load((const __bf16*)a.q + node * a.ldq, a.heads, l, a.dim);
            g.load((const __bf16*)a.g + node * a.ldg, a.heads, l, a.dim);
        };
        auto put_row = [&](const Piece& of) {
            const int64_t row = (int64_t)max(of.node, 0) * a.heads + l.head;
            norm = a.norm[row];
            delta = delta_of(a, hg, max(of.node, 0), l, (float*)my_k);
            if (of.node >= 0 && l.real && l.g == 0 && l.n < 8) a.stats[row] = make_float4(norm.x, norm.y, delta, 0.0f);
            q.put(my_q);
            g.put(my_g);
        };
        load_row(max(p.node, 0));
        put_row(p);
        for (int64_t u = w.at; u < w.end; u += w.step) {
            Bounds later;
            f32x4 acc[kV<NT>] = {};
            bool redo = false;
            int e0 = p.begin;
            do {
                const int n = p.end - e0;
                const Step<FAR> st = step_of<BUCKETS, FAR>(block, l);
                VChunk<NT> k[8], v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) k[x] = load_edge<NT, FAR>(kb, st.edge[x].node, a.ldk, lane_at);
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = load_edge<NT, FAR>(vb, st.edge[x].node, a.ldv, lane_at);
                __builtin_amdgcn_sched_barrier(0);
                block = block_at<BUCKETS, FAR>(a.L, n > 32 ? e0 + 32 : next.begin, n > 32 ? p.end : next.end);
                later = bounds_at(a.L, w, u + 2 * w.step);
                __builtin_amdgcn_sched_barrier(0);
                float s[8], ds[8];
                auto slopes = [&](auto apart) {
                    constexpr bool APART = decltype(apart)::value;
                    const f32x4 qk[2] = {products<NT, APART>(my_k, l, a.dim, my_q, k, 0),
                                         products<NT, APART>(my_k, l, a.dim, my_q, k, 1)};
                    const f32x4 gv[2] = {products<NT, APART>(my_k, l, a.dim, my_g, v, 0),
                                         products<NT, APART>(my_k, l, a.dim, my_g, v, 1)};
                    logits<BUCKETS>(a, l, st, qk, n, scale2, takes_out, s_tab, s);
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        ds[x] = s[x] == -INFINITY ? 0.0f : exp2_fast(s[x] - norm.x) * norm.y * (gv[x / 4][x % 4] - delta);
                };
                slopes(std::false_type{});
                float all = 0;
#pragma unroll
                for (int x = 0; x < 8; ++x) all = fmaf(0.0f, ds[x], all);
                const bool odd = __any(all != 0.0f);  // (a NaN)
                if (odd) {
                    keep_branch();
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = load_edge<NT, FAR>(vb, st.edge[x].node, a.ldv, lane_at);
                    slopes(std::true_type{});
                }
                const bf16x8 weight = two_parts(ds, l.n >= 8 ? -1.0f : 0.0f);
                if (BUCKETS && takes_out) {
                    keep_branch();
                    redo |= hide<NT>(l, s, k);
                }
#pragma unroll
                for (int i = 0; i < kV<NT>; ++i) acc[i] = mfma(turned(k, i), weight, acc[i]);
                if constexpr (BUCKETS) {
                    if (odd) {
                        keep_branch();
                        for (int x = 0; x < 8; ++x) {
                            if (0.0f * ds[x] == 0.0f) continue;
                            if (l.real && l.n < 8) atomicAdd(&s_odd[bucket_of(st.edge[x]) * a.heads + l.head], ds[x]);
                            ds[x] = 0;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < BT; ++t)
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const float is = (int)bucket_of(st.edge[x]) == 16 * t + l.n ? 1.0f : 0.0f;
                            tab[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(is, ds[x], tab[t], 0, 0, 0);
                        }
                }
                e0 += 32;
            } while (e0 < p.end);
            load_row(max(next.node, 0));
            if (p.begin == p.end) {
                keep_branch();
#pragma unroll
                for (int i = 0; i < kV<NT>; ++i) acc[i] = f32x4{0, 0, 0, 0};
            }
            if (__any(redo) && p.node >= 0) {
                backward_q_apart(a, p, (int)blockIdx.y * hg.heads, hg.heads, s_tab);
            } else if (p.node >= 0) {
                each_chunk<NT>(l, a.dim, acc, [&](float (&x)[8], int ch) {
                    if (p.item >= 0) {
                        store8(a.part_acc + (p.item * a.heads + l.head) * a.dim + ch, x);
                        return;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] *= a.scale;
                    store8((__bf16*)a.dq + ((int64_t)p.node * a.heads + l.head) * a.dim + ch, x);
                });
            }
            p = next;
            put_row(p);
            next = piece_from(a.L, w, u + 2 * w.step, later);
        }
    }
    if constexpr (BUCKETS) {
        if (l.n < 8)
#pragma unroll
            for (int t = 0; t < BT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s_sum[(wave * 16 * BT + 16 * t + 4 * l.g + r) * 8 + l.n] = tab[t][r];
        __syncthreads();
        const int h0 = (int)blockIdx.y * hg.heads, h1 = min(h0 + hg.heads, a.heads);
        float* out = a.dtab + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * cells;
        for (int i = threadIdx.x; i < cells; i += 64 * kWaves) {
            const int h = i % a.heads, b = i / a.heads;
            float x = 0;
            if (h >= h0 && h < h1) {
                for (int j = 0; j < kWaves; ++j) x += s_sum[(j * 16 * BT + b) * 8 + h - h0];
                x += s_odd[i];
            }
            out[i] = x;
        }
    }
}

// ---------------------------------------------------------------- backward, by source
// Bound as the pass by target, with q's and g's rows for k's and v's and 16 bytes of statistics for
// each edge and head: of shared heads as many rows as q has.  3.0M edges of 8 heads of 32: 336 us, at
// 48 % of the vector units and 42 % of the L1's cycles; 7.8M edges of 8 heads over 2: 973 us, at 48 % and
// 45 %.  (These times are a profile's, which are the longer ones.)
// (waves: the whole backward pass, 8 heads of 32: 733 us with 1, 601 with 2, 1518 with 3; 4 heads of
// 16: 233 us with 2, 222 with 3, 398 with 4)
constexpr int waves_of_kv(int NT) { return NT == 2 ? 2 : 3; }

__device__ __forceinline__ Lane lane_of_kv(const AttnArgs& a, const KvGroups& kg, int pass)
{
    Lane l;
    const int lane = threadIdx.x & 63;
    l.n = lane & 15;
    l.g = lane >> 4;
    const int k0 = (int)blockIdx.y * kg.heads, kn = min(kg.heads, a.kv_heads - k0), columns = kn * kg.shared;
    const int c = min(l.n & 7, columns - 1);
    l.real = (l.n & 7) < columns;
    l.source = k0 + c / kg.shared;
    l.kv0 = k0 * a.per + pass * kg.shared;  // the first of the gathered heads: of q
    l.head = l.source * a.per + pass * kg.shared + c % kg.shared;
    l.base = c * a.dim;
    l.wide = columns * a.dim;
    return l;
}

// dk and dv of one row for heads [k0, k0 + kn) of k, as forward_apart.
__device__ void backward_kv_apart(const AttnArgs& a, const Piece& p, int k0, int kn, const float* tab)
{
    const int lane = anew(threadIdx.x & 63), ch = 4 * lane;
    const bool wide = ch < a.dim;
    for (int c = k0; c < min(k0 + kn, a.kv_heads); ++c) {
        float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0}, dk[4] = {0, 0, 0, 0}, dv[4] = {0, 0, 0, 0};
        if (wide) {
            load4((const __bf16*)a.k + p.node * a.ldk + (int64_t)c * a.dim + ch, k);
            load4((const __bf16*)a.v + p.node * a.ldv + (int64_t)c * a.dim + ch, v);
        }
        for (int e = p.begin; e < p.end; ++e) {
            const int64_t t = a.L.idx[e];
            for (int h = c * a.per; h < (c + 1) * a.per; ++h) {
                const float b = tab[(int)a.L.bucket[e] * a.heads + h];
                if (b == -INFINITY) continue;
                const float4 st = a.stats[t * a.heads + h];
                float q[4] = {0, 0, 0, 0}, g[4] = {0, 0, 0, 0};
                if (wide) {
                    load4((const __bf16*)a.q + t * a.ldq + (int64_t)h * a.dim + ch, q);
                    load4((const __bf16*)a.g + t * a.ldg + (int64_t)h * a.dim + ch, g);
                }
                float s = 0, dp = 0;
                for (int i = 0; i < 4; ++i) {
                    s = fmaf(q[i], k[i], s);
                    dp = fmaf(g[i], v[i], dp);
                }
                const float pr = exp2_fast(fmaf(sum_lanes<64>(s), a.scale * kLog2e, b) - st.x) * st.y;
                const float ds = pr * (sum_lanes<64>(dp) - st.z);
                for (int i = 0; i < 4; ++i) {
                    dk[i] = fmaf(ds, q[i], dk[i]);
                    dv[i] = fmaf(pr, g[i], dv[i]);
                }
            }
        }
        if (!wide) continue;
        if (p.item >= 0) {
            store4(a.part_acc + (p.item * a.kv_heads + c) * a.dim + ch, dk);
            store4(a.part_acc2 + (p.item * a.kv_heads + c) * a.dim + ch, dv);
        } else {
            for (int i = 0; i < 4; ++i) dk[i] *= a.scale;
            store4((__bf16*)a.dk + ((int64_t)p.node * a.kv_heads + c) * a.dim + ch, dk);
            store4((__bf16*)a.dv + ((int64_t)p.node * a.kv_heads + c) * a.dim + ch, dv);
        }
    }
}

// x of the lane eight columns over, for columns 8 .. 15; the others keep theirs
__device__ __forceinline__ float twin_of(float x, bool low)
{
    const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
    return low ? y : x;
}

struct __attribute__((aligned(4))) Stats3 {
    float m, inv, delta;
};

// dk and dv: the roles of the two sides are swapped, rows of q and g are gathered against the
// spread k and v.  A target's (m, 1 / l, delta) come with it, by the lanes of the first eight
// columns; their twins take over what follows from them.
// (SHARED: several q heads of a head of k, whose sums are added up in LDS.)
template <int NT, bool BUCKETS, bool FAR, bool SHARED>
__global__ __launch_bounds__(64 * kWaves, waves_of_kv(NT)) void backward_kv_mfma_kernel(AttnArgs a, KvGroups kg)
{
    extern __shared__ float s_tab[];
    __shared__ u32x4 s_kk[kWaves][2 * NT * 64], s_vv[kWaves][2 * NT * 64];
    __shared__ __attribute__((aligned(16))) char s_x[kWaves][16 * kRowBytes<NT>];
    __shared__ float s_sum[SHARED ? kWaves : 1][2][SHARED ? 64 * NT : 1];
    __shared__ int s_any;
    const bool takes_out = stage_table<BUCKETS>(a, s_tab, &s_any);
    const float scale2 = a.scale * kLog2e;
    const Walk w = walk_of(a.L, kWaves);
    if (w.at >= w.end) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    u32x4* my_k = s_kk[wave] + lane;
    u32x4* my_v = s_vv[wave] + lane;
    char* my_x = s_x[wave];
    float* sum_k = s_sum[SHARED ? wave : 0][0];
    float* sum_v = s_sum[SHARED ? wave : 0][1];
    const int k0 = (int)blockIdx.y * kg.heads, out_wide = min(kg.heads, a.kv_heads - k0) * a.dim;
    const int out_head = 2 * lane / a.dim;
    const Lane l0 = lane_of_kv(a, kg, 0);
    Spread<NT> k, v;
    auto load_row = [&](const Piece& of, const Lane& l) {
        k.load((const __bf16*)a.k + max(of.node, 0) * a.ldk, a.kv_heads, l, a.dim);
        v.load((const __bf16*)a.v + max(of.node, 0) * a.ldv, a.kv_heads, l, a.dim);
    };
    auto put_row = [&] {
        k.put(my_k);
        v.put(my_v);
    };
    Piece p = piece_from(a.L, w, w.at, bounds_at(a.L, w, w.at));
    Piece next = piece_from(a.L, w, w.at + w.step, bounds_at(a.L, w, w.at + w.step));
    Block<FAR> block = block_at<BUCKETS, FAR>(a.L, p.begin, p.end);
    if (!SHARED) {
        load_row(p, l0);
        put_row();
    }
    for (int64_t u = w.at; u < w.end; u += w.step) {
        Bounds later;
        bool redo = false;
        float rk[2] = {0, 0}, rv[2] = {0, 0};  // channels 2 lane, 2 lane + 1 of the group's heads of k
        for (int pass = 0; pass < (SHARED ? kg.passes : 1); ++pass) {
            const Lane l = SHARED ? lane_of_kv(a, kg, pass) : l0;
            const uint32_t lane_at = lane_bytes<NT>(l);
            const char* qb = (const char*)a.q + 2 * l.kv0 * a.dim;
            const char* gb = (const char*)a.g + 2 * l.kv0 * a.dim;
            if (SHARED) {
                load_row(p, l);
                put_row();
            }
            f32x4 acc_k[kV<NT>], acc_v[kV<NT>];
            float odd;
            auto row = [&](auto apart) {
                constexpr bool APART = decltype(apart)::value;
#pragma unroll
                for (int i = 0; i < kV<NT>; ++i) acc_k[i] = acc_v[i] = f32x4{0, 0, 0, 0};
                odd = 0;
                int e0 = p.begin;
                do {
                    const int n = p.end - e0;
                    const Step<FAR> st = step_of<BUCKETS, FAR>(block, l);
                    VChunk<NT> q[8], g[8];
                    Stats3 of[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) q[x] = load_edge<NT, FAR>(qb, st.edge[x].node, a.ldq, lane_at);
#pragma unroll
                    for (int x = 0; x < 8; ++x) g[x] = load_edge<NT, FAR>(gb, st.edge[x].node, a.ldg, lane_at);
                    if (l.n < 8) {
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            of[x] = *(const Stats3*)((const char*)a.stats +
                                                     (row_at<FAR>(st.edge[x].node, 16 * a.heads) + 16 * l.head));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    const bool again = SHARED && n <= 32 && pass + 1 < kg.passes;
                    block = block_at<BUCKETS, FAR>(a.L, n > 32 ? e0 + 32 : again ? p.begin : next.begin,
                                                   n > 32 || again ? p.end : next.end);
                    later = bounds_at(a.L, w, u + 2 * w.step);
                    __builtin_amdgcn_sched_barrier(0);
                    const f32x4 qk[2] = {products<NT, APART>(my_x, l, a.dim, my_k, q, 0),
                                         products<NT, APART>(my_x, l, a.dim, my_k, q, 1)};
                    const f32x4 gv[2] = {products<NT, APART>(my_x, l, a.dim, my_v, g, 0),
                                         products<NT, APART>(my_x, l, a.dim, my_v, g, 1)};
                    float s[8], pr[8], ds[8];
                    logits<BUCKETS>(a, l, st, qk, n, scale2, takes_out, s_tab, s);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        pr[x] = s[x] == -INFINITY ? 0.0f : exp2_fast(s[x] - of[x].m) * of[x].inv;
                        ds[x] = s[x] == -INFINITY ? 0.0f : pr[x] * (gv[x / 4][x % 4] - of[x].delta);
                        pr[x] = twin_of(pr[x], l.n >= 8);
                        ds[x] = twin_of(ds[x], l.n >= 8);
                        odd = fmaf(0.0f, ds[x], odd);
                    }
                    if (BUCKETS && takes_out) {
                        keep_branch();
                        redo |= hide<NT>(l, s, q);
                        redo |= hide<NT>(l, s, g);
                    }
                    const bf16x8 weight = two_parts(pr, l.n >= 8 ? -1.0f : 0.0f);
                    if constexpr (APART) {  // infinities of g meet weights that are whole
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (edge_of(l, x) >= n) g[x] = VChunk<NT>{};
                        const bf16x8 whole = above_zero(pr);
#pragma unroll
                        for (int i = 0; i < kV<NT>; ++i) {
                            const bf16x8 gi = turned(g, i);
                            acc_v[i] = mfma(only<true>(gi), weight, acc_v[i]);
                            acc_v[i] = mfma(only<false>(gi), whole, acc_v[i]);
                            __builtin_amdgcn_sched_barrier(0);  // (one at a time: few registers)
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kV<NT>; ++i) acc_v[i] = mfma(turned(g, i), weight, acc_v[i]);
                    }
                    if constexpr (APART) {  // those of ds have no parts
                        bf16x8 vast;
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const bool is = isinf(ds[x]);
                            vast[x] = (__bf16)(is ? ds[x] : 0.0f);
                            ds[x] = is ? 0.0f : ds[x];
                        }
#pragma unroll
                        for (int i = 0; i < kV<NT>; ++i) {
                            acc_k[i] = mfma(turned(q, i), vast, acc_k[i]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                    const bf16x8 change = two_parts(ds, l.n >= 8 ? -1.0f : 0.0f);
#pragma unroll
                    for (int i = 0; i < kV<NT>; ++i) acc_k[i] = mfma(turned(q, i), change, acc_k[i]);
                    e0 += 32;
                } while (e0 < p.end);
            };
            row(std::false_type{});
            if (__builtin_expect(__any(odd != 0.0f), 0)) {  // (a NaN)
                keep_branch();
                block = block_at<BUCKETS, FAR>(a.L, p.begin, p.end);
                row(std::true_type{});
            }
            if (!SHARED) load_row(next, l);
            if (p.begin == p.end) {
                keep_branch();
#pragma unroll
                for (int i = 0; i < kV<NT>; ++i) acc_k[i] = acc_v[i] = f32x4{0, 0, 0, 0};
            }
            if constexpr (SHARED) {
                each_chunk<NT>(l, a.dim, acc_k, [&](float (&x)[8], int ch) { store8(sum_k + l.base + ch, x); });
                each_chunk<NT>(l, a.dim, acc_v, [&](float (&x)[8], int ch) { store8(sum_v + l.base + ch, x); });
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (2 * lane < out_wide) {
                    const int at = 2 * lane + out_head * (kg.shared - 1) * a.dim;
                    for (int i = 0; i < kg.shared; ++i) {
                        const float2 xk = *(const float2*)(sum_k + at + i * a.dim), xv = *(const float2*)(sum_v + at + i * a.dim);
                        rk[0] += xk.x;
                        rk[1] += xk.y;
                        rv[0] += xv.x;
                        rv[1] += xv.y;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            } else if (p.node >= 0 && !__any(redo)) {
                const int64_t at = ((p.item >= 0 ? p.item : (int64_t)p.node) * a.kv_heads + l.source) * a.dim;
                each_chunk<NT>(l, a.dim, acc_k, [&](float (&x)[8], int ch) {
                    if (p.item >= 0) {
                        store8(a.part_acc + at + ch, x);
                        return;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] *= a.scale;
                    store8((__bf16*)a.dk + at + ch, x);
                });
                each_chunk<NT>(l, a.dim, acc_v, [&](float (&x)[8], int ch) {
                    if (p.item >= 0) store8(a.part_acc2 + at + ch, x);
                    else store8((__bf16*)a.dv + at + ch, x);
                });
            }
        }
        if (__any(redo) && p.node >= 0) {
            backward_kv_apart(a, p, k0, kg.heads, s_tab);
        } else if (SHARED && p.node >= 0 && 2 * lane < out_wide) {
            if (p.item >= 0) {
                const int64_t at = (p.item * a.kv_heads + k0) * a.dim + 2 * lane;
                *(float2*)(a.part_acc + at) = make_float2(rk[0], rk[1]);
                *(float2*)(a.part_acc2 + at) = make_float2(rv[0], rv[1]);
            } else {
                const int64_t at = ((int64_t)p.node * a.kv_heads + k0) * a.dim + 2 * lane;
                *(bf16x2*)((__bf16*)a.dk + at) = bf16x2{(__bf16)(rk[0] * a.scale), (__bf16)(rk[1] * a.scale)};
                *(bf16x2*)((__bf16*)a.dv + at) = bf16x2{(__bf16)rv[0], (__bf16)rv[1]};
            }
        }
        if (!SHARED) put_row();
        p = next;
        next = piece_from(a.L, w, u + 2 * w.step, later);
    }
}

// ---------------------------------------------------------------- host
template <typename F>
void flag(bool x, F&& f)
{
    if (x) f(std::true_type{});
    else f(std::false_type{});
}
template <typename F>
void by_tiles(int tiles, F&& f)
{
    if (tiles == 1) f(std::integral_constant<int, 1>{});
    else f(std::integral_constant<int, 2>{});
}

// Whether the offset of a row (`bytes` long, of `rows`) can pass what 24-bit products of 32 bits
// hold; with as many nodes, an index leaves no room for a bucket either.
bool is_far(int64_t rows, int64_t bytes) { return rows >= 1 << 24 || bytes >= 1 << 24 || bytes * rows >= 1ll << 32; }

// A wave for each row (or part) of each group of heads, up to what the card holds at once (a
// workgroup has a wave on each SIMD of its CU).
dim3 grid_of(const AttnArgs& a, int groups, int per_simd)
{
    const int64_t rows = a.L.n_items + a.L.n_rows, most = std::max(1, 256 * per_simd / groups);
    return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((rows + kWaves - 1) / kWaves, most)), (unsigned)groups);
}

}  // namespace

void forward_mfma(const AttnArgs& a, hipStream_t s)
{
    const HeadGroups hg = head_groups(a.heads, a.per, a.dim);
    const bool far = is_far(a.n_nodes, 2 * std::max(a.ldk, a.ldv));
    by_tiles(hg.tiles, [&](auto nt) {
        flag(a.table != nullptr, [&](auto buckets) {
            flag(far, [&](auto is) {
                constexpr int NT = decltype(nt)::value;
                hipLaunchKernelGGL((forward_mfma_kernel<NT, decltype(buckets)::value, decltype(is)::value>),
                                   grid_of(a, hg.groups, waves_of(NT)), dim3(64 * kWaves),
                                   4 * (size_t)a.n_buckets * a.heads, s, a, hg);
            });
        });
    });
}

int backward_q_mfma(const AttnArgs& a, hipStream_t s)
{
    const HeadGroups hg = head_groups(a.heads, a.per, a.dim);
    const bool far = is_far(a.n_nodes, 2 * std::max(a.ldk, a.ldv));
    const int bucket_tiles = a.table ? (a.n_buckets + 15) / 16 : 0;
    int parts = 0;
    auto launch = [&](auto nt, auto bt, auto is) {
        constexpr int NT = decltype(nt)::value, BT = decltype(bt)::value;
        const dim3 grid = grid_of(a, hg.groups, waves_of_q(NT));
        parts = (int)(grid.x * grid.y);
        const size_t lds = 4 * (2 * (size_t)a.n_buckets * a.heads + kWaves * 16 * BT * 8);
        hipLaunchKernelGGL((backward_q_mfma_kernel<NT, BT, decltype(is)::value>), grid, dim3(64 * kWaves), lds, s, a, hg);
    };
    by_tiles(hg.tiles, [&](auto nt) {
        flag(far, [&](auto is) {
            if (bucket_tiles == 0) launch(nt, std::integral_constant<int, 0>{}, is);
            else if (bucket_tiles <= 2) launch(nt, std::integral_constant<int, 2>{}, is);
            else if (bucket_tiles <= 4) launch(nt, std::integral_constant<int, 4>{}, is);
            else launch(nt, std::integral_constant<int, 8>{}, is);
        });
    });
    return parts;
}

void backward_kv_mfma(const AttnArgs& a, hipStream_t s)
{
    const KvGroups kg = kv_groups(a.kv_heads, a.per, a.dim);
    const bool far = is_far(a.n_targets, std::max(2 * std::max(a.ldq, a.ldg), (int64_t)16 * a.heads)) || a.n_nodes >= 1 << 24;
    by_tiles(kg.tiles, [&](auto nt) {
        flag(a.table != nullptr, [&](auto buckets) {
            flag(far, [&](auto is) {
                constexpr int NT = decltype(nt)::value;
                flag(a.per > 1, [&](auto shared) {
                    hipLaunchKernelGGL((backward_kv_mfma_kernel<NT, decltype(buckets)::value, decltype(is)::value,
                                                                decltype(shared)::value>),
                                       grid_of(a, kg.groups, waves_of_kv(NT)), dim3(64 * kWaves),
                                       4 * (size_t)a.n_buckets * a.heads, s, a, kg);
                });
            });
        });
    });
}

}  // namespace dg
