// dg_grouped.hip -- linear maps whose weights go by group, ragged rows: forward and backward.
//
//   y[i] = W[g(i)] x[i] + b[g(i)]        rows of a group follow each other
//   dx[i] = W[g(i)]^T dy[i]   dW[g] = sum_{i in g} dy[i] x[i]^T   db[g] = sum_{i in g} dy[i]
// and with an activation f and a residual r, in the epilogue of the same product (z is y above)
//   y[i] = f(z[i]) + r[i]     dz[i] = dy[i] f'(z[i]), which takes dy's place above     dr = dy
// In bfloat16 dz goes on as two of them, its rounding and what that left (16 bits and their sign), and the products
// that take it sum over both: gradients are then as near to 64 bits as their own rounding (0.0017 of their norm; with dz
// rounded to one 0.0024, and a training step of 128 groups of 250 rows of 256 by 256 in 117 us, with two 143).
//
// Tiles of 128 x 128 on the matrix units, 32 x 32 a step, sums in 32 bits.  Both operands pass
// through LDS in rows of 128 bytes along the summed index (64 bfloat16 or 32 float), in chunks
// of 16 bytes that are swapped within a row so that neither the rows' writes nor the matrix
// operands' reads meet on a bank.  An operand that lies the other way in memory (W for dx, both
// for dW) is turned in registers on its way, a block of one chunk squared a time.  Half of the
// workgroup stages each operand: eight 16-byte loads a thread, in flight while the previous
// slab is multiplied.  The group's row count is not a multiple of a tile: rows past it are
// zeros in LDS and are not stored.
//
// In bfloat16, widths of 64 to 512 make these products bound by memory more than by arithmetic: a row
// tile's workgroup takes all its column tiles in turn, so x is read once from HBM, and the
// workgroups of an XCD hold neighbouring rows, whose weights then stay in its L2.
#include <hip/hip_runtime.h>
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

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

inline size_t al(size_t x) { return (x + 255) & ~(size_t)255; }

constexpr int kTile = 128;
constexpr int kRowBytes = 128;                   // of a slab's row in LDS
constexpr int kSlabBytes = kTile * kRowBytes;    // of one operand
constexpr int kXcds = 8;
constexpr int64_t kMaxGroups = 1 << 20;

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);  // elements of 16 bytes
template <typename T>
constexpr int kSlab = kRowBytes / (int)sizeof(T);  // summed indices of a slab

struct Args {
    const void* a;  // [rows, depth] (forward, dx); dy (dW)
    const void* a_low;  // what is added to it, where it comes in two parts
    const void* b;  // weights [groups, ...]; x (dW)
    const void* bias;
    void* out;
    void* out_low;    // (dz) what its rounding left, or NULL
    const void* aux;  // of out's layout: the residual, or dy (dz)
    int act;
    const int64_t* sizes;
    int64_t rows, groups;
    int cols, depth;  // of the result and of the sum (dW: the result is [cols = N, K = depth])
    // dW
    void* dbias;
    float* part;
    float* part_bias;
    int64_t chunk;  // rows of an item
};

// 16 bytes from an address aligned to the element alone (gfx950 reads any alignment).
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p)
{
    struct __attribute__((packed, aligned(2))) U { u32x4 v; };
    return ((const U*)p)->v;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, u32x4 v)
{
    struct __attribute__((packed, aligned(2))) U { u32x4 v; };
    ((U*)p)->v = v;
}

// The first n elements of a chunk (the rest zeros); n >= kChunk: all.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p, int n)
{
    if (n >= kChunk<T>) return load16(p);
    u32x4 v = {0, 0, 0, 0};
    if (n > 0) {
        if constexpr (sizeof(T) == 4) {
            for (int i = 0; i < 4; ++i)
                if (i < n) v[i] = ((const uint32_t*)p)[i];
        } else {
            for (int i = 0; i < 8; ++i)
                if (i < n) v[i / 2] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i % 2));
        }
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, u32x4 v, int n)
{
    if (n >= kChunk<T>) {
        store16(p, v);
    } else if constexpr (sizeof(T) == 4) {
        for (int i = 0; i < 4; ++i)
            if (i < n) ((uint32_t*)p)[i] = v[i];
    } else {
        for (int i = 0; i < 8; ++i)
            if (i < n) ((uint16_t*)p)[i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
    }
}

__device__ __forceinline__ int swapped(int row, int chunk) { return chunk ^ ((row ^ (row >> 3)) & 7); }

// One thread's eight 16-byte loads of a slab of an operand: `n` of its rows and `c_n` summed
// indices from c0 are real.  TURNED: memory holds [summed][row], else [row][summed].
template <typename T, bool TURNED, int ROWS = kTile>
struct Stage {
    static constexpr int N = ROWS / 16, R = TURNED && N < kChunk<T> ? kChunk<T> : N;
    static __device__ __forceinline__ void load(u32x4 (&r)[R], const T* p, int64_t ld, int n, int c0, int c_n, int t)
    {
        constexpr int C = kChunk<T>;
        if constexpr (!TURNED) {
            const int chunk = t % 8, left = c_n - (c0 + chunk * C);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = t / 8 + 16 * i;
                r[i] = load_chunk(p + row * ld + c0 + chunk * C, row < n ? left : 0);
            }
        } else {
            constexpr int across = ROWS / C;
#pragma unroll
            for (int b = 0; b < (N + C - 1) / C; ++b) {
                const int id = t + 128 * b, jb = id % across, cb = id / across;
                if (N < C && cb >= 8) break;  // (half of the threads have a block)
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const int c = c0 + cb * C + i;
                    r[b * C + i] = load_chunk(p + c * ld + jb * C, c < c_n ? n - jb * C : 0);
                }
            }
        }
    }
    static __device__ __forceinline__ void store(const u32x4 (&r)[R], char* lds, int t)
    {
        constexpr int C = kChunk<T>;
        if constexpr (!TURNED) {
            const int chunk = t % 8;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = t / 8 + 16 * i;
                *(u32x4*)(lds + row * kRowBytes + swapped(row, chunk) * 16) = r[i];
            }
        } else {
            constexpr int across = ROWS / C;
#pragma unroll
            for (int b = 0; b < (N + C - 1) / C; ++b) {
                const int id = t + 128 * b, jb = id % across, cb = id / across;
                if (N < C && cb >= 8) break;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    u32x4 v;
                    if constexpr (sizeof(T) == 4) {
                        for (int d = 0; d < 4; ++d) v[d] = r[b * 4 + d][j];
                    } else {  // pairs of rows, the low or the high halves of their words
                        for (int d = 0; d < 4; ++d)
                            v[d] = __builtin_amdgcn_perm(r[2 * d + 1][j / 2], r[2 * d][j / 2],
                                                         j % 2 ? 0x07060302u : 0x05040100u);
                    }
                    const int row = jb * C + j;
                    *(u32x4*)(lds + row * kRowBytes + swapped(row, cb) * 16) = v;
                }
            }
        }
    }
};

// acc[i][j] += the wave's 64 x 64 products of one slab: rows of `lo` by columns of `hi`.
template <typename T>
__device__ __forceinline__ void multiply(const char* rows, const char* cols, int w_row, int w_col, int lane,
                                         f32x16 (&acc)[2][2])
{
    const int x = lane & 31, half = lane >> 5;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        u32x4 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int ra = w_row + 32 * i + x, rb = w_col + 32 * i + x;
            a[i] = *(const u32x4*)(rows + ra * kRowBytes + swapped(ra, 2 * s + half) * 16);
            b[i] = *(const u32x4*)(cols + rb * kRowBytes + swapped(rb, 2 * s + half) * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if constexpr (sizeof(T) == 2) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[i]),
                                                                        __builtin_bit_cast(bf16x8, b[j]), acc[i][j], 0, 0, 0);
                } else {
                    // the summed indices of a step: element c of both halves' chunks
                    const f32x4 fa = __builtin_bit_cast(f32x4, a[i]), fb = __builtin_bit_cast(f32x4, b[j]);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[c], fb[c], acc[i][j], 0, 0, 0);
                }
            }
    }
}

// What becomes of a result: nothing, f(z) + r, or dy f'(z).
enum { kPlain, kApply, kSlope };

// f(z) (SLOPE: its derivative), in some ten to thirty instructions, which the library's functions would take
// twice.  silu: its slope from exp(-|z|), which neither overflows nor loses 1 - s.  gelu: the normal distribution's share
// beyond |z| is exp(-z^2 / 2) t Q(t) with t = 1 / (1 + 0.318 |z|), so that it keeps its digits far out; Q is a
// least-maximum fit of degree 9 to it in relative error (0.55 2^-24, 5.1 2^-24 as evaluated near zero; further out the
// roundings of z^2 count, up to 1.5 z^2 2^-24 of that share: 30 2^-24 at 3 to 6, 80 to 10, where the share is 1e-3 and less).
template <int ACT, bool SLOPE>
__device__ __forceinline__ float activation(float z)
{
    if constexpr (ACT == DG_ACT_SILU) {
        // (below -87 the reciprocal of what has no 32-bit inverse is 0: values beneath 1e-36 are)
        if constexpr (!SLOPE) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
        const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
        return (z < 0.0f ? e * r : r) * fmaf(z, z < 0.0f ? r : e * r, 1.0f);
    }
    if constexpr (ACT == DG_ACT_GELU) {
        const float e = __builtin_amdgcn_exp2f(-0.72134752f * (z * z)), t = __builtin_amdgcn_rcpf(fmaf(0.318f, fabsf(z), 1.0f));
        float q = -0.020624028518795967f;
        q = fmaf(q, t, 0.09520687907934189f);
        q = fmaf(q, t, -0.15045107901096344f);
        q = fmaf(q, t, 0.07162534445524216f);
        q = fmaf(q, t, -0.011254116892814636f);
        q = fmaf(q, t, 0.06007798761129379f);
        q = fmaf(q, t, 0.08761146664619446f);
        q = fmaf(q, t, 0.11408133804798126f);
        q = fmaf(q, t, 0.1268625557422638f);
        q = fmaf(q, t, 0.12686364352703094f);
        const float beyond = e * (t * q), share = z < 0.0f ? beyond : 1.0f - beyond;
        if constexpr (!SLOPE) return z * share;
        return fmaf(z * e, 0.39894228f, share);
    }
    return SLOPE ? 1.0f : z;
}
// N results at once (the branch is the same for the whole grid, and the N chains overlap).
template <int EPI, int ACT, int N>
__device__ __forceinline__ void finish_as(bool more, float (&z)[N], const float (&aux)[N])
{
    for (int i = 0; i < N; ++i) z[i] = activation<ACT, EPI == kSlope>(z[i]);
    if (EPI == kSlope)
        for (int i = 0; i < N; ++i) z[i] *= aux[i];
    else if (more)
        for (int i = 0; i < N; ++i) z[i] += aux[i];
}
template <int EPI, int N>
__device__ __forceinline__ void finish(int act, bool more, float (&z)[N], const float (&aux)[N])
{
    if (act == DG_ACT_SILU) finish_as<EPI, DG_ACT_SILU>(more, z, aux);
    else if (act == DG_ACT_GELU) finish_as<EPI, DG_ACT_GELU>(more, z, aux);
    else finish_as<EPI, DG_ACT_NONE>(more, z, aux);
}

// Sums that begin with their columns' bias, 64 columns from c0 on.
template <typename T>
__device__ __forceinline__ void begin_with(f32x16 (&acc)[2][2], const T* bias, int c0, int cols, int lane)
{
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int c = c0 + 32 * i + 8 * (q / 4) + 4 * (lane >> 5) + q % 4;
            acc[i][0][q] = acc[i][1][q] = c < cols ? (float)bias[c] : 0.0f;
        }
}

// What a rounding to bfloat16 leaves (of what is not finite then: nothing, or it would make a NaN of an infinity).
__device__ __forceinline__ float left_over(float v)
{
    const float h = (float)(__bf16)v;
    return fabsf(h) <= 3.4e38f ? v - h : 0.0f;
}

// A wave's 64 x 64 of the result to memory: in the accumulators a lane holds four neighbouring
// columns of one row, which LDS turns into whole chunks of rows.  `s` is the wave's own.  LOW: what the rounding leaves.
constexpr int kOutRows = 32;
template <typename T>
constexpr int kOutPitch = 64 * (int)sizeof(T) + 16;

template <typename T, int EPI = kPlain, bool LOW = false>
__device__ __forceinline__ void write_out(const f32x16 (&acc)[2][2], char* s, int lane, T* out, int64_t ld, int n_rows,
                                          int n_cols, const T* bias, const T* aux = nullptr, int act = 0)
{
    const int x = lane & 31, half = lane >> 5;
    constexpr int chunks = 64 / kChunk<T>;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = 32 * i + 8 * q + 4 * half;
                f32x4 v;
                for (int c = 0; c < 4; ++c) {
                    v[c] = acc[i][j][4 * q + c];
                    if (bias && col + c < n_cols) v[c] += (float)bias[col + c];
                }
                if constexpr (EPI != kPlain) {
                    float z[4], r[4] = {};
                    for (int c = 0; c < 4; ++c) z[c] = v[c];
                    if (aux && 32 * j + x < n_rows)
                        for (int c = 0; c < 4; ++c)
                            if (col + c < n_cols) r[c] = (float)aux[(int64_t)(32 * j + x) * ld + col + c];
                    finish<EPI>(act, aux != nullptr, z, r);
                    for (int c = 0; c < 4; ++c) v[c] = z[c];
                }
                if constexpr (sizeof(T) == 4) {
                    *(f32x4*)(s + x * kOutPitch<T> + col * 4) = v;
                } else {
                    __attribute__((ext_vector_type(4))) __bf16 y;
                    for (int c = 0; c < 4; ++c) y[c] = (__bf16)(LOW ? left_over(v[c]) : v[c]);
                    *(decltype(y)*)(s + x * kOutPitch<T> + col * 2) = y;
                }
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < kOutRows * chunks / 64; ++k) {
            const int id = k * 64 + lane, row = id / chunks, c = id % chunks;
            if (32 * j + row < n_rows && c * kChunk<T> < n_cols)
                store_chunk(out + (int64_t)(32 * j + row) * ld + c * kChunk<T>,
                            *(const u32x4*)(s + row * kOutPitch<T> + c * 16), n_cols - c * kChunk<T>);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Pieces (row tiles, or dW's items) of the groups.
struct Cuts {
    int64_t unit;  // rows of a piece
    int least;     // pieces of an empty group
    __device__ __forceinline__ int64_t of(int64_t size) const
    {
        const int64_t n = (size + unit - 1) / unit;
        return n < least ? least : n;
    }
};

struct Place {
    int64_t group, piece;  // the piece's number in its group
    int64_t row, size;     // the group's first row, its rows
    int64_t many;          // pieces of the groups before that have more than one
    int64_t split;         // those groups' number
};
constexpr int kSplitBit = 40;  // in the scan: groups above pieces (2^20 groups, 2^40 rows)

// A group's rows, were there enough: a negative size is empty, none is larger than all rows.
__device__ __forceinline__ int64_t claim(const Args& a, int64_t g)
{
    return g < a.groups ? min(max(a.sizes[g], (int64_t)0), a.rows) : 0;
}

// One pass of the workgroup (256 threads, or 512) over the groups: all pieces and rows, and where `found`
// holds, of (its first piece, its pieces, split groups before), that group's place (piece: its
// first piece).
template <int WAVES, typename F>
__device__ __forceinline__ void pass(const Args& a, const Cuts& c, int64_t* s_w, Place* s_p, int64_t& pieces, int64_t& rows,
                                     F&& found)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    pieces = 0;
    int64_t claimed = 0, many = 0;
    for (int64_t g0 = 0; g0 < a.groups; g0 += 64 * WAVES) {
        const int64_t g = g0 + threadIdx.x, n = claim(a, g);
        int64_t in = n;
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up(in, o, 64);
            if (lane >= o) in += y;
        }
        if (lane == 63) s_w[w] = in;
        __syncthreads();
        int64_t row = claimed + in - n;
        for (int i = 0; i < WAVES; ++i) {
            if (i < w) row += s_w[i];
            claimed += s_w[i];
        }
        const int64_t size = min(n, max(a.rows - row, (int64_t)0));
        const int64_t p = g < a.groups ? c.of(size) : 0, m = p > 1 ? p | 1ll << kSplitBit : 0;
        int64_t ip = p, im = m;
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(ip, o, 64), z = __shfl_up(im, o, 64);
            if (lane >= o) {
                ip += x;
                im += z;
            }
        }
        if (lane == 63) {
            s_w[WAVES + w] = ip;
            s_w[2 * WAVES + w] = im;
        }
        __syncthreads();
        int64_t bp = pieces + ip - p, bm = many + im - m;
        for (int i = 0; i < WAVES; ++i) {
            if (i < w) {
                bp += s_w[WAVES + i];
                bm += s_w[2 * WAVES + i];
            }
            pieces += s_w[WAVES + i];
            many += s_w[2 * WAVES + i];
        }
        if (g < a.groups && found(bp, p, bm >> kSplitBit))
            *s_p = Place{g, bp, min(row, a.rows), size, bm & ((1ll << kSplitBit) - 1), bm >> kSplitBit};
    }
    __syncthreads();
    rows = min(claimed, a.rows);
}

// The place of piece `at` (there is one).
template <int WAVES>
__device__ __forceinline__ Place locate(const Args& a, const Cuts& c, int64_t at, int64_t* s_w, Place* s_p)
{
    int64_t pieces, rows;
    pass<WAVES>(a, c, s_w, s_p, pieces, rows, [&](int64_t first, int64_t n, int64_t) { return n > 0 && at >= first && at < first + n; });
    Place p = *s_p;
    p.piece = at - p.piece;
    return p;
}

__device__ __forceinline__ int64_t scalar64(int64_t x)
{
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// The first group after `group` that claims rows (there is one), its first row given; `size`: its rows.
// 64 groups a load: a run of empty ones costs little.
__device__ __forceinline__ int64_t next_group(const Args& a, int64_t group, int64_t row, int64_t& size)
{
    for (++group; group < a.groups; group += 64) {
        const int64_t n = claim(a, group + (threadIdx.x & 63));
        const unsigned long long some = __ballot(n > 0);
        if (!some) continue;
        const int first = __builtin_ctzll(some);
        size = min(scalar64(__shfl(n, first, 64)), max(a.rows - row, (int64_t)0));
        return group + first;
    }
    size = 0x7fffffffffffffffll;  // (not reached: ends the caller's search)
    return a.groups - 1;
}

// This workgroup's place in an order in which an XCD's workgroups are neighbours.
__device__ __forceinline__ int64_t xcd_order(int64_t b, int64_t n)
{
    if (n % kXcds) return b;
    return b % kXcds * (n / kXcds) + b / kXcds;
}

// result[i, j] = sum_c a[i, c] W(j, c) (+ bias[j]), W(j, c) at weight[g][j][c], or (DX) [g][c][j].  PARTS: of a, each
// with all of the summed indices, one part after the other.
template <typename T, bool DX, int EPI, int PARTS>
__global__ __launch_bounds__(256, 2) void rows_kernel(Args a)
{
    __shared__ __attribute__((aligned(16))) char s_a[kSlabBytes], s_b[kSlabBytes];
    __shared__ __attribute__((aligned(16))) char s_out[4 * kOutRows * kOutPitch<T>];
    __shared__ int64_t s_w[12];
    __shared__ Place s_p;
    const Cuts cuts{kTile, 0};
    int64_t tiles, covered;
    pass<4>(a, cuts, s_w, &s_p, tiles, covered, [](int64_t, int64_t, int64_t) { return false; });
    const int col_tiles = (a.cols + kTile - 1) / kTile;
    const int64_t units = tiles * col_tiles, me = xcd_order(blockIdx.x, gridDim.x);
    int64_t u = units * me / gridDim.x;
    const int64_t end = units * (me + 1) / gridDim.x;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x % 128;
    const bool first_half = threadIdx.x < 128;
    if (u < end) {
        Place p = locate<4>(a, cuts, u / col_tiles, s_w, &s_p);
        int64_t group = scalar64(p.group), piece = scalar64(p.piece), row = scalar64(p.row), size = scalar64(p.size);
        const int slabs = (a.depth + kSlab<T> - 1) / kSlab<T>, all_slabs = PARTS * slabs;
        using SA = Stage<T, false>;
        using SB = Stage<T, DX>;
        u32x4 r[8];
        auto fetch = [&](int64_t uu, int slab) {
            const int col = (int)(uu % col_tiles) * kTile;
            const int64_t r0 = row + piece * kTile;
            const bool low = PARTS == 2 && slab >= slabs;
            if (low) slab -= slabs;
            if (first_half)
                SA::load(r, (const T*)(low ? a.a_low : a.a) + r0 * a.depth, a.depth,
                        (int)max((int64_t)0, min(min(size - piece * kTile, a.rows - r0), (int64_t)kTile)), slab * kSlab<T>,
                        a.depth, t);
            else {
                const T* wt = (const T*)a.b + group * a.cols * a.depth;
                if constexpr (DX)
                    SB::load(r, wt + col, a.cols, min(a.cols - col, kTile), slab * kSlab<T>, a.depth, t);
                else
                    SB::load(r, wt + (int64_t)col * a.depth, a.depth, min(a.cols - col, kTile), slab * kSlab<T>, a.depth, t);
            }
        };
        fetch(u, 0);
        while (u < end) {
            const int64_t my_row = row + piece * kTile, my_group = group;
            const int n_rows = (int)max((int64_t)0, min(min(size - piece * kTile, a.rows - my_row), (int64_t)kTile));
            const int col = (int)(u % col_tiles) * kTile;
            f32x16 acc[2][2] = {};
            if constexpr (EPI != kPlain)  // (as stream_kernel has it: the same bits)
                if (a.bias) begin_with(acc, (const T*)a.bias + my_group * a.cols, col + (w / 2) * 64, a.cols, lane);
            for (int slab = 0; slab < all_slabs; ++slab) {
                __syncthreads();
                if (first_half) SA::store(r, s_a, t);
                else SB::store(r, s_b, t);
                __syncthreads();
                if (slab + 1 < all_slabs) {
                    fetch(u, slab + 1);
                } else {  // the next unit's first slab
                    ++u;
                    if (u < end) {
                        if (u % col_tiles == 0) {
                            ++piece;
                            while (piece * kTile >= size) {  // (a later group has rows: u < end)
                                row += size;
                                piece = 0;
                                group = next_group(a, group, row, size);
                            }
                        }
                        fetch(u, 0);
                    }
                }
                multiply<T>(s_b, s_a, (w / 2) * 64, (w % 2) * 64, lane, acc);
            }
            const int c0 = col + (w / 2) * 64, r0 = (w % 2) * 64;
            const int64_t at = (my_row + r0) * a.cols + c0;
            write_out<T, EPI>(acc, s_out + w * kOutRows * kOutPitch<T>, lane, (T*)a.out + at, a.cols, n_rows - r0, a.cols - c0,
                              !DX && EPI == kPlain && a.bias ? (const T*)a.bias + my_group * a.cols + c0 : nullptr,
                              EPI != kPlain && a.aux ? (const T*)a.aux + at : nullptr, a.act);
            if constexpr (EPI == kSlope && sizeof(T) == 2)
                if (a.out_low)
                    write_out<T, EPI, true>(acc, s_out + w * kOutRows * kOutPitch<T>, lane, (T*)a.out_low + at, a.cols, n_rows - r0,
                                            a.cols - c0, nullptr, (const T*)a.aux + at, a.act);
        }
    }
    // rows of no group
    const int64_t from = min(covered, a.rows) * a.cols, all = a.rows * a.cols;
    for (int64_t i = from + blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll)
        ((T*)a.out)[i] = EPI == kApply && a.aux ? ((const T*)a.aux)[i] : (T)0.0f;
}

// The same for rows whose chunks of 16 bytes are whole, with at most 1 KB of summed indices: eight
// waves share a panel of W in LDS, PN columns by all summed indices, made once for all of the
// workgroup's rows of a group, and each streams strips of 32 rows through 8 KB of its own: 256
// bytes of each row a step, the next step's loads in flight while one is multiplied, and the
// strip's result back through the same 8 KB to whole rows.  No barrier but at a change of group.
// Loads and stores go through buffer descriptors of the strip: what lies outside reads as zero and
// is not written, so every step has the same instructions and the waits between them are counted.
// 2.2M rows of 128 by 128 in bfloat16: 232 us, 4.86 TB/s, what a copy reaches (4.9).  100,000 rows of
// 256 by 256 floats: 135 us, 97 TFLOP/s of the 153 that a product of 8192 cubed reaches.
// With an epilogue (200,003 rows of 256 by 512 in bfloat16, 16 groups; bytes at a copy's rate 60 us, products 44 at a
// library's): silu 105 us, gelu 138, a residual 117; in float silu 462, gelu 494.  864 rows, 8 groups: 8 us, in float 17.
// Four panels read x four times, from L2; the rest is instructions, 14 a value for silu and 25 for gelu, next to the
// products at two waves a SIMD (16 waves with panels half as wide: 168).
constexpr int kStreamWaves = 8;
constexpr int kStripRows = 32;
constexpr int kStreamRows = kStreamWaves * kStripRows;
constexpr int kStepBytes = 256;
constexpr int kOutside = 0x7ffffff0;

using Buffer = __amdgpu_buffer_rsrc_t;
__device__ __forceinline__ Buffer buffer_of(const void* p, int64_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)min(bytes, (int64_t)kOutside), 0x00020000);
}

template <typename T, bool DX, int PN, int EPI, int PARTS>
__global__ __launch_bounds__(64 * kStreamWaves) void stream_kernel(Args a, bool single)
{
    __shared__ __attribute__((aligned(16))) char s_panel[65536];
    __shared__ __attribute__((aligned(16))) char s_x[kStreamWaves][kStripRows * kStepBytes];
    __shared__ __attribute__((aligned(16))) float s_bias[EPI == kPlain ? 4 : PN];
    __shared__ int64_t s_w[3 * kStreamWaves];
    __shared__ Place s_p;
    constexpr int C = kChunk<T>, kStep = kStepBytes / (int)sizeof(T), kTiles = PN / 32;
    const Cuts cuts{kStreamRows, 0};
    const int panels = (a.cols + PN - 1) / PN;
    const int64_t me = xcd_order(blockIdx.x, gridDim.x), lane_of_work = me / panels, lanes_of_work = gridDim.x / panels;
    const int col = (int)(me % panels) * PN;
    // (with a workgroup for each tile there may be, the place of the tile comes from the same pass)
    int64_t tiles, covered;
    pass<kStreamWaves>(a, cuts, s_w, &s_p, tiles, covered, [&](int64_t first, int64_t n, int64_t) {
        return single && lane_of_work >= first && lane_of_work < first + n;
    });
    int64_t u = single ? lane_of_work : tiles * lane_of_work / lanes_of_work;
    const int64_t end = single ? min(u + 1, tiles) : lane_of_work < lanes_of_work ? tiles * (lane_of_work + 1) / lanes_of_work : u;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = lane & 31, half = lane >> 5, quarter = lane >> 4, chunk = lane & 15;
    char* my_x = s_x[w];
    if (u < end) {
        Place p = s_p;
        p.piece = u - p.piece;
        if (!single) p = locate<kStreamWaves>(a, cuts, u, s_w, &s_p);
        int64_t group = scalar64(p.group), piece = scalar64(p.piece), row = scalar64(p.row), size = scalar64(p.size);
        const int steps = (a.depth + kStep - 1) / kStep, slabs = (a.depth + kSlab<T> - 1) / kSlab<T>;
        const int64_t ld = (int64_t)a.depth * sizeof(T), ld_out = (int64_t)a.cols * sizeof(T);
        auto fill_panel = [&](int64_t g) {
            const T* wt = (const T*)a.b + g * a.cols * a.depth;
            __syncthreads();
            for (int s = threadIdx.x / 128; s < slabs; s += kStreamWaves / 2) {
                using S = Stage<T, DX, PN>;
                u32x4 st[S::R];
                const int t = threadIdx.x % 128;
                if constexpr (DX) S::load(st, wt + col, a.cols, min(a.cols - col, PN), s * kSlab<T>, a.depth, t);
                else S::load(st, wt + (int64_t)col * a.depth, a.depth, min(a.cols - col, PN), s * kSlab<T>, a.depth, t);
                S::store(st, s_panel + s * PN * kRowBytes, t);
            }
            if constexpr (EPI != kPlain)
                if ((int)threadIdx.x < PN)
                    s_bias[threadIdx.x] = a.bias && col + (int)threadIdx.x < a.cols
                                              ? (float)((const T*)a.bias)[g * a.cols + col + threadIdx.x] : 0.0f;
            __syncthreads();
        };
        // where a lane's operands of a slab lie: x's chunks 2 s + half of row x, the panel's of rows 32 t + x (whose
        // swap is that of row x, and another chunk's fourth for each second t)
        int at_x[4], at_w[2][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            at_x[s] = x * kStepBytes + ((2 * s + half) ^ (x & 15)) * 16;
            for (int t = 0; t < 2; ++t) at_w[t][s] = x * kRowBytes + swapped(32 * t + x, 2 * s + half) * 16;
        }
        // a lane loads a chunk of 16 bytes of each eighth row of 256: rows 4 i + quarter
        u32x4 r[8];
        auto fetch = [&](int64_t first_row, int n_rows, int step) {
            const bool low = PARTS == 2 && step >= steps;
            if (low) step -= steps;
            const Buffer b = buffer_of((const char*)(low ? a.a_low : a.a) + first_row * ld, n_rows * ld);
            const int at = step * kStepBytes + chunk * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                r[i] = __builtin_amdgcn_raw_buffer_load_b128(b, at < ld ? (4 * i + quarter) * (int)ld + at : kOutside, 0, 0);
        };
        auto rows_here = [&](int64_t r0) {  // of the wave's strip of this piece
            return (int)max((int64_t)0, min(min(size - piece * kStreamRows - w * kStripRows, a.rows - r0), (int64_t)kStripRows));
        };
        int64_t r0 = row + piece * kStreamRows + w * kStripRows;
        int n_rows = rows_here(r0);
        fetch(r0, n_rows, 0);
        fill_panel(group);
        while (u < end) {
            const int64_t my_row = r0, my_group = group;
            const int my_rows = n_rows;
            f32x16 acc[kTiles] = {};
            if constexpr (EPI != kPlain)  // (the bias is what the sums begin with: no instruction of its own)
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 f = *(const f32x4*)(s_bias + 32 * t + 8 * q + 4 * half);
                        for (int k = 0; k < 4; ++k) acc[t][4 * q + k] = f[k];
                    }
            for (int at_step = 0; at_step < PARTS * steps; ++at_step) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rr = 4 * i + quarter;
                    *(u32x4*)(my_x + rr * kStepBytes + (chunk ^ (rr & 15)) * 16) = r[i];
                }
                if (at_step + 1 < PARTS * steps) {
                    fetch(r0, n_rows, at_step + 1);
                } else {
                    ++u;
                    if (u < end) {
                        ++piece;
                        while (piece * kStreamRows >= size) {  // (a later group has rows: u < end)
                            row += size;
                            piece = 0;
                            group = next_group(a, group, row, size);
                        }
                        r0 = row + piece * kStreamRows + w * kStripRows;
                        n_rows = rows_here(r0);
                        fetch(r0, n_rows, 0);
                    }
                }
                const int step = PARTS == 2 && at_step >= steps ? at_step - steps : at_step;
                const char* panel = s_panel + step * 2 * PN * kRowBytes;
                const int inner = min(2, slabs - 2 * step);  // slabs of 128 bytes in this step
                for (int b = 0; b < inner; ++b)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const u32x4 v = *(const u32x4*)(my_x + (at_x[s] ^ b << 7));
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            const u32x4 y = *(const u32x4*)(panel + b * PN * kRowBytes + at_w[t & 1][s] + 32 * t * kRowBytes);
                            if constexpr (sizeof(T) == 2) {
                                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, y),
                                                                                 __builtin_bit_cast(bf16x8, v), acc[t], 0, 0, 0);
                            } else {
                                const f32x4 fy = __builtin_bit_cast(f32x4, y), fv = __builtin_bit_cast(f32x4, v);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(fy[k], fv[k], acc[t], 0, 0, 0);
                            }
                        }
                    }
            }
            if constexpr (EPI == kPlain) {
                // the strip's result, 256 bytes (or the panel's) of each row at once
                constexpr int kWide = PN * (int)sizeof(T) < kStepBytes ? PN : kStep, kPieces = PN / kWide, kChunks = kWide / C;
                const Buffer out = buffer_of((const char*)a.out + my_row * ld_out, my_rows * ld_out);
                const T* bias = !DX && a.bias ? (const T*)a.bias + my_group * a.cols + col : nullptr;
#pragma unroll
                for (int piece_at = 0; piece_at < kPieces; ++piece_at) {
#pragma unroll
                    for (int t = 0; t < kWide / 32; ++t)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int at = 32 * t + 8 * q + 4 * half, c = piece_at * kWide + at;
                            f32x4 v;
                            for (int k = 0; k < 4; ++k) v[k] = acc[piece_at * (kWide / 32) + t][4 * q + k];
                            if (bias && col + c < a.cols)
                                for (int k = 0; k < 4; ++k) v[k] += (float)bias[c + k];  // (whole chunks: four are there)
                            if constexpr (sizeof(T) == 4) {
                                *(f32x4*)(my_x + x * (kWide * 4) + ((at / 4) ^ (x & (kChunks - 1))) * 16) = v;
                            } else {
                                __attribute__((ext_vector_type(4))) __bf16 y;
                                for (int k = 0; k < 4; ++k) y[k] = (__bf16)v[k];
                                *(decltype(y)*)(my_x + x * (kWide * 2) + ((at / 8) ^ (x & (kChunks - 1))) * 16 + at % 8 * 2) = y;
                            }
                        }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int k = 0; k < kStripRows * kChunks / 64; ++k) {
                        const int id = k * 64 + lane, rr = id / kChunks, c = id % kChunks;
                        const int at = (col + piece_at * kWide) * (int)sizeof(T) + c * 16;
                        const u32x4 v = *(const u32x4*)(my_x + rr * (kWide * (int)sizeof(T)) + (c ^ (rr & (kChunks - 1))) * 16);
                        __builtin_amdgcn_raw_buffer_store_b128(v, out, at < ld_out ? rr * (int)ld_out + at : kOutside, 0, 0);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
            } else {
                // In 32 bits through the same 8 KB, 64 columns of each row at once, so that a lane has
                // whole chunks of rows, the same columns in each of them: residual (or dy) and
                // activation there, and one rounding.  The chunks of `aux` are under way meanwhile.
                constexpr int kWide = PN < 64 ? PN : 64, kPieces = PN / kWide, kChunks = kWide / C, kEach = kStripRows * kChunks / 64;
                const Buffer out = buffer_of((const char*)a.out + my_row * ld_out, my_rows * ld_out);
                const Buffer in = buffer_of((const char*)a.aux + my_row * ld_out, a.aux ? my_rows * ld_out : 0);
                const Buffer low = buffer_of((const char*)a.out_low + my_row * ld_out, a.out_low ? my_rows * ld_out : 0);
                const int c = lane % kChunks, r_first = lane / kChunks;
#pragma unroll
                for (int piece_at = 0; piece_at < kPieces; ++piece_at) {
                    const int first = col + piece_at * kWide + c * C;  // the lane's first column
                    const int at = first < a.cols ? first * (int)sizeof(T) : kOutside;
                    u32x4 aux[kEach];
#pragma unroll
                    for (int k = 0; k < kEach; ++k)
                        aux[k] = __builtin_amdgcn_raw_buffer_load_b128(in, at == kOutside ? at : (r_first + k * (64 / kChunks)) * (int)ld_out + at, 0, 0);
#pragma unroll
                    for (int t = 0; t < kWide / 32; ++t)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            f32x4 v;
                            for (int k = 0; k < 4; ++k) v[k] = acc[piece_at * (kWide / 32) + t][4 * q + k];
                            *(f32x4*)(my_x + x * (kWide * 4) + ((8 * t + 2 * q + half) ^ (x & (kWide / 4 - 1))) * 16) = v;
                        }
                    wave_sync();
#pragma unroll
                    for (int k = 0; k < kEach; ++k) {
                        const int rr = r_first + k * (64 / kChunks);
                        float v[C];
#pragma unroll
                        for (int h = 0; h < C / 4; ++h) {
                            const f32x4 f = *(const f32x4*)(my_x + rr * (kWide * 4) + ((c * (C / 4) + h) ^ (rr & (kWide / 4 - 1))) * 16);
                            for (int i = 0; i < 4; ++i) v[4 * h + i] = f[i];
                        }
                        float r[C];
                        for (int i = 0; i < C; ++i) {
                            const uint32_t word = aux[k][i * (int)sizeof(T) / 4];
                            r[i] = as_float(sizeof(T) == 4 ? word : i % 2 ? word & 0xffff0000u : word << 16);
                        }
                        finish<EPI>(a.act, a.aux, v, r);
                        u32x4 y;
                        if constexpr (sizeof(T) == 4) {
                            for (int i = 0; i < 4; ++i) y[i] = as_bits(v[i]);
                        } else {
                            bf16x8 f;
                            for (int i = 0; i < 8; ++i) f[i] = (__bf16)v[i];
                            y = __builtin_bit_cast(u32x4, f);
                        }
                        __builtin_amdgcn_raw_buffer_store_b128(y, out, at == kOutside ? at : rr * (int)ld_out + at, 0, 0);
                        if constexpr (EPI == kSlope && sizeof(T) == 2)
                            if (a.out_low) {
                                bf16x8 f;
                                for (int i = 0; i < 8; ++i) f[i] = (__bf16)left_over(v[i]);
                                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f), low,
                                                                       at == kOutside ? at : rr * (int)ld_out + at, 0, 0);
                            }
                    }
                    wave_sync();
                }
            }
            if (u < end && group != my_group) fill_panel(group);
        }
    }
    // rows of no group
    const int64_t from = min(covered, a.rows) * a.cols, all = a.rows * a.cols;
    for (int64_t i = from + blockIdx.x * (64ll * kStreamWaves) + threadIdx.x; i < all; i += gridDim.x * (64ll * kStreamWaves))
        ((T*)a.out)[i] = EPI == kApply && a.aux ? ((const T*)a.aux)[i] : (T)0.0f;
}

// dW[g][n][k] = sum_i dy[i, n] x[i, k] over an item's rows of a group, 128 x 128 of it; the
// first column tile's workgroups sum dy itself.  Groups of one item write their result,
// others partial sums that weight_join_kernel adds up in order.  128 groups of 250 rows, 256 by 512:
// 40 us, bound by the turning of both operands in registers (each is read twice to four times, from
// L2): 83 MB in and out, 2.1 TB/s.  PARTS of dy: its rows once for each, and x's again.
template <typename T, int PARTS>
__global__ __launch_bounds__(256, 2) void weight_kernel(Args a, int64_t max_items)
{
    __shared__ __attribute__((aligned(16))) char s_a[kSlabBytes], s_b[kSlabBytes];
    __shared__ __attribute__((aligned(16))) char s_out[4 * kOutRows * kOutPitch<T>];
    __shared__ int64_t s_w[12];
    __shared__ Place s_p;
    constexpr int C = kChunk<T>;
    const Cuts cuts{a.chunk, 1};
    const int n_tiles = (a.cols + kTile - 1) / kTile, k_tiles = (a.depth + kTile - 1) / kTile;
    const int64_t at = xcd_order(workgroup(), (int64_t)gridDim.y * gridDim.x);
    const int64_t item = at / (n_tiles * k_tiles);
    int64_t items, covered;
    pass<4>(a, cuts, s_w, &s_p, items, covered,
            [&](int64_t first, int64_t n, int64_t) { return item >= first && item < first + n; });
    if (item >= items || item >= max_items) return;
    const int tile = (int)(at % (n_tiles * k_tiles)), n0 = tile / k_tiles * kTile, k0 = tile % k_tiles * kTile;
    const Place p = s_p;
    const int64_t group = scalar64(p.group), row = scalar64(p.row), size = scalar64(p.size), piece = item - scalar64(p.piece);
    const int64_t r0 = row + piece * a.chunk;
    const int64_t n_rows = max((int64_t)0, min(min(size - piece * a.chunk, a.chunk), a.rows - r0));
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x % 128;
    const bool first_half = threadIdx.x < 128;
    const bool sums = a.dbias && k0 == 0;
    using S = Stage<T, true>;
    u32x4 st[S::R];
    float col_sum[8 / C][C] = {};
    const int64_t span = PARTS == 1 ? n_rows : (n_rows + kSlab<T> - 1) / kSlab<T> * kSlab<T>, end = PARTS * span;
    auto fetch = [&](int64_t r) {
        const bool low = PARTS == 2 && r >= span;
        if (low) r -= span;
        const int left = (int)min(n_rows - r, (int64_t)kSlab<T>);
        if (first_half)
            S::load(st, (const T*)(low ? a.a_low : a.a) + (r0 + r) * a.cols + n0, a.cols, min(a.cols - n0, kTile), 0, left, t);
        else
            S::load(st, (const T*)a.b + (r0 + r) * a.depth + k0, a.depth, min(a.depth - k0, kTile), 0, left, t);
    };
    f32x16 acc[2][2] = {};
    if (n_rows > 0) fetch(0);
    for (int64_t r = 0; r < end; r += kSlab<T>) {
        __syncthreads();
        S::store(st, first_half ? s_a : s_b, t);
        if (sums && first_half) {
#pragma unroll
            for (int b = 0; b < 8 / C; ++b)
#pragma unroll
                for (int j = 0; j < C; ++j)
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const uint32_t word = st[b * C + i][j * (int)sizeof(T) / 4];
                        col_sum[b][j] += __builtin_bit_cast(float, sizeof(T) == 4 ? word : j % 2 ? word & 0xffff0000u : word << 16);
                    }
        }
        __syncthreads();
        if (r + kSlab<T> < end) fetch(r + kSlab<T>);
        multiply<T>(s_b, s_a, (w / 2) * 64, (w % 2) * 64, lane, acc);
    }
    const bool whole = cuts.of(size) == 1;
    const int64_t slot = scalar64(p.many) + piece;
    if (sums) {  // the threads of a column are kTile / C apart
        __syncthreads();
        constexpr int across = kTile / C, strands = kSlab<T> / C;
        float* s_sum = (float*)s_a;  // [strands][kTile]
        if (first_half)
            for (int b = 0; b < 8 / C; ++b)
                for (int j = 0; j < C; ++j) {
                    const int id = t + 128 * b;
                    s_sum[id / across * kTile + id % across * C + j] = col_sum[b][j];
                }
        __syncthreads();
        const int n = n0 + threadIdx.x;
        if (threadIdx.x < kTile && n < a.cols) {
            float x = 0;
            for (int i = 0; i < strands; ++i) x += s_sum[i * kTile + threadIdx.x];
            if (whole) ((T*)a.dbias)[group * a.cols + n] = (T)x;
            else a.part_bias[slot * a.cols + n] = x;
        }
    }
    if (whole) {
        const int c0 = k0 + (w / 2) * 64, m0 = n0 + (w % 2) * 64;
        write_out<T>(acc, s_out + w * kOutRows * kOutPitch<T>, lane,
                     (T*)a.out + (group * a.cols + m0) * (int64_t)a.depth + c0, a.depth, a.cols - m0, a.depth - c0,
                     (const T*)nullptr);
    } else {
        f32x4* part = (f32x4*)a.part + ((slot * n_tiles * k_tiles + tile) * 4 + w) * 1024 + lane;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            f32x4 v;
            for (int c = 0; c < 4; ++c) v[c] = acc[q / 8][q / 4 % 2][4 * (q % 4) + c];
            part[q * 64] = v;
        }
    }
}

// Adds up the partial sums of groups of more than one item, in the items' order: a thread for four
// neighbouring columns a time, `parts` workgroups (a divisor of sixteen) for a tile of a split group.
constexpr int kJoinParts = 16;
template <typename T>
__global__ __launch_bounds__(256) void weight_join_kernel(Args a, int parts)
{
    __shared__ int64_t s_w[12];
    __shared__ Place s_p;
    const int n_tiles = (a.cols + kTile - 1) / kTile, k_tiles = (a.depth + kTile - 1) / kTile;
    const int64_t unit = blockIdx.x / parts, rank = unit / (n_tiles * k_tiles);
    const int first_part = (int)(blockIdx.x % parts);
    const int tile = (int)(unit % (n_tiles * k_tiles)), n0 = tile / k_tiles * kTile, k0 = tile % k_tiles * kTile;
    const Cuts cuts{a.chunk, 1};
    if (threadIdx.x == 0) s_p.group = -1;
    int64_t all_pieces, all_rows;
    pass<4>(a, cuts, s_w, &s_p, all_pieces, all_rows, [&](int64_t, int64_t n, int64_t split) { return n > 1 && split == rank; });
    const int64_t group = scalar64(s_p.group);
    if (group < 0) return;
    const int64_t pieces = scalar64(cuts.of(s_p.size)), slot = scalar64(s_p.many);
    // (the layout of weight_kernel's accumulators: four waves of sixteen times 64 lanes)
    const int lane = threadIdx.x & 63;
    const int64_t step = (int64_t)n_tiles * k_tiles * 4096;
    for (int part_of = first_part; part_of < kJoinParts; part_of += parts) {
        const int w = part_of / 4, q = part_of % 4 * 4 + threadIdx.x / 64;
        const f32x4* part = (const f32x4*)a.part + slot * step + ((int64_t)tile * 4 + w) * 1024 + q * 64 + lane;
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
        for (int64_t i = 0; i < pieces; ++i) sum += part[i * step];
        const int i = q / 8, j = q / 4 % 2;
        const int n = n0 + (w % 2) * 64 + 32 * j + (lane & 31);
        const int k = k0 + (w / 2) * 64 + 32 * i + 8 * (q % 4) + 4 * (lane >> 5);
        if (n < a.cols)
            for (int c = 0; c < 4; ++c)
                if (k + c < a.depth) ((T*)a.out)[(group * a.cols + n) * a.depth + k + c] = (T)sum[c];
    }
    const int col = n0 + threadIdx.x;
    if (a.dbias && k0 == 0 && first_part == 0 && threadIdx.x < kTile && col < a.cols) {
        float x = 0;
#pragma unroll 4
        for (int64_t i2 = 0; i2 < pieces; ++i2) x += a.part_bias[(slot + i2) * a.cols + col];
        ((T*)a.dbias)[group * a.cols + col] = (T)x;
    }
}

// ---------------------------------------------------------------- host
// Rows of an item of dW.  Splitting a group costs the join's launch and its partial sums' traffic, as
// much time as 512 rows of bfloat16 or 128 of float take to add up (one 128 x 128 tile, 128 groups
// of 250 rows: 17 us whole, 25 us in items of 128 rows; 7 groups of 1400 rows of 100 by 164 floats:
// 182 us whole, 27 us in items of 128).  Groups of fewer rows, and groups whose tiles alone give
// every CU two workgroups (128 groups of 256 by 512: 41 us, split 71 to 102 us), are taken whole up
// to four times their mean.  Else as many items as make two workgroups for every CU (8 groups of
// 25,000 rows: 32 us, four workgroups 41 us, whole 538 us), of 128 rows and more.
template <typename T>
int64_t item_rows(const dg_grouped_desc* d)
{
    const int64_t tiles = (int64_t)((d->n + kTile - 1) / kTile) * ((d->k + kTile - 1) / kTile);
    const int64_t mean = d->n_rows / d->n_groups + 1, each = 512 / (d->n_groups * tiles);
    const int64_t c = each <= 1 || mean <= (sizeof(T) == 2 ? 512 : 128) ? 4 * mean : mean / each;
    return std::max<int64_t>(128, (c + 63) / 64 * 64);
}
int64_t rows_of_item(const dg_grouped_desc* d)
{
    return d->dtype == DG_BF16 ? item_rows<__bf16>(d) : item_rows<float>(d);
}

struct Layout {
    size_t o_part, o_bias, total;
};

Layout layout(const dg_grouped_desc* d)
{
    // groups of several items have at most twice as many as their rows alone would make
    const int64_t slots = 2 * (d->n_rows / rows_of_item(d));
    const int64_t tiles = (int64_t)((d->n + kTile - 1) / kTile) * ((d->k + kTile - 1) / kTile);
    Layout L;
    L.o_part = 0;
    L.o_bias = al(4 * (size_t)(slots * tiles * kTile * kTile));
    L.total = L.o_bias + al(4 * (size_t)(slots * d->n) + 1);
    return L;
}

dg_status check(const dg_grouped_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->dtype != DG_F32 && d->dtype != DG_BF16)
        return fail(DG_ERR_INVALID, "x and weight must be float32 or bfloat16");
    if (d->n_rows < 0 || d->n_rows > (1ll << 40)) return fail(DG_ERR_INVALID, "rows must be in [0, 2^40]");
    if (d->n_groups < 1 || d->n_groups > kMaxGroups) return fail(DG_ERR_INVALID, "groups must be in [1, 2^20]");
    if (d->k < 1 || d->n < 1 || d->k > (1 << 20) || d->n > (1 << 20))
        return fail(DG_ERR_INVALID, "the widths must be in [1, 2^20]");
    return DG_OK;
}

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

// Workgroups of the streaming kernel: one a CU (its LDS), for each panel a share of the row tiles.
constexpr int kCus = 256;
int64_t stream_tiles(const Args& a) { return a.rows / kStreamRows + std::min(a.groups, a.rows) + 1; }

template <typename T, bool DX, int PN, int EPI, int PARTS>
void run_stream(const Args& a, hipStream_t s)
{
    const int64_t panels = (a.cols + PN - 1) / PN, tiles = stream_tiles(a);
    const int64_t lanes = std::max<int64_t>(1, std::min<int64_t>(tiles, kCus / panels));
    hipLaunchKernelGGL((stream_kernel<T, DX, PN, EPI, PARTS>), dim3((unsigned)(panels * lanes)), dim3(64 * kStreamWaves), 0, s, a,
                       lanes == tiles);
}

template <typename T, bool DX, int EPI = kPlain, int PARTS = 1>
void run_rows(const Args& a, hipStream_t s)
{
    // Whole chunks and a panel that fits: the streaming kernel (128 by 128 in bfloat16, 864 rows: 6.3
    // us, the other 10.0 us; 200,000 rows: 24.5 us, 33.0 us).  Narrower panels read x more often and
    // need less time to fill; they pay where wide ones would leave most CUs without work (128 by 128,
    // panels of 32, 64 and 128: 864 rows 6.3, 6.8 and 8.1 us; 30,000 rows 10.6, 8.2 and 9.3 us; 60,000
    // rows 13.9, 12.6 and 11.1 us).  Rows of more than 512 bytes leave the panel's LDS 64 columns.
    const int64_t bytes = a.depth * (int64_t)sizeof(T);
    const bool whole = bytes % 16 == 0 && a.cols % kChunk<T> == 0 && ((uintptr_t)a.a & 15) == 0 &&
                       ((uintptr_t)a.out & 15) == 0 && ((uintptr_t)a.aux & 15) == 0 && ((uintptr_t)a.a_low & 15) == 0 &&
                       ((uintptr_t)a.out_low & 15) == 0 && a.cols * (int64_t)sizeof(T) <= 1 << 24;
    if (whole && bytes <= 1024) {
        const int64_t work = stream_tiles(a) * ((a.cols + 127) / 128);  // workgroups with panels of 128
        if (work <= kCus / 4) run_stream<T, DX, 32, EPI, PARTS>(a, s);
        else if (bytes > 512 || work <= kCus / 2) run_stream<T, DX, 64, EPI, PARTS>(a, s);
        else run_stream<T, DX, 128, EPI, PARTS>(a, s);
        return;
    }

    const int64_t tiles = (a.rows / kTile + std::min(a.groups, a.rows) + 1) * ((a.cols + kTile - 1) / kTile);
    unsigned grid = (unsigned)std::min<int64_t>(tiles, 256 * 2);
    if (grid > kXcds) grid = (grid + kXcds - 1) / kXcds * kXcds;
    hipLaunchKernelGGL((rows_kernel<T, DX, EPI, PARTS>), dim3(grid), dim3(256), 0, s, a);
}

template <typename T, int PARTS = 1>
void run_weight(const Args& a, hipStream_t s)
{
    const int64_t tiles = (int64_t)((a.cols + kTile - 1) / kTile) * ((a.depth + kTile - 1) / kTile);
    const int64_t items = a.rows / a.chunk + a.groups;
    int64_t grid = items * tiles;
    if (grid > kXcds) grid = (grid + kXcds - 1) / kXcds * kXcds;
    hipLaunchKernelGGL((weight_kernel<T, PARTS>), workgroups(grid), dim3(256), 0, s, a, items);
    const int64_t split = std::min(a.groups, a.rows / a.chunk);  // groups above an item, at most
    if (split > 0) {
        // (most of a large number find no group: one round of workgroups, each with more to do)
        int parts = kJoinParts;
        while (parts > 1 && split * tiles * parts > 4 * kCus) parts /= 2;
        hipLaunchKernelGGL(weight_join_kernel<T>, dim3((unsigned)(split * tiles * parts)), dim3(256), 0, s, a, parts);
    }
}

}  // namespace

extern "C" {

dg_status dg_grouped_forward(const dg_grouped_desc* d, const void* x, const void* weight, const int64_t* sizes,
                             const void* bias, void* y, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (d->n_rows == 0) return DG_OK;
    if (!x || !weight || !sizes || !y) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    Args a = {};
    a.a = x;
    a.b = weight;
    a.bias = bias;
    a.out = y;
    a.sizes = sizes;
    a.rows = d->n_rows;
    a.groups = d->n_groups;
    a.cols = d->n;
    a.depth = d->k;
    if (d->dtype == DG_BF16) run_rows<__bf16, false>(a, s);
    else run_rows<float, false>(a, s);
    return launched("dg_grouped_forward");
}

static dg_status apply(const dg_grouped_desc* d, int32_t act, bool slope, const void* x, const void* weight, const int64_t* sizes,
                       const void* bias, const void* aux, void* out, void* out_low, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (act != DG_ACT_NONE && act != DG_ACT_SILU && act != DG_ACT_GELU) return fail(DG_ERR_INVALID, "unknown activation");
    if (d->n_rows == 0) return DG_OK;
    if (!x || !weight || !sizes || !out || (slope && !aux)) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    Args a = {};
    a.a = x;
    a.b = weight;
    a.bias = bias;
    a.aux = aux;
    a.act = act;
    a.out = out;
    a.out_low = out_low;
    a.sizes = sizes;
    a.rows = d->n_rows;
    a.groups = d->n_groups;
    a.cols = d->n;
    a.depth = d->k;
    if (d->dtype == DG_BF16) {
        if (slope) run_rows<__bf16, false, kSlope>(a, s);
        else run_rows<__bf16, false, kApply>(a, s);
    } else {
        if (slope) run_rows<float, false, kSlope>(a, s);
        else run_rows<float, false, kApply>(a, s);
    }
    return launched("dg_grouped_apply");
}

dg_status dg_grouped_apply(const dg_grouped_desc* d, int32_t act, const void* x, const void* weight, const int64_t* sizes,
                           const void* bias, const void* residual, void* y, hipStream_t s)
{
    return apply(d, act, false, x, weight, sizes, bias, residual, y, nullptr, s);
}

dg_status dg_grouped_apply_backward(const dg_grouped_desc* d, int32_t act, const void* x, const void* weight,
                                    const int64_t* sizes, const void* bias, const void* grad_y, void* dz, hipStream_t s)
{
    return apply(d, act, true, x, weight, sizes, bias, grad_y, dz, nullptr, s);
}

size_t dg_grouped_workspace_size(const dg_grouped_desc* d)
{
    if (check(d) != DG_OK) return 0;
    return layout(d).total;
}

// The gradients from those of the product's results, in one part or two (grad_low; 8 and 16 bits apart, bfloat16).
static dg_status backward(const dg_grouped_desc* d, const void* x, const void* weight, const int64_t* sizes, const void* grad,
                          const void* grad_low, void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes, hipStream_t s)
{
    const Layout L = layout(d);
    Args a = {};
    a.sizes = sizes;
    a.rows = d->n_rows;
    a.groups = d->n_groups;
    a.a = grad;
    a.a_low = grad_low;
    if (dx && d->n_rows > 0) {
        a.b = weight;
        a.out = dx;
        a.cols = d->k;
        a.depth = d->n;
        if (d->dtype != DG_BF16) run_rows<float, true>(a, s);
        else if (grad_low) run_rows<__bf16, true, kPlain, 2>(a, s);
        else run_rows<__bf16, true>(a, s);
    }
    if (dweight) {
        if (!ws || ws_bytes < L.total) return fail(DG_ERR_WORKSPACE, "workspace too small");
        a.b = x;
        a.out = dweight;
        a.dbias = dbias;
        a.cols = d->n;
        a.depth = d->k;
        a.chunk = rows_of_item(d);
        a.part = (float*)((char*)ws + L.o_part);
        a.part_bias = (float*)((char*)ws + L.o_bias);
        if (d->dtype != DG_BF16) run_weight<float>(a, s);
        else if (grad_low) run_weight<__bf16, 2>(a, s);
        else run_weight<__bf16>(a, s);
    } else if (dbias) {
        return fail(DG_ERR_INVALID, "dbias comes with dweight");
    }
    return launched("dg_grouped_backward");
}

dg_status dg_grouped_backward(const dg_grouped_desc* d, const void* x, const void* weight, const int64_t* sizes,
                              const void* grad_y, void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes,
                              hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (!sizes || (d->n_rows > 0 && (!x || !weight || !grad_y)))
        return fail(DG_ERR_INVALID, "inputs are NULL");
    return backward(d, x, weight, sizes, grad_y, nullptr, dx, dweight, dbias, ws, ws_bytes, s);
}

// dz: float, or two of bfloat16
static size_t dz_bytes(const dg_grouped_desc* d) { return al((size_t)d->n_rows * d->n * (d->dtype == DG_BF16 ? 2 : 4)); }

size_t dg_grouped_apply_workspace_size(const dg_grouped_desc* d)
{
    if (check(d) != DG_OK) return 0;
    return layout(d).total + dz_bytes(d) * (d->dtype == DG_BF16 ? 2 : 1);
}

dg_status dg_grouped_apply_gradients(const dg_grouped_desc* d, int32_t act, const void* x, const void* weight, const int64_t* sizes,
                                     const void* bias, const void* grad_y, void* dx, void* dweight, void* dbias, void* ws,
                                     size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (act == DG_ACT_NONE) return dg_grouped_backward(d, x, weight, sizes, grad_y, dx, dweight, dbias, ws, ws_bytes, s);
    if (act != DG_ACT_SILU && act != DG_ACT_GELU) return fail(DG_ERR_INVALID, "unknown activation");
    if (!sizes || (d->n_rows > 0 && (!x || !weight || !grad_y))) return fail(DG_ERR_INVALID, "inputs are NULL");
    if (dbias && !dweight) return fail(DG_ERR_INVALID, "dbias comes with dweight");
    const size_t each = dz_bytes(d), sums = dweight ? layout(d).total : 0, dzs = dg_grouped_apply_workspace_size(d) - layout(d).total;
    if (!ws || ws_bytes < dzs + sums) return fail(DG_ERR_WORKSPACE, "workspace too small");
    char* const dz = (char*)ws;
    char* const low = d->dtype == DG_BF16 ? dz + each : nullptr;
    st = apply(d, act, true, x, weight, sizes, bias, grad_y, dz, low, s);
    if (st != DG_OK) return st;
    return backward(d, x, weight, sizes, dz, low, dx, dweight, dbias, dz + dzs, sums, s);
}

}  // extern "C"
