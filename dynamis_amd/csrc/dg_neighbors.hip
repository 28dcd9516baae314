// dg_neighbors.hip -- the index lists that the attention over a built graph reads.
//
// From an edge list grouped by target (as every builder here writes it) and, optionally, a
// mask, distances and bucket boundaries, two compressed lists come out: for every target the
// sources of its edges (the forward pass and the gradient of q), for every source its targets
// (the gradients of k and v), each entry with its distance bucket.  Rows sit in slots: a
// node's slot is the place of its run in the edge list, nodes without a run follow by number (so
// the targets, being the first nodes, hold the first slots).
// Slots keep the builder's space-filling order, so rows that run at the same time read
// neighbouring atoms whatever the caller's numbering is.
//
// Two passes over the edge list with one scan between them; the second reads sources and targets twice,
// to count its waves' runs and entries and to write them.  26.5M edges take 465 us for the lists by
// target, 8.8M edges 224 us, where 57 bytes an edge (three times 16, 4 of distance, 5 written) at a
// copy's rate take 310 us and 103 us; 74,000 edges 111 us, launches and the wait.  The lists by source need no sort when
// the kept edges are symmetric -- for each (i, j, bucket) as many (j, i, bucket), which holds
// for every complete radius graph, the canonical distance being exact under negation: then
// the sources of a node are its targets, and the lists are the same arrays.  Symmetry is
// decided by two 64-bit sums over the edges of hash(i, j, b) - hash(j, i, b), both of which
// are zero for a symmetric list and, for any other, with a probability of about 2^-128.
// Otherwise a stable sort by the source's slot gives them.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "../../include/dynamis_graph.h"
#include "dg_scan.hpp"

namespace dg {
dg_status fail(dg_status st, const std::string& msg);  // dg_graph.hip
}

namespace {

using namespace dg;

inline size_t al(size_t x) { return (x + 255) & ~(size_t)255; }
inline unsigned nblk(int64_t n, int b = 256) { return (unsigned)((n + b - 1) / b); }

constexpr int kWaveEdges = 512;              // edges of a wave: eight steps of 64
constexpr int kTileEdges = 4 * kWaveEdges;   // of a workgroup
constexpr int kFingerSlots = 64;             // the hash sums are spread over so many addresses
constexpr int kMaxBuckets = 128;
constexpr int64_t kMaxEdges = 0x7fffff00LL;

// totals[]: what the host reads
enum { kKept = 0, kFlags, kRuns, kLongest, kLongRows, kLongEntries, kAsym, kTotals = 8 };

struct Args {
    const int64_t* src;
    const int64_t* dst;
    const uint8_t* mask;
    const void* dist;
    const void* bounds;
    int dist64, n_bounds;
    int64_t E, N, T;
    int64_t* tile;  // [tiles + 1] runs << 32 | kept
    int32_t* slot_of;
    int32_t* order;
    int32_t* ptr;
    int32_t* idx;
    uint8_t* bucket;
    int32_t* dst32;
    unsigned long long* finger;
    int64_t* totals;
};

__device__ __forceinline__ uint64_t mix64(uint64_t x)
{
    // the finaliser of splitmix64 (Steele, Lea, Flood 2014)
    x = (x ^ (x >> 30)) * 0xbf58476d1ce4e5b9ull;
    x = (x ^ (x >> 27)) * 0x94d049bb133111ebull;
    return x ^ (x >> 31);
}

__global__ void clear_kernel(Args a)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < kTotals) a.totals[i] = 0;
    if (i < 2 * kFingerSlots) a.finger[i] = 0;
    if (i < a.N) a.slot_of[i] = -1;
}

// One step of a wave: is lane's edge the first of its target's run, is it kept.
__device__ __forceinline__ void classify(const Args& a, int64_t e, int lane, int64_t& s, int64_t& d,
                                         bool& first, bool& kept, int& bad)
{
    const bool in = e < a.E;
    s = in ? a.src[e] : 0;
    d = in ? a.dst[e] : -1;
    int64_t before = __shfl_up(d, 1, 64);
    if (lane == 0) before = in && e > 0 ? a.dst[e - 1] : -1;
    const bool ok = in && s >= 0 && s < a.N && d >= 0 && d < a.T;
    if (in && !ok) bad |= DG_FLAG_RANGE;
    first = ok && (e == 0 || before != d);
    kept = ok && (!a.mask || a.mask[e]);
}

__global__ __launch_bounds__(256) void tile_kernel(Args a)
{
    __shared__ int s_w[4][2];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t base = (int64_t)blockIdx.x * kTileEdges + w * kWaveEdges;
    int runs = 0, kept = 0, bad = 0;
    for (int t = 0; t < kWaveEdges / 64; ++t) {
        int64_t s, d;
        bool f, k;
        classify(a, base + t * 64 + lane, lane, s, d, f, k, bad);
        runs += __popcll(__ballot(f));
        kept += __popcll(__ballot(k));
    }
    if (__any(bad) && lane == 0) atomicOr((unsigned long long*)&a.totals[kFlags], (unsigned long long)DG_FLAG_RANGE);
    if (lane == 0) {
        s_w[w][0] = runs;
        s_w[w][1] = kept;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t r = 0, k = 0;
        for (int i = 0; i < 4; ++i) {
            r += s_w[i][0];
            k += s_w[i][1];
        }
        a.tile[blockIdx.x] = (r << 32) | k;
    }
}

template <typename D>
__device__ __forceinline__ int bucket_of(D x, const D* b, int n)
{
    // the number of boundaries <= x (they ascend); 0 for a NaN
    int lo = 0;
#pragma unroll
    for (int step = 64; step > 0; step >>= 1)
        if (lo + step <= n && b[lo + step - 1] <= x) lo += step;
    return lo;
}

template <typename D>
__global__ __launch_bounds__(256) void write_kernel(Args a, const int64_t* __restrict__ tile_at)
{
    __shared__ int s_w[4][2];
    __shared__ D s_b[kMaxBuckets];
    __shared__ unsigned long long s_f[4][2];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < a.n_bounds; i += 256) s_b[i] = ((const D*)a.bounds)[i];
    const int64_t base = (int64_t)blockIdx.x * kTileEdges + w * kWaveEdges;
    int runs = 0, kept = 0, bad = 0;
    for (int t = 0; t < kWaveEdges / 64; ++t) {
        int64_t s, d;
        bool f, k;
        classify(a, base + t * 64 + lane, lane, s, d, f, k, bad);
        runs += __popcll(__ballot(f));
        kept += __popcll(__ballot(k));
    }
    if (lane == 0) {
        s_w[w][0] = runs;
        s_w[w][1] = kept;
    }
    __syncthreads();
    int64_t run = tile_at[blockIdx.x] >> 32, at = tile_at[blockIdx.x] & 0xffffffffLL;
    for (int i = 0; i < w; ++i) {
        run += s_w[i][0];
        at += s_w[i][1];
    }
    uint64_t f0 = 0, f1 = 0;
    bool twice = false;
    for (int t = 0; t < kWaveEdges / 64; ++t) {
        const int64_t e = base + t * 64 + lane;
        int64_t s, d;
        bool f, k;
        classify(a, e, lane, s, d, f, k, bad);
        const uint64_t fm = __ballot(f), km = __ballot(k), below = (1ull << lane) - 1;
        const int64_t my_at = at + __popcll(km & below);
        if (f) {
            const int64_t slot = run + __popcll(fm & below);
            if (slot < a.N) {  // more runs than nodes: not grouped, seen as a second run of some node
                a.order[slot] = (int32_t)d;
                a.ptr[slot] = (int32_t)my_at;
            }
            twice |= atomicExch(&a.slot_of[d], (int32_t)min(slot, a.N - 1)) != -1;
        }
        if (k) {
            int b = 0;
            if (a.dist) b = bucket_of<D>(((const D*)a.dist)[e], s_b, a.n_bounds);
            a.idx[my_at] = (int32_t)s;
            if (a.bucket) a.bucket[my_at] = (uint8_t)b;
            if (a.dst32) {
                a.dst32[my_at] = (int32_t)d;
                const uint64_t u = ((uint64_t)s << 32) | (uint64_t)d, v = ((uint64_t)d << 32) | (uint64_t)s;
                const uint64_t k0 = 0x9e3779b97f4a7c15ull * (2 * b + 1), k1 = 0xd1342543de82ef95ull * (2 * b + 1);
                f0 += mix64(u + k0) - mix64(v + k0);
                f1 += mix64((u ^ 0xa0761d6478bd642full) + k1) - mix64((v ^ 0xa0761d6478bd642full) + k1);
            }
        }
        run += __popcll(fm);
        at += __popcll(km);
    }
    if (__any(twice) && lane == 0)
        atomicOr((unsigned long long*)&a.totals[kFlags], (unsigned long long)DG_FLAG_UNGROUPED);
    if (a.dst32) {
        for (int o = 32; o > 0; o >>= 1) {
            f0 += __shfl_xor(f0, o, 64);
            f1 += __shfl_xor(f1, o, 64);
        }
        if (lane == 0) {
            s_f[w][0] = f0;
            s_f[w][1] = f1;
        }
        __syncthreads();
        if (threadIdx.x < 2)
            atomicAdd(&a.finger[2 * (blockIdx.x % kFingerSlots) + threadIdx.x],
                      s_f[0][threadIdx.x] + s_f[1][threadIdx.x] + s_f[2][threadIdx.x] + s_f[3][threadIdx.x]);
    }
}

__global__ void unseen_kernel(const int32_t* __restrict__ slot_of, int64_t n, int* __restrict__ flag)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) flag[i] = slot_of[i] < 0;
}

// Nodes without a run take the slots behind the runs; the list's end closes the pointers.
__global__ void rest_kernel(Args a, const int* __restrict__ place, const int64_t* __restrict__ tile_total)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t runs = *tile_total >> 32, kept = *tile_total & 0xffffffffLL;
    if (i == 0) {
        a.ptr[a.N] = (int32_t)kept;
        a.totals[kKept] = kept;
        a.totals[kRuns] = runs;
        if (a.dst32) {
            unsigned long long f0 = 0, f1 = 0;
            for (int k = 0; k < kFingerSlots; ++k) {
                f0 += a.finger[2 * k];
                f1 += a.finger[2 * k + 1];
            }
            a.totals[kAsym] = (f0 | f1) != 0;
        }
    }
    // the padding behind the entries, whose first a row of an empty list reads
    if (i < DG_NEIGHBOR_PAD) {
        a.idx[kept + i] = 0;
        if (a.bucket) a.bucket[kept + i] = 0;
    }
    if (i < a.N && a.slot_of[i] < 0) {
        const int64_t slot = runs + place[i];
        if (slot < a.N) {
            a.order[slot] = (int32_t)i;
            a.ptr[slot] = (int32_t)kept;
            a.slot_of[i] = (int32_t)slot;
        }
    }
}

// Longest row, and the rows above `split` with their entries.
__global__ __launch_bounds__(256) void longest_kernel(const int32_t* __restrict__ ptr, int64_t n, int split,
                                                      int64_t* __restrict__ totals)
{
    int longest = 0;
    long long rows = 0, entries = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int len = ptr[i + 1] - ptr[i];
        longest = max(longest, len);
        if (len > split) {
            ++rows;
            entries += len;
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        longest = max(longest, __shfl_xor(longest, o, 64));
        rows += __shfl_xor(rows, o, 64);
        entries += __shfl_xor(entries, o, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        atomicMax((unsigned long long*)&totals[kLongest], (unsigned long long)longest);
        if (rows) {
            atomicAdd((unsigned long long*)&totals[kLongRows], (unsigned long long)rows);
            atomicAdd((unsigned long long*)&totals[kLongEntries], (unsigned long long)entries);
        }
    }
}

// ---------------------------------------------------------------- lists by source
__global__ void keys_kernel(const int32_t* __restrict__ idx, const int32_t* __restrict__ slot_of, int64_t n,
                            int64_t* __restrict__ key)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) key[i] = slot_of[idx[i]];
}

__global__ void gather_kernel(const int64_t* __restrict__ perm, const int64_t* __restrict__ key,
                              const int32_t* __restrict__ dst32, const uint8_t* __restrict__ bucket, int64_t n,
                              int32_t* __restrict__ sorted, int32_t* __restrict__ tgt, uint8_t* __restrict__ sbucket)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) {
        const int64_t p = perm[i];
        sorted[i] = (int32_t)key[p];
        tgt[i] = dst32[p];
        if (bucket) sbucket[i] = bucket[p];
    } else if (i < n + DG_NEIGHBOR_PAD) {
        tgt[i] = 0;
        if (bucket) sbucket[i] = 0;
    }
}

__global__ void bounds_kernel(const int32_t* __restrict__ sorted, int64_t n, int64_t rows, int32_t* __restrict__ ptr)
{
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r > rows) return;
    int64_t lo = 0, hi = n;  // the first entry of a slot >= r
    while (lo < hi) {
        const int64_t m = (lo + hi) >> 1;
        if (sorted[m] < r) lo = m + 1;
        else hi = m;
    }
    ptr[r] = (int32_t)lo;
}

// ---------------------------------------------------------------- long rows in parts
__global__ void parts_kernel(const int32_t* __restrict__ ptr, int64_t n, int split, int chunk, int* __restrict__ parts,
                             int* __restrict__ is_long)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int len = ptr[i + 1] - ptr[i];
    parts[i] = len > split ? (len - 1) / chunk + 1 : 0;  // (len may be near 2^31)
    is_long[i] = len > split;
}

__global__ void long_kernel(const int* __restrict__ rank, int64_t n, int64_t n_long, int32_t* __restrict__ long_slot)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n && rank[i + 1] > rank[i] && rank[i] < n_long) long_slot[rank[i]] = (int32_t)i;
    if (i < n_long && i >= rank[n]) long_slot[i] = -1;
}

__global__ void items_kernel(const int32_t* __restrict__ first, const int32_t* __restrict__ ptr,
                             const int32_t* __restrict__ order, int64_t n, int chunk, int64_t max_items,
                             int4* __restrict__ item)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < max_items && i >= first[n]) item[i] = make_int4(0, 0, -1, 0);  // (the bound is not reached)
    if (i >= n) return;
    for (int64_t k = first[i]; k < first[i + 1] && k < max_items; ++k) {
        const int at = ptr[i] + (int)(k - first[i]) * chunk;  // (below the row's end; at + chunk may pass 2^31)
        item[k] = make_int4(at, at + min(chunk, ptr[i + 1] - at), order[i], (int)i);
    }
}

struct Layout {
    size_t o_totals, o_finger, o_tile, o_part, o_slot, o_dst, o_flag, o_place, total;
    int64_t tiles;
};

Layout layout(int64_t E, int64_t N)
{
    Layout L;
    size_t o = 0;
    auto take = [&](size_t b) { size_t r = o; o = al(o + (b ? b : 1)); return r; };
    L.tiles = (E + kTileEdges - 1) / kTileEdges;
    L.o_totals = take(8 * kTotals);
    L.o_finger = take(16 * kFingerSlots);
    L.o_tile = take(16 * (size_t)(L.tiles + 1));  // the tiles' counts, then their scan
    L.o_part = take(8 * (size_t)(std::max<int64_t>(L.tiles, N) / kScanTile + 2));
    L.o_slot = take(4 * (size_t)(N + 1));
    L.o_dst = take(4 * (size_t)E);
    L.o_flag = take(4 * (size_t)(N + 1));
    L.o_place = take(4 * (size_t)(N + 1));
    L.total = o;
    return L;
}

struct SortLayout {
    size_t o_key, o_perm, o_sorted, o_sort, total, sort_bytes;
};

SortLayout sort_layout(int64_t n)
{
    SortLayout L;
    size_t o = 0;
    auto take = [&](size_t b) { size_t r = o; o = al(o + (b ? b : 1)); return r; };
    L.o_key = take(8 * (size_t)n);
    L.o_perm = take(8 * (size_t)n);
    L.o_sorted = take(4 * (size_t)n);
    L.sort_bytes = dg_sfc_workspace_size(std::max<int64_t>(n, 1));
    L.o_sort = take(L.sort_bytes);
    L.total = o;
    return L;
}

dg_status check(const dg_neighbor_desc* d)
{
    if (!d) return fail(DG_ERR_INVALID, "desc is NULL");
    if (d->n_edges < 0 || d->n_edges > kMaxEdges) return fail(DG_ERR_INVALID, "n_edges must be in [0, 2^31 - 256]");
    if (d->n_nodes < 0 || d->n_nodes > kMaxEdges) return fail(DG_ERR_INVALID, "n_nodes must be in [0, 2^31 - 256]");
    if (d->n_targets < 0 || d->n_targets > d->n_nodes)
        return fail(DG_ERR_INVALID, "n_targets must be in [0, n_nodes]");
    if (d->n_boundaries < 0 || d->n_boundaries >= kMaxBuckets)
        return fail(DG_ERR_INVALID, "at most 127 boundaries (128 buckets)");
    if (d->dist_dtype != DG_F32 && d->dist_dtype != DG_F64)
        return fail(DG_ERR_INVALID, "distances must be float32 or float64");
    return DG_OK;
}

dg_status launched(const char* what)
{
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return DG_OK;
}

}  // namespace

extern "C" {

size_t dg_neighbors_workspace_size(const dg_neighbor_desc* d)
{
    if (check(d) != DG_OK) return 0;
    return layout(d->n_edges, d->n_nodes).total;
}

dg_status dg_neighbors_by_target(const dg_neighbor_desc* d, const int64_t* src, const int64_t* dst,
                                 const uint8_t* mask, const void* dist, const void* boundaries, int32_t* order,
                                 int32_t* ptr, int32_t* idx, uint8_t* bucket, int32_t by_source, void* ws,
                                 size_t ws_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    const Layout L = layout(d->n_edges, d->n_nodes);
    if (!ws || ws_bytes < L.total) return fail(DG_ERR_WORKSPACE, "workspace too small");
    if (!ptr || !idx || (d->n_nodes > 0 && !order) || (d->n_edges > 0 && (!src || !dst)) ||
        (bucket && d->n_edges > 0 && !dist) || (dist && d->n_boundaries > 0 && !boundaries))
        return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    char* w = (char*)ws;
    Args a = {};
    a.src = src;
    a.dst = dst;
    a.mask = mask;
    a.dist = bucket ? dist : nullptr;
    a.bounds = boundaries;
    a.dist64 = d->dist_dtype == DG_F64;
    a.n_bounds = bucket ? d->n_boundaries : 0;
    a.E = d->n_edges;
    a.N = d->n_nodes;
    a.T = d->n_targets;
    a.tile = (int64_t*)(w + L.o_tile);
    a.slot_of = (int32_t*)(w + L.o_slot);
    a.order = order;
    a.ptr = ptr;
    a.idx = idx;
    a.bucket = bucket;
    a.dst32 = by_source ? (int32_t*)(w + L.o_dst) : nullptr;
    a.finger = (unsigned long long*)(w + L.o_finger);
    a.totals = (int64_t*)(w + L.o_totals);
    int64_t* at = a.tile + L.tiles + 1;
    int64_t* part = (int64_t*)(w + L.o_part);
    int* flag = (int*)(w + L.o_flag);
    int* place = (int*)(w + L.o_place);
    hipLaunchKernelGGL(clear_kernel, dim3(nblk(std::max<int64_t>(a.N, 2 * kFingerSlots))), dim3(256), 0, s, a);
    if (L.tiles) hipLaunchKernelGGL(tile_kernel, dim3((unsigned)L.tiles), dim3(256), 0, s, a);
    excl_scan<int64_t, int64_t>(a.tile, L.tiles, at, part, s);
    if (L.tiles) {
        if (a.dist64)
            hipLaunchKernelGGL(write_kernel<double>, dim3((unsigned)L.tiles), dim3(256), 0, s, a, (const int64_t*)at);
        else
            hipLaunchKernelGGL(write_kernel<float>, dim3((unsigned)L.tiles), dim3(256), 0, s, a, (const int64_t*)at);
    }
    if (a.N > 0) hipLaunchKernelGGL(unseen_kernel, dim3(nblk(a.N)), dim3(256), 0, s, a.slot_of, a.N, flag);
    excl_scan<int, int>(flag, a.N, place, (int*)part, s);
    hipLaunchKernelGGL(rest_kernel, dim3(nblk(std::max<int64_t>(a.N, DG_NEIGHBOR_PAD))), dim3(256), 0, s, a,
                       (const int*)place, (const int64_t*)(at + L.tiles));
    if (a.N > 0)
        hipLaunchKernelGGL(longest_kernel, dim3(std::min(nblk(a.N), 512u)), dim3(256), 0, s, ptr, a.N,
                           DG_NEIGHBOR_SPLIT, a.totals);
    return launched("dg_neighbors_by_target");
}

dg_status dg_neighbors_read_totals(const dg_neighbor_desc* d, const void* ws, dg_neighbor_totals* out, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    if (!ws || !out) return fail(DG_ERR_INVALID, "workspace or totals is NULL");
    int64_t t[kTotals];
    hipError_t e = hipMemcpyAsync(t, (const char*)ws + layout(d->n_edges, d->n_nodes).o_totals, sizeof t,
                                  hipMemcpyDeviceToHost, s);
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) return fail(DG_ERR_HIP, std::string("dg_neighbors_read_totals: ") + hipGetErrorString(e));
    out->n_entries = t[kKept];
    out->longest = t[kLongest];
    out->long_rows = t[kLongRows];
    out->long_entries = t[kLongEntries];
    out->grouped = !(t[kFlags] & DG_FLAG_UNGROUPED);
    out->symmetric = t[kAsym] == 0;
    if (t[kFlags] & DG_FLAG_RANGE)
        return fail(DG_ERR_RANGE, "edge_index holds targets outside [0, " + std::to_string(d->n_targets) +
                                      ") or sources outside [0, " + std::to_string(d->n_nodes) + ")");
    return DG_OK;
}

size_t dg_neighbors_sort_workspace_size(int64_t n_entries)
{
    if (n_entries < 0 || n_entries > kMaxEdges) {
        fail(DG_ERR_INVALID, "n_entries must be in [0, 2^31 - 256]");
        return 0;
    }
    return sort_layout(n_entries).total;
}

dg_status dg_neighbors_by_source(const dg_neighbor_desc* d, int64_t n, const int32_t* idx, const uint8_t* bucket,
                                 int32_t* ptr, int32_t* tgt, uint8_t* tgt_bucket, void* ws, size_t ws_bytes,
                                 void* sort_ws, size_t sort_bytes, hipStream_t s)
{
    dg_status st = check(d);
    if (st != DG_OK) return st;
    const Layout L = layout(d->n_edges, d->n_nodes);
    if (n < 0 || n > d->n_edges) return fail(DG_ERR_INVALID, "n_entries must be in [0, n_edges]");
    const SortLayout S = sort_layout(n);
    if (!ws || ws_bytes < L.total || !sort_ws || sort_bytes < S.total)
        return fail(DG_ERR_WORKSPACE, "workspace too small");
    if (!idx || !ptr || !tgt || (bucket && !tgt_bucket)) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    char* w = (char*)ws;
    char* u = (char*)sort_ws;
    int64_t* key = (int64_t*)(u + S.o_key);
    int64_t* perm = (int64_t*)(u + S.o_perm);
    int32_t* sorted = (int32_t*)(u + S.o_sorted);
    if (n > 0) {
        hipLaunchKernelGGL(keys_kernel, dim3(nblk(n)), dim3(256), 0, s, idx, (const int32_t*)(w + L.o_slot), n, key);
        st = dg_sfc_order(key, n, perm, u + S.o_sort, S.sort_bytes, s);
        if (st != DG_OK) return st;
    }
    hipLaunchKernelGGL(gather_kernel, dim3(nblk(n + DG_NEIGHBOR_PAD)), dim3(256), 0, s, (const int64_t*)perm,
                       (const int64_t*)key, (const int32_t*)(w + L.o_dst), bucket, n, sorted, tgt, tgt_bucket);
    hipLaunchKernelGGL(bounds_kernel, dim3(nblk(d->n_nodes + 1)), dim3(256), 0, s, (const int32_t*)sorted, n,
                       d->n_nodes, ptr);
    int64_t* totals = (int64_t*)(w + L.o_totals);
    Args clear = {};
    clear.finger = (unsigned long long*)(w + L.o_finger);
    clear.totals = totals;
    hipLaunchKernelGGL(clear_kernel, dim3(nblk(2 * kFingerSlots)), dim3(256), 0, s, clear);
    if (d->n_nodes > 0)
        hipLaunchKernelGGL(longest_kernel, dim3(std::min(nblk(d->n_nodes), 512u)), dim3(256), 0, s, ptr, d->n_nodes,
                           DG_NEIGHBOR_SPLIT, totals);
    return launched("dg_neighbors_by_source");
}

size_t dg_neighbors_parts_workspace_size(int64_t n_rows)
{
    if (n_rows < 0 || n_rows > kMaxEdges) {
        fail(DG_ERR_INVALID, "n_rows must be in [0, 2^31 - 256]");
        return 0;
    }
    return 3 * al(4 * (size_t)(n_rows + 1)) + al(4 * (size_t)(n_rows / kScanTile + 2));
}

dg_status dg_neighbors_parts(const int32_t* order, const int32_t* ptr, int64_t n_rows, int32_t chunk,
                             int64_t max_items, int64_t n_long, int32_t* item_first, int32_t* items,
                             int32_t* long_slot, void* ws, size_t ws_bytes, hipStream_t s)
{
    if (n_rows < 1 || n_rows > kMaxEdges || chunk < 1 || max_items < 1 || n_long < 1)
        return fail(DG_ERR_INVALID, "n_rows, chunk, max_items and n_long must be positive");
    if (!order || !ptr || !item_first || !items || !long_slot) return fail(DG_ERR_INVALID, "inputs or outputs are NULL");
    if (!ws || ws_bytes < dg_neighbors_parts_workspace_size(n_rows))
        return fail(DG_ERR_WORKSPACE, "workspace too small");
    int* parts = (int*)ws;
    const size_t each = al(4 * (size_t)(n_rows + 1));
    int* is_long = (int*)((char*)ws + each);
    int* rank = (int*)((char*)ws + 2 * each);
    int* part = (int*)((char*)ws + 3 * each);
    hipLaunchKernelGGL(parts_kernel, dim3(nblk(n_rows)), dim3(256), 0, s, ptr, n_rows, DG_NEIGHBOR_SPLIT, (int)chunk,
                       parts, is_long);
    excl_scan<int, int>(parts, n_rows, item_first, part, s);
    excl_scan<int, int>(is_long, n_rows, rank, part, s);
    hipLaunchKernelGGL(long_kernel, dim3(nblk(std::max(n_rows, n_long))), dim3(256), 0, s, (const int*)rank, n_rows, n_long,
                       long_slot);
    hipLaunchKernelGGL(items_kernel, dim3(nblk(std::max(n_rows, max_items))), dim3(256), 0, s, (const int32_t*)item_first,
                       ptr, order, n_rows, (int)chunk, max_items, (int4*)items);
    return launched("dg_neighbors_parts");
}

}  // extern "C"
