// Host-side sanitizer driver for the entry points of the operators on a built graph, test
// infrastructure only: tests/test_operators_sanitizers.py compiles the library's sources with
// AddressSanitizer and UndefinedBehaviorSanitizer on the host code together with this file and runs
// it without a GPU.  Workspace sizes on random and extreme descriptions (their products must not
// overflow, and a size is given or refused with a message), and calls that have to be refused
// before anything is launched: a bad description, a NULL pointer, a workspace one byte short.
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <random>

#include "dynamis_graph.h"

static int failures = 0;
#define CHECK(c, ...)                                            \
    do {                                                         \
        if (!(c)) {                                              \
            fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
            fprintf(stderr, __VA_ARGS__);                        \
            fprintf(stderr, "\n");                               \
            failures++;                                          \
        }                                                        \
    } while (0)

static long given = 0, refused = 0;
static size_t note(size_t s)
{
    if (s) ++given;
    else {
        ++refused;
        CHECK(strlen(dg_last_error()) > 0, "size 0 without an error message");
    }
    return s;
}

int main()
{
    std::mt19937_64 g(11);
    const int64_t counts[] = {0, 1, 2, 7, 511, 513, 1000, 1 << 20, 0x7fffff00LL, 0x7fffff01LL, 0x7fffffffLL,
                              1ll << 40, 1ll << 62, INT64_MAX, -1, INT64_MIN};
    const int32_t small[] = {0, 1, 2, 3, 4, 8, 12, 16, 32, 64, 128, 256, 264, 1024, 1025, 1 << 20, INT_MAX, -1, INT_MIN};
    auto count = [&] { return counts[g() % (sizeof counts / sizeof *counts)]; };
    auto some = [&] { return small[g() % (sizeof small / sizeof *small)]; };
    const float scales[] = {1.0f, 0.25f, -3.0f, 0.0f, INFINITY, NAN, 3e38f};
    void* const p = (void*)4096;  // never read: the calls are refused first
    int32_t* const ints = (int32_t*)p;
    float* const floats = (float*)p;
    for (int it = 0; it < 40000; ++it) {
        dg_neighbor_desc n;
        memset(&n, 0, sizeof n);
        n.n_edges = count();
        n.n_nodes = count();
        n.n_targets = g() % 2 ? n.n_nodes : count();
        n.n_boundaries = g() % 2 ? 31 : some();
        n.dist_dtype = (int32_t)(g() % 3);
        const size_t sn = note(dg_neighbors_workspace_size(&n));
        if (sn) {
            CHECK(n.n_edges >= 0 && n.n_edges <= 0x7fffff00LL && n.n_nodes >= 0 && n.n_targets <= n.n_nodes, "accepted lists");
            CHECK(sn >= (size_t)n.n_edges * 4 + (size_t)n.n_nodes * 12, "workspace of %zu bytes", sn);
            CHECK(dg_neighbors_by_target(&n, (int64_t*)p, (int64_t*)p, nullptr, nullptr, nullptr, ints, ints, ints, nullptr, 1, p,
                                         sn - 1, nullptr) == DG_ERR_WORKSPACE, "a workspace one byte short");
            CHECK(dg_neighbors_by_target(&n, (int64_t*)p, (int64_t*)p, nullptr, nullptr, nullptr, ints, nullptr, ints, nullptr, 1,
                                         p, sn, nullptr) == DG_ERR_INVALID, "no pointers");
            CHECK(dg_neighbors_read_totals(&n, nullptr, nullptr, nullptr) == DG_ERR_INVALID, "no totals");
        }
        (void)note(dg_neighbors_sort_workspace_size(n.n_edges));
        (void)note(dg_neighbors_parts_workspace_size(n.n_nodes));

        dg_attention_desc a;
        memset(&a, 0, sizeof a);
        const bool plain = g() % 2;  // (else hardly any is accepted)
        a.n_nodes = count();
        a.n_targets = g() % 2 ? a.n_nodes : count();
        a.kv_heads = plain ? 1 << g() % 4 : some();
        a.heads = plain ? a.kv_heads << g() % 4 : some();
        a.dim = plain ? 8 * (1 + (int)(g() % 32)) : some();
        a.n_buckets = plain ? (int)(g() % 33) : some();
        a.dtype = g() % 4 ? (g() % 2 ? DG_F32 : DG_BF16) : (int32_t)(g() % 6);
        a.scale = plain ? 1.0f : scales[g() % 7];
        for (int64_t* ld : {&a.ld_q, &a.ld_k, &a.ld_v, &a.ld_g})
            *ld = g() % 4 ? 8 * (int64_t)(g() % 4096) : count();
        dg_neighbor_lists l;
        memset(&l, 0, sizeof l);
        l.n_rows = g() % 8 ? a.n_nodes : count();
        l.order = l.ptr = l.idx = ints;
        l.bucket = g() % 8 ? (uint8_t*)p : nullptr;
        if (g() % 2) {
            l.n_items = count();
            l.n_long = g() % 2 ? 1 : count();
            l.items = l.item_first = ints;
            l.long_slot = g() % 8 ? ints : nullptr;
        }
        const size_t sa = note(dg_attention_workspace_size(&a, &l, g() % 2 ? &l : nullptr));
        const size_t sb = note(dg_attention_workspace_size(&a, &l, &l));
        if (sb) {
            CHECK(sa > 0 && isfinite(a.scale) && a.heads % a.kv_heads == 0, "accepted attention");
            const double need = 16.0 * a.n_targets * a.heads + 4.0 * l.n_items * a.heads * a.dim;
            CHECK((double)sb >= need, "workspace of %zu bytes for %g", sb, need);
            CHECK(dg_attention_backward(&a, &l, &l, p, p, p, floats, floats, floats, p, p, p, p, floats, p, sb - 1, nullptr) ==
                      DG_ERR_WORKSPACE, "a workspace one byte short");
            if (a.n_targets > 0)
                CHECK(dg_attention_forward(&a, &l, nullptr, p, p, floats, p, nullptr, nullptr, nullptr, p, SIZE_MAX, nullptr) ==
                          DG_ERR_INVALID, "no q");
            if (a.n_nodes > 0)
                CHECK(dg_attention_backward(&a, &l, &l, p, p, p, floats, floats, floats, p, p, nullptr, p, floats, p, sb,
                                            nullptr) == DG_ERR_INVALID, "no dk");
        } else {
            CHECK(dg_attention_forward(&a, &l, p, p, p, floats, p, nullptr, nullptr, nullptr, p, SIZE_MAX, nullptr) ==
                      DG_ERR_INVALID, "launched what has no workspace");
        }

        dg_grouped_desc w;
        memset(&w, 0, sizeof w);
        w.n_rows = count();
        w.n_groups = g() % 2 ? 1 + (int64_t)(g() % (1 << 20)) : count();
        w.k = some();
        w.n = some();
        w.dtype = g() % 4 ? (g() % 2 ? DG_F32 : DG_BF16) : (int32_t)(g() % 6);
        const size_t sg = note(dg_grouped_workspace_size(&w));
        if (sg) {
            CHECK(dg_grouped_backward(&w, p, p, (int64_t*)p, p, nullptr, p, nullptr, p, sg - 1, nullptr) == DG_ERR_WORKSPACE,
                  "a workspace one byte short");
            CHECK(dg_grouped_backward(&w, p, p, nullptr, p, p, p, nullptr, p, sg, nullptr) == DG_ERR_INVALID, "no sizes");
            CHECK(dg_grouped_backward(&w, p, p, (int64_t*)p, p, nullptr, nullptr, p, p, sg, nullptr) == DG_ERR_INVALID,
                  "a bias's gradient alone");
        } else {
            CHECK(dg_grouped_forward(&w, p, p, (int64_t*)p, p, p, nullptr) == DG_ERR_INVALID, "launched a bad description");
        }
    }
    CHECK(given > 10000 && refused > 10000, "%ld given, %ld refused", given, refused);
    printf("operators' host code: %ld sizes given, %ld refused\n", given, refused);
    if (failures) {
        fprintf(stderr, "%d failures\n", failures);
        return 1;
    }
    printf("all checks passed\n");
    return 0;
}
