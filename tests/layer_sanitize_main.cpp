// Host-side sanitizer driver for the entry points of a layer's operators, test infrastructure only:
// tests/test_layer_sanitizers.py compiles the library's sources with AddressSanitizer and
// UndefinedBehaviorSanitizer on the host code together with this file and runs it without a GPU.
// Random and extreme descriptions: a size is given or refused with a message, and every call here
// has to be refused before anything is launched.
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
    std::mt19937_64 g(12);
    const int64_t counts[] = {0, 1, 2, 7, 64, 1000, 1 << 20, 0x7fffffffLL, 1ll << 31, 1ll << 40, 1ll << 41, 1ll << 62, INT64_MAX, -1,
                              INT64_MIN};
    const int32_t small[] = {0, 1, 2, 3, 4, 8, 9, 12, 16, 32, 60, 64, 65, 128, 256, 264, 1024, 1025, 1 << 20, INT_MAX, -1, INT_MIN};
    auto count = [&] { return counts[g() % (sizeof counts / sizeof *counts)]; };
    auto some = [&] { return small[g() % (sizeof small / sizeof *small)]; };
    const float floats_of[] = {1.0f, 1e-6f, 0.0f, -3.0f, INFINITY, -INFINITY, NAN, 3e38f};
    auto number = [&] { return g() % 2 ? 1.0f : floats_of[g() % 8]; };
    void* const p = (void*)4096;  // never read: the calls are refused first
    void* const odd = (void*)4104;
    int32_t* const ints = (int32_t*)p;
    int64_t* const longs = (int64_t*)p;
    float* const floats = (float*)p;
    for (int it = 0; it < 60000; ++it) {
        const bool plain = g() % 2;  // (else hardly any is accepted)
        dg_rotate_desc r;
        memset(&r, 0, sizeof r);
        r.n_nodes = plain ? 1 + (int64_t)(g() % 1000000) : count();
        r.n_targets = g() % 2 ? r.n_nodes : plain ? r.n_nodes / 2 : count();
        for (int64_t* ld : {&r.ld_q, &r.ld_k, &r.ld_gq, &r.ld_gk}) *ld = g() % 8 ? 8 * (int64_t)(g() % 4096) : count();
        r.heads = plain ? 1 + (int)(g() % 64) : some();
        r.kv_heads = plain ? 1 + (int)(g() % 64) : some();
        r.dim = plain ? 8 * (1 + (int)(g() % 32)) : some();
        r.axes = plain ? 1 + (int)(g() % 8) : some();
        for (int i = 0; i < 8; ++i) r.sections[i] = plain ? (int)(g() % 3) : some();
        r.dtype = g() % 8 ? (g() % 2 ? DG_F32 : DG_BF16) : (int32_t)(g() % 6);
        r.weight_dtype = g() % 8 ? r.dtype : (int32_t)(g() % 6);
        r.pos_dtype = (int32_t)(g() % (plain ? 3 : 6));
        r.norm = (int32_t)(g() % 2);
        r.interleaved = (int32_t)(g() % 2);
        r.eps = plain ? 1e-6f : number();
        const size_t sr = note(dg_rotate_workspace_size(&r));
        const dg_status bad = dg_rotate_forward(&r, odd, p, p, floats, nullptr, nullptr, p, p, nullptr);
        if (sr) {
            CHECK(sr <= (size_t)1024 * 2 * 256 * 4 && sr >= (size_t)r.dim * 8, "workspace of %zu bytes", sr);
            if (r.n_nodes > 0) CHECK(bad == DG_ERR_INVALID, "misaligned rows");
            if (r.norm && r.n_nodes > 0)
                CHECK(dg_rotate_backward(&r, p, p, p, floats, p, p, p, p, p, p, nullptr, p, p, p, sr - 1, nullptr) == DG_ERR_WORKSPACE,
                      "a workspace one byte short");
            if (!r.norm)
                CHECK(dg_rotate_backward(&r, p, p, p, floats, p, p, p, p, p, p, nullptr, p, p, p, sr, nullptr) == DG_ERR_INVALID,
                      "weights without a norm");
        } else {
            CHECK(bad == DG_ERR_INVALID, "launched a bad description");
        }

        dg_route_desc u;
        memset(&u, 0, sizeof u);
        u.n_rows = plain ? (int64_t)(g() % 10000000) : count();
        u.ld = g() % 8 ? 1024 : count();
        u.groups = plain ? 1 << g() % 4 : some();
        u.n_experts = plain ? u.groups * (1 + (int)(g() % 64)) : some();
        u.k = plain ? 1 + (int)(g() % 8) : some();
        u.top_groups = plain ? 1 + (int)(g() % u.groups) : some();
        u.group_best = plain ? 1 + (int)(g() % 2) : some();
        u.sigmoid = (int32_t)(g() % 2);
        u.renormalize = (int32_t)(g() % 2);
        u.dtype = g() % 8 ? (g() % 2 ? DG_F32 : DG_BF16) : (int32_t)(g() % 6);
        u.scale = plain ? 1.0f : number();
        const size_t su = note(dg_route_workspace_size(&u));
        if (su) {
            CHECK((double)su >= (double)u.n_rows / 256 * 4 * (u.n_experts + 1), "workspace of %zu bytes", su);
            CHECK(dg_route_forward(&u, p, floats, floats, ints, longs, ints, p, su - 1, nullptr) == DG_ERR_WORKSPACE,
                  "a workspace one byte short");
            CHECK(dg_route_forward(&u, p, floats, floats, ints, nullptr, ints, p, su, nullptr) == DG_ERR_INVALID, "no sizes");
            if (u.n_rows > 0)
                CHECK(dg_route_backward(&u, p, ints, nullptr, p, nullptr) == DG_ERR_INVALID, "no gradient");
        } else {
            CHECK(dg_route_forward(&u, p, floats, floats, ints, longs, ints, p, SIZE_MAX, nullptr) == DG_ERR_INVALID,
                  "launched a bad description");
        }

        dg_exchange_desc x;
        memset(&x, 0, sizeof x);
        x.n_rows = count();
        x.ld = count();
        x.k = some();
        x.width = some();
        x.dtype = (int32_t)(g() % 6);
        const dg_status sx = dg_exchange_dispatch(&x, nullptr, ints, p, nullptr);
        CHECK(sx == DG_ERR_INVALID || x.n_rows == 0, "no rows");
        CHECK(dg_exchange_combine(&x, p, nullptr, floats, p, p, nullptr) == DG_ERR_INVALID || x.n_rows == 0, "no places");
        CHECK(dg_exchange_combine_backward(&x, p, ints, floats, nullptr, p, floats, nullptr) == DG_ERR_INVALID || x.n_rows == 0,
              "no gradient");

        dg_grouped_desc w;
        memset(&w, 0, sizeof w);
        w.n_rows = count();
        w.n_groups = count();
        w.k = some();
        w.n = some();
        w.dtype = (int32_t)(g() % 6);
        CHECK(dg_grouped_apply(&w, (int32_t)(g() % 5) - 1, nullptr, p, longs, p, p, p, nullptr) == DG_ERR_INVALID || w.n_rows == 0, "no x");
        CHECK(dg_grouped_apply_backward(&w, (int32_t)(g() % 5) - 1, p, p, longs, p, nullptr, p, nullptr) == DG_ERR_INVALID ||
                  w.n_rows == 0, "no gradient");
    }
    CHECK(given > 10000 && refused > 10000, "%ld given, %ld refused", given, refused);
    printf("layer operators' host code: %ld sizes given, %ld refused\n", given, refused);
    if (failures) {
        fprintf(stderr, "%d failures\n", failures);
        return 1;
    }
    printf("all checks passed\n");
    return 0;
}
