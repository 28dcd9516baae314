// Host-side sanitizer driver for dg_grouped_apply_gradients, test infrastructure only:
// tests/test_grouped_gradients_sanitizers.py compiles the library's sources with AddressSanitizer and
// UndefinedBehaviorSanitizer on the host code together with this file and runs it without a GPU.
// Random and extreme descriptions: a size is given or refused with a message, and every call here
// has to be refused before anything is launched.
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

int main()
{
    std::mt19937_64 g(21);
    char buffer[64];
    void* const p = buffer;  // (nothing is read or written through it)
    long given = 0, refused = 0;
    for (int i = 0; i < 200000; ++i) {
        auto upto = [&](int64_t most) {
            switch (g() % 6) {
                case 0: return most;
                case 1: return most + 1;
                case 2: return (int64_t)0;
                case 3: return -(int64_t)(g() % 3);
                default: return (int64_t)(g() % (uint64_t)(g() % 2 ? most : 1000)) + 1;
            }
        };
        dg_grouped_desc d;
        memset(&d, 0, sizeof d);
        d.n_rows = upto(1ll << 40);
        d.n_groups = upto(1 << 20);
        d.k = (int32_t)upto(1 << 20);
        d.n = (int32_t)upto(1 << 20);
        d.dtype = g() % 4 ? (g() % 2 ? DG_BF16 : DG_F32) : (int32_t)(g() % 8) - 1;
        const size_t all = dg_grouped_apply_workspace_size(&d), sums = dg_grouped_workspace_size(&d);
        CHECK((all == 0) == (sums == 0), "one size of two");
        const int32_t act = 1 + (int32_t)(g() % 2);
        if (!all) {
            ++refused;
            CHECK(strlen(dg_last_error()) > 0, "size 0 without an error message");
            CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, p, p, p, p, p, ~(size_t)0, nullptr) == DG_ERR_INVALID, "bad desc");
            continue;
        }
        ++given;
        CHECK(all >= sums && all - sums >= (size_t)d.n_rows * (size_t)d.n * 4, "no room for the activation's gradient");
        CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, p, p, p, p, p, all - 1, nullptr) == DG_ERR_WORKSPACE, "small");
        CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, p, p, p, p, nullptr, all, nullptr) == DG_ERR_WORKSPACE, "none");
        if (all > sums)
            CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, p, p, nullptr, nullptr, p, all - sums - 1, nullptr) ==
                      DG_ERR_WORKSPACE, "small without sums");
        CHECK(dg_grouped_apply_gradients(&d, act, p, p, nullptr, p, p, p, p, p, p, all, nullptr) == DG_ERR_INVALID, "no sizes");
        CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, p, p, nullptr, p, p, all, nullptr) == DG_ERR_INVALID, "dbias alone");
        CHECK(dg_grouped_apply_gradients(&d, 3 + (int32_t)(g() % 5), p, p, (int64_t*)p, p, p, p, p, p, p, all, nullptr) == DG_ERR_INVALID, "act");
        if (d.n_rows > 0)
            CHECK(dg_grouped_apply_gradients(&d, act, p, p, (int64_t*)p, p, nullptr, p, p, p, p, all, nullptr) == DG_ERR_INVALID, "no gradient");
    }
    CHECK(given > 10000 && refused > 10000, "%ld given, %ld refused", given, refused);
    if (failures) {
        fprintf(stderr, "%d failures\n", failures);
        return 1;
    }
    printf("all checks passed\n");
    return 0;
}
