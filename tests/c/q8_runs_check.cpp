// Host check of the cut into runs (csrc/sp_q8_runs.h): every tile belongs to one
// run, a tile's run is found again, and differences of places' low 32 bits hold,
// for totals on both sides of 2^32.
#include <cstdio>

#include "sp_q8_runs.h"

static int fails = 0;
#define CHECK(x)                                                              \
    do {                                                                      \
        if (!(x)) {                                                           \
            printf("total %llu, grid %u, run %u: %s\n", total, grid, i, #x);  \
            fails++;                                                          \
        }                                                                     \
    } while (0)

int main()
{
    using namespace q8;
    const unsigned long long totals[] = {0, 1, 2, 147, 148, 149, 4095, 1000003, (1ull << 31) - 1, 1ull << 31, (1ull << 32) - 1,
                                         1ull << 32, (1ull << 32) + 1, (1ull << 32) + 147, 3ull << 32, (1ull << 37) + 12345,
                                         147ull << 31};
    const unsigned grids[] = {1, 2, 148, 160};
    for (unsigned long long total : totals) {
        for (unsigned grid : grids) {
            if ((total + grid - 1) / grid >= (1ull << 31)) continue;      // a run longer than it may be
            const LongRuns s = long_runs_of(total, grid);
            unsigned i = 0;
            CHECK(s.n == (total < grid ? total : grid));
            CHECK(run_begin(s, s.n) == total);
            for (i = 0; i < s.n; i++) {
                const unsigned long long b = run_begin(s, i), e = run_begin(s, i + 1);
                CHECK(b < e && e - b - total / s.n <= 1);
                CHECK(run_of_tile(s, b) == i && run_of_tile(s, e - 1) == i && run_of_tile(s, b + (e - b) / 2) == i);
                // a run as the kernel walks it: low 32 bits of its end, of a unit that
                // began before it and of one that goes on past it
                CHECK((unsigned long long)apart((unsigned)e, (unsigned)b) == e - b);
                CHECK(apart((unsigned)(b - 77), (unsigned)b) == -77);
                CHECK(b + apart((unsigned)(e + 9), (unsigned)b) == e + 9 || e - b + 9 >= (1ull << 31));
            }
        }
    }
    if (!fails) printf("ok\n");
    return fails != 0;
}
