// test_spans.cpp -- distances of rows and heads that a call takes or refuses (vq_b200/csrc/spans.hpp).  Built and run by tests/test_spans.py.
#include <cstdio>
#include <cstring>

#include "../../vq_b200/csrc/spans.hpp"

using namespace vqb;
typedef unsigned __int128 wide;

static int failed = 0;
static void expect(bool ok, const char *what, size_t n, size_t heads, size_t width, size_t ld, size_t head_ld)
{
    if (!ok) std::printf("FAIL %s: n %zu heads %zu width %zu ld %zu head_ld %zu\n", what, n, heads, width, ld, head_ld), ++failed;
}

int main()
{
    const size_t one = 1;
    const size_t steps[] = {0, 1, 3, 4, 64, 1000, one << 20, one << 28, (one << 28) + 1, one << 34, one << 40, (one << 40) + 1, one << 41, one << 53, one << 57, one << 58, one << 62, one << 63, ~size_t(0)};
    const size_t rows[] = {1, 2, 3, 65, (one << 23) + 1, (one << 24) + 1, (one << 30) - 1}, all_heads[] = {1, 2, 8, 4096}, widths[] = {1, 4, 256};
    int taken = 0;
    for (size_t n : rows)
        for (size_t heads : all_heads)
            for (size_t width : widths)
                for (size_t ld : steps)
                    for (size_t head_ld : steps) {
                        const char *fault = heads_fault(n, heads, width, ld, head_ld);
                        if (fault) continue;
                        ++taken;
                        // what is taken reaches as far as its numbers say, in bytes too
                        const wide far = (wide)(n - 1) * ld + (wide)(heads - 1) * head_ld + width;
                        expect(far * 4 < (wide(1) << 63) && far == heads_values(n, heads, width, ld, head_ld), "a span that leaves 64 bits is taken", n, heads, width, ld, head_ld);
                        // and no two rows of any heads share a value
                        const bool heads_inside = (heads == 1 || head_ld >= width) && (n == 1 || (wide)ld >= (wide)(heads - 1) * head_ld + width);
                        const bool rows_inside = (n == 1 || ld >= width) && (heads == 1 || (wide)head_ld >= (wide)(n - 1) * ld + width);
                        expect(heads_inside || rows_inside, "rows that overlap are taken", n, heads, width, ld, head_ld);
                    }
    expect(taken > 500, "hardly anything is taken", taken, 0, 0, 0, 0);
    for (size_t n : rows)
        for (size_t ld : steps) expect(too_far(n, ld) == ((wide)(n - 1) * ld > MOST_SPAN), "rows alone", n, 1, 0, ld, 0);
    // the bytes of these came out as 8, 0 and 0
    expect(heads_fault((one << 23) + 1, 1, 4, one << 40, 4), "8388609 rows 2^40 values apart", 0, 0, 0, 0, 0);
    expect(heads_fault((one << 24) + 1, 1, 4, one << 40, 4), "16777217 rows 2^40 values apart", 0, 0, 0, 0, 0);
    expect(heads_fault(2, 1, 4, one << 63, 4), "2 rows 2^63 values apart", 0, 0, 0, 0, 0);
    // heads as far apart as many rows of one make it
    expect(!heads_fault((one << 21) + 1, 2, 128, 128, (one << 28) + 128), "2^21 + 1 rows of 128 values, head behind head", 0, 0, 0, 0, 0);
    expect(!heads_fault(3, 4096, 64, 64, one << 40), "4096 heads 2^40 values apart", 0, 0, 0, 0, 0);
    expect(heads_fault(3, 3, 64, 64, one << 58), "3 heads 2^58 values apart", 0, 0, 0, 0, 0);
    expect(heads_fault(3, 4096, 64, 64, ~size_t(0)), "heads 2^64 - 1 values apart", 0, 0, 0, 0, 0);
    // distances that do not count
    expect(!heads_fault(1, 1, 4, ~size_t(0), ~size_t(0)), "one row of one head", 0, 0, 0, 0, 0);
    std::printf("%d taken, %d failed\n", taken, failed);
    return failed != 0;
}
