// rows_overlap (csrc/gpx_overlap.hpp) against the list of all rows, over random layouts and some at the ends.
#include <cstdio>
#include <random>
#include <vector>

#include "gpx_overlap.hpp"

using gpxh::rows_overlap;

static bool listed(const std::array<int64_t, 3> &s, const std::array<int64_t, 3> &n, int64_t dim)
{
    std::vector<int64_t> at;
    for (int64_t i = 0; i < n[0]; ++i)
        for (int64_t j = 0; j < n[1]; ++j)
            for (int64_t k = 0; k < n[2]; ++k)
                at.push_back(i * s[0] + j * s[1] + k * s[2]);
    std::sort(at.begin(), at.end());
    for (size_t i = 1; i < at.size(); ++i)
        if (at[i] - at[i - 1] < dim)
            return true;
    return false;
}

static int wrong = 0;
static void expect(const std::array<int64_t, 3> &s, const std::array<int64_t, 3> &n, int64_t dim, int want)
{
    const int got = rows_overlap(s, n, dim);
    if (got != want) {
        printf("strides %lld %lld %lld, %lld x %lld x %lld rows of %lld: %d instead of %d\n", (long long)s[0], (long long)s[1], (long long)s[2],
               (long long)n[0], (long long)n[1], (long long)n[2], (long long)dim, got, want);
        ++wrong;
    }
}

int main()
{
    std::mt19937 g(1);
    const auto upto = [&](int n) { return (int64_t)(g() % n); };
    int yes = 0, interleaved = 0;
    for (int i = 0; i < 200000; ++i) {
        const std::array<int64_t, 3> n = {1 + upto(5), 1 + upto(6), 1 + upto(4)}, s = {8 * upto(40), 8 * upto(40), 8 * upto(40)};
        const int64_t dim = 8 * (1 + upto(4));
        const bool want = listed(s, n, dim);
        yes += want;
        interleaved += !want;
        expect(s, n, dim, want);
    }
    // dense, heads first, packed with others, a batch stride of zero, equal strides of rows and heads
    expect({768, 256, 64}, {2, 3, 4}, 64, 0);
    expect({768, 64, 192}, {2, 3, 4}, 64, 0);
    expect({2304, 768, 64}, {2, 3, 4}, 64, 0);
    expect({0, 256, 64}, {2, 3, 4}, 64, 1);
    expect({0, 256, 64}, {1, 3, 4}, 64, 0);
    expect({768, 64, 64}, {2, 3, 4}, 64, 1);
    expect({704, 256, 64}, {2, 3, 4}, 64, 1);
    // strides and counts at their ends
    expect({INT64_MAX - 7, 256, 64}, {1 << 28, 4, 4}, 64, 0);
    expect({INT64_MAX - 7, (int64_t)1 << 22, 64}, {3, 1 << 28, 4}, 64, 0);
    expect({(int64_t)1 << 50, 256, 64}, {2, 1 << 28, 4}, 64, 0);
    expect({(int64_t)1 << 35, 256, 64}, {2, 1 << 28, 4}, 64, 1);
    // neither nested nor few
    expect({40, 24, 16}, {1 << 11, 1 << 12, 1 << 11}, 8, -1);
    printf("%d overlapping, %d not, %d wrong\n", yes, interleaved, wrong);
    return wrong != 0 || yes < 1000 || interleaved < 1000;
}
