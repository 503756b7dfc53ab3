// gpx_overlap.hpp -- whether the rows of a strided output share an element (gpx_attend.hip; no HIP type, so that the CPU suite can build
// it by itself).
#pragma once
#include <algorithm>
#include <array>
#include <cstdint>

namespace gpxh {

// Rows of `dim` elements at the indices of three axes (n indices each, none negative or above 2^28; strides from 0 on): 0 no two share
// an element, 1 some do, -1 too long to tell.  Nested strides, each at least what the smaller ones span, are told at once; others by
// the distances of all pairs of rows, of which the axis with the most indices needs no loop: up to 2^20 pairs of the other two.
inline int rows_overlap(std::array<int64_t, 3> stride, std::array<int64_t, 3> n, int64_t dim)
{
    struct Axis {
        __int128 stride;
        int64_t n;
    } x[3];
    for (int i = 0; i < 3; ++i)
        x[i] = {n[i] > 1 ? stride[i] : 0, n[i]};
    std::sort(x, x + 3, [](const Axis &a, const Axis &b) { return a.stride < b.stride; });
    __int128 span = dim;
    bool nested = true;
    for (const Axis &y : x)
        if (y.n > 1) {
            if (y.stride < dim)
                return 1;
            nested = nested && y.stride >= span;
            span += y.stride * (y.n - 1);
        }
    if (nested)
        return 0;
    std::sort(x, x + 3, [](const Axis &a, const Axis &b) { return a.n < b.n; });
    if (x[0].n * x[1].n > (1 << 20))
        return -1;
    for (int64_t i = 0; i < x[0].n; ++i)
        for (int64_t j = 1 - x[1].n; j < x[1].n; ++j) {
            const __int128 at = i * x[0].stride + j * x[1].stride, far = at < 0 ? -at : at, k = far / x[2].stride;
            for (__int128 m = k; m <= k + 1; ++m) {  // the multiples of the third stride next to that distance
                const __int128 d = far - m * x[2].stride;
                if (m < x[2].n && (i || j || m) && d < dim && -d < dim)
                    return 1;
            }
        }
    return 0;
}

}  // namespace gpxh
