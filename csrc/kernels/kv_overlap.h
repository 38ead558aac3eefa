// Whether two strided tensors share memory, decided exactly: tensors of one
// fused projection, interleaved by rows, heads or elements, span each other
// and share nothing.
#ifndef MPCOMM_B200_CSRC_KERNELS_KV_OVERLAP_H_
#define MPCOMM_B200_CSRC_KERNELS_KV_OVERLAP_H_

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <utility>

namespace mpcomm {
namespace kern {

// The elements base + sum of i_k * stride[k], 0 <= i_k < extent[k].
struct StridedSet {
    uintptr_t base = 0;
    int axes = 0;
    int64_t stride[5] = {}, extent[5] = {};
    int64_t first = 0, last = 0;  // the least and the greatest sum
    bool empty = false;
    StridedSet() = default;
    StridedSet(const void *p, std::initializer_list<std::pair<int64_t, int64_t>> strides_extents)
        : base(reinterpret_cast<uintptr_t>(p)) {
        for (const auto &a : strides_extents) {
            empty = empty || a.second <= 0;
            if (a.second <= 1 || a.first == 0) continue;  // one place, however it is reached
            stride[axes] = a.first;
            extent[axes++] = a.second;
            (a.first > 0 ? last : first) += a.first * (a.second - 1);
        }
    }
    // The same places in the same order.
    bool operator==(const StridedSet &o) const {
        return base == o.base && axes == o.axes && std::equal(stride, stride + axes, o.stride) &&
               std::equal(extent, extent + axes, o.extent);
    }
};

struct OverlapAxis {
    int64_t stride, lo, hi;  // stride > 0
};

// Whether some lo_k <= d_k <= hi_k give sum of d_k * stride_k = target; axes by falling stride. Where the strides are
// nested, as in any slice of a tensor, an axis leaves one or two values to try. Sets that are not end at `tries`, as
// sets that meet.
inline bool sum_reaches(const OverlapAxis *axis, int n, int64_t target, int *tries) {
    if (n == 0) return target == 0;
    if (--*tries < 0) return true;
    int64_t least = 0, most = 0;
    for (int k = 1; k < n; ++k) {
        least += axis[k].lo * axis[k].stride;
        most += axis[k].hi * axis[k].stride;
    }
    const int64_t s = axis[0].stride;
    auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t first = std::max(axis[0].lo, -floor_div(most - target, s)), last = std::min(axis[0].hi, floor_div(target - least, s));
    for (int64_t d = first; d <= last; ++d)
        if (sum_reaches(axis + 1, n - 1, target - d * s, tries)) return true;
    return false;
}

// Whether elements of `size` bytes of the two sets share a byte.
inline bool sets_overlap(const StridedSet &a, const StridedSet &b, int size) {
    if (a.empty || b.empty) return false;
    const int64_t bytes = static_cast<int64_t>(b.base - a.base);
    if (bytes + b.first * size >= (a.last + 1) * size || bytes + (b.last + 1) * size <= a.first * size) return false;
    OverlapAxis axis[10];
    int n = 0;
    // of a: 0 .. extent - 1, of b: the same, subtracted
    auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
        if (stride < 0) stride = -stride, lo = -lo, hi = -hi, std::swap(lo, hi);
        for (int k = 0; k < n; ++k)
            if (axis[k].stride == stride) {
                axis[k].lo += lo;
                axis[k].hi += hi;
                return;
            }
        axis[n++] = OverlapAxis{stride, lo, hi};
    };
    for (int k = 0; k < a.axes; ++k) add(a.stride[k], 0, a.extent[k] - 1);
    for (int k = 0; k < b.axes; ++k) add(b.stride[k], 1 - b.extent[k], 0);
    std::sort(axis, axis + n, [](const OverlapAxis &x, const OverlapAxis &y) { return x.stride > y.stride; });
    const int64_t at = bytes / size - (bytes % size < 0);  // rounded down
    int tries = 4096;
    return sum_reaches(axis, n, at, &tries) || (bytes % size && sum_reaches(axis, n, at + 1, &tries));
}

}  // namespace kern
}  // namespace mpcomm

#endif  // MPCOMM_B200_CSRC_KERNELS_KV_OVERLAP_H_
