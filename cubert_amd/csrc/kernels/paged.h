// What the kernels of a key/value cache in pages have in common.
#pragma once

namespace cubert {

// Whether no two elements of pools [pages, heads, page, size] with these strides (rows are contiguous) share a place: the dimensions, from
// the closest to the farthest, each step over all that the closer ones reach.
inline bool pages_apart(long long page_stride, long long head_stride, long long row_stride, long long pages, long long heads, long long page,
                        long long size) {
    long long stride[3] = {page_stride, head_stride, row_stride}, count[3] = {pages, heads, page};
    for (int i = 0; i < 3; ++i)
        if (count[i] == 1) stride[i] = 1ll << 62;  // never stepped
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
            if (stride[j] > stride[j + 1]) {
                const long long s = stride[j], c = count[j];
                stride[j] = stride[j + 1], count[j] = count[j + 1], stride[j + 1] = s, count[j + 1] = c;
            }
    long long reach = size;
    for (int i = 0; i < 3; ++i) {
        if (count[i] == 1) continue;
        if (stride[i] < reach || stride[i] > (1ll << 61) / count[i]) return false;
        reach = stride[i] * (count[i] - 1) + reach;
    }
    return true;
}

}  // namespace cubert
