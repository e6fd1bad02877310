// Which elements a strided tensor [size0][size1][size2][inner] names: whether all are distinct, and whether two
// tensors share one.  Host code without CUDA; strides are not negative, and a stride times its size is below 2^60.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace levo {

struct Strided {
    uintptr_t at;
    int64_t stride[3], size[3], inner;  // in elements, the inner dimension's is 1

    int64_t last() const {  // offset of the last element; -1: none
        int64_t e = inner - 1;
        for (int i = 0; i < 3; ++i) {
            if (size[i] <= 0 || inner <= 0) return -1;
            e += stride[i] * (size[i] - 1);
        }
        return e;
    }

    // Sorted by stride, each dimension steps past all that the smaller ones reach.
    bool distinct() const {
        int64_t reach = inner;
        bool done[3] = {false, false, false};
        for (int round = 0; round < 3; ++round) {
            int least = -1;
            for (int i = 0; i < 3; ++i)
                if (!done[i] && (least < 0 || stride[i] < stride[least])) least = i;
            done[least] = true;
            if (size[least] <= 1) continue;
            if (stride[least] < reach) return false;
            reach += stride[least] * (size[least] - 1);
        }
        return true;
    }
};

// Whether a and b share an element: whether integers within the sizes solve
//   sum of i_k a.stride_k - sum of j_k b.stride_k = (b.at - a.at) + (a place in b's inner run - one in a's),
// the right side an interval.  A dimension that steps no wider than the interval only widens it; the others are
// tried from the widest stride down, each by the few steps that what is left can make up for.  Sensible layouts take
// some ten trials; strides that take kTrials count as overlapping.
inline bool overlap(const Strided &a, const Strided &b, size_t element) {
    const int64_t a_last = a.last(), b_last = b.last();
    if (a_last < 0 || b_last < 0) return false;
    const int64_t apart =
        static_cast<int64_t>(b.at - a.at) / static_cast<int64_t>(element);  // both are aligned to an element
    if (apart > a_last || -apart > b_last) return false;

    struct Term {
        int64_t stride, from, to;
    } terms[6];
    int n = 0;
    auto add = [&](int64_t stride, int64_t from, int64_t to) {
        if (stride == 0 || from == to) return;
        int i = 0;
        while (i < n && terms[i].stride > stride) ++i;
        if (i < n && terms[i].stride == stride) {
            terms[i].from += from, terms[i].to += to;
            return;
        }
        std::copy_backward(terms + i, terms + n, terms + n + 1);
        terms[i] = {stride, from, to};
        ++n;
    };
    for (int i = 0; i < 3; ++i) {
        add(a.stride[i], 0, a.size[i] - 1);
        add(b.stride[i], 1 - b.size[i], 0);
    }
    int64_t low = apart - (a.inner - 1), high = apart + (b.inner - 1);
    while (n > 0 && terms[n - 1].stride <= high - low + 1) {
        const Term &t = terms[--n];
        low -= t.stride * t.to;
        high -= t.stride * t.from;
    }
    int64_t least[7], most[7];  // of the terms from the k-th on
    least[n] = most[n] = 0;
    for (int k = n - 1; k >= 0; --k) {
        least[k] = least[k + 1] + terms[k].stride * terms[k].from;
        most[k] = most[k + 1] + terms[k].stride * terms[k].to;
    }
    constexpr int kTrials = 1 << 18;
    struct Search {
        const Term *terms;
        const int64_t *least, *most;
        int n, left;
        static int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y < 0); }
        bool solve(int k, int64_t low, int64_t high) {
            if (k == n) return low <= 0 && high >= 0;
            const Term &t = terms[k];
            const int64_t from = std::max(t.from, -floor_div(most[k + 1] - low, t.stride));
            const int64_t to = std::min(t.to, floor_div(high - least[k + 1], t.stride));
            for (int64_t c = from; c <= to; ++c)
                if (--left < 0 || solve(k + 1, low - c * t.stride, high - c * t.stride)) return true;
            return false;
        }
    } search{terms, least, most, n, kTrials};
    return search.solve(0, low, high);
}

}  // namespace levo
