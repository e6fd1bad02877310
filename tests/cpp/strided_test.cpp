// levo::overlap and Strided::distinct against sets of element offsets, on small tensors drawn at random, and on the
// layouts that calls have.
#include <cstdio>
#include <random>
#include <set>

#include "strided.h"

namespace {

std::multiset<int64_t> elements(const levo::Strided &t, int64_t element) {
    std::multiset<int64_t> all;
    for (int64_t i = 0; i < t.size[0]; ++i)
        for (int64_t j = 0; j < t.size[1]; ++j)
            for (int64_t k = 0; k < t.size[2]; ++k)
                for (int64_t l = 0; l < t.inner; ++l)
                    all.insert(static_cast<int64_t>(t.at) / element + i * t.stride[0] + j * t.stride[1] +
                               k * t.stride[2] + l);
    return all;
}

int failures = 0;
void expect(bool ok, const char *what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what);
    ++failures;
}

}  // namespace

int main() {
    std::mt19937_64 rng(1);
    auto below = [&](int64_t n) { return static_cast<int64_t>(rng() % static_cast<uint64_t>(n)); };
    int shared = 0, apart = 0, distinct = 0;
    for (int round = 0; round < 40000; ++round) {
        levo::Strided t[2];
        const int64_t element = round % 2 ? 2 : 4, wide = 1 + below(60);
        for (auto &x : t) {
            x.at = static_cast<uintptr_t>(element * (1000 + below(1 + wide * 3)));
            x.inner = 1 + below(5);
            for (int i = 0; i < 3; ++i) x.size[i] = below(20) ? 1 + below(4) : 0, x.stride[i] = below(wide);
        }
        if (below(2))
            for (int i = 0; i < 3; ++i) t[1].stride[i] = t[0].stride[i];
        const auto a = elements(t[0], element), b = elements(t[1], element);
        bool common = false;
        for (int64_t e : a) common = common || b.count(e) > 0;
        expect(levo::overlap(t[0], t[1], element) == common, "overlap of a random pair");
        expect(levo::overlap(t[1], t[0], element) == common, "overlap the other way round");
        ++(common ? shared : apart);
        if (t[0].last() >= 0) {  // distinct() may refuse a layout that interleaves, never take one that repeats
            const bool once = std::set<int64_t>(a.begin(), a.end()).size() == a.size();
            expect(!t[0].distinct() || once, "distinct elements repeat");
            distinct += t[0].distinct();
        }
    }
    expect(shared > 3000 && apart > 3000 && distinct > 3000, "the draws meet both answers");

    // q, k and v side by side in a projection's output, turned in place; a transposed copy behind it
    const int64_t B = 64, S = 16001, H = 32, D = 128, row = 3 * H * D;
    const uintptr_t base = 1 << 20;
    auto view = [&](int64_t offset, int64_t b, int64_t s, int64_t h, int64_t tokens) {
        return levo::Strided{base + static_cast<uintptr_t>(2 * offset), {b, s, h}, {B, tokens, H}, D};
    };
    const auto q = view(0, S * row, row, D, S), k = view(H * D, S * row, row, D, S);
    expect(!levo::overlap(q, k, 2), "q beside k");
    expect(levo::overlap(q, view(H * D - 1, S * row, row, D, S), 2), "k one element too early");
    expect(levo::overlap(q, view(row, S * row, row, D, S - 1), 2), "q one token on");
    expect(!levo::overlap(q, view(B * S * row, H * S * D, D, S * D, S), 2), "behind the whole");
    expect(levo::overlap(q, view(B * S * row - 1 - 2 * H * D, H * S * D, D, S * D, S), 2), "at its last element");
    expect(!levo::overlap(q, view(B * S * row - 2 * H * D, H * S * D, D, S * D, S), 2), "right behind it");
    expect(levo::overlap(q, view(5 * row + H * D, H * S * D, D, S * D, S), 2), "transposed, inside");
    // odd rows against even ones, and strides that meet late
    expect(!levo::overlap(view(0, 4 * S * row, 2 * row, D, S), view(row, 4 * S * row, 2 * row, D, S), 2), "every other row");
    levo::Strided x{base, {0, 1000, 0}, {1, 5000, 1}, 1}, y{base + 2 * 999, {0, 1001, 0}, {1, 5000, 1}, 1};
    expect(levo::overlap(x, y, 2), "1000 i = 1001 j + 999 at j = 1");
    y.size[1] = 1;
    expect(!levo::overlap(x, y, 2), "not at j = 0");
    // as far out as the checks let strides go
    const int64_t far = int64_t(1) << 59;
    levo::Strided u{base, {far, far, far}, {2, 2, 2}, 8}, w{base + 16, {far, far, far}, {2, 2, 2}, 1};
    expect(!levo::overlap(u, w, 2), "far strides, one element beyond the run");
    w.stride[0] = far - 1;
    expect(levo::overlap(u, w, 2), "8 + (far - 1) is the last element of the run at far");
    w.stride[0] = far;
    w.at = base + 14;
    expect(levo::overlap(u, w, 2), "far strides, the run's last element");
    if (failures == 0) std::printf("strided: ok\n");
    return failures != 0;
}
