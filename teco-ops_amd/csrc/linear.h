// linear.h — how linear.hip cuts a product into tiles: host code, shared with
// the tests.
#pragma once

#include <cstddef>

namespace tecoops {

// Rows of x up to which gemv_batch.hip streams W past them.
constexpr int kLinearStreamRows = 64;
// Longest row (of x or W, in elements): 256 rows of it stay within the 32-bit
// offsets of a tile's copies.
constexpr int kLinearMaxRow = 1 << 21;

struct LinearPlan {
    int bm, bn;            // rows of x and of W per tile
    int tiles_m, tiles_n;
    int splits, stages;    // workgroups along K, stages of 64 in each
    size_t bytes;          // of workspace
};

inline LinearPlan linear_plan(int m, int n, int k, bool gated, bool copy, size_t workspace, int cus) {
    const auto up = [](long long a, long long b) { return static_cast<int>((a + b - 1) / b); };
    const long long wrows = gated ? 2LL * n : n;
    LinearPlan p{};
    p.bm = p.bn = 256;
    const auto cut = [&] {
        p.tiles_m = up(m, p.bm);
        p.tiles_n = gated ? up(n, p.bn / 2) : up(n, p.bn);
    };
    cut();
    if (!copy || static_cast<long long>(p.tiles_m) * p.tiles_n < cus) {
        p.bm = p.bn = 128;
        cut();
    }
    p.splits = 1;
    p.stages = up(k, 64);
    const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
    if (p.bm == 128 && tiles < cus) {
        int want = static_cast<int>(2 * cus / tiles);  // two workgroups to a CU
        if (want > p.stages / 8) want = p.stages / 8;  // 512 of K each or more
        while (want > 1 && static_cast<size_t>(want) * m * wrows * 4 > workspace) --want;
        if (want > 1) {
            const int per = up(p.stages, want);
            p.splits = up(p.stages, per);
            p.stages = per;
        }
    }
    p.bytes = p.splits > 1 ? static_cast<size_t>(p.splits) * m * wrows * 4 : 0;
    return p;
}

}  // namespace tecoops
