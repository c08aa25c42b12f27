// linear.h — how linear.hip cuts a product into tiles: host code, shared with
// the tests.
#pragma once

#include "gemv_batch.h"

#include <cstddef>
#include <cstdint>

namespace tecoops {

// Rows of x up to which gemv_batch.hip can stream W past them.
constexpr int kLinearStreamRows = 64;
// Longest row (of x or W, in elements): 256 rows of it stay within the 32-bit
// offsets of a tile's copies.
constexpr int kLinearMaxRow = 1 << 21;
constexpr int kLinearMaxOutputs = 1 << 23;

// The tiles built: rows of x and of W, stages in the ring, workgroups that fit a
// CU, and the microseconds of a workgroup on 256 CUs: per stage of 64 of K at
// full CUs, per stage at least (its copies' way), and besides its stages.  Fitted
// to the times of all tiles and splits over 127 products (m 65..8000, n
// 256..14336, k 256..14336, bf16), on which the size and split of the least
// estimate take 1.3 % longer than the best in the mean, 21 % at most.  One tile
// for all is worse by up to: 256 x 256 3.1 times, 64 x 64 2.4 times.
struct LinearTile {
    int bm, bn, depth, occupancy;
    float stage, latency, besides;
};
constexpr LinearTile kLinearTiles[] = {
    {256, 256, 2, 1, 0.097f, 1.405f, 8.4f},
    {128, 256, 3, 1, 0.057f, 0.809f, 5.0f},
    {128, 128, 3, 1, 0.033f, 0.507f, 4.0f},
    {64, 128, 3, 2, 0.353f, 0.008f, 3.0f},
    {64, 64, 3, 3, 0.225f, 0.267f, 3.1f},
};
constexpr int kLinearTileCount = sizeof(kLinearTiles) / sizeof(kLinearTiles[0]);
// Tiles whose rows can also be loaded through registers (the larger ones have no
// registers left to hold a stage).
constexpr int kLinearFirstLoaded = 2;

struct LinearPlan {
    bool stream;           // gemv_batch.hip takes it (the rest is 0)
    int tile;              // of kLinearTiles
    int tiles_m, tiles_n;
    int splits, stages;    // workgroups along K, stages of 64 in each
    size_t bytes;          // of workspace
};

// copy: rows in whole 16-byte words.  workspace: bytes there are for the sums of
// a split K.
inline LinearPlan linear_plan(int m, int n, int k, bool gated, bool copy, size_t workspace, int cus) {
    const auto up = [](int a, int b) { return (a - 1) / b + 1; };
    const long long wrows = gated ? 2LL * n : n;
    LinearPlan best{};
    // Streamed: HBM's rate for W, or a CU's for the rows of W and x it copies; in
    // tiles W is read at 5.5 TB/s at best.  Few rows of W with a long K leave the
    // copies of x, which every workgroup makes: [1024, 14336], 64 rows, 32.2 us
    // streamed, 15.7 in tiles; [14336, 4096], 32 rows, 21.5 and 27.8.  Over 96
    // products (m 8..64) the choice is 0.7 % slower than the better in the mean,
    // 11 % at most.
    double streamed = -1;
    if (copy && m <= kLinearStreamRows) {
        const int rows = gemv_batch_rows(static_cast<int>(wrows), k, m, false, cus, gated ? 16 : 8);
        const double hbm = 2.0 * wrows * k / 6.6e6;
        const double lds = static_cast<double>(gemv_batch_bytes(wrows, rows, gemv_batch_staged(m), false, cus)) *
                           k / 65e3;
        streamed = 3.2 + (hbm > lds ? hbm : lds);
        best.stream = streamed <= 6.2 + 2.0 * wrows * k / 5.5e6;
        if (best.stream) return best;
    }
    const int all = up(k, 64);
    double least = 0;
    for (int t = copy ? 0 : kLinearFirstLoaded; t < kLinearTileCount; ++t) {
        const LinearTile &c = kLinearTiles[t];
        const int tm = up(m, c.bm), tn = up(n, gated ? c.bn / 2 : c.bn);
        const long long tiles = static_cast<long long>(tm) * tn;
        for (const int want : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16}) {
            // a split of 256 of K or more, where tiles alone do not fill the CUs
            // and with workspace for its sums
            if (want > 1 && (tiles * (want - 1) >= static_cast<long long>(cus) * c.occupancy || all < 4 * want)) break;
            const int per = up(all, want), splits = up(all, per);
            const size_t bytes = splits > 1 ? static_cast<size_t>(splits) * m * wrows * 4 : 0;
            if (bytes > workspace) break;
            if (splits != want) continue;
            const long long wgs = tiles * splits;
            const int each = wgs > 0x7fffffff ? 0x7fffffff : up(static_cast<int>(wgs), cus);  // of a CU
            const int rounds = up(each, c.occupancy);
            const double busy = static_cast<double>(each) * per * c.stage;
            const double wait = static_cast<double>(rounds) * per * c.latency;
            double time = 2.2 + static_cast<double>(rounds) * c.besides + (busy > wait ? busy : wait);
            if (splits > 1) time += 1.4 + splits * 8.0 * m * wrows / 7e6;  // written and read again
            if (least == 0 || time < least) {
                least = time;
                best.tile = t;
                best.tiles_m = tm;
                best.tiles_n = tn;
                best.splits = splits;
                best.stages = per;
                best.bytes = bytes;
            }
        }
    }
    if (streamed >= 0 && streamed <= least) {
        best.stream = true;
        best.bytes = 0;
    }
    return best;
}

// Whether rows of x and W can be copied into LDS: in whole, aligned 16-byte words.
inline bool linear_copies(int k, long long x_stride, const void *x, const void *weight) {
    const auto whole = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return k % 8 == 0 && x_stride % 8 == 0 && whole(x) && whole(weight);
}

// Bytes of workspace that such a product can use (linear.hip).
size_t linear_workspace(int m, int n, int k, bool gated, bool copy);

}  // namespace tecoops
