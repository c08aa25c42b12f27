// fa_int4.h — host-side plan of attention over the 4-bit cache (fa_int4.hip).
#pragma once

#include <algorithm>
#include <cstddef>

namespace tecoops {
namespace fa4 {

// Both routes serve the (query row, query head of a group) pairs of each sequence
// and kv head as columns, in tiles, over keys cut into splits.
struct Plan {
    bool split;      // the split route, else the tile route
    int ct;          // split route: column tiles of 16 in a workgroup
    int waves;       // tile route: waves of 32 columns in a workgroup
    int tiles;       // column tiles of a sequence and kv head
    int cols;        // its columns in them (others: the same workgroups go on to them)
    int split_len, splits;
    size_t bytes;    // workspace: partial states where splits > 1
};

constexpr int kWaves = 4;                 // of a workgroup of the split route
constexpr int kLeastSplit = 32 * kWaves;  // keys: a block of 32 for each wave
// Columns that the split route serves: two tiles of 32, past which it takes a third and the
// other is faster (split / tile route, us, bf16, 8 kv heads of 128: 16 sequences of 4096
// keys, 32 columns 38.5 / 49.7, 64 53.2 / 56.0, 72 72.2 / 63.4, 96 73.2 / 66.6; 4 of 2048, 64
// columns 20.1 / 20.2, 72 26.0 / 20.7; one of 16384, 64 columns 27.8 / 33.7, 72 34.6 / 35.3;
// 64 of 1000, 64 columns 60.1 / 56.6, 72 83.1 / 57.9).  In fp16 it serves any number: the
// widened tiles' roundings are seen there (5e-4 against 2.1e-4, rms, of the output's own).
// 8 sequences of 1000 keys, 400 columns 60 / 48 us, 4 of 4096, 8192 columns 934 / 435.
constexpr int kSplitCols = 64;

constexpr long long kMostWorkgroups = 1ll << 22;  // of a grid, whose threads stay within 32 bits
constexpr long long kMostAcross = 65535;          // of its second axis: splits (tile route: tiles * splits)

// Bound on a sequence's query rows: the caller's, at least their mean and at most all.
inline int row_bound(int max_seqlen_q, int total_q, int batch) {
    const int mean = std::max(1, static_cast<int>((static_cast<long long>(total_q) + batch - 1) / batch));
    return std::min(std::max(max_seqlen_q, mean), std::max(total_q, 1));
}

inline size_t state_bytes(int batch, int kv_heads, int splits, int cols, int head_size) {
    return splits <= 1 ? 0
                       : static_cast<size_t>(batch) * kv_heads * splits * cols * (head_size + 2) * sizeof(float);
}

// rows, keys: bounds on a sequence's query rows and keys; room: the workspace's
// bytes; cus: compute units; exact: for any number of columns the split route.  Where
// the bounds ask for more workgroups than a grid has, each takes several tiles.
inline Plan make_plan(int batch, int heads, int kv_heads, int head_size, int rows, int keys, size_t room, int cus,
                      bool exact = false) {
    Plan p{};
    const long long cols = std::min<long long>(static_cast<long long>(heads / kv_heads) * rows, 0x7fffffff);
    p.cols = static_cast<int>(cols);
    p.split = exact || cols <= kSplitCols;
    p.splits = 1;
    long long len = 0;
    const auto splits = [&](long long l) { return std::max(1ll, (keys + l - 1) / l); };
    const long long heads_all = static_cast<long long>(batch) * kv_heads;
    const auto cut = [&](long long tile) {
        p.tiles = static_cast<int>((cols + tile - 1) / tile);
        const long long most = std::min(std::max(1ll, kMostWorkgroups / heads_all), kMostAcross);
        if (p.tiles <= most) return;
        p.tiles = static_cast<int>(most);
        p.cols = static_cast<int>(most * tile);
    };
    if (p.split) {
        p.ct = cols <= 16 ? 1 : 2;
        cut(16 * p.ct);
        // 2048 keys, or as much shorter as gives each CU a workgroup, down to one block a
        // wave.  What a workgroup costs besides its keys, and the splits' states, are
        // more than a fuller chip gains (one workgroup a CU / four, us: a sequence of
        // 16384 keys 12.5 / 23.6, 8 of 2048 9.9 / 14.3, 64 of 1000 18.1 / 23.8, 16 of
        // 4096 22.6 / 23.9; heads 32 on 8 of 128)
        const long long units = heads_all * p.tiles;
        // (two tiles of 16 columns write more states: no splits where there are two
        // workgroups a CU or more, else no more than make four of them.  2048 keys a split /
        // none, us, fp16: 2 sequences of 16300 keys, 1015 columns 318 / 248, 32 of 6000, 48
        // columns 127 / 105)
        len = 2048;
        if (p.ct > 1) {
            const long long most = units >= 2ll * cus ? 1 : 4ll * cus / units, each = (keys + most - 1) / most;
            len = std::max(len, (each + 127) / 128 * 128);
        }
        while (len > kLeastSplit && units * splits(len) < cus) len /= 2;
    } else {
        const int wide = head_size <= 128 ? 12 : 8;
        p.waves = cols <= 128 ? 4 : wide;
        cut(32 * p.waves);
        // where the tiles leave workgroup slots empty, as many splits as fill them, of
        // two tiles of 96 keys or more (least 512 / 192 / 96 keys, us: one sequence of
        // 1000 keys, 96 columns 45.1 / 19.8 / 16.6, of 4096 31.9 / 22.2 / 19.7, 256
        // columns 34.0 / 26.5 / 26.9; 4 of 2048, 96 columns 32.3 / 23.0 / 24.0)
        const long long units = heads_all * p.tiles;
        const long long slots = static_cast<long long>(cus) * (p.waves == 4 ? 3 : 1);
        const long long want = std::min(slots / std::max(units, 1ll), static_cast<long long>(keys) / 192);
        len = want > 1 ? ((keys + want - 1) / want + 95) / 96 * 96 : std::max(keys, 1);
    }
    const auto too_many = [&](long long n) {
        return heads_all * p.tiles * n > kMostWorkgroups || (p.split ? 1 : p.tiles) * n > kMostAcross ||
               state_bytes(batch, kv_heads, static_cast<int>(n), p.cols, head_size) > room;
    };
    while (splits(len) > 1 && too_many(splits(len))) len *= 2;
    p.split_len = static_cast<int>(std::min(len, (1ll << 30) / 384 * 384));
    p.splits = static_cast<int>(splits(len));
    p.bytes = state_bytes(batch, kv_heads, p.splits, p.cols, head_size);
    return p;
}

}  // namespace fa4
}  // namespace tecoops
