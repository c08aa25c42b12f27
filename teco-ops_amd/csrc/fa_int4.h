// fa_int4.h — host-side plan of attention over the 4-bit cache (fa_int4.hip).
#pragma once

#include <algorithm>
#include <cstddef>

namespace tecoops {
namespace fa4 {

// The split route serves `cols` (query head of a group, query row) pairs of each
// sequence and kv head in tiles of 16 * ct columns, over keys cut into splits.
struct Plan {
    bool split;      // the split route, else query tiles over all their keys
    int rows;        // the bound on a sequence's query rows
    int ct, tiles;   // column tiles of 16 in a workgroup, and such workgroups
    int cols;        // columns of a sequence and kv head in the workspace
    int split_len, splits;
    size_t bytes;    // workspace: partial states where splits > 1
};

constexpr int kWaves = 4;              // of a workgroup
constexpr int kLeastSplit = 32 * kWaves;  // keys: a block of 32 for each wave

inline size_t state_bytes(int batch, int kv_heads, int splits, int cols, int head_size) {
    return splits <= 1 ? 0
                       : static_cast<size_t>(batch) * kv_heads * splits * cols * (head_size + 2) * sizeof(float);
}

// rows, keys: bounds on a sequence's query rows and keys; room: the workspace's
// bytes; cus: compute units.
inline Plan make_plan(int batch, int heads, int kv_heads, int head_size, int rows, int keys, size_t room, int cus) {
    Plan p{};
    const long long group = heads / kv_heads;
    const long long cols = group * rows;
    p.rows = rows;
    p.split = cols <= 64;
    if (!p.split) return p;
    p.cols = static_cast<int>(cols);
    p.ct = cols <= 16 ? 1 : 2;
    p.tiles = static_cast<int>((cols + 16 * p.ct - 1) / (16 * p.ct));
    // as long as the grid has four workgroups a CU, else down to one block a wave
    const long long units = static_cast<long long>(batch) * kv_heads * p.tiles;
    long long len = 2048;
    while (len > kLeastSplit && units * ((keys + len - 1) / len) < 4ll * cus) len /= 2;
    const auto splits = [&](long long l) { return std::max(1ll, (keys + l - 1) / l); };
    while (splits(len) > 1 && state_bytes(batch, kv_heads, static_cast<int>(splits(len)), p.cols, head_size) > room)
        len *= 2;
    p.split_len = static_cast<int>(std::min(len, 1ll << 30));
    p.splits = static_cast<int>(splits(len));
    p.bytes = state_bytes(batch, kv_heads, p.splits, p.cols, head_size);
    return p;
}

}  // namespace fa4
}  // namespace tecoops
