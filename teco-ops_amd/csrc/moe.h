// moe.h — how moe.hip cuts a mixture-of-experts layer into work items and where
// they lie in its workspace: host code, shared with the tests.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace tecoops {

constexpr int kMoeMaxExperts = 1024;
constexpr int kMoeMaxTopK = 32;
constexpr int kMoeMaxTokens = 1 << 30;  // slices are counted in 32 bits
constexpr int kMoeMaxWidth = 1 << 16;  // the threads of every grid stay below 2^32
constexpr int kMoeFew = 8;  // tokens that route, and sum over the experts, within the products
constexpr int kMoeSlice = 512;  // tokens routed together; more run slice by slice

// Rows of x staged for an item: the tokens of an expert go through in chunks of
// this many, and W is read again for each.  Few tokens never need a second one;
// many take the size that an even spread over the experts fills about half, so
// that few experts overflow it (a skewed routing does, and reads W again).
inline int moe_rows(int tokens, int top_k, int experts) {
    if (tokens <= 4) return 4;
    if (tokens <= 8) return 8;
    if (tokens <= 16) return 16;
    const int even = (tokens * top_k + experts - 1) / experts;
    return even <= 8 ? 16 : even <= 20 ? 32 : 64;
}

struct MoeSpace {
    int pairs, items;      // most (token, expert) pairs and items of a slice
    int rows;              // of x per item
    long long h_stride;    // values between the rows of h, 4 bytes each
    size_t items_at, ids_at, token_at, slot_at, weight_at, cols_at, h_at, part_at;  // bytes
    size_t bytes;
};

inline MoeSpace moe_space(int tokens, int hidden, int inter, int experts, int top_k) {
    MoeSpace s{};
    const int slice = tokens < kMoeSlice ? tokens : kMoeSlice;
    s.pairs = slice * top_k;
    s.rows = moe_rows(slice, top_k, experts);
    s.items = experts + s.pairs / s.rows;
    if (s.items > s.pairs) s.items = s.pairs;
    s.h_stride = (inter + 7) / 8 * 8LL;
    size_t at = 256;  // the number of items
    const auto take = [&](size_t bytes) {
        const size_t from = at;
        at = (at + bytes + 255) / 256 * 256;
        return from;
    };
    s.items_at = take(16 * static_cast<size_t>(s.items));
    s.ids_at = take(4 * static_cast<size_t>(s.pairs));
    s.token_at = take(4 * static_cast<size_t>(s.pairs));
    s.slot_at = take(4 * static_cast<size_t>(s.pairs));
    s.weight_at = take(4 * static_cast<size_t>(s.pairs));
    s.cols_at = take(slice <= kMoeFew ? 8 * static_cast<size_t>(s.items) * kMoeFew : 0);
    s.h_at = take(4 * static_cast<size_t>(s.pairs) * s.h_stride);
    s.part_at = take(4 * static_cast<size_t>(s.pairs) * hidden);
    s.bytes = at;
    return s;
}

// Experts that `tokens` random choices of top_k reach, expected.
inline double moe_reached(int tokens, int top_k, int experts) {
    double missed = 1.0;
    for (int t = 0; t < tokens && missed > 1e-3; ++t) missed *= 1.0 - static_cast<double>(top_k) / experts;
    return experts * (1.0 - missed);
}

// Whether few tokens sum over the experts within the second product.  It spares
// the parts, their sum and a launch, about 5 us, but has a workgroup per 8 (or
// 16) rows of the result only, which leave part of the chip's bandwidth when they
// are few (6 tokens, 6 of 60 experts of [640, 9920]: 289 us, 182 in parts; 1 token,
// 3 of 4 of [1024, 896]: 12.6 and 14.7 us).
inline bool moe_out_few(int tokens, int hidden, int inter, int experts, int top_k, int cus) {
    if (tokens > kMoeFew) return false;
    const double bytes = 2.0 * hidden * inter * moe_reached(tokens, top_k, experts);
    const double share = (hidden + 7) / 8 / (0.875 * cus);
    return bytes / (5.8e6 * (share < 1 ? share : 1)) <= bytes / 5.5e6 + 5;
}

// Rows of W per workgroup: the size whose busiest CU copies the fewest bytes of
// W and x (`rows` rows of 16-bit values, or twice as many of two-term ones), with as
// many items as tokens spread evenly would make.
inline int moe_wrows(int wrows, int tokens, int top_k, int experts, int rows, int cus) {
    const double items = moe_reached(tokens, top_k, experts);
    int best = 0;
    double least = 0;
    for (int r : {128, 64, 32, 16}) {
        const long long wgs = static_cast<long long>(items + 0.5) * ((wrows + r - 1) / r);
        const double bytes = static_cast<double>((wgs + cus - 1) / cus) * (2.0 * r + 2.0 * rows);
        if (best == 0 || bytes < least) {
            least = bytes;
            best = r;
        }
    }
    return best;
}

}  // namespace tecoops
