// gemv_int4.h — how a product with 4-bit weights (gemv_int4.hip) is cut.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace tecoops {

constexpr int kGemvInt4Stage = 512;  // of K, staged at a time by the matrix-core kernel
constexpr int kGemvInt4DotK = 8192;  // the longest K of the kernel of one row of x
constexpr int kGemvInt4Rows = 64;    // rows of W of its workgroups

// Stages of a K of up to 2^31 - 1.
constexpr int gemv_int4_stages(int k) { return k <= 0 ? 0 : (k - 1) / kGemvInt4Stage + 1; }

// Elements (or bytes) of [from, from + count) that lie past `end`; from at most end + a stage.
constexpr int gemv_int4_past(int from, int count, int end) {
    return from - end + count > 0 ? from - end + count : 0;
}

// a / d as a product with 2^32 / d rounded up where that is exact for every a up to
// `most` (inv of gemv_int4_inverse), else a division: the group that a use of the
// scales lies in.
constexpr uint32_t gemv_int4_inverse(int d, int most) {
    if (d < 2) return 0;
    const uint64_t inv = ((1ull << 32) + d - 1) / d, off = inv * d - (1ull << 32);
    return static_cast<uint64_t>(most) * off < (1ull << 32) ? static_cast<uint32_t>(inv) : 0u;
}
constexpr int gemv_int4_quotient(int a, int d, uint32_t inv) {
    return d == 1 ? a : inv != 0u ? static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(a)) * inv >> 32) : a / d;
}

// Rows of x that a workgroup of it stages.
inline int gemv_int4_staged(int batch) { return batch <= 8 ? 8 : batch >= 64 ? 64 : (batch + 15) / 16 * 16; }

struct GemvInt4Plan {
    bool dot;      // the kernel of one row of x
    int parts;     // parts of K, their sums in the workspace where more than one
    size_t bytes;  // of it
};

// room: bytes of workspace.
inline GemvInt4Plan gemv_int4_plan(int batch, int n, int k, size_t room, int cus) {
    GemvInt4Plan p{};
    p.parts = 1;
    const long long staged = gemv_int4_staged(batch);
    const long long wgs = (n + kGemvInt4Rows - 1ll) / kGemvInt4Rows * ((batch + staged - 1) / staged);
    const int stages = gemv_int4_stages(k);
    const size_t part = static_cast<size_t>(batch) * n * sizeof(float);
    // as many parts as leave a workgroup a CU, two stages each or more
    const long long most = std::min<long long>(cus / std::max(wgs, 1ll), stages / 2);
    p.parts = static_cast<int>(std::max(1ll, std::min<long long>(most, static_cast<long long>(room / part))));
    // one row where K would be split, which takes a second launch (us, dot / this and
    // the sums of its parts, fp16, groups of 128, calls of a graph: 2048 x 2048 3.6 / 6.5,
    // 4096 x 4096 4.6 / 7.5, 256 x 8192 5.3 / 7.0, 8192 x 8192 9.8 / 13.0; past that a few
    // long rows are faster split, 256 x 14336 7.9 / 7.0, and many are not, 4096 x 14336
    // 9.7 / 12.7).  Unsplit, this is the faster: 28672 x 4096 20.7 / 15.5
    p.dot = batch == 1 && most > 1 && k <= kGemvInt4DotK;
    if (p.dot) p.parts = 1;
    p.bytes = p.parts > 1 ? part * p.parts : 0;
    return p;
}

}  // namespace tecoops
