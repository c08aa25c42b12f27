// rotary.h — positions and rotation shared by the kernels that turn queries and
// keys (rotary.hip, qk_norm_rotary.hip): the angles of a token's positions, the
// rotation of a pair, and the checks of a call's arguments.
#pragma once

#include "common.h"
#include "device.h"

namespace {

using namespace tecoops::dev;

constexpr int kMaxHalf = 256;  // rot_dim <= 512

// One position per token and axis, positions[axis * stride + t].  first[a] is
// the first frequency of axis a in ranges of them, first[a + 1] - first[a] its
// number of frequencies.  Angles are computed in turns in 64 bits and reduced
// to half a turn before sin and cos, so that far positions lose nothing: in 32
// bits an angle of 200000 is off by up to 0.008.
struct AxisPositions {
    const int64_t *__restrict__ positions;
    long long stride;
    const float *__restrict__ cos_sin_cache;
    int max_position, rot_dim, axes, layout;
    int first[TECOOPS_ROTARY_MAX_AXES + 1];
    double log2_base;

    static constexpr bool kCopySkipped = true;  // as they are, whatever they hold
    // The 64-bit angles take a good part of a microsecond: a workgroup's first loads
    // of q, k and v are under way meanwhile, and few tasks take 128 threads (q and k
    // [16380, 16, 128] fp16 in rows of 12288 bytes 49.7 us without, 46.0 with; with
    // the store, 4 tokens 4.2 and 3.8 us, 8191 tokens 40 us either way).
    static constexpr bool kEarlyLoads = true;

    __device__ __forceinline__ float2 angle(int t, int i) const {
        const int half = rot_dim >> 1;
        int axis = 0, from = 0, n = first[1];
        if (layout == TECOOPS_ROTARY_INTERLEAVED) {
            const int a = i % axes;
#pragma unroll
            for (int b = 1; b < TECOOPS_ROTARY_MAX_AXES; ++b)
                if (a == b && i < axes * (first[b + 1] - first[b])) axis = b;
        } else {
#pragma unroll
            for (int b = 1; b < TECOOPS_ROTARY_MAX_AXES; ++b)
                if (b < axes && i >= first[b]) {
                    axis = b;
                    from = first[b];
                    n = first[b + 1] - first[b];
                }
        }
        const int64_t pos = positions[axis * stride + t];
        float c = 1.0f, s = 0.0f;
        if (cos_sin_cache != nullptr) {
            if (pos >= 0 && pos < max_position) {
                c = cos_sin_cache[pos * rot_dim + i];
                s = cos_sin_cache[pos * rot_dim + half + i];
            }
            return make_float2(c, s);
        }
        const double power = layout == TECOOPS_ROTARY_PER_AXIS
                                 ? static_cast<double>(i - from) / n
                                 : static_cast<double>(i) / half;
        const double turns = static_cast<double>(pos) * (exp2(-power * log2_base) * 0.15915494309189535);
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
        return make_float2(c, s);
    }
    __device__ __forceinline__ bool skipped(int t) const {
        if (cos_sin_cache == nullptr) return false;
        bool out = false;
        for (int a = 0; a < axes; ++a) {
            const int64_t pos = positions[a * stride + t];
            out = out || pos < 0 || pos >= max_position;
        }
        return out;
    }
};

// o1 = x1 cos - x2 sin, o2 = x2 cos + x1 sin with the roundings spelled out
// (one product, then one fused multiply-add), so every kernel that rotates
// gets bit-identical results whatever the compiler would contract.
__device__ __forceinline__ float rot1(float x1, float x2, float c, float s) {
    return fmaf(x1, c, -(x2 * s));
}
__device__ __forceinline__ float rot2(float x1, float x2, float c, float s) {
    return fmaf(x2, c, x1 * s);
}

// Heads and strides of a call, and the widest words it can be done in.
struct Rows {
    void *query, *key;
    int num_tokens, num_heads, num_kv_heads, head_size, rot_dim;
    long long query_stride, key_stride;
};

// Arguments that both kinds of positions share.
inline tecoopsStatus_t check_rows(const Rows &r, const void *positions, const float *cos_sin_cache,
                           int max_position, float base, tecoopsDataType_t dataType) {
    if (positions == nullptr || r.query == nullptr) return TECOOPS_STATUS_BAD_PARAM;
    if (r.num_tokens <= 0 || r.num_heads <= 0 || r.head_size <= 0) return TECOOPS_STATUS_BAD_PARAM;
    if (r.key != nullptr && r.num_kv_heads <= 0) return TECOOPS_STATUS_BAD_PARAM;
    if (r.rot_dim <= 0 || (r.rot_dim & 1) || r.rot_dim > r.head_size || r.rot_dim / 2 > kMaxHalf)
        return TECOOPS_STATUS_BAD_PARAM;
    if (r.query_stride < static_cast<long long>(r.num_heads) * r.head_size)
        return TECOOPS_STATUS_BAD_PARAM;
    if (r.key != nullptr && r.key_stride < static_cast<long long>(r.num_kv_heads) * r.head_size)
        return TECOOPS_STATUS_BAD_PARAM;
    if (cos_sin_cache != nullptr && max_position <= 0) return TECOOPS_STATUS_BAD_PARAM;
    if (cos_sin_cache == nullptr && !(base > 0.0f)) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    return TECOOPS_STATUS_SUCCESS;
}

// The paged caches that the fused kernel writes to.
struct Pages {
    const void *value;
    const int64_t *slot_mapping;
    void *key_cache, *value_cache;
    long long value_stride;
    int num_blocks, block_size, write_key;
};

inline tecoopsStatus_t check_pages(const Rows &r, const Pages &g) {
    if (r.key == nullptr || g.value == nullptr || g.slot_mapping == nullptr ||
        g.key_cache == nullptr || g.value_cache == nullptr)
        return TECOOPS_STATUS_BAD_PARAM;
    if (g.num_blocks <= 0 || g.block_size <= 0) return TECOOPS_STATUS_BAD_PARAM;
    if (g.value_stride < static_cast<long long>(r.num_kv_heads) * r.head_size)
        return TECOOPS_STATUS_BAD_PARAM;
    if (static_cast<long long>(g.num_blocks) * g.block_size >= (1ll << 31))
        return TECOOPS_STATUS_NOT_SUPPORTED;
    return TECOOPS_STATUS_SUCCESS;
}

// The axes' frequencies have to fill the rotated half; interleaved, frequency
// i belongs to axis i % axes while that axis has any left, so every axis but
// the first has to find its last one inside the half.
inline tecoopsStatus_t axis_positions(AxisPositions *out, const int64_t *positions,
                               long long position_stride, int axes, const int *sections, int layout,
                               const Rows &r, const float *cos_sin_cache, int max_position,
                               float base) {
    if (axes < 1 || axes > TECOOPS_ROTARY_MAX_AXES || sections == nullptr)
        return TECOOPS_STATUS_BAD_PARAM;
    if (layout < TECOOPS_ROTARY_CONTIGUOUS || layout > TECOOPS_ROTARY_PER_AXIS)
        return TECOOPS_STATUS_BAD_PARAM;
    // positions are only read: all axes may share one row of them (stride 0)
    if (axes > 1 && position_stride != 0 && position_stride < r.num_tokens)
        return TECOOPS_STATUS_BAD_PARAM;
    const int half = r.rot_dim / 2;
    int sum = 0;
    for (int a = 0; a < TECOOPS_ROTARY_MAX_AXES; ++a) {
        out->first[a] = sum;
        if (a >= axes) continue;
        if (sections[a] < 0 || sections[a] > half - sum) return TECOOPS_STATUS_BAD_PARAM;
        if (layout == TECOOPS_ROTARY_INTERLEAVED && a > 0 && sections[a] > 0 &&
            axes * (sections[a] - 1) + a >= half)
            return TECOOPS_STATUS_BAD_PARAM;
        sum += sections[a];
    }
    out->first[TECOOPS_ROTARY_MAX_AXES] = sum;
    if (sum != half) return TECOOPS_STATUS_BAD_PARAM;
    out->positions = positions;
    out->stride = position_stride;
    out->cos_sin_cache = cos_sin_cache;
    out->max_position = max_position;
    out->rot_dim = r.rot_dim;
    out->axes = axes;
    out->layout = layout;
    out->log2_base = cos_sin_cache ? 0.0 : log2(static_cast<double>(base));
    return TECOOPS_STATUS_SUCCESS;
}

}  // namespace
