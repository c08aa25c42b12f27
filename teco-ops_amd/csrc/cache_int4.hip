// cache_int4.hip — keys and values stored into a paged cache held in 4 bits.
//
// A row x of a head (head_size elements) is held as codes n of 0..15 and a pair
// (scale, low) in x's type, x ~ scale * n + low:
//   low = min x,  scale = T((max x - min x) / 15),  n = (x - low) / scale to the
//   nearest (ties to even), at most 15; all codes 0 where scale is 0.
// The quotients are IEEE divisions of fp32 values, so the codes do not depend on
// how they are computed.  A row with a NaN, or whose range is not finite, has
// the pair (NaN, NaN) and codes 0: it reads as NaN throughout.
//
//   codes   uint8 [num_blocks, kv heads, block_size, head_size / 2], element 2j in
//           the low and 2j + 1 in the high half of byte j
//   scales  T [num_blocks, kv heads, block_size, 2]
//
// gfx950 design: a row is a group of lanes, one 16-byte chunk each, whose least
// and largest are a few DPP steps; each lane holds a key and a value chunk of
// kBatch rows, all loaded before the first is used.  HBM-bound: 2.5 bytes per
// element and 4 per row.
#include "common.h"
#include "device.h"
#include "epilogue.h"

namespace {

using namespace tecoops::dev;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;  // (16-byte loads need no alignment)

constexpr int kThreads = 256;
constexpr int kBatch = 2;  // (token, head) rows a thread has under way

struct Args {
    const uint16_t *key, *value;
    long long k_stride, v_stride;  // elements between tokens
    const int64_t *slots;
    uint8_t *kcodes, *vcodes;
    uint16_t *kscales, *vscales;
    int heads, head_size, block_size, lbs;
    long long capacity;  // num_blocks * block_size
    long long rows;      // tokens * heads
};

template <int LANES>
__device__ __forceinline__ void group_range(float &lo, float &hi) {
    const auto step = [&](auto f) {
        lo = fminf(lo, f(lo));
        hi = fmaxf(hi, f(hi));
    };
    step([](float v) { return dpp<kDppXor1>(v); });
    step([](float v) { return dpp<kDppXor2>(v); });
    step([](float v) { return dpp<kDppHalfMirror>(v); });
    if constexpr (LANES >= 16) step([](float v) { return dpp<kDppMirror>(v); });
    if constexpr (LANES >= 32) {
        lo = -row_swap_max(-lo);
        hi = row_swap_max(hi);
    }
    if constexpr (LANES >= 64) {
        lo = -half_swap_max(-lo);
        hi = half_swap_max(hi);
    }
}

// Codes and pair of one row from this lane's chunk of it.
template <typename T, int LANES>
__device__ __forceinline__ void quantise(const u32x4 &x, uint32_t &codes, uint32_t &pair) {
    float f[8], lo_ = INFINITY, hi_ = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = lo<T>(x[i]);
        f[2 * i + 1] = hi<T>(x[i]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo_ = fminf(lo_, f[e]);
        hi_ = fmaxf(hi_, f[e]);
        nan = nan || f[e] != f[e];
    }
    group_range<LANES>(lo_, hi_);
    const uint64_t any = __ballot(nan);
    const int lane = threadIdx.x & 63;
    const uint64_t group = LANES == 64 ? ~0ull : ((1ull << (LANES & 63)) - 1) << (lane & ~(LANES - 1));
    const float range = hi_ - lo_;
    const uint16_t s16 = static_cast<uint16_t>(round2<T>(range / 15.0f, 0.0f));
    const float scale = Cvt<T>::to(s16);
    codes = 0;
    if ((any & group) != 0 || !(range < INFINITY)) {
        pair = __is_same(T, f16) ? 0x7e007e00u : 0x7fc07fc0u;
        return;
    }
    pair = s16 | (round2<T>(lo_, lo_) << 16);
    if (!(scale > 0.0f)) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        codes |= static_cast<uint32_t>(fminf(rintf((f[e] - lo_) / scale), 15.0f)) << (4 * e);
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) append_kernel(Args a) {
    constexpr int ROWS = kThreads / LANES;
    const int c = threadIdx.x % LANES, chunks = a.head_size / 8, cc = min(c, chunks - 1);
    const long long row0 = static_cast<long long>(blockIdx.x) * (ROWS * kBatch) + threadIdx.x / LANES;
    u32x4 x[kBatch][2];
    int64_t slot[kBatch];
    int head[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const long long row = min(row0 + u * ROWS, a.rows - 1);
        const long long t = row / a.heads;
        head[u] = static_cast<int>(row - t * a.heads);
        slot[u] = row0 + u * ROWS < a.rows ? a.slots[t] : -1;
        const uint16_t *src[2] = {a.key + t * a.k_stride + head[u] * a.head_size + 8 * cc,
                                  a.value + t * a.v_stride + head[u] * a.head_size + 8 * cc};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(src[i]));
        }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        uint32_t codes[2], pair[2];
        quantise<T, LANES>(x[u][0], codes[0], pair[0]);
        quantise<T, LANES>(x[u][1], codes[1], pair[1]);
        if (slot[u] < 0 || slot[u] >= a.capacity || c >= chunks) continue;
        const int s32 = static_cast<int>(slot[u]);
        const int blk = a.lbs >= 0 ? s32 >> a.lbs : s32 / a.block_size;
        const long long at = (static_cast<long long>(blk) * a.heads + head[u]) * a.block_size +
                             (s32 - blk * a.block_size);
        *reinterpret_cast<uint32_t *>(a.kcodes + at * (a.head_size / 2) + 4 * c) = codes[0];
        *reinterpret_cast<uint32_t *>(a.vcodes + at * (a.head_size / 2) + 4 * c) = codes[1];
        if (c == 0) {
            *reinterpret_cast<uint32_t *>(a.kscales + at * 2) = pair[0];
            *reinterpret_cast<uint32_t *>(a.vscales + at * 2) = pair[1];
        }
    }
}

template <typename T>
void launch(const Args &a, hipStream_t s) {
    const int chunks = a.head_size / 8;
#define TECO_APPEND(L)                                                                              \
    hipLaunchKernelGGL((append_kernel<T, L>), dim3(tecoops::ceil_div(a.rows, kThreads / L * kBatch)), \
                       dim3(kThreads), 0, s, a)
    if (chunks <= 8) TECO_APPEND(8);
    else if (chunks <= 16) TECO_APPEND(16);
    else if (chunks <= 32) TECO_APPEND(32);
    else TECO_APPEND(64);
#undef TECO_APPEND
}

}  // namespace

extern "C" tecoopsStatus_t tecoopsReshapeAndCacheInt4(
    tecoopsHandle_t handle, const void *key, const void *value, const int64_t *slot_mapping,
    void *key_cache, void *value_cache, void *key_scales, void *value_scales, int num_tokens,
    int num_kv_heads, int head_size, long long key_stride, long long value_stride, int num_blocks,
    int block_size, tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (!key || !value || !slot_mapping || !key_cache || !value_cache || !key_scales || !value_scales)
        return TECOOPS_STATUS_BAD_PARAM;
    if (num_tokens < 0 || num_kv_heads <= 0 || head_size <= 0 || num_blocks <= 0 || block_size <= 0)
        return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    const long long width = static_cast<long long>(num_kv_heads) * head_size;
    if (key_stride < width || value_stride < width) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::aligned(key, 2) || !tecoops::aligned(value, 2) || !tecoops::aligned(key_cache, 4) ||
        !tecoops::aligned(value_cache, 4) || !tecoops::aligned(key_scales, 4) || !tecoops::aligned(value_scales, 4))
        return TECOOPS_STATUS_BAD_PARAM;
    TECO_RETURN_IF(head_size % 8 != 0 || head_size > 512, TECOOPS_STATUS_NOT_SUPPORTED,
                   "reshape_and_cache_int4: head_size %d not supported (multiples of 8 up to 512)", head_size);
    const long long rows = static_cast<long long>(num_tokens) * num_kv_heads;
    // (up to 64 lanes a row: the grid stays within 32-bit thread counts)
    if (static_cast<long long>(num_blocks) * block_size >= (1ll << 31) || rows >= (1ll << 26) || width >= (1ll << 30))
        return TECOOPS_STATUS_NOT_SUPPORTED;
    if (num_tokens == 0) return TECOOPS_STATUS_SUCCESS;
    Args a{};
    a.key = static_cast<const uint16_t *>(key);
    a.value = static_cast<const uint16_t *>(value);
    a.k_stride = key_stride;
    a.v_stride = value_stride;
    a.slots = slot_mapping;
    a.kcodes = static_cast<uint8_t *>(key_cache);
    a.vcodes = static_cast<uint8_t *>(value_cache);
    a.kscales = static_cast<uint16_t *>(key_scales);
    a.vscales = static_cast<uint16_t *>(value_scales);
    a.heads = num_kv_heads;
    a.head_size = head_size;
    a.block_size = block_size;
    a.lbs = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
    a.capacity = static_cast<long long>(num_blocks) * block_size;
    a.rows = rows;
    if (dataType == TECOOPS_DATA_HALF) launch<f16>(a, handle->stream);
    else launch<bf16>(a, handle->stream);
    TECO_CHECK_LAUNCH("reshape_and_cache_int4");
    return TECOOPS_STATUS_SUCCESS;
}
