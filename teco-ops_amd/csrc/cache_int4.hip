// cache_int4.hip — keys and values stored into a paged cache held in 4 bits.
//
// A row x of a head (head_size elements) is held as codes n of 0..15 and a pair
// (scale, low) in x's type, x ~ scale * n + low:
//   low = min x,  scale = T((max x - min x) / 15),  n = (x - low) / scale to the
//   nearest (ties to even), at most 15; all codes 0 where scale is 0.
// The quotients are IEEE divisions of fp32 values, so the codes do not depend on
// how they are computed (here as products with 1 / scale, whose rounded values are the
// quotients' unless one is next to the middle of two codes; then they are divided).  A row with a NaN, or whose range is not finite, has
// the pair (NaN, NaN) and codes 0: it reads as NaN throughout.
//
//   codes   uint8 [num_blocks, kv heads, block_size, head_size / 2], element 2j in
//           the low and 2j + 1 in the high half of byte j
//   scales  T [num_blocks, kv heads, block_size, 2]
//
// gfx950 design: a row is a group of lanes, one 16-byte chunk each, whose least and
// largest are a few DPP steps; each lane has one chunk of a key and one of its value,
// both loaded before the first is used.  2.5 bytes of memory an element and 4 a row,
// and some 20 vector instructions an element (least and largest as integers, two at a
// time): many short waves hide one under the other.  8192 tokens, 8 heads of 128, fp16
// (42 MB): 12.9 us, 3.3 TB/s; with 2, 3 and 4 rows a lane 13.8, 15.4 and 15.2, and with a
// division for each code 16.5 (2 rows).
#include "common.h"
#include "device.h"
#include "epilogue.h"

namespace {

using namespace tecoops::dev;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;  // (16-byte loads need no alignment)

constexpr int kThreads = 256;

struct Args {
    const uint16_t *key, *value;
    uint32_t k_stride, v_stride;  // elements between tokens
    const int64_t *slots;
    uint8_t *kcodes, *vcodes;
    uint16_t *kscales, *vscales;
    uint32_t heads, head_size, block_size, block_rows;  // rows of a block: heads * block_size
    int lbs;
    uint32_t inv_heads;  // 2^32 / heads rounded up, where that divides every row by it; else 0
    long long capacity;  // num_blocks * block_size
    uint32_t rows;       // tokens * heads
};

typedef short i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, a), __builtin_bit_cast(i16x2, b)));
}
// 16-bit floats as integers of the same order (-0 below 0), and back.
__device__ __forceinline__ uint32_t ordered(uint32_t v) {
    const i16x2 sign = __builtin_bit_cast(i16x2, v) >> 15;
    return v ^ (__builtin_bit_cast(uint32_t, sign) & 0x7fff7fffu);
}

// Over a row's lanes, the most of each half of w.
template <int LANES>
__device__ __forceinline__ uint32_t group_most(uint32_t w) {
    const auto moved = [](uint32_t v, auto f) { return __float_as_uint(f(__uint_as_float(v))); };
    w = most2(w, moved(w, [](float v) { return dpp<kDppXor1>(v); }));
    w = most2(w, moved(w, [](float v) { return dpp<kDppXor2>(v); }));
    w = most2(w, moved(w, [](float v) { return dpp<kDppHalfMirror>(v); }));
    if constexpr (LANES >= 16) w = most2(w, moved(w, [](float v) { return dpp<kDppMirror>(v); }));
    if constexpr (LANES >= 32) w = most2(w, static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), 16)));
    if constexpr (LANES >= 64) w = most2(w, static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), 32)));
    return w;
}

// Codes and pair of one row from this lane's chunk of it.
template <typename T, int LANES>
__device__ __forceinline__ void quantise(const u32x4 &x, uint32_t &codes, uint32_t &pair) {
    // the largest and the least as ordered integers, the second as its complement, two
    // halves of a word
    uint32_t o[4], top, low;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = ordered(x[i]);
    top = most2(most2(o[0], o[1]), most2(o[2], o[3]));
    low = most2(most2(~o[0], ~o[1]), most2(~o[2], ~o[3]));
    const uint32_t w = group_most<LANES>(
        most2(__builtin_amdgcn_perm(low, top, 0x05040100u), __builtin_amdgcn_perm(low, top, 0x07060302u)));
    constexpr int kInf = __is_same(T, f16) ? 0x7c00 : 0x7f80;
    const int top_at = static_cast<int16_t>(w), low_at = ~(static_cast<int>(w) >> 16);
    // a NaN lies above infinity, or below minus it
    const bool nan = top_at > kInf || low_at < ~kInf;
    const uint32_t ends = ordered(static_cast<uint16_t>(top_at) | static_cast<uint32_t>(low_at) << 16);
    const float hi_ = lo<T>(ends), lo_ = hi<T>(ends);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = lo<T>(x[i]);
        f[2 * i + 1] = hi<T>(x[i]);
    }
    const float range = hi_ - lo_;
    const uint16_t s16 = static_cast<uint16_t>(round2<T>(range / 15.0f, 0.0f));
    const float scale = Cvt<T>::to(s16);
    codes = 0;
    if (nan || !(range < INFINITY)) {
        pair = __is_same(T, f16) ? 0x7e007e00u : 0x7fc07fc0u;
        return;
    }
    pair = s16 | (ends & 0xffff0000u);
    if (!(scale > 0.0f)) return;
    // With inv off by 2^-23 and a rounding of 2^-24 in each of product and quotient, the
    // two are within 2^-22 of 23 (15.1, but for subnormal scales): farther than that from
    // the middle of two codes they round alike.  (An infinite inv is none of that.)
    constexpr float kClear = 0.5f - 0x1p-17f;
    const float inv = __builtin_amdgcn_rcpf(scale);
    float n[8], off = 0.0f;
    bool clear = inv < INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = (f[e] - lo_) * inv;
        n[e] = rintf(q);
        off = fmaxf(off, fabsf(q - n[e]));
    }
    clear = clear && off < kClear;
    if (!clear) {
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] = rintf((f[e] - lo_) / scale);
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        codes |= static_cast<uint32_t>(fmaf(16.0f, fminf(n[e + 1], 15.0f), fminf(n[e], 15.0f))) << (4 * e);
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) append_kernel(Args a) {
    constexpr int ROWS = kThreads / LANES;
    const uint32_t c = threadIdx.x % LANES, chunks = a.head_size / 8, cc = min(c, chunks - 1);
    // (32-bit factors and 64-bit sums: a product is one instruction)
    const auto mad = [](uint32_t x, uint32_t y, uint64_t z) { return static_cast<uint64_t>(x) * y + z; };
    const uint32_t at = blockIdx.x * ROWS + threadIdx.x / LANES, row = min(at, a.rows - 1);
    const uint32_t t = a.heads == 1 ? row : a.inv_heads != 0u ? __umulhi(row, a.inv_heads) : row / a.heads;
    const uint32_t head = row - t * a.heads, in = head * a.head_size + 8 * cc;
    const u32x4 key = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(a.key + mad(t, a.k_stride, in)));
    const u32x4 value = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(a.value + mad(t, a.v_stride, in)));
    const int64_t slot = at < a.rows ? a.slots[t] : -1;
    uint32_t codes[2], pair[2];
    quantise<T, LANES>(key, codes[0], pair[0]);
    quantise<T, LANES>(value, codes[1], pair[1]);
    if (slot < 0 || slot >= a.capacity || c >= chunks) return;
    const uint32_t s32 = static_cast<uint32_t>(slot);
    const uint32_t blk = a.lbs >= 0 ? s32 >> a.lbs : s32 / a.block_size;
    const uint64_t to = mad(blk, a.block_rows, mad(head, a.block_size, s32 - blk * a.block_size));
    const uint64_t byte = to * (a.head_size / 2) + 4 * c;
    *reinterpret_cast<uint32_t *>(a.kcodes + byte) = codes[0];
    *reinterpret_cast<uint32_t *>(a.vcodes + byte) = codes[1];
    if (c == 0) {
        *reinterpret_cast<uint32_t *>(a.kscales + to * 2) = pair[0];
        *reinterpret_cast<uint32_t *>(a.vscales + to * 2) = pair[1];
    }
}

template <typename T>
void launch(const Args &a, hipStream_t s) {
    const int chunks = a.head_size / 8;
#define TECO_APPEND(L)                                                                              \
    hipLaunchKernelGGL((append_kernel<T, L>), dim3(tecoops::ceil_div(a.rows, kThreads / L)), \
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
    if (num_tokens == 1) key_stride = value_stride = width;  // (of no use)
    const long long block_rows = static_cast<long long>(num_kv_heads) * block_size;
    if (key_stride >= (1ll << 32) || value_stride >= (1ll << 32) || block_rows >= (1ll << 32))
        return TECOOPS_STATUS_NOT_SUPPORTED;
    Args a{};
    a.key = static_cast<const uint16_t *>(key);
    a.value = static_cast<const uint16_t *>(value);
    a.k_stride = static_cast<uint32_t>(key_stride);
    a.v_stride = static_cast<uint32_t>(value_stride);
    a.slots = slot_mapping;
    a.kcodes = static_cast<uint8_t *>(key_cache);
    a.vcodes = static_cast<uint8_t *>(value_cache);
    a.kscales = static_cast<uint16_t *>(key_scales);
    a.vscales = static_cast<uint16_t *>(value_scales);
    a.heads = num_kv_heads;
    a.head_size = head_size;
    a.block_size = block_size;
    a.block_rows = static_cast<uint32_t>(block_rows);
    const uint64_t inv = ((1ull << 32) + num_kv_heads - 1) / num_kv_heads, off = inv * num_kv_heads - (1ull << 32);
    a.inv_heads = num_kv_heads > 1 && static_cast<uint64_t>(rows) * off < (1ull << 32) ? static_cast<uint32_t>(inv) : 0u;  // (exact up to 2^32 / off)
    a.lbs = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
    a.capacity = static_cast<long long>(num_blocks) * block_size;
    a.rows = static_cast<uint32_t>(rows);
    if (dataType == TECOOPS_DATA_HALF) launch<f16>(a, handle->stream);
    else launch<bf16>(a, handle->stream);
    TECO_CHECK_LAUNCH("reshape_and_cache_int4");
    return TECOOPS_STATUS_SUCCESS;
}
