// qk_norm_rotary.hip — the norm of each head of query and key and the rotation
// by the token's position in one pass, with the store into the paged cache or
// without.
//
//   y = x / sqrt(mean(x^2) + eps) * w       over the head_size elements of a head,
//   o = y turned by the angles of the token's positions (rotary.h),
//
// w the query's or the key's weight [head_size]; all in fp32, one rounding.  Read
// and written once each, where a norm and a rotation in turn move q and k twice
// and round twice.
//
// gfx950 design: a head is a row of lanes, one 16-byte chunk each (a power of
// two of lanes, those past the head idle), so that its sum of squares is a few
// DPP steps and the other halves of the pairs of NeoX order are one exchange
// between lanes away.  A lane keeps its chunk's place in every head that it
// works on: its angles and weights are loaded once.  Memory-bound: the loads of
// kBatch heads are under way before the first is used.  8191 tokens, 32 heads and 8 of
// 128, bf16, with the store (201 MB): 43.1 us, 4.7 TB/s (a large copy: 4.95); a decode
// step of 4 tokens 8, of which the kernel 4.5: the ramp of a launch.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "epilogue.h"
#include "rotary.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;          // heads a thread loads before it stores any
constexpr int kMaxVecHead = 512;   // elements of a head in one wave
constexpr int kMaxHead = 1024;     // ... in the LDS of the general kernel

struct Args {
    uint16_t *query, *key;
    const uint16_t *q_weight, *k_weight;
    const uint16_t *value;
    const int64_t *slots;
    uint16_t *kcache, *vcache;  // null: no cache
    int num_tokens, num_heads, num_kv_heads, head_size, rot_dim;
    long long q_stride, k_stride, v_stride;
    int block_size, lbs;  // lbs = log2(block_size) or -1
    long long capacity;   // num_blocks * block_size
    int write_key;
    float eps;
};

// First element of the cache row of `slot` at kv head 0, or -1.
__device__ __forceinline__ long long cache_row(const Args &a, int64_t slot) {
    if (slot < 0 || slot >= a.capacity) return -1;
    const int s32 = static_cast<int>(slot);
    const int blk = a.lbs >= 0 ? s32 >> a.lbs : s32 / a.block_size;
    return (static_cast<long long>(blk) * a.num_kv_heads * a.block_size + (s32 - blk * a.block_size)) *
           a.head_size;
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp<kDppXor1>(v);
    v += dpp<kDppXor2>(v);
    v += dpp<kDppHalfMirror>(v);
    if constexpr (LANES >= 16) v += dpp<kDppMirror>(v);
    if constexpr (LANES >= 32) v = row_swap_sum(v);
    if constexpr (LANES >= 64) v = half_swap_sum(v);
    return v;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &x, float (&f)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = lo<T>(w[i]);
        f[2 * i + 1] = hi<T>(w[i]);
    }
}

// Workgroup (token, part): heads query, then key, then (with a cache) value, a
// group of LANES lanes each, dealt to the groups of all parts in turn.
template <typename T, bool NEOX, int LANES, bool CACHE>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(AxisPositions angles, Args a) {
    __shared__ float2 cs[kMaxHalf];
    constexpr int GROUPS = kThreads / LANES;
    const int t = blockIdx.x;
    const int c = threadIdx.x % LANES, chunks = a.head_size / 8;
    const int cc = min(c, chunks - 1);
    const int half = a.rot_dim >> 1;
    const int nq = a.num_heads, nk = nq + a.num_kv_heads, total = nk + (CACHE ? a.num_kv_heads : 0);
    const int step = gridDim.y * GROUPS, first = blockIdx.y * GROUPS + threadIdx.x / LANES;
    uint16_t *const q = a.query + t * a.q_stride + 8 * cc;
    uint16_t *const k = a.key + t * a.k_stride + 8 * cc;
    const uint16_t *const v = a.value + t * a.v_stride + 8 * cc;
    // the head of the wave's first group: where that is past the last, the wave is done
    const int ahead = __builtin_amdgcn_readfirstlane(first);
    uint4 x[kBatch];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (base + u * step + ahead >= total) break;
            const int h = min(base + u * step + first, total - 1);
            const uint16_t *row = h < nq ? q + h * a.head_size
                                  : !CACHE || h < nk ? k + (h - nq) * a.head_size
                                                     : v + (h - nk) * a.head_size;
            x[u] = ld_stream(reinterpret_cast<const uint4 *>(row));
        }
    };
    load(0);
    // this lane's chunk: its weights and, in NeoX order, those of the chunk that
    // holds the other halves of its pairs
    const int hc = half / 8;
    const bool turns = NEOX ? c < 2 * hc : 8 * c < a.rot_dim;
    const int other = NEOX && turns ? (c < hc ? hc : -hc) : 0;
    const auto weight = [&](const uint16_t *w, int at) { return *reinterpret_cast<const uint4 *>(w + 8 * at); };
    const uint4 wq = weight(a.q_weight, cc), wk = a.key ? weight(a.k_weight, cc) : wq;
    uint4 wqo = wq, wko = wk;
    if (NEOX) {
        wqo = weight(a.q_weight, cc + other);
        if (a.key) wko = weight(a.k_weight, cc + other);
    }
    const bool skip = angles.skipped(t);
    const long long at = CACHE ? cache_row(a, a.slots[t]) : -1;
    if (!skip)
        for (int i = threadIdx.x; i < half; i += kThreads) cs[i] = angles.angle(t, i);
    __syncthreads();
    constexpr int NA = NEOX ? 8 : 4;  // angles of a chunk
    float2 an[NA];
#pragma unroll
    for (int e = 0; e < NA; ++e) {
        an[e] = cs[turns ? (NEOX ? 8 * (c < hc ? c : c - hc) + e : 4 * c + e) : 0];
        if (NEOX && c < hc) an[e].y = -an[e].y;
    }
    const float inv_d = 1.0f / static_cast<float>(a.head_size);
    const long long head_step = static_cast<long long>(a.block_size) * a.head_size;  // in the cache
    for (int base = 0; base < total; base += step * kBatch) {
        if (base != 0) load(base);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (base + u * step + ahead >= total) break;
            const int h = base + u * step + first;
            const bool is_q = h < nq, is_v = CACHE && h >= nk;
            float f[8], w[8];
            unpack8<T>(x[u], f);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e], f[e], sum);
            sum = group_sum<LANES>(c < chunks ? sum : 0.0f);
            const float r = rsqrtf(fmaf(sum, inv_d, a.eps));
            unpack8<T>(is_q ? wq : wk, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = f[e] * r * w[e];
            if constexpr (NEOX) {
                uint4 xo;
                const int from = static_cast<int>(threadIdx.x & 63) + other;
                xo.x = __shfl(x[u].x, from, 64);
                xo.y = __shfl(x[u].y, from, 64);
                xo.z = __shfl(x[u].z, from, 64);
                xo.w = __shfl(x[u].w, from, 64);
                float o[8];
                unpack8<T>(xo, o);
                unpack8<T>(is_q ? wqo : wko, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float turned = fmaf(f[e], an[e].x, o[e] * r * w[e] * an[e].y);
                    f[e] = turns ? turned : f[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y1 = f[2 * e], y2 = f[2 * e + 1];
                    if (turns) {
                        f[2 * e] = rot1(y1, y2, an[e].x, an[e].y);
                        f[2 * e + 1] = rot2(y1, y2, an[e].x, an[e].y);
                    }
                }
            }
            uint4 out = x[u];
            if (!skip && !is_v)
                out = make_uint4(round2<T>(f[0], f[1]), round2<T>(f[2], f[3]), round2<T>(f[4], f[5]),
                                 round2<T>(f[6], f[7]));
            if (h >= total || c >= chunks) continue;
            if (!skip && !is_v && (is_q || !CACHE || a.write_key))
                st_stream(reinterpret_cast<uint4 *>(is_q ? q + h * a.head_size : k + (h - nq) * a.head_size), out);
            if (CACHE && !is_q && at >= 0)
                st_stream(reinterpret_cast<uint4 *>((is_v ? a.vcache : a.kcache) + at +
                                                    (h - (is_v ? nk : nq)) * head_step + 8 * c), out);
        }
    }
}

// Any head size, alignment and order: a wave per head, an element a lane at a time.
template <typename T, bool NEOX, bool CACHE>
__global__ void __launch_bounds__(kThreads) qk_norm_any_kernel(AxisPositions angles, Args a) {
    __shared__ __attribute__((aligned(16))) float rows[kThreads / 64][kMaxHead];
    const int lane = threadIdx.x & 63, D = a.head_size;
    const int nq = a.num_heads, nk = nq + a.num_kv_heads, total = nk + (CACHE ? a.num_kv_heads : 0);
    const long long unit = static_cast<long long>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    if (unit >= static_cast<long long>(a.num_tokens) * total) return;
    const int t = static_cast<int>(unit / total), h = static_cast<int>(unit - static_cast<long long>(t) * total);
    const bool is_q = h < nq, is_v = CACHE && h >= nk;
    uint16_t *row = is_q ? a.query + t * a.q_stride + static_cast<long long>(h) * D
                         : a.key + t * a.k_stride + static_cast<long long>(h - nq) * D;
    const long long at = CACHE ? cache_row(a, a.slots[t]) : -1;
    const long long to = at + static_cast<long long>(h - (is_v ? nk : nq)) * a.block_size * D;
    const bool skip = angles.skipped(t);
    if (is_v || skip) {
        if (!CACHE || is_q || at < 0) return;
        const uint16_t *src = is_v ? a.value + t * a.v_stride + static_cast<long long>(h - nk) * D : row;
        for (int e = lane; e < D; e += 64) (is_v ? a.vcache : a.kcache)[to + e] = src[e];
        return;
    }
    float *y = rows[threadIdx.x >> 6];
    const uint16_t *w = is_q ? a.q_weight : a.k_weight;
    // (the wave's own LDS writes, before it reads them)
    const auto written = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    for (int e = lane; e < D; e += 64) y[e] = Cvt<T>::to(row[e]);
    written();
    // runs of 8 a lane and a tree over the lanes, as in the kernel above: a row comes out
    // of both with the same bits
    float sum = 0.0f;
    for (int c = 8 * lane; c < D; c += 8 * 64) {
        float run = 0.0f;
        if (c + 8 <= D) {
            const float4_t f[2] = {*reinterpret_cast<const float4_t *>(y + c), *reinterpret_cast<const float4_t *>(y + c + 4)};
#pragma unroll
            for (int e = 0; e < 8; ++e) run = fmaf(f[e >> 2][e & 3], f[e >> 2][e & 3], run);
        } else {
            for (int e = c; e < D; ++e) run = fmaf(y[e], y[e], run);
        }
        sum += run;
    }
    const float r = rsqrtf(fmaf(wave_sum(sum), 1.0f / static_cast<float>(D), a.eps));
    written();
    for (int e = lane; e < D; e += 64) y[e] = y[e] * r * Cvt<T>::to(w[e]);
    written();
    const int half = a.rot_dim >> 1;
    for (int e = lane; e < D; e += 64) {
        float o = y[e];
        if (e < a.rot_dim) {
            const int i = NEOX ? (e < half ? e : e - half) : e >> 1;
            const bool low = NEOX ? e < half : (e & 1) == 0;
            const float other = y[NEOX ? (low ? e + half : e - half) : e ^ 1];
            const float2 an = angles.angle(t, i);
            o = low ? rot1(o, other, an.x, an.y) : rot2(other, o, an.x, an.y);
        }
        const uint16_t b = Cvt<T>::from(o);
        if (is_q || !CACHE || a.write_key) row[e] = b;
        if (CACHE && !is_q && at >= 0) a.kcache[to + e] = b;
    }
}

template <typename T, bool NEOX, bool CACHE>
void launch(const AxisPositions &an, const Args &a, bool vec, hipStream_t s) {
    const int total = a.num_heads + a.num_kv_heads * (CACHE ? 2 : 1);
    if (!vec) {
        const long long units = static_cast<long long>(a.num_tokens) * total;
        hipLaunchKernelGGL((qk_norm_any_kernel<T, NEOX, CACHE>), dim3(tecoops::ceil_div(units, kThreads / 64)),
                           dim3(kThreads), 0, s, an, a);
        return;
    }
    const int chunks = a.head_size / 8;
    const int lanes = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64;
    // a few tokens are cut into as many workgroups as leave each thread one head
    const int most = static_cast<int>(tecoops::ceil_div(static_cast<long long>(total) * lanes, kThreads));
    const int room = std::max(1, 2 * tecoops::device_cus() / a.num_tokens);
    const dim3 grid(a.num_tokens, std::min(most, room));
#define TECO_QK_NORM(L) \
    hipLaunchKernelGGL((qk_norm_kernel<T, NEOX, L, CACHE>), grid, dim3(kThreads), 0, s, an, a)
    switch (lanes) {
        case 8: TECO_QK_NORM(8); break;
        case 16: TECO_QK_NORM(16); break;
        case 32: TECO_QK_NORM(32); break;
        default: TECO_QK_NORM(64); break;
    }
#undef TECO_QK_NORM
}

tecoopsStatus_t run(tecoopsHandle_t handle, const AxisPositions &an, Rows r, const Pages *g, const void *qw,
                    const void *kw, float eps, int is_neox, tecoopsDataType_t dataType) {
    const size_t el = sizeof(uint16_t);
    if (qw == nullptr || (r.key != nullptr && kw == nullptr)) return TECOOPS_STATUS_BAD_PARAM;
    if (!(eps >= 0.0f) || !(eps < INFINITY)) return TECOOPS_STATUS_BAD_PARAM;
    for (const void *p : {static_cast<const void *>(r.query), static_cast<const void *>(r.key), qw, kw})
        if (!tecoops::aligned(p, el)) return TECOOPS_STATUS_BAD_PARAM;
    if (r.head_size > kMaxHead || r.num_tokens >= (1 << 24)) return TECOOPS_STATUS_NOT_SUPPORTED;
    if (r.key == nullptr) r.num_kv_heads = 0;
    const long long heads = static_cast<long long>(r.num_heads) + r.num_kv_heads * (g ? 2ll : 1ll);
    if (heads > (1 << 20)) return TECOOPS_STATUS_NOT_SUPPORTED;
    Args a{};
    a.query = static_cast<uint16_t *>(r.query);
    a.key = static_cast<uint16_t *>(r.key);
    a.q_weight = static_cast<const uint16_t *>(qw);
    a.k_weight = static_cast<const uint16_t *>(kw);
    a.num_tokens = r.num_tokens;
    a.num_heads = r.num_heads;
    a.num_kv_heads = r.num_kv_heads;
    a.head_size = r.head_size;
    a.rot_dim = r.rot_dim;
    a.q_stride = r.query_stride;
    a.k_stride = r.key_stride;
    a.eps = eps;
    const int half = r.rot_dim / 2;
    bool vec = r.head_size % 8 == 0 && r.head_size <= kMaxVecHead && (is_neox ? half % 8 == 0 : half % 4 == 0) &&
               r.query_stride % 8 == 0 && tecoops::aligned(r.query, 16) && tecoops::aligned(qw, 16);
    if (r.key != nullptr)
        vec = vec && r.key_stride % 8 == 0 && tecoops::aligned(r.key, 16) && tecoops::aligned(kw, 16);
    if (g != nullptr) {
        a.value = static_cast<const uint16_t *>(g->value);
        a.slots = g->slot_mapping;
        a.kcache = static_cast<uint16_t *>(g->key_cache);
        a.vcache = static_cast<uint16_t *>(g->value_cache);
        a.v_stride = g->value_stride;
        a.block_size = g->block_size;
        a.lbs = (g->block_size & (g->block_size - 1)) == 0 ? __builtin_ctz(g->block_size) : -1;
        a.capacity = static_cast<long long>(g->num_blocks) * g->block_size;
        a.write_key = g->write_key;
        for (const void *p : {g->value, static_cast<const void *>(g->key_cache), static_cast<const void *>(g->value_cache)})
            if (!tecoops::aligned(p, el)) return TECOOPS_STATUS_BAD_PARAM;
        vec = vec && g->value_stride % 8 == 0 && tecoops::aligned(g->value, 16) &&
              tecoops::aligned(g->key_cache, 16) && tecoops::aligned(g->value_cache, 16);
    }
    // (a wave per head keeps the grid within 32-bit thread counts)
    if (!vec && heads * r.num_tokens > (1ll << 25)) return TECOOPS_STATUS_NOT_SUPPORTED;
    hipStream_t s = handle->stream;
    const bool h16 = dataType == TECOOPS_DATA_HALF;
    const auto go = [&](auto neox, auto cache) {
        constexpr bool NX = decltype(neox)::value, CA = decltype(cache)::value;
        if (h16) launch<f16, NX, CA>(an, a, vec, s);
        else launch<bf16, NX, CA>(an, a, vec, s);
    };
    if (is_neox) g ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    else g ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
    TECO_CHECK_LAUNCH("qk_norm_rotary");
    return TECOOPS_STATUS_SUCCESS;
}

}  // namespace

extern "C" tecoopsStatus_t tecoopsQkNormRotary(
    tecoopsHandle_t handle, const int64_t *positions, long long position_stride, int axes,
    const int *sections, tecoopsRotaryLayout_t layout, void *query, void *key,
    const void *query_weight, const void *key_weight, float eps, int num_tokens, int num_heads,
    int num_kv_heads, int head_size, int rot_dim, long long query_stride, long long key_stride,
    const float *cos_sin_cache, int max_position, float base, int is_neox,
    tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    const Rows r{query, key, num_tokens, num_heads, num_kv_heads, head_size, rot_dim, query_stride,
                 key_stride};
    AxisPositions an{};
    const int whole[1] = {rot_dim / 2};
    tecoopsStatus_t st = check_rows(r, positions, cos_sin_cache, max_position, base, dataType);
    if (st == TECOOPS_STATUS_SUCCESS)
        st = axis_positions(&an, positions, position_stride, axes, axes == 1 && !sections ? whole : sections,
                            layout, r, cos_sin_cache, max_position, base);
    if (st != TECOOPS_STATUS_SUCCESS) return st;
    return run(handle, an, r, nullptr, query_weight, key_weight, eps, is_neox, dataType);
}

extern "C" tecoopsStatus_t tecoopsQkNormRotaryReshapeAndCache(
    tecoopsHandle_t handle, const int64_t *positions, long long position_stride, int axes,
    const int *sections, tecoopsRotaryLayout_t layout, void *query, void *key, const void *value,
    const void *query_weight, const void *key_weight, float eps, const int64_t *slot_mapping,
    void *key_cache, void *value_cache, int num_tokens, int num_heads, int num_kv_heads,
    int head_size, int rot_dim, long long query_stride, long long key_stride,
    long long value_stride, const float *cos_sin_cache, int max_position, float base, int is_neox,
    int num_blocks, int block_size, int write_key, tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    const Rows r{query, key, num_tokens, num_heads, num_kv_heads, head_size, rot_dim, query_stride,
                 key_stride};
    const Pages g{value, slot_mapping, key_cache, value_cache, value_stride, num_blocks, block_size,
                  write_key};
    AxisPositions an{};
    const int whole[1] = {rot_dim / 2};
    tecoopsStatus_t st = check_rows(r, positions, cos_sin_cache, max_position, base, dataType);
    if (st == TECOOPS_STATUS_SUCCESS) st = check_pages(r, g);
    if (st == TECOOPS_STATUS_SUCCESS)
        st = axis_positions(&an, positions, position_stride, axes, axes == 1 && !sections ? whole : sections,
                            layout, r, cos_sin_cache, max_position, base);
    if (st != TECOOPS_STATUS_SUCCESS) return st;
    return run(handle, an, r, &g, query_weight, key_weight, eps, is_neox, dataType);
}
