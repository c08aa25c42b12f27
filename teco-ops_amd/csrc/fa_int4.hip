// fa_int4.hip — attention over the paged cache held in 4 bits (cache_int4.hip).
//
//   K[j] = s_j n_j + a_j   (n_j codes 0..15 of a row, s_j its scale, a_j its least),
//   S[i, j] = scale q_i . K[j],  P = softmax over the keys that row i sees,
//   O[i] = sum_j P[i, j] V[j];  rows, masks and lengths as in flash_attention.hip.
//
// Split route (few query rows: decode).  HBM-bound: a key and a value cost
// head_size + 8 bytes together.  At that rate a SIMD has about three lane
// operations for a cached element, so the codes are never widened to numbers one
// by one: as 16-bit patterns they are fp16 subnormals, n 2^-24, and go into the
// matrix core as they come out of a mask,
//   q . K[j] = s_j (q . n_j) + a_j sum(q),
//   sum_j P V = sum_j W_j n_j - c sum_j W_j + sum_j P (a_j + c s_j),  W = fp16(P s),
// with s and a applied to the fp32 scores, 1/16 of the work of the elements (and
// no rounding of K or V at all).  c = 7.5, the middle of the codes: what rounds W
// then weighs a value's distance from the middle of its row, not from its least,
// which for rows around 0 is 3 times as far.  A nibble in bits 4-7 is 16 n; the 1/16 goes into
// q's elements and into the sums of those value channels.  q and the weights P s
// are fp16, scaled by powers of two to the top of its range (q by its largest
// element in its column, P s by the running maximum and the largest scale so far),
// so that bf16's range is kept and small weights of long contexts lose nothing.
//   * Scores are computed transposed (keys x columns, 16x16x32), so that a lane
//     holds 8 keys of one column, which are the operand of the second product as
//     they are: neither P nor the codes go through LDS.
//   * A wave takes every 4th block of 32 keys; the next block's loads are under
//     way meanwhile.  Partial states meet in LDS, those of splits in a second
//     kernel.
//
// Tile route (prefill).  K and V tiles are widened to fp16 once per workgroup, on
// the way into LDS, and attended as in flash_attention.hip (fa_device.h).  fp16
// for bf16 models too, 8 times closer than bf16 and a fixed range: rows of the
// cache are first taken as they are, and a tile in which one is too large or all
// are too small is done again with a power of two that fits.
#include <cmath>

#include "fa_device.h"
#include "fa_int4.h"

namespace {

using tecoops::fa4::kWaves;
using tecoops::fa4::Plan;

struct Params {
    const uint16_t *q;
    const uint8_t *kc, *vc;
    const uint32_t *ks, *vs;  // (scale, least) of a row in one word
    uint16_t *o;
    const int *bt;
    long long bt_stride;
    const int *cu_q, *kv_lens;
    int batch, H, Hkv, G, bs, lbs, num_blocks;  // lbs = log2(bs) or -1
    int kv_cap;                                 // keys that a table row can name
    float scale_log2;
    int causal;
    long long total_q;
    float *ws_o, *ws_ml;
    int cols, tiles, split_len, splits;
};

typedef unsigned __attribute__((aligned(4))) u32_a4;
typedef float4_t f32x4_t;
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mma16(const u32x4 &a, const u32x4 &b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
}

// 2^e, e within a float's normal exponents.
__device__ __forceinline__ float power2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ void sequence(const Params &p, int b, long long &q_off, int &L, int &S) {
    q_off = p.cu_q[b];
    L = p.cu_q[b + 1] - p.cu_q[b];
    S = min(max(p.kv_lens[b], 0), p.kv_cap);
}

// Output rows of no sequence are written as zeros, as by the 16-bit cache's
// attention.
__device__ __forceinline__ void zero_tail(const Params &p, int D) {
    const long long end = max(p.cu_q[p.batch], 0);
    if (end >= p.total_q) return;
    const long long chunks = static_cast<long long>(p.H) * D / 8;
    u32x4 *o = reinterpret_cast<u32x4 *>(p.o);
    for (long long c = end * chunks + threadIdx.x; c < p.total_q * chunks; c += blockDim.x)
        o[c] = u32x4{0u, 0u, 0u, 0u};
}

__device__ __forceinline__ int block_at(const Params &p, int key) { return p.lbs >= 0 ? key >> p.lbs : key / p.bs; }

// Row of the cache, in rows of all blocks and heads, of a key whose block-table
// entry is `page`; entries out of range are taken as block 0.
__device__ __forceinline__ long long row_of(const Params &p, int kvh, int page, int key, int blk) {
    if (page < 0 || page >= p.num_blocks) page = 0;
    return (static_cast<long long>(page) * p.Hkv + kvh) * p.bs + (key - blk * p.bs);
}

// Weights are at most 2^kTop * 2^kSlack before the maximum is raised; scales at
// most twice the reference: P s stays below 2^15.
constexpr float kTop = 10.0f, kSlack = 4.0f;
constexpr float kMiddle = 7.5f;  // of the codes
constexpr int kLeastRef = -90;   // (sums of 2^24 weights stay within fp32)
constexpr float kNever = -1e30f;  // the running maximum before any key

// Block-size modes: 1 a multiple of 16 (a block of 16 keys lies in one page: its
// entry is a scalar), 2 a multiple of 4 (so do a lane's 4 keys), 0 any.
template <int D, int BSM>
struct Block {
    static constexpr int KW = D / 32;  // 32-bit words of a key row in a lane
    static constexpr int N128 = D / 128, N64 = D % 128 / 64, N32 = D % 64 / 32;
    static constexpr int VP = BSM == 0 ? 4 : 1;  // table entries of a lane's 4 keys
    uint32_t k[2][KW];
    uint32_t v[2][4][N128 + N64 + N32];
    u32x4 ks[2], vs[2];

    // The block-table entries that a load() needs, fetched one load ahead of it.
    struct Pages {
        int kp[2], vp[2][VP];
    };

    static __device__ __forceinline__ void pages(Pages &g, const Params &p, const int *table, int j0, int limit) {
        const int lane = threadIdx.x & 63;
        int(&kp)[2] = g.kp, (&vp)[2][VP] = g.vp;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if constexpr (BSM == 1) {
                const int row = __builtin_amdgcn_readfirstlane(j0 + 16 * b);
                const auto *t4 = (const __attribute__((address_space(4))) int *)(table);
                kp[b] = row < limit ? t4[block_at(p, row)] : 0;
            } else {
                const int key = j0 + 16 * b + (lane & 15);
                kp[b] = table[block_at(p, key < limit ? key : 0)];
#pragma unroll
                for (int i = 0; i < VP; ++i) {
                    const int kv = j0 + 16 * b + 4 * (lane >> 4) + i;
                    vp[b][i] = table[block_at(p, kv < limit ? kv : 0)];
                }
            }
        }
    }

    // The 32 keys (load_k) or values (load_v) from j0 on; what lies at `limit` or
    // behind it is some row.
    __device__ __forceinline__ void load_k(const Pages &pg, const Params &p, int kvh, int j0, int limit) {
        const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            int key = j0 + 16 * b + (BSM == 1 ? 0 : m);
            key = key < limit ? key : 0;
            long long kr = row_of(p, kvh, pg.kp[b], key, block_at(p, key));
            long long sr = kr + 4 * g;
            if (BSM == 1) kr += m;
            const u32_a4 *kw = reinterpret_cast<const u32_a4 *>(p.kc + kr * (D / 2)) + g * KW;
#pragma unroll
            for (int w = 0; w < KW; ++w) k[b][w] = __builtin_nontemporal_load(kw + w);
            if constexpr (BSM != 1) sr = row4(pg, p, kvh, j0, limit, b, 0);
            ks[b] = pairs4(pg, p, p.ks, kvh, j0, limit, b, sr);
        }
    }
    __device__ __forceinline__ void load_v(const Pages &pg, const Params &p, int kvh, int j0, int limit) {
        const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            long long r0;
            if constexpr (BSM == 1) {
                const int key = j0 + 16 * b < limit ? j0 + 16 * b : 0;
                r0 = row_of(p, kvh, pg.kp[b], key, block_at(p, key)) + 4 * g;
            } else {
                r0 = row4(pg, p, kvh, j0, limit, b, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *row = p.vc + (BSM == 0 && i > 0 ? row4(pg, p, kvh, j0, limit, b, i) : r0 + i) * (D / 2);
#pragma unroll
                for (int n = 0; n < N128; ++n)
                    v[b][i][n] = __builtin_nontemporal_load(reinterpret_cast<const u32_a4 *>(row + 64 * n) + m);
                if constexpr (N64 > 0)
                    v[b][i][N128] = *(reinterpret_cast<const uint16_t *>(row + 64 * N128) + m);
                if constexpr (N32 > 0) v[b][i][N128 + N64] = row[64 * N128 + 32 * N64 + m];
            }
            vs[b] = pairs4(pg, p, p.vs, kvh, j0, limit, b, r0);
        }
    }

private:
    // Row of this lane's key i of its four of half b.
    static __device__ __forceinline__ long long row4(const Pages &pg, const Params &p, int kvh, int j0, int limit, int b,
                                                     int i) {
        int key = j0 + 16 * b + 4 * static_cast<int>(threadIdx.x >> 4 & 3) + i;
        key = key < limit ? key : 0;
        return row_of(p, kvh, pg.vp[b][BSM == 0 ? i : 0], key, block_at(p, key));
    }
    // The pairs of its four keys, the first in row r0.
    static __device__ __forceinline__ u32x4 pairs4(const Pages &pg, const Params &p, const uint32_t *pairs, int kvh, int j0,
                                                   int limit, int b, long long r0) {
        if constexpr (BSM == 0) {
            u32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pairs[i == 0 ? r0 : row4(pg, p, kvh, j0, limit, b, i)];
            return x;
        } else {
            typedef u32x4 __attribute__((aligned(4))) u32x4_a4;
            return *reinterpret_cast<const u32x4_a4 *>(pairs + r0);
        }
    }
};

// 8 codes of a word as fp16 subnormals: pairs (0, 4), (1, 5) * 16, (2, 6),
// (3, 7) * 16 of elements, in units of 2^-24.
__device__ __forceinline__ u32x4 widen8(uint32_t w) {
    const uint32_t h = w >> 8;
    return u32x4{w & 0x000f000fu, w & 0x00f000f0u, h & 0x000f000fu, h & 0x00f000f0u};
}

// State of a wave: per column tile the running maximum (log2 domain), the sums of
// the weights and of weight * middle of the row over this lane's keys, and the
// unnormalised sums of weight * scale * code, all in units of the power of two `ref`
// that the scales are taken relative to.
template <int D, int CT>
struct State {
    f32x4_t acc[CT][D / 16], w[CT];  // w: sums of the weights * scale as rounded
    float m[CT], l[CT], r[CT];
    float twice_ref;
    int ref;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            m[t] = kNever;
            l[t] = r[t] = 0.0f;
            w[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < D / 16; ++i) acc[t][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        ref = kLeastRef;
        twice_ref = power2(kLeastRef + 1);
    }
};

// A lane's column: its query in fp16, scaled, as the operand of the first product.
template <int D>
struct Column {
    u32x4 q[D / 32];
    float to_log2;  // raw score (codes in units of 2^-24) to log2 domain
    float sum;      // of the query's elements, as a raw score of codes 1
    int vis;        // keys that it sees
};

template <typename T, int D>
__device__ __forceinline__ void load_column(const Params &p, Column<D> &c, const uint16_t *src, bool there) {
    // this lane's quarter of the head: elements [g D/4, (g + 1) D/4)
    const int g = (threadIdx.x & 63) >> 4;
    u32x4 raw[D / 32];
    uint32_t most = 0;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        raw[w] = *reinterpret_cast<const u32x4 *>(src + g * (D / 4) + 8 * w);
        if (!there) raw[w] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = raw[w][i] & 0x7fff7fffu;
            most = max(most, max(a & 0xffffu, a >> 16));
        }
    }
    const float big = row_swap_max(half_swap_max(Cvt<T>::to(static_cast<uint16_t>(most))));
    // the largest element to [2^14, 2^15); infinities and NaN stay what they are
    int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
    e = min(max(e, -100), 120);
    const float up = power2(14 - e);
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = lo<T>(raw[w][i]) * up;
            f[2 * i + 1] = hi<T>(raw[w][i]) * up;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float unit = i & 1 ? 0.0625f : 1.0f;
            c.q[w][i] = __builtin_bit_cast(
                uint32_t, f16x2_t{static_cast<_Float16>(f[i] * unit), static_cast<_Float16>(f[i + 4] * unit)});
        }
    }
    c.sum = row_swap_sum(half_swap_sum(s)) * 0x1p-24f;
    c.to_log2 = p.scale_log2 * power2(e - 14) * 0x1p24f;
}

// Scores of the 32 keys from j0 on, held in `b`, before their factor to_log2.  Keys at
// `limit` or behind it, and keys that a column does not see, score -inf and have pairs
// of 0, whatever the cache holds there; `edge`: some are among these.
template <typename T, int D, int CT, int BSM>
__device__ __forceinline__ void scores(Block<D, BSM> &b, const Column<D> (&col)[CT], f32x4_t (&s)[CT][2], int j0,
                                       int limit, bool edge) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[t][h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 a = widen8(b.k[h][w]);
#pragma unroll
            for (int t = 0; t < CT; ++t) s[t][h] = mma16(a, col[t].q[w], s[t][h]);
        }
    if (edge) {
        asm volatile("");  // (a branch, taken in the last block alone)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (j0 + 16 * h + 4 * g + i >= limit) b.ks[h][i] = 0u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float sk = lo<T>(b.ks[h][i]), ak = hi<T>(b.ks[h][i]);
#pragma unroll
            for (int t = 0; t < CT; ++t) s[t][h][i] = fmaf(sk, s[t][h][i], ak * col[t].sum);
        }
    if (edge) {
        asm volatile("");
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (j0 + 16 * h + 4 * g + i >= min(limit, col[t].vis)) s[t][h][i] = kNegInf;
    }
}

// Their values, weighted by the softmax of the scores, into the state.
template <typename T, int D, int CT, int BSM>
__device__ __forceinline__ void weigh(Block<D, BSM> &b, const Column<D> (&col)[CT], const f32x4_t (&s)[CT][2],
                                      State<D, CT> &st, int j0, int limit, bool edge) {
    const int g = (threadIdx.x & 63) >> 4;
    if (edge) {
        asm volatile("");
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (j0 + 16 * h + 4 * g + i >= limit) b.vs[h][i] = 0u;
    }
    float sv[2][4], av[2][4];
    float top = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sv[h][i] = lo<T>(b.vs[h][i]);
            av[h][i] = fmaf(kMiddle, sv[h][i], hi<T>(b.vs[h][i]));
            top = fmaxf(top, fabsf(sv[h][i]));
        }
    // scales relative to a power of two that is at least half of the largest seen
    if (!__all(top <= st.twice_ref)) {
        top = row_swap_max(half_swap_max(top));
        const int e = min(static_cast<int>(__float_as_uint(top) >> 23) - 127, 100);
        if (e > st.ref) {
            const float down = e - st.ref > 120 ? 0.0f : power2(st.ref - e);
            st.ref = e;
            st.twice_ref = power2(e + 1);
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                st.l[t] *= down;
                st.r[t] *= down;
                st.w[t] *= down;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) st.acc[t][i] *= down;
            }
        }
    }
    u32x4 pw[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        float mx = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                         fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3]))) * col[t].to_log2;
        if (!__all(mx <= st.m[t] + kSlack)) {
            mx = row_swap_max(half_swap_max(mx));
            const float next = fmaxf(st.m[t], mx);
            const float f = __builtin_amdgcn_exp2f(st.m[t] - next);
            st.m[t] = next;
            st.l[t] *= f;
            st.r[t] *= f;
            st.w[t] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) st.acc[t][i] *= f;
        }
        const float shift = kTop - st.m[t] - static_cast<float>(st.ref);
        float w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][h][i], col[t].to_log2, shift));
                st.l[t] += e;
                st.r[t] = fmaf(e, av[h][i], st.r[t]);
                w[h][i] = e * sv[h][i];
            }
        pw[t] = u32x4{Mma<f16>::pack2(w[0][0], w[0][1]), Mma<f16>::pack2(w[0][2], w[0][3]),
                      Mma<f16>::pack2(w[1][0], w[1][1]), Mma<f16>::pack2(w[1][2], w[1][3])};
        constexpr uint32_t one = 0x3c003c00u;
        st.w[t] = mma16(u32x4{one, one, one, one}, pw[t], st.w[t]);
    }
    // values: words of 8, 4 or 2 channels of a key become, per pair of keys, words
    // of one channel each
    using B = Block<D, BSM>;
    const auto product = [&](int tile, const u32x4 &a) {
#pragma unroll
        for (int t = 0; t < CT; ++t) st.acc[t][tile] = mma16(a, pw[t], st.acc[t][tile]);
    };
    const auto four = [&](int tile, const u32x4 &x) {  // x[i]: 16 bits of two keys
        const u32x4 y = x >> 8;
        product(tile, x & 0x000f000fu);
        product(tile + 1, x & 0x00f000f0u);
        product(tile + 2, y & 0x000f000fu);
        product(tile + 3, y & 0x00f000f0u);
    };
    const auto pairs = [&](int n, uint32_t select) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_amdgcn_perm(b.v[i >> 1][2 * (i & 1) + 1][n], b.v[i >> 1][2 * (i & 1)][n], select);
        return x;
    };
#pragma unroll
    for (int n = 0; n < B::N128; ++n) {
        four(8 * n, pairs(n, 0x05040100u));
        four(8 * n + 4, pairs(n, 0x07060302u));
    }
    if constexpr (B::N64 > 0) four(8 * B::N128, pairs(B::N128, 0x05040100u));
    if constexpr (B::N32 > 0) {
        const u32x4 x = pairs(B::N128 + B::N64, 0x05040100u);
        product(8 * B::N128 + 4 * B::N64, x & 0x000f000fu);
        product(8 * B::N128 + 4 * B::N64 + 1, x & 0x00f000f0u);
    }
}

// Channel of row m of an accumulator tile.
template <int D>
__device__ __forceinline__ int channel_of(int tile, int m) {
    constexpr int N128 = D / 128, N64 = D % 128 / 64;
    if (tile < 8 * N128) return 128 * (tile >> 3) + 8 * m + (tile & 7);
    if (tile < 8 * N128 + 4 * N64) return 128 * N128 + 4 * m + (tile - 8 * N128);
    return 128 * N128 + 64 * N64 + 2 * m + (tile - 8 * N128 - 4 * N64);
}

template <int D, int CT>
constexpr size_t split_lds() {
    return sizeof(float) * kWaves * 16 * CT * (D + 2);
}

// Columns [c0, c0 + 16 CT) of (sequence, kv head) over the keys [lo, hi): column j
// is query row j / G, head j % G of the group.  Leaves the waves' states in LDS,
// after a barrier: maximum, sum and unnormalised output of each column.
template <typename T, int D, int CT, int BSM>
__device__ __forceinline__ void split_pass(const Params &p, float *lds, int b, int kvh, long long q_off, int L, int S,
                                           int c0, int lo, int hi) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q_start = p.causal ? max(S - L, 0) : 0;
    const int last = min(c0 + 16 * CT, p.G * L) - 1;
    // no column sees more than the last one
    const int limit = p.causal ? min(hi, q_start + last / p.G + 1) : hi;
    const int least = p.causal ? min(limit, q_start + c0 / p.G + 1) : limit;
    const int *table = p.bt + b * p.bt_stride;
    Column<D> col[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int j = min(c0 + 16 * t + n, last);
        const int row = j / p.G, head = j - row * p.G;
        load_column<T, D>(p, col[t], p.q + ((q_off + row) * p.H + kvh * p.G + head) * D, c0 + 16 * t + n <= last);
        col[t].vis = p.causal ? q_start + row + 1 : S;
    }
    State<D, CT> st;
    st.clear();
    // The next block's keys are asked for once this one's scores are done, its values
    // once these are used: one set of registers each, and more waves, whose loads
    // overlap, in place of a second set.
    using B = Block<D, BSM>;
    B blk;
    typename B::Pages pages, next;
    constexpr int STEP = 32 * kWaves;
    int j0 = lo + 32 * wave;
    if (j0 < limit) {
        B::pages(pages, p, table, j0, limit);
        blk.load_k(pages, p, kvh, j0, limit);
        blk.load_v(pages, p, kvh, j0, limit);
        if (j0 + STEP < limit) B::pages(next, p, table, j0 + STEP, limit);
    }
    for (; j0 < limit; j0 += STEP) {
        const bool edge = j0 + 32 > least, more = j0 + STEP < limit;
        f32x4_t s[CT][2];
        scores<T, D, CT, BSM>(blk, col, s, j0, limit, edge);
        pages = next;
        if (more) {
            blk.load_k(pages, p, kvh, j0 + STEP, limit);
            if (j0 + 2 * STEP < limit) B::pages(next, p, table, j0 + 2 * STEP, limit);
        }
        weigh<T, D, CT, BSM>(blk, col, s, st, j0, limit, edge);
        if (more) blk.load_v(pages, p, kvh, j0 + STEP, limit);
    }
    constexpr int COLS = 16 * CT;
    float *lm = lds, *ll = lm + kWaves * COLS, *lout = ll + kWaves * COLS;
    const float ref = power2(st.ref);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const float l = row_swap_sum(half_swap_sum(st.l[t])), r = row_swap_sum(half_swap_sum(st.r[t]));
        const int c = wave * COLS + 16 * t + n;
        if (g == 0) {
            lm[c] = st.m[t];
            ll[c] = l * ref;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const float unit = (i & 1) ? 0x1p20f : 0x1p24f;
#pragma unroll
            for (int v = 0; v < 4; ++v)
                lout[c * D + channel_of<D>(i, 4 * g + v)] =
                    ref * (fmaf(st.acc[t][i][v], unit, -kMiddle * st.w[t][v]) + r);
        }
    }
    __syncthreads();
}

// sink(column, channel, output, maximum, sum) of the waves' states in LDS.
template <int D, int CT, typename Sink>
__device__ __forceinline__ void merge_states(const float *lds, int cols, Sink sink) {
    constexpr int COLS = 16 * CT;
    const float *lm = lds, *ll = lm + kWaves * COLS, *lout = ll + kWaves * COLS;
    for (int task = threadIdx.x; task < cols * D; task += blockDim.x) {
        const int c = task / D, d = task % D;
        float M = lm[c];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) M = fmaxf(M, lm[w * COLS + c]);
        float out = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(lm[w * COLS + c] - M);
            out = fmaf(f, lout[(w * COLS + c) * D + d], out);
            sum = fmaf(f, ll[w * COLS + c], sum);
        }
        sink(c, d, out, M, sum);
    }
}

__device__ __forceinline__ int splits_of(const Params &p, int S) {
    return min(max((S + p.split_len - 1) / p.split_len, 1), p.splits);
}

// Workgroup (sequence, kv head, column tile) and split: the last split holds every
// key past the splits, and rows past the bound that the grid was made for are done
// by the workgroups of split 0, over all keys, so that the bounds shape the launch
// alone.
template <typename T, int D, int CT, int BSM>
__global__ void __launch_bounds__(64 * kWaves, D * CT <= 64 && CT == 1 ? 4 : D * CT <= 128 ? 3 : D * CT <= 256 ? 2 : 1) split_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float states[];
    if (blockIdx.x == 0 && blockIdx.y == 0) zero_tail(p, D);
    const int tile = blockIdx.x % p.tiles;
    const int kvh = blockIdx.x / p.tiles % p.Hkv;
    const int b = blockIdx.x / p.tiles / p.Hkv;
    const int split = blockIdx.y;
    long long q_off;
    int L, S;
    sequence(p, b, q_off, L, S);
    const int all = p.G * max(L, 0), ns = splits_of(p, S);
    const auto write = [&](int c0) {
        return [&, c0](int c, int d, float out, float, float sum) {
            const int j = c0 + c, row = j / p.G;
            p.o[((q_off + row) * p.H + kvh * p.G + (j - row * p.G)) * D + d] =
                Cvt<T>::from(sum > 0.0f ? out / sum : 0.0f * sum);
        };
    };
    int c0 = tile * 16 * CT;
    if (c0 < min(all, p.cols) && split < ns) {
        const int lo = split * p.split_len, hi = split == ns - 1 ? S : lo + p.split_len;
        const int cols = min(16 * CT, min(all, p.cols) - c0);
        split_pass<T, D, CT, BSM>(p, states, b, kvh, q_off, L, S, c0, lo, hi);
        if (p.splits == 1) {
            merge_states<D, CT>(states, cols, write(c0));
        } else {
            const long long base = ((static_cast<long long>(b) * p.Hkv + kvh) * p.splits + split) * p.cols + c0;
            merge_states<D, CT>(states, cols, [&](int c, int d, float out, float M, float sum) {
                p.ws_o[(base + c) * D + d] = out;
                if (d == 0) {
                    p.ws_ml[(base + c) * 2] = M;
                    p.ws_ml[(base + c) * 2 + 1] = sum;
                }
            });
        }
    }
    if (split != 0) return;
    // (p.cols need not be a whole number of tiles: the rest starts at it)
    for (c0 = p.cols + tile * 16 * CT; c0 < all; c0 += p.tiles * 16 * CT) {
        __syncthreads();
        split_pass<T, D, CT, BSM>(p, states, b, kvh, q_off, L, S, c0, 0, S);
        merge_states<D, CT>(states, min(16 * CT, all - c0), write(c0));
    }
}

// The splits' states of a column into its output row: D / 4 lanes a column.
template <typename T, int D>
__global__ void __launch_bounds__(256) combine_kernel(Params p) {
    constexpr int V = D / 4, COLS = 256 / V, AHEAD = 4;
    const int kvh = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int c = blockIdx.y * COLS + threadIdx.x / V, e = threadIdx.x % V;
    long long q_off;
    int L, S;
    sequence(p, b, q_off, L, S);
    if (threadIdx.x >= COLS * V || c >= min(p.cols, p.G * L)) return;
    const int ns = splits_of(p, S);
    const long long base = (static_cast<long long>(b) * p.Hkv + kvh) * p.splits * p.cols + c;
    float M = kNever, sum = 0.0f;
    float4_t out = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < ns; s0 += AHEAD) {
        float4_t o[AHEAD];
        float2_t ml[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const long long at = base + static_cast<long long>(min(s0 + u, ns - 1)) * p.cols;
            o[u] = *reinterpret_cast<const float4_t *>(p.ws_o + at * D + 4 * e);
            ml[u] = *reinterpret_cast<const float2_t *>(p.ws_ml + at * 2);
        }
        float next = M;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) next = fmaxf(next, ml[u].x);
        const float f = __builtin_amdgcn_exp2f(M - next);
        M = next;
        sum *= f;
        out *= f;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float w = s0 + u < ns ? __builtin_amdgcn_exp2f(ml[u].x - M) : 0.0f;
            sum = fmaf(w, ml[u].y, sum);
            out += w * o[u];
        }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f * sum;
    const int row = c / p.G;
    uint16_t *dst = p.o + ((q_off + row) * p.H + kvh * p.G + (c - row * p.G)) * D + 4 * e;
    store_row4<T>(dst, out.x * inv, out.y * inv, out.z * inv, out.w * inv);
}

// ---------------------------------------------------------------- tile route

// K and V tiles of TILE keys from the cache into LDS as fp16, both row-major (the
// layout that wave_attend reads with transposing loads): a thread's tasks are
// 16-byte words of codes, 32 elements of a row.
template <typename T, int D, int TILE, int NT>
struct Widener {
    static constexpr int KP = D + 8, VR = D + kVRowPad;
    static constexpr int VOFF = TILE * KP, ELEMS = TILE * (KP + VR);
    static constexpr int WORDS = D / 32;  // of a row
    static constexpr int HALF = TILE * WORDS, TASKS = 2 * HALF;
    static constexpr int PER = (TASKS + NT - 1) / NT;
    u32x4 codes[PER];
    uint32_t pair[PER];
    int page[PER];
    float most_k, most_v;  // largest magnitude seen

    __device__ __forceinline__ void pages(const Params &p, const int *table, int j0, int limit) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int task = (static_cast<int>(threadIdx.x) + i * NT) % HALF;
            const int key = j0 + task / WORDS;
            page[i] = table[block_at(p, key < limit ? key : 0)];
        }
    }
    __device__ __forceinline__ void load(const Params &p, int kvh, int j0, int limit) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = static_cast<int>(threadIdx.x) + i * NT;
            const int task = t % HALF, word = task % WORDS;
            const bool is_v = t >= HALF;
            int key = j0 + task / WORDS;
            const bool there = key < limit;
            key = there ? key : 0;
            const long long row = row_of(p, kvh, page[i], key, block_at(p, key));
            codes[i] = *reinterpret_cast<const u32x4 *>((is_v ? p.vc : p.kc) + row * (D / 2) + 16 * word);
            pair[i] = (is_v ? p.vs : p.ks)[row];
            if (!there) pair[i] = 0u;
        }
    }
    // rows times down_k (keys) and down_v (values)
    __device__ __forceinline__ void store(uint16_t *buf, float down_k, float down_v) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = static_cast<int>(threadIdx.x) + i * NT;
            if (TASKS % NT != 0 && t >= TASKS) continue;
            const int task = t % HALF, word = task % WORDS, row = task / WORDS;
            const bool is_v = t >= HALF;
            const float s = lo<T>(pair[i]), a = hi<T>(pair[i]);
            const float most = fmaxf(fabsf(a), fabsf(fmaf(15.0f, s, a)));
            if (is_v) most_v = fmaxf(most_v, most);
            else most_k = fmaxf(most_k, most);
            const float down = is_v ? down_v : down_k;
            const _Float16 sh = static_cast<_Float16>(s * down), ah = static_cast<_Float16>(a * down);
            const f16x2_t s2 = {sh, sh}, a2 = {ah, ah}, bias = {static_cast<_Float16>(-1024.0f), static_cast<_Float16>(-1024.0f)};
            uint16_t *dst = buf + (is_v ? VOFF + row * VR : row * KP) + 32 * word;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t x[4];  // elements (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t n = ((codes[i][w] >> (4 * e)) & 0x000f000fu) | 0x64006400u;  // 1024 + n
                    x[e] = __builtin_bit_cast(
                        uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, n) + bias, s2, a2));
                }
                *reinterpret_cast<u32x4 *>(dst + 8 * w) =
                    u32x4{__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                          __builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
            }
        }
    }
};

template <int D, int TILE, int W>
constexpr size_t tile_lds() {
    constexpr size_t kv = 2ull * Widener<f16, D, TILE, W * 64>::ELEMS, o = static_cast<size_t>(32 * W) * (D + 8);
    return sizeof(uint16_t) * (kv > o ? kv : o);
}

// Columns [c0, c0 + 32 W) below `all` of (sequence, kv head) over the keys [from, to): wave w
// serves columns 32 w .. + 31, column j being query row j / G, head j % G of the
// group, so that heads of any number fill the waves.  Into the output rows, or with
// `part` into the states [column][D], (maximum, sum) [column].  Ends with a barrier.
template <typename T, int D, int W, int TILE>
__device__ __forceinline__ void column_tile(const Params &p, uint16_t *lds, float *meet, int b, int kvh, long long q_off,
                                            int L, int S, int all, int c0, int from, int to, float *part,
                                            float *part_ml) {
    constexpr int NKB = TILE % 64 == 0 ? 2 : 1, KB = 32 * NKB, COLS = 32 * W;
    using Wd = Widener<T, D, TILE, W * 64>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 5, r32 = lane & 31;
    const int cw0 = c0 + 32 * wave;
    const int q_start = p.causal ? max(S - L, 0) : 0;
    const auto seen = [&](int j) { return p.causal ? min(to, q_start + j / p.G + 1) : to; };
    const int kv_end = seen(min(c0 + COLS, all) - 1);
    const int wave_end = __builtin_amdgcn_readfirstlane(cw0 < all ? seen(min(cw0 + 32, all) - 1) : from);
    const int wave_least = __builtin_amdgcn_readfirstlane(seen(min(cw0, all - 1)));
    const int *table = p.bt + b * p.bt_stride;
    const int j = min(cw0 + r32, all - 1), row = j / p.G;
    const int vis = seen(j);

    // the wave's queries in fp16, their largest element to [2^8, 2^9)
    u32x4 qf[1][D / 16];
    float q_unit;
    {
        const uint16_t *src = p.q + ((q_off + row) * p.H + kvh * p.G + (j - row * p.G)) * D;
        uint32_t most = 0;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const u32x4 x = *reinterpret_cast<const u32x4 *>(src + 16 * ks + 8 * g);
            qf[0][ks] = x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = x[i] & 0x7fff7fffu;
                most = max(most, max(a & 0xffffu, a >> 16));
            }
        }
        const float big = wave_max(Cvt<T>::to(static_cast<uint16_t>(most)));
        int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
        e = min(max(e, -100), 120);
        const float up = power2(8 - e);
        q_unit = power2(e - 8);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                qf[0][ks][i] = Mma<f16>::pack2(tecoops::dev::lo<T>(qf[0][ks][i]) * up, tecoops::dev::hi<T>(qf[0][ks][i]) * up);
    }

    float m[1], lsum[1];
    f32x16_t oacc[1][D / 32];
    Wd wd;
    int ek = 0, ev = 0;
    const int ntiles = kv_end > from ? (kv_end - from + TILE - 1) / TILE : 0;
    for (int pass = 0;; ++pass) {
        const float down_k = power2(-ek), down_v = power2(-ev);
        const float scale = p.scale_log2 * q_unit * power2(ek), inv_scale = 1.0f / scale;
        m[0] = kNever;
        lsum[0] = 0.0f;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int v = 0; v < 16; ++v) oacc[0][db][v] = 0.0f;
        wd.most_k = wd.most_v = 0.0f;
        const auto buf = [&](int t) { return lds + __builtin_amdgcn_readfirstlane((t & 1) * Wd::ELEMS); };
        if (ntiles > 0) {
            wd.pages(p, table, from, to);
            wd.load(p, kvh, from, to);
            wd.pages(p, table, from + TILE, to);
            wd.store(buf(0), down_k, down_v);
        }
        __syncthreads();
        for (int it = 0; it < ntiles; ++it) {
            const uint16_t *cur = buf(it);
            if (it + 1 < ntiles) {
                wd.load(p, kvh, from + (it + 1) * TILE, to);
                wd.pages(p, table, from + (it + 2) * TILE, to);
            }
#pragma unroll
            for (int hb = 0; hb < TILE / KB; ++hb) {
                const int j0 = from + it * TILE + KB * hb;
                if (j0 < wave_end) {
                    const int lim[1] = {vis - j0 - 4 * g};
                    wave_attend<f16, D, Wd::KP, 0, Wd::VR, NKB, 1, true>(cur, cur + Wd::VOFF, KB * hb, qf, oacc, m, lsum,
                                                                        lim, scale, inv_scale, j0 + KB > wave_least);
                }
            }
            if (it + 1 < ntiles) wd.store(buf(it + 1), down_k, down_v);
            __syncthreads();
        }
        // rows out of fp16's range, or all of them down where it has few bits: once
        // more, with the power of two that their largest asks for
        if (pass == 1) break;
        const float mk = wave_max(wd.most_k), mv = wave_max(wd.most_v);
        if (lane == 0) {
            meet[wave] = mk;
            meet[W + wave] = mv;
        }
        __syncthreads();
        float all_k = 0.0f, all_v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            all_k = fmaxf(all_k, meet[w]);
            all_v = fmaxf(all_v, meet[W + w]);
        }
        __syncthreads();
        const auto outside = [](float most) { return most < INFINITY && most > 0.0f && (most > 0x1p15f || most < 0x1p-6f); };
        if (!outside(all_k) && !outside(all_v)) break;
        const auto power = [&](float most) {
            return outside(most) ? min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127 - 10, -110), 110) : 0;
        };
        ek = __builtin_amdgcn_readfirstlane(power(all_k));
        ev = __builtin_amdgcn_readfirstlane(power(all_v));
    }
    const float lt = half_swap_sum(lsum[0]);
    if (part != nullptr) {
        if (cw0 + r32 < all) {
            float *dst = part + static_cast<long long>(j) * D;
            const float unit = power2(ev);
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    *reinterpret_cast<float4_t *>(dst + 32 * db + 8 * u + 4 * g) =
                        float4_t{oacc[0][db][4 * u] * unit, oacc[0][db][4 * u + 1] * unit, oacc[0][db][4 * u + 2] * unit,
                                 oacc[0][db][4 * u + 3] * unit};
            if (g == 0) *reinterpret_cast<float2_t *>(part_ml + static_cast<long long>(j) * 2) = float2_t{m[0], lt};
        }
        return;  // (the loop's last barrier has passed)
    }
    // O leaves through LDS, a column at a time
    constexpr int OROW = D + 8, RCH = D / 8, NOC = (COLS * RCH + W * 64 - 1) / (W * 64);
    const float inv = (lt > 0.0f ? 1.0f / lt : 0.0f * lt) * power2(ev);
    uint16_t *dst = lds + (32 * wave + r32) * OROW;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int u = 0; u < 4; ++u)
            store_row4<T>(dst + 32 * db + 8 * u + 4 * g, oacc[0][db][4 * u] * inv, oacc[0][db][4 * u + 1] * inv,
                          oacc[0][db][4 * u + 2] * inv, oacc[0][db][4 * u + 3] * inv);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NOC; ++i) {
        const int t = static_cast<int>(threadIdx.x) + i * W * 64, c = t / RCH, jj = c0 + c;
        if (t >= COLS * RCH || jj >= all) continue;
        const int r = jj / p.G;
        *reinterpret_cast<u32x4 *>(p.o + ((q_off + r) * p.H + kvh * p.G + (jj - r * p.G)) * D + (t - c * RCH) * 8) =
            *reinterpret_cast<const u32x4 *>(lds + c * OROW + (t - c * RCH) * 8);
    }
    __syncthreads();
}

// Workgroup (sequence, kv head) and (column tile, split), the heaviest tiles first;
// that of tile 0 and split 0 goes on to the columns past the grid, of which there
// are none where the bound on the rows holds.
template <typename T, int D, int W, int TILE>
__global__ void __launch_bounds__(W * 64, W >= 12 ? 3 : D <= 128 && W == 4 ? 3 : 2) tile_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) uint16_t tiles_lds[];
    __shared__ float meet[2 * W];
    if (blockIdx.x == 0 && blockIdx.y == 0) zero_tail(p, D);
    constexpr int COLS = 32 * W;
    const int kvh = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
    const int split = blockIdx.y % p.splits, tile = p.tiles - 1 - blockIdx.y / p.splits;
    long long q_off;
    int L, S;
    sequence(p, b, q_off, L, S);
    if (L <= 0) return;
    const int all = p.G * L, bound = min(all, p.cols);
    int c0 = tile * COLS;
    if (c0 < bound && p.splits == 1) {
        column_tile<T, D, W, TILE>(p, tiles_lds, meet, b, kvh, q_off, L, S, bound, c0, 0, S, nullptr, nullptr);
    } else if (c0 < bound) {
        const int ns = splits_of(p, S);
        const long long at = (static_cast<long long>(b) * p.Hkv + kvh) * p.splits + split;
        if (split < ns)
            column_tile<T, D, W, TILE>(p, tiles_lds, meet, b, kvh, q_off, L, S, bound, c0, split * p.split_len,
                                       split == ns - 1 ? S : (split + 1) * p.split_len, p.ws_o + at * p.cols * D,
                                       p.ws_ml + at * p.cols * 2);
    }
    if (tile != 0 || split != 0) return;
    for (c0 = p.cols; c0 < all; c0 += COLS) {
        __syncthreads();
        column_tile<T, D, W, TILE>(p, tiles_lds, meet, b, kvh, q_off, L, S, all, c0, 0, S, nullptr, nullptr);
    }
}

// ------------------------------------------------------------------- host

template <typename T, int D>
tecoopsStatus_t launch_combine(const Params &p, const Plan &pl, hipStream_t s) {
    if (pl.splits <= 1) return TECOOPS_STATUS_SUCCESS;
    constexpr int COLS = 256 / (D / 4);
    hipLaunchKernelGGL((combine_kernel<T, D>), dim3(p.batch * p.Hkv, tecoops::ceil_div(pl.cols, COLS)), dim3(256), 0, s, p);
    TECO_CHECK_LAUNCH("flash_attention_int4 combine");
    return TECOOPS_STATUS_SUCCESS;
}

template <typename T, int D, int CT>
tecoopsStatus_t launch_split(const Params &p, const Plan &pl, hipStream_t s) {
    const size_t lds = split_lds<D, CT>();
    auto *kern = p.bs % 16 == 0  ? &split_kernel<T, D, CT, 1>
                 : p.bs % 4 == 0 ? &split_kernel<T, D, CT, 2>
                                 : &split_kernel<T, D, CT, 0>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return TECOOPS_STATUS_INTERNAL_ERROR;
    hipLaunchKernelGGL(kern, dim3(p.batch * p.Hkv * pl.tiles, pl.splits), dim3(64 * kWaves), lds, s, p);
    TECO_CHECK_LAUNCH("flash_attention_int4");
    return launch_combine<T, D>(p, pl, s);
}

template <typename T, int D, int W, int TILE>
tecoopsStatus_t launch_tiles(const Params &p, const Plan &pl, hipStream_t s) {
    constexpr size_t lds = tile_lds<D, TILE, W>();
    static_assert(lds + 8 * W <= tecoops::kLdsMax, "fits the LDS");
    auto *kern = &tile_kernel<T, D, W, TILE>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return TECOOPS_STATUS_INTERNAL_ERROR;
    hipLaunchKernelGGL(kern, dim3(p.batch * p.Hkv, pl.tiles * pl.splits), dim3(W * 64), lds, s, p);
    TECO_CHECK_LAUNCH("flash_attention_int4");
    return launch_combine<T, D>(p, pl, s);
}

template <typename T, int D>
tecoopsStatus_t launch_size(const Params &p, const Plan &pl, hipStream_t s) {
    if (pl.split) return pl.ct == 1 ? launch_split<T, D, 1>(p, pl, s) : launch_split<T, D, 2>(p, pl, s);
    if (pl.waves == 4) return launch_tiles<T, D, 4, 32>(p, pl, s);
    if constexpr (D <= 128) return launch_tiles<T, D, 12, 96>(p, pl, s);
    else return launch_tiles<T, D, 8, 64>(p, pl, s);
}

template <typename T>
tecoopsStatus_t launch_type(const Params &p, const Plan &pl, int head_size, hipStream_t s) {
    switch (head_size) {
        case 32: return launch_size<T, 32>(p, pl, s);
        case 64: return launch_size<T, 64>(p, pl, s);
        case 96: return launch_size<T, 96>(p, pl, s);
        case 128: return launch_size<T, 128>(p, pl, s);
        case 160: return launch_size<T, 160>(p, pl, s);
        default: return launch_size<T, 192>(p, pl, s);
    }
}

bool head_size_ok(int D) { return D >= 32 && D <= 192 && D % 32 == 0; }

}  // namespace

extern "C" tecoopsStatus_t tecoopsGetFlashAttentionInt4WorkspaceSize(int batch, int total_q, int num_heads,
                                                                     int num_kv_heads, int head_size,
                                                                     int max_seqlen_q, int max_seqlen_k,
                                                                     size_t *bytes) {
    if (bytes == nullptr || batch <= 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        num_heads % num_kv_heads != 0 || max_seqlen_k <= 0)
        return TECOOPS_STATUS_BAD_PARAM;
    if (!head_size_ok(head_size)) return TECOOPS_STATUS_NOT_SUPPORTED;
    const int rows = std::max(max_seqlen_q, static_cast<int>(tecoops::ceil_div(std::max(total_q, 1), batch)));
    *bytes = tecoops::fa4::make_plan(batch, num_heads, num_kv_heads, head_size, rows, max_seqlen_k, ~size_t{0},
                                     tecoops::device_cus())
                 .bytes;
    return TECOOPS_STATUS_SUCCESS;
}

extern "C" tecoopsStatus_t tecoopsFlashAttentionInt4(
    tecoopsHandle_t handle, int max_seqlen_q, int max_seqlen_k, const int *cu_seqlens_q, const int *kv_seq_lens,
    const int *block_table, long long block_table_stride, int batch, int blocks_per_seq, const void *q,
    const void *key_cache, const void *value_cache, const void *key_scales, const void *value_scales, void *out,
    int total_q, int num_heads, int num_kv_heads, int head_size, int num_blocks, int block_size, float softmax_scale,
    int causal, void *workspace, size_t workspace_bytes, tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (!cu_seqlens_q || !kv_seq_lens || !block_table || !q || !key_cache || !value_cache || !key_scales ||
        !value_scales || !out)
        return TECOOPS_STATUS_BAD_PARAM;
    if (batch <= 0 || total_q < 0 || blocks_per_seq < 0 || num_blocks <= 0 || block_size <= 0 || num_heads <= 0 ||
        num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || block_table_stride < 0)
        return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    TECO_RETURN_IF(!head_size_ok(head_size), TECOOPS_STATUS_NOT_SUPPORTED,
                   "flash_attention_int4: head_size %d not supported (32, 64, 96, 128, 160, 192)", head_size);
    for (const void *ptr : {q, key_cache, value_cache, static_cast<const void *>(out)})
        if (!tecoops::aligned(ptr, 16)) return TECOOPS_STATUS_BAD_PARAM;
    for (const void *ptr : {key_scales, value_scales, static_cast<const void *>(cu_seqlens_q),
                            static_cast<const void *>(kv_seq_lens), static_cast<const void *>(block_table)})
        if (!tecoops::aligned(ptr, 4)) return TECOOPS_STATUS_BAD_PARAM;
    if (workspace != nullptr && !tecoops::aligned(workspace, 16)) return TECOOPS_STATUS_BAD_PARAM;
    if (total_q == 0) return TECOOPS_STATUS_SUCCESS;
    Params p{};
    p.q = static_cast<const uint16_t *>(q);
    p.kc = static_cast<const uint8_t *>(key_cache);
    p.vc = static_cast<const uint8_t *>(value_cache);
    p.ks = static_cast<const uint32_t *>(key_scales);
    p.vs = static_cast<const uint32_t *>(value_scales);
    p.o = static_cast<uint16_t *>(out);
    p.bt = block_table;
    p.bt_stride = block_table_stride;
    p.cu_q = cu_seqlens_q;
    p.kv_lens = kv_seq_lens;
    p.batch = batch;
    p.H = num_heads;
    p.Hkv = num_kv_heads;
    p.G = num_heads / num_kv_heads;
    p.bs = block_size;
    p.lbs = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(block_size)) : -1;
    p.num_blocks = num_blocks;
    // (a block of keys past the last stays within an int)
    p.kv_cap = static_cast<int>(std::min(static_cast<long long>(blocks_per_seq) * block_size, 0x7fffffffll - 4096));
    const float scale = softmax_scale > 0.0f ? softmax_scale : 1.0f / std::sqrt(static_cast<float>(head_size));
    p.scale_log2 = scale * 1.4426950408889634f;
    p.causal = causal != 0;
    p.total_q = total_q;
    const int rows = std::max(max_seqlen_q, static_cast<int>(tecoops::ceil_div(total_q, batch)));
    const int keys = max_seqlen_k > 0 ? max_seqlen_k : std::max(p.kv_cap, 1);
    TECO_RETURN_IF(static_cast<long long>(total_q) * p.G >= (1ll << 31), TECOOPS_STATUS_NOT_SUPPORTED,
                   "flash_attention_int4: too many query rows");
    const int cus = tecoops::device_cus();
    const auto plan = [&](size_t room) {
        return tecoops::fa4::make_plan(batch, num_heads, num_kv_heads, head_size, rows, keys, room, cus);
    };
    Plan pl = plan(workspace != nullptr ? workspace_bytes : ~size_t{0});
    if (pl.bytes > 0 && workspace == nullptr) {
        workspace = tecoops::handle_scratch_if_any(handle, pl.bytes);
        if (workspace == nullptr) pl = plan(0);
    }
    // the grid within 32-bit thread counts
    if (static_cast<long long>(batch) * num_kv_heads * pl.tiles * pl.splits > (1ll << 22)) return TECOOPS_STATUS_NOT_SUPPORTED;
    p.cols = pl.cols;
    p.tiles = pl.tiles;
    p.split_len = pl.split_len;
    p.splits = pl.splits;
    if (pl.splits > 1) {
        p.ws_o = static_cast<float *>(workspace);
        p.ws_ml = p.ws_o + pl.bytes / sizeof(float) / (head_size + 2) * head_size;
    }
    hipStream_t s = handle->stream;
    return dataType == TECOOPS_DATA_HALF ? launch_type<f16>(p, pl, head_size, s) : launch_type<bf16>(p, pl, head_size, s);
}
