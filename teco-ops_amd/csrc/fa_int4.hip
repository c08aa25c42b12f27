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
// element in its column, P s by the running maximum and the largest scale that the
// column has seen), so that bf16's range is kept and small weights of long contexts lose
// nothing.
//   * Scores are computed transposed (keys x columns, 16x16x32), so that a lane
//     holds 8 keys of one column, which are the operand of the second product as
//     they are: neither P nor the codes go through LDS.  With at most 8 or 4 columns
//     the 16 of the matrix core hold each 2 or 4 times, and a lane takes 4 or 2 of the
//     8 keys through the softmax.
//   * A wave takes every 4th block of 32 keys, copied into a ring in LDS without
//     registers while it works on the blocks before.  Partial states meet in LDS,
//     those of splits in a second kernel.
//   * [64 sequences of 512 to 8192 keys, 32 heads on 8 of 128, bf16] 72 us, 60 of them this
//     kernel at 4.8 TB/s (287 MB; a large read alone 5.9) and 5 the second one.  Issue:
//     per block some 150 vector, 120 scalar and 17 matrix instructions.  Loads through
//     registers and all 8 keys in each lane took 84; rings of 2 / 3 blocks 72.7 / 71.6;
//     splits of 4096 / 2048 / 1024 / 512 keys 73.7 / 71.5 / 75.1 / 87.5.
//
// Tile route (prefill in bf16).  K and V tiles are widened to fp16 once per workgroup, on
// the way into LDS, and attended as in flash_attention.hip (fa_device.h).  fp16 is 8 times
// closer than bf16 and a fixed range: rows of the cache are first taken as they are.  A
// tile of columns in which a row is too large, all are too small, or all that some column
// sees have too few bits is done again with powers of two that fit, and where its largest
// row is more than 2^24 above all that some column sees, key by key in fp32.  Rounded are
// K, V and the weights, each to 2^-11, which is unseen beside a bf16 output.  Beside an
// fp16 one it is seen (4e-4 to 6e-4, rms, against 2.1e-4), so that fp16 models have the
// split route for any number of columns, at up to twice the time.  Matrix cores are busy
// 39 % of the cycles, vector units 44 %, at the 12 waves a CU that LDS leaves room for: issue
// and waits in between.  [4 sequences, 2048 rows on up to 4096 keys, 32 heads on 8 of 128]
// 404 us, 800 TFLOP/s of visible pairs (fp16 by the split route 700); [2 of up to 203 rows on
// 16300 keys, 40 heads] 142 us, 760 (fp16 220).
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
    uint32_t inv_bs;                            // 2^32 / bs rounded up, or 0
    int kv_cap;                                 // keys that a table row can name
    long long page_rows;                        // rows of a block: heads * keys
    float scale_log2;
    int causal;
    long long total_q;
    float *ws_o, *ws_ml;
    int cols, tiles, split_len, splits;
};

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

// The power of two that brings a sum of weights next to 2^-10: with it a state's output
// is at most the largest value, whatever the number of keys.
__device__ __forceinline__ int near_1024th(float sum) {
    return sum > 0.0f && sum < INFINITY ? 117 - static_cast<int>(__float_as_uint(sum) >> 23) : 0;
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

// Cache block of a key: a shift, a product with 2^32 / bs where that is exact for
// every key that the table can name, or a division.
__device__ __forceinline__ int block_at(const Params &p, int key) {
    if (p.lbs >= 0) return key >> p.lbs;
    return p.inv_bs != 0u ? static_cast<int>(__umulhi(static_cast<uint32_t>(key), p.inv_bs)) : key / p.bs;
}

// Row of the cache, in rows of all blocks and heads, of a key whose block-table
// entry is `page`; entries out of range are taken as block 0.
__device__ __forceinline__ long long row_of(const Params &p, int kvh, int page, int key, int blk) {
    if (page < 0 || page >= p.num_blocks) page = 0;
    return (static_cast<long long>(page) * p.Hkv + kvh) * p.bs + (key - blk * p.bs);
}

// Weights are at most 2^kTop * 2^kSlack before the maximum is raised; scales at
// most twice the reference: P s stays below 2^15.  Rows of equal elements have scale 0
// whatever they hold: middles of rows are at most 2^kAside above that, so that P * middle
// stays below 2^56.
constexpr float kTop = 10.0f, kSlack = 4.0f;
constexpr float kMiddle = 7.5f;  // of the codes
constexpr int kLeastRef = -90;   // (sums of 2^24 weights stay within fp32)
constexpr float kAside = 0x1p40f;
// Past a reference of 2^kMostRef (in bf16 alone), sums in the values' units come near
// fp32's end, and past 2^100 small weights its start: from there on a wave takes its
// values in units of 2^kFar, and leaves a state whose sum is near 2^-10.
constexpr int kMostRef = 40, kFar = 64;
constexpr float kNever = -1e30f;  // the running maximum before any key

// N words of each lane from `base` + `off` (or `src`) to `dst` in LDS, lane after lane
// (M0 holds where; a copy has to be a wait state behind its write).
__device__ __forceinline__ uint32_t lds_address(char *at) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)(at)));
}
__device__ __forceinline__ void copy4(const void *base, uint32_t off, char *dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base),
                 "s"(lds_address(dst))
                 : "memory");
}
__device__ __forceinline__ void copy4(const void *src, char *dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_address(dst))
                 : "memory");
}
__device__ __forceinline__ void copy1(const void *src, char *dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds_address(dst))
                 : "memory");
}

// A wave's blocks of 32 keys on their way: keys, values and pairs go from the cache
// straight into LDS (global_load_lds, no registers), DEPTH blocks in a ring of the
// wave's own, so that a block is worked on while the next ones are under way.
//
//   keys    head_size 128: 16 bytes at 16 (64 h + 16 g + m), the words that lane
//           (g, m) reads for key 16 h + m; else rows as they are
//   values  rows, that of key 16 h + 4 g + i at 16 h + 4 i + g: the four rows that a
//           read touches lie together
//   pairs   32 of the keys, 32 of the values
//
// UNIFORM: pages hold a multiple of 16 keys, so that the pages of a block's halves are
// scalars, followed from block to block without a division, and where a copy's rows
// are of one half (head size 128) it costs no vector instruction but itself;
// else each lane looks its rows' entries up in a copy of the table's part in LDS
// (kTable entries; what lies behind them, in memory).
constexpr int kTable = 2048;

template <int D, bool UNIFORM>
struct Ring {
    static constexpr int KW = D / 32;               // 32-bit words of a key row in a lane
    static constexpr int N128 = D / 128, N64 = D % 128 / 64, N32 = D % 64 / 32;
    static constexpr int NI = (D + 63) / 64;        // copies of the keys, and of the values
    static constexpr int PER = 2 * NI + 1;          // copies of a block
    static constexpr int V_AT = NI * 1024, P_AT = 2 * NI * 1024, BYTES = P_AT + 256;
    static constexpr int DEPTH = D <= 64 ? 4 : 3;
    static constexpr int STEP = 32 * kWaves;        // keys from a wave's block to its next
    static constexpr bool SCALAR = UNIFORM && D == 128;
    static_assert((DEPTH - 1) * PER < 64, "vmcnt");

    const Params &p;
    const int *table, *copy;
    int kvh, first, limit;
    const uint32_t *pairs;  // of the lane: the keys' or the values'
    uint32_t koff, voff;    // SCALAR: the lane's 16 bytes within 16 rows
    // UNIFORM: the pages and places in them of the block to ask for next
    uint32_t in, step_in, within[2] = {0, 0};
    int blk, step_blk, last, page[2] = {0, 0};

    __device__ __forceinline__ Ring(const Params &params, int kv_head, const int *entries, const int *copied, int from,
                                    int end, int j0)
        : p(params), table(entries), copy(copied), kvh(kv_head), first(from), limit(end) {
        const int lane = threadIdx.x & 63;
        pairs = lane < 32 ? p.ks : p.vs;
        asm volatile("" : "+v"(pairs));  // (in registers, not loaded again for each block)
        koff = (lane & 15) * (D / 2) + 16 * (lane >> 4);
        voff = (4 * (lane >> 2 & 3) + (lane >> 4)) * (D / 2) + 16 * (lane & 3);
        if constexpr (UNIFORM) {
            const int b = block_at(p, j0);
            blk = __builtin_amdgcn_readfirstlane(b);
            in = __builtin_amdgcn_readfirstlane(j0 - b * p.bs);
            step_blk = __builtin_amdgcn_readfirstlane(block_at(p, STEP));
            step_in = __builtin_amdgcn_readfirstlane(STEP - block_at(p, STEP) * p.bs);
            last = __builtin_amdgcn_readfirstlane(block_at(p, max(limit - 1, 0)));
        }
    }

    // Asks for the table entries of the next block's halves (read-only for the launch:
    // scalar loads).  Behind the last key's page it is that page again.
    __device__ __forceinline__ void turn() {
        if constexpr (UNIFORM) {
            const auto *entry = (const __attribute__((address_space(4))) int *)(table);
            const bool next = in + 16 >= static_cast<uint32_t>(p.bs);
            within[0] = in;
            within[1] = next ? 0u : in + 16;
            page[0] = entry[min(blk, last)];
            page[1] = entry[min(next ? blk + 1 : blk, last)];
            blk += step_blk;
            in += step_in;
            if (in >= static_cast<uint32_t>(p.bs)) {
                in -= p.bs;
                ++blk;
            }
        }
    }

    // Row of key j0 + r of a block; half0, half1: the first rows of its halves (UNIFORM).
    __device__ __forceinline__ long long row(long long half0, long long half1, int j0, int r) const {
        if constexpr (UNIFORM) return half0 + (r < 16 ? 0 : half1 - half0) + (r & 15);
        const int key = j0 + r < limit ? j0 + r : first;
        const int b = block_at(p, key), at = b - block_at(p, first);
        return row_of(p, kvh, at < kTable ? copy[at] : table[b], key, b);
    }

    // Asks for the 32 keys from j0 on (UNIFORM: of the pages of the last turn()).
    __device__ __forceinline__ void load(int j0, char *dst) const {
        const int lane = threadIdx.x & 63;
        const auto first_row = [&](int pg, uint32_t at) {
            if (pg < 0 || pg >= p.num_blocks) pg = 0;
            return static_cast<uint32_t>(pg) * p.page_rows + static_cast<long long>(kvh) * p.bs + at;
        };
        const long long half0 = UNIFORM ? first_row(page[0], within[0]) : 0;
        const long long half1 = UNIFORM ? first_row(page[1], within[1]) : 0;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            if constexpr (SCALAR) {
                copy4(p.kc + (n == 0 ? half0 : half1) * (D / 2), koff, dst + 1024 * n);
            } else {
                const int c = min(64 * n + lane, D - 1);  // 16-byte words of 32 rows: D of them
                const int r = D == 128 ? 16 * n + (lane & 15) : c / KW, w = D == 128 ? lane >> 4 : c - r * KW;
                copy4(p.kc + row(half0, half1, j0, r) * (D / 2) + 16 * w, dst + 1024 * n);
            }
        }
        copy1(pairs + row(half0, half1, j0, lane & 31), dst + P_AT);
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            if constexpr (SCALAR) {
                copy4(p.vc + (n == 0 ? half0 : half1) * (D / 2), voff, dst + V_AT + 1024 * n);
            } else {
                const int c = min(64 * n + lane, D - 1), q = c / KW, w = c - q * KW;
                const int r = (q & 16) + 4 * (q & 3) + (q >> 2 & 3);
                copy4(p.vc + row(half0, half1, j0, r) * (D / 2) + 16 * w, dst + V_AT + 1024 * n);
            }
        }
    }

    // Waits until at most `newer` blocks asked for after this one are under way (any
    // other load under way only makes it wait for more).
    template <int NEWER>
    static __device__ __forceinline__ void wait() {
        constexpr int n = NEWER * PER;
        __builtin_amdgcn_s_waitcnt(((n >> 4) << 14) | 0x0F70 | (n & 15));
        asm volatile("" ::: "memory");
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
// unnormalised sums of weight * scale * code, all in units of the power of two ref()
// that the scales of the rows that the column sees are taken relative to.
template <typename T, int D, int CT>
struct State {
    f32x4_t acc[CT][D / 16], w[CT];  // w: sums of the weights * scale as rounded
    float m[CT], l[CT], r[CT];
    float shift[CT];      // of a score to its weight: kTop - maximum - ref
    float twice_ref[CT];  // 0: no sums yet; below 0: in units of 2^kFar (every block is looked at)

    __device__ __forceinline__ int ref(int t) const {
        return max(static_cast<int>(__float_as_uint(twice_ref[t]) >> 23 & 255u) - 128, kLeastRef);
    }
    // twice_ref's sign, the same in all columns.
    __device__ __forceinline__ int state() const { return __builtin_amdgcn_readfirstlane(__float_as_int(twice_ref[0])); }
    __device__ __forceinline__ bool far() const { return __is_same(T, bf16) && state() < 0; }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            m[t] = kNever;
            l[t] = r[t] = 0.0f;
            w[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < D / 16; ++i) acc[t][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            shift[t] = -kNever;
            twice_ref[t] = 0.0f;
        }
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

// A column's sum or maximum over the lanes that hold its keys: 4 groups of 16, and
// with PACK > 1 the lanes n of a group that are alike modulo 16 / PACK.
template <int PACK>
__device__ __forceinline__ float column_sum(float v) {
    if (PACK >= 4) v += dpp<kDppRor4>(v);
    if (PACK >= 2) v += dpp<kDppRor8>(v);
    return row_swap_sum(half_swap_sum(v));
}
template <int PACK>
__device__ __forceinline__ float column_max(float v) {
    if (PACK >= 4) v = fmaxf(v, dpp<kDppRor4>(v));
    if (PACK >= 2) v = fmaxf(v, dpp<kDppRor8>(v));
    return row_swap_max(half_swap_max(v));
}

// Lane l's value from lane l + N of its row of 16 (N 4, 8 or 12; 0 from past its end).
template <int N>
__device__ __forceinline__ uint32_t from_right(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x100 + N, 0xF, 0xF, true));
}

// The 32 keys from j0 on, whose block lies at `blk`, into the state.  Keys at `limit`
// or behind it, and keys that a column does not see, weigh nothing, whatever the cache
// holds there; `edge`: some are among these.
//
// PACK (one column tile): with at most 16 / PACK columns the matrix core's 16 hold
// each of them PACK times, all with the same scores, and each of the copies' lanes
// takes 8 / PACK of its 8 keys through the softmax instead of all: 4 heads of a group
// are then a quarter of that work (the larger part of what is not a mask or a product).
template <typename T, int D, int CT, int PACK>
__device__ __forceinline__ void attend(const char *blk, const Column<D> (&col)[CT], State<T, D, CT> &st, int j0, int limit,
                                       bool edge) {
    using R = Ring<D, true>;
    static_assert(CT == 1 || PACK == 1, "copies of one tile's columns");
    constexpr int V = 8 / PACK;  // keys of a lane: (half h, i) in order, V from V part on
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const int part = PACK == 1 ? 0 : m / (16 / PACK);
    const int k0 = V * part >= 4 ? 16 + 4 * g : V == 2 ? 4 * g + 2 * (part & 1) : 4 * g;  // its first key
    const int first = V == 2 && part >= 2 ? 16 + 4 * g + 2 * (part & 1) : k0;
    const auto key_of = [&](int e) { return PACK == 1 ? 16 * (e >> 2) + 4 * g + (e & 3) : first + e; };
    const auto pairs = [&](uint32_t(&pair)[V], int at) {
        if constexpr (V == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(blk + at + 4 * first);
            pair[0] = w[0];
            pair[1] = w[1];
        } else {
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(blk + at + 4 * (V == 4 ? first : 16 * h + 4 * g));
#pragma unroll
                for (int i = 0; i < 4; ++i) pair[4 * h + i] = w[i];
            }
        }
    };
    uint32_t k[2][R::KW], kp[V], vp[V];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t *src = reinterpret_cast<const uint32_t *>(blk + (D == 128 ? 1024 * h + 16 * lane
                                                                                 : (16 * h + m) * (D / 2) + g * (D / 8)));
        if constexpr (D == 128) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
            for (int i = 0; i < 4; ++i) k[h][i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < R::KW; ++i) k[h][i] = src[i];
        }
    }
    pairs(kp, R::P_AT);
    pairs(vp, R::P_AT + 128);
    f32x4_t raw[CT][2];
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 a = widen8(k[h][w]);
#pragma unroll
            for (int t = 0; t < CT; ++t)
                raw[t][h] = mma16(a, col[t].q[w], w == 0 ? f32x4_t{0.0f, 0.0f, 0.0f, 0.0f} : raw[t][h]);
        }
    uint32_t v[2][4][R::N128 + R::N64 + R::N32];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const char *row = blk + R::V_AT + (16 * h + 4 * i + g) * (D / 2);
#pragma unroll
            for (int n = 0; n < R::N128; ++n) v[h][i][n] = *(reinterpret_cast<const uint32_t *>(row + 64 * n) + m);
            if constexpr (R::N64 > 0)
                v[h][i][R::N128] = *(reinterpret_cast<const uint16_t *>(row + 64 * R::N128) + m);
            if constexpr (R::N32 > 0)
                v[h][i][R::N128 + R::N64] = *(reinterpret_cast<const uint8_t *>(row + 64 * R::N128 + 32 * R::N64) + m);
        }
    float s[CT][V];
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float x;
            if constexpr (PACK == 1) {
                x = raw[t][e >> 2][e & 3];
            } else if constexpr (PACK == 2) {
                x = part ? raw[t][1][e] : raw[t][0][e];
            } else {
                const float x0 = part & 1 ? raw[t][0][2 + e] : raw[t][0][e], x1 = part & 1 ? raw[t][1][2 + e] : raw[t][1][e];
                x = part & 2 ? x1 : x0;
            }
            s[t][e] = fmaf(lo<T>(kp[e]), x, hi<T>(kp[e]) * col[t].sum);
        }
    // (a branch, taken in the last blocks alone; none stands between a product and the
    // reads of it, across which the compiler has left out waits that those need)
    if (edge) {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (j0 + key_of(e) >= limit) vp[e] = 0u;
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (j0 + key_of(e) >= min(limit, col[t].vis)) s[t][e] = kNegInf;
    }
    float sv[V], av[V];
    float top = 0.0f, aside = 0.0f;  // largest scale, middle (NaN where one is)
#pragma unroll
    for (int e = 0; e < V; ++e) {
        sv[e] = lo<T>(vp[e]);
        av[e] = fmaf(kMiddle, sv[e], hi<T>(vp[e]));
        top = fmaxf(top, fabsf(sv[e]));
        aside = __builtin_elementwise_maximum(aside, fabsf(av[e]));
    }
    float mx[CT];
    const float size = __builtin_elementwise_maximum(top, aside * (1.0f / kAside));
    bool raise = false;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        raise = raise || !(size <= st.twice_ref[t]);
        mx[t] = s[t][0];
#pragma unroll
        for (int e = 1; e < V; ++e) mx[t] = fmaxf(mx[t], s[t][e]);
        mx[t] *= col[t].to_log2;
        raise = raise || !(mx[t] <= st.m[t] + kSlack);
    }
    if (__any(raise)) {
        // a value row that is no finite number: its score is none, where it is seen (so that
        // it reaches the rows that see it), and the values 0 (and no others)
        if (__builtin_expect(__any(!(aside < INFINITY)), 0)) {
            aside = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (!(fabsf(av[e]) < INFINITY)) {
#pragma unroll
                    for (int t = 0; t < CT; ++t)
                        if (s[t][e] != kNegInf) s[t][e] = NAN;
                    sv[e] = av[e] = 0.0f;
                }
                aside = fmaxf(aside, fabsf(av[e]));
            }
        }
        // scales relative to a power of two that is at least half of the largest that the
        // column sees (a larger one behind its mask would leave nothing of the others)
        const int before = st.state();
        const auto exponent = [](float most) {
            return static_cast<int>(__float_as_uint(column_max<PACK>(most)) >> 23) - 127;
        };
        int e[CT], old[CT], now[CT], down[CT], down_l[CT];
        const int all = exponent(fmaxf(top, aside * (1.0f / kAside)));
#pragma unroll
        for (int t = 0; t < CT; ++t) e[t] = all;
        if (edge) {
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < V; ++k)
                    most = s[t][k] == kNegInf ? most : fmaxf(most, fmaxf(fabsf(sv[k]), fabsf(av[k]) * (1.0f / kAside)));
                e[t] = exponent(most);
            }
        }
        bool strange = before < 0;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            old[t] = st.ref(t);
            now[t] = max(old[t], min(e[t], kMostRef));
            st.twice_ref[t] = power2(now[t] + 1);
            down[t] = down_l[t] = before == 0 ? 0 : old[t] - now[t];  // (without a sum: any)
            strange = strange || e[t] > kMostRef || down[t] < -80;
        }
        if (__builtin_expect(__any(strange), 0)) {
            bool far = before < 0;
#pragma unroll
            for (int t = 0; t < CT; ++t) far = far || e[t] > kMostRef;
            if (__is_same(T, bf16) && __any(far)) {
                const int enter = before < 0 ? 0 : kFar;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    sv[k] *= power2(-kFar);
                    av[k] *= power2(-kFar);
                }
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    now[t] = max(max(old[t] - enter, kLeastRef), min(e[t] - kFar, kFar));
                    st.twice_ref[t] = -power2(now[t] + 1);
                    down_l[t] = before == 0 ? 0 : old[t] - now[t];
                    down[t] = before == 0 ? 0 : down_l[t] - enter;
                }
            }
            // (such a power of two may be past a float's, though nothing scaled by it is: in
            // steps.  What a factor above 2^-80 and a fall of the weights make 0 is nothing)
#pragma unroll
            for (int t = 0; t < CT; ++t) {
#pragma unroll 1
                for (int step = 0; step < 4; ++step) {
                    const float f = down[t] < -80 ? 0x1p-80f : 1.0f, fl = down_l[t] < -80 ? 0x1p-80f : 1.0f;
                    down[t] += down[t] < -80 ? 80 : 0;
                    down_l[t] += down_l[t] < -80 ? 80 : 0;
                    st.l[t] *= fl;
                    st.r[t] *= f;
                    st.w[t] *= f;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) st.acc[t][i] *= f;
                }
            }
        }
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const float next = fmaxf(st.m[t], column_max<PACK>(mx[t]));
            const float fall = __builtin_amdgcn_exp2f(st.m[t] - next), f = fall * power2(down[t]);
            st.m[t] = next;
            st.shift[t] = kTop - next - static_cast<float>(now[t]);
            st.l[t] *= fall * power2(down_l[t]);
            st.r[t] *= f;
            st.w[t] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) st.acc[t][i] *= f;
        }
    }
    // the weights in fp16, in fp16 models as sums of two terms: one term's rounding,
    // next to that of such an output, is seen (2.5e-4 to 3.1e-4 against 2.1e-4, rms)
    constexpr int TERMS = __is_same(T, f16) ? 2 : 1;
    u32x4 pw[TERMS][CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        uint32_t w[TERMS][V / 2];
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float a = __builtin_amdgcn_exp2f(fmaf(s[t][e], col[t].to_log2, st.shift[t]));
            const float b = __builtin_amdgcn_exp2f(fmaf(s[t][e + 1], col[t].to_log2, st.shift[t]));
            st.l[t] += a + b;
            st.r[t] = fmaf(b, av[e + 1], fmaf(a, av[e], st.r[t]));
            const uint32_t one = Mma<f16>::pack2(a * sv[e], b * sv[e + 1]);
            w[0][e / 2] = one;
            if constexpr (TERMS == 2)
                w[1][e / 2] = Mma<f16>::pack2(fmaf(a, sv[e], -lo<f16>(one)), fmaf(b, sv[e + 1], -hi<f16>(one)));
        }
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
            // (of the copies of a column the first alone has all its weights after this)
            const uint32_t *x = w[k];
            if constexpr (PACK == 1) pw[k][t] = u32x4{x[0], x[1], x[2], x[3]};
            else if constexpr (PACK == 2) pw[k][t] = u32x4{x[0], x[1], from_right<8>(x[0]), from_right<8>(x[1])};
            else pw[k][t] = u32x4{x[0], from_right<4>(x[0]), from_right<8>(x[0]), from_right<12>(x[0])};
            constexpr uint32_t one = 0x3c003c00u;
            st.w[t] = mma16(u32x4{one, one, one, one}, pw[k][t], st.w[t]);
        }
    }
    // values: words of 8, 4 or 2 channels of a key become, per pair of keys, words
    // of one channel each
    const auto product = [&](int tile, const u32x4 &a) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int k = 0; k < TERMS; ++k) st.acc[t][tile] = mma16(a, pw[k][t], st.acc[t][tile]);
    };
    const auto four = [&](int tile, const u32x4 &x) {  // x[i]: 16 bits of two keys
        const u32x4 y = x >> 8;
        product(tile, x & 0x000f000fu);
        product(tile + 1, x & 0x00f000f0u);
        product(tile + 2, y & 0x000f000fu);
        product(tile + 3, y & 0x00f000f0u);
    };
    const auto of_two = [&](int n, uint32_t select) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_amdgcn_perm(v[i >> 1][2 * (i & 1) + 1][n], v[i >> 1][2 * (i & 1)][n], select);
        return x;
    };
#pragma unroll
    for (int n = 0; n < R::N128; ++n) {
        four(8 * n, of_two(n, 0x05040100u));
        four(8 * n + 4, of_two(n, 0x07060302u));
    }
    if constexpr (R::N64 > 0) four(8 * R::N128, of_two(R::N128, 0x05040100u));
    if constexpr (R::N32 > 0) {
        const u32x4 x = of_two(R::N128 + R::N64, 0x05040100u);
        product(8 * R::N128 + 4 * R::N64, x & 0x000f000fu);
        product(8 * R::N128 + 4 * R::N64 + 1, x & 0x00f000f0u);
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

template <int D, int CT, bool UNIFORM>
constexpr size_t split_lds() {
    constexpr size_t states = sizeof(float) * kWaves * 16 * CT * (D + 2);
    constexpr size_t rings = kWaves * Ring<D, UNIFORM>::DEPTH * Ring<D, UNIFORM>::BYTES + (UNIFORM ? 0 : kTable * 4);
    return states > rings ? states : rings;
}

// Columns of a workgroup.
template <int CT, int PACK>
constexpr int kSpan = PACK > 1 ? 16 / PACK : 16 * CT;

// Columns [c0, c0 + kSpan) of (sequence, kv head) over the keys [lo, hi): column j
// is query row j / G, head j % G of the group.  Leaves the waves' states in LDS,
// after a barrier: maximum, sum and unnormalised output of each column.
template <typename T, int D, int CT, int PACK, bool UNIFORM>
__device__ __forceinline__ void split_pass(const Params &p, float *lds, int b, int kvh, long long q_off, int L, int S,
                                           int c0, int lo, int hi) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q_start = p.causal ? max(S - L, 0) : 0;
    const int last = min(c0 + kSpan<CT, PACK>, p.G * L) - 1;
    // no column sees more than the last one
    const int limit = p.causal ? min(hi, q_start + last / p.G + 1) : hi;
    const int least = p.causal ? min(limit, q_start + c0 / p.G + 1) : limit;
    const int *table = p.bt + b * p.bt_stride;
    Column<D> col[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int nc = PACK == 1 ? 16 * t + n : n & (16 / PACK - 1);
        const int j = min(c0 + nc, last);
        const int row = j / p.G, head = j - row * p.G;
        load_column<T, D>(p, col[t], p.q + ((q_off + row) * p.H + kvh * p.G + head) * D, c0 + nc <= last);
        col[t].vis = p.causal ? q_start + row + 1 : S;
    }
    State<T, D, CT> st;
    st.clear();
    using R = Ring<D, UNIFORM>;
    constexpr int STEP = R::STEP, DEPTH = R::DEPTH;
    char *const ring = reinterpret_cast<char *>(lds) + wave * (DEPTH * R::BYTES);
    int *const copy = reinterpret_cast<int *>(reinterpret_cast<char *>(lds) + kWaves * DEPTH * R::BYTES);
    if constexpr (!UNIFORM) {
        if (lo < limit) {
            const int b0 = block_at(p, lo), used = min(block_at(p, limit - 1) - b0 + 1, kTable);
            for (int i = threadIdx.x; i < used; i += 64 * kWaves) copy[i] = table[b0 + i];
        }
        __syncthreads();
    }
    const int j0 = lo + 32 * wave;
    R asked(p, kvh, table, copy, lo, limit, j0);
    const auto load = [&](int i) {
        asked.load(j0 + i * STEP, ring + __builtin_amdgcn_readfirstlane((i % DEPTH) * R::BYTES));
        asked.turn();
    };
    const int blocks = j0 < limit ? (limit - j0 + STEP - 1) / STEP : 0;
    // (the queries are there before the first copy: no wait for them among the copies)
    __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("" ::: "memory");
    if (blocks > 0) asked.turn();
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i)
        if (i < blocks) load(i);
    for (int i = 0; i < blocks; ++i) {
        const int j = j0 + i * STEP;
        // the reads of the block before this one are done: its place is free
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + DEPTH - 1 < blocks) {
            load(i + DEPTH - 1);
            R::template wait<DEPTH - 1>();
        } else {
            // fewer blocks behind this one than the ring holds
            if (DEPTH > 3 && i + 2 < blocks) R::template wait<2>();
            else if (DEPTH > 2 && i + 1 < blocks) R::template wait<1>();
            else R::template wait<0>();
        }
        const char *blk = ring + __builtin_amdgcn_readfirstlane((i % DEPTH) * R::BYTES);
        const bool edge = j + 32 > least;
        attend<T, D, CT, PACK>(blk, col, st, j, limit, edge);
    }
    __syncthreads();  // the states take the rings' place
    constexpr int COLS = 16 * CT;
    float *lm = lds, *ll = lm + kWaves * COLS, *lout = ll + kWaves * COLS;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const float l = column_sum<PACK>(st.l[t]), r = column_sum<PACK>(st.r[t]);
        const int c = wave * COLS + 16 * t + n;
        if (n >= 16 / PACK) continue;  // a copy
        // the sum's unit 2^ref, or one that brings it to 2^-10, which the maximum takes up
        const int unit = st.far() ? near_1024th(l) : st.ref(t);
        const float value = power2(st.far() ? unit + kFar : unit);
        if (g == 0) {
            lm[c] = st.m[t] + static_cast<float>(st.ref(t) - unit);
            ll[c] = l * power2(unit);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const float code = (i & 1) ? 0x1p20f : 0x1p24f;
#pragma unroll
            for (int v = 0; v < 4; ++v)
                lout[c * D + channel_of<D>(i, 4 * g + v)] =
                    value * (fmaf(st.acc[t][i][v], code, -kMiddle * st.w[t][v]) + r);
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
    return min(max((S - 1) / p.split_len + 1, 1), p.splits);
}

// Workgroup (sequence, kv head, column tile) and split: the last split holds every
// key past the splits, and rows past the bound that the grid was made for are done
// by the workgroups of split 0, over all keys, so that the bounds shape the launch
// alone.
template <typename T, int D, int CT, int PACK, bool UNIFORM>
__global__ void __launch_bounds__(64 * kWaves, D * CT <= 64 && CT == 1 ? 4 : D * CT <= 128 ? 3 : D * CT <= 256 ? 2 : 1) split_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float states[];
    if (blockIdx.x == 0 && blockIdx.y == 0) zero_tail(p, D);
    const int tile = p.tiles - 1 - blockIdx.x % p.tiles;  // (the heaviest first)
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
    constexpr int SPAN = kSpan<CT, PACK>;
    int c0 = tile * SPAN;
    if (c0 < min(all, p.cols) && split < ns) {
        const int lo = split * p.split_len, hi = split == ns - 1 ? S : lo + p.split_len;
        const int cols = min(SPAN, min(all, p.cols) - c0);
        split_pass<T, D, CT, PACK, UNIFORM>(p, states, b, kvh, q_off, L, S, c0, lo, hi);
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
    for (long long past = static_cast<long long>(p.cols) + tile * SPAN; past < all; past += p.tiles * SPAN) {
        c0 = static_cast<int>(past);
        __syncthreads();
        split_pass<T, D, CT, PACK, UNIFORM>(p, states, b, kvh, q_off, L, S, c0, 0, S);
        merge_states<D, CT>(states, min(SPAN, all - c0), write(c0));
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

// The largest magnitude that a row of this pair can hold.
template <typename T>
__device__ __forceinline__ float magnitude(uint32_t pair) {
    return fmaxf(fabsf(hi<T>(pair)), fabsf(fmaf(15.0f, lo<T>(pair), hi<T>(pair))));
}
// fp16 holds a row to 2^-11 of this and more, which is enough for columns that see one
// such key and such a value.
constexpr float kEnough = 0x1p-14f;
// Out of what fp16 holds well, of the largest magnitude of all rows.
__device__ __forceinline__ bool outside(float most) {
    return most < INFINITY && most > 0.0f && (most > 0x1p15f || most < 0x1p-6f);
}

// Maxima over the workgroup, through `meet` [N][W].
template <int N, int W>
__device__ __forceinline__ void over_waves(float (&x)[N], float *meet) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = wave_max(x[i]);
        if (lane == 0) meet[i * W + wave] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) x[i] = fmaxf(x[i], meet[i * W + w]);
    __syncthreads();
}

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
    uint32_t kpair[PER], vpair[PER];
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
            kpair[i] = p.ks[row];
            vpair[i] = p.vs[row];
            if (!there) kpair[i] = vpair[i] = 0u;
        }
    }
    // Whether a key, and a value, of the loaded tile's first `rows` is at least kEnough.
    __device__ __forceinline__ void enough(int rows, bool &key, bool &value) const {
        key = value = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = static_cast<int>(threadIdx.x) + i * NT;
            if (t % HALF / WORDS >= rows) continue;
            key = key || magnitude<T>(kpair[i]) >= kEnough;
            value = value || magnitude<T>(vpair[i]) >= kEnough;
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
            const float vs = lo<T>(vpair[i]), va = hi<T>(vpair[i]);
            // a value row that is no finite number: its key is none (so that it reaches the
            // rows that see it) and the values 0 (so that it reaches no others)
            const bool none = !(fabsf(fmaf(kMiddle, vs, va)) < INFINITY);
            float s = is_v ? vs : lo<T>(kpair[i]), a = is_v ? va : hi<T>(kpair[i]);
            if (none) s = a = is_v ? 0.0f : NAN;
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

// Columns [c, end) of (sequence, kv head) over the keys [from, to), one key after the other
// in fp32, into the output rows or the states as by column_tile: for sequences whose rows
// have magnitudes too far apart for one power of two, where a row that a column does not
// see would leave nothing of those that it sees.
template <typename T, int D>
__device__ __forceinline__ void plain_columns(const Params &p, int b, int kvh, long long q_off, int q_start, int c, int end,
                                              int from, int to, float *part, float *part_ml) {
    constexpr int N = (D + 63) / 64, AHEAD = 4;
    const int lane = threadIdx.x & 63;
    const int *table = p.bt + b * p.bt_stride;
#pragma unroll 1
    for (; c < end; ++c) {
        const int row = c / p.G, seen = p.causal ? min(to, q_start + row + 1) : to;
        const long long at = ((q_off + row) * p.H + kvh * p.G + (c - row * p.G)) * D;
        float q[N], out[N], m = kNever, sum = 0.0f;  // out: the mean of the values so far
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = lane + 64 * i;
            q[i] = d < D ? Cvt<T>::to(p.q[at + d]) * p.scale_log2 : 0.0f;
            out[i] = 0.0f;
        }
#pragma unroll 1
        for (int j0 = from; j0 < seen; j0 += AHEAD) {
            uint32_t kp[AHEAD], vp[AHEAD];
            uint8_t k[AHEAD][N], v[AHEAD][N];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int key = min(j0 + u, seen - 1), blk = block_at(p, key);
                const long long r = row_of(p, kvh, table[blk], key, blk);
                kp[u] = p.ks[r];
                vp[u] = p.vs[r];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const long long byte = r * (D / 2) + min(lane + 64 * i, D - 1) / 2;
                    k[u][i] = p.kc[byte];
                    v[u][i] = p.vc[byte];
                }
            }
            const auto code = [&](uint8_t x) { return static_cast<float>(lane & 1 ? x >> 4 : x & 15); };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (j0 + u >= seen) break;
                float score = 0.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) score = fmaf(q[i], fmaf(lo<T>(kp[u]), code(k[u][i]), hi<T>(kp[u])), score);
                score = wave_sum(score);
                if (!(fabsf(fmaf(kMiddle, lo<T>(vp[u]), hi<T>(vp[u]))) < INFINITY)) score = NAN;  // (as in the tiles)
                const float next = fmaxf(m, score), before = sum * __builtin_amdgcn_exp2f(m - next);
                const float weight = __builtin_amdgcn_exp2f(score - next);
                m = next;
                sum = before + weight;
                const float now = weight / sum, rest = before / sum;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    out[i] = fmaf(out[i], rest, now * fmaf(lo<T>(vp[u]), code(v[u][i]), hi<T>(vp[u])));
            }
        }
        // (as a state: the mean of weights of sum 2^-10)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) continue;
            if (part != nullptr) part[static_cast<long long>(c) * D + d] = out[i] * 0x1p-10f;
            else p.o[at + d] = Cvt<T>::from(out[i]);
        }
        if (part != nullptr && lane == 0) {
            part_ml[static_cast<long long>(c) * 2] = sum == 0.0f ? kNever : m + log2f(sum) + 10.0f;
            part_ml[static_cast<long long>(c) * 2 + 1] = sum == 0.0f ? 0.0f : sum == sum ? 0x1p-10f : sum;
        }
    }
}

// Columns [c0, c0 + 32 W) below `all` of (sequence, kv head) over the keys [from, to): wave w
// serves columns 32 w .. + 31, column j being query row j / G, head j % G of the
// group, so that heads of any number fill the waves.  Into the output rows, or with
// `part` into the states [column][D], (maximum, sum) [column].  Ends with a barrier.
// Keys and values are taken times 2^-ek and 2^-ev.  LOOK: as they are, and false, with
// nothing written, where fp16 does not hold them well: rows out of its range, or all that
// some column sees down where it has few bits.
template <typename T, int D, int W, int TILE, bool LOOK>
__device__ __forceinline__ bool column_tile(const Params &p, uint16_t *lds, float *meet, int b, int kvh, long long q_off,
                                            int L, int S, int all, int c0, int from, int to, float *part,
                                            float *part_ml, int ek = 0, int ev = 0) {
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

    // the wave's queries in fp16, each with its largest element to [2^8, 2^9)
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
        const float big = half_swap_max(Cvt<T>::to(static_cast<uint16_t>(most)));
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
    if (LOOK) ek = ev = 0;
    bool enough_k = true, enough_v = true;  // among the first tile's keys that all columns see
    const int ntiles = kv_end > from ? (kv_end - from + TILE - 1) / TILE : 0;
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
        // (the first column that sees a key sees the first)
        if (LOOK) wd.enough(max(seen(c0) - from, 1), enough_k, enough_v);
        wd.store(buf(0), down_k, down_v);
    }
    const bool wave_k = __any(enough_k), wave_v = __any(enough_v);
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
    if (LOOK) {
        float of[4] = {wd.most_k, wd.most_v, wave_k ? 1.0f : 0.0f, wave_v ? 1.0f : 0.0f};
        over_waves<4, W>(of, meet);
        if (outside(of[0]) || outside(of[1]) || of[2] * of[3] == 0.0f) return false;
    }
    const float lt = half_swap_sum(lsum[0]);
    if (part != nullptr) {
        if (cw0 + r32 < all) {
            float *dst = part + static_cast<long long>(j) * D;
            // (sums of large values, of any number of keys, stay within fp32)
            const int up = ev > 40 ? near_1024th(lt) : 0;
            const float unit = power2(ev + up);
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    *reinterpret_cast<float4_t *>(dst + 32 * db + 8 * u + 4 * g) =
                        float4_t{oacc[0][db][4 * u] * unit, oacc[0][db][4 * u + 1] * unit, oacc[0][db][4 * u + 2] * unit,
                                 oacc[0][db][4 * u + 3] * unit};
            if (g == 0)
                *reinterpret_cast<float2_t *>(part_ml + static_cast<long long>(j) * 2) =
                    float2_t{m[0] - static_cast<float>(up), lt * power2(up)};
        }
        return true;  // (the loop's last barrier has passed)
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
    return true;
}

// The tiles of a workgroup once more (from the start, so that nothing is kept for it
// through them), with the powers of two that their rows ask for.  A tile whose largest row
// is more than 2^24 above all that some column sees is done without: one power of two
// would leave that column less than 11 bits.
template <typename T, int D, int W, int TILE>
__device__ __forceinline__ void careful_tiles(const Params &p, uint16_t *lds, float *meet) {
    constexpr long long COLS = 32 * W;
    const int kvh = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv, wave = threadIdx.x >> 6;
    const int split = blockIdx.y % p.splits, tile = p.tiles - 1 - blockIdx.y / p.splits;
    const int *table = p.bt + b * p.bt_stride;
    long long q_off;
    int L, S;
    sequence(p, b, q_off, L, S);
    const int all = p.G * L, q_start = p.causal ? max(S - L, 0) : 0, ns = splits_of(p, S);
    const long long at = (static_cast<long long>(b) * p.Hkv + kvh) * p.splits + split, step = COLS * p.tiles;
#pragma unroll 1
    for (long long c = tile * COLS; c < all; c += step) {
        const bool in_grid = c < p.cols, split_up = in_grid && p.splits > 1;
        if (split >= ns || (split != 0 && !in_grid)) return;
        const int c0 = static_cast<int>(c), end = in_grid ? min(all, p.cols) : all;
        const int from = split_up ? split * p.split_len : 0, to = split_up && split < ns - 1 ? from + p.split_len : S;
        float *const part = split_up ? p.ws_o + at * p.cols * D : nullptr;
        float *const part_ml = split_up ? p.ws_ml + at * p.cols * 2 : nullptr;
        const auto seen = [&](int j) { return p.causal ? min(to, q_start + j / p.G + 1) : to; };
        const int last = seen(static_cast<int>(min(c + COLS, static_cast<long long>(end))) - 1);
        const int first_end = max(seen(c0), from + 1);
        // of keys and values: the largest, the largest that all columns see, the least of the rest
        float most[2] = {0.0f, 0.0f}, own[4] = {0.0f, 0.0f, -INFINITY, -INFINITY};
        for (int key = from + static_cast<int>(threadIdx.x); key < last; key += W * 64) {
            const int blk = block_at(p, key);
            const long long r = row_of(p, kvh, table[blk], key, blk);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = magnitude<T>(i == 0 ? p.ks[r] : p.vs[r]);
                if (!(x < INFINITY)) continue;
                most[i] = fmaxf(most[i], x);
                if (key < first_end) own[i] = fmaxf(own[i], x);
                else if (x > 0.0f) own[2 + i] = fmaxf(own[2 + i], -x);
            }
        }
        over_waves<2, W>(most, meet);
        over_waves<4, W>(own, meet);
        int e[2];
        bool apart = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float least = own[i] > 0.0f ? own[i] : -own[2 + i];  // (rows of zeros are held whole)
            const bool again = outside(most[i]) || least < kEnough;
            apart = apart || (again && least < most[i] * 0x1p-24f);
            e[i] = __builtin_amdgcn_readfirstlane(
                again ? min(max(static_cast<int>(__float_as_uint(most[i]) >> 23) - 127 - 10, -110), 118) : 0);
        }
        const int cw0 = c0 + 32 * wave;
        if (apart) plain_columns<T, D>(p, b, kvh, q_off, q_start, cw0, min(cw0 + 32, end), from, to, part, part_ml);
        else column_tile<T, D, W, TILE, false>(p, lds, meet, b, kvh, q_off, L, S, end, c0, from, to, part, part_ml, e[0], e[1]);
        __syncthreads();
        if (in_grid) c = p.cols + tile * COLS - step;  // (those past the grid start at its end)
    }
}

// Workgroup (sequence, kv head) and (column tile, split), the heaviest tiles first;
// those of split 0 go on to the columns past the grid, of which there are none where
// the bound on the rows holds and the grid has room for it.
template <typename T, int D, int W, int TILE>
__global__ void __launch_bounds__(W * 64, W >= 12 ? 3 : D <= 128 && W == 4 ? 3 : 2) tile_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) uint16_t tiles_lds[];
    __shared__ float meet[4 * W];
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
    bool done = true;
    if (c0 < bound && p.splits == 1) {
        done = column_tile<T, D, W, TILE, true>(p, tiles_lds, meet, b, kvh, q_off, L, S, bound, c0, 0, S, nullptr, nullptr);
    } else if (c0 < bound) {
        const int ns = splits_of(p, S);
        const long long at = (static_cast<long long>(b) * p.Hkv + kvh) * p.splits + split;
        if (split < ns)
            done = column_tile<T, D, W, TILE, true>(p, tiles_lds, meet, b, kvh, q_off, L, S, bound, c0, split * p.split_len,
                                              split == ns - 1 ? S : (split + 1) * p.split_len, p.ws_o + at * p.cols * D,
                                              p.ws_ml + at * p.cols * 2);
    }
    if (split == 0) {
        for (long long past = p.cols + static_cast<long long>(tile) * COLS; past < all;
             past += static_cast<long long>(p.tiles) * COLS) {
            c0 = static_cast<int>(past);
            __syncthreads();
            if (!column_tile<T, D, W, TILE, true>(p, tiles_lds, meet, b, kvh, q_off, L, S, all, c0, 0, S, nullptr, nullptr))
                done = false;
        }
    }
    if (!done) careful_tiles<T, D, W, TILE>(p, tiles_lds, meet);
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

template <typename T, int D, int CT, int PACK>
tecoopsStatus_t launch_split(const Params &p, const Plan &pl, hipStream_t s) {
    const bool uniform = p.bs % 16 == 0;
    const size_t lds = uniform ? split_lds<D, CT, true>() : split_lds<D, CT, false>();
    auto *kern = uniform ? &split_kernel<T, D, CT, PACK, true> : &split_kernel<T, D, CT, PACK, false>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return TECOOPS_STATUS_INTERNAL_ERROR;
    hipLaunchKernelGGL(kern, dim3(p.batch * p.Hkv * pl.tiles, pl.splits), dim3(64 * kWaves), lds, s, p);
    TECO_CHECK_LAUNCH("flash_attention_int4");
    return launch_combine<T, D>(p, pl, s);
}

template <typename T, int D, int W, int TILE>
tecoopsStatus_t launch_tiles(const Params &p, const Plan &pl, hipStream_t s) {
    constexpr size_t lds = tile_lds<D, TILE, W>();
    static_assert(lds + 16 * W <= tecoops::kLdsMax, "fits the LDS");
    auto *kern = &tile_kernel<T, D, W, TILE>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return TECOOPS_STATUS_INTERNAL_ERROR;
    hipLaunchKernelGGL(kern, dim3(p.batch * p.Hkv, pl.tiles * pl.splits), dim3(W * 64), lds, s, p);
    TECO_CHECK_LAUNCH("flash_attention_int4");
    return launch_combine<T, D>(p, pl, s);
}

template <typename T, int D>
tecoopsStatus_t launch_size(const Params &p, const Plan &pl, hipStream_t s) {
    if (pl.split && pl.ct > 1) return launch_split<T, D, 2, 1>(p, pl, s);
    if (pl.split && pl.cols > 8) return launch_split<T, D, 1, 1>(p, pl, s);
    if (pl.split) return pl.cols > 4 ? launch_split<T, D, 1, 2>(p, pl, s) : launch_split<T, D, 1, 4>(p, pl, s);
    if constexpr (__is_same(T, f16)) return TECOOPS_STATUS_INTERNAL_ERROR;  // (make_plan's exact)
    else if (pl.waves == 4) return launch_tiles<T, D, 4, 32>(p, pl, s);
    else if constexpr (D <= 128) return launch_tiles<T, D, 12, 96>(p, pl, s);
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
    const int rows = tecoops::fa4::row_bound(max_seqlen_q, total_q, batch);
    *bytes = 0;
    for (const bool exact : {false, true})  // (of either type)
        *bytes = std::max(*bytes, tecoops::fa4::make_plan(batch, num_heads, num_kv_heads, head_size, rows, max_seqlen_k,
                                                          ~size_t{0}, tecoops::device_cus(), exact)
                                      .bytes);
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
    p.page_rows = static_cast<long long>(num_kv_heads) * block_size;
    const uint64_t inv = ((1ull << 32) + block_size - 1) / block_size;
    const uint64_t off = inv * block_size - (1ull << 32);  // exact up to 2^32 / off
    // (a block of keys past the last stays within an int)
    p.kv_cap = static_cast<int>(std::min(static_cast<long long>(blocks_per_seq) * block_size, 0x7fffffffll - 4096));
    p.inv_bs = block_size > 1 && (static_cast<uint64_t>(p.kv_cap) + 8192) * off < (1ull << 32) ? static_cast<uint32_t>(inv) : 0u;
    const float scale = softmax_scale > 0.0f ? softmax_scale : 1.0f / std::sqrt(static_cast<float>(head_size));
    p.scale_log2 = scale * 1.4426950408889634f;
    p.causal = causal != 0;
    p.total_q = total_q;
    const int rows = tecoops::fa4::row_bound(max_seqlen_q, total_q, batch);
    const int keys = std::max(max_seqlen_k > 0 ? std::min(max_seqlen_k, p.kv_cap) : p.kv_cap, 1);
    TECO_RETURN_IF(static_cast<long long>(total_q) * p.G >= (1ll << 31), TECOOPS_STATUS_NOT_SUPPORTED,
                   "flash_attention_int4: too many query rows");
    if (static_cast<long long>(batch) * num_kv_heads > tecoops::fa4::kMostWorkgroups) return TECOOPS_STATUS_NOT_SUPPORTED;
    const int cus = tecoops::device_cus();
    const auto plan = [&](size_t room) {
        return tecoops::fa4::make_plan(batch, num_heads, num_kv_heads, head_size, rows, keys, room, cus,
                                       dataType == TECOOPS_DATA_HALF);
    };
    Plan pl = plan(workspace != nullptr ? workspace_bytes : ~size_t{0});
    if (pl.bytes > 0 && workspace == nullptr) {
        workspace = tecoops::handle_scratch_if_any(handle, pl.bytes);
        if (workspace == nullptr) pl = plan(0);
    }
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
