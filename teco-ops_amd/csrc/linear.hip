// linear.hip — matrix products with their epilogue, for any number of rows.
//
//   out[m, n] = T( act( sum_k x[m, k] W[n, k] + bias[n] ) + residual[m, n] )
//   gated: W holds n gate rows, then n up rows;
//   out[m, n] = T( act(gate[m, n]) * up[m, n] + residual[m, n] )
//
// Up to 64 rows of x mostly stream W through gemv_batch.hip.  Other products run
// here, a tile of out per workgroup on v_mfma_f32_16x16x32_{f16,bf16} with W as the
// first operand, so that a lane ends with 4 neighbouring outputs of a row.  (With
// 32x32x16 the same kernel is slower: 8192 x 28672 x 4096 bf16 gated 1577 us for
// 1523, 4096^3 115 for 108.5, 333 x 4096 x 14336 60 for 55.6.)
//
// A stage is 64 of K: 128 bytes of each row of W and x of the tile, copied into
// LDS with no registers (global_load_lds_dwordx4), D stages in a ring.  The
// 16-byte chunk c of row r sits at chunk c ^ (r / 2 % 8) of its LDS row, so that
// 16 rows read at one chunk fall on distinct banks (two rows to the 256 bytes of
// all banks); the copy's source address carries the permutation.  A wave reads the
// second half of stage i while it multiplies the first, and the first half of
// stage i + 1 while it multiplies the second, the reads and copies dealt between
// its matrix instructions, so that the matrix cores wait for LDS at neither.  One
// barrier per stage, in between, says that stage i + 1 has landed and that the
// slot of stage i is free for stage i + D.
//
// Rows that are not in whole 16-byte words (odd K, views) cannot be copied that
// way: the same kernel then loads chunks to registers, zero past K, and writes
// them to the same LDS places.
//
// Few tiles leave CUs without work: K is then split over several workgroups,
// whose fp32 sums a second kernel adds in their order and finishes.
#include "linear.h"

#include "common.h"
#include "device.h"
#include "epilogue.h"
#include "gemv_batch.h"

#include <type_traits>

namespace {

using namespace tecoops::dev;
using tecoops::Epilogue;

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <typename T> struct Mma;
template <> struct Mma<f16> {
    static __device__ __forceinline__ float4_t run(u32x4_t a, u32x4_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct Mma<bf16> {
    static __device__ __forceinline__ float4_t run(u32x4_t a, u32x4_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};

// Global -> LDS with no register staging: 16 bytes per lane from base + off
// into dst + 16 * lane (dst wave-uniform, in M0).  Inline assembly, so that the
// compiler does not wait for every copy in flight before each LDS read; the
// kernel waits for all of its copies at once.
__device__ __forceinline__ void dma16(const char *base, uint32_t off, const char *dst) {
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)(dst)));
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory");
}

// LDS written by lanes of this wave is read by others of it: the wave's LDS
// operations stay in order, the compiler has to keep them so.
__device__ __forceinline__ void wave_lds_fence() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

struct TileArgs {
    const char *w, *x;
    uint16_t *out;
    float *part;        // split K: [splits, m, rows of W] fp32
    int m, n, k;        // n: outputs per row (half the rows of W when gated)
    int wrows;
    long long x_stride;  // bytes
    int tiles_m, tiles_n, splits, stages_per_split;
    int wide8;          // 8 outputs of a row in one 16-byte word
    Epilogue e;
};

// Output that row r of a tile belongs to, from the tile's first (clamped, so
// that rows past the end repeat the last).  Gated: blocks of 32 rows of the
// tile alternate between gate and up, so a wave has both sums of an output in
// the same lane.
__device__ __forceinline__ int tile_output(const TileArgs &a, int n0, int r) {
    return min(a.e.gated ? (r >> 6) * 32 + (r & 31) : r, a.n - 1 - n0);
}

// Four sums of row r of a wave's part of LDS, from its row 4 q of W on.
__device__ __forceinline__ float4_t sums4(const char *mine, int r, int q) {
    return *reinterpret_cast<const float4_t *>(mine + r * 256 + ((q ^ r) & 15) * 16);
}

// The sum of row r and its row c of W.
__device__ __forceinline__ float sum1(const char *mine, int r, int c) {
    return *reinterpret_cast<const float *>(mine + r * 256 + ((c / 4 ^ r) & 15) * 16 + c % 4 * 4);
}

// Rows of outputs n .. from 64 rows of W in a wave's part of LDS, finished and
// stored.  A lane has 8 neighbouring outputs of a row (two rows of 4 sums, and
// their up sums 32 rows of W on) and keeps them for all of its rows.
template <typename T, int ACT, bool GATED>
__device__ __forceinline__ void store_rows_as(const TileArgs &a, const char *mine, int lane, long long m,
                                              int rows, int n) {
    constexpr int PER = GATED ? 4 : 8;  // lanes of a row
    const int q = 2 * (lane % PER);
    n += 4 * q;
    if (n >= a.n) return;  // n is a multiple of 8, and so is a.n
    float b[8], bu[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        b[i] = a.e.bias != nullptr ? Cvt<T>::to(a.e.bias[n + i]) : 0.0f;
        bu[i] = GATED && a.e.bias != nullptr ? Cvt<T>::to(a.e.bias[a.n + n + i]) : 0.0f;
    }
    const auto row = [&](int r, const uint4 &res) {
        float v[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float4_t s = sums4(mine, r, q + half);
            float4_t u = s;
            if (GATED) u = sums4(mine, r, q + half + 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int o = 4 * half + i;
                v[o] = activate(s[i] + b[o], ACT);
                if (GATED) v[o] *= u[i] + bu[o];
            }
        }
        const uint32_t w[4] = {res.x, res.y, res.z, res.w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (a.e.residual != nullptr) {
                v[2 * i] += lo<T>(w[i]);
                v[2 * i + 1] += hi<T>(w[i]);
            }
            o[i] = round2<T>(v[2 * i], v[2 * i + 1]);
        }
        *reinterpret_cast<uint4 *>(a.out + (m + r) * a.e.out_stride + n) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    // several rows at once, so that their LDS reads and residuals overlap
    constexpr int STEP = 64 / PER, B = 2;
    for (int r = lane / PER; r < rows; r += STEP * B) {
        uint4 res[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (a.e.residual != nullptr && r + STEP * i < rows)
                res[i] = *reinterpret_cast<const uint4 *>(a.e.residual + (m + r + STEP * i) * a.e.res_stride + n);
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (r + STEP * i < rows) row(r + STEP * i, res[i]);
    }
}

// Rows that are not in whole 16-byte words: a lane per output, so that a store
// still covers 128 neighbouring bytes (64 when gated).  [14337, 588] times 3000
// rows took 236 us with 8 outputs to a lane stored one by one.
template <typename T>
__device__ __forceinline__ void store_rows_narrow(const TileArgs &a, const char *mine, int lane, long long m,
                                                  int rows, int n) {
    const int per = a.e.gated ? 32 : 64;
    const int c = lane & (per - 1);
    n += c;
    if (n >= a.n) return;
    const float b = a.e.bias != nullptr ? Cvt<T>::to(a.e.bias[n]) : 0.0f;
    const float bu = a.e.gated && a.e.bias != nullptr ? Cvt<T>::to(a.e.bias[a.n + n]) : 0.0f;
    const uint16_t *res = a.e.residual + m * a.e.res_stride + n;
    uint16_t *dst = a.out + m * a.e.out_stride + n;
#pragma unroll 2
    for (int r = lane / per; r < rows; r += 64 / per) {
        float v = activate(sum1(mine, r, c) + b, a.e.act);
        if (a.e.gated) v *= sum1(mine, r, c + 32) + bu;
        if (a.e.residual != nullptr) v += Cvt<T>::to(res[r * a.e.res_stride]);
        dst[r * a.e.out_stride] = static_cast<uint16_t>(round2<T>(v, v));
    }
}

template <typename T>
__device__ __forceinline__ void store_rows(const TileArgs &a, const char *mine, int lane, long long m, int rows,
                                           int n) {
    if (!a.wide8) return store_rows_narrow<T>(a, mine, lane, m, rows, n);
#define TECO_STORE(ACT)                                                        \
    case ACT:                                                                  \
        if (a.e.gated) store_rows_as<T, ACT, true>(a, mine, lane, m, rows, n); \
        else store_rows_as<T, ACT, false>(a, mine, lane, m, rows, n);          \
        break
    switch (a.e.act) {
        TECO_STORE(TECOOPS_ACTIVATION_RELU);
        TECO_STORE(TECOOPS_ACTIVATION_SILU);
        TECO_STORE(TECOOPS_ACTIVATION_GELU);
        TECO_STORE(TECOOPS_ACTIVATION_GELU_TANH);
        default: TECO_STORE(TECOOPS_ACTIVATION_NONE);
    }
#undef TECO_STORE
}

// The same for a part of K: the sums themselves, at their rows of W.
__device__ __forceinline__ void store_part(const TileArgs &a, int split, const char *mine, int lane, long long m,
                                           int rows, int n0, int r0) {
    const int q = lane & 15, r4 = r0 + 4 * q;  // 4 rows of W of the tile
    const int o = a.e.gated ? n0 + (r4 >> 6) * 32 + (r4 & 31) : n0 + r4;
    if (o >= a.n) return;
    float *p = a.part + (split * static_cast<long long>(a.m) + m) * a.wrows + (a.e.gated && (r4 & 32) ? a.n : 0) + o;
#pragma unroll 4
    for (int r = lane >> 4; r < rows; r += 4) {
        const float4_t s = sums4(mine, r, q);
        float *dst = p + static_cast<long long>(r) * a.wrows;
        if (a.n % 4 == 0) {
            *reinterpret_cast<float4_t *>(dst) = s;
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (o + t < a.n) dst[t] = s[t];
        }
    }
}

// Waits until this wave has at most N younger copies in flight (no other vector
// memory operation of its is younger than the copies it waits for) and its LDS
// reads and writes are done, then for the other waves.
template <int N>
__device__ __forceinline__ void settle() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt(((N >> 4) << 14) | 0x0070 | (N & 15));
    asm volatile("s_barrier" ::: "memory");
}

template <typename T, int BM, int BN, int WM, int WN, int D, bool COPY, bool SPLIT>
__global__ void __launch_bounds__(WM * WN * 64, 2)
linear_tile_kernel(TileArgs a) {
    constexpr int NW = WM * WN;
    constexpr int MT = BM / WM / 32, NT = BN / WN / 32;  // blocks of 32 rows of a wave
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int CW = BN / 8 / NW, CX = BM / 8 / NW;  // copies of a wave and stage
    static_assert(CW * 8 * NW == BN && CX * 8 * NW == BM, "whole copies");
    static_assert(NT % 2 == 0 && NW * MT * 32 * 256 <= D * STAGE, "the epilogue's part of LDS");
    static_assert(D >= 2, "a stage to read and one to copy to");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // Consecutive workgroups go to the 8 XCDs in turn; each XCD takes a contiguous
    // range of tiles (of parts of K and their tiles), in bands of 8 rows of tiles, so
    // that the workgroups an XCD runs at a time share rows of W and x in its L2.
    // Parts dealt to all XCDs alike read x eight times (3000 x 256 x 14336 42.5 us for
    // 40.5, 1500 x 1024 x 14336 57.7 for 55.4).
    const int tiles = a.tiles_m * a.tiles_n;
    const int all_wgs = SPLIT ? tiles * a.splits : tiles;
    const int xcd = blockIdx.x % 8;
    int id = xcd * (all_wgs / 8) + min(xcd, all_wgs % 8) + static_cast<int>(blockIdx.x / 8);
    const int split = SPLIT ? id / tiles : 0;
    if (SPLIT) id -= split * tiles;
    constexpr int kBand = 8;
    const int band = id / (kBand * a.tiles_n);
    const int in_band = id - band * kBand * a.tiles_n;
    const int band_rows = min(kBand, a.tiles_m - band * kBand);
    const int tm = band * kBand + in_band % band_rows, tn = in_band / band_rows;
    const int m0 = tm * BM;
    const int n0 = tn * (a.e.gated ? BN / 2 : BN);

    const int kbytes = a.k * 2;
    const int all = (a.k + 63) / 64;
    const int st0 = SPLIT ? split * a.stages_per_split : 0;
    const int nst = SPLIT ? min(a.stages_per_split, all - st0) : all;

    // copy c of this wave: rows 8 (wave + NW c) + lane / 8, LDS chunk lane % 8
    const int lrow = lane >> 3;
    static_assert(NW % 2 == 0, "rows 8 (wave + NW c) swap chunks alike for every c");
    const int cof = ((lane & 7) ^ ((8 * wave + lrow) >> 1 & 7)) * 16;  // byte in the stage's row
    const char *const gate = a.w + static_cast<long long>(n0) * kbytes;
    const char *const up = a.e.gated ? gate + static_cast<long long>(a.n) * kbytes : gate;
    const auto wbase = [&](int c) { return (wave + NW * c) & 4 ? up : gate; };
    const char *xbase = a.x + m0 * a.x_stride;
    uint32_t woff[CW], xoff[CX];
#pragma unroll
    for (int c = 0; c < CW; ++c)
        woff[c] = static_cast<uint32_t>(tile_output(a, n0, 8 * (wave + NW * c) + lrow)) *
                  static_cast<uint32_t>(kbytes);
#pragma unroll
    for (int c = 0; c < CX; ++c)
        xoff[c] = static_cast<uint32_t>(min(8 * (wave + NW * c) + lrow, a.m - 1 - m0)) *
                  static_cast<uint32_t>(a.x_stride);

    struct Hold {
        u32x4_t c[COPY ? 1 : CW + CX];
    };
    // The chunk at byte b of a row, zero past its kbytes: 2 bytes at a time, none
    // past the end, all loaded before the first is used.
    const auto chunk = [&](const char *row, int b) {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            h[i] = *reinterpret_cast<const uint16_t *>(row + min(b + 2 * i, kbytes - 2));
        u32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = (b + 4 * i < kbytes ? h[2 * i] : 0u) | (b + 4 * i + 2 < kbytes ? h[2 * i + 1] << 16 : 0u);
        return v;
    };
    const auto fetch = [&](Hold &hold, int i) {  // registers <- stage i
        if constexpr (!COPY) {
            const int b = (st0 + i) * 128 + cof;
            if ((st0 + i) * 128 + 128 <= kbytes) {  // the whole stage within the rows
#pragma unroll
                for (int c = 0; c < CW; ++c) __builtin_memcpy(&hold.c[c], wbase(c) + woff[c] + b, 16);
#pragma unroll
                for (int c = 0; c < CX; ++c) __builtin_memcpy(&hold.c[CW + c], xbase + xoff[c] + b, 16);
            } else if ((st0 + i) * 128 < kbytes) {  // stages past the last are never read
#pragma unroll
                for (int c = 0; c < CW; ++c) hold.c[c] = chunk(wbase(c) + woff[c], b);
#pragma unroll
                for (int c = 0; c < CX; ++c) hold.c[CW + c] = chunk(xbase + xoff[c], b);
            }
        }
    };
    // LDS <- stage i, in CW + CX pieces.  Copies past a row's end take its last
    // chunk: stages past the last are never read, and the last masks what is past
    // K.
    const auto commit = [&](const Hold &hold, int i, int slot, int c) {
        char *dst = lds + slot + (c < CW ? 0 : BN * 128) + (wave + NW * (c < CW ? c : c - CW)) * 1024;
        if constexpr (COPY) {
            const uint32_t b = min((st0 + i) * 128 + cof, kbytes - 16);
            if (c < CW) dma16(wbase(c), woff[c < CW ? c : 0] + b, dst);
            else dma16(xbase, xoff[c < CW ? 0 : c - CW] + b, dst);
        } else {
            *reinterpret_cast<u32x4_t *>(dst + lane * 16) = hold.c[c];
        }
    };

    float4_t acc[2 * NT][2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    // fragments: row lane % 16 of a 16-row block, 8 of K at 8 (lane / 16)
    const int fr = lane & 15, fg = lane >> 4;
    struct Frags {
        u32x4_t w[2 * NT], x[2 * MT];
    };
    const char *wl = lds + (wn * NT * 32 + fr) * 128;
    const char *xl = lds + BN * 128 + (wm * MT * 32 + fr) * 128;
    // Fragment number q of a half stage, in the order of their use.
    constexpr int NF = 2 * (MT + NT);
    const auto read = [&](Frags &f, int slot, int half, int q) {
        const int c = ((4 * half + fg) ^ (fr >> 1 & 7)) * 16 + slot;
        if (q < 2 * MT) f.x[q] = *reinterpret_cast<const u32x4_t *>(xl + q * 2048 + c);
        else f.w[q - 2 * MT] = *reinterpret_cast<const u32x4_t *>(wl + (q - 2 * MT) * 2048 + c);
    };
    const auto multiply = [&](const Frags &f, int p) {  // product p of 4 NT MT
        const int i = p / (2 * MT), j = p % (2 * MT);
        acc[i][j] = Mma<T>::run(f.w[i], f.x[j], acc[i][j]);
    };
    constexpr int NP = 4 * NT * MT;
    // Both operands are cleared past K: the bits there are some other chunk's,
    // which may hold inf or NaN.
    const auto mask = [&](Frags &f, int half) {
        const int left = a.k - (st0 + nst - 1) * 64;
        if (left >= 64) return;
        const int k0 = 32 * half + 8 * fg;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t keep = (k0 + 2 * e < left ? 0xffffu : 0u) | (k0 + 2 * e + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) f.w[i][e] &= keep;
#pragma unroll
            for (int j = 0; j < 2 * MT; ++j) f.x[j][e] &= keep;
        }
    };
    // The products of one half stage with the reads of the next half (and, with
    // `copies`, the copies of stage i into `to`) dealt between them in this order:
    // left to itself the compiler moves the reads to right before their use.
    const auto phase = [&](const Frags &f, Frags &next, int from, int half, auto copies, int i, int to) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            multiply(f, p);
#pragma unroll
            for (int q = p * NF / NP; q < (p + 1) * NF / NP; ++q) read(next, from, half, q);
            if constexpr (decltype(copies)::value) {
#pragma unroll
                for (int c = p * (CW + CX) / NP; c < (p + 1) * (CW + CX) / NP; ++c) commit(Hold{}, i, to, c);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Rows loaded through registers: stages 0 .. D - 2 go to LDS, D - 1 and D wait
    // in registers, all loaded at once.
    Hold hold[COPY ? 1 : D + 1];
#pragma unroll
    for (int d = 0; d < (COPY ? 0 : D + 1); ++d) fetch(hold[d], d);
#pragma unroll
    for (int d = 0; d < (COPY ? D : D - 1); ++d)
#pragma unroll
        for (int c = 0; c < CW + CX; ++c) commit(hold[COPY ? 0 : d], d, d * STAGE, c);
    settle<COPY ? (D - 1) * (CW + CX) : 63>();
    Frags f0, f1;
#pragma unroll
    for (int q = 0; q < NF; ++q) read(f0, 0, 0, q);
    int slot = 0;  // of stage i
    const auto stage = [&](int i, Hold &h) {
        const int from = slot + STAGE == D * STAGE ? 0 : slot + STAGE;
        if constexpr (!COPY) {
            // written two stages after it was loaded, to the slot of stage i - 1
            const int to = slot == 0 ? (D - 1) * STAGE : slot - STAGE;
#pragma unroll
            for (int c = 0; c < CW + CX; ++c) commit(h, i + D - 1, to, c);
            fetch(h, i + D + 1);
        }
        phase(f0, f1, slot, 1, std::false_type{}, 0, 0);
        settle<COPY ? (D - 2) * (CW + CX) : 63>();
        phase(f1, f0, from, 0, std::integral_constant<bool, COPY>{}, i + D, slot);
        slot = from;
    };
    int i = 0;
    if constexpr (!COPY) {
        for (; i + 2 < nst; i += 2) {
            stage(i, hold[D - 1]);
            stage(i + 1, hold[D]);
        }
    }
    for (; i + 1 < nst; ++i) stage(i, hold[COPY ? 0 : D - 1]);
#pragma unroll
    for (int q = 0; q < NF; ++q) read(f1, slot, 1, q);
    mask(f0, 0);
#pragma unroll
    for (int p = 0; p < NP; ++p) multiply(f0, p);
    mask(f1, 1);
#pragma unroll
    for (int p = 0; p < NP; ++p) multiply(f1, p);
    settle<0>();  // the last copies have landed, and everyone has read

    // A wave's sums pass through its own part of LDS, 64 rows of W at a time, so
    // that 8 lanes (4 when gated) end up with neighbouring outputs of one row and
    // the stores fill whole lines.  Lane l of an accumulator holds row l % 16 of its
    // 16 rows of x and 4 rows of W, from 4 (l / 16) on: a 16-byte chunk, at chunk
    // q ^ (row % 16) of the row's 256 bytes.
    char *mine = lds + wave * (MT * 32 * 256);
#pragma unroll 1
    for (int h = 0; h < NT / 2; ++h) {
#pragma unroll
        for (int hh = 0; hh < NT / 2; ++hh) {
            if (hh != h) continue;
#pragma unroll
            for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4_t *>(mine + (j * 16 + fr) * 256 + ((4 * i + fg) ^ fr) * 16) =
                        acc[4 * hh + i][j];
        }
        wave_lds_fence();
        const int r0 = (wn * NT + 2 * h) * 32;  // the tile's rows of W from here on
        const int mw = m0 + wm * MT * 32, rows = min(MT * 32, a.m - mw);
        if constexpr (SPLIT) store_part(a, split, mine, lane, mw, rows, n0, r0);
        else store_rows<T>(a, mine, lane, mw, rows, n0 + (a.e.gated ? r0 / 2 : r0));
        wave_lds_fence();
    }
}

// out from the partial sums of split K, added in the order of K.
template <typename T>
__global__ void __launch_bounds__(256) linear_finish_kernel(TileArgs a) {
    const int quads = (a.n + 3) / 4;
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long m = id / quads;
    if (m >= a.m) return;
    const int n = static_cast<int>(id - m * quads) * 4;
    float s[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
    const float *src = a.part + m * a.wrows + n;
    const long long next = static_cast<long long>(a.m) * a.wrows;
    if (a.n % 4 == 0) {
#pragma unroll 4
        for (int p = 0; p < a.splits; ++p, src += next) {
            const float4_t g = *reinterpret_cast<const float4_t *>(src);
            const float4_t h = *reinterpret_cast<const float4_t *>(src + (a.e.gated ? a.n : 0));
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                s[t] += g[t];
                u[t] += h[t];
            }
        }
    } else {
        for (int p = 0; p < a.splits; ++p, src += next)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (n + t < a.n) {
                    s[t] += src[t];
                    if (a.e.gated) u[t] += src[a.n + t];
                }
    }
    finish4<T>(a.e, a.out, m, n, a.n, s, u);
}

template <typename T, int BM, int BN, int WM, int WN, int D, bool COPY, bool SPLIT>
bool launch_tile(const TileArgs &a, hipStream_t s) {
    auto *kern = &linear_tile_kernel<T, BM, BN, WM, WN, D, COPY, SPLIT>;
    constexpr size_t lds = D * (BM + BN) * 128;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, dim3(a.tiles_m * a.tiles_n * a.splits), dim3(WM * WN * 64), lds, s, a);
    return true;
}

template <typename T, int TILE, int WM, int WN>
bool launch_as(const TileArgs &a, bool copy, hipStream_t s) {
    constexpr tecoops::LinearTile t = tecoops::kLinearTiles[TILE];
    if constexpr (TILE >= tecoops::kLinearFirstLoaded)
        if (!copy)
            return a.splits > 1 ? launch_tile<T, t.bm, t.bn, WM, WN, t.depth, false, true>(a, s)
                                : launch_tile<T, t.bm, t.bn, WM, WN, t.depth, false, false>(a, s);
    return a.splits > 1 ? launch_tile<T, t.bm, t.bn, WM, WN, t.depth, true, true>(a, s)
                        : launch_tile<T, t.bm, t.bn, WM, WN, t.depth, true, false>(a, s);
}

// The waves of each tile along its rows of x and of W.
template <typename T>
tecoopsStatus_t run_tiles(const TileArgs &a, const tecoops::LinearPlan &p, bool copy, hipStream_t s) {
    static_assert(tecoops::kLinearTileCount == 5, "a launch for every tile");
    const bool ok = p.tile == 0   ? launch_as<T, 0, 4, 2>(a, copy, s)
                    : p.tile == 1 ? launch_as<T, 1, 2, 4>(a, copy, s)
                    : p.tile == 2 ? launch_as<T, 2, 2, 2>(a, copy, s)
                    : p.tile == 3 ? launch_as<T, 3, 2, 2>(a, copy, s)
                                  : launch_as<T, 4, 2, 1>(a, copy, s);
    if (!ok) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("linear");
    if (p.splits > 1) {
        const long long quads = static_cast<long long>((a.n + 3) / 4) * a.m;
        hipLaunchKernelGGL((linear_finish_kernel<T>), dim3(tecoops::ceil_div(quads, 256)), dim3(256),
                           0, s, a);
        TECO_CHECK_LAUNCH("linear");
    }
    return TECOOPS_STATUS_SUCCESS;
}

// More workspace than this is not asked for: products that would split further
// write and read sums for longer than the split saves.
constexpr size_t kMostWorkspace = size_t{512} << 20;

}  // namespace

size_t tecoops::linear_workspace(int m, int n, int k, bool gated, bool copy) {
    return linear_plan(m, n, k, gated, copy, kMostWorkspace, device_cus()).bytes;
}

extern "C" tecoopsStatus_t tecoopsGetLinearWorkspaceSize(int m, int n, int k, int gated,
                                                         size_t *bytes) {
    if (bytes == nullptr || m < 0 || n <= 0 || k <= 0) return TECOOPS_STATUS_BAD_PARAM;
    *bytes = 0;
    if (m == 0) return TECOOPS_STATUS_SUCCESS;
    // enough wherever x and the weight lie: a view off 16 bytes or with another
    // stride is loaded through registers, by a plan of its own (8 rows of x, [4096,
    // 14336]: copied they stream W without a workspace, through registers K is split
    // 8 ways)
    *bytes = tecoops::linear_workspace(m, n, k, gated != 0, false);
    if (k % 8 == 0) {
        const size_t copied = tecoops::linear_workspace(m, n, k, gated != 0, true);
        if (copied > *bytes) *bytes = copied;
    }
    return TECOOPS_STATUS_SUCCESS;
}

extern "C" tecoopsStatus_t tecoopsLinear(tecoopsHandle_t handle, const void *x, long long x_stride,
                                         const void *weight, const void *bias, const void *residual,
                                         long long residual_stride, void *out, long long out_stride,
                                         int m, int n, int k, tecoopsActivation_t activation,
                                         int gated, void *workspace, size_t workspace_bytes,
                                         tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (x == nullptr || weight == nullptr || out == nullptr) return TECOOPS_STATUS_BAD_PARAM;
    if (m < 0 || n <= 0 || k <= 0) return TECOOPS_STATUS_BAD_PARAM;
    if (x_stride < k || out_stride < n || (residual != nullptr && residual_stride < n))
        return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::epilogue_act_ok(activation)) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    for (const void *p : {x, weight, bias, residual, const_cast<const void *>(out)})
        if (!tecoops::aligned(p, 2)) return TECOOPS_STATUS_BAD_PARAM;
    // a tile's offsets into x and W are 32-bit, and so is a grid's number of threads
    if (x_stride > tecoops::kLinearMaxRow || k > tecoops::kLinearMaxRow || n > tecoops::kLinearMaxOutputs)
        return TECOOPS_STATUS_NOT_SUPPORTED;
    if (m == 0) return TECOOPS_STATUS_SUCCESS;
    const int wrows = gated ? 2 * n : n;
    const bool copy = tecoops::linear_copies(k, x_stride, x, weight);
    Epilogue e;
    e.bias = static_cast<const uint16_t *>(bias);
    e.residual = static_cast<const uint16_t *>(residual);
    e.res_stride = residual_stride;
    e.out_stride = out_stride;
    e.act = activation;
    e.gated = gated != 0;
    e.wide = n % 4 == 0 && out_stride % 4 == 0 && tecoops::aligned(out, 8) &&
             (residual == nullptr || (residual_stride % 4 == 0 && tecoops::aligned(residual, 8)));
    if (workspace == nullptr || !tecoops::aligned(workspace, 16)) workspace_bytes = 0;
    const tecoops::LinearPlan p =
        tecoops::linear_plan(m, n, k, gated != 0, copy, workspace_bytes, tecoops::device_cus());
    if (p.stream)
        return tecoops::gemv_batch_epilogue(handle->stream, weight, x, x_stride, out, m, wrows, k,
                                            dataType, e);
    if (static_cast<long long>(p.tiles_m) * p.tiles_n * p.splits > 0x7fffff)
        return TECOOPS_STATUS_NOT_SUPPORTED;
    TileArgs a{};
    a.w = static_cast<const char *>(weight);
    a.x = static_cast<const char *>(x);
    a.out = static_cast<uint16_t *>(out);
    a.part = static_cast<float *>(workspace);
    a.m = m;
    a.n = n;
    a.k = k;
    a.wrows = wrows;
    a.x_stride = x_stride * 2;
    a.tiles_m = p.tiles_m;
    a.tiles_n = p.tiles_n;
    a.splits = p.splits;
    a.stages_per_split = p.stages;
    a.e = e;
    a.wide8 = n % 8 == 0 && out_stride % 8 == 0 && tecoops::aligned(out, 16) &&
              (residual == nullptr || (residual_stride % 8 == 0 && tecoops::aligned(residual, 16)));
    return dataType == TECOOPS_DATA_HALF ? run_tiles<f16>(a, p, copy, handle->stream)
                                         : run_tiles<bf16>(a, p, copy, handle->stream);
}
