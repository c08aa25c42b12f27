// gemv_stream.h — the sweep of W past a few staged rows of x that gemv_batch.hip
// and moe.hip are made of: a workgroup's RS * WR rows of W times up to XR rows
// of x on v_mfma_f32_16x16x32_{f16,bf16}, every W value read from memory once.
//
// W and x go from memory straight into LDS (global_load_lds_dwordx4, no
// registers) in stages of 256 bytes per row of W, D stages in a ring, and the
// MFMA operands are 16-byte LDS reads.  The 16-byte chunk c of row r sits at
// chunk c ^ (r % 16) of its LDS row, so that the 16 rows a fragment read touches
// fall on distinct banks; the copy's source address carries the permutation.
// Chunks past K are copied from a zero constant, for W and x alike, so any K in
// whole chunks works.
#pragma once

#include "common.h"
#include "device.h"

namespace tecoops {
namespace stream {

using namespace tecoops::dev;

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <typename T> struct Mma16;
template <> struct Mma16<f16> {
    static __device__ __forceinline__ f32x4_t run(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct Mma16<bf16> {
    static __device__ __forceinline__ f32x4_t run(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};

// 16 zero bytes: the source of chunks past K.
__device__ __attribute__((aligned(16))) const uint32_t kZero16[4] = {0u, 0u, 0u, 0u};

// Global -> LDS with no register staging: 16 bytes per lane into
// dst + 16 * lane (dst wave-uniform, in M0).  STREAM: read once (W), so not
// to displace x in L2.  Inline assembly, so that the compiler does not wait
// for every copy in flight before each LDS read; the copies are ordered by
// wait_copies().  No other code of these kernels uses M0 (build.py checks
// it in the assembly).
template <bool STREAM>
__device__ __forceinline__ void dma16(const void *src, void *dst) {
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)(dst)));
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "s"(lds)
                     : "memory");
    else
        asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds)
                     : "memory");
}

// Waits until this wave has at most N younger vector-memory operations in
// flight.  Every copy counts as one; any other load in flight only makes the
// wait stricter.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt(((N >> 4) << 14) | 0x0F70 | (N & 15));
    asm volatile("" ::: "memory");
}

// 16 int8 weights -> 16 fp16 values holding them exactly: bytes of w + 128
// under the exponent of 1024.0, then minus 1152.
__device__ __forceinline__ void widen_i8x16(u32x4_t q, u32x4_t &lo8, u32x4_t &hi8) {
    const half2_t bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t u = q[e] ^ 0x80808080u;
        const half2_t a = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
        const half2_t b = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
        u32x4_t &d = e < 2 ? lo8 : hi8;
        d[2 * (e & 1)] = __builtin_bit_cast(uint32_t, a);
        d[2 * (e & 1) + 1] = __builtin_bit_cast(uint32_t, b);
    }
}

// What W and x hold: both 16-bit values; int8 W, widened to fp16; or 16-bit W and
// x as sums of two 16-bit terms, hi + kLow * lo, whose row holds 8 his, then the 8
// los of the same values, and so on.
enum Operands { kPlain, kInt8, kTwoTerms };

// What the second term counts.  In fp16 it is kept 2^11 times its size, so that it
// loses no bits to the type's small exponents.
template <typename T> constexpr float kLow = __is_same(T, f16) ? 0x1p-11f : 1.0f;

// The sum of the terms' sums.  An infinite weight makes that of the second terms
// infinite or NaN whatever they are (0 or of the other sign, say): the first decides.
template <typename T>
__device__ __forceinline__ float both_terms(float high, float low) {
    return fabsf(low) < INFINITY ? fmaf(kLow<T>, low, high) : high;
}

// Sizes of a workgroup's stages.  XR: rows of x staged; WR: rows of W per wave.
template <Operands OP, int XR, int WR, int RS, int KS>
struct Shape {
    static constexpr int NW = RS * KS;
    static constexpr int CT = (XR + 15) / 16;      // column tiles of 16
    static constexpr int RT = (WR + 15) / 16;      // row tiles of 16
    static constexpr int WB = WR * 256;            // W bytes of a wave's stage
    static constexpr int WC = WR / 4;              // W copies of a wave and stage
    static constexpr int XROW = OP == kPlain ? 256 : 512;  // x bytes of a row and stage
    static constexpr int XB = XR * XROW;           // x bytes of a K part's stage
    static constexpr int SB = NW * WB + KS * XB;   // bytes of a stage
    static constexpr int XN = XB / 1024;           // x copies of a K part and stage
    static constexpr int XC = (XN + RS - 1) / RS;  // ... of a wave
    static constexpr int PER = WC + XC;            // copies of a wave and stage
    static constexpr int FIT = static_cast<int>(tecoops::kLdsMax) / SB;
    static constexpr int D = FIT > 4 ? 4 : FIT;    // stages in the ring
    static constexpr int RED = NW * RT * CT * 1024;  // partial sums (KS > 1)
    static constexpr size_t LDS = D * SB > RED ? D * SB : RED;
    static_assert(XR == 4 || XR == 8 || XR % 16 == 0, "whole column tiles, or part of one");
    static_assert(WR == 8 || WR % 16 == 0, "whole row tiles, or half of one");
    static_assert(D < 3 || (D - 2) * PER < 64, "vmcnt");
};

// One workgroup's product.  w_row(r) is the workgroup's row r of W, x_row(r) row
// r of x (any valid row where there is none: what comes of it is not kept);
// `unit` numbers the workgroups.  put(r, col, s) takes the sums s of rows r ..
// r + 3 of W and row col of x: lane l has column l % 16 of rows 4 (l / 16) ..
// + 3 of each tile of 16 x 16, and all lanes of a wave call it together.  With
// WR < 16 the lanes l / 16 >= WR / 4 hold nothing.
//
// The wave's copies of stage i + D - 1 are issued while stage i is consumed.
// With RS > 1 one barrier per stage publishes the x copies of the other waves
// and, since every wave passes it after reading stage i - 1, frees the slot
// the next copies go to.  With RS = 1 a wave reads only what it copied.
template <typename T, Operands OP, int XR, int WR, int RS, int KS, typename WRow, typename XRow,
          typename Put>
__device__ __forceinline__ void product(char *lds, int K, int unit, WRow &&w_row, XRow &&x_row,
                                        Put &&put) {
    using S = Shape<OP, XR, WR, RS, KS>;
    constexpr bool I8 = OP == kInt8, TWO = OP == kTwoTerms;
    constexpr int NW = S::NW, CT = S::CT, RT = S::RT, D = S::D, WC = S::WC, XC = S::XC, PER = S::PER;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rs = wave % RS, kp = wave / RS;
    const int g = lane >> 4, c = lane & 15;
    const int kw = I8 ? K / 16 : K / 8, kx = TWO ? K / 4 : K / 8;  // 16-byte chunks of a row of W / x
    constexpr int XCH = S::XROW / 16;                // x chunks of a row and stage
    const int nst = ((kw + 15) / 16 + KS - 1) / KS;  // stages of a K part
    // W copy m: rows 4m + lane / 16, chunk slot lane % 16
    const char *wsrc[WC];
    int wch[WC];
#pragma unroll
    for (int m = 0; m < WC; ++m) {
        const int row = 4 * m + (lane >> 4);
        wsrc[m] = w_row(rs * WR + row);
        wch[m] = kp * nst * 16 + ((lane & 15) ^ (row & 15));
    }
    // x copy q: rows (1024 / XROW) q + lane / XCH, slot lane % XCH; a K part's
    // copies are dealt to its RS waves (the last ones repeated to fill up)
    const char *xsrc[XC];
    int xch[XC], xdst[XC];
#pragma unroll
    for (int m = 0; m < XC; ++m) {
        const int q = (rs + m * RS) % S::XN;
        const int row = (1024 / S::XROW) * q + lane / XCH;
        xsrc[m] = x_row(row);
        xch[m] = kp * nst * XCH + ((lane % XCH) ^ (row & 15));
        xdst[m] = q * 1024;
    }
    f32x4_t acc[RT][CT], low[TWO ? RT : 1][TWO ? CT : 1];  // low: of the second terms
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            acc[r][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (TWO) low[r][t] = acc[r][t];
        }
    // Workgroups start their sweep of K at different stages, so that the
    // requests in flight spread over the HBM channels (rows a power of two
    // bytes apart start on the same one).  The step is odd: nst mostly is a
    // power of two, and an even step would leave most starts unused (bf16
    // batch 8, steps of 2 / 3 stages: [16384, 8192] 81.0 / 47.6 µs, [32768,
    // 4096] 44.3 / 42.8; steps of 8 / 9 at 128 rows [32768, 4096] 51.2 / 43.1).
    const int rot = (unit * (RS | 1) + (RS == 1 ? wave : 0)) % nst;
    char *wbuf = lds + wave * S::WB;
    char *xbuf = lds + NW * S::WB + kp * S::XB;
    const auto slot = [&](int i) { return __builtin_amdgcn_readfirstlane((i % D) * S::SB); };
    const auto load = [&](int i) {
        const int st = i + rot < nst ? i + rot : i + rot - nst;
        const int so = slot(i);
#pragma unroll
        for (int m = 0; m < XC; ++m) {
            const int q = xch[m] + XCH * st;
            dma16<false>(q < kx ? static_cast<const void *>(xsrc[m] + 16 * q)
                                : static_cast<const void *>(kZero16),
                         xbuf + so + xdst[m]);
        }
#pragma unroll
        for (int m = 0; m < WC; ++m) {
            const int q = wch[m] + 16 * st;
            dma16<true>(q < kw ? static_cast<const void *>(wsrc[m] + 16 * q)
                               : static_cast<const void *>(kZero16),
                        wbuf + so + m * 1024);
        }
    };
    // this lane's fragment rows: W row c of a row tile, x row c of a column
    // tile (in a tile of fewer rows the lanes past them repeat its rows, and
    // what they produce is never stored)
    const int wc = WR < 16 ? c & 7 : c, xc = XR < 16 ? c & (XR - 1) : c;
    const int wsw = wc, xsw = xc;
    const char *wl = wbuf + wc * 256, *xl = xbuf + xc * S::XROW;
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (d < nst) load(d);
    for (int i = 0; i < nst; ++i) {
        // stages i + 1 .. min(i + D - 2, nst - 1) may still be in flight
        if (D > 3 && i + 2 < nst) wait_copies<(D > 3 ? 2 : 1) * PER>();
        else if (D > 2 && i + 1 < nst) wait_copies<PER>();
        else wait_copies<0>();
        if constexpr (RS > 1) __syncthreads();
        if (i + D - 1 < nst) load(i + D - 1);
        const int so = slot(i);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            u32x4_t a[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r)
                a[r] = *reinterpret_cast<const u32x4_t *>(wl + so + r * 4096 + 16 * ((4 * u + g) ^ wsw));
            if constexpr (OP != kPlain) {
                u32x4_t b0[CT], b1[CT];
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    const char *p = xl + so + t * 16 * S::XROW;
                    b0[t] = *reinterpret_cast<const u32x4_t *>(p + 16 * ((8 * u + 2 * g) ^ xsw));
                    b1[t] = *reinterpret_cast<const u32x4_t *>(p + 16 * ((8 * u + 2 * g + 1) ^ xsw));
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    u32x4_t a0 = a[r], a1;
                    if constexpr (I8) widen_i8x16(a[r], a0, a1);
#pragma unroll
                    for (int t = 0; t < CT; ++t) {
                        acc[r][t] = Mma16<T>::run(a0, b0[t], acc[r][t]);
                        if constexpr (TWO) low[r][t] = Mma16<T>::run(a0, b1[t], low[r][t]);
                        else acc[r][t] = Mma16<T>::run(a1, b1[t], acc[r][t]);
                    }
                }
            } else {
                u32x4_t b[CT];
#pragma unroll
                for (int t = 0; t < CT; ++t)
                    b[t] = *reinterpret_cast<const u32x4_t *>(xl + so + t * 16 * S::XROW +
                                                              16 * ((4 * u + g) ^ xsw));
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < CT; ++t) acc[r][t] = Mma16<T>::run(a[r], b[t], acc[r][t]);
            }
        }
        // the reads of stage i are done before its slot is copied over
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if constexpr (TWO)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[r][t][v] = both_terms<T>(acc[r][t][v], low[r][t][v]);
    if constexpr (KS > 1) {
        __syncthreads();  // every wave is done with the ring
        float *red = reinterpret_cast<float *>(lds);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t)
                *reinterpret_cast<f32x4_t *>(red + (((wave * RT + r) * CT + t) * 64 + lane) * 4) = acc[r][t];
        __syncthreads();
        for (int q = wave; q < RS * RT * CT; q += NW) {
            const int rr = q / (RT * CT), r = q / CT % RT, t = q % CT;
            f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < KS; ++p)
                s += *reinterpret_cast<const f32x4_t *>(
                    red + ((((p * RS + rr) * RT + r) * CT + t) * 64 + lane) * 4);
            put(rr * WR + 16 * r + 4 * g, 16 * t + c, s);
        }
    } else {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t) put(rs * WR + 16 * r + 4 * g, 16 * t + c, acc[r][t]);
    }
}

}  // namespace stream
}  // namespace tecoops
