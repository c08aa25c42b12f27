// gemv_int4.hip — products with 4-bit weights in groups along a row.
//
//   y[b, n] = sum_k (code[n, k] - zero[n, k / g]) scale[n, k / g] x[b, k]
//           = sum over groups of scale * (sum_k code x - zero * sum_k x),
//
// codes 0..15 two to a byte (element 2j in the low half of byte j), fp32 sums and
// one rounding.  Read once each: K / 2 bytes of a row and 2 or 4 per group.
//
// gfx950 design, one row of x over a short K: a wave streams kRows rows of W, 16
// bytes (32 codes) per lane and load, 1 KiB of a row together.  Codes are not
// converted: under the exponent of 1024 (fp16) or 128 (bf16) they are numbers as
// they come out of a mask, products of two are summed by v_dot2, and what the
// exponent added is taken off with the zero, from the sum of the x of the 32.  x
// is staged in LDS in the order in which masks yield the codes (0, 4, 1, 5, 2, 6,
// 3, 7), a plane for each word of the 16 bytes, so that lanes read neighbouring
// words.  [4096, 4096], groups of 128: 6.1 us, 4.2 of them the kernel: the ramp of a
// launch (8.7 MB at a large read's rate take 1.5).
//
// Several rows of x, or a long K or many rows of W: 16x16x32 matrix instructions over
// 64 rows of W and 8 to 64 of x a workgroup; 8 waves, 2 of rows and 4 of K, whose sums
// meet in LDS.  Stages of 512 of K go through registers into LDS one stage ahead, x in
// the order of the masked codes.  Scales are applied to the fp32 sums of a group (at
// most 128 of K), with the zero's share taken from the sums of x, which one more matrix
// instruction with ones yields.  [28672, 4096], 16 rows, groups of 64: 23 us, 2.9 TB/s;
// [4096, 14336], 33 rows, groups of 128: 22, 4 of them for the sum of 4 parts of K.  What
// bounds them: a workgroup's chain of a few stages (load, barrier, LDS, products) beside a
// ramp of some 5 us, and x through L2 once for every 64 rows of W.  Tried without a
// gain: stages copied straight into LDS, four in a ring (19 to 27 us and 19 to 25 over
// eight shapes of a workgroup; one row of x then 18.4 for 15.5), two stages ahead in
// registers, two buffers in LDS.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "device.h"
#include "epilogue.h"
#include "gemv_int4.h"

namespace {

using namespace tecoops::dev;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;  // (16-byte loads need no alignment)

constexpr int kThreads = 256;
constexpr int kRows = 4;   // rows of W of a wave
constexpr int kAhead = 2;  // 16-byte words of each under way

template <typename T> struct Code;
template <> struct Code<f16> {
    static constexpr uint32_t kExponent = 0x64006400u;
    static constexpr float kOffset = 1024.0f;
    static __device__ __forceinline__ float dot(uint32_t a, uint32_t b, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, a), __builtin_bit_cast(half2_t, b), c, false);
    }
};
template <> struct Code<bf16> {
    static constexpr uint32_t kExponent = 0x43004300u;
    static constexpr float kOffset = 128.0f;
    static __device__ __forceinline__ float dot(uint32_t a, uint32_t b, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf162_t, a), __builtin_bit_cast(bf162_t, b), c, false);
    }
};

struct Args {
    const uint8_t *w;
    const uint16_t *scales, *zeros, *x;
    uint16_t *y;
    int n, k, batch, group;
    int pairs;   // four outputs of a row in one 8-byte word
    int groups;  // of a row
    int slots_a_group = 0;   // uses of a group's scales
    uint32_t inv_slots = 0;  // for gemv_int4_quotient by that
    int split = 0;           // stages of a part of K
    float *parts = nullptr;  // [parts of K][batch][n] sums, null: one part
};

// Eight values of x in the order of the masked codes.
__device__ __forceinline__ u32x4 interleaved(const u32x4 &v) {
    return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// For sums that are no finite number: an infinite x, or one whose multiple by 128 + n
// passes fp32's range, makes the difference of two sums NaN where the sum of the
// products is infinite or finite.  Then elements [k0, k1) (whole runs of 32) of output
// (n, b) are summed by the whole wave, each weight on its own, but for rows of x with a
// NaN there, whose outputs are NaN.  ([28672, 4096], 16 rows of x, the same call again and
// again: 20.4 us, one row with a NaN 24, all of them 86.  Looking for such sums costs less
// than 0.2.)
template <typename T>
__device__ __forceinline__ bool holds_nan(const Args &a, int b, int k0, int k1) {
    constexpr uint32_t kInf = __is_same(T, f16) ? 0x7c00u : 0x7f80u;
    bool nan = false;
#pragma unroll 1
    for (int q = k0 / 8 + static_cast<int>(threadIdx.x & 63); q < k1 / 8; q += 64) {
        const u32x4 v = *reinterpret_cast<const u32x4_a2 *>(a.x + static_cast<long long>(b) * a.k + 8ll * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) nan = nan || (v[e] & 0x7fffu) > kInf || (v[e] >> 16 & 0x7fffu) > kInf;
    }
    return __any(nan);
}

template <typename T>
__device__ __forceinline__ float direct_sum(const Args &a, int n, int b, int k0, int k1) {
    const long long row = n;
    float sum = 0.0f;
#pragma unroll 1
    for (int q = k0 / 32 + static_cast<int>(threadIdx.x & 63); q < k1 / 32; q += 64) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(a.w + row * (a.k / 2) + 16ll * q);
        const uint16_t *x = a.x + static_cast<long long>(b) * a.k + 32ll * q;
        const long long at = row * a.groups + 32 * q / a.group;
        const float s = Cvt<T>::to(a.scales[at]), z = a.zeros != nullptr ? Cvt<T>::to(a.zeros[at]) : 8.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4 v = *reinterpret_cast<const u32x4_a2 *>(x + 8 * j);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float code = static_cast<float>((w[j] >> (4 * e)) & 15u);
                sum = fmaf((code - z) * s, e & 1 ? hi<T>(v[e >> 1]) : lo<T>(v[e >> 1]), sum);
            }
        }
    }
    return wave_sum(sum);
}

// Bytes of a staged panel: x, and the sums of its runs of 32.
constexpr size_t panel_bytes(int panel) { return static_cast<size_t>(panel) * 2 + panel / 32 * 4; }

template <typename T>
__global__ void __launch_bounds__(kThreads) dot_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int n0 = (blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * kRows;
    uint32_t exponent = Code<T>::kExponent;  // (in a vector register, as the mask is in a scalar one)
    asm("" : "+v"(exponent));
    const int runs = a.k / 32;  // of 32 elements
    u32x4 *xs = reinterpret_cast<u32x4 *>(lds);               // [4][runs]
    float *sums = reinterpret_cast<float *>(xs + 4 * runs);  // [runs]
    for (int q = threadIdx.x; q < runs; q += kThreads) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4 v = *reinterpret_cast<const u32x4_a2 *>(a.x + 32 * q + 8 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += lo<T>(v[e]) + hi<T>(v[e]);
            xs[j * runs + q] = interleaved(v);
        }
        sums[q] = sum;
    }
    __syncthreads();
    float acc[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[r] = 0.0f;
    for (int q0 = lane; q0 < runs; q0 += 64 * kAhead) {
        u32x4 w[kAhead][kRows];
        float s[kAhead][kRows], z[kAhead][kRows];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int q = min(q0 + 64 * u, runs - 1);
            const int gi = 32 * q / a.group;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const long long row = min(n0 + r, a.n - 1);
                w[u][r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(a.w + row * (a.k / 2) + 16 * q));
                s[u][r] = Cvt<T>::to(a.scales[row * a.groups + gi]);
                z[u][r] = a.zeros != nullptr ? Cvt<T>::to(a.zeros[row * a.groups + gi]) : 8.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int q = q0 + 64 * u;
            if (q >= runs) continue;
            u32x4 xv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) xv[j] = xs[j * runs + q];
            const float xsum = sums[q];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float d = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d = Code<T>::dot(((w[u][r][j] >> (4 * e)) & 0x000f000fu) | exponent, xv[j][e], d);
                acc[r] = fmaf(s[u][r], fmaf(-(Code<T>::kOffset + z[u][r]), xsum, d), acc[r]);
            }
        }
    }
    bool whole = true;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        acc[r] = wave_sum(acc[r]);
        whole = whole && (fabsf(acc[r]) < INFINITY || n0 + r >= a.n);
    }
    if (__builtin_expect(!whole, 0)) {
        const bool nan = holds_nan<T>(a, 0, 0, a.k);
#pragma unroll 1
        for (int i = 0; i < kRows && n0 + i < a.n; ++i) {
            const float sum = nan ? NAN : direct_sum<T>(a, n0 + i, 0, 0, a.k);
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (r == i && !(fabsf(acc[r]) < INFINITY)) acc[r] = sum;
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (lane == 0 && n0 + r < a.n) a.y[n0 + r] = Cvt<T>::from(acc[r]);
}

template <typename T>
bool launch_dot(const Args &a, hipStream_t s) {
    static_assert(panel_bytes(tecoops::kGemvInt4DotK) <= tecoops::kLdsDefault, "x fits in LDS");
    hipLaunchKernelGGL((dot_kernel<T>), dim3(tecoops::ceil_div(a.n, kThreads / 64 * kRows)), dim3(kThreads),
                       panel_bytes(a.k), s, a);
    return true;
}

// ------------------------------------------------------ several rows of x

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// Codes in the matrix core: as fp16 they are subnormals as they are, n 2^-24; in
// bf16, whose subnormals times x would leave fp32, under the exponent of 128.
template <typename T> struct Mma;
template <> struct Mma<f16> {
    static constexpr uint32_t kExponent = 0u;
    static constexpr float kUnit = 0x1p24f, kOffset = 0.0f;
    static __device__ __forceinline__ u32x4 ones() { return u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}; }
    static __device__ __forceinline__ float4_t run(const u32x4 &a, const u32x4 &b, const float4_t &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct Mma<bf16> {
    static constexpr uint32_t kExponent = Code<bf16>::kExponent;
    static constexpr float kUnit = 1.0f, kOffset = Code<bf16>::kOffset;
    static __device__ __forceinline__ u32x4 ones() { return u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}; }
    static __device__ __forceinline__ float4_t run(const u32x4 &a, const u32x4 &b, const float4_t &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};

// Sizes of a workgroup: RS * 16 RT rows of W, XR rows of x, stages of kStage of K;
// KS groups of waves share a stage's steps of 32.  PER: steps between two uses of
// the scales (groups of more than 128 use theirs every 128).
constexpr int kStage = tecoops::kGemvInt4Stage, kSteps = kStage / 32;

template <int XR, int RT, int RS, int KS, int PER>
struct Shape {
    static constexpr int NT = 64 * RS * KS, R = 16 * RT * RS, CT = (XR + 15) / 16;
    static constexpr int MINE = kSteps / KS, SLOTS = kSteps / PER;
    static constexpr int USE = PER < MINE ? PER : MINE;           // steps between two uses in a wave
    static constexpr int AHEAD = CT > 2 && USE > 2 ? 2 : USE;  // steps whose words are loaded together
    static constexpr int WCH = R * kSteps, XCH = XR * kStage / 8, SCH = R * SLOTS;
    static constexpr int WT = WCH / NT, XT = (XCH + NT - 1) / NT, ST = (SCH + NT - 1) / NT;
    static constexpr int X_AT = R * kStage / 2, S_AT = X_AT + XR * kStage * 2, Z_AT = S_AT + SCH * 4;
    static constexpr int STAGE = Z_AT + SCH * 4;
    static constexpr int RED = KS > 1 ? RS * KS * RT * CT * 1024 : 0;  // sums of the K groups
    static constexpr int LDS = STAGE > RED ? STAGE : RED;
    static_assert(WCH % NT == 0 && kSteps % KS == 0 && MINE % USE == 0 && PER % USE == 0, "whole steps");
    static_assert(LDS <= static_cast<int>(tecoops::kLdsMax), "a stage fits");
};

template <typename T, int XR, int RT, int RS, int KS, int PER>
__global__ void __launch_bounds__(64 * RS * KS) mma_kernel(Args a) {
    using S = Shape<XR, RT, RS, KS, PER>;
    using M = Mma<T>;
    constexpr int CT = S::CT, R = S::R, NT = S::NT;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rs = wave % RS, kp = wave / RS;
    const int n0 = blockIdx.x * R, b0 = blockIdx.z * XR, nb = min(XR, a.batch - b0);
    const int st0 = blockIdx.y * a.split, st1 = min(st0 + a.split, tecoops::gemv_int4_stages(a.k));

    // this thread's words of the first stage: of W row / step, of x row / 8
    // elements, of the scales row, and its slot
    const uint8_t *wp[S::WT];
    const uint16_t *xp[S::XT];
    long long sp[S::ST];
#pragma unroll
    for (int i = 0; i < S::WT; ++i)
        wp[i] = a.w + static_cast<long long>(min(n0 + (tid + i * NT) / kSteps, a.n - 1)) * (a.k / 2) +
                (tid + i * NT) % kSteps * 16;
#pragma unroll
    for (int i = 0; i < S::XT; ++i)
        xp[i] = a.x + static_cast<long long>(b0 + min((tid + i * NT) / (kStage / 8), nb - 1)) * a.k +
                (tid + i * NT) % (kStage / 8) * 8;
#pragma unroll
    for (int i = 0; i < S::ST; ++i)
        sp[i] = static_cast<long long>(min(n0 + (tid + i * NT) % R, a.n - 1)) * a.groups;
    u32x4 w[S::WT], x[S::XT];
    uint16_t sc[S::ST], ze[S::ST];
    const auto load = [&](int st) {
        const int k0 = st * kStage;
        const bool whole = a.k - k0 >= kStage;  // words past K: the last ones instead
#pragma unroll
        for (int i = 0; i < S::XT; ++i) {
            const uint16_t *src = xp[i] + k0;
            if (!whole) src -= tecoops::gemv_int4_past(k0 + (tid + i * NT) % (kStage / 8) * 8, 8, a.k);
            x[i] = *reinterpret_cast<const u32x4_a2 *>(src);
        }
#pragma unroll
        for (int i = 0; i < S::ST; ++i) {
            // the group that the slot's first element is in (those past K are not used)
            const int slot = st * S::SLOTS + min((tid + i * NT) / R, S::SLOTS - 1);
            const int gi = tecoops::gemv_int4_quotient(slot, a.slots_a_group, a.inv_slots);
            const long long at = sp[i] + min(gi, a.groups - 1);
            sc[i] = a.scales[at];
            if (a.zeros != nullptr) ze[i] = a.zeros[at];
        }
#pragma unroll
        for (int i = 0; i < S::WT; ++i) {
            const uint8_t *src = wp[i] + k0 / 2;
            if (!whole) src -= tecoops::gemv_int4_past(k0 / 2 + (tid + i * NT) % kSteps * 16, 16, a.k / 2);
            w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src));
        }
    };
    const auto store = [&](int st) {
        const bool tail = a.k - st * kStage < kStage;  // past K, x is 0
#pragma unroll
        for (int i = 0; i < S::XT; ++i) {
            const int t = tid + i * NT, row = t / (kStage / 8), q = t % (kStage / 8);
            if (S::XCH % NT != 0 && t >= S::XCH) continue;
            u32x4 v = x[i];
            if (row >= nb || (tail && st * kStage + 8 * q >= a.k)) v = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4 *>(lds + S::X_AT + row * kStage * 2 + (q ^ (row & 15)) * 16) = interleaved(v);
        }
        float *const ss = reinterpret_cast<float *>(lds + S::S_AT), *const zs = reinterpret_cast<float *>(lds + S::Z_AT);
#pragma unroll
        for (int i = 0; i < S::ST; ++i) {
            const int t = tid + i * NT;
            if (S::SCH % NT != 0 && t >= S::SCH) continue;
            ss[t] = Cvt<T>::to(sc[i]) * M::kUnit;
            zs[t] = a.zeros != nullptr ? (M::kOffset + Cvt<T>::to(ze[i])) * (1.0f / M::kUnit)
                                       : (M::kOffset + 8.0f) / M::kUnit;
        }
#pragma unroll
        for (int i = 0; i < S::WT; ++i) {
            const int t = tid + i * NT, row = t / kSteps;
            *reinterpret_cast<u32x4 *>(lds + row * (kStage / 2) + ((t ^ row) & (kSteps - 1)) * 16) = w[i];
        }
    };
    const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
    float4_t acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) acc[r][t] = zero;
    const int xr = XR < 16 ? c & (XR - 1) : c;  // (columns past XR repeat its rows and are not stored)
    const u32x4 ones = M::ones();
    // (in a vector register: an instruction takes one scalar, and that is the mask)
    uint32_t exponent = M::kExponent;
    asm("" : "+v"(exponent));
    if (st0 < st1) load(st0);
    for (int st = st0; st < st1; ++st) {
        __syncthreads();
        store(st);
        __syncthreads();
        if (st + 1 < st1) load(st + 1);
        const float *ss = reinterpret_cast<const float *>(lds + S::S_AT);
        const float *zs = reinterpret_cast<const float *>(lds + S::Z_AT);
#pragma unroll
        for (int u0 = 0; u0 < S::MINE; u0 += S::USE) {
            float4_t raw[RT][CT], xsum[CT];  // of codes * x, of x (the same in all rows)
#pragma unroll
            for (int p0 = 0; p0 < S::USE; p0 += S::AHEAD) {
                // the words of these steps first: a product waits for its own alone
                u32x4 b[S::AHEAD][CT];
                uint32_t v[S::AHEAD][RT];
#pragma unroll
                for (int u = 0; u < S::AHEAD; ++u) {
                    const int step = kp * S::MINE + u0 + p0 + u;
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        v[u][r] = *reinterpret_cast<const uint32_t *>(
                            lds + ((rs * RT + r) * 16 + c) * (kStage / 2) + ((step ^ c) & (kSteps - 1)) * 16 + 4 * g);
#pragma unroll
                    for (int t = 0; t < CT; ++t)
                        b[u][t] = *reinterpret_cast<const u32x4 *>(lds + S::X_AT + (16 * t + xr) * kStage * 2 +
                                                                   ((4 * step + g) ^ (xr & 15)) * 16);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < S::AHEAD; ++u) {
                    const bool first = p0 + u == 0;
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        u32x4 code;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            code[e] = (v[u][r] >> (4 * e)) & 0x000f000fu;
                            if (M::kExponent != 0u) code[e] |= exponent;
                        }
#pragma unroll
                        for (int t = 0; t < CT; ++t) raw[r][t] = M::run(code, b[u][t], first ? zero : raw[r][t]);
                    }
#pragma unroll
                    for (int t = 0; t < CT; ++t) xsum[t] = M::run(ones, b[u][t], first ? zero : xsum[t]);
                }
            }
            const int slot = (kp * S::MINE + u0) / PER;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int row = slot * R + (rs * RT + r) * 16 + 4 * g;
                const float4_t sv = *reinterpret_cast<const float4_t *>(ss + row);
                const float4_t zv = *reinterpret_cast<const float4_t *>(zs + row);
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        acc[r][t][v] = fmaf(sv[v], fmaf(-zv[v], xsum[t][v], raw[r][t][v]), acc[r][t][v]);
            }
        }
    }
    const auto put = [&](int tile, int t, float4_t s) {  // 16 rows and columns, a whole wave
        const int n = n0 + tile * 16 + 4 * g, col = 16 * t + c;
        const auto finite = [](float v) { return fabsf(v) < INFINITY; };
        const bool whole = finite(s[0]) && finite(s[1]) && finite(s[2]) && finite(s[3]);
#pragma unroll 1
        for (uint64_t left = __ballot(!whole && col < nb && n < a.n); left != 0;) {
            const int at = __builtin_ctzll(left) & 15;  // a column of these
            left &= ~(0x0001000100010001ull << at);
            const int k0 = st0 * kStage, k1 = min(static_cast<long long>(st1) * kStage, static_cast<long long>(a.k));
            const bool nan = holds_nan<T>(a, b0 + 16 * t + at, k0, k1);
#pragma unroll 1
            for (int r = 0; r < 16 && n0 + tile * 16 + r < a.n; ++r) {
                const float sum = nan ? NAN : direct_sum<T>(a, n0 + tile * 16 + r, b0 + 16 * t + at, k0, k1);
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (4 * g + v == r && c == at && !finite(s[v])) s[v] = sum;
            }
        }
        if (col >= nb || n >= a.n) return;
        const long long at = static_cast<long long>(b0 + col) * a.n + n;
        if (a.parts != nullptr) {
            float *dst = a.parts + static_cast<long long>(blockIdx.y) * a.batch * a.n + at;
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (n + v < a.n) dst[v] = s[v];
        } else if (a.pairs) {
            *reinterpret_cast<uint2 *>(a.y + at) = make_uint2(round2<T>(s[0], s[1]), round2<T>(s[2], s[3]));
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (n + v < a.n) a.y[at + v] = Cvt<T>::from(s[v]);
        }
    };
    if constexpr (KS == 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t) put(rs * RT + r, t, acc[r][t]);
    } else {
        __syncthreads();
        float4_t *red = reinterpret_cast<float4_t *>(lds);  // [KS][RS * RT][CT][64]
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < CT; ++t) red[((kp * RS * RT + rs * RT + r) * CT + t) * 64 + lane] = acc[r][t];
        __syncthreads();
        for (int q = wave; q < RS * RT * CT; q += RS * KS) {
            float4_t s = red[q * 64 + lane];
#pragma unroll
            for (int k = 1; k < KS; ++k) s += red[(k * RS * RT * CT + q) * 64 + lane];
            put(q / CT, q % CT, s);
        }
    }
}

// The sums of the parts of K, V outputs a thread.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) parts_kernel(const float *parts, uint16_t *y, long long count, int n) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const long long i = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) * V;
    if (i >= count) return;
    vec s = *reinterpret_cast<const vec *>(parts + i);
#pragma unroll 4
    for (int p = 1; p < n; ++p) s += *reinterpret_cast<const vec *>(parts + p * count + i);
#pragma unroll
    for (int v = 0; v < V; ++v) y[i + v] = Cvt<T>::from(s[v]);
}

template <typename T, int XR, int RT, int RS, int KS, int PER>
bool launch_mma(Args a, int splits, hipStream_t s) {
    using S = Shape<XR, RT, RS, KS, PER>;
    auto *kern = &mma_kernel<T, XR, RT, RS, KS, PER>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), S::LDS)) return false;
    a.slots_a_group = a.group / (32 * PER);
    const int stages = tecoops::gemv_int4_stages(a.k);
    a.inv_slots = tecoops::gemv_int4_inverse(a.slots_a_group, stages * S::SLOTS);
    a.split = (stages + splits - 1) / splits;
    splits = (stages + a.split - 1) / a.split;
    if (splits == 1) a.parts = nullptr;
    hipLaunchKernelGGL(kern, dim3(tecoops::ceil_div(a.n, S::R), splits, tecoops::ceil_div(a.batch, XR)), dim3(S::NT),
                       S::LDS, s, a);
    if (splits > 1) {
        const long long count = static_cast<long long>(a.batch) * a.n;
        const bool pairs = count % 2 == 0 && tecoops::aligned(a.parts, 8) && tecoops::aligned(a.y, 4);
        auto *sum = pairs ? &parts_kernel<T, 2> : &parts_kernel<T, 1>;
        hipLaunchKernelGGL(sum, dim3(tecoops::ceil_div(count, kThreads * (pairs ? 2 : 1))), dim3(kThreads), 0, s,
                           a.parts, a.y, count, splits);
    }
    return true;
}

template <typename T, int XR, int PER>
bool launch_rows(const Args &a, int parts, hipStream_t s) {
    return launch_mma<T, XR, 2, 2, 4, PER>(a, parts, s);
}

template <typename T, int PER>
bool launch_group(const Args &a, int parts, hipStream_t s) {
    switch (tecoops::gemv_int4_staged(a.batch)) {
        case 8: return launch_rows<T, 8, PER>(a, parts, s);
        case 16: return launch_rows<T, 16, PER>(a, parts, s);
        case 32: return launch_rows<T, 32, PER>(a, parts, s);
        case 48: return launch_rows<T, 48, PER>(a, parts, s);
        default: return launch_rows<T, 64, PER>(a, parts, s);
    }
}

template <typename T>
bool launch(const Args &a, size_t room, hipStream_t s) {
    const tecoops::GemvInt4Plan p = tecoops::gemv_int4_plan(a.batch, a.n, a.k, room, tecoops::device_cus());
    if (p.dot) return launch_dot<T>(a, s);
    if (a.group % 128 == 0) return launch_group<T, 4>(a, p.parts, s);
    return a.group % 64 == 0 ? launch_group<T, 2>(a, p.parts, s) : launch_group<T, 1>(a, p.parts, s);
}

}  // namespace

extern "C" tecoopsStatus_t tecoopsGemvInt4(tecoopsHandle_t handle, const void *weight, const void *scales,
                                           const void *zeros, const void *x, void *y, int batch, int n, int k,
                                           int group_size, void *workspace, size_t workspace_bytes,
                                           tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (weight == nullptr || scales == nullptr || x == nullptr || y == nullptr) return TECOOPS_STATUS_BAD_PARAM;
    if (batch < 0 || n <= 0 || k <= 0 || group_size <= 0 || k % group_size != 0) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::aligned(weight, 16) || !tecoops::aligned(scales, 2) || !tecoops::aligned(zeros, 2) ||
        !tecoops::aligned(x, 2) || !tecoops::aligned(y, 2) || !tecoops::aligned(workspace, 4))
        return TECOOPS_STATUS_BAD_PARAM;
    TECO_RETURN_IF(group_size % 32 != 0, TECOOPS_STATUS_NOT_SUPPORTED,
                   "gemv_int4: group_size %d not supported (multiples of 32)", group_size);
    // the grid within 32-bit thread counts
    if (n > (1 << 26) || batch > (1 << 16) || static_cast<long long>(n) * batch >= (1ll << 27)) return TECOOPS_STATUS_NOT_SUPPORTED;
    if (batch == 0) return TECOOPS_STATUS_SUCCESS;
    Args a{static_cast<const uint8_t *>(weight), static_cast<const uint16_t *>(scales),
                 static_cast<const uint16_t *>(zeros), static_cast<const uint16_t *>(x), static_cast<uint16_t *>(y),
                 n, k, batch, group_size, n % 4 == 0 && tecoops::aligned(y, 8), k / group_size};
    const size_t room = workspace != nullptr ? workspace_bytes : 0;
    a.parts = static_cast<float *>(workspace);
    const bool ok = dataType == TECOOPS_DATA_HALF ? launch<f16>(a, room, handle->stream) : launch<bf16>(a, room, handle->stream);
    if (!ok) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("gemv_int4");
    return TECOOPS_STATUS_SUCCESS;
}

extern "C" tecoopsStatus_t tecoopsGetGemvInt4WorkspaceSize(int batch, int n, int k, size_t *bytes) {
    if (bytes == nullptr || batch < 0 || n <= 0 || k <= 0) return TECOOPS_STATUS_BAD_PARAM;
    *bytes = batch == 0 ? 0 : tecoops::gemv_int4_plan(batch, n, k, ~size_t{0}, tecoops::device_cus()).bytes;
    return TECOOPS_STATUS_SUCCESS;
}
