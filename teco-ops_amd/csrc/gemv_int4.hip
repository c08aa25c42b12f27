// gemv_int4.hip — products with 4-bit weights in groups along a row.
//
//   y[b, n] = sum_k (code[n, k] - zero[n, k / g]) scale[n, k / g] x[b, k]
//           = sum over groups of scale * (sum_k code x - zero * sum_k x),
//
// codes 0..15 two to a byte (element 2j in the low half of byte j), fp32 sums and
// one rounding.  Read once each: K / 2 bytes of a row and 2 or 4 per group.
//
// gfx950 design, up to four rows of x at a time: a wave streams kRows rows of W,
// 16 bytes (32 codes) per lane and load, 1 KiB of a row together.  Codes are not
// converted: under the exponent of 1024 (fp16) or 128 (bf16) they are numbers as
// they come out of a mask, products of two are summed by v_dot2, and what the
// exponent added is taken off with the zero, from the sum of the x of the 32.  x
// is staged in LDS in the order in which masks yield the codes (0, 4, 1, 5, 2, 6,
// 3, 7), a plane for each word of the 16 bytes, so that lanes read neighbouring
// words.
#include <algorithm>

#include "common.h"
#include "device.h"
#include "epilogue.h"

namespace {

using namespace tecoops::dev;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

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
    int panel;   // elements of K staged at a time, a multiple of 32
    int narrow;  // x is not in aligned 16-byte words
};

// Eight values of x in the order of the masked codes.
__device__ __forceinline__ u32x4 interleaved(const u32x4 &v) {
    return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// Bytes of a staged panel: x, and the sums of its runs of 32.
size_t panel_bytes(int rows, int panel) { return static_cast<size_t>(rows) * (panel * 2 + panel / 32 * 4); }

// B: rows of x in this pass.
template <typename T, int B>
__global__ void __launch_bounds__(kThreads) dot_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int b0 = blockIdx.y * B, nb = min(B, a.batch - b0);
    const int n0 = (blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * kRows;
    const int groups = a.k / a.group;
    float acc[kRows][B];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int b = 0; b < B; ++b) acc[r][b] = 0.0f;
    for (int k0 = 0; k0 < a.k; k0 += a.panel) {
        const int runs = min(a.panel, a.k - k0) / 32;  // of 32 elements
        u32x4 *xs = reinterpret_cast<u32x4 *>(lds);               // [B][4][runs]
        float *sums = reinterpret_cast<float *>(xs + B * 4 * runs);  // [B][runs]
        if (k0 != 0) __syncthreads();
        for (int i = threadIdx.x; i < B * runs; i += kThreads) {
            const int b = i / runs, q = i - b * runs;
            const uint16_t *src = a.x + static_cast<long long>(b0 + min(b, nb - 1)) * a.k + k0 + 32 * q;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 v;
                if (!a.narrow) {
                    v = *reinterpret_cast<const u32x4 *>(src + 8 * j);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = src[8 * j + 2 * e] | (static_cast<uint32_t>(src[8 * j + 2 * e + 1]) << 16);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += lo<T>(v[e]) + hi<T>(v[e]);
                xs[(b * 4 + j) * runs + q] = interleaved(v);
            }
            sums[i] = sum;
        }
        __syncthreads();
        for (int q0 = lane; q0 < runs; q0 += 64 * kAhead) {
            u32x4 w[kAhead][kRows];
            float s[kAhead][kRows], z[kAhead][kRows];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int q = min(q0 + 64 * u, runs - 1);
                const int gi = (k0 + 32 * q) / a.group;
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const long long row = min(n0 + r, a.n - 1);
                    w[u][r] = __builtin_nontemporal_load(
                        reinterpret_cast<const u32x4 *>(a.w + row * (a.k / 2) + (k0 / 2 + 16 * q)));
                    s[u][r] = Cvt<T>::to(a.scales[row * groups + gi]);
                    z[u][r] = a.zeros != nullptr ? Cvt<T>::to(a.zeros[row * groups + gi]) : 8.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int q = q0 + 64 * u;
                if (q >= runs) continue;
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    u32x4 xv[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) xv[j] = xs[(b * 4 + j) * runs + q];
                    const float xsum = sums[b * runs + q];
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        float d = 0.0f;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                d = Code<T>::dot(((w[u][r][j] >> (4 * e)) & 0x000f000fu) | Code<T>::kExponent, xv[j][e], d);
                        acc[r][b] = fmaf(s[u][r], fmaf(-(Code<T>::kOffset + z[u][r]), xsum, d), acc[r][b]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const float v = wave_sum(acc[r][b]);
            if (lane == 0 && b < nb && n0 + r < a.n)
                a.y[static_cast<long long>(b0 + b) * a.n + n0 + r] = Cvt<T>::from(v);
        }
}

template <typename T, int B>
bool launch_dot(Args a, hipStream_t s) {
    a.panel = std::min(a.k, 16384 / B);
    auto *kern = &dot_kernel<T, B>;
    const size_t lds = panel_bytes(B, a.panel);
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, dim3(tecoops::ceil_div(a.n, kThreads / 64 * kRows), tecoops::ceil_div(a.batch, B)),
                       dim3(kThreads), lds, s, a);
    return true;
}

template <typename T>
bool launch(const Args &a, hipStream_t s) {
    if (a.batch == 1) return launch_dot<T, 1>(a, s);
    if (a.batch == 2) return launch_dot<T, 2>(a, s);
    return launch_dot<T, 4>(a, s);
}

}  // namespace

extern "C" tecoopsStatus_t tecoopsGemvInt4(tecoopsHandle_t handle, const void *weight, const void *scales,
                                           const void *zeros, const void *x, void *y, int batch, int n, int k,
                                           int group_size, tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (weight == nullptr || scales == nullptr || x == nullptr || y == nullptr) return TECOOPS_STATUS_BAD_PARAM;
    if (batch < 0 || n <= 0 || k <= 0 || group_size <= 0 || k % group_size != 0) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::is_16bit_float(dataType)) return TECOOPS_STATUS_BAD_PARAM;
    if (!tecoops::aligned(weight, 16) || !tecoops::aligned(scales, 2) || !tecoops::aligned(zeros, 2) ||
        !tecoops::aligned(x, 2) || !tecoops::aligned(y, 2))
        return TECOOPS_STATUS_BAD_PARAM;
    TECO_RETURN_IF(group_size % 32 != 0, TECOOPS_STATUS_NOT_SUPPORTED,
                   "gemv_int4: group_size %d not supported (multiples of 32)", group_size);
    // the grid within 32-bit thread counts
    if (n > (1 << 26) || batch > (1 << 16) || static_cast<long long>(n) * batch >= (1ll << 27)) return TECOOPS_STATUS_NOT_SUPPORTED;
    if (batch == 0) return TECOOPS_STATUS_SUCCESS;
    const Args a{static_cast<const uint8_t *>(weight), static_cast<const uint16_t *>(scales),
                 static_cast<const uint16_t *>(zeros), static_cast<const uint16_t *>(x), static_cast<uint16_t *>(y),
                 n, k, batch, group_size, 0, !tecoops::aligned(x, 16)};
    const bool ok = dataType == TECOOPS_DATA_HALF ? launch<f16>(a, handle->stream) : launch<bf16>(a, handle->stream);
    if (!ok) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("gemv_int4");
    return TECOOPS_STATUS_SUCCESS;
}
