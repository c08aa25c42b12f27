// gemv_batch.hip — weight products for a batch of rows of x: one stream of W
// for up to 64 rows.
//
//   y[b, n] = T( sum_k W[n, k] x[b, k] )            fp32 accumulation
//   y[b, n] = fp16( s[n] sum_k Wq[n, k] x[b, k] )   int8 weights
//
// gfx950 design: Y^T = W X^T on v_mfma_f32_16x16x32_{f16,bf16}; a wave owns
// WR rows of W and all XR columns (rows of x), so each W value is read
// from HBM once whatever the batch.  W and x go from memory straight into LDS
// (global_load_lds_dwordx4, no registers) in stages of 256 bytes per row of
// W, D stages in a ring, and the MFMA operands are 16-byte LDS reads.  What
// bounds it is HBM for W and, for few rows per workgroup, the L2 -> LDS
// traffic of x (every workgroup copies all of x); both want whole row
// segments per copy:
//   * a copy instruction moves four 256-byte row segments (1 KiB).  Loading
//     the operands straight from memory instead touches 16 rows x 64 bytes
//     per instruction: [28672, 4096] bf16, batch 16, 60-76 µs for that over
//     12 launch shapes, 40-53 µs with W copied and x loaded, 36-40 µs with
//     both copied; batch 64 112-170 / 85-140 / 43-48 µs.
//   * RS waves of a workgroup take different rows and share the x stage; KS
//     groups of waves take different ranges of K and add their sums through
//     LDS at the end, so that few rows still fill the chip with copies in
//     flight.
#include "gemv_batch.h"

#include "common.h"
#include "epilogue.h"
#include "gemv_stream.h"

namespace {

using namespace tecoops::stream;
using tecoops::Epilogue;
using tecoops::gemv_batch_rows;

// EPI: rows of x are x_stride bytes apart and the sums end in `epi`.  Gated
// products hold 8 gate rows and the 8 up rows of the same outputs in each tile
// of 16, so that the two sums of an output meet 32 lanes apart; N is then the
// number of outputs, half the rows of W.
template <typename T, bool I8, int XR, int WR, int RS, int KS, bool EPI>
__global__ void __launch_bounds__(RS * KS * 64)
gemv_batch_kernel(const char *__restrict__ W, const uint16_t *__restrict__ scales,
                  const char *__restrict__ x, uint16_t *y, int N, int K, int B,
                  int pairs, long long x_stride, Epilogue epi) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int g = (threadIdx.x & 63) >> 4;
    const int n0 = blockIdx.x * RS * WR;
    const auto w_row = [&](int r) {
        int from = min(n0 + r, N - 1);
        if (EPI && epi.gated)
            from = min(n0 / 2 + (r >> 4) * 8 + (r & 7), N - 1) + ((r & 8) ? N : 0);
        return W + static_cast<long long>(from) * (I8 ? K / 16 : K / 8) * 16;
    };
    const auto x_row = [&](int r) { return x + min(r, B - 1) * (EPI ? x_stride : K / 8 * 16LL); };
    const auto put = [&](int r, int col, f32x4_t s) {
        int n = n0 + r;
        if constexpr (EPI) {
            f32x4_t u = s;
            if (epi.gated) {
                n = n / 16 * 8 + (n & 7);
#pragma unroll
                for (int v = 0; v < 4; ++v) u[v] = from_upper_half(s[v]);
            }
            if (col >= B || (epi.gated && g >= 2) || (WR < 16 && g >= WR / 4)) return;
            const float sv[4] = {s[0], s[1], s[2], s[3]}, uv[4] = {u[0], u[1], u[2], u[3]};
            finish4<T>(epi, y, col, n, N, sv, uv);
            return;
        }
        if (col >= B || n >= N || (WR < 16 && g >= WR / 4)) return;
        if constexpr (I8) {
#pragma unroll
            for (int v = 0; v < 4; ++v) s[v] *= h2f(scales[min(n + v, N - 1)]);
        }
        uint16_t *dst = y + static_cast<long long>(col) * N + n;
        if (pairs) {  // N % 4 == 0 and y 8-byte aligned
            *reinterpret_cast<uint2 *>(dst) = make_uint2(pack<T>(s[0], s[1]), pack<T>(s[2], s[3]));
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (n + v < N) dst[v] = Cvt<T>::from(s[v]);
        }
    };
    tecoops::stream::product<T, I8 ? kInt8 : kPlain, XR, WR, RS, KS>(lds, K, blockIdx.x, w_row, x_row, put);
}

// A product's operands; N counts the rows of W.
struct Product {
    const void *W, *scales, *x;
    void *y;
    int N, K;
    long long x_stride;  // elements
    const Epilogue *epi;  // null: the sums are stored as they are
    hipStream_t stream;
};

template <typename T, bool I8, int XR, int WR, int RS, int KS, bool EPI>
bool launch(const Product &p, int B) {
    using S = Shape<I8 ? kInt8 : kPlain, XR, WR, RS, KS>;
    static_assert(S::D >= 2, "two stages fit in LDS");
    auto *kern = &gemv_batch_kernel<T, I8, XR, WR, RS, KS, EPI>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), S::LDS)) return false;
    const int pairs = p.N % 4 == 0 && tecoops::aligned(p.y, 8);
    Epilogue e;
    if (EPI) e = *p.epi;
    hipLaunchKernelGGL(kern, dim3(tecoops::ceil_div(p.N, WR * RS)), dim3(S::NW * 64), S::LDS,
                       p.stream, static_cast<const char *>(p.W),
                       static_cast<const uint16_t *>(p.scales), static_cast<const char *>(p.x),
                       static_cast<uint16_t *>(p.y), EPI && e.gated ? p.N / 2 : p.N, p.K, B, pairs,
                       p.x_stride * 2, e);
    return true;
}

// The waves of each size (gemv_batch_rows): K split over as many groups of
// waves as leave two stages or more in LDS.  A wave's stages are a serial chain
// of copies, LDS reads and MFMAs, so that where few rows leave a CU few waves,
// more groups of shorter ranges are faster, as long as a group has enough
// stages to run through:
//   * 16 rows split K eight ways where that leaves each group 4 stages or more
//     and x is short ([4096, 14336] batch 8, four / eight ways: fp16 21.0 /
//     20.0, int8 13.1 / 12.4 µs; int8 [4096, 4096], 2 stages a group: 5.5 / 6.3);
//   * 8 rows of int8 W with short x likewise, from 2 stages a group ([256,
//     8192] batch 3, four / eight ways 7.0 / 6.0 µs, [1024, 13824] 10.7 / 8.5,
//     [2048, 4096] 5.3 / 5.1);
//   * 32 rows of int8 W with short x four ways where at most three quarters of
//     the CUs have a workgroup ([5120, 13824] two / four ways: batch 3 19.1 /
//     17.0, batch 8 20.2 / 18.1, [5120, 4096] 7.8 / 7.8, 8.1 / 7.6; two of the
//     smaller workgroups share a CU, so full grids lose: [8192, 8192] batch 4
//     14.1 / 15.9).
// 64 rows: two waves of 32 for 16-bit W (one LDS read of x serves two row
// tiles), four of 16 for int8 ([14336, 4096] batch 8: fp16 19.1 / 21.6, int8
// 13.6 / 12.3 µs).
template <typename T, bool I8, int XR, bool EPI>
bool launch_rows(const Product &p, int B) {
    const int N = p.N, K = p.K;
    // int8 stages hold twice the x: above 32 rows of x two of them fit only
    // with K split two ways, and 16 rows of W per workgroup are then no
    // faster than 32 ([4096, 14336] batch 64: 43.4 / 41.8 µs)
    constexpr bool kShortX = I8 && XR > 32;
    const int stages = (K / (I8 ? 16 : 8) + 15) / 16;
    const int cus = tecoops::device_cus();
    switch (gemv_batch_rows(N, K, B, I8, cus, EPI && p.epi->gated ? 16 : 8)) {
        case 8:
            if constexpr (I8 && XR <= 8)
                if (stages >= 16) return launch<T, I8, XR, 8, 1, 8, EPI>(p, B);
            if constexpr (!kShortX) return launch<T, I8, XR, 8, 1, 4, EPI>(p, B);
            return false;
        case 16:
            if constexpr (XR <= 8)
                if (stages >= 32) return launch<T, I8, XR, 16, 1, 8, EPI>(p, B);
            if constexpr (!kShortX) return launch<T, I8, XR, 16, 1, 4, EPI>(p, B);
            return false;
        case 32:
            if constexpr (I8 && XR <= 8)
                if (stages >= (XR <= 4 ? 32 : 16) && N <= 24 * cus)
                    return launch<T, I8, XR, 16, 2, 4, EPI>(p, B);
            return launch<T, I8, XR, 16, 2, 2, EPI>(p, B);
        case 48:
            if constexpr (XR <= 8) return launch<T, I8, XR, 16, 3, 2, EPI>(p, B);
            return false;
        case 64:
            if constexpr (I8)
                return launch<T, I8, XR, 16, 4, (kShortX ? 1 : 2), EPI>(p, B);
            else
                return launch<T, I8, XR, 32, 2, 2, EPI>(p, B);
        case 96: return launch<T, I8, XR, 16, 6, 1, EPI>(p, B);
        case 112: return launch<T, I8, XR, 16, 7, 1, EPI>(p, B);
        default: return launch<T, I8, XR, 16, 8, 1, EPI>(p, B);
    }
}

template <typename T, bool I8, bool EPI>
bool launch_batch(const Product &p, int B) {
    if (B <= 4) return launch_rows<T, I8, 4, EPI>(p, B);
    if (B <= 8) return launch_rows<T, I8, 8, EPI>(p, B);
    if (B <= 16) return launch_rows<T, I8, 16, EPI>(p, B);
    if (B <= 32) return launch_rows<T, I8, 32, EPI>(p, B);
    if (B <= 48) return launch_rows<T, I8, 48, EPI>(p, B);
    return launch_rows<T, I8, 64, EPI>(p, B);
}

}  // namespace

tecoopsStatus_t tecoops::gemv_batch(hipStream_t s, const void *W, const void *scales,
                                    const void *x, void *y, int batch, int n, int k,
                                    tecoopsDataType_t dataType, bool i8) {
    constexpr int kSlice = 64;
    for (int b0 = 0; b0 < batch; b0 += kSlice) {
        const int nb = batch - b0 < kSlice ? batch - b0 : kSlice;
        Product p{W, scales, static_cast<const uint16_t *>(x) + static_cast<long long>(b0) * k,
                  static_cast<uint16_t *>(y) + static_cast<long long>(b0) * n, n, k, k, nullptr, s};
        const bool ok = i8 ? launch_batch<f16, true, false>(p, nb)
                        : dataType == TECOOPS_DATA_HALF ? launch_batch<f16, false, false>(p, nb)
                                                        : launch_batch<bf16, false, false>(p, nb);
        if (!ok) return TECOOPS_STATUS_INTERNAL_ERROR;
        TECO_CHECK_LAUNCH("gemv");
    }
    return TECOOPS_STATUS_SUCCESS;
}

tecoopsStatus_t tecoops::gemv_batch_epilogue(hipStream_t s, const void *W, const void *x,
                                             long long x_stride, void *y, int batch, int wrows,
                                             int k, tecoopsDataType_t dataType, const Epilogue &e) {
    if (batch > 64) return TECOOPS_STATUS_INTERNAL_ERROR;
    Product p{W, nullptr, x, y, wrows, k, x_stride, &e, s};
    const bool ok = dataType == TECOOPS_DATA_HALF ? launch_batch<f16, false, true>(p, batch)
                                                  : launch_batch<bf16, false, true>(p, batch);
    if (!ok) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("linear");
    return TECOOPS_STATUS_SUCCESS;
}
