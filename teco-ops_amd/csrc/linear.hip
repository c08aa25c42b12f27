// linear.hip — matrix products with their epilogue, for any number of rows.
//
//   out[m, n] = T( act( sum_k x[m, k] W[n, k] + bias[n] ) + residual[m, n] )
//   gated: W holds n gate rows, then n up rows;
//   out[m, n] = T( act(gate[m, n]) * up[m, n] + residual[m, n] )
//
// Up to 64 rows of x stream W through gemv_batch.hip.  More rows run here, a
// tile of out per workgroup on v_mfma_f32_32x32x16_{f16,bf16} with W as the
// first operand, so that a lane ends with 4 neighbouring outputs of a row.
//
// A stage is 64 of K: 128 bytes of each row of W and x of the tile, copied
// into LDS with no registers (global_load_lds_dwordx4), two stages deep.  The
// 16-byte chunk c of row r sits at chunk c ^ (r % 8) of its LDS row, so that 8
// rows read at one chunk fall on distinct banks; the copy's source address
// carries the permutation.  A wave reads the second half of stage i while it
// multiplies the first, and the first half of stage i + 1 while it multiplies
// the second, so the matrix cores wait for LDS at neither; one barrier per
// stage, in between, says that stage i + 1 has landed and that the slot of
// stage i is free for stage i + 2.
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

namespace {

using namespace tecoops::dev;
using tecoops::Epilogue;

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <typename T> struct Mma32;
template <> struct Mma32<f16> {
    static __device__ __forceinline__ f32x16_t run(u32x4_t a, u32x4_t b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct Mma32<bf16> {
    static __device__ __forceinline__ f32x16_t run(u32x4_t a, u32x4_t b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
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
    Epilogue e;
};

// Output that row r of a tile belongs to, from the tile's first (clamped, so
// that rows past the end repeat the last).  Gated: blocks of 32 rows of the
// tile alternate between gate and up, so a wave has both sums of an output in
// the same lane.
__device__ __forceinline__ int tile_output(const TileArgs &a, int n0, int r) {
    return min(a.e.gated ? (r >> 6) * 32 + (r & 31) : r, a.n - 1 - n0);
}

template <typename T, int BM, int BN, int WM, int WN, bool COPY, bool SPLIT>
__global__ void __launch_bounds__(WM * WN * 64, 2)
linear_tile_kernel(TileArgs a) {
    constexpr int NW = WM * WN;
    constexpr int MT = BM / WM / 32, NT = BN / WN / 32;  // 32 x 32 tiles of a wave
    constexpr int STAGE = (BM + BN) * 128;
    constexpr int CW = BN / 8 / NW, CX = BM / 8 / NW;  // copies of a wave and stage
    static_assert(CW * 8 * NW == BN && CX * 8 * NW == BM, "whole copies");
    static_assert(NT % 2 == 0 && NW * MT * 32 * 256 <= 2 * STAGE, "the epilogue's part of LDS");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // Consecutive workgroups go to the 8 XCDs in turn; each XCD takes a
    // contiguous range of tiles, in bands of 8 rows of tiles, so that the
    // workgroups an XCD runs at a time share rows of W and x in its L2.
    const int tiles = a.tiles_m * a.tiles_n;
    int id = blockIdx.x;
    const int split = SPLIT ? id / tiles : 0;
    if (SPLIT) id -= split * tiles;
    {
        const int q = tiles / 8, r = tiles % 8, xcd = id % 8;
        id = xcd * q + min(xcd, r) + id / 8;
    }
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
    const int cof = ((lane & 7) ^ lrow) * 16;  // byte in the stage's row
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

    u32x4_t hold[COPY ? 1 : CW + CX];
    // chunk of a row at byte b of its kbytes (any alignment of 2), zero past K
    const auto chunk = [&](const char *row, int b) {
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (b + 16 <= kbytes) {
            __builtin_memcpy(&v, row + b, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (b + 2 * i < kbytes)
                    v[i >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(row + b + 2 * i))
                                 << (16 * (i & 1));
        }
        return v;
    };
    const auto fetch = [&](int i) {  // registers <- stage i
        if constexpr (!COPY) {
            const int b = (st0 + i) * 128 + cof;
#pragma unroll
            for (int c = 0; c < CW; ++c) hold[c] = chunk(wbase(c) + woff[c], b);
#pragma unroll
            for (int c = 0; c < CX; ++c) hold[CW + c] = chunk(xbase + xoff[c], b);
        }
    };
    // LDS <- stage i.  Copies past a row's end take its last chunk: stages past
    // the last are never read, and the last masks what is past K.
    const auto commit = [&](int i) {
        char *dst = lds + (i & 1) * STAGE;
        if constexpr (COPY) {
            const uint32_t b = min((st0 + i) * 128 + cof, kbytes - 16);
#pragma unroll
            for (int c = 0; c < CW; ++c) dma16(wbase(c), woff[c] + b, dst + (wave + NW * c) * 1024);
#pragma unroll
            for (int c = 0; c < CX; ++c)
                dma16(xbase, xoff[c] + b, dst + BN * 128 + (wave + NW * c) * 1024);
        } else {
#pragma unroll
            for (int c = 0; c < CW; ++c)
                *reinterpret_cast<u32x4_t *>(dst + (wave + NW * c) * 1024 + lane * 16) = hold[c];
#pragma unroll
            for (int c = 0; c < CX; ++c)
                *reinterpret_cast<u32x4_t *>(dst + BN * 128 + (wave + NW * c) * 1024 + lane * 16) =
                    hold[CW + c];
        }
    };

    f32x16_t acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    // fragments: row lane % 32 of a 32-row block, 8 of K at 8 (lane / 32)
    const int fr = lane & 31, fg = lane >> 5;
    struct Frags {
        u32x4_t w[2][NT], x[2][MT];
    };
    const char *wl = lds + (wn * NT * 32 + fr) * 128;
    const char *xl = lds + BN * 128 + (wm * MT * 32 + fr) * 128;
    const auto read = [&](Frags &f, int slot, int half) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int c = ((4 * half + 2 * s + fg) ^ (fr & 7)) * 16 + slot * STAGE;
#pragma unroll
            for (int i = 0; i < NT; ++i)
                f.w[s][i] = *reinterpret_cast<const u32x4_t *>(wl + i * 4096 + c);
#pragma unroll
            for (int j = 0; j < MT; ++j)
                f.x[s][j] = *reinterpret_cast<const u32x4_t *>(xl + j * 4096 + c);
        }
    };
    const auto multiply = [&](const Frags &f) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = Mma32<T>::run(f.w[s][i], f.x[s][j], acc[i][j]);
    };
    // Both operands are cleared past K: the bits there are some other chunk's,
    // which may hold inf or NaN.
    const auto mask = [&](Frags &f, int half) {
        const int left = a.k - (st0 + nst - 1) * 64;
        if (left >= 64) return;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k0 = 32 * half + 16 * s + 8 * fg;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t keep = (k0 + 2 * e < left ? 0xffffu : 0u) |
                                      (k0 + 2 * e + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
                for (int i = 0; i < NT; ++i) f.w[s][i][e] &= keep;
#pragma unroll
                for (int j = 0; j < MT; ++j) f.x[s][j][e] &= keep;
            }
        }
    };
    // this wave's copies have landed and its LDS reads and writes are done
    const auto settle = [&] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
    };

    fetch(0);
    commit(0);
    settle();
    Frags f0, f1;
    read(f0, 0, 0);
    fetch(1);
    commit(1);
    for (int i = 0; i + 1 < nst; ++i) {
        fetch(i + 2);
        read(f1, i & 1, 1);
        multiply(f0);
        settle();
        commit(i + 2);
        read(f0, (i + 1) & 1, 0);
        multiply(f1);
    }
    read(f1, (nst - 1) & 1, 1);
    mask(f0, 0);
    multiply(f0);
    mask(f1, 1);
    multiply(f1);
    settle();  // the last copies land in LDS before the workgroup's end

    // A wave's sums pass through its own part of LDS, 64 rows of W at a time, so
    // that 16 lanes (8 when gated) end up with neighbouring outputs of one row
    // and the stores fill whole lines.  Lane l of an accumulator holds row
    // l % 32 of x and 4 rows of W, from 8 v + 4 (l / 32) on: a 16-byte chunk,
    // at chunk q ^ (row % 16) of the row's 256 bytes.
    char *mine = lds + wave * (MT * 32 * 256);
    const int per = a.e.gated ? 8 : 16;  // lanes per row
#pragma unroll
    for (int h = 0; h < NT / 2; ++h) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const f32x16_t &t = acc[2 * h + i][j];
                    *reinterpret_cast<float4_t *>(mine + (j * 32 + fr) * 256 +
                                                  ((8 * i + 2 * v + fg) ^ (fr & 15)) * 16) =
                        float4_t{t[4 * v], t[4 * v + 1], t[4 * v + 2], t[4 * v + 3]};
                }
        wave_lds_fence();
        const int q = lane & (per - 1);
        const int r0 = (wn * NT + 2 * h) * 32;  // the tile's rows of W from here on
        const int n = n0 + (a.e.gated ? r0 / 2 : r0) + 4 * q;
#pragma unroll 1
        for (int r = lane / per; r < MT * 32; r += 64 / per) {
            const long long m = m0 + wm * MT * 32 + r;
            if (m >= a.m) break;
            const float4_t s = *reinterpret_cast<const float4_t *>(mine + r * 256 + (q ^ (r & 15)) * 16);
            const float4_t u = *reinterpret_cast<const float4_t *>(mine + r * 256 + (((q + 8) & 15) ^ (r & 15)) * 16);
            const float sv[4] = {s[0], s[1], s[2], s[3]}, uv[4] = {u[0], u[1], u[2], u[3]};
            if constexpr (SPLIT) {
                float *p = a.part + (static_cast<long long>(split) * a.m + m) * a.wrows + n;
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (n + t < a.n) {
                        p[t] = sv[t];
                        if (a.e.gated) p[a.n + t] = uv[t];
                    }
            } else {
                finish4<T>(a.e, a.out, m, n, a.n, sv, uv);
            }
        }
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
    for (int p = 0; p < a.splits; ++p) {
        const float *src = a.part + (static_cast<long long>(p) * a.m + m) * a.wrows + n;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (n + t >= a.n) break;
            s[t] += src[t];
            if (a.e.gated) u[t] += src[a.n + t];
        }
    }
    finish4<T>(a.e, a.out, m, n, a.n, s, u);
}

template <typename T, int BM, int BN, int WM, int WN, bool COPY, bool SPLIT>
bool launch_tile(const TileArgs &a, hipStream_t s) {
    auto *kern = &linear_tile_kernel<T, BM, BN, WM, WN, COPY, SPLIT>;
    constexpr size_t lds = 2 * (BM + BN) * 128;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, dim3(a.tiles_m * a.tiles_n * a.splits), dim3(WM * WN * 64), lds, s, a);
    return true;
}

template <typename T>
tecoopsStatus_t run_tiles(TileArgs a, const tecoops::LinearPlan &p, bool copy, hipStream_t s) {
    bool ok;
    if (p.bm == 256)
        ok = launch_tile<T, 256, 256, 4, 2, true, false>(a, s);
    else if (copy)
        ok = p.splits > 1 ? launch_tile<T, 128, 128, 2, 2, true, true>(a, s)
                          : launch_tile<T, 128, 128, 2, 2, true, false>(a, s);
    else
        ok = p.splits > 1 ? launch_tile<T, 128, 128, 2, 2, false, true>(a, s)
                          : launch_tile<T, 128, 128, 2, 2, false, false>(a, s);
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

}  // namespace

extern "C" tecoopsStatus_t tecoopsGetLinearWorkspaceSize(int m, int n, int k, int gated,
                                                         size_t *bytes) {
    if (bytes == nullptr || m < 0 || n <= 0 || k <= 0) return TECOOPS_STATUS_BAD_PARAM;
    *bytes = 0;
    if (m == 0) return TECOOPS_STATUS_SUCCESS;
    const bool copy = k % 8 == 0;
    if (copy && m <= tecoops::kLinearStreamRows) return TECOOPS_STATUS_SUCCESS;
    *bytes = tecoops::linear_plan(m, n, k, gated != 0, copy, ~size_t{0}, tecoops::device_cus()).bytes;
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
    // a tile's offsets into x and W and the rows of W are 32-bit
    if (x_stride > tecoops::kLinearMaxRow || k > tecoops::kLinearMaxRow || n > (1 << 30))
        return TECOOPS_STATUS_NOT_SUPPORTED;
    if (m == 0) return TECOOPS_STATUS_SUCCESS;
    const int wrows = gated ? 2 * n : n;
    const bool copy = k % 8 == 0 && x_stride % 8 == 0 && tecoops::aligned(weight, 16) &&
                      tecoops::aligned(x, 16);
    Epilogue e;
    e.bias = static_cast<const uint16_t *>(bias);
    e.residual = static_cast<const uint16_t *>(residual);
    e.res_stride = residual_stride;
    e.out_stride = out_stride;
    e.act = activation;
    e.gated = gated != 0;
    e.wide = n % 4 == 0 && out_stride % 4 == 0 && tecoops::aligned(out, 8) &&
             (residual == nullptr || (residual_stride % 4 == 0 && tecoops::aligned(residual, 8)));
    if (copy && m <= tecoops::kLinearStreamRows)
        return tecoops::gemv_batch_epilogue(handle->stream, weight, x, x_stride, out, m, wrows, k,
                                            dataType, e);
    if (workspace == nullptr || !tecoops::aligned(workspace, 4)) workspace_bytes = 0;
    const tecoops::LinearPlan p =
        tecoops::linear_plan(m, n, k, gated != 0, copy, workspace_bytes, tecoops::device_cus());
    if (static_cast<long long>(p.tiles_m) * p.tiles_n * p.splits > 0x7fffffffll)
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
    return dataType == TECOOPS_DATA_HALF ? run_tiles<f16>(a, p, copy, handle->stream)
                                         : run_tiles<bf16>(a, p, copy, handle->stream);
}
