// moe.hip — a mixture-of-experts layer for a few tokens (a decode batch).
//
//   p = softmax(router_logits[t]);  e_0 .. e_{k-1}: the top k experts
//   w_j = p[e_j]  (/ sum_j p[e_j] when renormalised)
//   h_j = act(x W_in[e_j][:I]^T) * (x W_in[e_j][I:]^T)
//   out[t] = T( sum_j w_j (h_j W_out[e_j]^T) )
//
// What bounds it is reading the chosen experts' weights, 3 H I values each.
// Tokens are therefore grouped by expert: a weight is read from HBM once for an item
// of up to XR tokens of its expert (gemv_stream.h), not once per token.  XR comes of
// an even spread of the tokens, and the whole of W is swept again for the items past
// an expert's first: 512 tokens, 1 of 128 experts of [2048, 768], 204 us spread at
// random (188 to read the weights), 54 all at one expert; 512 tokens, 2 of 8 of [4096,
// 14336], 1305 us where one pass of the weights would take 447.
//   route    softmax, top k and the groups: per expert a list of its (token, j)
//            pairs, cut into items of up to XR pairs
//   in       per item and block of rows of W_in: h of its pairs
//   out      per item and block of rows of W_out: w_j (h_j W_out^T) in fp32
//   combine  the k parts of each token, added in the order of j
// h is a matrix operand of the second product, where one 16-bit value in its place
// would cost as much as the result's own rounding (rms against 64 bits 0.0023 in
// bf16 and 0.0003 in fp16, for 0.0016 and 0.0002).  It is therefore the sum of two
// (`two_terms`), which the product takes in turn: 4 bytes a value instead of 2, and
// twice the matrix instructions, of which the stream of W leaves enough (256 tokens, 8
// of 128 experts of [4096, 1024] bf16: 559 us with one value, 574 with two; 1 token, 2
// of 8 of [4096, 14336] 111 either way).
// No sum depends on the order in which workgroups run: a pair's place in its
// group decides only which column of an MFMA it is.
#include "moe.h"

#include "common.h"
#include "epilogue.h"
#include "gemv_stream.h"

namespace {

using namespace tecoops::stream;
using tecoops::MoeSpace;

struct MoeArgs {
    const char *x, *w_in, *w_out;
    const void *logits;
    uint16_t *out;
    int *topk_ids;         // or null
    float *topk_weights;   // or null
    long long x_stride;    // bytes
    int tokens, hidden, inter, experts, top_k;
    int logits16, renorm, act;
    int rows;              // of x per item
    int units;             // blocks of rows of W per item
    // workspace
    int *n_items;
    int4 *items;           // expert, first pair, pairs
    int *ids;              // [tokens, top_k], -1: none
    int *token, *slot;     // of a pair in the experts' order: its row of x, t * top_k + j
    float *weight;
    uint16_t *h;           // [pairs, h_stride] in two terms; fp32 for the scalar kernels
    long long h_stride;    // values
    float *part;           // [tokens, top_k, hidden]
    // few tokens: of item i and token t, the pair or -1 and its weight
    int *col_pair;         // [items, kMoeFew]
    float *col_weight;
};

// ------------------------------------------------------------------- routing

// Softmax and top k of token t by one wave, R logits per lane (of expert 64 r +
// lane).  The best logit left is a maximum over the wave, its expert the lowest
// one that holds it; -inf and NaN are never chosen, so a token may have fewer
// than k.  Lane j ends with choice j: its expert or -1, and its weight.
template <typename T, int R>
__device__ __forceinline__ void choose(const MoeArgs &a, int t, int lane, int &id, float &weight) {
    float v[R];
    float local = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int e = 64 * r + lane;
        v[r] = -INFINITY;
        if (e < a.experts) {
            const long long at = static_cast<long long>(t) * a.experts + e;
            v[r] = a.logits16 ? Cvt<T>::to(static_cast<const uint16_t *>(a.logits)[at])
                              : static_cast<const float *>(a.logits)[at];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (!(v[r] > -INFINITY)) v[r] = -INFINITY;  // NaN
        v[r] += 0.0f;                               // -0 ties with 0
        local = fmaxf(local, v[r]);
    }
    const float top = wave_max(local);
    float sum = 0.0f, mine = 0.0f;  // mine: exp(logit - top) of choice `lane`
    id = -1;
    if (!a.renorm) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float p = v[r] == top ? 1.0f : expf(v[r] - top);
            sum += v[r] > -INFINITY ? p : 0.0f;
        }
        sum = wave_sum(sum);
    }
    for (int j = 0; j < a.top_k; ++j) {
        float best = v[R - 1];
        int e = 64 * (R - 1) + lane;
#pragma unroll
        for (int r = R - 2; r >= 0; --r)
            if (v[r] >= best) {
                best = v[r];
                e = 64 * r + lane;
            }
        const float m = j == 0 ? top : wave_max(best);
        if (!(m > -INFINITY)) break;
        const int won = static_cast<int>(-wave_max(best == m ? -static_cast<float>(e) : -INFINITY));
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (won == 64 * r + lane) v[r] = -INFINITY;
        if (lane == j) {
            id = won;
            mine = m;
        }
    }
    mine = id < 0 ? 0.0f : mine == top ? 1.0f : expf(mine - top);
    if (a.renorm) sum = wave_sum(mine);
    weight = id < 0 ? 0.0f : mine / sum;
}

__device__ __forceinline__ void store_choice(const MoeArgs &a, int p, int id, float weight) {
    a.ids[p] = id;
    if (a.topk_ids != nullptr) a.topk_ids[p] = id;
    if (a.topk_weights != nullptr) a.topk_weights[p] = weight;
}

// Groups the pairs by expert and cuts the groups into items, by a workgroup of
// 1024: pair(p, e, w) gives pair p's expert and weight.  A pair's place in its
// group follows the order of the atomics; it decides which column of an MFMA
// the pair is, and no result depends on it.
template <typename Pair>
__device__ __forceinline__ void group(const MoeArgs &a, Pair &&pair) {
    __shared__ int count[tecoops::kMoeMaxExperts], first[tecoops::kMoeMaxExperts];
    __shared__ int wave_pairs[16], wave_items[16];
    const int me = threadIdx.x, lane = me & 63, wave = me >> 6;
    const int pairs = a.tokens * a.top_k;
    count[me] = 0;
    __syncthreads();
    for (int p = me; p < pairs; p += 1024) {
        int e;
        float w;
        pair(p, e, w);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    // first pair and first item of expert `me`: prefix sums over the experts
    const int c = count[me];
    const int items = (c + a.rows - 1) / a.rows;
    int sc = c, si = items;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int oc = __shfl_up(sc, d), oi = __shfl_up(si, d);
        if (lane >= d) {
            sc += oc;
            si += oi;
        }
    }
    if (lane == 63) {
        wave_pairs[wave] = sc;
        wave_items[wave] = si;
    }
    __syncthreads();
    int bc = 0, bi = 0, total = 0;
    for (int w = 0; w < 16; ++w) {
        if (w < wave) {
            bc += wave_pairs[w];
            bi += wave_items[w];
        }
        total += wave_items[w];
    }
    bc += sc - c;
    bi += si - items;
    for (int i = 0; i < items; ++i)
        a.items[bi + i] = make_int4(me, bc + i * a.rows, min(a.rows, c - i * a.rows), 0);
    if (me == 0) *a.n_items = total;
    first[me] = bc;
    count[me] = 0;
    __syncthreads();
    for (int p = me; p < pairs; p += 1024) {
        int e;
        float w;
        pair(p, e, w);
        if (e < 0) continue;
        const int at = first[e] + atomicAdd(&count[e], 1);
        a.token[at] = p / a.top_k;
        a.slot[at] = p;
        a.weight[at] = w;
    }
}

// Few tokens: groups without atomics, in one workgroup of their own or in every
// workgroup of the first product, whose first one then also writes what the later
// kernels read.  An expert is one item, as no token has it twice: pair p's place is
// the number of pairs before it in the order of experts, then of pairs, counted
// over all of them.
constexpr int kFewPairs = tecoops::kMoeFew * tecoops::kMoeMaxTopK;

struct FewItem {
    int items, expert, first, count;
    int token[tecoops::kMoeFew];  // of its pairs
};

// Fills `out` (shared) for `item`; `lds` is scratch, free again at the return.
template <typename T, int R>
__device__ __forceinline__ void route_few(const MoeArgs &a, char *lds, int item, FewItem *out) {
    int *const id = reinterpret_cast<int *>(lds), *const fresh = id + kFewPairs;
    float *const weight = reinterpret_cast<float *>(fresh + kFewPairs);
    const int me = threadIdx.x, lane = me & 63;
    const bool store = blockIdx.x == 0;
    for (int t = me >> 6; t < a.tokens; t += blockDim.x >> 6) {
        int e;
        float w;
        choose<T, R>(a, t, lane, e, w);
        if (lane < a.top_k) {
            const int p = t * a.top_k + lane;
            id[p] = e;
            weight[p] = w;
            if (store) store_choice(a, p, e, w);
        }
    }
    __syncthreads();
    const int pairs = a.tokens * a.top_k;  // at most blockDim.x
    const int e = me < pairs ? id[me] : -1;
    int before = 0, same = 0, count = 0;
#pragma unroll 8
    for (int q = 0; q < pairs; ++q) {
        const int o = id[q];
        before += o >= 0 && o < e;
        same += o == e && q < me;
        count += o == e;
    }
    if (me < pairs) fresh[me] = e >= 0 && same == 0 ? e : -1;
    __syncthreads();
    int mine = 0, total = 0;  // experts below e, and all
#pragma unroll 8
    for (int q = 0; q < pairs; ++q) {
        const int o = fresh[q];
        mine += o >= 0 && o < e;
        total += o >= 0;
    }
    if (me == 0) out->items = total;
    if (e >= 0 && mine == item) {
        out->token[same] = me / a.top_k;
        if (same == 0) {
            out->expert = e;
            out->first = before;
            out->count = count;
        }
    }
    if (store) {
        if (me == 0) *a.n_items = total;
        for (int i = me; i < total * tecoops::kMoeFew; i += blockDim.x) a.col_pair[i] = -1;
        __syncthreads();
        if (e >= 0) {
            const int at = before + same, token = me / a.top_k;
            a.token[at] = token;
            a.slot[at] = me;
            a.weight[at] = weight[me];
            if (same == 0) a.items[mine] = make_int4(e, before, count, 0);
            a.col_pair[mine * tecoops::kMoeFew + token] = at;
            a.col_weight[mine * tecoops::kMoeFew + token] = weight[me];
        }
    }
    __syncthreads();
}

template <typename T, int R>
__global__ void __launch_bounds__(tecoops::kMoeFew * 64) moe_route_kernel(MoeArgs a) {
    __shared__ int scratch[3 * kFewPairs];
    __shared__ FewItem none;
    route_few<T, R>(a, reinterpret_cast<char *>(scratch), -1, &none);
}

// More tokens: a wave each over the chip, then one workgroup for the groups.
template <typename T, int R>
__global__ void __launch_bounds__(256) moe_choose_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.tokens) return;
    int e;
    float w;
    choose<T, R>(a, t, lane, e, w);
    if (lane < a.top_k) {
        const int p = t * a.top_k + lane;
        store_choice(a, p, e, w);
        a.part[p] = w;  // free until the second product
    }
}

__global__ void __launch_bounds__(1024) moe_group_kernel(MoeArgs a) {
    group(a, [&](int p, int &e, float &w) {
        e = a.ids[p];
        w = a.part[p];
    });
}

// Whether there is a table of the tokens' pairs: few tokens, rows in whole words.
bool few_tokens(const MoeArgs &a, bool copy) { return copy && a.tokens <= tecoops::kMoeFew && a.rows <= 8; }

template <typename T>
void launch_route(const MoeArgs &a, bool copy, hipStream_t s) {
    if (few_tokens(a, copy)) {
        if (a.experts <= 128)
            hipLaunchKernelGGL((moe_route_kernel<T, 2>), dim3(1), dim3(tecoops::kMoeFew * 64), 0, s, a);
        else
            hipLaunchKernelGGL((moe_route_kernel<T, tecoops::kMoeMaxExperts / 64>), dim3(1),
                               dim3(tecoops::kMoeFew * 64), 0, s, a);
        return;
    }
    const dim3 grid(tecoops::ceil_div(a.tokens, 4));
    if (a.experts <= 64) hipLaunchKernelGGL((moe_choose_kernel<T, 1>), grid, dim3(256), 0, s, a);
    else if (a.experts <= 128) hipLaunchKernelGGL((moe_choose_kernel<T, 2>), grid, dim3(256), 0, s, a);
    else if (a.experts <= 256) hipLaunchKernelGGL((moe_choose_kernel<T, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((moe_choose_kernel<T, tecoops::kMoeMaxExperts / 64>), grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL(moe_group_kernel, dim3(1), dim3(1024), 0, s, a);
}

// ------------------------------------------------------------------ products

// h = kUnit (hi + kLow lo), with 16 bits of it in bf16 and 22 in fp16.  kUnit moves
// fp16's range to 65520 * 256 (beyond, hi is infinite and lo is 0) and its smallest
// step, that of lo, to 2^-27.
template <typename T> constexpr float kUnit = __is_same(T, f16) ? 256.0f : 1.0f;

template <typename T>
__device__ __forceinline__ void two_terms(float v0, float v1, uint32_t &hi2, uint32_t &lo2) {
    v0 *= 1.0f / kUnit<T>;
    v1 *= 1.0f / kUnit<T>;
    hi2 = round2<T>(v0, v1);
    const float h0 = lo<T>(hi2), h1 = hi<T>(hi2);
    lo2 = round2<T>(fabsf(h0) < INFINITY ? (v0 - h0) * (1.0f / kLow<T>) : 0.0f,
                    fabsf(h1) < INFINITY ? (v1 - h1) * (1.0f / kLow<T>) : 0.0f);
}

// IN: rows of W_in, 8 gate rows and the 8 up rows of the same outputs in each
// tile of 16; OUT: rows of W_out.
// R > 0: few tokens, routed here (R logits per lane).
template <typename T, int XR, int WR, int RS, int KS, bool OUT, int R>
__global__ void __launch_bounds__(RS * KS * 64) moe_product_kernel(MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ FewItem few;
    const int item = blockIdx.x / a.units, unit = blockIdx.x - item * a.units;
    if constexpr (R > 0) {
        static_assert(RS * KS * 64 >= kFewPairs, "a thread per pair");
        route_few<T, R>(a, lds, item, &few);
    }
    if (item >= (R > 0 ? few.items : *a.n_items)) return;
    const int4 it = R > 0 ? make_int4(few.expert, few.first, few.count, 0) : a.items[item];
    const int expert = __builtin_amdgcn_readfirstlane(it.x), first = __builtin_amdgcn_readfirstlane(it.y);
    const int count = __builtin_amdgcn_readfirstlane(it.z);
    const int g = (threadIdx.x & 63) >> 4;
    const int K = OUT ? a.inter : a.hidden, N = OUT ? a.hidden : a.inter;
    const char *w = (OUT ? a.w_out : a.w_in) +
                    static_cast<long long>(expert) * (OUT ? 2 : 4) * a.hidden * a.inter;
    const int n0 = unit * RS * WR / (OUT ? 1 : 2);
    const auto w_row = [&](int r) {
        const int from = OUT ? min(n0 + r, N - 1)
                             : min(n0 + (r >> 4) * 8 + (r & 7), N - 1) + ((r & 8) ? N : 0);
        return w + static_cast<long long>(from) * K * 2;
    };
    const auto x_row = [&](int r) {
        const int i = min(r, count - 1);
        return OUT ? reinterpret_cast<const char *>(a.h) + (first + i) * a.h_stride * 4
                   : a.x + (R > 0 ? few.token[i] : a.token[first + i]) * a.x_stride;
    };
    const auto put = [&](int r, int col, f32x4_t s) {
        if constexpr (OUT) {
            const int n = n0 + r;
            if (col >= count || n >= N) return;  // N % 8 == 0: four at a time
            const float wt = kUnit<T> * a.weight[first + col];
            *reinterpret_cast<f32x4_t *>(a.part + static_cast<long long>(a.slot[first + col]) * N + n) =
                f32x4_t{wt * s[0], wt * s[1], wt * s[2], wt * s[3]};
        } else {
            f32x4_t u;
#pragma unroll
            for (int v = 0; v < 4; ++v) u[v] = from_upper_half(s[v]);
            const int n = n0 + (r >> 4) * 8 + (r & 7);
            if (col >= count || g >= 2 || n >= N) return;
            uint2 high, low;
            two_terms<T>(activate(s[0], a.act) * u[0], activate(s[1], a.act) * u[1], high.x, low.x);
            two_terms<T>(activate(s[2], a.act) * u[2], activate(s[3], a.act) * u[3], high.y, low.y);
            uint16_t *dst = a.h + (first + col) * a.h_stride * 2 + n / 8 * 16 + n % 8;
            *reinterpret_cast<uint2 *>(dst) = high;
            *reinterpret_cast<uint2 *>(dst + 8) = low;
        }
    };
    product<T, OUT ? kTwoTerms : kPlain, XR, WR, RS, KS>(lds, K, unit, w_row, x_row, put);
}

// Few tokens: the second product with the sum over the experts in it, straight to
// out.  A workgroup has WR rows of every expert's W_out; its KS waves share the
// items' stages of K out evenly, one item after the other, in a ring of D stages
// each.  The columns are the tokens; at the end of an item (or of a wave's share
// of it) a column adds its sums with its routing weight, or nothing where the
// token has not chosen the expert, whatever was multiplied there.
template <typename T, int XR, int WR, int KS, int D>
__global__ void __launch_bounds__(KS * 64) moe_out_few_kernel(MoeArgs a) {
    constexpr int RT = (WR + 15) / 16, WC = WR / 4, XC = XR / 2, PER = WC + XC;
    constexpr int SB = WR * 256 + XR * 512;
    static_assert(RT == 1 && D <= 4 && D >= 3 && (D - 2) * PER < 64, "one row tile, vmcnt");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int expert[kFewPairs];
    __shared__ uint16_t col_pair[kFewPairs * XR];
    __shared__ float col_weight[kFewPairs * XR];  // -1: the token has not chosen the expert
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * WR;
    const int items = *a.n_items;
    for (int i = threadIdx.x; i < items; i += KS * 64) expert[i] = a.items[i].x;
    for (int i = threadIdx.x; i < items * XR; i += KS * 64) {
        const int at = i / XR * tecoops::kMoeFew + i % XR;
        const int p = a.col_pair[at];
        col_pair[i] = static_cast<uint16_t>(max(p, 0));  // any pair's row of h
        col_weight[i] = p >= 0 ? a.col_weight[at] : -1.0f;
    }
    __syncthreads();
    const int kw = a.inter / 8;          // chunks of a row
    const int spi = (kw + 15) / 16;      // stages of an item
    const int stages = items * spi;
    const int s0 = static_cast<int>(static_cast<long long>(stages) * wave / KS);
    const int s1 = static_cast<int>(static_cast<long long>(stages) * (wave + 1) / KS);
    char *ring = lds + wave * D * SB;
    const int row = lane >> 4;
    // load of the next stage: li, lst its item and stage in it
    int li = s0 / spi, lst = s0 - li * spi, lslot = 0;
    const auto load = [&] {
        const int e = __builtin_amdgcn_readfirstlane(expert[li]);
        const char *w = a.w_out + static_cast<long long>(e) * a.hidden * a.inter * 2;
        char *dst = ring + lslot * SB;
#pragma unroll
        for (int m = 0; m < XC; ++m) {
            const int xr = 2 * m + (lane >> 5), q = 32 * lst + ((lane & 31) ^ xr);
            const int p = col_pair[li * XR + xr];
            dma16<false>(q < 2 * kw ? static_cast<const void *>(reinterpret_cast<const char *>(a.h) +
                                                                p * a.h_stride * 4 + 16 * q)
                                    : static_cast<const void *>(kZero16),
                         dst + WR * 256 + m * 1024);
        }
#pragma unroll
        for (int m = 0; m < WC; ++m) {
            const int q = 16 * lst + ((lane & 15) ^ (4 * m + row));
            const long long r = min(n0 + 4 * m + row, a.hidden - 1);
            dma16<true>(q < kw ? static_cast<const void *>(w + r * a.inter * 2 + 16 * q)
                               : static_cast<const void *>(kZero16),
                        dst + m * 1024);
        }
        if (++lst == spi) {
            lst = 0;
            ++li;
        }
        lslot = lslot + 1 == D ? 0 : lslot + 1;
    };
    const int wc = WR < 16 ? c & 7 : c, xc = c & (XR - 1);
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f}, low = acc, tot = acc;
    int ui = li, ust = lst, slot = 0;
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (s0 + d < s1) load();
    for (int s = s0; s < s1; ++s) {
        // stages s + 1 .. min(s + D - 2, s1 - 1) may still be in flight
        if (D > 3 && s + 2 < s1) wait_copies<(D > 3 ? 2 : 1) * PER>();
        else if (s + 1 < s1) wait_copies<PER>();
        else wait_copies<0>();
        if (s + D - 1 < s1) load();
        const char *wl = ring + slot * SB + wc * 256, *xl = ring + slot * SB + WR * 256 + xc * 512;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const u32x4_t w = *reinterpret_cast<const u32x4_t *>(wl + 16 * ((4 * u + g) ^ wc));
            acc = Mma16<T>::run(w, *reinterpret_cast<const u32x4_t *>(xl + 16 * ((8 * u + 2 * g) ^ xc)), acc);
            low = Mma16<T>::run(w, *reinterpret_cast<const u32x4_t *>(xl + 16 * ((8 * u + 2 * g + 1) ^ xc)), low);
        }
        slot = slot + 1 == D ? 0 : slot + 1;
        if (++ust == spi || s + 1 == s1) {
            const float wt = kUnit<T> * col_weight[ui * XR + xc];
#pragma unroll
            for (int v = 0; v < 4; ++v) tot[v] += wt >= 0.0f ? wt * both_terms<T>(acc[v], low[v]) : 0.0f;
            acc = low = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            ust = 0;
            ++ui;
        }
        // the reads of stage s are done before its slot is copied over
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    __syncthreads();
    float4_t *red = reinterpret_cast<float4_t *>(lds);
    red[wave * 64 + lane] = float4_t{tot[0], tot[1], tot[2], tot[3]};
    __syncthreads();
    if (wave != 0) return;
    float4_t sum = red[lane];
#pragma unroll
    for (int w = 1; w < KS; ++w) sum += red[w * 64 + lane];
    const int n = n0 + 4 * g;
    if (c >= a.tokens || g >= WR / 4 || n >= a.hidden) return;  // hidden % 8 == 0: four at a time
    uint16_t *dst = a.out + static_cast<long long>(c) * a.hidden + n;
    const uint32_t lo2 = tecoops::dev::round2<T>(sum[0], sum[1]), hi2 = tecoops::dev::round2<T>(sum[2], sum[3]);
    if (tecoops::aligned(dst, 8)) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(lo2, hi2);
    } else {
        dst[0] = static_cast<uint16_t>(lo2);
        dst[1] = static_cast<uint16_t>(lo2 >> 16);
        dst[2] = static_cast<uint16_t>(hi2);
        dst[3] = static_cast<uint16_t>(hi2 >> 16);
    }
}

template <typename T, int XR, int WR, int KS, int D>
bool launch_out_few(const MoeArgs &a, hipStream_t s) {
    auto *kern = &moe_out_few_kernel<T, XR, WR, KS, D>;
    constexpr size_t lds = KS * D * (WR * 256 + XR * 512);
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, dim3(tecoops::ceil_div(a.hidden, WR)), dim3(KS * 64), lds, s, a);
    return true;
}

// 16 rows of W_out to a workgroup where that leaves every CU one, else 8.
template <typename T>
bool run_out_few(const MoeArgs &a, hipStream_t s) {
    const bool wide = a.hidden >= 16 * tecoops::device_cus();
    if (a.rows == 4) return wide ? launch_out_few<T, 4, 16, 8, 3>(a, s) : launch_out_few<T, 4, 8, 8, 4>(a, s);
    return wide ? launch_out_few<T, 8, 16, 4, 4>(a, s) : launch_out_few<T, 8, 8, 8, 3>(a, s);
}

// Widths that are not in whole 16-byte words, or tensors that are not aligned: a
// wave per pair and row of the product.
template <typename T, bool OUT>
__global__ void __launch_bounds__(256) moe_scalar_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63;
    const int N = OUT ? a.hidden : a.inter, K = OUT ? a.inter : a.hidden;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int item = blockIdx.y;
    if (n >= N || item >= *a.n_items) return;
    const int4 it = a.items[item];
    const uint16_t *w = reinterpret_cast<const uint16_t *>(OUT ? a.w_out : a.w_in) +
                        static_cast<long long>(it.x) * (OUT ? 1 : 2) * a.hidden * a.inter +
                        static_cast<long long>(n) * K;
    for (int p = it.y; p < it.y + it.z; ++p) {
        float *const h = reinterpret_cast<float *>(a.h) + p * a.h_stride;
        const uint16_t *x = reinterpret_cast<const uint16_t *>(a.x + a.token[p] * a.x_stride);
        float s = 0.0f, u = 0.0f;
        for (int k = lane; k < K; k += 64) {
            const float xv = OUT ? h[k] : Cvt<T>::to(x[k]);
            s += Cvt<T>::to(w[k]) * xv;
            if (!OUT) u += Cvt<T>::to(w[static_cast<long long>(N) * K + k]) * xv;
        }
        s = wave_sum(s);
        if (!OUT) u = wave_sum(u);
        if (lane != 0) continue;
        if (OUT)
            a.part[static_cast<long long>(a.slot[p]) * N + n] = a.weight[p] * s;
        else
            h[n] = activate(s, a.act) * u;
    }
}

// out[t] from the parts of its pairs, in the order of j; zero where it has none.
template <typename T>
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeArgs a) {
    const int t = blockIdx.y;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    const bool whole = a.hidden % 4 == 0;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // a token's choices come first, so their number is that of its ids >= 0; the
    // parts are then loaded without a wait between them
    const int lane = threadIdx.x & 63;
    const int id = lane < a.top_k ? a.ids[t * a.top_k + lane] : -1;
    const int chosen = __builtin_popcountll(__ballot(id >= 0));
    if (n >= a.hidden) return;
    const float *src = a.part + static_cast<long long>(t) * a.top_k * a.hidden + n;
    if (whole) {
#pragma unroll 8
        for (int j = 0; j < chosen; ++j) {
            const f32x4_t v = *reinterpret_cast<const f32x4_t *>(src + static_cast<long long>(j) * a.hidden);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        }
    } else {
        for (int j = 0; j < chosen; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.hidden) s[i] += src[static_cast<long long>(j) * a.hidden + i];
    }
    uint16_t *dst = a.out + static_cast<long long>(t) * a.hidden + n;
    if (whole && tecoops::aligned(dst, 8)) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack<T>(s[0], s[1]), pack<T>(s[2], s[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.hidden) dst[i] = Cvt<T>::from(s[i]);
    }
}

template <typename T, int XR, int WR, int RS, int KS, bool OUT, int R>
bool launch_as(MoeArgs a, int items, hipStream_t s) {
    using S = Shape<OUT ? kTwoTerms : kPlain, XR, WR, RS, KS>;
    static_assert(S::D >= 2, "two stages fit in LDS");
    auto *kern = &moe_product_kernel<T, XR, WR, RS, KS, OUT, R>;
    if (!tecoops::reserve_lds(reinterpret_cast<const void *>(kern), S::LDS)) return false;
    a.units = static_cast<int>(tecoops::ceil_div(OUT ? a.hidden : 2LL * a.inter, RS * WR));
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(a.units) * items), dim3(S::NW * 64), S::LDS, s, a);
    return true;
}

// Whether the tokens are routed within the first product: it spares a launch and
// its wait, but every workgroup does it again at its start, so only where each CU
// has one of them (2 tokens, 1 of 128 experts of [1792, 672]: 12.3 us with a
// launch, 10.5 within; 6 tokens, 6 of 60 of [640, 9920], many to a CU: 182 and 286).
bool routes_within(const MoeArgs &a, int items, bool copy) {
    const int cus = tecoops::device_cus();
    return few_tokens(a, copy) &&
           static_cast<long long>(items) * tecoops::ceil_div(2LL * a.inter,
               tecoops::moe_wrows(2 * a.inter, a.tokens, a.top_k, a.experts, a.rows, cus)) <= cus;
}

template <typename T, int XR, int WR, int RS, int KS, bool OUT>
bool launch(const MoeArgs &a, int items, hipStream_t s) {
    if constexpr (!OUT && XR <= 8)
        if (routes_within(a, items, true))
            return a.experts <= 128
                       ? launch_as<T, XR, WR, RS, KS, OUT, 2>(a, items, s)
                       : launch_as<T, XR, WR, RS, KS, OUT, tecoops::kMoeMaxExperts / 64>(a, items, s);
    return launch_as<T, XR, WR, RS, KS, OUT, 0>(a, items, s);
}

template <typename T, int XR, bool OUT>
bool launch_wrows(const MoeArgs &a, int items, hipStream_t s) {
    // 64 rows of two-term x leave two stages in LDS from 32 rows of W on
    constexpr bool kLong = OUT && XR > 32;
    switch (tecoops::moe_wrows(OUT ? a.hidden : 2 * a.inter, a.tokens, a.top_k, a.experts, OUT ? 2 * XR : XR,
                               tecoops::device_cus())) {
        case 16:
            if constexpr (!kLong) return launch<T, XR, 16, 1, 4, OUT>(a, items, s);
            [[fallthrough]];
        case 32: return launch<T, XR, 16, 2, 2, OUT>(a, items, s);
        case 64: return launch<T, XR, kLong ? 16 : 32, kLong ? 4 : 2, kLong ? 1 : 2, OUT>(a, items, s);
        default: return launch<T, XR, 16, 8, 1, OUT>(a, items, s);
    }
}

template <typename T, bool OUT>
bool launch_product(const MoeArgs &a, int items, bool copy, hipStream_t s) {
    if (!copy) {
        hipLaunchKernelGGL((moe_scalar_kernel<T, OUT>),
                           dim3(tecoops::ceil_div(OUT ? a.hidden : a.inter, 4), items), dim3(256), 0,
                           s, a);
        return true;
    }
    switch (a.rows) {
        case 4: return launch_wrows<T, 4, OUT>(a, items, s);
        case 8: return launch_wrows<T, 8, OUT>(a, items, s);
        case 16: return launch_wrows<T, 16, OUT>(a, items, s);
        case 32: return launch_wrows<T, 32, OUT>(a, items, s);
        default: return launch_wrows<T, 64, OUT>(a, items, s);
    }
}

template <typename T>
tecoopsStatus_t run_slice(const MoeArgs &a, int items, bool copy, hipStream_t s) {
    if (!routes_within(a, items, copy)) {
        launch_route<T>(a, copy, s);
        TECO_CHECK_LAUNCH("moe_layer");
    }
    if (!launch_product<T, false>(a, items, copy, s)) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("moe_layer");
    if (few_tokens(a, copy) && tecoops::moe_out_few(a.tokens, a.hidden, a.inter, a.experts, a.top_k, tecoops::device_cus())) {
        if (!run_out_few<T>(a, s)) return TECOOPS_STATUS_INTERNAL_ERROR;
        TECO_CHECK_LAUNCH("moe_layer");
        return TECOOPS_STATUS_SUCCESS;
    }
    if (!launch_product<T, true>(a, items, copy, s)) return TECOOPS_STATUS_INTERNAL_ERROR;
    TECO_CHECK_LAUNCH("moe_layer");
    hipLaunchKernelGGL((moe_combine_kernel<T>), dim3(tecoops::ceil_div(a.hidden, 1024), a.tokens),
                       dim3(256), 0, s, a);
    TECO_CHECK_LAUNCH("moe_layer");
    return TECOOPS_STATUS_SUCCESS;
}

tecoopsStatus_t check_sizes(int tokens, int hidden, int inter, int experts, int top_k) {
    if (tokens < 0 || hidden <= 0 || inter <= 0 || experts <= 0 || top_k <= 0 || top_k > experts)
        return TECOOPS_STATUS_BAD_PARAM;
    if (tokens > tecoops::kMoeMaxTokens || experts > tecoops::kMoeMaxExperts || top_k > tecoops::kMoeMaxTopK ||
        hidden > tecoops::kMoeMaxWidth || inter > tecoops::kMoeMaxWidth)
        return TECOOPS_STATUS_NOT_SUPPORTED;
    return TECOOPS_STATUS_SUCCESS;
}

}  // namespace

extern "C" tecoopsStatus_t tecoopsGetMoeLayerWorkspaceSize(int tokens, int hidden, int inter,
                                                           int experts, int top_k, size_t *bytes) {
    if (bytes == nullptr) return TECOOPS_STATUS_BAD_PARAM;
    const tecoopsStatus_t st = check_sizes(tokens, hidden, inter, experts, top_k);
    if (st != TECOOPS_STATUS_SUCCESS) return st;
    *bytes = tokens == 0 ? 0 : tecoops::moe_space(tokens, hidden, inter, experts, top_k).bytes;
    return TECOOPS_STATUS_SUCCESS;
}

extern "C" tecoopsStatus_t tecoopsMoeLayer(tecoopsHandle_t handle, const void *x, long long x_stride,
                                           const void *w_in, const void *w_out,
                                           const void *router_logits, tecoopsDataType_t logitsType,
                                           void *out, int *topk_ids, float *topk_weights, int tokens,
                                           int hidden, int inter, int experts, int top_k,
                                           int renormalize, tecoopsActivation_t activation,
                                           void *workspace, size_t workspace_bytes,
                                           tecoopsDataType_t dataType) {
    if (handle == nullptr) return TECOOPS_STATUS_NOT_INITIALIZED;
    if (x == nullptr || w_in == nullptr || w_out == nullptr || router_logits == nullptr ||
        out == nullptr)
        return TECOOPS_STATUS_BAD_PARAM;
    const tecoopsStatus_t st = check_sizes(tokens, hidden, inter, experts, top_k);
    if (st != TECOOPS_STATUS_SUCCESS) return st;
    if (x_stride < hidden || !tecoops::epilogue_act_ok(activation) ||
        !tecoops::is_16bit_float(dataType))
        return TECOOPS_STATUS_BAD_PARAM;
    if (logitsType != TECOOPS_DATA_FLOAT && logitsType != dataType) return TECOOPS_STATUS_BAD_PARAM;
    const size_t logit = logitsType == TECOOPS_DATA_FLOAT ? 4 : 2;
    if (!tecoops::aligned(x, 2) || !tecoops::aligned(w_in, 2) || !tecoops::aligned(w_out, 2) ||
        !tecoops::aligned(out, 2) || !tecoops::aligned(router_logits, logit) ||
        !tecoops::aligned(topk_ids, 4) || !tecoops::aligned(topk_weights, 4))
        return TECOOPS_STATUS_BAD_PARAM;
    if (tokens == 0) return TECOOPS_STATUS_SUCCESS;
    const MoeSpace sp = tecoops::moe_space(tokens, hidden, inter, experts, top_k);
    if (workspace == nullptr) {
        const tecoopsStatus_t got = tecoops::handle_scratch(handle, sp.bytes, &workspace);
        if (got != TECOOPS_STATUS_SUCCESS) return got;
    } else if (workspace_bytes < sp.bytes || !tecoops::aligned(workspace, 16)) {
        return TECOOPS_STATUS_BAD_PARAM;
    }
    char *ws = static_cast<char *>(workspace);
    MoeArgs a{};
    a.w_in = static_cast<const char *>(w_in);
    a.w_out = static_cast<const char *>(w_out);
    a.x_stride = x_stride * 2;
    a.hidden = hidden;
    a.inter = inter;
    a.experts = experts;
    a.top_k = top_k;
    a.logits16 = logit == 2;
    a.renorm = renormalize != 0;
    a.act = activation;
    a.rows = sp.rows;
    a.n_items = reinterpret_cast<int *>(ws);
    a.items = reinterpret_cast<int4 *>(ws + sp.items_at);
    a.ids = reinterpret_cast<int *>(ws + sp.ids_at);
    a.token = reinterpret_cast<int *>(ws + sp.token_at);
    a.slot = reinterpret_cast<int *>(ws + sp.slot_at);
    a.weight = reinterpret_cast<float *>(ws + sp.weight_at);
    a.h = reinterpret_cast<uint16_t *>(ws + sp.h_at);
    a.h_stride = sp.h_stride;
    a.part = reinterpret_cast<float *>(ws + sp.part_at);
    a.col_pair = reinterpret_cast<int *>(ws + sp.cols_at);
    a.col_weight = reinterpret_cast<float *>(ws + sp.cols_at) + sp.items * tecoops::kMoeFew;
    const bool copy = hidden % 8 == 0 && inter % 8 == 0 && x_stride % 8 == 0 &&
                      tecoops::aligned(x, 16) && tecoops::aligned(w_in, 16) &&
                      tecoops::aligned(w_out, 16);
    for (int t0 = 0; t0 < tokens; t0 += tecoops::kMoeSlice) {
        a.tokens = tokens - t0 < tecoops::kMoeSlice ? tokens - t0 : tecoops::kMoeSlice;
        a.x = static_cast<const char *>(x) + t0 * a.x_stride;
        a.logits = static_cast<const char *>(router_logits) + static_cast<long long>(t0) * experts * logit;
        a.out = static_cast<uint16_t *>(out) + static_cast<long long>(t0) * hidden;
        a.topk_ids = topk_ids ? topk_ids + static_cast<long long>(t0) * top_k : nullptr;
        a.topk_weights = topk_weights ? topk_weights + static_cast<long long>(t0) * top_k : nullptr;
        const tecoopsStatus_t done = dataType == TECOOPS_DATA_HALF
                                         ? run_slice<f16>(a, sp.items, copy, handle->stream)
                                         : run_slice<bf16>(a, sp.items, copy, handle->stream);
        if (done != TECOOPS_STATUS_SUCCESS) return done;
    }
    return TECOOPS_STATUS_SUCCESS;
}
