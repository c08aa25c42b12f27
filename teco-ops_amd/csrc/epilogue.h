// epilogue.h — what a weight product does with its sums before they are
// rounded and stored: bias, activation, gate, residual.
//
//   out = T( act(s + bias) + residual )
//   out = T( act(g + bias_g) * (u + bias_u) + residual )     gated
//
// All in fp32, one rounding at the end.
#pragma once

#include "device.h"
#include "tecoops.h"

namespace tecoops {

struct Epilogue {
    const uint16_t *bias = nullptr;      // [rows of W] or null
    const uint16_t *residual = nullptr;  // [m, n] or null
    long long res_stride = 0;            // elements between rows
    long long out_stride = 0;
    int act = TECOOPS_ACTIVATION_NONE;
    int gated = 0;                       // W holds n gate rows, then n up rows
    int wide = 0;                        // 4 outputs of a row in one 8-byte word
};

inline bool epilogue_act_ok(int act) {
    return act >= TECOOPS_ACTIVATION_NONE && act <= TECOOPS_ACTIVATION_GELU_TANH;
}

namespace dev {

// Two results rounded to T (to nearest even; one instruction on gfx950).
template <typename T>
__device__ __forceinline__ uint32_t round2(float a, float b) {
    if constexpr (__is_same(T, f16))
        return __builtin_bit_cast(uint32_t, half2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)});
    else
        return __builtin_bit_cast(uint32_t, bf162_t{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}

// The exponentials are of the hardware's base-2 one: a relative error of about
// |v| 2^-24, far below half a step of the 16-bit result.  The sigmoid forms
// overflow to inf in the denominator for very negative v and give -0, their
// limit; gelu through erfc keeps its relative accuracy there, where 1 + erf
// cancels.
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case TECOOPS_ACTIVATION_RELU: return v < 0.0f ? 0.0f : v;
        case TECOOPS_ACTIVATION_SILU: return v / (1.0f + __expf(-v));
        case TECOOPS_ACTIVATION_GELU: return 0.5f * v * erfcf(v * -0.70710678f);
        case TECOOPS_ACTIVATION_GELU_TANH:
            return v / (1.0f + __expf(-1.5957691f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

// Four neighbouring outputs n .. n + 3 of row m from their sums s (and u, the
// up sums, when gated); columns from N on are not touched.
template <typename T>
__device__ __forceinline__ void finish4(const Epilogue &e, uint16_t *out, long long m, int n, int N,
                                        const float *s, const float *u) {
    if (n >= N) return;
    float v[4];
    const int last = N - 1 - n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = n + (i < last ? i : last);
        v[i] = s[i];
        if (e.bias != nullptr) v[i] += Cvt<T>::to(e.bias[c]);
        v[i] = activate(v[i], e.act);
        if (e.gated) v[i] *= u[i] + (e.bias != nullptr ? Cvt<T>::to(e.bias[N + c]) : 0.0f);
    }
    uint16_t *dst = out + m * e.out_stride + n;
    const uint16_t *res = e.residual + m * e.res_stride + n;
    if (e.wide) {
        if (e.residual != nullptr) {
            const uint2 r = *reinterpret_cast<const uint2 *>(res);
            v[0] += lo<T>(r.x);
            v[1] += hi<T>(r.x);
            v[2] += lo<T>(r.y);
            v[3] += hi<T>(r.y);
        }
        *reinterpret_cast<uint2 *>(dst) = make_uint2(round2<T>(v[0], v[1]), round2<T>(v[2], v[3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i <= last) {
            const float f = e.residual != nullptr ? v[i] + Cvt<T>::to(res[i]) : v[i];
            dst[i] = static_cast<uint16_t>(round2<T>(f, f));
        }
}

}  // namespace dev
}  // namespace tecoops
