// tg_recurrence.hpp -- what the kernels of the gated linear recurrence share: gates, sizes, and how rows and columns are split.
#pragma once
#include "tg_elements.hpp"

namespace tg {

struct Gate {
    real a, rest, slope;  // a, 1 - a, da / dgate
};

#ifdef TG_DOUBLE_PRECISION
__device__ __forceinline__ real exp_real(real g) { return exp(g); }
__device__ __forceinline__ real one_minus_exp(real g, real) { return -expm1(g); }
__device__ __forceinline__ real reciprocal(real v) { return 1.0 / v; }
#else
// exp(g) to about one unit: 2^(g log2 e) with the product's rounding error, and the constant's, put back to first order.  Where that
// would meet an infinity (beyond e^87) the plain power is left as it is: 0, infinity, NaN, or off by 2^-18 of a value that small or large.
__device__ __forceinline__ float exp_real(float g) {
    const float t = g * 1.44269504f, low = fmaf(g, 1.44269504f, -t), r = __builtin_amdgcn_exp2f(t);
    const float fine = fmaf(r, fmaf(g, 1.925963033e-8f, low) * 0.693147181f, r);
    return fabsf(g) < 87.0f ? fine : r;
}
// 1 - exp(g) without the loss of its leading digits: near 0 by its series (the first term left out is below 2^-25 of it).
__device__ __forceinline__ float one_minus_exp(float g, float e) {
    const float s = g * (1.0f + g * (1.0f / 2) * (1.0f + g * (1.0f / 3) * (1.0f + g * (1.0f / 4) * (1.0f + g * (1.0f / 5) *
                    (1.0f + g * (1.0f / 6) * (1.0f + g * (1.0f / 7)))))));
    return fabsf(g) < 0.35f ? -s : 1.0f - e;
}
// 1 / v for v in [1, 2]: the hardware's approximation and one step of Newton's.
__device__ __forceinline__ float reciprocal(float v) {
    const float r = __builtin_amdgcn_rcpf(v);
    return fmaf(r, fmaf(-v, r, 1.0f), r);
}
#endif

__device__ __forceinline__ Gate gate_of(int form, real g) {
    Gate r;
    if (form == TG_GATE_VALUE) {
        r.a = g;
        r.rest = (real)1 - g;
        r.slope = (real)1;
    } else if (form == TG_GATE_LOG) {
        r.a = exp_real(g);
        r.rest = one_minus_exp(g, r.a);
        r.slope = r.a;
    } else {
        const real e = exp_real(-fabs(g)), big = reciprocal((real)1 + e), small = e * big;
        r.a = g >= 0 ? big : small;
        r.rest = g >= 0 ? small : big;
        r.slope = big * small;
    }
    return r;
}

struct Shape {
    int64_t sequences, length, channels, gates, shared;  // shared: channels of a gate
    int gate_form;
    bool complement, reverse;
};

int recurrence_shape(const char *fn, const tg_recurrence &r, Shape &m);

}  // namespace tg
