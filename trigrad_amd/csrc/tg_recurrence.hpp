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
// exp(g) as a power of two: off by |g| / 2 + 1 units of 2^-24 of itself, so by more than a few units only where it is below e^-8.  (Putting the
// product's rounding error back took four more instructions of the about twenty that an element has.)
__device__ __forceinline__ float exp_real(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504f); }
// 1 - exp(g) without the loss of its leading digits: near 0 by its series (the first term left out is below 2^-25 of it).
__device__ __forceinline__ float one_minus_exp(float g, float e) {
    float s = fmaf(g, 1.0f / 5040, 1.0f / 720);
    s = fmaf(g, s, 1.0f / 120);
    s = fmaf(g, s, 1.0f / 24);
    s = fmaf(g, s, 1.0f / 6);
    s = fmaf(g, s, 0.5f);
    s = -fmaf(g * g, s, g);
    return fabsf(g) < 0.35f ? s : 1.0f - e;
}
__device__ __forceinline__ float reciprocal(float v) { return __builtin_amdgcn_rcpf(v); }  // to one unit
#endif

template <int Form> __device__ __forceinline__ Gate gate_of(real g) {
    Gate r;
    if (Form == TG_GATE_VALUE) {
        r.a = g;
        r.rest = (real)1 - g;
        r.slope = (real)1;
    } else if (Form == TG_GATE_LOG) {
        r.a = exp_real(g);
        r.rest = one_minus_exp(g, r.a);
        r.slope = r.a;
    } else {
        // from exp(-|g|), so that neither 1 - a near a = 1 nor a near 0 loses digits, and infinite logits are 0 and 1
        const real e = exp_real(-fabs(g)), big = reciprocal((real)1 + e), small = e * big;
        r.a = g >= 0 ? big : small;
        r.rest = g >= 0 ? small : big;
        r.slope = big * small;
    }
    return r;
}
__device__ __forceinline__ Gate gate_of(int form, real g) {
    return form == TG_GATE_VALUE ? gate_of<TG_GATE_VALUE>(g) : form == TG_GATE_LOG ? gate_of<TG_GATE_LOG>(g) : gate_of<TG_GATE_LOGIT>(g);
}

struct Shape {
    int64_t sequences, length, channels, gates, shared;  // shared: channels of a gate
    int gate_form;
    bool complement, reverse;
};

int recurrence_shape(const char *fn, const tg_recurrence &r, Shape &m);

}  // namespace tg
