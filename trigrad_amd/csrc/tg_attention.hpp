// tg_attention.hpp -- what the kernels of linear attention share: sizes, strides and gates.
#pragma once
#include "tg_elements.hpp"

namespace tg {

struct Strides {  // in elements
    int64_t sequence, row, head;
};

struct Attention {
    int64_t sequences, length, rows;  // rows: of all sequences, with those of none
    int heads, key_heads, shared;     // shared: value heads of a key head
    int key_size, value_size;
    Strides q, k, v, g;
    int gate_form;
    bool fixed, packed;
    real scale;
};

// The rows of a sequence: `first` counts as the outputs' rows do.
struct AttentionRows {
    int64_t first, count;
};
__device__ __forceinline__ AttentionRows rows_of(const Attention &m, const int32_t *offsets, int64_t s) {
    if (!m.packed) return {s * m.length, m.length};
    const int64_t first = min((int64_t)max(offsets[s], 0), m.length);
    return {first, max(first, min((int64_t)max(offsets[s + 1], 0), m.length)) - first};
}
// Where a sequence's first row lies in a tensor of these strides.
__device__ __forceinline__ int64_t place_of(const Attention &m, const Strides &t, int64_t s, int64_t first, int head) {
    return (m.packed ? first * t.row : s * t.sequence) + head * t.head;
}

// log2 of a gate in 64 bits, of which differences over a sequence are taken: logarithms of successive gates add up to thousands, and a decay
// between two rows needs 24 bits of their difference.  Minus infinity counts as 2^-300, which no float32 survives.
__device__ __forceinline__ double log2_gate(int form, float g) {
    double l = (double)g;
    if (form == TG_GATE_LOGIT) {  // -log(1 + exp(-g)), from exp(-|g|): neither end loses digits
        const float e = expf(-fabsf(g));
        l = fmin(l, 0.0) - (double)log1pf(e);
    }
    l *= 1.4426950408889634;
    return l < -300.0 ? -300.0 : l;
}
__device__ __forceinline__ double log2_gate(int form, double g) {
    const double l = (form == TG_GATE_LOGIT ? fmin(g, 0.0) - log1p(exp(-fabs(g))) : g) * 1.4426950408889634;
    return l < -4000.0 ? -4000.0 : l;
}
// d log a / d gate
__device__ __forceinline__ double slope_of(int form, double g) { return form == TG_GATE_LOGIT ? 1.0 / (1.0 + exp(g)) : 1.0; }

int attention_shape(const char *fn, const tg_attention &a, Attention &m);

}  // namespace tg
