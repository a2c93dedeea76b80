// tg_recurrence.hip -- the gated linear recurrence h_t = a_t h_{t-1} + u_t: whole sequences forward and backward, and a single step.
//
// With a = f(gate) and u = x or (1 - a) x, and l_t the gradient of h_t with all that follows from it,
//     l_t = dh_t + a_{t+1} l_{t+1},   dx_t = l_t or (1 - a_t) l_t,   da_t = l_t h_{t-1} or l_t (h_{t-1} - x_t),   dgate = f'(gate) sum da
// over the channels that share the gate.
#include "tg_elements.hpp"

namespace tg {

// 1 - exp(g) for g <= 0 without the loss of its leading digits: near 0 by its series (the first term left out is below 2^-25 of it).
__device__ __forceinline__ real one_minus_exp(real g, real e) {
#ifdef TG_DOUBLE_PRECISION
    return -expm1(g);
#else
    const float s = g * (1.0f + g * (1.0f / 2) * (1.0f + g * (1.0f / 3) * (1.0f + g * (1.0f / 4) * (1.0f + g * (1.0f / 5) *
                    (1.0f + g * (1.0f / 6) * (1.0f + g * (1.0f / 7)))))));
    return fabsf(g) < 0.35f ? -s : 1.0f - e;
#endif
}

struct Gate {
    real a, rest, slope;  // a, 1 - a, da / dgate
};

__device__ __forceinline__ Gate gate_of(int form, real g) {
    Gate r;
    if (form == TG_GATE_VALUE) {
        r.a = g;
        r.rest = (real)1 - g;
        r.slope = (real)1;
    } else if (form == TG_GATE_LOG) {
        r.a = exp(g);
        r.rest = one_minus_exp(g, r.a);
        r.slope = r.a;
    } else {
        const real e = exp(-fabs(g)), big = (real)1 / ((real)1 + e), small = e * big;
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

__device__ __forceinline__ real fma_real(real a, real b, real c) { return fma(a, b, c); }

// ---- one thread a sequence and channel ------------------------------------------------

struct Rows {
    int64_t begin, end;
};
__device__ __forceinline__ Rows rows_of(const Shape &m, const int32_t *offsets, int64_t s) {
    Rows r;
    if (!offsets) {
        r.begin = s * m.length;
        r.end = r.begin + m.length;
    } else {
        r.begin = min((int64_t)max(offsets[s], 0), m.length);
        r.end = max(r.begin, min((int64_t)max(offsets[s + 1], 0), m.length));
    }
    return r;
}

// The rows in front of the first sequence and behind the last one: zeros.
template <class T> __device__ void clear_outside(const Shape &m, const int32_t *offsets, int64_t s, T *out, int64_t column, int64_t columns) {
    if (!offsets || !out) return;
    const int64_t first = s == 0 ? 0 : rows_of(m, offsets, s).end;
    const int64_t begin = s == 0 ? rows_of(m, offsets, 0).begin : 0;
    if (s == 0)
        for (int64_t r = first; r < begin; r++) out[r * columns + column] = (T)(real)0;
    if (s == m.sequences - 1)
        for (int64_t r = rows_of(m, offsets, s).end; r < m.length; r++) out[r * columns + column] = (T)(real)0;
}

template <class T, class S>
__global__ void recurrence_forward_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates, const real *__restrict__ initial,
                                          const int32_t *__restrict__ offsets, T *__restrict__ states, real *__restrict__ final,
                                          real *__restrict__ kept) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= m.sequences * m.channels) return;
    const int64_t s = id / m.channels, d = id % m.channels, g = d / m.shared;
    const Rows rows = rows_of(m, offsets, s);
    real h = initial ? initial[id] : (real)0;
    for (int64_t i = rows.begin; i < rows.end; i++) {
        const int64_t r = m.reverse ? rows.end - 1 - (i - rows.begin) : i;
        const Gate gate = gate_of(m.gate_form, (real)gates[r * m.gates + g]);
        const real x = (real)inputs[r * m.channels + d];
        if (kept) kept[r * m.channels + d] = h;
        h = fma_real(gate.a, h, m.complement ? gate.rest * x : x);
        if (states) states[r * m.channels + d] = (T)h;
    }
    final[id] = h;
    clear_outside(m, offsets, s, states, d, m.channels);
}

template <class T, class S>
__global__ void recurrence_backward_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates, const int32_t *__restrict__ offsets,
                                           const real *__restrict__ kept, const T *__restrict__ grad_states,
                                           const real *__restrict__ grad_final, T *__restrict__ grad_inputs, S *__restrict__ grad_gates,
                                           real *__restrict__ grad_initial, real *__restrict__ carried) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= m.sequences * m.gates) return;
    const int64_t s = id / m.gates, g = id % m.gates;
    const Rows rows = rows_of(m, offsets, s);
    real *e = carried + s * m.channels;
    for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) e[d] = grad_final ? grad_final[s * m.channels + d] : (real)0;
    for (int64_t i = rows.begin; i < rows.end; i++) {
        const int64_t r = m.reverse ? i : rows.end - 1 - (i - rows.begin);
        const Gate gate = gate_of(m.gate_form, (real)gates[r * m.gates + g]);
        real sum = 0;
        for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) {
            const int64_t at = r * m.channels + d;
            const real l = e[d] + (grad_states ? (real)grad_states[at] : (real)0);
            sum = fma_real(l, m.complement ? kept[at] - (real)inputs[at] : kept[at], sum);
            if (grad_inputs) grad_inputs[at] = (T)(m.complement ? gate.rest * l : l);
            e[d] = gate.a * l;
        }
        if (grad_gates) grad_gates[r * m.gates + g] = (S)(sum * gate.slope);
    }
    for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) {
        if (grad_initial) grad_initial[s * m.channels + d] = e[d];
        clear_outside(m, offsets, s, grad_inputs, d, m.channels);
    }
    clear_outside(m, offsets, s, grad_gates, g, m.gates);
}

// ---- a single step ----------------------------------------------------------------------

constexpr int kStepThreads = 256;

template <class T, class S>
__global__ __launch_bounds__(kStepThreads) void recurrence_step_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates,
                                                                       const real *state, T *__restrict__ states, real *new_state) {
    const int64_t id = (int64_t)blockIdx.x * kStepThreads + threadIdx.x;
    if (id >= m.sequences * m.channels) return;
    const int64_t s = id / m.channels, g = id % m.channels / m.shared;
    const Gate gate = gate_of(m.gate_form, (real)gates[s * m.gates + g]);
    const real x = (real)inputs[id];
    const real h = fma_real(gate.a, state[id], m.complement ? gate.rest * x : x);
    new_state[id] = h;
    states[id] = (T)h;
}

// ---- host ---------------------------------------------------------------------------------

static int check_shape(const char *fn, const tg_recurrence &r, Shape &m) {
    if (r.sequences < 0 || r.length < 0 || r.channels < 0 || r.gate_count < 0 || (r.gate_count == 0) != (r.channels == 0) ||
        (r.gate_count > 0 && r.channels % r.gate_count != 0)) {
        set_error("%s: sizes", fn);
        return TG_E_ARG;
    }
    if (!type_known(r.type) || (r.gate_type != r.type && r.gate_type != kRealType)) {
        set_error("%s: types %lld and %lld", fn, (long long)r.type, (long long)r.gate_type);
        return TG_E_ARG;
    }
    if (r.gate_form < TG_GATE_VALUE || r.gate_form > TG_GATE_LOGIT || r.input_form < TG_INPUT_PLAIN || r.input_form > TG_INPUT_COMPLEMENT) {
        set_error("%s: gate_form %lld, input_form %lld", fn, (long long)r.gate_form, (long long)r.input_form);
        return TG_E_ARG;
    }
    const int64_t limit = (int64_t)1 << 40;
    const int64_t rows = r.offsets ? r.length : r.length == 0 ? 0 : r.sequences > limit / r.length ? limit : r.sequences * r.length;
    if (rows >= limit || (r.offsets && r.length > 0x7fffffff) || r.channels >= ((int64_t)1 << 31) || r.sequences >= ((int64_t)1 << 31) ||
        (r.channels > 0 && (rows > limit / r.channels || r.sequences > limit / r.channels))) {
        set_error("%s: more than 2^40 elements, or a size of 2^31", fn);
        return TG_E_ARG;
    }
    m.sequences = r.sequences;
    m.length = r.length;
    m.channels = r.channels;
    m.gates = r.gate_count;
    m.shared = r.gate_count ? r.channels / r.gate_count : 1;
    m.gate_form = (int)r.gate_form;
    m.complement = r.input_form == TG_INPUT_COMPLEMENT;
    m.reverse = r.reverse != 0;
    return 0;
}

}  // namespace tg

extern "C" int tg_linear_recurrence_sizes(const tg_recurrence *r, int64_t out[3]) {
    using namespace tg;
    if (!r || !out) {
        set_error("tg_linear_recurrence_sizes: null pointer");
        return TG_E_ARG;
    }
    Shape m;
    if (const int code = check_shape("tg_linear_recurrence_sizes", *r, m)) return code;
    const int64_t rows = r->offsets ? m.length : m.sequences * m.length;
    out[0] = rows * m.channels * (int64_t)sizeof(real);
    out[1] = 0;
    out[2] = m.sequences * m.channels * (int64_t)sizeof(real);
    return 0;
}

extern "C" int tg_linear_recurrence_forward(const tg_recurrence *r) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_forward";
    Shape m;
    int64_t sizes[3];
    if (!r) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    if (const int code = check_shape(fn, *r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    tg_linear_recurrence_sizes(r, sizes);
    if ((m.length > 0 && (!r->inputs || !r->gates)) || !r->final || (r->kept && r->kept_bytes < sizes[0])) {
        set_error("%s: null pointer, or kept too small", fn);
        return TG_E_ARG;
    }
    hipStream_t stream = (hipStream_t)r->stream;
    return by_types(r->type, r->gate_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        const int64_t n = m.sequences * m.channels;
        TG_LAUNCH_AS("recurrence_forward", (recurrence_forward_kernel<T, S>), dim3((unsigned)ceil_div64(n, 256)), dim3(256), 0, stream, m,
                     (const T *)r->inputs, (const S *)r->gates, r->initial, r->offsets, (T *)r->states, r->final, (real *)r->kept);
        return check_launch(fn);
    });
}

extern "C" int tg_linear_recurrence_backward(const tg_recurrence *r) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_backward";
    Shape m;
    int64_t sizes[3];
    if (!r) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    if (const int code = check_shape(fn, *r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    tg_linear_recurrence_sizes(r, sizes);
    if (m.length > 0 && (!r->inputs || !r->gates || !r->kept || r->kept_bytes < sizes[0])) {
        set_error("%s: null pointer, or kept too small", fn);
        return TG_E_ARG;
    }
    if (!r->workspace || r->workspace_bytes < sizes[2]) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)r->workspace_bytes, (long long)sizes[2]);
        return TG_E_WORKSPACE;
    }
    hipStream_t stream = (hipStream_t)r->stream;
    return by_types(r->type, r->gate_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        const int64_t n = m.sequences * m.gates;
        TG_LAUNCH_AS("recurrence_backward", (recurrence_backward_kernel<T, S>), dim3((unsigned)ceil_div64(n, 256)), dim3(256), 0, stream, m,
                     (const T *)r->inputs, (const S *)r->gates, r->offsets, (const real *)r->kept, (const T *)r->grad_states, r->grad_final,
                     (T *)r->grad_inputs, (S *)r->grad_gates, r->grad_initial, (real *)r->workspace);
        return check_launch(fn);
    });
}

extern "C" int tg_linear_recurrence_step(const void *inputs, const void *gates, const tg_real *state, void *states, tg_real *new_state,
                                         int64_t sequences, int64_t channels, int64_t gate_count, int type, int gate_type, int gate_form,
                                         int input_form, void *stream) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_step";
    tg_recurrence r = {};
    r.sequences = sequences;
    r.length = 1;
    r.channels = channels;
    r.gate_count = gate_count;
    r.type = type;
    r.gate_type = gate_type;
    r.gate_form = gate_form;
    r.input_form = input_form;
    Shape m;
    if (const int code = check_shape(fn, r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    if (!inputs || !gates || !state || !states || !new_state) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    return by_types(type, gate_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        const int64_t n = m.sequences * m.channels;
        TG_LAUNCH_AS("recurrence_step", (recurrence_step_kernel<T, S>), dim3((unsigned)ceil_div64(n, kStepThreads)), dim3(kStepThreads), 0,
                     (hipStream_t)stream, m, (const T *)inputs, (const S *)gates, state, (T *)states, new_state);
        return check_launch(fn);
    });
}
