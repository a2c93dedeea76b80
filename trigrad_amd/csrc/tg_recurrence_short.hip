// tg_recurrence_short.hip -- the gated linear recurrence over sequences of at most eight rows: compositing a few slabs of an image.
//
// A thread has a sequence's rows of V channels in registers and walks them, so nothing is composed and nothing waits: memory traffic alone
// bounds it: eight slabs of 1920 x 1080 take 72 us forward (290 MB read or written, 4.0 TB/s) and 95 backward (555 MB, 5.8 TB/s; the inputs were
// read by the forward pass just before).  The kernels for longer sequences, with their tables of where sequences begin, took 90 and 175.
#include "tg_recurrence_scan.hpp"

#ifndef TG_DOUBLE_PRECISION
namespace tg {

struct ShortPlace {
    int64_t sequence, channel, gate, row, step;
    int part;
    bool valid;
};
template <int V, bool Shared> __device__ __forceinline__ ShortPlace short_place(const Split &m) {
    ShortPlace p;
    const uint32_t id = blockIdx.x * (uint32_t)kShortThreads + threadIdx.x;  // of fewer than 2^32, which the host sees to
    p.sequence = id / (uint32_t)m.columns;
    const int64_t column = id - p.sequence * m.columns;
    p.valid = p.sequence < m.sequences;
    p.part = 0;
    if (!Shared) {
        p.channel = p.gate = column * V;
    } else {
        const uint32_t run = (uint32_t)(column >> m.gate_lanes_log2), g = run / (uint32_t)m.parts;
        p.part = (int)(run - g * (uint32_t)m.parts);
        const int64_t within = (((int64_t)p.part << m.gate_lanes_log2) + (column & ((1 << m.gate_lanes_log2) - 1))) * V;
        p.gate = g;
        p.channel = p.gate * m.shared + within;
        p.valid = p.valid && within < m.shared;
    }
    if (!p.valid) p.sequence = p.channel = p.gate = 0;
    p.row = p.sequence * m.length + (m.reverse ? m.length - 1 : 0);
    p.step = m.reverse ? -1 : 1;
    return p;
}

template <class T, int V> __device__ __forceinline__ void load_short(const Split &m, const ShortPlace &p, const T *from, Pack<T, V> (&x)[kShortRows]) {
    const T *at = from + p.row * m.channels + p.channel;
#pragma unroll
    for (int k = 0; k < kShortRows; k++)
        if (k < m.length) x[k] = load_pack<V>(at + k * p.step * m.channels);
}
template <class T, int GV>
__device__ __forceinline__ void load_short_gates(const Split &m, const ShortPlace &p, const void *gates, float (&g)[kShortRows][GV]) {
    const int64_t at = p.row * m.gates + p.gate;
    if (sizeof(T) == 4 || m.wide_gates) {
#pragma unroll
        for (int k = 0; k < kShortRows; k++)
            if (k < m.length) {
                const Pack<float, GV> raw = load_pack<GV>((const float *)gates + at + k * p.step * m.gates);
#pragma unroll
                for (int v = 0; v < GV; v++) g[k][v] = raw.v[v];
            }
    } else {
        Pack<T, GV> raw[kShortRows];
#pragma unroll
        for (int k = 0; k < kShortRows; k++)
            if (k < m.length) raw[k] = load_pack<GV>((const T *)gates + at + k * p.step * m.gates);
#pragma unroll
        for (int k = 0; k < kShortRows; k++)
            if (k < m.length)
#pragma unroll
                for (int v = 0; v < GV; v++) g[k][v] = raw[k][v];
    }
}

template <class T, int V, bool Shared>
__global__ __launch_bounds__(kShortThreads) void recurrence_short_forward_kernel(Split m, const T *__restrict__ inputs, const void *__restrict__ gates,
                                                                                 const float *__restrict__ initial, T *__restrict__ states,
                                                                                 float *__restrict__ final) {
    constexpr int GV = Shared ? 1 : V;
    const ShortPlace p = short_place<V, Shared>(m);
    if (!p.valid) return;
    Pack<T, V> x[kShortRows];
    float g[kShortRows][GV], h[V];
    load_short(m, p, inputs, x);
    load_short_gates<T, GV>(m, p, gates, g);
    const int64_t at = p.sequence * m.channels + p.channel;
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = initial ? initial[at + v] : 0.0f;
#pragma unroll
    for (int k = 0; k < kShortRows; k++) {
        if (k >= m.length) break;
        Gate gate[GV];
#pragma unroll
        for (int v = 0; v < GV; v++) gate[v] = gate_of(m.gate_form, g[k][v]);
#pragma unroll
        for (int v = 0; v < V; v++) h[v] = fmaf(gate[Shared ? 0 : v].a, h[v], m.complement ? gate[Shared ? 0 : v].rest * x[k][v] : x[k][v]);
        if (states) store_pack<V>(states + (p.row + k * p.step) * m.channels + p.channel, h);
    }
#pragma unroll
    for (int v = 0; v < V; v++) final[at + v] = h[v];
}

template <class T, int V, bool Shared>
__global__ __launch_bounds__(kShortThreads) void recurrence_short_backward_kernel(Split m, const T *__restrict__ inputs, const void *__restrict__ gates,
                                                                                  const float *__restrict__ initial, const T *__restrict__ grad_states,
                                                                                  const float *__restrict__ grad_final, T *__restrict__ grad_inputs,
                                                                                  void *__restrict__ grad_gates, float *__restrict__ grad_initial,
                                                                                  float *__restrict__ partial) {
    constexpr int GV = Shared ? 1 : V;
    const ShortPlace p = short_place<V, Shared>(m);
    const int64_t at = p.sequence * m.channels + p.channel;
    Pack<T, V> x[kShortRows], dh[kShortRows];
    float a[kShortRows][GV], rest[kShortRows][GV], before[kShortRows][V], h[V], e[V];
    load_short(m, p, inputs, x);
    load_short_gates<T, GV>(m, p, gates, a);
    if (grad_states) load_short(m, p, grad_states, dh);
#pragma unroll
    for (int v = 0; v < V; v++) {
        h[v] = initial ? initial[at + v] : 0.0f;
        e[v] = grad_final ? grad_final[at + v] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kShortRows; k++) {
        if (k >= m.length) break;
#pragma unroll
        for (int v = 0; v < GV; v++) {
            const Gate gate = gate_of(m.gate_form, a[k][v]);
            a[k][v] = gate.a;
            rest[k][v] = gate.rest;
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            before[k][v] = h[v];
            h[v] = fmaf(a[k][Shared ? 0 : v], h[v], m.complement ? rest[k][Shared ? 0 : v] * x[k][v] : x[k][v]);
        }
    }
    const bool wide = sizeof(T) == 4 || m.wide_gates;
#pragma unroll
    for (int k = kShortRows - 1; k >= 0; k--) {
        if (k >= m.length) continue;
        const int64_t row = p.row + k * p.step;
        float dx[V], dg[V], sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float ak = a[k][Shared ? 0 : v], rk = rest[k][Shared ? 0 : v], l = grad_states ? e[v] + dh[k][v] : e[v];
            dx[v] = m.complement ? rk * l : l;
            dg[v] = l * (m.complement ? before[k][v] - x[k][v] : before[k][v]);
            e[v] = ak * l;
            if (Shared) sum = v == 0 ? dg[0] : sum + dg[v];
            else dg[v] *= m.gate_form == TG_GATE_VALUE ? 1.0f : m.gate_form == TG_GATE_LOG ? ak : ak * rk;
        }
        if (grad_inputs && p.valid) store_pack<V>(grad_inputs + row * m.channels + p.channel, dx);
        if (!grad_gates) continue;
        const int64_t to = row * m.gates + p.gate;
        if (!Shared) {
            if (!p.valid) continue;
            if (wide) store_pack<V>((float *)grad_gates + to, dg);
            else store_pack<V>((T *)grad_gates + to, dg);
        } else {
            sum = sum_lanes(p.valid ? sum : 0.0f, 1 << m.gate_lanes_log2);
            if (!p.valid || (threadIdx.x & ((1 << m.gate_lanes_log2) - 1)) != 0) continue;
            if (m.parts > 1) {
                partial[p.part * m.rows * m.gates + to] = sum;
                continue;
            }
            sum *= m.gate_form == TG_GATE_VALUE ? 1.0f : m.gate_form == TG_GATE_LOG ? a[k][0] : a[k][0] * rest[k][0];
            if (wide) ((float *)grad_gates)[to] = sum;
            else ((T *)grad_gates)[to] = (T)sum;
        }
    }
    if (grad_initial && p.valid)
#pragma unroll
        for (int v = 0; v < V; v++) grad_initial[at + v] = e[v];
}

int launch_short(const tg_recurrence &r, const Split &m, float *partial, int vector, bool backward, hipStream_t stream) {
    const unsigned blocks = (unsigned)ceil_div64(m.sequences * m.columns, kShortThreads);
    const int code = by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        constexpr bool Shared = decltype(shared)::value;
        if (backward)
            TG_LAUNCH_AS("recurrence_short_backward", (recurrence_short_backward_kernel<T, V, Shared>), dim3(blocks), dim3(kShortThreads), 0, stream, m,
                         (const T *)r.inputs, r.gates, r.initial, (const T *)r.grad_states, r.grad_final, (T *)r.grad_inputs, r.grad_gates,
                         r.grad_initial, partial);
        else
            TG_LAUNCH_AS("recurrence_short_forward", (recurrence_short_forward_kernel<T, V, Shared>), dim3(blocks), dim3(kShortThreads), 0, stream, m,
                         (const T *)r.inputs, r.gates, r.initial, (T *)r.states, r.final);
        return check_launch("tg_linear_recurrence");
    });
    if (code) return code;
    return backward ? launch_gate_sums(r, m, partial, stream) : 0;
}

}  // namespace tg
#endif  // !TG_DOUBLE_PRECISION
