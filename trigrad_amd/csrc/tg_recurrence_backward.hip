// tg_recurrence_backward.hip -- whole sequences of the gated linear recurrence, backward.
//
// e_t = a_{t+1} l_{t+1} is what reaches h_t from behind: l_t = dh_t + e_t, e_{t-1} = a_t l_t, a chain of maps like the forward one, against
// the order.  The states h_{t-1} that the gates' gradients need are not read but computed again, from the float32 states that the
// forward call kept every chunk_rows rows: x has to be read where the input is (1 - a) x or not, in the place of h, and h comes
// without having been rounded.
#include "tg_recurrence_scan.hpp"

#ifndef TG_DOUBLE_PRECISION
namespace tg {

template <class T, int V, bool Shared, int K, int Threads>
__global__ __launch_bounds__(Threads) void recurrence_backward_kernel(Split m, Chain c, const T *__restrict__ inputs, const void *__restrict__ gates,
                                                                      const float *__restrict__ initial, const int32_t *__restrict__ offsets,
                                                                      const float *__restrict__ kept, const T *__restrict__ grad_states,
                                                                      const float *__restrict__ grad_final, T *__restrict__ grad_inputs,
                                                                      void *__restrict__ grad_gates, float *__restrict__ grad_initial,
                                                                      float *__restrict__ partial) {
    constexpr int GV = Shared ? 1 : V;
    extern __shared__ int32_t table[];
    __shared__ Joint<V, Threads> joint;
    __shared__ uint32_t ticket;
    int64_t order, tile, channel, gate;
    int part;
    numbered(m, c, &ticket, order, tile);
    const int64_t chunk = m.chunks - 1 - order;
    const Place p = place_of<Threads>(m);
    const int places = (Threads >> m.lanes_log2) * K, at = p.turn * K;
    const int64_t start = chunk * m.chunk_rows;
    const int there = (int)min(m.chunk_rows, m.rows - start);
    const int n = max(0, min(there - at, K)), last = max(n - 1, 0);
    const bool valid = column_of<V, Shared>(m, (tile << m.lanes_log2) + p.lane, channel, gate, part);
    if (!valid) channel = gate = 0;
    const int64_t place = start + (n > 0 ? at : 0), row = m.reverse ? m.rows - 1 - place : place, step = m.reverse ? -1 : 1;
    const int64_t pitch = m.channels * step;

    Pack<T, V> x[K], dh[K];
    float a[K][GV], rest[K][GV];
    {
        const T *from = inputs + row * m.channels + channel;
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = load_pack<V>(from + pitch * min(k, last));
    }
    load_gates<T, K, GV>(m, gates, row, step, gate, last, a);
    if (grad_states) {
        const T *from = grad_states + row * m.channels + channel;
#pragma unroll
        for (int k = 0; k < K; k++) dh[k] = load_pack<V>(from + pitch * min(k, last));
    } else {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) dh[k].v[v] = (T)0.0f;
    }
    float known[V];
#pragma unroll
    for (int v = 0; v < V; v++) known[v] = m.chained ? kept[chunk * m.channels + channel + v] : 0.0f;

    uint32_t firsts = 0, lasts = 0, outside = 0;
    bool chunk_closed = false;
    int32_t *seq = table;
    if (!inside_one_sequence(m, c, offsets, chunk)) {
        uint8_t *flags = (uint8_t *)(table + places);
        chunk_table<Threads>(m, c, offsets, chunk, places, seq, flags);
        __syncthreads();
        for (int k = 0; k < n; k++) {
            const uint32_t f = flags[at + k];
            firsts |= (f & kFirst ? 1u : 0u) << k;
            lasts |= (f & kLast ? 1u : 0u) << k;
            outside |= (f & kOutside ? 1u : 0u) << k;
        }
        chunk_closed = (flags[there - 1] & kLast) != 0;
    }

#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int v = 0; v < GV; v++) {
            const Gate g = gate_of(m.gate_form, a[k][v]);
            a[k][v] = g.a;
            rest[k][v] = g.rest;
        }
    }
    if (n < K || outside) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool none = k >= n, out = (outside >> k & 1) != 0;
#pragma unroll
            for (int v = 0; v < GV; v++) {
                a[k][v] = none ? 1.0f : out ? 0.0f : a[k][v];
                rest[k][v] = none || out ? 0.0f : rest[k][v];
            }
            if (none || out) {
#pragma unroll
                for (int v = 0; v < V; v++) x[k].v[v] = dh[k].v[v] = (T)0.0f;
            }
        }
    }
    const auto begin = [&](int k, int v) {
        return initial && !(outside >> k & 1) && valid ? initial[seq[at + k] * m.channels + channel + v] : 0.0f;
    };
    const auto end = [&](int k, int v) {
        return grad_final && !(outside >> k & 1) && valid ? grad_final[seq[at + k] * m.channels + channel + v] : 0.0f;
    };
    const auto input = [&](int k, int v) { return m.complement ? rest[k][Shared ? 0 : v] * x[k][v] : x[k][v]; };

    // the states again
    Map<V> map = unit_map<V>();
    map.closed = firsts != 0;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (firsts >> k & 1) map.u[v] = begin(k, v);
            map.u[v] = fmaf(a[k][Shared ? 0 : v], map.u[v], input(k, v));
            map.a[v] *= a[k][Shared ? 0 : v];
        }
    float h[V], before[K][V];
    join<V, Threads, false>(m, c, joint, p, tile, chunk, map, false, false, known, h);
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (firsts >> k & 1) h[v] = begin(k, v);
            before[k][v] = h[v];
            h[v] = fmaf(a[k][Shared ? 0 : v], h[v], input(k, v));
        }

    // what reaches the last of the thread's rows from behind
    map = unit_map<V>();
    map.closed = lasts != 0;
#pragma unroll
    for (int k = K - 1; k >= 0; k--)
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (lasts >> k & 1) map.u[v] = end(k, v);
            map.u[v] = a[k][Shared ? 0 : v] * (map.u[v] + dh[k][v]);
            map.a[v] *= a[k][Shared ? 0 : v];
        }
    __syncthreads();
    float e[V];
    join<V, Threads, true>(m, c, joint, p, tile, order, map, chunk_closed, m.chained, nullptr, e);

    float q[K];
    const int64_t gate_pitch = m.gates * step;
#pragma unroll
    for (int k = K - 1; k >= 0; k--) {
        float dx[V], dg[V];
        q[k] = 0.0f;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float ak = a[k][Shared ? 0 : v], rk = rest[k][Shared ? 0 : v];
            if (lasts >> k & 1) e[v] = end(k, v);
            const float l = e[v] + dh[k][v];
            dx[v] = m.complement ? rk * l : l;
            const float da = l * (m.complement ? before[k][v] - x[k][v] : before[k][v]);
            e[v] = ak * l;
            if (Shared) q[k] += da;
            else dg[v] = m.gate_form == TG_GATE_VALUE ? da : m.gate_form == TG_GATE_LOG ? da * ak : da * (ak * rk);
        }
        if (valid && k < n) {
            if (grad_inputs) store_pack<V>(grad_inputs + row * m.channels + channel + pitch * k, dx);
            if (!Shared && grad_gates) {
                const int64_t to = row * m.gates + gate + gate_pitch * k;
                if (sizeof(T) == 4 || m.wide_gates) store_pack<V>((float *)grad_gates + to, dg);
                else store_pack<V>((T *)grad_gates + to, dg);
            }
            if (grad_initial && ((firsts & ~outside) >> k & 1)) {
#pragma unroll
                for (int v = 0; v < V; v++) grad_initial[seq[at + k] * m.channels + channel + v] = e[v];
            }
        }
    }
    if (!Shared || !grad_gates) return;
    const int gate_lanes = 1 << m.gate_lanes_log2, lane = threadIdx.x & (gate_lanes - 1);
#pragma unroll
    for (int k = 0; k < K; k++) {
        float sum = valid && !(outside >> k & 1) ? q[k] : 0.0f;
        for (int d = gate_lanes >> 1; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane == 0 && valid && k < n) {
            const int64_t to = row * m.gates + gate + gate_pitch * k;
            if (m.parts > 1) {
                partial[part * m.rows * m.gates + to] = sum;
                continue;
            }
            const float ak = a[k][0];
            sum = m.gate_form == TG_GATE_VALUE ? sum : m.gate_form == TG_GATE_LOG ? sum * ak : sum * (ak * rest[k][0]);
            if (sizeof(T) == 4 || m.wide_gates) ((float *)grad_gates)[to] = sum;
            else ((T *)grad_gates)[to] = (T)sum;
        }
    }
}

// Gates of more channels than a wave has: the sum of the waves' sums.
template <class T>
__global__ __launch_bounds__(256) void recurrence_gate_sums_kernel(Split m, const void *__restrict__ gates, const float *__restrict__ partial,
                                                                   void *__restrict__ grad_gates) {
    const int64_t n = m.rows * m.gates;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float sum = 0.0f;
        for (int part = 0; part < m.parts; part++) sum += partial[part * n + i];
        const bool wide = sizeof(T) == 4 || m.wide_gates;
        // a row of no sequence has sums of zero, whatever its gate is
        if (m.gate_form != TG_GATE_VALUE && sum != 0.0f) sum *= gate_of(m.gate_form, wide ? ((const float *)gates)[i] : (float)((const T *)gates)[i]).slope;
        if (wide) ((float *)grad_gates)[i] = sum;
        else ((T *)grad_gates)[i] = (T)sum;
    }
}

template <class T, int V, bool Shared>
int launch_backward(const tg_recurrence &r, const Split &m, const Chain &c, float *partial, unsigned blocks, hipStream_t stream) {
    constexpr int K = kBackwardRows, Threads = kBackwardThreads;
    const size_t lds = (size_t)(Threads >> m.lanes_log2) * K * 5;
    TG_LAUNCH_AS("recurrence_backward", (recurrence_backward_kernel<T, V, Shared, K, Threads>), dim3(blocks), dim3(Threads), lds, stream, m, c,
                 (const T *)r.inputs, r.gates, r.initial, r.offsets, (const float *)r.kept, (const T *)r.grad_states, r.grad_final,
                 (T *)r.grad_inputs, r.grad_gates, r.grad_initial, partial);
    if (Shared && r.grad_gates && m.parts > 1) {
        const unsigned sum_blocks = (unsigned)std::min<int64_t>(ceil_div64(m.rows * m.gates, 256), 4096);
        TG_LAUNCH_AS("recurrence_gate_sums", (recurrence_gate_sums_kernel<T>), dim3(sum_blocks), dim3(256), 0, stream, m, r.gates, partial, r.grad_gates);
    }
    return check_launch("tg_linear_recurrence_backward");
}

int launch_backward(const tg_recurrence &r, const Split &m, const Chain &c, float *partial, int vector, unsigned blocks, hipStream_t stream) {
    return by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        return launch_backward<decltype(t), decltype(v)::value, decltype(shared)::value>(r, m, c, partial, blocks, stream);
    });
}

}  // namespace tg
#endif  // !TG_DOUBLE_PRECISION
