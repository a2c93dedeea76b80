// tg_recurrence_backward.hip -- whole sequences of the gated linear recurrence, backward.
//
// e_t = a_{t+1} l_{t+1} is what reaches h_t from behind: l_t = dh_t + e_t, e_{t-1} = a_t l_t, a chain of maps like the forward one, against
// the order.  The states h_{t-1} that the gates' gradients need are not read but computed again, from the float32 states that the
// forward call kept for every chunk: x is read in the place of h, which comes without having been rounded.
//
// Eight rows a thread, since x, dh, the gates and eight states of each channel are held: 116 registers with shared gates, 136 without (three waves a
// SIMD; held to 128 it spills and takes 94 us where it takes 63, 2 x 8192 x 1536 in half precision).  4 x 4096 x 2048 with 16 gates: 56 us,
// 3.6 TB/s, of which the vector instructions are 35.
#include "tg_recurrence_scan.hpp"

#ifndef TG_DOUBLE_PRECISION
namespace tg {

template <class T, int V, bool Shared, int K, int Threads>
__global__ __launch_bounds__(Threads, Shared || Threads == kWideThreads ? 4 : 3) void recurrence_backward_kernel(
    Split m, const int32_t *__restrict__ first_sequence, const float *__restrict__ starts, const T *__restrict__ inputs, const void *__restrict__ gates,
    const float *__restrict__ initial, const int32_t *__restrict__ offsets, const float *__restrict__ kept, const T *__restrict__ grad_states,
    const float *__restrict__ grad_final, T *__restrict__ grad_inputs, void *__restrict__ grad_gates, float *__restrict__ grad_initial,
    float *__restrict__ partial) {
    constexpr int GV = Shared ? 1 : V;
    extern __shared__ uint32_t table[];
    __shared__ Joint<V, Threads> joint;
    int64_t channel, gate;
    int part;
    const int64_t chunk = blockIdx.x / (uint32_t)m.tiles, tile = blockIdx.x % (uint32_t)m.tiles;
    const Place p = place_of<Threads>(m);
    const int places = (Threads >> m.lanes_log2) * K, at = p.turn * K;
    const int64_t start = chunk * m.chunk_rows;
    const int there = (int)min(m.chunk_rows, m.rows - start);
    const int n = max(0, min(there - at, K));
    const bool valid = column_of<V, Shared>(m, (tile << m.lanes_log2) + p.lane, channel, gate, part);
    const Walk w = walk_of<K, Threads>(m, start, p.turn, n);
    const Column cx = column(m.channels, channel), cg = column(m.gates, gate);

    Pack<T, V> x[K], dh[K];
    float a[K][GV], rest[K][GV];
    each_row<K>(w, cx, inputs, [&](int k, const T *from) { x[k] = load_pack<V>(from); });
    read_gates<T, K, GV>(m, gates, w, cg, a);
    if (grad_states) {
        each_row<K>(w, cx, grad_states, [&](int k, const T *from) { dh[k] = load_pack<V>(from); });
    } else {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) dh[k].v[v] = (T)0.0f;
    }
    float h[V], e[V];  // the state in front of the chunk, what comes from behind it
#pragma unroll
    for (int v = 0; v < V; v++) {
        h[v] = m.chained ? kept[chunk * m.channels + channel + v] : 0.0f;
        e[v] = m.chained ? starts[chunk * m.channels + channel + v] : 0.0f;
    }

    uint32_t firsts = 0, lasts = 0, outside = 0;
    const bool open = inside_one_sequence(m, first_sequence, offsets, chunk);
    if (!open) {
        chunk_table<Threads>(m, first_sequence, offsets, chunk, places, table);
        __syncthreads();
        const Marks marks = marks_of(table + at, n);
        firsts = marks.firsts;
        lasts = marks.lasts;
        outside = marks.outside;
    }

    compute_gates<K, GV>(m, a, rest);
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
        return initial && !(outside >> k & 1) && valid ? initial[sequence_of(table[at + k]) * m.channels + channel + v] : 0.0f;
    };
    const auto end = [&](int k, int v) {
        return grad_final && !(outside >> k & 1) && valid ? grad_final[sequence_of(table[at + k]) * m.channels + channel + v] : 0.0f;
    };
    // Where none of the wave's rows begins or ends a sequence the loops know it, and the form of the input too.
    const bool marked = __any((firsts | lasts) != 0);
    const auto by_rows = [&](auto &&call) {
        if (marked) call(std::true_type(), std::integral_constant<int, 2>());
        else if (!Shared) call(std::false_type(), std::integral_constant<int, 2>());
        else if (m.complement) call(std::false_type(), std::integral_constant<int, 1>());
        else call(std::false_type(), std::integral_constant<int, 0>());
    };
    const auto input = [&](auto form, int k, int v) {
        const bool complement = decltype(form)::value == 2 ? m.complement : decltype(form)::value == 1;
        return complement ? rest[k][Shared ? 0 : v] * x[k][v] : x[k][v];
    };

    // the states again
    const bool alone = Threads >> m.lanes_log2 == 1;  // a thread has all rows of its chunk: nothing comes from another
    Map<V> map = unit_map<V>();
    map.closed = firsts != 0;
    if (!alone) by_rows([&](auto with_marks, auto form) {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (with_marks.value && (firsts >> k & 1)) map.u[v] = begin(k, v);
                map.u[v] = fmaf(a[k][Shared ? 0 : v], map.u[v], input(form, k, v));
                map.a[v] *= a[k][Shared ? 0 : v];
            }
    });
    float before[K][V];
    if (!alone) join<V, Threads, false>(m, joint, p, map, open, h);
    by_rows([&](auto with_marks, auto form) {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (with_marks.value && (firsts >> k & 1)) h[v] = begin(k, v);
                before[k][v] = h[v];
                h[v] = fmaf(a[k][Shared ? 0 : v], h[v], input(form, k, v));
            }
    });

    // what reaches the last of the thread's rows from behind
    map = unit_map<V>();
    map.closed = lasts != 0;
    const auto map_of_gradients = [&](auto with_marks) {
#pragma unroll
        for (int k = K - 1; k >= 0; k--)
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (with_marks.value && (lasts >> k & 1)) map.u[v] = end(k, v);
                map.u[v] = a[k][Shared ? 0 : v] * (map.u[v] + dh[k][v]);
                map.a[v] *= a[k][Shared ? 0 : v];
            }
    };
    if (!alone) {
        if (marked) map_of_gradients(std::true_type());
        else map_of_gradients(std::false_type());
        __syncthreads();
        join<V, Threads, true>(m, joint, p, map, open, e);
    }

    float q[K];  // of a shared gate: the sum over the lane's channels
    // dx of row k, and da in its place in before[]
    const auto gradients = [&](auto with_marks, auto form, int k, float (&dx)[V]) {
        const bool complement = decltype(form)::value == 2 ? m.complement : decltype(form)::value == 1;
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (with_marks.value && (lasts >> k & 1)) e[v] = end(k, v);
            const float l = e[v] + dh[k][v];
            dx[v] = complement ? rest[k][Shared ? 0 : v] * l : l;
            before[k][v] = l * (complement ? before[k][v] - x[k][v] : before[k][v]);
            e[v] = a[k][Shared ? 0 : v] * l;
        }
        if (Shared) {
            q[k] = before[k][0];
#pragma unroll
            for (int v = 1; v < V; v++) q[k] += before[k][v];
        }
    };
    const auto slope = [&](int k, int v) {
        return m.gate_form == TG_GATE_VALUE ? 1.0f : m.gate_form == TG_GATE_LOG ? a[k][v] : a[k][v] * rest[k][v];
    };
    const auto gate_gradients = [&](int k, float (&dg)[V]) {
#pragma unroll
        for (int v = 0; v < V; v++) dg[v] = before[k][v] * slope(k, Shared ? 0 : v);
    };
    const bool wide = sizeof(T) == 4 || m.wide_gates;
    if (w.whole && !marked) {
        const Walk back = against<K>(w);
        by_rows([&](auto with_marks, auto form) {
            if (with_marks.value) return;
            each_row<K>(back, cx, grad_inputs ? grad_inputs : const_cast<T *>(inputs), [&](int i, T *to) {
                float dx[V];
                gradients(with_marks, form, K - 1 - i, dx);
                if (grad_inputs && valid) store_pack<V>(to, dx);
            });
        });
        if (!Shared && grad_gates && valid) {
            if (wide)
                each_row<K>(w, cg, (float *)grad_gates, [&](int k, float *to) {
                    float dg[V];
                    gate_gradients(k, dg);
                    store_pack<V>(to, dg);
                });
            else
                each_row<K>(w, cg, (T *)grad_gates, [&](int k, T *to) {
                    float dg[V];
                    gate_gradients(k, dg);
                    store_pack<V>(to, dg);
                });
        }
    } else {
#pragma unroll
        for (int k = K - 1; k >= 0; k--) {
            float dx[V], dg[V];
            gradients(std::true_type(), std::integral_constant<int, 2>(), k, dx);
            if (!valid || k >= n) continue;
            const int64_t row = w.row + k * w.step;
            if (grad_inputs) store_pack<V>(grad_inputs + row * m.channels + channel, dx);
            if (!Shared && grad_gates) {
                gate_gradients(k, dg);
                if (wide) store_pack<V>((float *)grad_gates + row * m.gates + gate, dg);
                else store_pack<V>((T *)grad_gates + row * m.gates + gate, dg);
            }
            if (grad_initial && ((firsts & ~outside) >> k & 1)) {
#pragma unroll
                for (int v = 0; v < V; v++) grad_initial[sequence_of(table[at + k]) * m.channels + channel + v] = e[v];
            }
        }
    }
    if (!Shared || !grad_gates) return;
    const auto store_gate = [&](int k, float sum, float s) {
        const int64_t to = (w.row + k * w.step) * m.gates + gate;
        if (m.parts > 1) partial[part * m.rows * m.gates + to] = sum;
        else if (wide) ((float *)grad_gates)[to] = sum * s;
        else ((T *)grad_gates)[to] = (T)(sum * s);
    };
    if (!valid) {
#pragma unroll
        for (int k = 0; k < K; k++) q[k] = 0.0f;
    }
    const bool any_valid = __builtin_amdgcn_readfirstlane(valid ? 1 : 0) != 0;
    if (m.gate_lanes_log2 == 6) {
        const float sum = sum_rows(q);
        const int k = (threadIdx.x & (kWave - 1)) >> 3;
        float s = 1.0f;
#pragma unroll
        for (int i = 0; i < K; i++) s = i == k ? slope(i, 0) : s;
        if ((threadIdx.x & 7) == 0 && k < n && any_valid) store_gate(k, sum, s);
    } else {
        const int gate_lanes = 1 << m.gate_lanes_log2, lane = threadIdx.x & (gate_lanes - 1);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const float sum = sum_lanes(q[k], gate_lanes);
            if (lane == 0 && valid && k < n) store_gate(k, sum, slope(k, 0));
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

int launch_backward(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, const float *starts, float *partial, int vector,
                    unsigned blocks, hipStream_t stream) {
    return by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        using T = decltype(t);
        const auto with = [&](auto rows, auto threads) {
            constexpr int K = decltype(rows)::value, Threads = decltype(threads)::value;
            TG_LAUNCH_AS("recurrence_backward", (recurrence_backward_kernel<T, decltype(v)::value, decltype(shared)::value, K, Threads>), dim3(blocks),
                         dim3(Threads), table_bytes(m, Threads * K), stream, m, first_sequence, starts, (const T *)r.inputs, r.gates, r.initial,
                         r.offsets, (const float *)r.kept, (const T *)r.grad_states, r.grad_final, (T *)r.grad_inputs, r.grad_gates,
                         r.grad_initial, partial);
            return check_launch("tg_linear_recurrence_backward");
        };
        const int code = m.wide ? with(std::integral_constant<int, kWideRows>(), std::integral_constant<int, kWideThreads>())
                                : with(std::integral_constant<int, kBackwardRows>(), std::integral_constant<int, kBackwardThreads>());
        return code ? code : launch_gate_sums(r, m, partial, stream);
    });
}

int launch_gate_sums(const tg_recurrence &r, const Split &m, const float *partial, hipStream_t stream) {
    if (m.shared == 1 || !r.grad_gates || m.parts == 1) return 0;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div64(m.rows * m.gates, 256), 4096);
    const auto with = [&](auto t) {
        TG_LAUNCH_AS("recurrence_gate_sums", (recurrence_gate_sums_kernel<decltype(t)>), dim3(blocks), dim3(256), 0, stream, m, r.gates, partial,
                     r.grad_gates);
        return check_launch("tg_linear_recurrence_backward");
    };
    return r.type == TG_TYPE_F32 ? with(float()) : r.type == TG_TYPE_F16 ? with(half_t()) : with(bf16_t());
}

}  // namespace tg
#endif  // !TG_DOUBLE_PRECISION
