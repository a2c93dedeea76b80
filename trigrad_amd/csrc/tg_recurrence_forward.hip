// tg_recurrence_forward.hip -- whole sequences of the gated linear recurrence, forward, and what both directions need before them.
#include "tg_recurrence_scan.hpp"

#ifndef TG_DOUBLE_PRECISION
namespace tg {

// What a thread's rows are: places [at, at + n) of the chunk, by the table's flags.
struct Marks {
    uint32_t firsts, lasts, outside;
};

template <class T, int V, bool Shared, int K, int Threads>
__global__ __launch_bounds__(Threads, 4) void recurrence_forward_kernel(Split m, Chain c, const T *__restrict__ inputs, const void *__restrict__ gates,
                                                                     const float *__restrict__ initial, const int32_t *__restrict__ offsets,
                                                                     T *__restrict__ states, float *__restrict__ final, float *__restrict__ kept) {
    constexpr int GV = Shared ? 1 : V;
    extern __shared__ int32_t table[];
    __shared__ Joint<V, Threads> joint;
    __shared__ uint32_t ticket;
    int64_t chunk, tile, channel, gate;
    int part;
    numbered(m, c, &ticket, chunk, tile);
    const Place p = place_of<Threads>(m);
    const int places = (Threads >> m.lanes_log2) * K, at = p.turn * K;
    const int64_t start = chunk * m.chunk_rows;
    const int n = (int)max((int64_t)0, min(min(m.chunk_rows, m.rows - start) - at, (int64_t)K)), last = max(n - 1, 0);
    const bool valid = column_of<V, Shared>(m, (tile << m.lanes_log2) + p.lane, channel, gate, part);
    if (!valid) channel = gate = 0;
    const int64_t place = start + (n > 0 ? at : 0), row = m.reverse ? m.rows - 1 - place : place, step = m.reverse ? -1 : 1;

    Pack<T, V> x[K];
    {
        const T *from = inputs + row * m.channels + channel;
        const int64_t pitch = m.channels * step;
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = load_pack<V>(from + pitch * min(k, last));
    }
    float a[K][GV], u[K][V];
    load_gates<T, K, GV>(m, gates, row, step, gate, last, a);

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
        chunk_closed = (flags[0] & kFirst) != 0;
    }

#pragma unroll
    for (int k = 0; k < K; k++) {
        float rest[GV];
#pragma unroll
        for (int v = 0; v < GV; v++) {
            const Gate g = gate_of(m.gate_form, a[k][v]);
            a[k][v] = g.a;
            rest[v] = g.rest;
        }
#pragma unroll
        for (int v = 0; v < V; v++) u[k][v] = m.complement ? rest[Shared ? 0 : v] * x[k][v] : x[k][v];
    }
    if (n < K || outside) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool none = k >= n, out = (outside >> k & 1) != 0;
#pragma unroll
            for (int v = 0; v < GV; v++) a[k][v] = none ? 1.0f : out ? 0.0f : a[k][v];
#pragma unroll
            for (int v = 0; v < V; v++) u[k][v] = none || out ? 0.0f : u[k][v];
        }
    }
    const auto begin = [&](int k, int v) {
        return initial && !(outside >> k & 1) && valid ? initial[seq[at + k] * m.channels + channel + v] : 0.0f;
    };

    Map<V> map = unit_map<V>();
    if (!firsts) {
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                map.u[v] = fmaf(a[k][Shared ? 0 : v], map.u[v], u[k][v]);
                map.a[v] *= a[k][Shared ? 0 : v];
            }
    } else {
        map.closed = true;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (firsts >> k & 1) map.u[v] = begin(k, v);
                map.u[v] = fmaf(a[k][Shared ? 0 : v], map.u[v], u[k][v]);
            }
    }
    float h[V];
    join<V, Threads, false>(m, c, joint, p, tile, chunk, map, chunk_closed, m.chained, nullptr, h);
    if (!valid || n == 0) return;
    if (kept && at % m.block_rows == 0) {
#pragma unroll
        for (int v = 0; v < V; v++) kept[(start + at) / m.block_rows * m.channels + channel + v] = h[v];
    }
    T *to = states ? states + row * m.channels + channel : nullptr;
    const int64_t pitch = m.channels * step;
    if (n == K && !(firsts | lasts)) {
        if (!to) return;
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = fmaf(a[k][Shared ? 0 : v], h[v], u[k][v]);
            store_pack<V>(to + pitch * k, h);
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (firsts >> k & 1) h[v] = begin(k, v);
                h[v] = fmaf(a[k][Shared ? 0 : v], h[v], u[k][v]);
            }
            if (to && k < n) store_pack<V>(to + pitch * k, h);
            if ((lasts & ~outside) >> k & 1) {
#pragma unroll
                for (int v = 0; v < V; v++) final[seq[at + k] * m.channels + channel + v] = h[v];
            }
        }
    }
}

// In front of a chained or packed call: words that say "not there yet", the ticket, the sequences that each chunk's rows are searched
// between, and the final states (or, backward, the initial states' gradients) of sequences without rows.
__global__ __launch_bounds__(256) void recurrence_prepare_kernel(Split m, Chain c, uint64_t *words, int64_t n_words, const int32_t *__restrict__ offsets,
                                                                 const float *__restrict__ from, float *__restrict__ to) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    for (int64_t i = id; i < n_words; i += all) words[i] = ~(uint64_t)0;
    if (id == 0 && m.chained) *c.ticket = 0;
    if (m.packed) {
        for (int64_t i = id; i < 2 * m.chunks; i += all) {
            const int64_t start = (i >> 1) * m.chunk_rows, place = (i & 1) ? min(start + m.chunk_rows, m.rows) - 1 : start;
            const int64_t row = m.reverse ? m.rows - 1 - place : place;
            int32_t lo = 0, hi = (int32_t)(m.sequences - 1);
            while (lo < hi) {
                const int32_t mid = lo + (hi - lo + 1) / 2;
                if (offsets[mid] <= row) lo = mid; else hi = mid - 1;
            }
            c.first_sequence[m.reverse ? i ^ 1 : i] = lo;
        }
    }
    if (to) {
        for (int64_t i = id; i < m.sequences * m.channels; i += all) {
            const int64_t s = i / m.channels;
            if (!m.packed || offsets[s + 1] <= offsets[s]) to[i] = from ? from[i] : 0.0f;
        }
    }
}

template <class T, int V, bool Shared>
int launch_forward(const tg_recurrence &r, const Split &m, const Chain &c, unsigned blocks, hipStream_t stream) {
    constexpr int K = kForwardRows, Threads = kForwardThreads;
    const size_t lds = (size_t)(Threads >> m.lanes_log2) * K * 5;
    TG_LAUNCH_AS("recurrence_forward", (recurrence_forward_kernel<T, V, Shared, K, Threads>), dim3(blocks), dim3(Threads), lds, stream, m, c,
                 (const T *)r.inputs, r.gates, r.initial, r.offsets, (T *)r.states, r.final, (float *)r.kept);
    return check_launch("tg_linear_recurrence_forward");
}

int launch_forward(const tg_recurrence &r, const Split &m, const Chain &c, int vector, unsigned blocks, hipStream_t stream) {
    return by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        return launch_forward<decltype(t), decltype(v)::value, decltype(shared)::value>(r, m, c, blocks, stream);
    });
}

int launch_prepare(const Split &m, const Chain &c, uint64_t *words, int64_t n_words, const int32_t *offsets, const float *from, float *to,
                   hipStream_t stream) {
    const int64_t most = std::max(std::max(n_words, 2 * m.chunks), to ? m.sequences * m.channels : 0);
    const unsigned blocks = (unsigned)std::min<int64_t>(std::max<int64_t>(ceil_div64(most, 1024), 1), 2048);
    TG_LAUNCH_AS("recurrence_prepare", recurrence_prepare_kernel, dim3(blocks), dim3(256), 0, stream, m, c, words, n_words, offsets, from, to);
    return check_launch("tg_linear_recurrence");
}

}  // namespace tg
#endif  // !TG_DOUBLE_PRECISION
