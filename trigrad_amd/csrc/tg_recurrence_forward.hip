// tg_recurrence_forward.hip -- whole sequences of the gated linear recurrence, forward, and what both directions need before them.
//
// The forward kernel has a and u of sixteen rows of two channels in 64 registers and the workgroup's maps in LDS: loads, one pass for the maps, one for
// the states.  32768 x 2048 with logits: 89 us, 402 MB, 4.5 TB/s.
#include "tg_recurrence_scan.hpp"

#ifndef TG_DOUBLE_PRECISION
namespace tg {

template <class T, int V, bool Shared, int K, int Threads>
__global__ __launch_bounds__(Threads, 4) void recurrence_forward_kernel(Split m, const int32_t *__restrict__ first_sequence,
                                                                        const float *__restrict__ starts, const T *__restrict__ inputs,
                                                                        const void *__restrict__ gates, const float *__restrict__ initial,
                                                                        const int32_t *__restrict__ offsets, T *__restrict__ states,
                                                                        float *__restrict__ final, float *__restrict__ kept) {
    constexpr int GV = Shared ? 1 : V;
    extern __shared__ uint32_t table[];
    __shared__ Joint<V, Threads> joint;
    int64_t channel, gate;
    int part;
    const int64_t chunk = blockIdx.x / (uint32_t)m.tiles, tile = blockIdx.x % (uint32_t)m.tiles;
    const Place p = place_of<Threads>(m);
    const int places = (Threads >> m.lanes_log2) * K, at = p.turn * K;
    const int64_t start = chunk * m.chunk_rows;
    const int n = (int)max((int64_t)0, min(min(m.chunk_rows, m.rows - start) - at, (int64_t)K));
    const bool valid = column_of<V, Shared>(m, (tile << m.lanes_log2) + p.lane, channel, gate, part);
    const Walk w = walk_of<K, Threads>(m, start, p.turn, n);
    const Column cx = column(m.channels, channel), cg = column(m.gates, gate);

    Pack<T, V> x[K];
    each_row<K>(w, cx, inputs, [&](int k, const T *from) { x[k] = load_pack<V>(from); });
    float a[K][GV], u[K][V];
    read_gates<T, K, GV>(m, gates, w, cg, a);

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

    {
        float rest[K][GV];
        compute_gates<K, GV>(m, a, rest);
        if (m.complement) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < V; v++) u[k][v] = rest[k][Shared ? 0 : v] * x[k][v];
        } else {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < V; v++) u[k][v] = x[k][v];
        }
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
        return initial && !(outside >> k & 1) && valid ? initial[sequence_of(table[at + k]) * m.channels + channel + v] : 0.0f;
    };

    const bool alone = Threads >> m.lanes_log2 == 1;  // a thread has all rows of its chunk: nothing comes from another
    Map<V> map = unit_map<V>();
    if (alone) {
    } else if (!firsts) {
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
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = m.chained ? starts[chunk * m.channels + channel + v] : 0.0f;
    if (!alone) join<V, Threads, false>(m, joint, p, map, open, h);
    if (!valid || n == 0) return;
    if (kept && at % (int)m.kept_rows == 0) {
#pragma unroll
        for (int v = 0; v < V; v++) kept[(start + at) / m.kept_rows * m.channels + channel + v] = h[v];
    }
    if (w.whole && !(firsts | lasts)) {
        if (!states) return;
        each_row<K>(w, cx, states, [&](int k, T *to) {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = fmaf(a[k][Shared ? 0 : v], h[v], u[k][v]);
            store_pack<V>(to, h);
        });
    } else {
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (firsts >> k & 1) h[v] = begin(k, v);
                h[v] = fmaf(a[k][Shared ? 0 : v], h[v], u[k][v]);
            }
            if (states && k < n) store_pack<V>(states + (w.row + k * w.step) * m.channels + channel, h);
            if ((lasts & ~outside) >> k & 1) {
#pragma unroll
                for (int v = 0; v < V; v++) final[sequence_of(table[at + k]) * m.channels + channel + v] = h[v];
            }
        }
    }
}

// The map of each chunk, by a first look at what it needs: inputs and gates, or, Backward, gradients of the states and gates.  A thread
// goes over its rows as they were read, eight at a time, so little else is held.
template <class T, int V, bool Shared, bool Backward>
__global__ __launch_bounds__(kMapThreads) void recurrence_maps_kernel(Split m, const int32_t *__restrict__ first_sequence, const T *__restrict__ inputs,
                                                                      const void *__restrict__ gates, const float *__restrict__ ends,
                                                                      const int32_t *__restrict__ offsets, MapWords *__restrict__ maps) {
    constexpr int GV = Shared ? 1 : V, Threads = kMapThreads, Rows = (Backward ? kBackwardChunk : kForwardChunk) / Threads;
    extern __shared__ uint32_t table[];
    __shared__ Joint<V, Threads> joint;
    int64_t channel, gate;
    int part;
    const int64_t chunk = blockIdx.x / (uint32_t)m.tiles, tile = blockIdx.x % (uint32_t)m.tiles;
    const Place p = place_of<Threads>(m);
    const int64_t start = chunk * m.chunk_rows;
    const bool valid = column_of<V, Shared>(m, (tile << m.lanes_log2) + p.lane, channel, gate, part);
    const Column cx = column(m.channels, channel), cg = column(m.gates, gate);
    const bool wide = sizeof(T) == 4 || m.wide_gates;
    Map<V> map = unit_map<V>();
    const auto step = [&](int v, const Gate &g, float x) {
        if (Backward) map.u[v] = g.a * (map.u[v] + x);
        else map.u[v] = fmaf(g.a, map.u[v], m.complement ? g.rest * x : x);
        map.a[v] *= g.a;
    };
    const auto read = [&](auto &x, const Walk &w) {
        constexpr int K = sizeof(x) / sizeof(x[0]);
        if (inputs) {
            each_row<K>(w, cx, inputs, [&](int k, const T *from) { x[k] = load_pack<V>(from); });
        } else {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < V; v++) x[k].v[v] = (T)0.0f;
        }
    };
    if (start + m.chunk_rows <= m.rows && inside_one_sequence(m, first_sequence, offsets, chunk)) {
        constexpr int K = 8, Batches = Rows / K;
        for (int batch = 0; batch < Batches; batch++) {
            const Walk w = walk_of<K, Threads>(m, start, p.turn * Batches + (Backward ? Batches - 1 - batch : batch), K, Batches);
            Pack<T, V> x[K];
            read(x, w);
            const auto all = [&](auto &&gate_at) {
#pragma unroll
                for (int i = 0; i < K; i++) {
                    const int k = Backward ? K - 1 - i : i;
#pragma unroll
                    for (int v = 0; v < V; v++) step(v, gate_at(k, Shared ? 0 : v), x[k][v]);
                }
            };
            if (Shared && m.gate_lanes_log2 == 6) {
                // all lanes share a gate: lane k computes that of row k
                const int64_t at = (w.row + min((int)(threadIdx.x & (kWave - 1)), K - 1) * w.step) * m.gates + gate;
                const Gate own = gate_of(m.gate_form, wide ? ((const float *)gates)[at] : (float)((const T *)gates)[at]);
                all([&](int k, int) {
                    Gate g;
                    g.a = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own.a), k));
                    g.rest = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own.rest), k));
                    return g;
                });
                continue;
            }
            const auto by_type = [&](auto like) {
                Pack<decltype(like), GV> g[K];
                each_row<K>(w, cg, (const decltype(like) *)gates, [&](int k, const decltype(like) *from) { g[k] = load_pack<GV>(from); });
                if (m.gate_form == TG_GATE_VALUE) all([&](int k, int v) { return gate_of<TG_GATE_VALUE>(g[k][v]); });
                else if (m.gate_form == TG_GATE_LOG) all([&](int k, int v) { return gate_of<TG_GATE_LOG>(g[k][v]); });
                else all([&](int k, int v) { return gate_of<TG_GATE_LOGIT>(g[k][v]); });
            };
            if (wide) by_type(float());
            else by_type(T());
        }
    } else {
        constexpr int K = 8, Batches = Rows / K;
        const int places = (Threads >> m.lanes_log2) * Rows;
        chunk_table<Threads>(m, first_sequence, offsets, chunk, places, table);
        __syncthreads();
        for (int batch = 0; batch < Batches; batch++) {
            const int turn = p.turn * Batches + (Backward ? Batches - 1 - batch : batch), at = turn * K;
            const int n = (int)max((int64_t)0, min(min(m.chunk_rows, m.rows - start) - at, (int64_t)K));
            const Walk w = walk_of<K, Threads>(m, start, turn, n, Batches);
            Pack<T, V> x[K];
            float g[K][GV];
            read(x, w);
            load_gates<T, K, GV>(m, gates, w, cg, g);
            const Marks marks = marks_of(table + at, n);
#pragma unroll
            for (int i = 0; i < K; i++) {
                const int k = Backward ? K - 1 - i : i;
                const bool out = (marks.outside >> k & 1) != 0;
                if (k >= n) continue;
                if ((Backward ? marks.lasts : marks.firsts) >> k & 1) {
#pragma unroll
                    for (int v = 0; v < V; v++)
                        map.u[v] = ends && !out && valid ? ends[sequence_of(table[at + k]) * m.channels + channel + v] : 0.0f;
                    map.closed = true;
                }
                if (out) continue;
#pragma unroll
                for (int v = 0; v < V; v++) step(v, gate_of(m.gate_form, g[k][Shared ? 0 : v]), x[k][v]);
            }
        }
    }
    gather<V, Threads, Backward>(m, joint, p, map);
    if (!p.leads || !valid) return;
    Map<V> total = unit_map<V>();
    for (int i = 0; i < p.entries; i++) {
        Map<V> next = joint.at(Backward ? p.entries - 1 - i : i, 1 << m.lanes_log2, p.lane);
        compose(next, total);
        total = next;
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        MapWords words;
        words.a = total.closed ? __uint_as_float(kClosedMap) : total.a[v] != total.a[v] ? __uint_as_float(0x7fc00000u) : total.a[v];
        words.u = total.u[v];
        maps[chunk * m.channels + channel + v] = words;
    }
}

// The states that the chunks start from: the chunks' maps composed as a thread's rows are, 8 channels and 128 runs of chunks a workgroup.  A run
// of up to Ahead chunks is read at once and kept; longer ones are read again.  1094 and 2188 chunks of 384 channels, runs of 9 and 18: 24 us
// together with 24 ahead, 31 with 8; 512 chunks of 2048: 8.5 with 8, 11 with 24.
constexpr int kStartRuns = kStartThreads >> kStartLanesLog2, kStartAhead = 8, kStartFurther = 24;
template <int Ahead>
__global__ __launch_bounds__(kStartThreads) void recurrence_starts_kernel(int64_t chunks, int64_t channels, bool backward,
                                                                          const MapWords *__restrict__ maps, float *__restrict__ starts) {
    __shared__ Joint<1, kStartThreads> joint;
    Split m = {};
    m.lanes_log2 = kStartLanesLog2;
    const Place p = place_of<kStartThreads>(m);
    const int64_t channel = ((int64_t)blockIdx.x << kStartLanesLog2) + p.lane, run = (chunks + kStartRuns - 1) / kStartRuns;
    const int64_t begin = min(p.turn * run, chunks), end = min(begin + run, chunks);
    const bool valid = channel < channels;
    MapWords next[Ahead];
    const auto read = [&](int64_t i) {
#pragma unroll
        for (int k = 0; k < Ahead; k++) {
            const int64_t c = min(i + k, max(end - 1, (int64_t)0));
            next[k] = maps[(backward ? chunks - 1 - c : c) * channels + (valid ? channel : 0)];
        }
    };
    const auto over = [&](int64_t i, auto &&call) {
#pragma unroll
        for (int k = 0; k < Ahead; k++) {
            Map<1> map;
            map.closed = __float_as_uint(next[k].a) == kClosedMap;
            map.a[0] = map.closed ? 0.0f : next[k].a;
            map.u[0] = next[k].u;
            if (i + k < end) call(i + k, map);
        }
    };
    Map<1> total = unit_map<1>();
    for (int64_t i = begin; i < end; i += Ahead) {
        read(i);
        over(i, [&](int64_t, Map<1> map) {
            compose(map, total);
            total = map;
        });
    }
    float h[1] = {0.0f};
    join<1, kStartThreads, false>(m, joint, p, total, false, h);
    for (int64_t i = begin; i < end; i += Ahead) {
        if (run > Ahead) read(i);
        over(i, [&](int64_t c, const Map<1> &map) {
            if (valid) starts[(backward ? chunks - 1 - c : c) * channels + channel] = h[0];
            step_over(h, map);
        });
    }
}

// In front of a call on packed sequences: those that each chunk's rows are searched between, and the final states (or, backward, the initial
// states' gradients) of sequences without rows; the latter alone where no sequence has any.
__global__ __launch_bounds__(256) void recurrence_prepare_kernel(Split m, int32_t *__restrict__ first_sequence, const int32_t *__restrict__ offsets,
                                                                 const float *__restrict__ from, float *__restrict__ to) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    if (m.packed) {
        for (int64_t i = id; i < 2 * m.chunks; i += all) {
            const int64_t start = (i >> 1) * m.chunk_rows, place = (i & 1) ? min(start + m.chunk_rows, m.rows) - 1 : start;
            const int64_t row = m.reverse ? m.rows - 1 - place : place;
            int32_t lo = 0, hi = (int32_t)(m.sequences - 1);
            while (lo < hi) {
                const int32_t mid = lo + (hi - lo + 1) / 2;
                if (offsets[mid] <= row) lo = mid; else hi = mid - 1;
            }
            first_sequence[m.reverse ? i ^ 1 : i] = lo;
        }
    }
    if (to) {
        for (int64_t i = id; i < m.sequences * m.channels; i += all) {
            const int64_t s = i / m.channels;
            if (!m.packed || min((int64_t)offsets[s + 1], m.rows) <= max((int64_t)offsets[s], (int64_t)0)) to[i] = from ? from[i] : 0.0f;
        }
    }
}

int launch_forward(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, const float *starts, int vector, unsigned blocks,
                   hipStream_t stream) {
    return by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        using T = decltype(t);
        const auto with = [&](auto rows, auto threads) {
            constexpr int K = decltype(rows)::value, Threads = decltype(threads)::value;
            TG_LAUNCH_AS("recurrence_forward", (recurrence_forward_kernel<T, decltype(v)::value, decltype(shared)::value, K, Threads>), dim3(blocks),
                         dim3(Threads), table_bytes(m, Threads * K), stream, m, first_sequence, starts, (const T *)r.inputs, r.gates, r.initial,
                         r.offsets, (T *)r.states, r.final, m.chained ? (float *)r.kept : nullptr);
            return check_launch("tg_linear_recurrence_forward");
        };
        return m.wide ? with(std::integral_constant<int, kWideRows>(), std::integral_constant<int, kWideThreads>())
                      : with(std::integral_constant<int, kForwardRows>(), std::integral_constant<int, kForwardThreads>());
    });
}

int launch_starts(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, MapWords *maps, float *starts, int vector, bool backward,
                  hipStream_t stream) {
    const unsigned blocks = (unsigned)(m.chunks * m.tiles);
    const int code = by_layout(r.type, vector, m.shared, [&](auto t, auto v, auto shared) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        constexpr bool Shared = decltype(shared)::value;
        if (backward)
            TG_LAUNCH_AS("recurrence_maps_backward", (recurrence_maps_kernel<T, V, Shared, true>), dim3(blocks), dim3(kMapThreads), table_bytes(m, kBackwardChunk),
                         stream, m, first_sequence, (const T *)r.grad_states, r.gates, r.grad_final, r.offsets, maps);
        else
            TG_LAUNCH_AS("recurrence_maps", (recurrence_maps_kernel<T, V, Shared, false>), dim3(blocks), dim3(kMapThreads), table_bytes(m, kForwardChunk), stream,
                         m, first_sequence, (const T *)r.inputs, r.gates, r.initial, r.offsets, maps);
        return check_launch("tg_linear_recurrence");
    });
    if (code) return code;
    const dim3 grid((unsigned)ceil_div64(m.channels, 1 << kStartLanesLog2)), block(kStartThreads);
    if (m.chunks <= kStartRuns * kStartAhead)
        TG_LAUNCH_AS("recurrence_starts", recurrence_starts_kernel<kStartAhead>, grid, block, 0, stream, m.chunks, m.channels, backward, maps, starts);
    else
        TG_LAUNCH_AS("recurrence_starts", recurrence_starts_kernel<kStartFurther>, grid, block, 0, stream, m.chunks, m.channels, backward, maps, starts);
    return check_launch("tg_linear_recurrence");
}

int launch_prepare(const Split &m, int32_t *first_sequence, const int32_t *offsets, const float *from, float *to, hipStream_t stream) {
    const int64_t most = std::max(2 * m.chunks, to ? m.sequences * m.channels : 0);
    const unsigned blocks = (unsigned)std::min<int64_t>(std::max<int64_t>(ceil_div64(most, 1024), 1), 2048);
    TG_LAUNCH_AS("recurrence_prepare", recurrence_prepare_kernel, dim3(blocks), dim3(256), 0, stream, m, first_sequence, offsets, from, to);
    return check_launch("tg_linear_recurrence");
}

}  // namespace tg
#endif  // !TG_DOUBLE_PRECISION
