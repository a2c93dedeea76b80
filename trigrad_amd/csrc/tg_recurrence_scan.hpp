// tg_recurrence_scan.hpp -- how the rows and channels of a gated linear recurrence are split over threads and workgroups, and how the
// pieces are joined again (float library).
//
// A step is the map h -> a h + u; maps compose, (a2, u2) after (a1, u1) = (a2 a1, a2 u1 + u2), and a map whose sequence began within it
// does not look at what came before ("closed").  All sequences laid end to end are one axis of rows; every thread holds kRows successive
// rows of V channels in registers, so the inputs are read once.  Its map is composed
//   1. over the threads of a wave that hold other rows of the same channels (there are some where there are few channels),
//   2. over the workgroup's waves, through LDS,
//   3. over the workgroups: a chunk of rows publishes its map; the last of every kChain chunks that of their group; the last of every
//      kChain groups the state behind it.  A chunk starts from the last such state and goes over the groups and then the chunks
//      between: a fixed order of operations, so results do not depend on timing, and one wait for kChain^2 chunks in the chain from the
//      first chunk to the last.  Nothing in front of a closed map is waited for.
// Chunks are numbered by a ticket, taken when a workgroup starts, so every chunk that is waited for is running or done and waits
// only on lower ones itself.  Waits are bounded all the same: one that expires makes its chunk's states NaN.
// A published word holds its own "not there yet" (all ones, a NaN that no result has), so no fence orders a flag with its data: 8 bytes
// (map) and 4 bytes (state) are written and read whole.
#pragma once
#include <algorithm>
#include <type_traits>

#include "tg_recurrence.hpp"

namespace tg {

constexpr int kForwardThreads = 256, kForwardRows = 16;    // rows of a thread; at most 32, a bit each
constexpr int kBackwardThreads = 256, kBackwardRows = 16;
constexpr int kChain = 8;
constexpr uint32_t kAbsent = 0xffffffffu;    // not published yet
constexpr uint32_t kClosedMap = 0xfffffffeu;  // in the place of a map's factor: closed
constexpr uint32_t kWaitLimit = 1u << 20;

// Rows in the order of the recurrence ("places"): row = reverse ? rows - 1 - place : place.  Columns are lanes: a lane has V successive
// channels; the lanes of a shared gate are padded to a power of two (gate_lanes), above 64 of them it has `parts` such runs.
struct Split {
    int64_t rows, channels, gates, shared, length, sequences;
    int64_t chunks, columns, tiles;  // columns: lanes of a row, padding included
    int64_t chunk_rows;
    int64_t block_rows;              // rows between two states that are kept for the backward call
    int lanes_log2, gate_lanes_log2, parts;
    int gate_form, wide_gates;       // gates are float whatever T is
    bool complement, reverse, chained, packed;
};

// Workspace of a chained or packed call; where[] says at what byte.
struct Chain {
    uint64_t *maps;       // [chunks][tiles * lanes * V]
    uint64_t *groups;     // [chunks / kChain][tiles * lanes * V]
    uint32_t *states;     // [chunks / kChain^2][tiles * lanes * V]
    uint32_t *ticket;
    int32_t *first_sequence;  // [chunks][2] (packed): the sequences that the chunk's first and last row are searched between
};

constexpr uint8_t kFirst = 1, kLast = 2, kOutside = 4;

template <int V> struct Map {
    float a[V], u[V];
    bool closed;
};

// A factor may have left the range of float32 while the state it is applied to is 0: that stays 0.
__device__ __forceinline__ float apply(float a, float h, float u) { return h == 0.0f ? u : fmaf(a, h, u); }

template <int V> __device__ __forceinline__ void compose(Map<V> &later, const Map<V> &earlier) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        later.u[v] = later.closed ? later.u[v] : apply(later.a[v], earlier.u[v], later.u[v]);
        later.a[v] *= earlier.a[v];
    }
    later.closed = later.closed || earlier.closed;
}

__device__ __forceinline__ uint32_t word_of(float f) { return f != f ? 0x7fc00000u : __float_as_uint(f); }

template <class W> __device__ __forceinline__ W look(const W *word) {
    return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The word, once it is there; `seen` is what a look at it found.
template <class W> __device__ __forceinline__ W wait_for(const W *word, W absent, W seen, bool &expired) {
    for (uint32_t spins = 0; seen == absent && spins < kWaitLimit; spins++) {
        __builtin_amdgcn_s_sleep(1);
        seen = look(word);
    }
    if (seen == absent) expired = true;
    return seen;
}

template <int V> __device__ __forceinline__ void publish(uint64_t *words, const Map<V> &map) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        const uint32_t a = map.closed ? kClosedMap : word_of(map.a[v]);
        __hip_atomic_store(&words[v], (uint64_t)a << 32 | word_of(map.u[v]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
template <int V> __device__ __forceinline__ void publish(uint32_t *words, const float (&h)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) __hip_atomic_store(&words[v], word_of(h[v]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int V> __device__ __forceinline__ void step_over(float (&h)[V], const Map<V> &map) {
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = map.closed ? map.u[v] : apply(map.a[v], h[v], map.u[v]);
}

// What each place of the chunk is, and whose: by one thread a place.  seq[i] is in [0, sequences) wherever flags say it is used.
template <int Threads>
__device__ __forceinline__ void chunk_table(const Split &m, const Chain &c, const int32_t *offsets, int64_t chunk, int places, int32_t *seq,
                                            uint8_t *flags) {
    const int64_t start = chunk * m.chunk_rows;
    if (!m.packed) {
        const int64_t s0 = start / m.length;
        const int64_t q0 = start - s0 * m.length;
        for (int i = threadIdx.x; i < places; i += Threads) {
            int64_t q = q0 + i, s = s0;
            if (q >= m.length) {
                const uint32_t over = m.length >= m.chunk_rows ? 1u : (uint32_t)q / (uint32_t)m.length;
                s += over;
                q -= (int64_t)over * m.length;
            }
            seq[i] = (int32_t)(m.reverse ? m.sequences - 1 - s : s);
            flags[i] = start + i >= m.rows ? 0 : (q == 0 ? kFirst : 0) | (q == m.length - 1 ? kLast : 0);
        }
    } else {
        const int32_t low = c.first_sequence[2 * chunk], high = c.first_sequence[2 * chunk + 1];
        for (int i = threadIdx.x; i < places; i += Threads) {
            const int64_t place = start + i, row = m.reverse ? m.rows - 1 - place : place;
            int32_t lo = low, hi = high;  // the last sequence that begins at or in front of the row
            while (lo < hi) {
                const int32_t mid = lo + (hi - lo + 1) / 2;
                if (offsets[mid] <= row) lo = mid; else hi = mid - 1;
            }
            const int64_t begin = offsets[lo], end = offsets[lo + 1];
            seq[i] = lo;
            if (place >= m.rows) flags[i] = 0;
            else if (row < begin || row >= end) flags[i] = kFirst | kLast | kOutside;
            else flags[i] = (row == (m.reverse ? end - 1 : begin) ? kFirst : 0) | (row == (m.reverse ? begin : end - 1) ? kLast : 0);
        }
    }
}

// Whether all rows of the chunk are of one sequence that neither begins nor ends among them: no table is needed then.
__device__ __forceinline__ bool inside_one_sequence(const Split &m, const Chain &c, const int32_t *offsets, int64_t chunk) {
    const int64_t start = chunk * m.chunk_rows, end = min(start + m.chunk_rows, m.rows);
    if (!m.packed) {
        const int64_t q = start % m.length;
        return q > 0 && q + (end - start) < m.length;
    }
    const int32_t s = c.first_sequence[2 * chunk];
    const int64_t low = m.reverse ? m.rows - end : start, high = m.reverse ? m.rows - start : end;
    return s == c.first_sequence[2 * chunk + 1] && offsets[s] < low && high < offsets[s + 1];
}

// The channel and the gate of a lane's column; false: padding.
template <int V, bool Shared> __device__ __forceinline__ bool column_of(const Split &m, int64_t column, int64_t &channel, int64_t &gate, int &part) {
    part = 0;
    if (!Shared) {
        channel = gate = column * V;
        return channel < m.channels;
    }
    const uint32_t run = (uint32_t)(column >> m.gate_lanes_log2);
    const uint32_t g = run / (uint32_t)m.parts;
    part = (int)(run - g * (uint32_t)m.parts);
    const int64_t within = (((int64_t)part << m.gate_lanes_log2) + (column & ((1 << m.gate_lanes_log2) - 1))) * V;
    gate = g;
    channel = gate * m.shared + within;
    return g < m.gates && within < m.shared;
}

// K successive gates of a lane from place `first` on, GV of them a row.  Nothing behind `last` is read.
template <class T, int K, int GV>
__device__ __forceinline__ void load_gates(const Split &m, const void *gates, int64_t row, int64_t step, int64_t at, int last, float (&g)[K][GV]) {
    const int64_t pitch = m.gates * step;
    if (sizeof(T) == 4 || m.wide_gates) {
        const float *p = (const float *)gates + row * m.gates + at;
        Pack<float, GV> raw[K];
#pragma unroll
        for (int k = 0; k < K; k++) raw[k] = load_pack<GV>(p + pitch * min(k, last));
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < GV; v++) g[k][v] = raw[k].v[v];
    } else {
        const T *p = (const T *)gates + row * m.gates + at;
        Pack<T, GV> raw[K];
#pragma unroll
        for (int k = 0; k < K; k++) raw[k] = load_pack<GV>(p + pitch * min(k, last));
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < GV; v++) g[k][v] = (float)raw[k].v[v];
    }
}

// Maps that other workgroups published, in LDS: [which][lane][V].
template <int V> struct Published {
    float a[kChain * kWave * V], u[kChain * kWave * V];
    bool closed[kChain];
    template <int W> __device__ __forceinline__ Map<W> at(int i, int lanes, int lane) const {
        Map<W> r;
#pragma unroll
        for (int v = 0; v < V; v++) {
            r.a[v] = a[(i * lanes + lane) * V + v];
            r.u[v] = u[(i * lanes + lane) * V + v];
        }
        r.closed = closed[i];
        return r;
    }
};

template <int V>
__device__ __forceinline__ void settle(Published<V> &to, int i, int lanes, int lane, const uint64_t (&seen)[V], const uint64_t *words, bool &expired) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        const uint64_t w = wait_for(&words[v], ~(uint64_t)0, seen[v], expired);
        const uint32_t a = (uint32_t)(w >> 32);
        to.a[(i * lanes + lane) * V + v] = __uint_as_float(a);
        to.u[(i * lanes + lane) * V + v] = __uint_as_float((uint32_t)w);
        if (lane == 0 && v == 0) to.closed[i] = a == kClosedMap;
    }
}

// The maps of the workgroup's threads, or waves, [entry][lane][V].
template <int V, int Threads> struct Joint {
    float a[Threads * V], u[Threads * V];
    Published<V> maps, groups;
    float state[Threads * V];
    bool closed[Threads];
};

template <int V> __device__ __forceinline__ Map<V> shifted(const Map<V> &m, int lanes, bool backward) {
    Map<V> r;
#pragma unroll
    for (int v = 0; v < V; v++) {
        r.a[v] = backward ? __shfl_down(m.a[v], lanes) : __shfl_up(m.a[v], lanes);
        r.u[v] = backward ? __shfl_down(m.u[v], lanes) : __shfl_up(m.u[v], lanes);
    }
    const int c = m.closed ? 1 : 0;
    r.closed = (backward ? __shfl_down(c, lanes) : __shfl_up(c, lanes)) != 0;
    return r;
}

template <int V> __device__ __forceinline__ Map<V> unit_map() {
    Map<V> r;
#pragma unroll
    for (int v = 0; v < V; v++) {
        r.a[v] = 1.0f;
        r.u[v] = 0.0f;
    }
    r.closed = false;
    return r;
}

// Where a thread stands: lane of the row, which of the threads that hold successive rows (`turn`), and its entry in the Joint.
struct Place {
    int lane, turn, entry, entries;
    bool leads;  // one thread for each lane of a row
};
template <int Threads> __device__ __forceinline__ Place place_of(const Split &m) {
    Place p;
    const int tid = threadIdx.x, lanes = 1 << m.lanes_log2;
    p.lane = tid & (lanes - 1);
    p.turn = tid >> m.lanes_log2;
    if (m.lanes_log2 < 6) {
        p.entry = tid >> 6;
        p.entries = Threads / kWave;
        p.leads = tid < lanes;
    } else {
        p.entry = p.turn;
        p.entries = Threads >> m.lanes_log2;
        p.leads = p.turn == 0;
    }
    return p;
}

// Composes `map` over the workgroup and the chunks before: returns the state (or, backward, what reaches the last row from behind) that the
// thread's own rows start from.  known: what the chunk starts from, for a call that knows (h of the leading threads).
template <int V, int Threads, bool Backward>
__device__ __forceinline__ void join(const Split &m, const Chain &c, Joint<V, Threads> &j, const Place &p, int64_t tile, int64_t order, Map<V> map,
                                     bool chunk_closed, bool chained, const float *known, float (&h)[V]) {
    const int lanes = 1 << m.lanes_log2;
    Map<V> before = unit_map<V>();
    if (m.lanes_log2 < 6) {
        const int sub = (threadIdx.x & (kWave - 1)) >> m.lanes_log2, subs = kWave >> m.lanes_log2;
        for (int d = 1; d < subs; d <<= 1) {
            const Map<V> other = shifted(map, d << m.lanes_log2, Backward);
            if (Backward ? sub + d < subs : sub >= d) compose(map, other);
        }
        const Map<V> other = shifted(map, lanes, Backward);
        if (Backward ? sub + 1 < subs : sub >= 1) before = other;
        if (sub == (Backward ? 0 : subs - 1)) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                j.a[(p.entry * lanes + p.lane) * V + v] = map.a[v];
                j.u[(p.entry * lanes + p.lane) * V + v] = map.u[v];
            }
            if (p.lane == 0) j.closed[p.entry] = map.closed;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            j.a[threadIdx.x * V + v] = map.a[v];
            j.u[threadIdx.x * V + v] = map.u[v];
        }
        if (p.lane == 0) j.closed[p.entry] = map.closed;
    }
    __syncthreads();
    const int64_t words = m.tiles * lanes * V, at = (tile * lanes + p.lane) * V;
    if (chained) {
        const bool ends_group = order % kChain == kChain - 1, ends_super = order % (kChain * kChain) == kChain * kChain - 1;
        const int64_t group = order / kChain, super = group / kChain;
        Map<V> total = unit_map<V>();
        if (p.leads) {
            for (int i = 0; i < p.entries; i++) {
                const int e = Backward ? p.entries - 1 - i : i;
                Map<V> next;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    next.a[v] = j.a[(e * lanes + p.lane) * V + v];
                    next.u[v] = j.u[(e * lanes + p.lane) * V + v];
                }
                next.closed = j.closed[e];
                compose(next, total);
                total = next;
            }
            if (!ends_group) publish(c.maps + order * words + at, total);
            else if (total.closed && !ends_super) publish(c.groups + group * words + at, total);
            if (ends_super && total.closed) publish(c.states + super * words + at, total.u);
        }
        const int maps = (int)(order % kChain), groups = (int)(group % kChain);
        if (!chunk_closed) {
            // one look at all that may be needed, then waits for what was not there
            constexpr int Turns = Threads / kWave, Rounds = kChain / Turns + (kChain % Turns ? 1 : 0);
            const int turns = Threads >> m.lanes_log2;
            bool expired = false;
            uint64_t seen_map[Rounds][V], seen_group[Rounds][V];
            uint32_t seen_state[V];
#pragma unroll
            for (int r = 0; r < Rounds; r++) {
                const int i = p.turn + r * turns;
#pragma unroll
                for (int v = 0; v < V; v++) {
                    seen_map[r][v] = i < maps ? look(&c.maps[(group * kChain + i) * words + at + v]) : 0;
                    seen_group[r][v] = i < groups ? look(&c.groups[(super * kChain + i) * words + at + v]) : 0;
                }
            }
#pragma unroll
            for (int v = 0; v < V; v++) seen_state[v] = p.leads && super > 0 ? look(&c.states[(super - 1) * words + at + v]) : 0;
#pragma unroll
            for (int r = 0; r < Rounds; r++) {
                const int i = p.turn + r * turns;
                if (i < maps) settle<V>(j.maps, i, lanes, p.lane, seen_map[r], c.maps + (group * kChain + i) * words + at, expired);
            }
            bool failed = __syncthreads_or(expired) != 0, shut = false;
            for (int i = 0; i < maps; i++) shut = shut || j.maps.closed[i];
            if (ends_group && !ends_super && !total.closed && p.leads) {
                Map<V> all = total;
                for (int i = maps - 1; i >= 0; i--) compose(all, j.maps.template at<V>(i, lanes, p.lane));
                if (failed)
#pragma unroll
                    for (int v = 0; v < V; v++) all.u[v] = __uint_as_float(0x7fc00000u);
                publish(c.groups + group * words + at, all);
            }
            if (!shut) {
#pragma unroll
                for (int r = 0; r < Rounds; r++) {
                    const int i = p.turn + r * turns;
                    if (i < groups) settle<V>(j.groups, i, lanes, p.lane, seen_group[r], c.groups + (super * kChain + i) * words + at, expired);
                }
                failed = __syncthreads_or(expired) != 0;
            }
            if (p.leads) {
                bool open = !shut;
                if (open)
                    for (int i = 0; i < groups; i++) open = open && !j.groups.closed[i];
                expired = false;
#pragma unroll
                for (int v = 0; v < V; v++)
                    h[v] = open && super > 0 ? __uint_as_float(wait_for(&c.states[(super - 1) * words + at + v], kAbsent, seen_state[v], expired)) : 0.0f;
                if (!shut)
                    for (int i = 0; i < groups; i++) step_over(h, j.groups.template at<V>(i, lanes, p.lane));
                for (int i = 0; i < maps; i++) step_over(h, j.maps.template at<V>(i, lanes, p.lane));
                if (failed || expired)
#pragma unroll
                    for (int v = 0; v < V; v++) h[v] = __uint_as_float(0x7fc00000u);
            }
        } else if (p.leads) {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = 0.0f;
        }
        if (p.leads) {
            if (ends_super && !total.closed) {
                float end[V];
#pragma unroll
                for (int v = 0; v < V; v++) end[v] = h[v];
                step_over(end, total);
                publish(c.states + super * words + at, end);
            }
#pragma unroll
            for (int v = 0; v < V; v++) j.state[p.lane * V + v] = h[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; v++) h[v] = j.state[p.lane * V + v];
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) h[v] = known ? known[v] : 0.0f;
    }
    // through the entries before the thread's own, then through the threads before it in its wave
    const int mine = Backward ? p.entries - 1 - p.entry : p.entry;
    for (int i = 0; i < mine; i++) {
        const int e = Backward ? p.entries - 1 - i : i;
        Map<V> next;
#pragma unroll
        for (int v = 0; v < V; v++) {
            next.a[v] = j.a[(e * lanes + p.lane) * V + v];
            next.u[v] = j.u[(e * lanes + p.lane) * V + v];
        }
        next.closed = j.closed[e];
        step_over(h, next);
    }
    step_over(h, before);
}

// The workgroup's chunk in the order of the chain, and its tile of columns.  Chained: by ticket.
__device__ __forceinline__ void numbered(const Split &m, const Chain &c, uint32_t *shared, int64_t &order, int64_t &tile) {
    uint32_t id = blockIdx.x;
    if (m.chained) {
        if (threadIdx.x == 0) *shared = __hip_atomic_fetch_add(c.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        id = *shared;
    }
    order = id / (uint32_t)m.tiles;
    tile = id - (uint32_t)order * (uint32_t)m.tiles;
}

// call(T(), integral_constant V, bool_constant Shared) for a layout that split_of makes.
template <class Call> int by_layout(int64_t type, int vector, int64_t shared, Call &&call) {
    const auto by_vector = [&](auto t) {
        using one = std::integral_constant<int, 1>;
        using two = std::integral_constant<int, 2>;
        using three = std::integral_constant<int, 3>;
        if (shared == 1) return vector == 2 ? call(t, two(), std::false_type()) : call(t, one(), std::false_type());
        if (vector == 3) return call(t, three(), std::true_type());
        return vector == 2 ? call(t, two(), std::true_type()) : call(t, one(), std::true_type());
    };
    return type == TG_TYPE_F32 ? by_vector(float()) : type == TG_TYPE_F16 ? by_vector(half_t()) : by_vector(bf16_t());
}

int launch_forward(const tg_recurrence &r, const Split &m, const Chain &c, int vector, unsigned blocks, hipStream_t stream);
int launch_backward(const tg_recurrence &r, const Split &m, const Chain &c, float *partial, int vector, unsigned blocks, hipStream_t stream);
int launch_prepare(const Split &m, const Chain &c, uint64_t *words, int64_t n_words, const int32_t *offsets, const float *from, float *to,
                   hipStream_t stream);

}  // namespace tg
