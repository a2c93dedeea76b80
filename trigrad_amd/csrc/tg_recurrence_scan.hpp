// tg_recurrence_scan.hpp -- how the rows and channels of a gated linear recurrence are split over threads and workgroups, and how the
// pieces are joined again (float library).
//
// A step is the map h -> a h + u; maps compose, (a2, u2) after (a1, u1) = (a2 a1, a2 u1 + u2), and a map whose sequence began within it
// does not look at what came before ("closed").  All sequences laid end to end are one axis of rows; every thread holds a few
// successive rows of V channels in registers.  Its map is composed
//   1. over the threads of a wave that hold other rows of the same channels (there are some where there are few channels),
//   2. over the workgroup's waves, through LDS,
//   3. over the chunks of rows that workgroups have, in three launches: the chunks' maps, from a first look at the inputs; the states that
//      the chunks start from, by going over the maps; and the chunks themselves, each from its state.  Calls whose sequences fit a chunk
//      are the third launch alone.
// The order of operations is fixed: results do not depend on timing, and no workgroup waits for another.
//
// Bound by memory traffic, and by vector instructions beside it (about 20 an element with a logistic function, 10 without).  The first look
// costs reading inputs twice (backward: gates and dh, not x).  For 32768 x 2048 in bfloat16 with a gate for every channel it takes 67 us (268 MB,
// 4.0 TB/s where a kernel that only reads reaches 5), the starting states 8, the chunks 89 (402 MB, 4.5 TB/s).  A single launch in which chunks waited
// for the maps of those before them read everything once and was no faster forward (155 us at 2.6 TB/s, and the clearing of its words) and slower
// backward (4 x 4096 x 2048, 16 gates: 148 us against 56 + 7 + 22): its chunks waited for each other, with their registers held for three
// round trips through memory more.
//
// Chunks are small, four or eight waves a SIMD's worth of workgroups beside each other, because a workgroup reads, computes and writes one after
// another: with 1024 threads, one workgroup a CU, the same backward pass took 80 us.  Chunks of half the rows again would double what the maps and
// starting states cost (24 bytes a chunk and channel).
#pragma once
#include <cfloat>
#include <algorithm>
#include <type_traits>

#include "tg_recurrence.hpp"

namespace tg {

// Rows of a thread (at most 32, a bit each) and threads; their product is a chunk's rows x lanes of a row, where there are several chunks to
// a sequence.  A forward chunk is a whole number of backward ones: the states in front of those are what the forward call keeps.
constexpr int kForwardThreads = 256, kForwardRows = 16, kForwardChunk = kForwardThreads * kForwardRows;
constexpr int kShortRows = 8, kShortThreads = 256;  // sequences of no more rows have kernels of their own
constexpr int kBackwardThreads = 256, kBackwardRows = 8, kBackwardChunk = kBackwardThreads * kBackwardRows;
constexpr int kMapThreads = 256;
constexpr int kStartThreads = 1024, kStartLanesLog2 = 3;  // of the starting states' launch: 8 channels a workgroup
// Sequences of one chunk to about four have a large workgroup each instead: no first look, no starting states, one launch.
constexpr int kWideThreads = 1024, kWideRows = 8, kWideChunk = kWideThreads * kWideRows;
static_assert(kForwardChunk % kBackwardChunk == 0 && kForwardChunk % (8 * kMapThreads) == 0 && kBackwardChunk % (8 * kMapThreads) == 0, "");
constexpr uint32_t kClosedMap = 0xfffffffeu;  // in the place of a map's factor: closed

// Rows in the order of the recurrence ("places"): row = reverse ? rows - 1 - place : place.  Columns are lanes: a lane has V successive
// channels; the lanes of a shared gate are padded to a power of two (gate_lanes), above 64 of them it has `parts` such runs.
struct Split {
    int64_t rows, channels, gates, shared, length, sequences;
    int64_t chunks, columns, tiles;  // columns: lanes of a row, padding included
    int64_t chunk_rows;
    int64_t kept_rows;               // rows between two states that the forward call keeps
    int lanes_log2, gate_lanes_log2, parts;
    int gate_form, wide_gates;       // gates are float whatever T is
    bool wide;                       // workgroups of kWideThreads
    bool complement, reverse, chained, packed;  // chained: chunks do not all begin with a sequence
};

// A word of the table of a chunk's places: its sequence, and what the place is in it.
constexpr uint32_t kSequences = 1u << 29, kFirst = 1u << 29, kLast = 1u << 30, kOutside = 1u << 31;
struct Marks {
    uint32_t firsts, lasts, outside;  // a bit for each of a thread's rows
};
__device__ __forceinline__ Marks marks_of(const uint32_t *table, int n) {
    Marks r = {0, 0, 0};
    for (int k = 0; k < n; k++) {
        const uint32_t w = table[k];
        r.firsts |= (w & kFirst ? 1u : 0u) << k;
        r.lasts |= (w & kLast ? 1u : 0u) << k;
        r.outside |= (w & kOutside ? 1u : 0u) << k;
    }
    return r;
}
__device__ __forceinline__ int64_t sequence_of(uint32_t word) { return word % kSequences; }

template <int V> struct Map {
    float a[V], u[V];
    bool closed;
};

// A factor may have left the range of float32 while the state it is applied to is 0: that stays 0.
__device__ __forceinline__ float apply(float a, float h, float u) { return h == 0.0f ? u : fmaf(a, h, u); }

// A factor that left the range as the largest number: times 0 that is 0.  (NaN becomes a number too: then the map's u is NaN.)
__device__ __forceinline__ float bounded(float a) { return __builtin_amdgcn_fmed3f(a, -FLT_MAX, FLT_MAX); }

template <int V> __device__ __forceinline__ void compose(Map<V> &later, const Map<V> &earlier) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        later.u[v] = later.closed ? later.u[v] : apply(later.a[v], earlier.u[v], later.u[v]);
        later.a[v] *= earlier.a[v];
    }
    later.closed = later.closed || earlier.closed;
}

template <int V> __device__ __forceinline__ void step_over(float (&h)[V], const Map<V> &map) {
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = map.closed ? map.u[v] : apply(map.a[v], h[v], map.u[v]);
}

// What each place of the chunk is, and whose (its sequence, in [0, sequences) for places that have one): by one thread a place.
template <int Threads>
__device__ __forceinline__ void chunk_table(const Split &m, const int32_t *first_sequence, const int32_t *offsets, int64_t chunk, int places, uint32_t *table) {
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
            const uint32_t flags = start + i >= m.rows ? 0 : (q == 0 ? kFirst : 0) | (q == m.length - 1 ? kLast : 0);
            table[i] = (uint32_t)(m.reverse ? m.sequences - 1 - s : s) % kSequences | flags;
        }
    } else {
        const int32_t low = first_sequence[2 * chunk], high = first_sequence[2 * chunk + 1];
        for (int i = threadIdx.x; i < places; i += Threads) {
            const int64_t place = start + i, row = m.reverse ? m.rows - 1 - place : place;
            int32_t lo = low, hi = high;  // the last sequence that begins at or in front of the row
            while (lo < hi) {
                const int32_t mid = lo + (hi - lo + 1) / 2;
                if (offsets[mid] <= row) lo = mid; else hi = mid - 1;
            }
            const int64_t begin = max(offsets[lo], 0), end = min((int64_t)offsets[lo + 1], m.rows);
            uint32_t flags = 0;
            if (place < m.rows) {
                if (row < begin || row >= end) flags = kFirst | kLast | kOutside;
                else flags = (row == (m.reverse ? end - 1 : begin) ? kFirst : 0) | (row == (m.reverse ? begin : end - 1) ? kLast : 0);
            }
            table[i] = (uint32_t)lo | flags;
        }
    }
}

// Whether all rows of the chunk are of one sequence that neither begins nor ends among them: no table is needed then.
__device__ __forceinline__ bool inside_one_sequence(const Split &m, const int32_t *first_sequence, const int32_t *offsets, int64_t chunk) {
    const int64_t start = chunk * m.chunk_rows, end = min(start + m.chunk_rows, m.rows);
    if (!m.packed) {
        const int64_t q = start % m.length;
        return q > 0 && q + (end - start) < m.length;
    }
    const int32_t s = first_sequence[2 * chunk];
    const int64_t low = m.reverse ? m.rows - end : start, high = m.reverse ? m.rows - start : end;
    return s == first_sequence[2 * chunk + 1] && max(offsets[s], 0) < low && high < min((int64_t)offsets[s + 1], m.rows);
}

__device__ __forceinline__ int64_t uniform(int64_t v) {  // of a wave whose lanes all have the same, or whose first lane's it is
    const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)v), high = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (int64_t)((uint64_t)high << 32 | low);
}

// The channel and the gate of a lane's column; false: padding (which no wave's first lane is unless all of its lanes are).
template <int V, bool Shared> __device__ __forceinline__ bool column_of(const Split &m, int64_t column, int64_t &channel, int64_t &gate, int &part) {
    part = 0;
    bool valid;
    if (!Shared) {
        channel = gate = column * V;
        valid = channel < m.channels;
    } else {
        const uint32_t run = (uint32_t)(column >> m.gate_lanes_log2);
        const uint32_t g = run / (uint32_t)m.parts;
        part = (int)(run - g * (uint32_t)m.parts);
        const int64_t within = (((int64_t)part << m.gate_lanes_log2) + (column & ((1 << m.gate_lanes_log2) - 1))) * V;
        gate = g;
        channel = gate * m.shared + within;
        valid = g < m.gates && within < m.shared;
    }
    // padding reads what the wave's first lane reads
    const bool any = __builtin_amdgcn_readfirstlane(valid ? 1 : 0) != 0;
    const int64_t first_channel = uniform(channel), first_gate = uniform(gate);
    if (!valid) {
        channel = any ? first_channel : 0;
        gate = any ? first_gate : 0;
    }
    return valid;
}

// Where a thread's K rows are.  Rows of a wave that has all of them are addressed from a scalar base with 32-bit offsets of the lanes: a
// row costs no vector instruction but its load.  (Lanes of a wave with several rows' threads have few channels: offsets stay small.)
struct Walk {
    int64_t row, step;       // the thread's first row; 1, or -1 where the order is reversed
    int64_t wave_row;        // the lowest of the wave's threads' first rows
    uint32_t above;          // the thread's first row, from there
    int last;                // the thread's last row, by number
    bool whole;              // all of the wave's threads have K rows
};

template <int K, int Threads> __device__ __forceinline__ Walk walk_of(const Split &m, int64_t start, int turn, int n, int batches = 1) {
    Walk w;
    const int at = turn * K, subs = m.lanes_log2 < 6 ? kWave >> m.lanes_log2 : 1;
    const int64_t place = start + (n > 0 ? at : 0);
    w.row = m.reverse ? m.rows - 1 - place : place;
    w.step = m.reverse ? -1 : 1;
    w.last = max(n - 1, 0);
    w.whole = __all(n == K);
    const int first_turn = __builtin_amdgcn_readfirstlane(turn), sub = turn - first_turn;
    const int reach = (subs - 1) * batches;  // a thread's rows are those of every batches-th turn
    w.wave_row = m.reverse ? m.rows - 1 - (start + (int64_t)(first_turn + reach) * K) : start + (int64_t)first_turn * K;
    w.above = (uint32_t)((m.reverse ? reach - sub : sub) * K);
    return w;
}

// A column of an array of `width` a row: the wave's first one, and the lane's from there.
struct Column {
    int64_t width, wave, lane;
    uint32_t offset;
};
__device__ __forceinline__ Column column(int64_t width, int64_t at) {
    Column c;
    c.width = width;
    c.lane = at;
    c.wave = uniform(at);
    c.offset = (uint32_t)(at - c.wave);
    return c;
}

// call(k, pointer to the thread's row k): rows behind the last are the last again.
template <int K, class T, class Call> __device__ __forceinline__ void each_row(const Walk &w, const Column &c, T *array, Call &&call) {
    const int64_t pitch = c.width * w.step;
    if (w.whole) {
        T *from = array + (w.wave_row * c.width + c.wave);
        const uint32_t offset = w.above * (uint32_t)c.width + c.offset;
#pragma unroll
        for (int k = 0; k < K; k++) call(k, from + pitch * k + offset);
    } else {
        T *from = array + (w.row * c.width + c.lane);
#pragma unroll
        for (int k = 0; k < K; k++) call(k, from + pitch * min(k, w.last));
    }
}

// K successive gates of a lane, GV of them a row.
template <class T, int K, int GV>
__device__ __forceinline__ void load_gates(const Split &m, const void *gates, const Walk &w, const Column &c, float (&g)[K][GV]) {
    if (sizeof(T) == 4 || m.wide_gates) {
        Pack<float, GV> raw[K];
        each_row<K>(w, c, (const float *)gates, [&](int k, const float *p) { raw[k] = load_pack<GV>(p); });
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < GV; v++) g[k][v] = raw[k].v[v];
    } else {
        Pack<T, GV> raw[K];
        each_row<K>(w, c, (const T *)gates, [&](int k, const T *p) { raw[k] = load_pack<GV>(p); });
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < GV; v++) g[k][v] = (float)raw[k].v[v];
    }
}

// The same rows from the last to the first (of a wave that has all of them).
template <int K> __device__ __forceinline__ Walk against(const Walk &w) {
    Walk b = w;
    b.row = w.row + (K - 1) * w.step;
    b.wave_row = w.wave_row + (K - 1) * w.step;
    b.step = -w.step;
    return b;
}

// The gates of a thread's rows in two steps, reading and computing.  Where all lanes of a wave share a gate, lane k reads and computes that
// of row k, for all.
template <class T, int K, int GV>
__device__ __forceinline__ void read_gates(const Split &m, const void *gates, const Walk &w, const Column &c, float (&g)[K][GV]) {
    if (GV == 1 && m.shared > 1 && m.gate_lanes_log2 == 6) {
        const int64_t at = (w.row + min((int)(threadIdx.x & (kWave - 1)), w.last) * w.step) * c.width + c.lane;
        g[0][0] = sizeof(T) == 4 || m.wide_gates ? ((const float *)gates)[at] : (float)((const T *)gates)[at];
    } else {
        load_gates<T, K, GV>(m, gates, w, c, g);
    }
}
template <int K, int GV> __device__ __forceinline__ void compute_gates(const Split &m, float (&a)[K][GV], float (&rest)[K][GV]) {
    if (GV == 1 && m.shared > 1 && m.gate_lanes_log2 == 6) {
        const Gate own = gate_of(m.gate_form, a[0][0]);
#pragma unroll
        for (int k = 0; k < K; k++) {
            a[k][0] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own.a), k));
            rest[k][0] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(own.rest), k));
        }
    } else {
        const auto all = [&](auto form) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < GV; v++) {
                    const Gate g = gate_of<decltype(form)::value>(a[k][v]);
                    a[k][v] = g.a;
                    rest[k][v] = g.rest;
                }
        };
        if (m.gate_form == TG_GATE_VALUE) all(std::integral_constant<int, TG_GATE_VALUE>());
        else if (m.gate_form == TG_GATE_LOGIT) all(std::integral_constant<int, TG_GATE_LOGIT>());
        else if (m.complement) all(std::integral_constant<int, TG_GATE_LOG>());
        else {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < GV; v++) a[k][v] = rest[k][v] = exp_real(a[k][v]);  // 1 - a is not asked for
        }
    }
}

// Sums of eight rows' values over the wave.  Each step hands half of the rows to half of the lanes, so 4 + 2 + 1 + 3 additions do what six
// for each row would; lane i ends with the sum of row i / 8.
__device__ __forceinline__ float sum_rows(float (&q)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(q[i]), __float_as_uint(q[i + 4]), false, false);
        q[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(q[i]), __float_as_uint(q[i + 2]), false, false);
        q[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const bool upper = (threadIdx.x & 8) != 0;
    const float keep = upper ? q[1] : q[0], give = upper ? q[0] : q[1];
    return sum_lanes(keep + from_lane<kRotate8>(give), 8);
}

// The maps of the workgroup's threads, or waves, [entry][lane][V].
template <int V, int Threads> struct Joint {
    float a[Threads * V], u[Threads * V];
    bool closed[Threads];
    __device__ __forceinline__ Map<V> at(int entry, int lanes, int lane) const {
        Map<V> r;
#pragma unroll
        for (int v = 0; v < V; v++) {
            r.a[v] = a[(entry * lanes + lane) * V + v];
            r.u[v] = u[(entry * lanes + lane) * V + v];
        }
        r.closed = closed[entry];
        return r;
    }
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

// Puts the threads' maps into the Joint, composed over the threads of a wave where several hold rows of the same channels, and returns the
// map of those in front of the thread in its wave.  Backward: the order is that against the rows.
template <int V, int Threads, bool Backward>
__device__ __forceinline__ Map<V> gather(const Split &m, Joint<V, Threads> &j, const Place &p, Map<V> map) {
    const int lanes = 1 << m.lanes_log2;
    Map<V> before = unit_map<V>();
    bool stores = true;
    if (m.lanes_log2 < 6) {
        const int sub = (threadIdx.x & (kWave - 1)) >> m.lanes_log2, subs = kWave >> m.lanes_log2;
        for (int d = 1; d < subs; d <<= 1) {
            const Map<V> other = shifted(map, d << m.lanes_log2, Backward);
            if (Backward ? sub + d < subs : sub >= d) compose(map, other);
        }
        const Map<V> other = shifted(map, lanes, Backward);
        if (Backward ? sub + 1 < subs : sub >= 1) before = other;
        stores = sub == (Backward ? 0 : subs - 1);
    }
    if (stores) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            j.a[(p.entry * lanes + p.lane) * V + v] = bounded(map.a[v]);
            j.u[(p.entry * lanes + p.lane) * V + v] = map.u[v];
        }
        if (p.lane == 0) j.closed[p.entry] = map.closed;
    }
    __syncthreads();
    return before;
}

// What the thread's own rows start from; h on entry is what the chunk starts from.  open: no map of the chunk is closed.
template <int V, int Threads, bool Backward>
__device__ __forceinline__ void join(const Split &m, Joint<V, Threads> &j, const Place &p, const Map<V> &map, bool open, float (&h)[V]) {
    const Map<V> before = gather<V, Threads, Backward>(m, j, p, map);
    const int mine = Backward ? p.entries - 1 - p.entry : p.entry, lanes = 1 << m.lanes_log2;
    if (open) {
        const int step = Backward ? -lanes * V : lanes * V;
        int at = ((Backward ? p.entries - 1 : 0) * lanes + p.lane) * V;
#pragma unroll 4
        for (int i = 0; i < mine; i++, at += step)
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = fmaf(j.a[at + v], h[v], j.u[at + v]);
        if (m.lanes_log2 < 6) step_over(h, before);
        return;
    }
    for (int i = 0; i < mine; i++) step_over(h, j.at(Backward ? p.entries - 1 - i : i, lanes, p.lane));
    step_over(h, before);
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

// LDS for the table of a chunk's places.
inline size_t table_bytes(const Split &m, int chunk) { return (size_t)(chunk >> m.lanes_log2) * 4; }

struct MapWords {
    float a, u;  // a: kClosedMap's bits where the map is closed
};

int launch_forward(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, const float *starts, int vector, unsigned blocks,
                   hipStream_t stream);
int launch_backward(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, const float *starts, float *partial, int vector,
                    unsigned blocks, hipStream_t stream);
// The sum of the waves' sums, where a gate has more channels than a wave.
int launch_gate_sums(const tg_recurrence &r, const Split &m, const float *partial, hipStream_t stream);
// Sequences of at most kShortRows rows, none of them of another length.
int launch_short(const tg_recurrence &r, const Split &m, float *partial, int vector, bool backward, hipStream_t stream);
int launch_prepare(const Split &m, int32_t *first_sequence, const int32_t *offsets, const float *from, float *to, hipStream_t stream);
// The states (backward: what comes from behind) that the chunks of `m` start from.
int launch_starts(const tg_recurrence &r, const Split &m, const int32_t *first_sequence, MapWords *maps, float *starts, int vector, bool backward,
                  hipStream_t stream);

}  // namespace tg
