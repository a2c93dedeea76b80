// tg_attention_forward.hip -- linear attention by chunks, forward: what units of chunks add to the state, and the outputs.
#ifndef TG_DOUBLE_PRECISION
#include "tg_attention_chunk.hpp"

namespace tg {

template <class T, int D> constexpr int kStatesLds = 2 * Tile<typename Parts<T>::Element, Parts<T>::kInput, Parts<T>::kRows, D>::kBytes + 2 * (int)sizeof(Reach<Parts<T>::kRows>);
template <class T, int D> constexpr int kOutputsLds = 3 * Tile<typename Parts<T>::Element, Parts<T>::kInput, Parts<T>::kRows, D>::kBytes +
                                                      PairsOf<T>::kBytes + 2 * (int)sizeof(Reach<Parts<T>::kRows>);
constexpr int W = 1;  // see State
template <int D> constexpr int kThreads = State<D, W>::kWaves * kWave;

// What a unit adds to the state, and its decay.  A chunk is on its way from memory while the one before is computed on.  32768 rows of 16 heads of 128
// in bfloat16: 73 us, 3.7 TB/s; weighted values in three parts are what it computes.
template <class T, int D, bool Vector>
__global__ __launch_bounds__(kThreads<D>, waves_of_simd(kThreads<D>, kStatesLds<T, D>, W * D / 4)) void attention_states_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput;
    using E = typename Parts<T>::Element;
    using In = Tile<E, N, R, D>;
    __shared__ __attribute__((aligned(16))) E lds[In::kBytes];
    __shared__ Reach<R> reaches[2];
    const int64_t u = blockIdx.x / c.m.heads;
    const int head = (int)(blockIdx.x % c.m.heads), wave = wave_of(), column = 16 * W * wave;
    const Unit unit = unit_of<R>(c, u);
    if (!unit.there) return;
    const AttentionRows rows = rows_of(c.m, c.offsets, unit.sequence);
    const T *k = (const T *)c.keys + place_of(c.m, c.m.k, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.k.row,
            *v = (const T *)c.values + place_of(c.m, c.m.v, unit.sequence, rows.first, head) + unit.base * c.m.v.row;
    State<D, W> state = {};
    double before = 0.0;
    Incoming<T, R, D, kThreads<D>, Vector> next_k, next_v;
    if (unit.count > 0) {
        next_k.load(k, c.m.k.row, unit.count, c.m.key_size);
        next_v.load(v, c.m.v.row, unit.count, c.m.value_size);
    }
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first, unit.count, head), unit.count, before);
    int turn = 0;
    for (int64_t at = 0; at < unit.count; at += R, turn ^= 1) {
        const int lane = lane_of_turn();
        const In keys{lds, lane}, values{lds + In::kBytes / 2, lane};
        next_k.template store<E, N>(keys, unit.count - at, c.m.key_size);
        next_v.template store<E, N>(values, unit.count - at, c.m.value_size);
        __syncthreads();
        if (at + R < unit.count) {
            next_k.load(k + (at + R) * c.m.k.row, c.m.k.row, unit.count - at - R, c.m.key_size);
            next_v.load(v + (at + R) * c.m.v.row, c.m.v.row, unit.count - at - R, c.m.value_size);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at + R, unit.count - at - R, head);
        }
        Operand<E, N> mine[R / 32][W];
        columns_of(values, column, mine);
        state.template fold<T, kFoldApart<T, D, W, true>>(reaches[turn].whole, keys, mine, reaches[turn].column);
        if (wave == 0 && at + R < unit.count) reach_of(c, reaches[turn ^ 1], gate, unit.count - at - R, before);
        __syncthreads();
    }
    state.template store<false>(c.states + (u * c.m.heads + head) * c.m.key_size * c.m.value_size, column, c.m.key_size, c.m.value_size);
    if (threadIdx.x == 0) c.decays[u * c.m.heads + head] = power_of_two((float)before);
}

// The outputs, from the states in front of the units, or through whole sequences.  A state is read through its accumulators, the pairs of a chunk
// through LDS.  32768 rows of 16 heads of 128 in bfloat16: 164 us, 3.3 TB/s; instructions that make a state's parts and the decays of pairs bound it.
template <class T, int D, bool Vector>
__global__ __launch_bounds__(kThreads<D>, waves_of_simd(kThreads<D>, kOutputsLds<T, D>, W * D / 4)) void attention_outputs_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, M = Parts<T>::kState, kTiles = R / 16, kWaves = State<D, W>::kWaves;
    using E = typename Parts<T>::Element;
    using In = Tile<E, N, R, D>;
    using Pairs = PairsOf<T>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Reach<R> *reaches = (Reach<R> *)(lds + 3 * In::kBytes + Pairs::kBytes);
    const int64_t which = blockIdx.x / c.m.heads;  // a unit, or a sequence
    const int head = (int)(blockIdx.x % c.m.heads), wave = wave_of(), column = 16 * W * wave;
    const int64_t state_size = (int64_t)c.m.key_size * c.m.value_size;
    Unit unit;
    int64_t u = which;
    if (c.through) {
        const AttentionRows rows = rows_of(c.m, c.offsets, which);
        unit = {which, 0, rows.first, rows.count, 0, true};
        u = c.m.packed ? (c.states ? c.plan[c.most_units + which] : 0) : which * c.units;
    } else {
        unit = unit_of<R>(c, which);
    }
    if (!unit.there) return;
    const AttentionRows rows = rows_of(c.m, c.offsets, unit.sequence);
    const T *q = (const T *)c.queries + place_of(c.m, c.m.q, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.q.row,
            *k = (const T *)c.keys + place_of(c.m, c.m.k, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.k.row,
            *v = (const T *)c.values + place_of(c.m, c.m.v, unit.sequence, rows.first, head) + unit.base * c.m.v.row;
    T *out = (T *)c.outputs + (unit.first * c.m.heads + head) * c.m.value_size;
    const int64_t out_row = (int64_t)c.m.heads * c.m.value_size;
    State<D, W> state;
    const float *start = c.through ? (c.initial ? c.initial + (unit.sequence * c.m.heads + head) * state_size : nullptr)
                                   : c.states + (u * c.m.heads + head) * state_size;
    state.template load<false>(start, column, c.m.key_size, c.m.value_size);
    double before = 0.0;
    Incoming<T, R, D, kThreads<D>, Vector> next_q, next_k, next_v;
    const auto load = [&](int64_t at) {
        const int64_t left = unit.count - at;
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size);
    };
    if (unit.count > 0) load(0);
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first, unit.count, head), unit.count, before);
    int turn = 0, chunk = 0;
    for (int64_t at = 0; at < unit.count; at += R, turn ^= 1) {
        const int lane = lane_of_turn();
        const In queries{(E *)lds, lane}, keys{(E *)(lds + In::kBytes), lane}, values{(E *)(lds + 2 * In::kBytes), lane};
        const Pairs pairs{(E *)(lds + 3 * In::kBytes), lane};
        if (c.through && c.states && chunk == 0) {
            if (u < c.most_units) state.template store<false>(c.states + (u * c.m.heads + head) * state_size, column, c.m.key_size, c.m.value_size);
            u++;
        }
        chunk = chunk + 1 == c.chunks ? 0 : chunk + 1;
        next_q.template store<E, N>(queries, unit.count - at, c.m.key_size);
        next_k.template store<E, N>(keys, unit.count - at, c.m.key_size);
        next_v.template store<E, N>(values, unit.count - at, c.m.value_size);
        __syncthreads();
        if (at + R < unit.count) {
            load(at + R);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at + R, unit.count - at - R, head);
        }
        const Reach<R> &reach = reaches[turn];
        // pairs: row s, column r
        const int all_tiles = tiles_of_chunk<T>(kWaves);
#pragma unroll 1
        for (int tiles = wave; tiles < all_tiles; tiles += kWaves) {
            const int s = tiles * kAcross<T> / kTiles, first = tiles * kAcross<T> % kTiles;
            if (first > (s | 1)) continue;
            floatx4 p[kAcross<T>] = {};
#pragma unroll
            for (int a = 0; a < kAcross<T>; a++) {
                const int r = first + a;
                if (r > s) continue;
#pragma unroll
                for (int i = 0; i < D; i += 32) p[a] = product(keys.straight(16 * r, i), queries.straight(16 * s, i), p[a]);
                p[a] *= decays_of<true>(reach, 16 * r, 16 * s, c.m.scale, lane);
            }
            put_pairs<T>(pairs, 16 * s, 16 * first, p);
        }
        floatx4 read[kTiles][W] = {};
        float down[W];
        state.template read_by<T, M>(queries, read, down);
        __syncthreads();
        Operand<E, N> mine[R / 32][W];
        columns_of(values, column, mine);
        each_of<kTiles>([&](auto number) {
            constexpr int s = decltype(number)::value;
            scale_read<T>(read[s], reach.row[16 * s + lane % 16], down, lane);
            add_pairs<T, 0, s / 2 + 1>(pairs, 16 * s, mine, read[s]);
            in_order();
            const int to = column + 4 * (lane / 16);
            if (16 * s + lane % 16 < unit.count - at) {
#pragma unroll
                for (int w = 0; w < W; w++)
                    put_row(out + (at + 16 * s) * out_row + 16 * w, (uint32_t)(lane % 16 * (int)out_row + to), to + 16 * w, c.m.value_size, Vector, read[s][w]);
            }
        });
        state.template fold<T, kFoldApart<T, D, W, true>>(reach.whole, keys, mine, reach.column);
        if (wave == 0 && at + R < unit.count) reach_of(c, reaches[turn ^ 1], gate, unit.count - at - R, before);
        __syncthreads();
    }
#pragma unroll 1
    for (float *to = c.through ? c.final : nullptr; to; to = to == c.final ? c.finals : nullptr)
        state.template store<false>(to + (unit.sequence * c.m.heads + head) * state_size, column, c.m.key_size, c.m.value_size);
}

int launch_attention_forward(int64_t type, const AttentionCall &c, int size, bool states_only, hipStream_t stream) {
    return by_attention_kernel(type, size, c.vector, [&](auto t, auto d, auto vector) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool Vector = decltype(vector)::value;
        const dim3 grid((unsigned)((c.through ? c.m.sequences : c.most_units) * c.m.heads));
        if (states_only) {
            TG_LAUNCH_AS("attention_states", (attention_states_kernel<T, D, Vector>), grid, dim3(kThreads<D>), 0, stream, c);
            return 0;
        }
        constexpr int kBytes = kOutputsLds<T, D>;
        static size_t reserved[kMaxDevices];
        const int code = reserve_lds("tg_linear_attention_forward", (const void *)attention_outputs_kernel<T, D, Vector>, kBytes, reserved);
        if (code) return code;
        TG_LAUNCH_AS("attention_outputs", (attention_outputs_kernel<T, D, Vector>), grid, dim3(kThreads<D>), kBytes, stream, c);
        return 0;
    });
}

}  // namespace tg
#endif
