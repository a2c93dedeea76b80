// tg_attention_backward.hip -- linear attention by chunks, backward: dq from the first chunk of a unit to its last, dk and dv from the last to the first.
//
// Both states are at hand in one chunk only if one of them is written out for every chunk, 64 KB a head and chunk of 16 KB tensors.  So the
// queries' gradients go with S, the keys' and values' with D, each over units whose first S the forward pass kept and whose last D is made of what
// the first of the two kernels adds up on its way.  dlog a is by row what <S_t, D_t> changes by, k.dk - q.dq without the pair of a row and itself, from
// <S, D> in front of the unit on: sums of at most a unit's rows, so that little is lost where they cancel.
#ifndef TG_DOUBLE_PRECISION
#include "tg_attention_chunk.hpp"

namespace tg {

// The sum over the lanes that hold the same row: 16, 32 and 48 on.
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

template <class T, int D, bool Vector> __global__ __launch_bounds__(4 * D) void attention_grad_queries_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, kTiles = R / 16, kWaves = D / 16;
    using In = Tile<N, R, D>;
    using Pairs = Tile<N, R, R>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const In queries{(__bf16 *)lds}, keys{(__bf16 *)(lds + In::kBytes)}, values{(__bf16 *)(lds + 2 * In::kBytes)}, grads{(__bf16 *)(lds + 3 * In::kBytes)};
    const Pairs pairs{(__bf16 *)(lds + 4 * In::kBytes)};
    Reach<R> *reaches = (Reach<R> *)(lds + 4 * In::kBytes + Pairs::kBytes);
    float(*by_wave)[R] = (float(*)[R])(reaches + 2);  // q.dq without the chunk's own pairs, of each wave's columns
    float(*by_later)[R] = by_wave + kWaves;           // by row s, of each tile's pairs
    float(*by_earlier)[R] = by_later + kTiles;        // by row r
    const int64_t u = blockIdx.x / c.m.heads;
    const int head = (int)(blockIdx.x % c.m.heads), lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, column = 16 * wave;
    const int64_t state_size = (int64_t)c.m.key_size * c.m.value_size;
    const Unit unit = unit_of<R>(c, u);
    if (!unit.there) return;
    const AttentionRows rows = rows_of(c.m, c.offsets, unit.sequence);
    const T *q = (const T *)c.queries + place_of(c.m, c.m.q, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.q.row,
            *k = (const T *)c.keys + place_of(c.m, c.m.k, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.k.row,
            *v = (const T *)c.values + place_of(c.m, c.m.v, unit.sequence, rows.first, head) + unit.base * c.m.v.row,
            *g = (const T *)c.grad_outputs + place_of(c.m, c.m.g, unit.sequence, rows.first, head) + unit.base * c.m.g.row;
    State<D> state, change = {};  // rows are values, columns keys
    state.template load<true>(c.states + (u * c.m.heads + head) * state_size, column, c.m.key_size, c.m.value_size);
    double before = 0.0;
    Incoming<T, R, D, Vector> next_q, next_k, next_v, next_g;
    const auto load = [&](int64_t at) {
        const int64_t left = unit.count - at;
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size);
        next_g.load(g + at * c.m.g.row, c.m.g.row, left, c.m.value_size);
    };
    load(0);
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first, unit.count, head), unit.count, before);
    int turn = 0;
    for (int64_t at = 0; at < unit.count; at += R, turn ^= 1) {
        next_q.store(queries, unit.count - at, c.m.key_size);
        next_k.store(keys, unit.count - at, c.m.key_size);
        next_v.store(values, unit.count - at, c.m.value_size);
        next_g.store(grads, c.grad_outputs_there ? unit.count - at : 0, c.m.value_size);
        __syncthreads();
        if (at + R < unit.count) {
            load(at + R);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at + R, unit.count - at - R, head);
        }
        const Reach<R> &reach = reaches[turn];
#pragma unroll 1
        for (int n = 0; n < (kTiles * kTiles + kWaves - 1) / kWaves; n++) {
            const int tile = wave + n * kWaves, s = tile / kTiles, r = tile % kTiles;
            if (tile >= kTiles * kTiles) continue;
            floatx4 p = {0.0f, 0.0f, 0.0f, 0.0f}, d = p;
            if (r <= s) {
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    p = product(keys.straight(16 * r, i), queries.straight(16 * s, i), p);
                    d = product(values.straight(16 * r, i), grads.straight(16 * s, i), d);
                }
                d *= decays_of<true>(reach, 16 * r, 16 * s, c.m.scale);
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] = 16 * s + lane % 16 > 16 * r + 4 * (lane / 16) + j ? p[j] * d[j] : 0.0f;
            }
            if (r <= (s | 1)) pairs.put(16 * s, 16 * r, d);
            const float later = sum_groups(p[0] + p[1] + p[2] + p[3]);
            if (lane < 16) by_later[r][16 * s + lane] = later;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float earlier = sum_lanes(p[j], 16);
                if (lane % 16 == 0) by_earlier[s][16 * r + 4 * (lane / 16) + j] = earlier;
            }
        }
        Operand<N> mine[R / 32];
#pragma unroll
        for (int n = 0; n < R / 32; n++) mine[n] = keys.transposed(32 * n, column);
        floatx4 read[kTiles] = {};
        state.template read_by<kWhole>(grads, read);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kTiles; s++) {
            floatx4 o = read[s];
            o *= reach.row[16 * s + lane % 16];
            const floatx4 x = queries.numbers(16 * s + lane % 16, column + 4 * (lane / 16));
            const float sum = sum_groups(o[0] * x[0] + o[1] * x[1] + o[2] * x[2] + o[3] * x[3]);
            if (lane < 16) by_wave[wave][16 * s + lane] = sum;
#pragma unroll
            for (int n = 0; n < R / 32; n++)
                if (2 * n <= s) o = product(mine[n], pairs.chained(16 * s, 32 * n), o);
            const int64_t row = at + 16 * s + lane % 16;
            if (row < unit.count && c.grad_queries) {
                const int64_t to = ((unit.first + row) * c.m.heads + head) * c.m.key_size;
                if (c.m.shared == 1)
                    put_row((T *)c.grad_queries + to, column + 4 * (lane / 16), c.m.key_size, Vector, o);
                else
                    put_row((float *)c.grad_queries + to, column + 4 * (lane / 16), c.m.key_size, Vector, o);
            }
        }
        Operand<kWhole> late[R / 32];
#pragma unroll
        for (int n = 0; n < R / 32; n++) late[n] = weighted<kWhole>(mine[n], reach.column, 32 * n);
        state.times(reach.whole);
        state.add(values, late);
#pragma unroll
        for (int n = 0; n < R / 32; n++) late[n] = weighted<kWhole>(queries.transposed(32 * n, column), reach.start, 32 * n);
        change.add(grads, late);
        if (wave == 0 && at + R < unit.count) reach_of(c, reaches[turn ^ 1], gate, unit.count - at - R, before);
        __syncthreads();
        if (threadIdx.x < R && at + threadIdx.x < unit.count) {
            float x = 0.0f;
#pragma unroll
            for (int n = 0; n < kTiles; n++) x += by_later[n][threadIdx.x] - by_earlier[n][threadIdx.x];
#pragma unroll
            for (int n = 0; n < kWaves; n++) x += by_wave[n][threadIdx.x];
            c.changes[0][head * c.m.rows + unit.first + at + threadIdx.x] = x;
        }
    }
    change.template store<true>(c.grad_states + (u * c.m.heads + head) * state_size, column, c.m.key_size, c.m.value_size);
    if (threadIdx.x == 0) c.decays[u * c.m.heads + head] = power_of_two((float)before);
}

template <class T, int D, bool Vector> __global__ __launch_bounds__(4 * D) void attention_grad_keys_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, M = Parts<T>::kState, kTiles = R / 16, kWaves = D / 16;
    using In = Tile<N, R, D>;
    using Pairs = Tile<N, R, R>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const In queries{(__bf16 *)lds}, keys{(__bf16 *)(lds + In::kBytes)}, values{(__bf16 *)(lds + 2 * In::kBytes)}, grads{(__bf16 *)(lds + 3 * In::kBytes)};
    const Pairs scores{(__bf16 *)(lds + 4 * In::kBytes)}, pairs{(__bf16 *)(lds + 4 * In::kBytes + Pairs::kBytes)};
    Reach<R> *reaches = (Reach<R> *)(lds + 4 * In::kBytes + 2 * Pairs::kBytes);
    float(*by_wave)[R] = (float(*)[R])(reaches + 2);  // k.dk without the chunk's own pairs, of each wave's columns
    const int64_t u = blockIdx.x / c.m.heads;
    const int head = (int)(blockIdx.x % c.m.heads), lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, column = 16 * wave;
    const int64_t state_size = (int64_t)c.m.key_size * c.m.value_size;
    const Unit unit = unit_of<R>(c, u);
    if (!unit.there || unit.count == 0) return;
    const AttentionRows rows = rows_of(c.m, c.offsets, unit.sequence);
    const T *q = (const T *)c.queries + place_of(c.m, c.m.q, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.q.row,
            *k = (const T *)c.keys + place_of(c.m, c.m.k, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.k.row,
            *v = (const T *)c.values + place_of(c.m, c.m.v, unit.sequence, rows.first, head) + unit.base * c.m.v.row,
            *g = (const T *)c.grad_outputs + place_of(c.m, c.m.g, unit.sequence, rows.first, head) + unit.base * c.m.g.row;
    State<D> state, turned;  // D: rows are keys and columns values, and the other way round
    const float *behind = c.grad_states + (u * c.m.heads + head) * state_size;
    state.template load<false>(behind, column, c.m.key_size, c.m.value_size);
    turned.template load<true>(behind, column, c.m.key_size, c.m.value_size);
    double before = 0.0;
    Incoming<T, R, D, Vector> next_q, next_k, next_v, next_g;
    const auto load = [&](int64_t at) {
        const int64_t left = unit.count - at;
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size);
        next_g.load(g + at * c.m.g.row, c.m.g.row, left, c.m.value_size);
    };
    const int64_t last = (unit.count - 1) / R * R;
    load(last);
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first + last, unit.count - last, head), unit.count - last, before);
    int turn = 0;
    for (int64_t at = last; at >= 0; at -= R, turn ^= 1) {
        next_q.store(queries, unit.count - at, c.m.key_size);
        next_k.store(keys, unit.count - at, c.m.key_size);
        next_v.store(values, unit.count - at, c.m.value_size);
        next_g.store(grads, c.grad_outputs_there ? unit.count - at : 0, c.m.value_size);
        __syncthreads();
        if (at > 0) {
            load(at - R);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at - R, R, head);
        }
        const Reach<R> &reach = reaches[turn];
#pragma unroll 1
        for (int n = 0; n < (kTiles * kTiles + kWaves - 1) / kWaves; n++) {
            const int tile = wave + n * kWaves, r = tile / kTiles, s = tile % kTiles;
            if (tile >= kTiles * kTiles || (s | 1) < r) continue;
            floatx4 p = {0.0f, 0.0f, 0.0f, 0.0f}, d = p;
            if (s >= r) {
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    p = product(queries.straight(16 * s, i), keys.straight(16 * r, i), p);
                    d = product(grads.straight(16 * s, i), values.straight(16 * r, i), d);
                }
                const floatx4 decay = decays_of<false>(reach, 16 * s, 16 * r, c.m.scale);
                p *= decay;
                d *= decay;
            }
            scores.put(16 * r, 16 * s, p);
            pairs.put(16 * r, 16 * s, d);
        }
        Operand<N> mine_g[R / 32], mine_q[R / 32];
#pragma unroll
        for (int n = 0; n < R / 32; n++) {
            mine_g[n] = grads.transposed(32 * n, column);
            mine_q[n] = queries.transposed(32 * n, column);
        }
        floatx4 read_x[kTiles] = {}, read_y[kTiles] = {};
        state.template read_by<M>(keys, read_x);
        turned.template read_by<kWhole>(values, read_y);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kTiles; r++) {
            floatx4 x = read_x[r], y = read_y[r];
            const float decay = reach.column[16 * r + lane % 16];
            x *= decay;
            y *= decay;
            const floatx4 own = keys.numbers(16 * r + lane % 16, column + 4 * (lane / 16));
            const float sum = sum_groups(y[0] * own[0] + y[1] * own[1] + y[2] * own[2] + y[3] * own[3]);
            if (lane < 16) by_wave[wave][16 * r + lane] = sum;
#pragma unroll
            for (int n = 0; n < R / 32; n++)
                if (2 * n + 1 >= r) {
                    x = product(mine_g[n], scores.chained(16 * r, 32 * n), x);
                    y = product(mine_q[n], pairs.chained(16 * r, 32 * n), y);
                }
            const int64_t row = at + 16 * r + lane % 16;
            if (row < unit.count) {
                const int64_t here = (unit.first + row) * c.m.heads + head;
                if (c.grad_values) put_row((T *)c.grad_values + here * c.m.value_size, column + 4 * (lane / 16), c.m.value_size, Vector, x);
                if (c.grad_keys && c.m.shared == 1)
                    put_row((T *)c.grad_keys + here * c.m.key_size, column + 4 * (lane / 16), c.m.key_size, Vector, y);
                else if (c.grad_keys)
                    put_row((float *)c.grad_keys + here * c.m.key_size, column + 4 * (lane / 16), c.m.key_size, Vector, y);
            }
        }
        Operand<kWhole> late[R / 32];
#pragma unroll
        for (int n = 0; n < R / 32; n++) late[n] = weighted<kWhole>(mine_g[n], reach.row, 32 * n);
        state.times(reach.whole);
        state.add(queries, late);
#pragma unroll
        for (int n = 0; n < R / 32; n++) late[n] = weighted<kWhole>(mine_q[n], reach.row, 32 * n);
        turned.times(reach.whole);
        turned.add(grads, late);
        if (wave == 0 && at > 0) reach_of(c, reaches[turn ^ 1], gate, R, before);
        __syncthreads();
        if (threadIdx.x < R && at + threadIdx.x < unit.count) {
            float x = 0.0f;
#pragma unroll
            for (int n = 0; n < kWaves; n++) x += by_wave[n][threadIdx.x];
            c.changes[1][head * c.m.rows + unit.first + at + threadIdx.x] = x;
        }
    }
}

int launch_attention_backward(int64_t type, const AttentionCall &c, int size, bool for_keys, hipStream_t stream) {
    return by_attention_kernel(type, size, c.vector, [&](auto t, auto d, auto vector) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value, R = Parts<T>::kRows, N = Parts<T>::kInput, kTiles = R / 16, kWaves = D / 16;
        constexpr bool Vector = decltype(vector)::value;
        constexpr size_t kShared = 4 * Tile<N, R, D>::kBytes + 2 * sizeof(Reach<R>) + kWaves * R * 4;
        constexpr size_t kQueries = kShared + Tile<N, R, R>::kBytes + 2 * kTiles * R * 4, kKeys = kShared + 2 * Tile<N, R, R>::kBytes;
        static_assert(kQueries <= 160 * 1024 && kKeys <= 160 * 1024, "LDS");
        static size_t reserved[2][kMaxDevices];
        const dim3 grid((unsigned)(c.most_units * c.m.heads));
        const void *kernel = for_keys ? (const void *)attention_grad_keys_kernel<T, D, Vector> : (const void *)attention_grad_queries_kernel<T, D, Vector>;
        const int code = reserve_lds("tg_linear_attention_backward", kernel, for_keys ? kKeys : kQueries, reserved[for_keys]);
        if (code) return code;
        if (for_keys)
            TG_LAUNCH_AS("attention_grad_keys", (attention_grad_keys_kernel<T, D, Vector>), grid, dim3(4 * D), kKeys, stream, c);
        else
            TG_LAUNCH_AS("attention_grad_queries", (attention_grad_queries_kernel<T, D, Vector>), grid, dim3(4 * D), kQueries, stream, c);
        return 0;
    });
}

}  // namespace tg
#endif
