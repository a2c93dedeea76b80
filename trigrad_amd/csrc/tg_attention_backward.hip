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

template <class T, int D> __global__ __launch_bounds__(4 * D) void attention_grad_queries_kernel(AttentionCall c) {
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
    Incoming<T, R, D> next_q, next_k, next_v, next_g;
    const auto load = [&](int64_t at) {
        const int64_t left = unit.count - at;
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size, c.vector);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size, c.vector);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size, c.vector);
        next_g.load(g + at * c.m.g.row, c.m.g.row, c.grad_outputs ? left : 0, c.m.value_size, c.vector);
    };
    load(0);
    if (wave == 0) reach_of<T>(c, reaches[0], unit.first, unit.count, head, before);
    int turn = 0;
    for (int64_t at = 0; at < unit.count; at += R, turn ^= 1) {
        next_q.store(queries);
        next_k.store(keys);
        next_v.store(values);
        next_g.store(grads);
        __syncthreads();
        if (at + R < unit.count) {
            load(at + R);
            if (wave == 0) reach_of<T>(c, reaches[turn ^ 1], unit.first + at + R, unit.count - at - R, head, before);
        }
        const Reach<R> &reach = reaches[turn];
#pragma unroll
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
                    put_row((T *)c.grad_queries + to, column + 4 * (lane / 16), c.m.key_size, c.vector, o);
                else
                    put_row((float *)c.grad_queries + to, column + 4 * (lane / 16), c.m.key_size, c.vector, o);
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
    if (threadIdx.x == 0) c.decays[u * c.m.heads + head] = exp2f((float)before);
}

template <class T, int D> __global__ __launch_bounds__(4 * D) void attention_grad_keys_kernel(AttentionCall c) {
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
    Incoming<T, R, D> next_q, next_k, next_v, next_g;
    const auto load = [&](int64_t at) {
        const int64_t left = unit.count - at;
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size, c.vector);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size, c.vector);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size, c.vector);
        next_g.load(g + at * c.m.g.row, c.m.g.row, c.grad_outputs ? left : 0, c.m.value_size, c.vector);
    };
    const int64_t last = (unit.count - 1) / R * R;
    load(last);
    if (wave == 0) reach_of<T>(c, reaches[0], unit.first + last, unit.count - last, head, before);
    int turn = 0;
    for (int64_t at = last; at >= 0; at -= R, turn ^= 1) {
        next_q.store(queries);
        next_k.store(keys);
        next_v.store(values);
        next_g.store(grads);
        __syncthreads();
        if (at > 0) {
            load(at - R);
            if (wave == 0) reach_of<T>(c, reaches[turn ^ 1], unit.first + at - R, R, head, before);
        }
        const Reach<R> &reach = reaches[turn];
#pragma unroll
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
                if (c.grad_values) put_row((T *)c.grad_values + here * c.m.value_size, column + 4 * (lane / 16), c.m.value_size, c.vector, x);
                if (c.grad_keys && c.m.shared == 1)
                    put_row((T *)c.grad_keys + here * c.m.key_size, column + 4 * (lane / 16), c.m.key_size, c.vector, y);
                else if (c.grad_keys)
                    put_row((float *)c.grad_keys + here * c.m.key_size, column + 4 * (lane / 16), c.m.key_size, c.vector, y);
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
        __syncthreads();
        if (threadIdx.x < R && at + threadIdx.x < unit.count) {
            float x = 0.0f;
#pragma unroll
            for (int n = 0; n < kWaves; n++) x += by_wave[n][threadIdx.x];
            c.changes[1][head * c.m.rows + unit.first + at + threadIdx.x] = x;
        }
    }
}

template <class T, int D> static int launch(const tg_attention &a, const AttentionCall &c, int which, hipStream_t stream) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, kTiles = R / 16, kWaves = D / 16;
    constexpr size_t kShared = 4 * Tile<N, R, D>::kBytes + 2 * sizeof(Reach<R>) + kWaves * R * 4;
    constexpr size_t kQueries = kShared + Tile<N, R, R>::kBytes + 2 * kTiles * R * 4, kKeys = kShared + 2 * Tile<N, R, R>::kBytes;
    static_assert(kQueries <= 160 * 1024 && kKeys <= 160 * 1024, "LDS");
    static size_t reserved[2][kMaxDevices];
    const dim3 grid((unsigned)(c.most_units * c.m.heads));
    const void *kernel = which ? (const void *)attention_grad_keys_kernel<T, D> : (const void *)attention_grad_queries_kernel<T, D>;
    const int code = reserve_lds("tg_linear_attention_backward", kernel, which ? kKeys : kQueries, reserved[which]);
    if (code) return code;
    if (which)
        TG_LAUNCH_AS("attention_grad_keys", (attention_grad_keys_kernel<T, D>), grid, dim3(4 * D), kKeys, stream, c);
    else
        TG_LAUNCH_AS("attention_grad_queries", (attention_grad_queries_kernel<T, D>), grid, dim3(4 * D), kQueries, stream, c);
    return 0;
}

int launch_attention_backward(const tg_attention &a, const AttentionCall &c, int size, int which, hipStream_t stream) {
    const auto with = [&](auto t) {
        using T = decltype(t);
        return size <= 32 ? launch<T, 32>(a, c, which, stream) : size <= 64 ? launch<T, 64>(a, c, which, stream) : launch<T, 128>(a, c, which, stream);
    };
    return a.type == TG_TYPE_F32 ? with(float()) : a.type == TG_TYPE_F16 ? with(half_t()) : with(bf16_t());
}

}  // namespace tg
#endif
