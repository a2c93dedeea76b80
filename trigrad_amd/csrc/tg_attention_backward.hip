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

// The two kernels have twice the waves of a state: the first half (`role` 0) has one state, the second half the other.  LDS, and waves of a SIMD that
// they are compiled for: two, with 256 registers, where LDS has room for one workgroup.
//
// W of State, 4 x 4096 rows of 16 heads of 128 in bfloat16, and 2 x 3000 of 8 in float32: the queries' kernel 183 and 82 us with one, 197 and 60 with
// two; the keys' 300 and 87 with one, 198 and 64 with two.  8 x 2048 rows of 32 heads of 64: 136 and 137 with one, 170 and 156 with two.  In float16,
// whose scalings take registers, the first of these forward and backward: 539 with one in the queries' kernel, 512 with two.
// Instructions bound both: making parts, matrix instructions and readings of LDS take a third to a half of the time each and hardly overlap, as all
// waves of a workgroup are in the same phase (1.8 TB/s of memory for heads of 128, 2.5 for those of 64).
template <class T, int D> constexpr int kQueriesColumns = D > 64 && (sizeof(T) == 4 || Parts<T>::kScaled) ? 2 : 1;
template <int D> constexpr int kKeysColumns = D > 64 ? 2 : 1;
template <class T, int D> constexpr int kQueriesThreads = 2 * State<D, kQueriesColumns<T, D>>::kWaves * kWave;
template <int D> constexpr int kKeysThreads = 2 * State<D, kKeysColumns<D>>::kWaves * kWave;
template <class T, int D> constexpr int kBackwardLds = 4 * Tile<typename Parts<T>::Element, Parts<T>::kInput, Parts<T>::kRows, D>::kBytes + 2 * (int)sizeof(Reach<Parts<T>::kRows>) +
                                                       D / 16 * Parts<T>::kRows * 4;
template <class T, int D> constexpr int kQueriesLds = kBackwardLds<T, D> + PairsOf<T>::kBytes + 2 * Parts<T>::kRows / 16 * Parts<T>::kRows * 4;
template <class T, int D> constexpr int kKeysLds = kBackwardLds<T, D> + 2 * PairsOf<T>::kBytes;

// The chunks of a unit's tensors on their way to LDS.
template <class T, int D, int Threads, bool Vector> struct Four {
    static constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput;
    const T *q, *k, *v, *g;
    Incoming<T, R, D, Threads, Vector> next_q, next_k, next_v, next_g;

    __device__ __forceinline__ Four(const AttentionCall &c, const Unit &unit, int head) {
        const AttentionRows rows = rows_of(c.m, c.offsets, unit.sequence);
        q = (const T *)c.queries + place_of(c.m, c.m.q, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.q.row;
        k = (const T *)c.keys + place_of(c.m, c.m.k, unit.sequence, rows.first, head / c.m.shared) + unit.base * c.m.k.row;
        v = (const T *)c.values + place_of(c.m, c.m.v, unit.sequence, rows.first, head) + unit.base * c.m.v.row;
        g = (const T *)c.grad_outputs + place_of(c.m, c.m.g, unit.sequence, rows.first, head) + unit.base * c.m.g.row;
    }
    __device__ __forceinline__ void load(const AttentionCall &c, int64_t at, int64_t left) {
        next_q.load(q + at * c.m.q.row, c.m.q.row, left, c.m.key_size);
        next_k.load(k + at * c.m.k.row, c.m.k.row, left, c.m.key_size);
        next_v.load(v + at * c.m.v.row, c.m.v.row, left, c.m.value_size);
        next_g.load(g + at * c.m.g.row, c.m.g.row, left, c.m.value_size);
    }
    template <class Tile> __device__ __forceinline__ void store(const AttentionCall &c, const Tile &queries, const Tile &keys, const Tile &values, const Tile &grads,
                                                                int64_t left) const {
        using E = typename Parts<T>::Element;
        next_q.template store<E, N>(queries, left, c.m.key_size);
        next_k.template store<E, N>(keys, left, c.m.key_size);
        next_v.template store<E, N>(values, left, c.m.value_size);
        next_g.template store<E, N>(grads, c.grad_outputs_there ? left : 0, c.m.value_size);
    }
};

// dq, what changes dlog a from q.dq and the pairs, and what the unit adds to D.
template <class T, int D, bool Vector>
__global__ __launch_bounds__((kQueriesThreads<T, D>), (waves_of_simd(kQueriesThreads<T, D>, kQueriesLds<T, D>, kQueriesColumns<T, D> * D / 4))) void attention_grad_queries_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, kTiles = R / 16, W = kQueriesColumns<T, D>, kWaves = State<D, W>::kWaves;
    using E = typename Parts<T>::Element;
    using In = Tile<E, N, R, D>;
    using Pairs = PairsOf<T>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Reach<R> *reaches = (Reach<R> *)(lds + 4 * In::kBytes + Pairs::kBytes);
    float(*by_wave)[R] = (float(*)[R])(reaches + 2);  // q.dq without the chunk's own pairs, of each wave's columns
    float(*by_later)[R] = by_wave + kWaves;           // by row s, of each tile's pairs
    float(*by_earlier)[R] = by_later + kTiles;        // by row r
    const int64_t u = blockIdx.x / c.m.heads;
    const int head = (int)(blockIdx.x % c.m.heads), wave = wave_of();
    const int role = wave / kWaves, column = 16 * W * (wave % kWaves);
    const int64_t state_size = (int64_t)c.m.key_size * c.m.value_size;
    const Unit unit = unit_of<R>(c, u);
    if (!unit.there) return;
    // rows are values, columns keys: S, which the queries' gradients read, or what the unit adds to D
    State<D, W> state;
    state.template load<true>(role == 0 ? c.states + (u * c.m.heads + head) * state_size : nullptr, column, c.m.key_size, c.m.value_size);
    double before = 0.0;
    Four<T, D, kQueriesThreads<T, D>, Vector> next(c, unit, head);
    if (unit.count > 0) next.load(c, 0, unit.count);  // offsets may have changed since the units were made of them
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first, unit.count, head), unit.count, before);
    int turn = 0;
    for (int64_t at = 0; at < unit.count; at += R, turn ^= 1) {
        const int lane = lane_of_turn();
        const In queries{(E *)lds, lane}, keys{(E *)(lds + In::kBytes), lane}, values{(E *)(lds + 2 * In::kBytes), lane},
            grads{(E *)(lds + 3 * In::kBytes), lane};
        const Pairs pairs{(E *)(lds + 4 * In::kBytes), lane};
        next.store(c, queries, keys, values, grads, unit.count - at);
        __syncthreads();
        if (at + R < unit.count) {
            next.load(c, at + R, unit.count - at - R);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at + R, unit.count - at - R, head);
        }
        const Reach<R> &reach = reaches[turn];
        // Pairs by all waves, or, with as many waves that the others have enough to do meanwhile, by those that add to D while those of S read it.
        constexpr bool kApart = D > 64;
        floatx4 read[kTiles][W] = {};
        float down[W];
        if (kApart && role == 0) state.template read_by<T, Parts<T>::kWhole>(grads, read, down);
        constexpr int kStep = kApart ? kWaves : 2 * kWaves;
        const int all_tiles = tiles_of_chunk<T>(kStep);
#pragma unroll 1
        for (int tiles = !kApart ? wave : role == 0 ? all_tiles : wave - kWaves; tiles < all_tiles; tiles += kStep) {
            const int s = tiles * kAcross<T> / kTiles, first = tiles * kAcross<T> % kTiles;
            const int lane = lane_of_turn();
            const In q{queries.at, lane}, k{keys.at, lane}, v{values.at, lane}, g{grads.at, lane};
            floatx4 p[kAcross<T>] = {}, d[kAcross<T>] = {};
#pragma unroll
            for (int a = 0; a < kAcross<T>; a++) {
                const int r = first + a;
                if (r > s) continue;
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    p[a] = product(k.straight(16 * r, i), q.straight(16 * s, i), p[a]);
                    d[a] = product(v.straight(16 * r, i), g.straight(16 * s, i), d[a]);
                    if (i % 64 == 32) in_order();
                }
                d[a] *= decays_of<true>(reach, 16 * r, 16 * s, c.m.scale, lane);
#pragma unroll
                for (int j = 0; j < 4; j++) p[a][j] = 16 * s + lane % 16 > 16 * r + 4 * (lane / 16) + j ? p[a][j] * d[a][j] : 0.0f;
            }
            if (first <= (s | 1)) put_pairs<T>(Pairs{pairs.at, lane}, 16 * s, 16 * first, d);
#pragma unroll
            for (int a = 0; a < kAcross<T>; a++) {
                const int r = first + a;
                const float later = sum_groups(p[a][0] + p[a][1] + p[a][2] + p[a][3]);
                if (lane < 16) by_later[r][16 * s + lane] = later;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float earlier = sum_lanes(p[a][j], 16);
                    if (lane % 16 == 0) by_earlier[s][16 * r + 4 * (lane / 16) + j] = earlier;
                }
            }
        }
        if (!kApart && role == 0) state.template read_by<T, Parts<T>::kWhole>(grads, read, down);
        __syncthreads();
        Operand<E, N> mine[R / 32][W];
        if (role == 0) {
            columns_of(keys, column, mine);
            each_of<kTiles>([&](auto number) {
                constexpr int s = decltype(number)::value;
                scale_read<T>(read[s], reach.row[16 * s + lane % 16], down, lane);
                const int to = column + 4 * (lane / 16);
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const floatx4 x = queries.numbers(16 * s, column + 16 * w);
#pragma unroll
                    for (int j = 0; j < 4; j++) sum = fmaf(read[s][w][j], x[j], sum);
                }
                sum = sum_groups(sum);
                if (lane < 16) by_wave[wave][16 * s + lane] = sum;
                add_pairs<T, 0, s / 2 + 1>(pairs, 16 * s, mine, read[s]);
                in_order();
                if (c.grad_queries && 16 * s + lane % 16 < unit.count - at) {
                    const int64_t base = ((unit.first + at + 16 * s) * c.m.heads + head) * c.m.key_size;
                    const uint32_t offset = (uint32_t)(lane % 16 * c.m.heads * c.m.key_size + to);
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        if (c.m.shared == 1)
                            put_row((T *)c.grad_queries + base + 16 * w, offset, to + 16 * w, c.m.key_size, Vector, read[s][w]);
                        else
                            put_row((float *)c.grad_queries + base + 16 * w, offset, to + 16 * w, c.m.key_size, Vector, read[s][w]);
                    }
                }
            });
            state.template fold<T, kFoldApart<T, D, W, false>>(reach.whole, values, mine, reach.column);
        } else {
            columns_of(queries, column, mine);
            state.template fold<T, kFoldApart<T, D, W, false>>(1.0f, grads, mine, reach.start);
        }
        if (wave == 0 && at + R < unit.count) reach_of(c, reaches[turn ^ 1], gate, unit.count - at - R, before);
        __syncthreads();
        if (threadIdx.x < R && at + threadIdx.x < unit.count) {
            double x = 0.0;
#pragma unroll
            for (int n = 0; n < kTiles; n++) x += (double)by_later[n][threadIdx.x] - (double)by_earlier[n][threadIdx.x];
#pragma unroll
            for (int n = 0; n < kWaves; n++) x += (double)by_wave[n][threadIdx.x];
            c.changes[0][head * c.m.rows + unit.first + at + threadIdx.x] = x;
        }
    }
    if (role == 1) state.template store<true>(c.grad_states + (u * c.m.heads + head) * state_size, column, c.m.key_size, c.m.value_size);
    if (threadIdx.x == 0) c.decays[u * c.m.heads + head] = power_of_two((float)before);
}

// dk, dv, and what changes dlog a from k.dk.
template <class T, int D, bool Vector>
__global__ __launch_bounds__(kKeysThreads<D>, (waves_of_simd(kKeysThreads<D>, kKeysLds<T, D>, kKeysColumns<D> * D / 4))) void attention_grad_keys_kernel(AttentionCall c) {
    constexpr int R = Parts<T>::kRows, N = Parts<T>::kInput, kTiles = R / 16, W = kKeysColumns<D>, kWaves = State<D, W>::kWaves;
    using E = typename Parts<T>::Element;
    using In = Tile<E, N, R, D>;
    using Pairs = PairsOf<T>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Reach<R> *reaches = (Reach<R> *)(lds + 4 * In::kBytes + 2 * Pairs::kBytes);
    float(*by_wave)[R] = (float(*)[R])(reaches + 2);  // k.dk without the chunk's own pairs, of each wave's columns
    const int64_t u = blockIdx.x / c.m.heads;
    const int head = (int)(blockIdx.x % c.m.heads), wave = wave_of();
    const int role = wave / kWaves, column = 16 * W * (wave % kWaves);
    const int64_t state_size = (int64_t)c.m.key_size * c.m.value_size;
    const Unit unit = unit_of<R>(c, u);
    if (!unit.there || unit.count == 0) return;
    State<D, W> state;  // D: rows are keys and columns values (role 0, the values' gradients), or the other way round
    const float *behind = c.grad_states + (u * c.m.heads + head) * state_size;
    if (role == 0)
        state.template load<false>(behind, column, c.m.key_size, c.m.value_size);
    else
        state.template load<true>(behind, column, c.m.key_size, c.m.value_size);
    void *const out = role ? c.grad_keys : c.grad_values;
    const int size = role ? c.m.key_size : c.m.value_size;
    double before = 0.0;
    Four<T, D, kKeysThreads<D>, Vector> next(c, unit, head);
    const int64_t last = (unit.count - 1) / R * R;
    next.load(c, last, unit.count - last);
    float gate = 0.0f;  // of the next chunk's row, in the first wave
    if (wave == 0) reach_of(c, reaches[0], gate_of_lane<T, R>(c, unit.first + last, unit.count - last, head), unit.count - last, before);
    int turn = 0;
    for (int64_t at = last; at >= 0; at -= R, turn ^= 1) {
        const int lane = lane_of_turn();
        const In queries{(E *)lds, lane}, keys{(E *)(lds + In::kBytes), lane}, values{(E *)(lds + 2 * In::kBytes), lane},
            grads{(E *)(lds + 3 * In::kBytes), lane};
        const Pairs scores{(E *)(lds + 4 * In::kBytes), lane}, pairs{(E *)(lds + 4 * In::kBytes + Pairs::kBytes), lane};
        next.store(c, queries, keys, values, grads, unit.count - at);
        __syncthreads();
        if (at > 0) {
            next.load(c, at - R, R);
            if (wave == 0) gate = gate_of_lane<T, R>(c, unit.first + at - R, R, head);
        }
        const Reach<R> &reach = reaches[turn];
        const int all_tiles = tiles_of_chunk<T>(2 * kWaves);
#pragma unroll 1
        for (int tiles = wave; tiles < all_tiles; tiles += 2 * kWaves) {
            const int r = tiles * kAcross<T> / kTiles, first = tiles * kAcross<T> % kTiles;
            if ((first | 1) < r) continue;
            floatx4 p[kAcross<T>] = {}, d[kAcross<T>] = {};
#pragma unroll
            for (int a = 0; a < kAcross<T>; a++) {
                const int s = first + a;
                if (s < r) continue;
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    p[a] = product(queries.straight(16 * s, i), keys.straight(16 * r, i), p[a]);
                    d[a] = product(grads.straight(16 * s, i), values.straight(16 * r, i), d[a]);
                    if (i % 64 == 32) in_order();
                }
                const floatx4 decay = decays_of<false>(reach, 16 * s, 16 * r, c.m.scale, lane);
                p[a] *= decay;
                d[a] *= decay;
            }
            put_pairs<T>(scores, 16 * r, 16 * first, p);
            put_pairs<T>(pairs, 16 * r, 16 * first, d);
        }
        // the same for both roles: what the state reads, what its transposed rows are added up with, and what of
        const In reading{(E *)(lds + (role ? 2 : 1) * In::kBytes), lane}, with{(E *)(lds + (role ? 0 : 3) * In::kBytes), lane},
            adding{(E *)(lds + (role ? 3 : 0) * In::kBytes), lane};
        const Pairs mine_of{(E *)(lds + 4 * In::kBytes + role * Pairs::kBytes), lane};
        floatx4 read[kTiles][W] = {};
        float down[W];
        if (role)
            state.template read_by<T, Parts<T>::kWhole>(reading, read, down);
        else
            state.template read_by<T, Parts<T>::kState>(reading, read, down);
        __syncthreads();
        Operand<E, N> mine[R / 32][W];
        columns_of(with, column, mine);
        each_of<kTiles>([&](auto number) {
            constexpr int r = decltype(number)::value;
            scale_read<T>(read[r], reach.column[16 * r + lane % 16], down, lane);
            const int to = column + 4 * (lane / 16);
            if (role) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const floatx4 k = keys.numbers(16 * r, column + 16 * w);
#pragma unroll
                    for (int j = 0; j < 4; j++) sum = fmaf(read[r][w][j], k[j], sum);
                }
                sum = sum_groups(sum);
                if (lane < 16) by_wave[wave - kWaves][16 * r + lane] = sum;
            }
            add_pairs<T, r / 2, R / 32>(mine_of, 16 * r, mine, read[r]);
            in_order();
            if (out && 16 * r + lane % 16 < unit.count - at) {
                const int64_t base = ((unit.first + at + 16 * r) * c.m.heads + head) * size;
                const uint32_t offset = (uint32_t)(lane % 16 * c.m.heads * size + to);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    if (!role || c.m.shared == 1)
                        put_row((T *)out + base + 16 * w, offset, to + 16 * w, size, Vector, read[r][w]);
                    else
                        put_row((float *)out + base + 16 * w, offset, to + 16 * w, size, Vector, read[r][w]);
                }
            }
        });
        state.template fold<T, kFoldApart<T, D, W, false>>(reach.whole, adding, mine, reach.row);
        if (wave == 0 && at > 0) reach_of(c, reaches[turn ^ 1], gate, R, before);
        __syncthreads();
        if (threadIdx.x < R && at + threadIdx.x < unit.count) {
            double x = 0.0;
#pragma unroll
            for (int n = 0; n < kWaves; n++) x += (double)by_wave[n][threadIdx.x];
            c.changes[1][head * c.m.rows + unit.first + at + threadIdx.x] = x;
        }
    }
}

int launch_attention_backward(int64_t type, const AttentionCall &c, int size, bool for_keys, hipStream_t stream) {
    return by_attention_kernel(type, size, c.vector, [&](auto t, auto d, auto vector) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value, kQueries = kQueriesLds<T, D>, kKeys = kKeysLds<T, D>;
        constexpr bool Vector = decltype(vector)::value;
        static_assert(kQueries <= 160 * 1024 && kKeys <= 160 * 1024, "LDS");
        static size_t reserved[2][kMaxDevices];
        const dim3 grid((unsigned)(c.most_units * c.m.heads));
        const void *kernel = for_keys ? (const void *)attention_grad_keys_kernel<T, D, Vector> : (const void *)attention_grad_queries_kernel<T, D, Vector>;
        const int code = reserve_lds("tg_linear_attention_backward", kernel, for_keys ? kKeys : kQueries, reserved[for_keys]);
        if (code) return code;
        if (for_keys)
            TG_LAUNCH_AS("attention_grad_keys", (attention_grad_keys_kernel<T, D, Vector>), grid, dim3(kKeysThreads<D>), kKeys, stream, c);
        else
            TG_LAUNCH_AS("attention_grad_queries", (attention_grad_queries_kernel<T, D, Vector>), grid, dim3((kQueriesThreads<T, D>)), kQueries, stream, c);
        return 0;
    });
}

}  // namespace tg
#endif
