// tg_attention_chunk.hpp -- linear attention by chunks of rows on the matrix units: what its kernels share.
//
// With L_t the sum of log2 a from a chunk's first row to row t, S_0 the state in front of the chunk and D_C the gradient of the state behind it,
//     o_s  = scale [ sum_{r <= s} 2^(L_s - L_r) (q_s.k_r) v_r + 2^L_s S_0^T q_s ],      S_C = 2^L_C S_0 + sum_r 2^(L_C - L_r) k_r v_r^T,
//     dq_s = scale [ sum_{r <= s} 2^(L_s - L_r) (do_s.v_r) k_r + 2^L_s S_0 do_s ],
//     dk_r = scale sum_{s >= r} 2^(L_s - L_r) (do_s.v_r) q_s + 2^(L_C - L_r) D_C v_r,   D_0 = 2^L_C D_C + scale sum_s 2^L_s q_s do_s^T,
//     dv_r = scale sum_{s >= r} 2^(L_s - L_r) (q_s.k_r) do_s + 2^(L_C - L_r) D_C^T k_r:
// products of matrices of at most 64 rows and TG_ATTENTION_SIZE columns.  A workgroup has a head and a run of chunks (a unit), one after another; the states stay in
// the accumulators of its waves, each of which has sixteen columns of them.
//
// Numbers.  Products are of numbers in 16 bits and summed in float32.  What is not one is a sum of "parts", each the rounded rest of those before.
// In bfloat16, whose range is float32's, inputs in float32 are three parts, exactly; so are states, and inputs that carry a decay, wherever what they
// go into is float32 in the end (states, their gradients, gates' gradients: two parts leave an error of 2e-6, three one of 1e-8, below that of the
// sums).  What goes into an output of 16 bits has two parts, states as well as the matrix of pairs inside a chunk: 2^-16 of a term, where the output's own
// rounding is 2^-8 (pairs in one part left outputs off by 2.3e-3 of their norm in place of 1.7e-3).  Inputs in
// float16 stay as they are, and what meets them is two parts in float16 (an error of 2^-22 of each, or 2^-39 of the largest): a column of a state or of
// weighted inputs, and 32 pairs of a row, by a power of two that brings the largest of them near 2^15.  What they are summed with has the same column, or row:
// no other has a part in how they are rounded, also where it is not finite.
#pragma once
#include "tg_attention.hpp"

#include <type_traits>

namespace tg {

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));

// Parts of an input, of a state or a pair that goes into an output of its type and of what goes into float32, their type, and rows of a chunk: as many
// as leave room in LDS for the parts.
template <class T> struct Parts;
template <> struct Parts<bf16_t> {
    using Element = __bf16;
    static constexpr int kInput = 1, kState = 2, kWhole = 3, kRows = 64;
    static constexpr bool kScaled = false;
};
template <> struct Parts<half_t> {
    using Element = _Float16;
    static constexpr int kInput = 1, kState = 2, kWhole = 2, kRows = 64;
    static constexpr bool kScaled = true;
};
template <> struct Parts<float> {
    using Element = __bf16;
    static constexpr int kInput = 3, kState = 3, kWhole = 3, kRows = 32;
    static constexpr bool kScaled = false;
};

template <class E> struct Vectors {
    typedef E x8 __attribute__((ext_vector_type(8)));
    typedef E x4 __attribute__((ext_vector_type(4)));
};

// Eight numbers of a lane for a product of 16 x 32 by 32 x 16 numbers: row (of A) or column (of B) lane % 16, and eight of the 32 that are summed over;
// which, both operands have to agree in.  "Straight": 8 (lane / 16) on.  "Chained": 4 (lane / 16) on, and sixteen further: as two accumulators one above
// the other hold them (rows 4 (lane / 16) on of column lane % 16), so that a state goes from one product into the next without leaving its lane.
template <class E, int N> struct Operand { typename Vectors<E>::x8 part[N]; };

__device__ __forceinline__ floatx4 multiply(Vectors<__bf16>::x8 a, Vectors<__bf16>::x8 b, floatx4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, sum, 0, 0, 0);
}
__device__ __forceinline__ floatx4 multiply(Vectors<_Float16>::x8 a, Vectors<_Float16>::x8 b, floatx4 sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, sum, 0, 0, 0);
}
template <class E, int NA, int NB> __device__ __forceinline__ floatx4 product(const Operand<E, NA> &a, const Operand<E, NB> &b, floatx4 sum) {
    constexpr int kTerms = NA > NB ? NA : NB;  // parts beyond are below the last ones' rounding
#pragma unroll
    for (int i = NA - 1; i >= 0; i--)
#pragma unroll
        for (int j = NB - 1; j >= 0; j--)
            if (i + j < kTerms) sum = multiply(a.part[i], b.part[j], sum);
    return sum;
}

// What two numbers' roundings leave of them: sums of two products and a number, exact here, one instruction each where taking a rounded number out of its
// half and subtracting it are two.  -1 and 0 come from a register: the compiler writes them as constants of another type into the instruction.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void without(bf16x2 rounded, float &x, float &y) {
    uint32_t first = 0x0000bf80u, second = 0xbf800000u;
    asm("" : "+s"(first), "+s"(second));
    x = __builtin_amdgcn_fdot2_f32_bf16(rounded, __builtin_bit_cast(bf16x2, first), x, false);
    y = __builtin_amdgcn_fdot2_f32_bf16(rounded, __builtin_bit_cast(bf16x2, second), y, false);
}
__device__ __forceinline__ void without(halfx2 rounded, float &x, float &y) {
    uint32_t first = 0x0000bc00u, second = 0xbc000000u;
    asm("" : "+s"(first), "+s"(second));
    x = __builtin_amdgcn_fdot2(rounded, __builtin_bit_cast(halfx2, first), x, false);
    y = __builtin_amdgcn_fdot2(rounded, __builtin_bit_cast(halfx2, second), y, false);
}

template <class E, int N> __device__ __forceinline__ Operand<E, N> parts_of(const float *x) {
    typedef E x2 __attribute__((ext_vector_type(2)));
    Operand<E, N> o;
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; j++) rest[j] = x[j];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const x2 rounded = {(E)rest[j], (E)rest[j + 1]};
            o.part[n][j] = rounded[0];
            o.part[n][j + 1] = rounded[1];
            if (n + 1 < N) without(rounded, rest[j], rest[j + 1]);
        }
    return o;
}

// A power of two that brings the largest of four lanes' numbers (16 lanes apart; `most` is this lane's, none is negative) to at most 2^15, and its reciprocal.
struct Scaling {
    float up, down;
};
__device__ __forceinline__ Scaling scaling_of(float most) {
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const int exponent = max(1, min(253, 268 - (int)(__float_as_uint(most) >> 23)));
    return {__uint_as_float((uint32_t)exponent << 23), __uint_as_float((uint32_t)(254 - exponent) << 23)};
}

// A matrix of Rows x Columns in LDS, N parts.  One that is only read by rows has rows 16 bytes longer than their numbers, so that sixteen rows begin in
// different banks; one that is read transposed too, 32 bytes of four rows at once, has them 32 bytes longer, which sets eight rows apart, and the
// other eight of sixteen with neighbouring 16 bytes exchanged: no reading meets another in a bank.
template <class E, int N, int Rows, int Columns, bool Turned = true> struct Tile {
    using x8 = typename Vectors<E>::x8;
    using x4 = typename Vectors<E>::x4;
    static constexpr int kExchanged = Turned ? 8 : 0, kStride = Columns + (Turned ? 16 : 8), kPart = Rows * kStride, kBytes = N * kPart * 2;
    E *at;
    int lane;

    __device__ __forceinline__ Operand<E, N> straight(int row, int column) const {
        const E *p = at + (row + lane % 16) * kStride + column + (8 * (lane / 16) ^ (lane & kExchanged));
        Operand<E, N> o;
#pragma unroll
        for (int n = 0; n < N; n++) o.part[n] = *(const x8 *)(p + n * kPart);
        return o;
    }
    __device__ __forceinline__ Operand<E, N> chained(int row, int column) const {
        const E *p = at + (row + lane % 16) * kStride + column + (4 * (lane / 16) ^ (lane & kExchanged));
        Operand<E, N> o;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const x4 a = *(const x4 *)(p + n * kPart), b = *(const x4 *)(p + n * kPart + 16);
            o.part[n] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return o;
    }
    // The transposed matrix's: row or column `column` + lane % 16, chained rows from `row`.  LDS hands out four rows of sixteen columns transposed to
    // sixteen lanes, of which each points at four neighbours of a row.
    __device__ __forceinline__ Operand<E, N> transposed(int row, int column) const {
        static_assert(Turned);
        const E *p = at + (row + 4 * (lane / 16) + lane % 16 / 4) * kStride + column + (4 * (lane % 4) ^ (lane >> 2 & kExchanged));
        Operand<E, N> o;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const x4 a = turned(p + n * kPart), b = turned(p + n * kPart + 16 * kStride);
            o.part[n] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return o;
    }
    static __device__ __forceinline__ x4 turned(const E *p) {
        return __builtin_bit_cast(x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t *)p));
    }
    // Four neighbours, as an accumulator has them: of row `row` + lane % 16, from `column` + 4 (lane / 16) on.
    __device__ __forceinline__ floatx4 numbers(int row, int column) const {
        const E *p = at + (row + lane % 16) * kStride + column + (4 * (lane / 16) ^ (lane & kExchanged));
        floatx4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = N - 1; n >= 0; n--) {
            const x4 v = *(const x4 *)(p + n * kPart);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] += (float)v[j];
        }
        return x;
    }
    // What 32 pairs of a row from column 32 `strip` on are to be multiplied with, in the bytes behind the row's numbers.
    __device__ __forceinline__ float &factor(int row, int strip) const {
        static_assert(!Turned && Columns <= 128);
        return ((float *)(at + row * kStride + Columns))[strip];
    }
    // An accumulator's four rows (columns here) of its column (a row here): the product's transpose.
    __device__ __forceinline__ void put(int row, int column, floatx4 x) const {
        static_assert(!Turned);
        E *p = at + (row + lane % 16) * kStride + column + 4 * (lane / 16);
#pragma unroll
        for (int n = 0; n < N; n++) {
            x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = (E)x[j];
                x[j] -= (float)v[j];
            }
            *(x4 *)(p + n * kPart) = v;
        }
    }
};

// A transposed input's numbers with a weight for each row.
template <class E, int N> __device__ __forceinline__ void weighted(const Operand<E, N> &o, const float *weights, int row, int lane, float *x) {
    const int group = lane / 16;
    const floatx4 a = *(const floatx4 *)(weights + row + 4 * group), b = *(const floatx4 *)(weights + row + 16 + 4 * group);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        x[j] = (float)o.part[N - 1][j];
#pragma unroll
        for (int n = N - 2; n >= 0; n--) x[j] += (float)o.part[n][j];
        x[j] *= j < 4 ? a[j] : b[j - 4];
    }
}

// The matrix of pairs inside a chunk.
template <class T> using PairsOf = Tile<typename Parts<T>::Element, Parts<T>::kState, Parts<T>::kRows, Parts<T>::kRows, false>;
// Neighbouring tiles of sixteen columns that a wave makes at a time: those of a product over 32 columns where they have one scaling.
template <class T> constexpr int kAcross = Parts<T>::kScaled ? 2 : 1;

// How many of a chunk's tiles there are for waves that take every `waves`th.  Where that is one turn the compiler does not know it: it would take the loop
// away, and fill the registers with what is read behind it.
template <class T> __device__ __forceinline__ int tiles_of_chunk(int waves) {
    int n = Parts<T>::kRows / 16 * Parts<T>::kRows / 16 / kAcross<T>;
    if (n <= waves) asm volatile("" : "+s"(n));
    return n;
}

// Puts sixteen rows of pairs from `row` on, scaled by row where they have to be.
template <class T> __device__ __forceinline__ void put_pairs(const PairsOf<T> &pairs, int row, int column, floatx4 (&p)[kAcross<T>]) {
    if constexpr (Parts<T>::kScaled) {
        float most = 0.0f;  // of the row's numbers in this lane
#pragma unroll
        for (int a = 0; a < kAcross<T>; a++)
#pragma unroll
            for (int j = 0; j < 4; j++) most = fmaxf(most, fabsf(p[a][j]));
        const Scaling scaling = scaling_of(most);
#pragma unroll
        for (int a = 0; a < kAcross<T>; a++) p[a] *= scaling.up;
        if (pairs.lane < 16) pairs.factor(row + pairs.lane, column / 32) = scaling.down;
    }
#pragma unroll
    for (int a = 0; a < kAcross<T>; a++) pairs.put(row, column + 16 * a, p[a]);
}

// Keeps the compiler from reading ahead over this point: operands of a whole chunk, read at its beginning, would not fit the registers.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }
// ---- reading a chunk ----------------------------------------------------------------------

// A thread's part of a chunk of Rows x D numbers, on its way to LDS: groups of eight neighbours.  Vector: in accesses of 16 bytes, which divide the
// rows and are aligned.
template <class T, int Rows, int D, int Threads, bool Vector> struct Incoming {
    static constexpr int kAll = Rows * D / 8, kGroups = (kAll + Threads - 1) / Threads, kWidest = Vector ? 16 / (int)sizeof(T) : 1;
    Pack<T, kWidest> x[kGroups][8 / kWidest];

    static __device__ __forceinline__ int row_of(int n) { return ((int)threadIdx.x + n * Threads) / (D / 8); }
    static __device__ __forceinline__ int column_of(int n) { return ((int)threadIdx.x + n * Threads) % (D / 8) * 8; }
    static __device__ __forceinline__ bool mine(int n) { return kAll % Threads == 0 || (int)threadIdx.x + n * Threads < kAll; }  // for whole waves alike

    // `count` > 0 rows from p on, `size` numbers each.  What lies beyond is read from places inside, and dropped by store: a load that no branch goes
    // around is waited for where its numbers are used, after a chunk's computation.
    __device__ __forceinline__ void load(const T *p, int64_t row_stride, int64_t count, int size) {
#pragma unroll
        for (int n = 0; n < kGroups; n++) {
            if (!mine(n)) continue;
            const T *from = p + min((int64_t)row_of(n), count - 1) * row_stride;
#pragma unroll
            for (int j = 0; j < 8; j += kWidest) x[n][j / kWidest] = load_pack<kWidest>(from + min(column_of(n) + j, size - kWidest));
        }
    }
    template <class E, int N> __device__ __forceinline__ void store(const Tile<E, N, Rows, D> &tile, int64_t count, int size) const {
#pragma unroll
        for (int n = 0; n < kGroups; n++) {
            if (!mine(n)) continue;
            using In = Tile<E, N, Rows, D>;
            const int row = row_of(n), column = column_of(n), place = row * In::kStride + (column ^ (row & In::kExchanged));
            if constexpr (Vector && N == 1) {  // as it is
                const uint32x4 w = __builtin_bit_cast(uint32x4, x[n][0]), none = {0, 0, 0, 0}, v = row < count && column < size ? w : none;
                *(uint32x4 *)(tile.at + place) = v;
                continue;
            }
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = row < count && column + j / kWidest * kWidest < size ? (float)x[n][j / kWidest].v[j % kWidest] : 0.0f;
            const Operand<E, N> o = parts_of<E, N>(v);
#pragma unroll
            for (int i = 0; i < N; i++)
                *(typename Vectors<E>::x8 *)(tile.at + i * In::kPart + place) = o.part[i];
        }
    }
};

// Waves of a SIMD that a kernel is compiled for: those of as many workgroups as a CU's 160 KB of LDS have room for, at most four (128 registers a
// lane), or two for a state of 64 registers.
constexpr int waves_of_simd(int threads, int lds_bytes, int state_registers) {
    const int groups = 160 * 1024 / lds_bytes, waves = groups * threads / kWave / 4, most = state_registers > 32 ? 2 : 4;
    return waves > most ? most : waves < 1 ? 1 : waves;
}

// Decays of a chunk.
template <int Rows> struct alignas(16) Reach {
    double reach[Rows];   // L
    float row[Rows];      // scale 2^L
    float column[Rows];   // 2^(L_C - L)
    float start[Rows];    // scale 2^L from the unit's beginning
    float whole;          // 2^L_C
};

struct AttentionCall {
    Attention m;
    const void *queries, *keys, *values, *gates;
    const float *initial;
    const int32_t *offsets;
    const int32_t *plan;    // packed: sequence of each unit, or -1; behind `most_units` of them the first unit of each sequence
    void *outputs;
    float *final;
    float *states;          // of each unit and head, in front of it
    float *finals;          // of each sequence and head, the state behind it, kept for the backward pass; or null
    float *decays;          // of each unit and head
    int64_t most_units;     // units there may be
    int64_t units;          // of a sequence, where all are alike
    int chunks;             // of a unit
    bool wide_gates;
    bool vector;            // see Incoming
    bool through;           // a workgroup has a whole sequence
    // the backward pass's
    const void *grad_outputs;
    bool grad_outputs_there;  // false: zeros, and the pointer is to something else of the values' shape
    const float *grad_final;
    void *grad_queries, *grad_keys, *grad_values, *grad_gates;
    float *grad_states;     // of each unit and head: what the unit adds to the gradient in front of it, then the gradient behind it
    double *changes[2];     // of each head and row: what dlog a changes by
    double *sums;           // of each unit and head: dlog a of all rows
};

struct Unit {
    int64_t sequence, index;  // index: in its sequence
    int64_t first, count;     // rows
    int64_t base;             // in the sequence
    bool there;
};
template <int Rows> __device__ __forceinline__ Unit unit_of(const AttentionCall &c, int64_t u) {
    Unit n;
    if (c.m.packed) {
        n.sequence = c.plan[u];
        n.there = n.sequence >= 0;
        if (!n.there) return n;
        n.index = u - c.plan[c.most_units + n.sequence];
    } else {
        n.sequence = u / c.units;
        n.index = u - n.sequence * c.units;
        n.there = true;
    }
    const AttentionRows rows = rows_of(c.m, c.offsets, n.sequence);
    n.base = n.index * c.chunks * Rows;
    n.first = rows.first + n.base;
    n.count = max((int64_t)0, min(rows.count - n.base, (int64_t)c.chunks * Rows));
    return n;
}

template <class T> __device__ __forceinline__ float gate_at(const AttentionCall &c, int64_t row, int head) {
    const int64_t at = c.m.fixed ? head : row * c.m.heads + head;
    return c.wide_gates ? ((const float *)c.gates)[at] : (float)((const T *)c.gates)[at];
}

// v plus that of another lane, where the data-parallel move's control has one, else v.
template <int Control, int RowMask> __device__ __forceinline__ double plus_lane(double v) {
    const uint64_t bits = (uint64_t)__double_as_longlong(v);
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, Control, RowMask, 0xf, false);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), Control, RowMask, 0xf, false);
    return v + __longlong_as_double((long long)((uint64_t)high << 32 | low));
}

__device__ __forceinline__ float power_of_two(float l) { return __builtin_amdgcn_exp2f(l); }  // what is below 2^-126 is zero

// One wave: the decays of `count` rows whose gates its lanes hold, where `before` is L from the unit's beginning, which moves on.
template <int Rows> __device__ __forceinline__ void reach_of(const AttentionCall &c, Reach<Rows> &out, float gate, int64_t count, double &before) {
    const int lane = threadIdx.x % kWave;
    double sum = lane < count && lane < Rows ? log2_gate(c.m.gate_form, gate) : 0.0;
    sum = plus_lane<0x111, 0xf>(sum);  // sums over sixteen lanes by moves of 1, 2, 4 and 8
    sum = plus_lane<0x112, 0xf>(sum);
    sum = plus_lane<0x114, 0xf>(sum);
    sum = plus_lane<0x118, 0xf>(sum);
    sum = plus_lane<0x142, 0xa>(sum);  // the last lane of sixteen to the next sixteen, of 32 to the next 32
    if (Rows > 32) sum = plus_lane<0x143, 0xc>(sum);
    const uint64_t bits = (uint64_t)__double_as_longlong(sum);
    const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, Rows - 1), high = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), Rows - 1);
    const double whole = __longlong_as_double((long long)((uint64_t)high << 32 | low));
    if (lane < Rows) {
        out.reach[lane] = sum;
        out.row[lane] = c.m.scale * power_of_two((float)sum);
        out.column[lane] = power_of_two((float)(whole - sum));
        out.start[lane] = c.m.scale * power_of_two((float)(before + sum));
        if (lane == 0) out.whole = power_of_two((float)whole);
    }
    before += whole;
}
template <class T, int Rows> __device__ __forceinline__ float gate_of_lane(const AttentionCall &c, int64_t first, int64_t count, int head) {
    const int lane = threadIdx.x % kWave;
    return lane < count && lane < Rows ? gate_at<T>(c, first + lane, head) : 0.0f;
}

// scale 2^(L_s - L_r) of an accumulator whose columns are rows s (or r) of the chunk, zero where s < r.
template <bool ColumnsAreLater, int Rows> __device__ __forceinline__ floatx4 decays_of(const Reach<Rows> &reach, int row, int column, float scale, int lane) {
    const int x = column + lane % 16, y = row + 4 * (lane / 16);
    const double here = reach.reach[x];
    floatx4 d;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const double other = reach.reach[y + j];
        const float l = (float)(ColumnsAreLater ? here - other : other - here);
        const bool in = ColumnsAreLater ? x >= y + j : x <= y + j;
        d[j] = in ? scale * power_of_two(l) : 0.0f;
    }
    return d;
}

// Four neighbours of an output's row, `offset` numbers from p on.
template <class T> __device__ __forceinline__ void put_row(T *p, uint32_t offset, int column, int size, bool vector, floatx4 x) {
    if (vector) {
        if (column < size) {
            const float v[4] = {x[0], x[1], x[2], x[3]};
            store_pack<4>(p + offset, v);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (column + j < size) p[offset + j] = (T)x[j];
    }
}

// The number of the wave, and a lane's in it.  What is made of lane_of_turn is made again in each turn of a loop: places in LDS and in memory that
// were kept over all of them would take more registers than the states.
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave); }
__device__ __forceinline__ int lane_of_turn() {
    int lane = threadIdx.x % kWave;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Whether State::fold adds up apart, where the registers are enough: 8 x 2048 rows of 32 heads of 64 with fixed decays near 1, states off by 1.1e-7 in
// place of 2.7e-7 and the decays' gradients by 5e-7 in place of 9e-7, in the same time; but 4 x 4096 rows of 16 heads of 128 the outputs' kernel 168 us
// in place of 115, and, with two times sixteen columns a wave, the keys' 261 in place of 198.
template <class T, int D, int W, bool Forward> constexpr bool kFoldApart = Forward ? D <= 64 || Parts<T>::kRows == 32 : W == 1;

// The state in accumulators: rows of keys and columns of values (Turned: the other way round), of a wave the 16 W columns from `column` on.  With W = 2 an
// operand from LDS goes into twice as many products, with W = 1 twice as many waves hide each other's latencies.
template <int D, int W> struct State {
    static constexpr int kWaves = D / (16 * W);
    floatx4 x[W][D / 16];

    // call(w, n, j, the place of x[w][n][j]) for all that are there, with one offset of a lane and a uniform one beside it.
    template <bool Turned, class Call> __device__ __forceinline__ void each(int column, int key_size, int value_size, Call &&call) {
        const int lane = lane_of_turn();
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int across = column + 16 * w + lane % 16, down = 4 * (lane / 16);
            const int most = Turned ? value_size : key_size, offset = Turned ? across * value_size + down : down * value_size + across;
            if (across < (Turned ? key_size : value_size)) {
#pragma unroll
                for (int n = 0; n < D / 16; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (down + 16 * n + j < most) call(w, n, j, offset + (Turned ? 16 * n + j : (16 * n + j) * value_size));
            }
        }
    }
    template <bool Turned> __device__ __forceinline__ void load(const float *from, int column, int key_size, int value_size) {
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int n = 0; n < D / 16; n++) x[w][n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if (from) each<Turned>(column, key_size, value_size, [&](int w, int n, int j, int at) { x[w][n][j] = from[at]; });
    }
    template <bool Turned> __device__ __forceinline__ void store(float *to, int column, int key_size, int value_size) {
        each<Turned>(column, key_size, value_size, [&](int w, int n, int j, int at) { to[at] = x[w][n][j]; });
    }
    // Adds its transpose times the rows' columns to `sums`, by sixteen rows of the tile; `down`: what the sums are to be multiplied with, by column (Scaled).
    template <class T, int M, class E, int N, int Rows>
    __device__ __forceinline__ void read_by(const Tile<E, N, Rows, D> &tile, floatx4 (&sums)[Rows / 16][W], float (&down)[W]) const {
        float up[W];
        if constexpr (Parts<T>::kScaled) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                float most = 0.0f;
#pragma unroll
                for (int n = 0; n < D / 16; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) most = fmaxf(most, fabsf(x[w][n][j]));
                const Scaling scaling = scaling_of(most);
                up[w] = scaling.up;
                down[w] = scaling.down;
            }
        }
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            Operand<E, M> mine[W];
#pragma unroll
            for (int w = 0; w < W; w++) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = Parts<T>::kScaled ? x[w][2 * i + j / 4][j % 4] * up[w] : x[w][2 * i + j / 4][j % 4];
                mine[w] = parts_of<E, M>(v);
            }
#pragma unroll
            for (int r = 0; r < Rows / 16; r++) {
                const Operand<E, N> theirs = tile.chained(16 * r, 32 * i);
#pragma unroll
                for (int w = 0; w < W; w++) sums[r][w] = product(mine[w], theirs, sums[r][w]);
            }
            in_order();
        }
    }
    // decay times itself, plus the tile, transposed, times this wave's columns `mine` of another with a weight for each row.  Apart: 32 rows are added
    // up apart, so that a long state is rounded twice a chunk and not by each of six products.
    template <class T, bool Apart, class E, int N, int Rows>
    __device__ __forceinline__ void fold(float decay, const Tile<E, N, Rows, D> &tile, const Operand<E, N> (&mine)[Rows / 32][W], const float *weights) {
        constexpr int M = Parts<T>::kWhole, K = Rows / 32;
        if constexpr (Parts<T>::kScaled) {
            Operand<E, M> late[K][W];
            float down[W];
#pragma unroll
            for (int w = 0; w < W; w++) {
                float v[K][8], most = 0.0f;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    weighted(mine[k][w], weights, 32 * k, tile.lane, v[k]);
#pragma unroll
                    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(v[k][j]));
                }
                const Scaling scaling = scaling_of(most);
                down[w] = scaling.down;
#pragma unroll
                for (int k = 0; k < K; k++) {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[k][j] *= scaling.up;
                    late[k][w] = parts_of<E, M>(v[k]);
                }
            }
#pragma unroll
            for (int n = 0; n < D / 16; n++) {
                floatx4 sum[W] = {};
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const Operand<E, N> theirs = tile.transposed(32 * k, 16 * n);
#pragma unroll
                    for (int w = 0; w < W; w++) sum[w] = product(theirs, late[k][w], sum[w]);
                }
#pragma unroll
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int j = 0; j < 4; j++) x[w][n][j] = fmaf(sum[w][j], down[w], x[w][n][j] * decay);
                if (n % 4 == 3) in_order();
            }
        } else {
            if (!Apart) {
#pragma unroll
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int n = 0; n < D / 16; n++) x[w][n] *= decay;
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                Operand<E, M> late[W];
#pragma unroll
                for (int w = 0; w < W; w++) {
                    float v[8];
                    weighted(mine[k][w], weights, 32 * k, tile.lane, v);
                    late[w] = parts_of<E, M>(v);
                }
#pragma unroll
                for (int n = 0; n < D / 16; n++) {
                    const Operand<E, N> theirs = tile.transposed(32 * k, 16 * n);
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        const floatx4 sum = product(theirs, late[w], Apart ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : x[w][n]);
#pragma unroll
                        for (int j = 0; j < 4; j++) x[w][n][j] = !Apart ? sum[j] : k == 0 ? fmaf(x[w][n][j], decay, sum[j]) : x[w][n][j] + sum[j];
                    }
                    if (n % 4 == 3) in_order();
                }
            }
        }
    }
};

// call(constant 0), ... up to before N
template <int N, class Call> __device__ __forceinline__ void each_of(Call &&call) {
    if constexpr (N > 0) {
        each_of<N - 1>(call);
        call(std::integral_constant<int, N - 1>());
    }
}

// What a state gave sixteen rows, times their decay, and times what lanes 0 to 15 have for its columns.
template <class T, int W> __device__ __forceinline__ void scale_read(floatx4 (&read)[W], float decay, const float (&down)[W], int lane) {
#pragma unroll
    for (int w = 0; w < W; w++) {
        read[w] *= decay;
        if constexpr (Parts<T>::kScaled) {
#pragma unroll
            for (int j = 0; j < 4; j++) read[w][j] *= __shfl(down[w], 4 * (lane / 16) + j);
        }
    }
}

// This wave's columns of a tile, for fold.
template <class E, int N, int Rows, int D, int W>
__device__ __forceinline__ void columns_of(const Tile<E, N, Rows, D> &tile, int column, Operand<E, N> (&mine)[Rows / 32][W]) {
#pragma unroll
    for (int k = 0; k < Rows / 32; k++)
#pragma unroll
        for (int w = 0; w < W; w++) mine[k][w] = tile.transposed(32 * k, column + 16 * w);
}

// += this wave's columns times sixteen rows of pairs from `row` on, those of the columns from First on to before Last.
template <class T, int First, int Last, class E, int N, int Rows, int W>
__device__ __forceinline__ void add_pairs(const Tile<E, Parts<T>::kState, Rows, Rows, false> &pairs, int row, const Operand<E, N> (&mine)[Rows / 32][W], floatx4 (&sums)[W]) {
#pragma unroll
    for (int k = First; k < Last; k++) {
        const Operand<E, Parts<T>::kState> p = pairs.chained(row, 32 * k);
        if constexpr (Parts<T>::kScaled) {
            const float down = pairs.factor(row + pairs.lane % 16, k);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const floatx4 inside = product(mine[k][w], p, floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int j = 0; j < 4; j++) sums[w][j] = fmaf(inside[j], down, sums[w][j]);
            }
        } else {
#pragma unroll
            for (int w = 0; w < W; w++) sums[w] = product(mine[k][w], p, sums[w]);
        }
    }
}

// `size`: 32, 64 or 128, of keys and values in the kernel
int launch_attention_forward(int64_t type, const AttentionCall &c, int size, bool states_only, hipStream_t stream);
int launch_attention_backward(int64_t type, const AttentionCall &c, int size, bool keys, hipStream_t stream);

// call(T(), constant D, constant Vector)
template <class Call> int by_attention_kernel(int64_t type, int size, bool vector, Call &&call) {
    const auto with_type = [&](auto t) {
        const auto with_size = [&](auto d) { return vector ? call(t, d, std::true_type()) : call(t, d, std::false_type()); };
        return size <= 32 ? with_size(std::integral_constant<int, 32>()) : size <= 64 ? with_size(std::integral_constant<int, 64>())
                                                                                       : with_size(std::integral_constant<int, 128>());
    };
    return type == TG_TYPE_F32 ? with_type(float()) : type == TG_TYPE_F16 ? with_type(half_t()) : with_type(bf16_t());
}

}  // namespace tg
