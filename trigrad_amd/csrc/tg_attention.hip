// tg_attention.hip -- linear attention S_t = a_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t: the calls, a walk through the rows, a single step.
//
// With D_t the gradient of S_t with all that follows from it,
//     D_t = a_{t+1} D_{t+1} + scale q_t do_t^T,   dq_t = scale S_t do_t,   dk_t = D_t v_t,   dv_t = D_t^T k_t,   dlog a_t = a_t <D_t, S_{t-1}>,
// and since <D_t, S_t> is both q_t.dq_t + dlog a_{t+1} and k_t.dk_t + dlog a_t,
//     dlog a_{t+1} = dlog a_t + k_t.dk_t - q_t.dq_t,   dlog a_1 = <S_0, a_1 D_1>.
#ifdef TG_DOUBLE_PRECISION
#include "tg_attention.hpp"
#else
#include "tg_attention_chunk.hpp"
#endif

namespace tg {

constexpr int kWalkThreads = 64;
constexpr int64_t kGridThreads = (int64_t)1 << 32;  // a grid has fewer
constexpr int kMost = TG_ATTENTION_SIZE;

template <class T> __device__ __forceinline__ double wide(T v) { return (double)(real)v; }

#ifdef TG_DOUBLE_PRECISION
// ---- a walk through the rows ----------------------------------------------------------

// A thread has a column of the state, in LDS.
template <class T, class S>
__global__ __launch_bounds__(kWalkThreads) void attention_walk_kernel(Attention m, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                      const T *__restrict__ values, const S *__restrict__ gates,
                                                                      const real *__restrict__ initial, const int32_t *__restrict__ offsets,
                                                                      T *__restrict__ outputs, real *__restrict__ final) {
    __shared__ double state[kMost][kWalkThreads];
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), lane = threadIdx.x, j = blockIdx.y * kWalkThreads + lane;
    if (j >= m.value_size) return;
    const AttentionRows rows = rows_of(m, offsets, s);
    const T *q = queries + place_of(m, m.q, s, rows.first, h / m.shared), *k = keys + place_of(m, m.k, s, rows.first, h / m.shared),
            *v = values + place_of(m, m.v, s, rows.first, h);
    const int64_t at = (s * m.heads + h) * m.key_size * m.value_size + j;
    for (int i = 0; i < m.key_size; i++) state[i][lane] = initial ? (double)initial[at + (int64_t)i * m.value_size] : 0.0;
    for (int64_t t = 0; t < rows.count; t++) {
        const double a = exp2(log2_gate(m.gate_form, (real)gates[m.fixed ? h : (rows.first + t) * m.heads + h]));
        const double x = wide(v[t * m.v.row + j]);
        double sum = 0.0;
        for (int i = 0; i < m.key_size; i++) {
            const double next = a * state[i][lane] + wide(k[t * m.k.row + i]) * x;
            state[i][lane] = next;
            sum += wide(q[t * m.q.row + i]) * next;
        }
        outputs[((rows.first + t) * m.heads + h) * m.value_size + j] = (T)(real)(sum * (double)m.scale);
    }
    for (int i = 0; i < m.key_size; i++) final[at + (int64_t)i * m.value_size] = (real)state[i][lane];
}

// A thread has a row of the state, or of its gradient (Back, from the last row to the first): dq, or dk and the initial state's gradient.
template <class T, class S, bool Back>
__global__ __launch_bounds__(kWalkThreads) void attention_walk_keys_kernel(Attention m, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                           const T *__restrict__ values, const S *__restrict__ gates,
                                                                           const real *__restrict__ first_state, const int32_t *__restrict__ offsets,
                                                                           const T *__restrict__ grad_outputs, double *__restrict__ out,
                                                                           double *__restrict__ last_state) {
    __shared__ double state[kMost][kWalkThreads];
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), lane = threadIdx.x, i = blockIdx.y * kWalkThreads + lane;
    if (i >= m.key_size) return;
    const AttentionRows rows = rows_of(m, offsets, s);
    const T *q = queries + place_of(m, m.q, s, rows.first, h / m.shared), *k = keys + place_of(m, m.k, s, rows.first, h / m.shared),
            *v = values + place_of(m, m.v, s, rows.first, h), *g = grad_outputs ? grad_outputs + place_of(m, m.g, s, rows.first, h) : nullptr;
    const int64_t at = ((s * m.heads + h) * m.key_size + i) * m.value_size;
    for (int j = 0; j < m.value_size; j++) state[j][lane] = first_state ? (double)first_state[at + j] : 0.0;
    for (int64_t n = 0; n < rows.count; n++) {
        const int64_t t = Back ? rows.count - 1 - n : n;
        const double a = exp2(log2_gate(m.gate_form, (real)gates[m.fixed ? h : (rows.first + t) * m.heads + h]));
        const double x = Back ? wide(q[t * m.q.row + i]) * (double)m.scale : wide(k[t * m.k.row + i]);
        double sum = 0.0;
        for (int j = 0; j < m.value_size; j++) {
            const double y = wide(v[t * m.v.row + j]), d = g ? wide(g[t * m.g.row + j]) : 0.0;
            const double next = (Back ? state[j][lane] : a * state[j][lane]) + x * (Back ? d : y);
            state[j][lane] = Back ? a * next : next;
            sum += next * (Back ? y : d);
        }
        out[((rows.first + t) * m.heads + h) * m.key_size + i] = Back ? sum : sum * (double)m.scale;
    }
    if (Back)
        for (int j = 0; j < m.value_size; j++) last_state[at + j] = state[j][lane];
}

template <class T, class S>
__global__ __launch_bounds__(kWalkThreads) void attention_walk_values_kernel(Attention m, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                             const S *__restrict__ gates, const real *__restrict__ grad_final,
                                                                             const int32_t *__restrict__ offsets, const T *__restrict__ grad_outputs,
                                                                             T *__restrict__ grad_values) {
    __shared__ double state[kMost][kWalkThreads];
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), lane = threadIdx.x, j = blockIdx.y * kWalkThreads + lane;
    if (j >= m.value_size) return;
    const AttentionRows rows = rows_of(m, offsets, s);
    const T *q = queries + place_of(m, m.q, s, rows.first, h / m.shared), *k = keys + place_of(m, m.k, s, rows.first, h / m.shared),
            *g = grad_outputs ? grad_outputs + place_of(m, m.g, s, rows.first, h) : nullptr;
    const int64_t at = (s * m.heads + h) * m.key_size * m.value_size + j;
    for (int i = 0; i < m.key_size; i++) state[i][lane] = grad_final ? (double)grad_final[at + (int64_t)i * m.value_size] : 0.0;
    for (int64_t t = rows.count - 1; t >= 0; t--) {
        const double a = exp2(log2_gate(m.gate_form, (real)gates[m.fixed ? h : (rows.first + t) * m.heads + h]));
        const double d = g ? wide(g[t * m.g.row + j]) * (double)m.scale : 0.0;
        double sum = 0.0;
        for (int i = 0; i < m.key_size; i++) {
            const double next = state[i][lane] + wide(q[t * m.q.row + i]) * d;
            state[i][lane] = a * next;
            sum += wide(k[t * m.k.row + i]) * next;
        }
        grad_values[((rows.first + t) * m.heads + h) * m.value_size + j] = (T)(real)sum;
    }
}

// A workgroup has a sequence and head: dlog a from row to row.
template <class T, class S>
__global__ __launch_bounds__(kWalkThreads) void attention_walk_gates_kernel(Attention m, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                            const S *__restrict__ gates, const real *__restrict__ initial,
                                                                            const int32_t *__restrict__ offsets, const double *__restrict__ dq,
                                                                            const double *__restrict__ dk, const double *__restrict__ dstate,
                                                                            S *__restrict__ grad_gates, double *__restrict__ sums) {
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), lane = threadIdx.x;
    const AttentionRows rows = rows_of(m, offsets, s);
    const T *q = queries + place_of(m, m.q, s, rows.first, h / m.shared), *k = keys + place_of(m, m.k, s, rows.first, h / m.shared);
    const int64_t size = (int64_t)m.key_size * m.value_size, at = (s * m.heads + h) * size;
    double log_a = 0.0, all = 0.0;
    if (initial)
        for (int64_t i = lane; i < size; i += kWalkThreads) log_a += (double)initial[at + i] * dstate[at + i];
    log_a = sum_lanes(log_a, 64);
    for (int64_t t = 0; t < rows.count; t++) {
        const int64_t row = rows.first + t, here = (row * m.heads + h) * m.key_size;
        all += log_a;
        if (!m.fixed && lane == 0)
            grad_gates[row * m.heads + h] = (S)(real)(log_a * slope_of(m.gate_form, wide(gates[row * m.heads + h])));
        double change = 0.0;
        for (int i = lane; i < m.key_size; i += kWalkThreads)
            change += wide(k[t * m.k.row + i]) * dk[here + i] - wide(q[t * m.q.row + i]) * dq[here + i];
        log_a += sum_lanes(change, 64);
    }
    if (m.fixed && lane == 0) sums[s * m.heads + h] = all;
}

#else
// ---- units of chunks -------------------------------------------------------------------

constexpr int kPlanThreads = 1024, kScanThreads = 256;

__device__ __forceinline__ int64_t units_of(const AttentionCall &c, int64_t s, int64_t unit_rows, int64_t &first) {
    if (!c.m.packed) {
        first = s * c.units;
        return c.units;
    }
    first = c.plan[c.most_units + s];
    return max((int64_t)0, min((rows_of(c.m, c.offsets, s).count + unit_rows - 1) / unit_rows, c.most_units - first));
}

// Packed sequences' units: which sequence each is of, and every sequence's first.  One workgroup.
__global__ __launch_bounds__(kPlanThreads) void attention_plan_kernel(Attention m, const int32_t *__restrict__ offsets, int64_t unit_rows, int64_t most, int32_t *plan) {
    __shared__ int64_t waves[kPlanThreads / kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int64_t before = 0;
    for (int64_t first = 0; first < m.sequences; first += kPlanThreads) {
        const int64_t s = first + threadIdx.x, n = s < m.sequences ? (rows_of(m, offsets, s).count + unit_rows - 1) / unit_rows : 0;
        int64_t sum = n;
#pragma unroll
        for (int step = 1; step < kWave; step *= 2) {
            const int64_t other = __shfl_up(sum, step);
            if (lane >= step) sum += other;
        }
        if (lane == kWave - 1) waves[wave] = sum;
        __syncthreads();
        int64_t at = before + sum - n;
        for (int w = 0; w < kPlanThreads / kWave; w++) {
            if (w < wave) at += waves[w];
            before += waves[w];
        }
        if (s < m.sequences) {
            plan[most + s] = (int32_t)min(at, most);
            for (int64_t i = at; i < min(at + n, most); i++) plan[i] = (int32_t)s;
        }
        __syncthreads();
    }
    for (int64_t i = before + threadIdx.x; i < most; i += kPlanThreads) plan[i] = -1;
}

// From what units add to a state, the states in front of them (or behind them, from the last to the first): x' = decay x + added.  A thread has V
// neighbours of the state and reads eight units ahead.  136 units, of 37 sequences, of 16 states of 64 x 128: 34 us, 4.2 TB/s (52 with V = 1).
template <int V>
__global__ __launch_bounds__(kScanThreads) void attention_scan_kernel(AttentionCall c, float *__restrict__ states, const float *__restrict__ from, float *__restrict__ to,
                                                                      float *__restrict__ kept, int64_t unit_rows, bool back) {
    constexpr int kAhead = 8;
    const int64_t s = blockIdx.x / c.m.heads, size = (int64_t)c.m.key_size * c.m.value_size, i = ((int64_t)blockIdx.y * kScanThreads + threadIdx.x) * V;
    const int head = (int)(blockIdx.x % c.m.heads);
    if (i >= size) return;
    int64_t first;
    const int64_t count = units_of(c, s, unit_rows, first);
    Pack<float, V> x = {};
    if (from) x = load_pack<V>(from + (s * c.m.heads + head) * size + i);
    for (int64_t n = 0; n < count; n += kAhead) {
        Pack<float, V> added[kAhead];
        float decay[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t here = min(n + j, count - 1), unit = (first + (back ? count - 1 - here : here)) * c.m.heads + head;
            added[j] = load_pack<V>(states + unit * size + i);
            decay[j] = c.decays[unit];
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int64_t unit = (first + (back ? count - 1 - n - j : n + j)) * c.m.heads + head;
            if (n + j < count) {
                store_pack<V>(states + unit * size + i, x.v);
#pragma unroll
                for (int v = 0; v < V; v++) x.v[v] = fmaf(decay[j], x.v[v], added[j].v[v]);
            }
        }
    }
    if (to) store_pack<V>(to + (s * c.m.heads + head) * size + i, x.v);
    if (kept) store_pack<V>(kept + (s * c.m.heads + head) * size + i, x.v);
}

// dlog a of a unit's rows: <S, D> in front of it, and what changes it from row to row.  What is missing at the unit's end to <S, D> behind it, the sum of
// roundings, goes to the rows in the share of their changes' squares: of a walk whose both ends are known a third of the variance is left.  It reads
// every state twice (once from the cache): 256 units' states of 128 x 128 in 18 us.
template <class S> __global__ __launch_bounds__(kScanThreads) void attention_gates_kernel(AttentionCall c, int64_t rows_of_chunk, const float *__restrict__ in_front) {
    __shared__ double waves[kScanThreads / kWave];
    const int64_t u = blockIdx.x / c.m.heads, size = (int64_t)c.m.key_size * c.m.value_size;
    const int head = (int)(blockIdx.x % c.m.heads), lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const Unit unit = rows_of_chunk == 32 ? unit_of<32>(c, u) : unit_of<64>(c, u);
    if (!unit.there) {
        if (c.m.fixed && threadIdx.x == 0) c.sums[u * c.m.heads + head] = 0.0;
        return;
    }
    const auto over_waves = [&](double v, double &all) {  // -> the sum over waves before this one
        __syncthreads();
        if (lane == kWave - 1) waves[wave] = v;
        __syncthreads();
        double before = 0.0;
        all = 0.0;
        for (int w = 0; w < kScanThreads / kWave; w++) {
            if (w < wave) before += waves[w];
            all += waves[w];
        }
        return before;
    };
    const auto product_of = [&](const float *state, const float *gradient) {  // this thread's part
        double product = 0.0;
        // eight products are added in float32, all others in 64 bits
#pragma unroll 2
        for (int64_t first = threadIdx.x; first < size; first += 8 * kScanThreads) {
            float x[8], y[8], sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int64_t at = min(first + j * kScanThreads, size - 1);
                x[j] = state[at];
                y[j] = gradient[at];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) sum = first + j * kScanThreads < size ? fmaf(x[j], y[j], sum) : sum;
            product += (double)sum;
        }
        return product;
    };
    const int64_t of_unit = (u * c.m.heads + head) * size, next = c.m.heads * size, of_sequence = (unit.sequence * c.m.heads + head) * size;
    const bool last_unit = unit.base + unit.count >= rows_of(c.m, c.offsets, unit.sequence).count;
    double product = 0.0, product_behind = 0.0, all, at_end;
    if (unit.index > 0)
        product = product_of(c.states + of_unit, c.grad_states + of_unit - next);
    else if (in_front)
        product = product_of(c.states + of_unit, in_front + of_sequence);
    if (!last_unit && u + 1 < c.most_units)
        product_behind = product_of(c.states + of_unit + next, c.grad_states + of_unit);
    else if (last_unit && c.grad_final)
        product_behind = product_of(c.finals + of_sequence, c.grad_final + of_sequence);
    over_waves(sum_lanes(product, kWave), all);
    over_waves(sum_lanes(product_behind, kWave), at_end);
    double log_a = all;  // of the first row
    const int64_t each = (unit.count + kScanThreads - 1) / kScanThreads, first = min(unit.count, threadIdx.x * each), last = min(unit.count, first + each);
    const int64_t at = head * c.m.rows + unit.first;
    double sum = 0.0, squares = 0.0, all_squares;
    const auto change_at = [&](int64_t t, double &square) {
        const double up = c.changes[1][at + t], down = c.changes[0][at + t];
        square = up * up + down * down;
        return up - down;
    };
    for (int64_t t = first; t < last; t++) {
        double square;
        sum += change_at(t, square);
        squares += square;
    }
    double upto = sum, squares_upto = squares;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
        const double other = __shfl_up(upto, step), other_squares = __shfl_up(squares_upto, step);
        if (lane >= step) upto += other, squares_upto += other_squares;
    }
    const double before = over_waves(upto, all) + upto - sum, squares_before = over_waves(squares_upto, all_squares) + squares_upto - squares;
    const double share = all_squares > 0.0 ? (at_end - (log_a + all)) / all_squares : 0.0;  // of what is missing, for a square
    log_a += before + share * squares_before;
    double total = 0.0;
    for (int64_t t = first; t < last; t++) {
        total += log_a;
        const int64_t to = (unit.first + t) * c.m.heads + head;
        if (!c.m.fixed) ((S *)c.grad_gates)[to] = (S)(float)(log_a * slope_of(c.m.gate_form, (double)(float)((const S *)c.gates)[to]));
        double square;
        const double change = change_at(t, square);
        log_a += change + share * square;
    }
    if (c.m.fixed) {
        over_waves(sum_lanes(total, kWave), all);
        if (threadIdx.x == 0) c.sums[u * c.m.heads + head] = all;
    }
}
#endif  // TG_DOUBLE_PRECISION

template <class S>
__global__ void attention_fixed_gates_kernel(Attention m, const S *__restrict__ gates, const double *__restrict__ sums, int64_t parts, S *__restrict__ grad_gates) {
    const int h = blockIdx.x;
    double all = 0.0;
    for (int64_t n = threadIdx.x; n < parts; n += kWalkThreads) all += sums[n * m.heads + h];
    all = sum_lanes(all, 64);
    if (threadIdx.x == 0) grad_gates[h] = (S)(real)(all * slope_of(m.gate_form, wide(gates[h])));
}

constexpr int kSharedThreads = 256;

// Key heads' gradients, the sums of their value heads': of queries (y = 0) and of keys.  A row of `lanes` threads (a power of two) has one key head of
// one row, a thread V of its numbers.  30011 rows of 16 heads of 64 into 4 key heads' in float16: 50 us for both, 5.5 TB/s.
template <class T, class P, int V> struct SharedParts {
    const P *parts[2];
    T *out[2];
};
template <class T, class P, int V> __global__ __launch_bounds__(kSharedThreads) void attention_shared_kernel(Attention m, int lanes, SharedParts<T, P, V> both) {
    const P *parts = both.parts[blockIdx.y];
    T *out = both.out[blockIdx.y];
    const int i = threadIdx.x % lanes * V;
    if (!out || i >= m.key_size) return;
    const int64_t step = (int64_t)gridDim.x * (kSharedThreads / lanes);
    for (int64_t head = (int64_t)blockIdx.x * (kSharedThreads / lanes) + threadIdx.x / lanes; head < m.rows * m.key_heads; head += step) {  // row and key head
        P sum[V] = {};
#pragma unroll 4
        for (int n = 0; n < m.shared; n++) {
            const Pack<P, V> part = load_pack<V>(parts + (head * m.shared + n) * m.key_size + i);
#pragma unroll
            for (int v = 0; v < V; v++) sum[v] += part.v[v];
        }
        real to[V];
#pragma unroll
        for (int v = 0; v < V; v++) to[v] = (real)sum[v];
        store_pack<V>(out + head * m.key_size + i, to);
    }
}

// Rows in front of the first sequence and behind the last one: zeros, in each of up to four tensors (y) whose rows have `width` pieces of 16 bits.
struct Outside {
    uint16_t *out[4];
    int64_t width[4];
};
__global__ void attention_outside_kernel(Attention m, const int32_t *__restrict__ offsets, Outside all) {
    const AttentionRows first = rows_of(m, offsets, 0), last = rows_of(m, offsets, m.sequences - 1);
    const int64_t end = last.first + last.count, begin = min(first.first, end), outside = m.rows - end + begin, width = all.width[blockIdx.y];
    for (int64_t row = blockIdx.x; row < outside; row += gridDim.x) {
        uint16_t *out = all.out[blockIdx.y] + (row < begin ? row : row - begin + end) * width;
        for (int64_t i = threadIdx.x; i < width; i += blockDim.x) out[i] = 0;
    }
}

// ---- host ---------------------------------------------------------------------------------

int attention_shape(const char *fn, const tg_attention &a, Attention &m) {
    if (a.sequences < 0 || a.length < 0 || a.heads < 1 || a.key_heads < 1 || a.heads % a.key_heads != 0 || a.key_size < 1 || a.value_size < 1 ||
        a.key_size > kMost || a.value_size > kMost) {
        set_error("%s: sizes (heads: a multiple of key_heads; key_size and value_size: 1 to %d)", fn, kMost);
        return TG_E_ARG;
    }
    if (!type_known(a.type) || (a.gate_type != a.type && a.gate_type != kRealType)) {
        set_error("%s: types %lld and %lld", fn, (long long)a.type, (long long)a.gate_type);
        return TG_E_ARG;
    }
    if (a.gate_form != TG_GATE_LOG && a.gate_form != TG_GATE_LOGIT) {
        set_error("%s: gate_form %lld", fn, (long long)a.gate_form);
        return TG_E_ARG;
    }
    const int64_t limit = (int64_t)1 << 40, heads = a.heads;
    const int64_t rows = a.offsets ? a.length : a.length == 0 ? 0 : a.sequences > limit / a.length ? limit : a.sequences * a.length;
    if (heads >= (1 << 16) || a.length > 0x7fffffff || a.sequences >= ((int64_t)1 << 29) || rows >= limit / (heads * kMost) ||
        a.sequences >= ((int64_t)1 << 31) / heads) {
        set_error("%s: %lld rows, %lld sequences of %lld heads are too many", fn, (long long)rows, (long long)a.sequences, (long long)heads);
        return TG_E_ARG;
    }
    const auto strides = [](const int64_t s[3]) { return Strides{s[0], s[1], s[2]}; };
    m = {a.sequences, a.length, rows, (int)a.heads, (int)a.key_heads, (int)(a.heads / a.key_heads), (int)a.key_size, (int)a.value_size,
         strides(a.query_strides), strides(a.key_strides), strides(a.value_strides), strides(a.grad_strides),
         (int)a.gate_form, a.fixed_gates != 0, a.offsets != nullptr, (real)a.scale};
    return 0;
}

// A workgroup of `threads` for each sequence and head.
static int refuse_many(const char *fn, const Attention &m, int threads) {
    if (m.sequences * m.heads < kGridThreads / threads) return 0;
    set_error("%s: %lld sequences of %d heads are too many", fn, (long long)m.sequences, m.heads);
    return TG_E_ARG;
}

static void clear_outside(const tg_attention &a, const Attention &m, std::initializer_list<std::pair<void *, int64_t>> tensors) {  // and bytes of a row
    Outside all = {};
    unsigned n = 0;
    for (const auto &t : tensors)
        if (t.first) all.out[n] = (uint16_t *)t.first, all.width[n++] = t.second / 2;
    if (!m.packed || !m.rows || !n) return;
    TG_LAUNCH_AS("attention_outside", attention_outside_kernel, dim3((unsigned)std::min<int64_t>(m.rows, 1024), n), dim3(256), 0, (hipStream_t)a.stream, m, a.offsets, all);
}
template <class T> static void clear_outputs(const tg_attention &a, const Attention &m) {
    clear_outside(a, m, {{a.outputs, (int64_t)sizeof(T) * m.heads * m.value_size}});
}
template <class T, class S> static void clear_gradients(const tg_attention &a, const Attention &m) {
    const int64_t keys = (int64_t)sizeof(T) * m.key_heads * m.key_size;
    clear_outside(a, m, {{a.grad_queries, keys}, {a.grad_keys, keys}, {a.grad_values, (int64_t)sizeof(T) * m.heads * m.value_size},
                         {m.fixed ? nullptr : a.grad_gates, (int64_t)sizeof(S) * m.heads}});
}

template <class T, class P> static void add_shared(const tg_attention &a, const Attention &m, const P *queries, const P *keys) {
    const auto launch = [&](auto vector) {
        constexpr int V = decltype(vector)::value;
        int lanes = 1;
        while (lanes * V < m.key_size) lanes *= 2;
        const SharedParts<T, P, V> both = {{queries, keys}, {(T *)a.grad_queries, (T *)a.grad_keys}};
        const int64_t groups = ceil_div64(m.rows * m.key_heads, kSharedThreads / lanes);
        TG_LAUNCH_AS("attention_shared", (attention_shared_kernel<T, P, V>), dim3((unsigned)std::min<int64_t>(groups, 1 << 16), 2), dim3(kSharedThreads), 0,
                     (hipStream_t)a.stream, m, lanes, both);
    };
    if (!m.rows || (!a.grad_queries && !a.grad_keys)) return;
    constexpr int kWidest = 16 / (int)sizeof(P);
    if (m.key_size % kWidest == 0 && (uintptr_t)a.grad_queries % 16 == 0 && (uintptr_t)a.grad_keys % 16 == 0 && (uintptr_t)a.workspace % 16 == 0)
        launch(std::integral_constant<int, kWidest>());
    else
        launch(std::integral_constant<int, 1>());
}

#ifdef TG_DOUBLE_PRECISION
struct WalkRoom {
    int64_t dq, dk, dstate, sums, all;
};
static WalkRoom walk_room(const Attention &m) {
    WalkRoom r;
    r.dq = 0;
    r.dk = r.dq + m.rows * m.heads * m.key_size * 8;
    r.dstate = r.dk + m.rows * m.heads * m.key_size * 8;
    r.sums = r.dstate + m.sequences * m.heads * m.key_size * m.value_size * 8;
    r.all = r.sums + (m.fixed ? m.sequences * m.heads * 8 : 0);
    return r;
}

template <class T, class S> static int walk_forward(const tg_attention &a, const Attention &m) {
    const hipStream_t stream = (hipStream_t)a.stream;
    TG_LAUNCH_AS("attention_walk", (attention_walk_kernel<T, S>), dim3((unsigned)(m.sequences * m.heads), (unsigned)ceil_div(m.value_size, kWalkThreads)),
                 dim3(kWalkThreads), 0, stream, m, (const T *)a.queries, (const T *)a.keys, (const T *)a.values, (const S *)a.gates, a.initial, a.offsets,
                 (T *)a.outputs, a.final);
    clear_outputs<T>(a, m);
    return check_launch("tg_linear_attention_forward");
}

template <class T> static __global__ void attention_round_kernel(const double *__restrict__ in, int64_t n, T *__restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) out[i] = (T)in[i];
}

template <class T, class S> static int walk_backward(const tg_attention &a, const Attention &m) {
    const hipStream_t stream = (hipStream_t)a.stream;
    const WalkRoom room = walk_room(m);
    char *w = (char *)a.workspace;
    double *dq = (double *)(w + room.dq), *dk = (double *)(w + room.dk), *dstate = (double *)(w + room.dstate), *sums = (double *)(w + room.sums);
    const unsigned heads = (unsigned)(m.sequences * m.heads);
    const dim3 keys(heads, (unsigned)ceil_div(m.key_size, kWalkThreads)), values(heads, (unsigned)ceil_div(m.value_size, kWalkThreads));
    const T *q = (const T *)a.queries, *k = (const T *)a.keys, *v = (const T *)a.values, *g = (const T *)a.grad_outputs;
    const S *gates = (const S *)a.gates;
    TG_LAUNCH_AS("attention_walk_queries", (attention_walk_keys_kernel<T, S, false>), keys, dim3(kWalkThreads), 0, stream, m, q, k, v, gates, a.initial, a.offsets,
                 g, dq, (double *)nullptr);
    TG_LAUNCH_AS("attention_walk_keys", (attention_walk_keys_kernel<T, S, true>), keys, dim3(kWalkThreads), 0, stream, m, q, k, v, gates, a.grad_final, a.offsets,
                 g, dk, dstate);
    if (a.grad_values)
        TG_LAUNCH_AS("attention_walk_values", (attention_walk_values_kernel<T, S>), values, dim3(kWalkThreads), 0, stream, m, q, k, gates, a.grad_final, a.offsets,
                     g, (T *)a.grad_values);
    if (a.grad_gates) {
        TG_LAUNCH_AS("attention_walk_gates", (attention_walk_gates_kernel<T, S>), dim3(heads), dim3(kWalkThreads), 0, stream, m, q, k, gates, a.initial, a.offsets,
                     dq, dk, dstate, (S *)a.grad_gates, sums);
        if (m.fixed)
            TG_LAUNCH_AS("attention_fixed_gates", (attention_fixed_gates_kernel<S>), dim3((unsigned)m.heads), dim3(kWalkThreads), 0, stream, m, gates, sums,
                         m.sequences, (S *)a.grad_gates);
    }
    const int64_t states = m.sequences * m.heads * m.key_size * m.value_size;
    if (a.grad_initial)
        TG_LAUNCH_AS("attention_round", (attention_round_kernel<real>), dim3((unsigned)std::min<int64_t>(ceil_div64(states, 256), 1 << 20)), dim3(256), 0, stream, dstate, states, a.grad_initial);
    add_shared<T>(a, m, dq, dk);
    clear_gradients<T, S>(a, m);
    return check_launch("tg_linear_attention_backward");
}

static int64_t room_for_walk(const Attention &m) { return walk_room(m).all; }

static int sizes_of(const char *fn, const tg_attention &, const Attention &m, int64_t out[4]) {
    const int code = refuse_many(fn, m, kWalkThreads);
    if (code) return code;
    out[0] = out[1] = out[2] = 0;
    out[3] = room_for_walk(m);
    return 0;
}
static int forward(const tg_attention &a, const Attention &m) { return walk_forward<real, real>(a, m); }
static int backward(const tg_attention &a, const Attention &m) { return walk_backward<real, real>(a, m); }

#else

static_assert(Parts<bf16_t>::kRows == Parts<half_t>::kRows, "rows of a chunk");
constexpr int64_t kComputeUnits = 256;
constexpr int64_t kMostChunks = 16;   // of a unit: 1024 rows, beside whose 16 chunks a state that is written and read is little
constexpr int64_t kMostUnits = 1024;  // of a sequence, which are gone through one after another
// How the rows of a call are split, the same forward and backward.
struct Split {
    int64_t rows_of_chunk, chunks, units, most_units, size;
    bool through;
};
static int split_of(const char *fn, const tg_attention &a, const Attention &m, Split &s) {
    s.rows_of_chunk = a.type == TG_TYPE_F32 ? Parts<float>::kRows : Parts<bf16_t>::kRows;
    s.size = std::max(m.key_size, m.value_size) <= 32 ? 32 : std::max(m.key_size, m.value_size) <= 64 ? 64 : 128;
    const int64_t of_one = ceil_div64(m.length, s.rows_of_chunk);
    s.chunks = 0;
    // Chunks of a unit, as if a compute unit took its units one after another, and a unit, whose state is written and read, as long as its chunks and two
    // more (four of half the rows).  2 x 3000 rows of 8 heads in float32: six chunks, 256 units, 184 us forward and backward; five, 304 units, 282.  Of
    // heads of at most 64 a compute unit has two or three at once, and packed sequences' last units are half empty: neither is in the model.
    int64_t least = 0;
    for (int64_t n = std::max<int64_t>(1, ceil_div64(of_one, kMostUnits)), most = std::max(n, kMostChunks); n <= most; n++) {
        const int64_t units = (m.packed ? of_one / n + m.sequences : ceil_div64(of_one, n) * m.sequences) * m.heads;
        const int64_t time = ceil_div64(units, kComputeUnits) * (n + 128 / s.rows_of_chunk);
        if (s.chunks == 0 || time < least) {
            s.chunks = n;
            least = time;
        }
    }
    s.units = ceil_div64(m.length, s.rows_of_chunk * s.chunks);
    s.most_units = m.packed ? m.length / (s.rows_of_chunk * s.chunks) + m.sequences : s.units * m.sequences;
    // sequences and heads enough: the forward pass goes through each from its first row to its last, and reads keys and values once
    s.through = s.units <= 1 || (!m.packed && m.sequences * m.heads >= 2 * kComputeUnits);
    if (s.most_units * m.heads >= kGridThreads / (8 * s.size) || m.sequences * m.heads >= kGridThreads / (8 * s.size) || s.most_units > 0x7fffffff) {
        set_error("%s: %lld rows, %lld sequences of %d heads are too many", fn, (long long)m.rows, (long long)m.sequences, m.heads);
        return TG_E_ARG;
    }
    return 0;
}

// Bytes from the beginning of what the forward call leaves, or of a workspace.
struct Room {
    int64_t states, finals, decays, plan, grad_states, changes, sums, grad_initial, shared_queries, shared_keys, all;
};
static Room room_of(const tg_attention &a, const Attention &m, const Split &s, bool states, bool backward) {
    Room r = {};
    int64_t at = 0;
    const auto take = [&](bool wanted, int64_t bytes) {
        const int64_t here = at;
        if (wanted) at += ceil_div64(bytes, 16) * 16;
        return here;
    };
    const int64_t size = (int64_t)m.key_size * m.value_size * 4, units = s.most_units * m.heads;
    r.states = take(states, units * size);
    r.finals = take(states, m.sequences * m.heads * size);
    r.plan = take(states && m.packed, (s.most_units + m.sequences) * 4);
    r.decays = take(backward || !states, units * 4);
    r.grad_states = take(backward, units * size);
    r.changes = take(backward, 2 * m.rows * m.heads * 8);
    r.sums = take(backward && m.fixed, units * 8);
    r.grad_initial = take(backward && a.initial, m.sequences * m.heads * size);
    r.shared_queries = take(backward && m.shared > 1, m.rows * m.heads * m.key_size * 4);
    r.shared_keys = take(backward && m.shared > 1, m.rows * m.heads * m.key_size * 4);
    r.all = at;
    return r;
}

static int sizes_of(const char *fn, const tg_attention &a, const Attention &m, int64_t out[4]) {
    Split s;
    const int code = split_of(fn, a, m, s);
    if (code) return code;
    const int64_t kept = room_of(a, m, s, true, false).all, decays = room_of(a, m, s, false, false).all;
    out[0] = kept;
    out[1] = s.through ? 0 : kept + decays;
    out[2] = s.through ? 0 : decays;
    tg_attention with = a;
    static const real some = 0;
    with.initial = &some;  // whether there is one need not be known yet
    out[3] = room_of(with, m, s, false, true).all;
    return 0;
}

static bool in_vectors(const tg_attention &a, const Attention &m) {
    const int64_t bytes = type_bytes(a.type);
    if (m.key_size * bytes % 16 != 0 || m.value_size * bytes % 16 != 0) return false;
    for (const void *p : {a.queries, a.keys, a.values, (const void *)a.outputs, a.grad_outputs, (const void *)a.grad_queries, (const void *)a.grad_keys, (const void *)a.grad_values})
        if ((uintptr_t)p % 16 != 0) return false;
    const auto dense = [&](const Strides &t, int heads) {
        return (m.packed || m.sequences == 1 || t.sequence * bytes % 16 == 0) && (m.length == 1 || t.row * bytes % 16 == 0) && (heads == 1 || t.head * bytes % 16 == 0);
    };
    return dense(m.q, m.key_heads) && dense(m.k, m.key_heads) && dense(m.v, m.heads) && (!a.grad_outputs || dense(m.g, m.heads));
}

static AttentionCall call_of(const tg_attention &a, const Attention &m, const Split &s) {
    AttentionCall c = {};
    c.m = m;
    c.queries = a.queries;
    c.keys = a.keys;
    c.values = a.values;
    c.gates = a.gates;
    c.initial = a.initial;
    c.offsets = a.offsets;
    c.outputs = a.outputs;
    c.final = a.final;
    c.most_units = s.most_units;
    c.units = s.units;
    c.chunks = (int)s.chunks;
    c.wide_gates = a.gate_type == TG_TYPE_F32;
    c.vector = in_vectors(a, m);
    c.through = s.through;
    c.grad_outputs_there = a.grad_outputs != nullptr;
    c.grad_outputs = a.grad_outputs ? a.grad_outputs : a.values;
    if (!a.grad_outputs) c.m.g = m.v;
    c.grad_final = a.grad_final;
    c.grad_values = a.grad_values;
    c.grad_gates = a.grad_gates;
    return c;
}

static void scan(const AttentionCall &c, const Split &s, float *states, const float *from, float *to, float *kept, bool back, hipStream_t stream) {
    const int64_t size = (int64_t)c.m.key_size * c.m.value_size;
    const auto launch = [&](auto vector) {
        constexpr int V = decltype(vector)::value;
        TG_LAUNCH_AS("attention_scan", (attention_scan_kernel<V>), dim3((unsigned)(c.m.sequences * c.m.heads), (unsigned)ceil_div64(size, kScanThreads * V)),
                     dim3(kScanThreads), 0, stream, c, states, from, to, kept, s.rows_of_chunk * s.chunks, back);
    };
    if (size % 4 == 0 && ((uintptr_t)states | (uintptr_t)from | (uintptr_t)to | (uintptr_t)kept) % 16 == 0)
        launch(std::integral_constant<int, 4>());
    else
        launch(std::integral_constant<int, 1>());
}

static int forward(const tg_attention &a, const Attention &m) {
    const hipStream_t stream = (hipStream_t)a.stream;
    Split s;
    int code = split_of("tg_linear_attention_forward", a, m, s);
    if (code) return code;
    AttentionCall c = call_of(a, m, s);
    const bool kept = a.kept != nullptr;
    if (kept || !s.through) {
        const Room room = room_of(a, m, s, true, false);
        char *p = (char *)(kept ? a.kept : a.workspace);
        c.states = (float *)(p + room.states);
        c.finals = kept ? (float *)(p + room.finals) : nullptr;
        c.plan = (const int32_t *)(p + room.plan);
        c.decays = (float *)((char *)a.workspace + (kept ? 0 : room.all));
        if (m.packed)
            TG_LAUNCH_AS("attention_plan", attention_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, m, a.offsets, s.rows_of_chunk * s.chunks, s.most_units,
                         (int32_t *)(p + room.plan));
    }
    if (m.rows == 0 || s.through) {
        c.through = true;
    } else {
        if ((code = launch_attention_forward(a.type, c, (int)s.size, true, stream))) return code;
        scan(c, s, c.states, a.initial, a.final, c.finals, false, stream);
    }
    if ((code = launch_attention_forward(a.type, c, (int)s.size, false, stream))) return code;
    return by_types(a.type, a.gate_type, [&](auto t, auto) {
        clear_outputs<decltype(t)>(a, m);
        return check_launch("tg_linear_attention_forward");
    });
}

template <class T, class S> static int backward(const tg_attention &a, const Attention &m) {
    const hipStream_t stream = (hipStream_t)a.stream;
    Split s;
    int code = split_of("tg_linear_attention_backward", a, m, s);
    if (code) return code;
    AttentionCall c = call_of(a, m, s);
    const Room kept = room_of(a, m, s, true, false), room = room_of(a, m, s, false, true);
    char *w = (char *)a.workspace;
    c.states = (float *)((char *)a.kept + kept.states);
    c.finals = (float *)((char *)a.kept + kept.finals);
    c.plan = (const int32_t *)((char *)a.kept + kept.plan);
    c.decays = (float *)(w + room.decays);
    c.grad_states = (float *)(w + room.grad_states);
    c.changes[0] = (double *)(w + room.changes);
    c.changes[1] = c.changes[0] + m.rows * m.heads;
    c.sums = (double *)(w + room.sums);
    c.grad_queries = m.shared > 1 && a.grad_queries ? w + room.shared_queries : a.grad_queries;
    c.grad_keys = m.shared > 1 && a.grad_keys ? w + room.shared_keys : a.grad_keys;
    float *in_front = a.initial && a.grad_gates ? (float *)(w + room.grad_initial) : nullptr;
    if (a.grad_initial) in_front = a.grad_initial;
    if (m.rows && (code = launch_attention_backward(a.type, c, (int)s.size, false, stream))) return code;
    scan(c, s, c.grad_states, a.grad_final, in_front, nullptr, true, stream);
    if (m.rows && (a.grad_keys || a.grad_values || a.grad_gates) && (code = launch_attention_backward(a.type, c, (int)s.size, true, stream))) return code;
    if (a.grad_gates) {
        if (m.rows)
            TG_LAUNCH_AS("attention_gates", (attention_gates_kernel<S>), dim3((unsigned)(s.most_units * m.heads)), dim3(kScanThreads), 0, stream, c, s.rows_of_chunk,
                         a.initial ? in_front : nullptr);
        if (m.fixed)
            TG_LAUNCH_AS("attention_fixed_gates", (attention_fixed_gates_kernel<S>), dim3((unsigned)m.heads), dim3(kWalkThreads), 0, stream, m, (const S *)a.gates, c.sums,
                         m.rows ? s.most_units : 0, (S *)a.grad_gates);
    }
    if (m.shared > 1) add_shared<T>(a, m, (const float *)c.grad_queries, (const float *)c.grad_keys);
    clear_gradients<T, S>(a, m);
    return check_launch("tg_linear_attention_backward");
}
static int backward(const tg_attention &a, const Attention &m) {
    return by_types(a.type, a.gate_type, [&](auto t, auto s) { return backward<decltype(t), decltype(s)>(a, m); });
}
#endif  // TG_DOUBLE_PRECISION

// ---- a single step ----------------------------------------------------------------------

constexpr int kStepThreads = 256;

__device__ __forceinline__ real decay_of(int form, real g) { return form == TG_GATE_LOGIT ? 1 / (1 + exp(-g)) : exp(g); }

// A workgroup has V x `lanes` columns of one state (lanes: a power of two), a thread V of them in every (256 / lanes)th row, eight rows on their way at
// once, the first ones while the key and the query come.  All there is to it is reading and writing states: 256 x 32 heads of 128 x 128, 205 us, 5.2 TB/s; 16 heads of
// 64 x 64, 4.6 us.
template <class T, class S, int V>
__global__ __launch_bounds__(kStepThreads) void attention_step_kernel(Attention m, int lanes, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                      const T *__restrict__ values, const S *__restrict__ gates, const real *state,
                                                                      T *__restrict__ outputs, real *new_state) {
    constexpr int kAhead = 8;
    __shared__ real q[kMost], k[kMost], partial[kStepThreads][V];
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), t = threadIdx.x;
    const int column = (blockIdx.y * lanes + (t & (lanes - 1))) * V, step = kStepThreads / lanes, first = t / lanes;
    const bool there = column < m.value_size;
    const int64_t at = (s * m.heads + h) * m.key_size * m.value_size + (there ? column : 0);
    Pack<real, V> before[kAhead];
    const auto load = [&](int from) {  // rows behind the last one: the last one, which nothing is made of
#pragma unroll
        for (int n = 0; n < kAhead; n++) before[n] = load_pack<V>(state + at + (int64_t)min(from + n * step, m.key_size - 1) * m.value_size);
    };
    load(first);
    const S gate = gates[m.fixed ? h : s * m.heads + h];
    T value[V];
#pragma unroll
    for (int j = 0; j < V; j++) value[j] = values[s * m.v.sequence + h * m.v.head + (there ? column + j : 0)];
    for (int i = t; i < m.key_size; i += kStepThreads) {
        q[i] = (real)queries[s * m.q.sequence + h / m.shared * m.q.head + i];
        k[i] = (real)keys[s * m.k.sequence + h / m.shared * m.k.head + i];
    }
    __syncthreads();
    real sum[V] = {};
    const real a = decay_of(m.gate_form, (real)gate);
    for (int from = first; from < m.key_size; from += kAhead * step) {
        if (from > first) load(from);
#pragma unroll
        for (int n = 0; n < kAhead; n++) {
            const int i = from + n * step;
            if (i >= m.key_size || !there) break;
            real next[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                next[j] = fma(a, before[n].v[j], k[i] * (real)value[j]);
                sum[j] = fma(q[i], next[j], sum[j]);
            }
            store_pack<V>(new_state + at + (int64_t)i * m.value_size, next);
        }
    }
    for (int apart = lanes; apart < kWave; apart *= 2)
#pragma unroll
        for (int j = 0; j < V; j++) sum[j] += __shfl_xor(sum[j], apart);
#pragma unroll
    for (int j = 0; j < V; j++) partial[t][j] = sum[j];
    __syncthreads();
    if (t >= lanes || !there) return;
    const int each = max(lanes, kWave);
#pragma unroll
    for (int j = 0; j < V; j++) {
        real all = 0;
        for (int i = t; i < kStepThreads; i += each) all += partial[i][j];
        outputs[(s * m.heads + h) * m.value_size + column + j] = (T)(all * (real)m.scale);
    }
}

template <class T, class S> static int step(const tg_attention &a, const Attention &m) {
    const auto launch = [&](auto vector) {
        constexpr int V = decltype(vector)::value;
        int lanes = 1;
        while (lanes * V < m.value_size) lanes *= 2;
        TG_LAUNCH_AS("attention_step", (attention_step_kernel<T, S, V>), dim3((unsigned)(m.sequences * m.heads), (unsigned)ceil_div(m.value_size, lanes * V)),
                     dim3(kStepThreads), 0, (hipStream_t)a.stream, m, lanes, (const T *)a.queries, (const T *)a.keys, (const T *)a.values, (const S *)a.gates,
                     a.initial, (T *)a.outputs, a.final);
    };
    constexpr int kWidest = 16 / (int)sizeof(real);
    if (m.value_size % kWidest == 0 && (uintptr_t)a.initial % 16 == 0 && (uintptr_t)a.final % 16 == 0)
        launch(std::integral_constant<int, kWidest>());
    else
        launch(std::integral_constant<int, 1>());
    return check_launch("tg_linear_attention_step");
}

}  // namespace tg

using namespace tg;

static int check_pointers(const char *fn, std::initializer_list<const void *> needed) {
    for (const void *p : needed)
        if (!p) {
            set_error("%s: null pointer", fn);
            return TG_E_ARG;
        }
    return 0;
}

extern "C" int tg_linear_attention_sizes(const tg_attention *a, int64_t out[4]) {
    const char *fn = "tg_linear_attention_sizes";
    if (!a || !out) return check_pointers(fn, {a, out});
    Attention m;
    const int code = attention_shape(fn, *a, m);
    return code ? code : sizes_of(fn, *a, m, out);
}

// A fixed decay has a gradient of zero then.
static int no_sequences(const tg_attention &a, const Attention &m) {
    if (!m.fixed || !a.grad_gates) return 0;
    return by_types(a.type, a.gate_type, [&](auto, auto s) {
        using S = decltype(s);
        TG_LAUNCH_AS("attention_fixed_gates", (attention_fixed_gates_kernel<S>), dim3((unsigned)m.heads), dim3(kWalkThreads), 0, (hipStream_t)a.stream, m,
                     (const S *)a.gates, (const double *)nullptr, (int64_t)0, (S *)a.grad_gates);
        return check_launch("tg_linear_attention_backward");
    });
}

static int attention_call(const char *fn, const tg_attention *a, bool backward_pass) {
    if (!a) return check_pointers(fn, {a});
    Attention m;
    int code = attention_shape(fn, *a, m);
    if (code) return code;
    int64_t sizes[4];
    if ((code = sizes_of(fn, *a, m, sizes))) return code;
    if (m.rows && (code = check_pointers(fn, {a->queries, a->keys, a->values, a->gates}))) return code;
    if (!backward_pass && m.sequences && (code = check_pointers(fn, {a->final}))) return code;
    if (!backward_pass && m.rows && (code = check_pointers(fn, {a->outputs}))) return code;
    if (backward_pass && sizes[0] && (code = check_pointers(fn, {a->kept}))) return code;
    if (a->kept && a->kept_bytes < sizes[0]) {
        set_error("%s: kept has %lld bytes, %lld needed", fn, (long long)a->kept_bytes, (long long)sizes[0]);
        return TG_E_WORKSPACE;
    }
    const int64_t room = sizes[backward_pass ? 3 : a->kept ? 2 : 1];
    if (a->workspace_bytes < room || (room && !a->workspace)) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)a->workspace_bytes, (long long)room);
        return TG_E_WORKSPACE;
    }
    if (((uintptr_t)a->kept | (uintptr_t)a->workspace) % 16 != 0) {
        set_error("%s: kept and workspace must be aligned to 16 bytes", fn);
        return TG_E_WORKSPACE;
    }
    if (m.sequences == 0) return backward_pass ? no_sequences(*a, m) : 0;
    return backward_pass ? backward(*a, m) : forward(*a, m);
}

extern "C" int tg_linear_attention_forward(const tg_attention *a) { return attention_call("tg_linear_attention_forward", a, false); }
extern "C" int tg_linear_attention_backward(const tg_attention *a) { return attention_call("tg_linear_attention_backward", a, true); }

extern "C" int tg_linear_attention_step(const tg_attention *a) {
    const char *fn = "tg_linear_attention_step";
    if (!a) return check_pointers(fn, {a});
    Attention m;
    int code = attention_shape(fn, *a, m);
    if (code) return code;
    if (m.length != 1 || m.packed) {
        set_error("%s: a step is one row", fn);
        return TG_E_ARG;
    }
    if (m.sequences == 0) return 0;
    if ((code = refuse_many(fn, m, kStepThreads))) return code;
    if ((code = check_pointers(fn, {a->queries, a->keys, a->values, a->gates, a->initial, a->outputs, a->final}))) return code;
    return by_types(a->type, a->gate_type, [&](auto t, auto s) { return step<decltype(t), decltype(s)>(*a, m); });
}
