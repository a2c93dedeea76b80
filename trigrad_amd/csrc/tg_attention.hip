// tg_attention.hip -- linear attention S_t = a_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t: the calls, a walk through the rows, a single step.
//
// With D_t the gradient of S_t with all that follows from it,
//     D_t = a_{t+1} D_{t+1} + scale q_t do_t^T,   dq_t = scale S_t do_t,   dk_t = D_t v_t,   dv_t = D_t^T k_t,   dlog a_t = a_t <D_t, S_{t-1}>,
// and since <D_t, S_t> is both q_t.dq_t + dlog a_{t+1} and k_t.dk_t + dlog a_t,
//     dlog a_{t+1} = dlog a_t + k_t.dk_t - q_t.dq_t,   dlog a_1 = <S_0, a_1 D_1>.
#include "tg_attention.hpp"

namespace tg {

// ---- a walk through the rows ----------------------------------------------------------

constexpr int kWalkThreads = 64;
constexpr int kMost = TG_ATTENTION_SIZE;

template <class T> __device__ __forceinline__ double wide(T v) { return (double)(real)v; }

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

template <class S>
__global__ void attention_fixed_gates_kernel(Attention m, const S *__restrict__ gates, const double *__restrict__ sums, int64_t parts, S *__restrict__ grad_gates) {
    const int h = blockIdx.x;
    double all = 0.0;
    for (int64_t n = threadIdx.x; n < parts; n += kWalkThreads) all += sums[n * m.heads + h];
    all = sum_lanes(all, 64);
    if (threadIdx.x == 0) grad_gates[h] = (S)(real)(all * slope_of(m.gate_form, wide(gates[h])));
}

// Key heads' gradients, the sums of their value heads'.
template <class T>
__global__ void attention_shared_kernel(Attention m, const double *__restrict__ parts, T *__restrict__ out) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= m.rows * m.key_heads * m.key_size) return;
    const int64_t i = id % m.key_size, head = id / m.key_size;  // row and key head
    double sum = 0.0;
    for (int n = 0; n < m.shared; n++) sum += parts[(head * m.shared + n) * m.key_size + i];
    out[id] = (T)(real)sum;
}

// Rows in front of the first sequence and behind the last one: zeros.
template <class T> __global__ void attention_outside_kernel(Attention m, const int32_t *__restrict__ offsets, int64_t width, T *__restrict__ out) {
    const AttentionRows first = rows_of(m, offsets, 0), last = rows_of(m, offsets, m.sequences - 1);
    const int64_t end = last.first + last.count, begin = min(first.first, end), outside = m.rows - end + begin;
    for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < outside * width; id += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = id / width;
        out[(row < begin ? row : row - begin + end) * width + id % width] = (T)(real)0;
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
    if (heads >= (1 << 20) || a.length > 0x7fffffff || a.sequences >= ((int64_t)1 << 29) || rows >= limit / (heads * kMost) ||
        a.sequences >= ((int64_t)1 << 31) / heads) {
        set_error("%s: %lld rows, %lld sequences of %lld heads are too many", fn, (long long)rows, (long long)a.sequences, (long long)heads);
        return TG_E_ARG;
    }
    const auto strides = [](const int64_t s[3]) { return Strides{s[0], s[1], s[2]}; };
    m = {a.sequences, a.length, rows, (int)a.heads, (int)a.key_heads, (int)(a.heads / a.key_heads), (int)a.key_size, (int)a.value_size,
         strides(a.query_strides), strides(a.key_strides), strides(a.value_strides), strides(a.grad_strides),
         (int)a.gate_form, a.fixed_gates != 0, a.offsets != nullptr, (float)a.scale};
    return 0;
}

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

static unsigned blocks_for(int64_t n) { return (unsigned)std::min<int64_t>(ceil_div64(n, 256), 1 << 20); }

template <class T, class S> static int walk_forward(const tg_attention &a, const Attention &m) {
    const hipStream_t stream = (hipStream_t)a.stream;
    TG_LAUNCH_AS("attention_walk", (attention_walk_kernel<T, S>), dim3((unsigned)(m.sequences * m.heads), (unsigned)ceil_div(m.value_size, kWalkThreads)),
                 dim3(kWalkThreads), 0, stream, m, (const T *)a.queries, (const T *)a.keys, (const T *)a.values, (const S *)a.gates, a.initial, a.offsets,
                 (T *)a.outputs, a.final);
    if (m.packed && m.rows) {
        const int64_t width = (int64_t)m.heads * m.value_size;
        TG_LAUNCH_AS("attention_outside", (attention_outside_kernel<T>), dim3(blocks_for(m.rows * width)), dim3(256), 0, stream, m, a.offsets, width, (T *)a.outputs);
    }
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
        TG_LAUNCH_AS("attention_round", (attention_round_kernel<real>), dim3(blocks_for(states)), dim3(256), 0, stream, dstate, states, a.grad_initial);
    const int64_t n = m.rows * m.key_heads * m.key_size;
    for (int which = 0; which < 2; which++) {
        T *out = (T *)(which ? a.grad_keys : a.grad_queries);
        if (out && n)
            TG_LAUNCH_AS("attention_shared", (attention_shared_kernel<T>), dim3((unsigned)ceil_div64(n, 256)), dim3(256), 0, stream, m, which ? dk : dq, out);
    }
    if (m.packed && m.rows) {
        const auto outside = [&](auto *out, int64_t width) {
            using U = std::remove_pointer_t<decltype(out)>;
            if (out)
                TG_LAUNCH_AS("attention_outside", (attention_outside_kernel<U>), dim3(blocks_for(m.rows * width)), dim3(256), 0, stream, m, a.offsets, width, out);
        };
        outside((T *)a.grad_queries, (int64_t)m.key_heads * m.key_size);
        outside((T *)a.grad_keys, (int64_t)m.key_heads * m.key_size);
        outside((T *)a.grad_values, (int64_t)m.heads * m.value_size);
        if (!m.fixed) outside((S *)a.grad_gates, (int64_t)m.heads);
    }
    return check_launch("tg_linear_attention_backward");
}

// ---- a single step ----------------------------------------------------------------------

constexpr int kStepThreads = 256;

// A workgroup has V x `lanes` columns of one state (lanes: a power of two), a thread V of them in every (256 / lanes)th row.
template <class T, class S, int V>
__global__ __launch_bounds__(kStepThreads) void attention_step_kernel(Attention m, int lanes, const T *__restrict__ queries, const T *__restrict__ keys,
                                                                      const T *__restrict__ values, const S *__restrict__ gates, const real *state,
                                                                      T *__restrict__ outputs, real *new_state) {
    __shared__ real q[kMost], k[kMost], partial[kStepThreads][V];
    const int64_t s = blockIdx.x / m.heads;
    const int h = (int)(blockIdx.x % m.heads), t = threadIdx.x;
    for (int i = t; i < m.key_size; i += kStepThreads) {
        q[i] = (real)queries[s * m.q.sequence + h / m.shared * m.q.head + i];
        k[i] = (real)keys[s * m.k.sequence + h / m.shared * m.k.head + i];
    }
    __syncthreads();
    const int column = (blockIdx.y * lanes + (t & (lanes - 1))) * V, step = kStepThreads / lanes;
    const bool there = column < m.value_size;
    real sum[V] = {};
    if (there) {
        const real a = (real)exp2(log2_gate(m.gate_form, (real)gates[m.fixed ? h : s * m.heads + h]));
        real v[V];
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = (real)values[s * m.v.sequence + h * m.v.head + column + j];
        const int64_t at = (s * m.heads + h) * m.key_size * m.value_size + column;
#pragma unroll 8
        for (int i = t / lanes; i < m.key_size; i += step) {
            const Pack<real, V> before = load_pack<V>(state + at + (int64_t)i * m.value_size);
            real next[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                next[j] = fma(a, before[j], k[i] * v[j]);
                sum[j] = fma(q[i], next[j], sum[j]);
            }
            store_pack<V>(new_state + at + (int64_t)i * m.value_size, next);
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) partial[t][j] = sum[j];
    __syncthreads();
    if (t >= lanes || !there) return;
#pragma unroll
    for (int j = 0; j < V; j++) {
        real all = 0;
        for (int i = t; i < kStepThreads; i += lanes) all += partial[i][j];
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
    if (!a || !out) return check_pointers("tg_linear_attention_sizes", {a, out});
    Attention m;
    const int code = attention_shape("tg_linear_attention_sizes", *a, m);
    if (code) return code;
    out[0] = out[1] = out[2] = 0;
    out[3] = walk_room(m).all;
    return 0;
}

static int attention_call(const char *fn, const tg_attention *a, bool backward) {
    if (!a) return check_pointers(fn, {a});
    Attention m;
    int code = attention_shape(fn, *a, m);
    if (code) return code;
    int64_t sizes[4];
    code = tg_linear_attention_sizes(a, sizes);
    if (code) return code;
    if (m.sequences == 0) return 0;
    if (m.rows && (code = check_pointers(fn, {a->queries, a->keys, a->values, a->gates}))) return code;
    if (!backward && (code = check_pointers(fn, {a->final}))) return code;
    if (!backward && m.rows && (code = check_pointers(fn, {a->outputs}))) return code;
    if (a->workspace_bytes < sizes[backward ? 3 : 1] || (sizes[backward ? 3 : 1] && !a->workspace)) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)a->workspace_bytes, (long long)sizes[backward ? 3 : 1]);
        return TG_E_WORKSPACE;
    }
    return by_types(a->type, a->gate_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        return backward ? walk_backward<T, S>(*a, m) : walk_forward<T, S>(*a, m);
    });
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
    if ((code = check_pointers(fn, {a->queries, a->keys, a->values, a->gates, a->initial, a->outputs, a->final}))) return code;
    return by_types(a->type, a->gate_type, [&](auto t, auto s) { return step<decltype(t), decltype(s)>(*a, m); });
}
