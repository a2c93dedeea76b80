// tg_recurrence.hip -- the gated linear recurrence h_t = a_t h_{t-1} + u_t: sizes, the calls, a single step (and, in the double library, a
// plain walk through the rows; the float library's kernels are in tg_recurrence_forward.hip and tg_recurrence_backward.hip).
//
// With a = f(gate) and u = x or (1 - a) x, and l_t the gradient of h_t with all that follows from it,
//     l_t = dh_t + a_{t+1} l_{t+1},   dx_t = l_t or (1 - a_t) l_t,   da_t = l_t h_{t-1} or l_t (h_{t-1} - x_t),   dgate = f'(gate) sum da
// over the channels that share the gate.
#ifdef TG_DOUBLE_PRECISION
#include "tg_recurrence.hpp"
#else
#include "tg_recurrence_scan.hpp"
#endif

namespace tg {

#ifndef TG_DOUBLE_PRECISION
static_assert(kForwardThreads == kBackwardThreads && kForwardThreads == kMapThreads, "one bound for the grids of all three");
#endif

#ifdef TG_DOUBLE_PRECISION
// ---- one thread a sequence and channel ------------------------------------------------

struct Rows {
    int64_t begin, end;
};
__device__ __forceinline__ Rows rows_of(const Shape &m, const int32_t *offsets, int64_t s) {
    Rows r;
    if (!offsets) {
        r.begin = s * m.length;
        r.end = r.begin + m.length;
    } else {
        r.begin = min((int64_t)max(offsets[s], 0), m.length);
        r.end = max(r.begin, min((int64_t)max(offsets[s + 1], 0), m.length));
    }
    return r;
}

// The rows in front of the first sequence and behind the last one: zeros.
template <class T> __device__ void clear_outside(const Shape &m, const int32_t *offsets, int64_t s, T *out, int64_t column, int64_t columns) {
    if (!offsets || !out) return;
    const int64_t first = s == 0 ? 0 : rows_of(m, offsets, s).end;
    const int64_t begin = s == 0 ? rows_of(m, offsets, 0).begin : 0;
    if (s == 0)
        for (int64_t r = first; r < begin; r++) out[r * columns + column] = (T)(real)0;
    if (s == m.sequences - 1)
        for (int64_t r = rows_of(m, offsets, s).end; r < m.length; r++) out[r * columns + column] = (T)(real)0;
}

template <class T, class S>
__global__ void recurrence_forward_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates, const real *__restrict__ initial,
                                          const int32_t *__restrict__ offsets, T *__restrict__ states, real *__restrict__ final,
                                          real *__restrict__ kept) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= m.sequences * m.channels) return;
    const int64_t s = id / m.channels, d = id % m.channels, g = d / m.shared;
    const Rows rows = rows_of(m, offsets, s);
    real h = initial ? initial[id] : (real)0;
    for (int64_t i = rows.begin; i < rows.end; i++) {
        const int64_t r = m.reverse ? rows.end - 1 - (i - rows.begin) : i;
        const Gate gate = gate_of(m.gate_form, (real)gates[r * m.gates + g]);
        const real x = (real)inputs[r * m.channels + d];
        if (kept) kept[r * m.channels + d] = h;
        h = fma(gate.a, h, m.complement ? gate.rest * x : x);
        if (states) states[r * m.channels + d] = (T)h;
    }
    final[id] = h;
    clear_outside(m, offsets, s, states, d, m.channels);
}

template <class T, class S>
__global__ void recurrence_backward_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates, const int32_t *__restrict__ offsets,
                                           const real *__restrict__ kept, const T *__restrict__ grad_states,
                                           const real *__restrict__ grad_final, T *__restrict__ grad_inputs, S *__restrict__ grad_gates,
                                           real *__restrict__ grad_initial, real *__restrict__ carried) {
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= m.sequences * m.gates) return;
    const int64_t s = id / m.gates, g = id % m.gates;
    const Rows rows = rows_of(m, offsets, s);
    real *e = carried + s * m.channels;
    for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) e[d] = grad_final ? grad_final[s * m.channels + d] : (real)0;
    for (int64_t i = rows.begin; i < rows.end; i++) {
        const int64_t r = m.reverse ? i : rows.end - 1 - (i - rows.begin);
        const Gate gate = gate_of(m.gate_form, (real)gates[r * m.gates + g]);
        real sum = 0;
        for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) {
            const int64_t at = r * m.channels + d;
            const real l = e[d] + (grad_states ? (real)grad_states[at] : (real)0);
            sum = fma(l, m.complement ? kept[at] - (real)inputs[at] : kept[at], sum);
            if (grad_inputs) grad_inputs[at] = (T)(m.complement ? gate.rest * l : l);
            e[d] = gate.a * l;
        }
        if (grad_gates) grad_gates[r * m.gates + g] = (S)(sum * gate.slope);
    }
    for (int64_t d = g * m.shared; d < (g + 1) * m.shared; d++) {
        if (grad_initial) grad_initial[s * m.channels + d] = e[d];
        clear_outside(m, offsets, s, grad_inputs, d, m.channels);
    }
    clear_outside(m, offsets, s, grad_gates, g, m.gates);
}
#endif  // TG_DOUBLE_PRECISION

// ---- a single step ----------------------------------------------------------------------

constexpr int kStepThreads = 256;

// A thread has V successive channels, of one gate (Shared) or of as many.  Bound by latency for a few sequences; for 512 x 4096 in bfloat16 with a
// gate by head 25 MB go by in 5.2 to 5.9 us of the kernel, and a thread a channel with 64-bit divisions took 9.5.
template <class T, class S, int V, bool Shared>
__global__ __launch_bounds__(kStepThreads) void recurrence_step_kernel(Shape m, const T *__restrict__ inputs, const S *__restrict__ gates,
                                                                       const real *state, T *__restrict__ states, real *new_state) {
    constexpr int GV = Shared ? 1 : V;
    const uint32_t id = blockIdx.x * (uint32_t)kStepThreads + threadIdx.x, row = (uint32_t)(m.channels / V);
    const uint32_t s = id / row;
    if (s >= (uint64_t)m.sequences) return;
    const int64_t at = (int64_t)id * V;
    const uint32_t channel = (id - s * row) * V;
    const Pack<S, GV> g = load_pack<GV>(gates + s * m.gates + (Shared ? channel / (uint32_t)m.shared : channel));
    const Pack<T, V> x = load_pack<V>(inputs + at);
    const Pack<real, V> before = load_pack<V>(state + at);
    real h[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const Gate gate = gate_of(m.gate_form, g[Shared ? 0 : v]);
        h[v] = fma(gate.a, before[v], m.complement ? gate.rest * x[v] : x[v]);
    }
    store_pack<V>(new_state + at, h);
    store_pack<V>(states + at, h);
}

// ---- host ---------------------------------------------------------------------------------

constexpr int64_t kGridThreads = (int64_t)1 << 32;  // a grid has fewer

static int too_many(const char *fn, int64_t rows, int64_t channels) {
    set_error("%s: %lld rows of %lld channels are too many", fn, (long long)rows, (long long)channels);
    return TG_E_ARG;
}

int recurrence_shape(const char *fn, const tg_recurrence &r, Shape &m) {
    if (r.sequences < 0 || r.length < 0 || r.channels < 0 || r.gate_count < 0 || (r.gate_count == 0) != (r.channels == 0) ||
        (r.gate_count > 0 && r.channels % r.gate_count != 0)) {
        set_error("%s: sizes", fn);
        return TG_E_ARG;
    }
    if (!type_known(r.type) || (r.gate_type != r.type && r.gate_type != kRealType)) {
        set_error("%s: types %lld and %lld", fn, (long long)r.type, (long long)r.gate_type);
        return TG_E_ARG;
    }
    if (r.gate_form < TG_GATE_VALUE || r.gate_form > TG_GATE_LOGIT || r.input_form < TG_INPUT_PLAIN || r.input_form > TG_INPUT_COMPLEMENT) {
        set_error("%s: gate_form %lld, input_form %lld", fn, (long long)r.gate_form, (long long)r.input_form);
        return TG_E_ARG;
    }
    const int64_t limit = (int64_t)1 << 40;
    const int64_t rows = r.offsets ? r.length : r.length == 0 ? 0 : r.sequences > limit / r.length ? limit : r.sequences * r.length;
    if (rows >= limit || (r.offsets && r.length > 0x7fffffff) || r.channels >= ((int64_t)1 << 31) || r.sequences >= ((int64_t)1 << 29) ||
        (r.channels > 0 && (rows > limit / r.channels || r.sequences > limit / r.channels))) {
        set_error("%s: more than 2^40 elements, 2^29 sequences or 2^31 channels", fn);
        return TG_E_ARG;
    }
    m.sequences = r.sequences;
    m.length = r.length;
    m.channels = r.channels;
    m.gates = r.gate_count;
    m.shared = r.gate_count ? r.channels / r.gate_count : 1;
    m.gate_form = (int)r.gate_form;
    m.complement = r.input_form == TG_INPUT_COMPLEMENT;
    m.reverse = r.reverse != 0;
    return 0;
}

#ifdef TG_DOUBLE_PRECISION

static int sizes_of(const char *fn, const tg_recurrence &r, const Shape &m, int64_t out[3]) {
    if (m.sequences * m.channels > kGridThreads - 256) return too_many(fn, m.sequences, m.channels);
    out[0] = (r.offsets ? m.length : m.sequences * m.length) * m.channels * (int64_t)sizeof(real);
    out[1] = 0;
    out[2] = m.sequences * m.channels * (int64_t)sizeof(real);
    return 0;
}

static int forward(const char *fn, const tg_recurrence &r, const Shape &m) {
    TG_LAUNCH_AS("recurrence_forward", (recurrence_forward_kernel<real, real>), dim3((unsigned)ceil_div64(m.sequences * m.channels, 256)), dim3(256), 0,
                 (hipStream_t)r.stream, m, (const real *)r.inputs, (const real *)r.gates, r.initial, r.offsets, (real *)r.states, r.final,
                 (real *)r.kept);
    return check_launch(fn);
}

static int backward(const char *fn, const tg_recurrence &r, const Shape &m) {
    TG_LAUNCH_AS("recurrence_backward", (recurrence_backward_kernel<real, real>), dim3((unsigned)ceil_div64(m.sequences * m.gates, 256)), dim3(256), 0,
                 (hipStream_t)r.stream, m, (const real *)r.inputs, (const real *)r.gates, r.offsets, (const real *)r.kept,
                 (const real *)r.grad_states, r.grad_final, (real *)r.grad_inputs, (real *)r.grad_gates, r.grad_initial, (real *)r.workspace);
    return check_launch(fn);
}

#else

static int log2_above(int64_t n) {  // of the power of two that is n or more
    int k = 0;
    while (((int64_t)1 << k) < n) k++;
    return k;
}

// Channels of a lane: two neighbours where they are aligned (or all three of a gate that has three), else one.
static int vector_of(int64_t shared, int64_t channels, bool aligned) {
    const int64_t run = shared > 1 ? shared : channels;
    return run % 2 == 0 ? (aligned ? 2 : 1) : shared % 3 == 0 ? 3 : 1;
}

static bool aligned_for(int64_t bytes, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if ((uintptr_t)p % (uintptr_t)bytes != 0) return false;
    return true;
}

// Rows and columns of a call in one direction.  What the two directions have to agree on (whether the rows are chained, and into which
// chunks) does not depend on alignment.
static Split split_of(const Shape &s, bool packed, int64_t wide_gates, int vector, bool backward) {
    Split m = {};
    m.packed = packed;
    m.rows = packed ? s.length : s.sequences * s.length;
    m.channels = s.channels;
    m.gates = s.gates;
    m.shared = s.shared;
    m.length = s.length;
    m.sequences = s.sequences;
    m.gate_form = s.gate_form;
    m.wide_gates = (int)wide_gates;
    m.complement = s.complement;
    m.reverse = s.reverse;
    const int best = vector_of(s.shared, s.channels, true);
    const auto columns = [&](int v, int most_lanes_log2) {
        m.parts = 1;
        m.gate_lanes_log2 = 0;
        if (s.shared == 1) return ceil_div64(s.channels, v);
        m.gate_lanes_log2 = std::min(log2_above(ceil_div64(s.shared, v)), most_lanes_log2);
        m.parts = (int)ceil_div64(ceil_div64(s.shared, v), (int64_t)1 << m.gate_lanes_log2);
        return s.gates * m.parts << m.gate_lanes_log2;
    };
    const int64_t wanted = columns(best, 6), axis = packed ? m.rows : s.length;
    const int narrow = std::min(6, log2_above(wanted));  // lanes of a row where there are many rows
    m.kept_rows = kBackwardChunk >> narrow;
    m.chained = axis > kWideChunk >> narrow;
    m.wide = !m.chained && axis > m.kept_rows;
    const int threads = m.wide ? kWideThreads : backward ? kBackwardThreads : kForwardThreads;
    const int rows = m.wide ? kWideRows : backward ? kBackwardRows : kForwardRows;
    const int threads_log2 = log2_above(threads);
    m.lanes_log2 = narrow;
    if (!m.chained) m.lanes_log2 = std::min(log2_above(wanted), std::max(narrow, threads_log2 - log2_above(ceil_div64(axis, rows))));
    m.columns = columns(vector, std::min(6, m.lanes_log2));
    m.tiles = ceil_div64(m.columns, (int64_t)1 << m.lanes_log2);
    m.chunk_rows = (int64_t)(threads >> m.lanes_log2) * rows;
    if (!m.chained) m.chunk_rows = packed ? std::max<int64_t>(m.rows, 1) : m.chunk_rows / s.length * s.length;
    m.chunks = ceil_div64(m.rows, m.chunk_rows);
    return m;
}

// The workspace: sequences to search between (packed), what chunks start from, their maps, sums of gates' gradients by waves.  Bytes.
struct Room {
    int64_t sequences, starts, maps, partial, all;
};
static Room room_of(const Split &m, bool backward) {
    Room r = {};
    r.maps = m.chained ? m.chunks * m.channels * (int64_t)sizeof(MapWords) : 0;
    r.starts = m.chained ? (m.chunks * m.channels + 1) / 2 * 8 : 0;
    r.sequences = m.packed ? m.chunks * 8 : 0;
    r.partial = backward && m.parts > 1 ? m.parts * m.rows * m.gates * 4 : 0;
    r.all = r.sequences + r.starts + r.maps + r.partial;
    return r;
}

static int sizes_of(const char *fn, const tg_recurrence &r, const Shape &m, int64_t out[3]) {
    out[0] = out[1] = out[2] = 0;
    if (m.length == 0 || m.sequences == 0 || m.channels == 0) return 0;
    const bool packed = r.offsets != nullptr;
    for (int aligned = 0; aligned < 2; aligned++)
        for (int backward = 0; backward < 2; backward++) {
            const Split s = split_of(m, packed, 0, vector_of(m.shared, m.channels, aligned), backward);
            if (s.chunks * s.tiles >= kGridThreads / (s.wide ? kWideThreads : kForwardThreads) ||
                (s.chained && ceil_div64(s.channels, 1 << kStartLanesLog2) >= kGridThreads / kStartThreads) ||
                (!packed && m.length <= kShortRows && m.sequences * s.columns >= kGridThreads - kShortThreads))
                return too_many(fn, s.rows, s.channels);
            const Room room = room_of(s, backward);
            out[1 + backward] = std::max(out[1 + backward], room.all);
            out[0] = s.chained ? ceil_div64(s.rows, s.kept_rows) * s.channels * 4 : 0;
        }
    return 0;
}

static int run(const tg_recurrence &r, const Shape &s, bool backward) {
    hipStream_t stream = (hipStream_t)r.stream;
    const float *from = backward ? r.grad_final : r.initial;
    float *to = backward ? r.grad_initial : r.final;
    if (s.length == 0) {
        const Split none = {0, s.channels, s.gates, s.shared, 0, s.sequences};
        return to ? launch_prepare(none, nullptr, nullptr, from, to, stream) : 0;
    }
    const int64_t bytes = type_bytes(r.type), gate_bytes = type_bytes(r.gate_type);
    bool aligned = aligned_for(2 * bytes, {r.inputs, r.states, r.grad_states, r.grad_inputs});
    if (s.shared == 1) aligned = aligned && aligned_for(2 * gate_bytes, {r.gates, r.grad_gates});
    const int vector = vector_of(s.shared, s.channels, aligned);
    const Split m = split_of(s, r.offsets != nullptr, r.gate_type == TG_TYPE_F32, vector, backward);
    const Room room = room_of(m, backward);
    char *at = (char *)r.workspace;
    int32_t *first_sequence = (int32_t *)at;
    float *starts = (float *)(at + room.sequences);
    MapWords *maps = (MapWords *)(at + room.sequences + room.starts);
    float *partial = (float *)(at + room.sequences + room.starts + room.maps);
    if (m.packed)
        if (const int code = launch_prepare(m, first_sequence, r.offsets, from, to, stream)) return code;
    if (m.chained)
        if (const int code = launch_starts(r, m, first_sequence, maps, starts, vector, backward, stream)) return code;
    if (!m.packed && m.length <= kShortRows) return launch_short(r, m, partial, vector, backward, stream);
    const unsigned blocks = (unsigned)(m.chunks * m.tiles);
    return backward ? launch_backward(r, m, first_sequence, starts, partial, vector, blocks, stream)
                    : launch_forward(r, m, first_sequence, starts, vector, blocks, stream);
}

static int forward(const char *, const tg_recurrence &r, const Shape &s) { return run(r, s, false); }
static int backward(const char *, const tg_recurrence &r, const Shape &s) { return run(r, s, true); }

#endif  // TG_DOUBLE_PRECISION

}  // namespace tg

extern "C" int tg_linear_recurrence_sizes(const tg_recurrence *r, int64_t out[3]) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_sizes";
    if (!r || !out) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    Shape m;
    if (const int code = recurrence_shape(fn, *r, m)) return code;
    return sizes_of(fn, *r, m, out);
}

extern "C" int tg_linear_recurrence_forward(const tg_recurrence *r) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_forward";
    Shape m;
    int64_t sizes[3];
    if (!r) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    if (const int code = recurrence_shape(fn, *r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    if (const int code = sizes_of(fn, *r, m, sizes)) return code;
    if ((m.length > 0 && (!r->inputs || !r->gates)) || !r->final || (r->kept && r->kept_bytes < sizes[0])) {
        set_error("%s: null pointer, or kept too small", fn);
        return TG_E_ARG;
    }
    if (sizes[1] > 0 && (!r->workspace || r->workspace_bytes < sizes[1])) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)r->workspace_bytes, (long long)sizes[1]);
        return TG_E_WORKSPACE;
    }
    return forward(fn, *r, m);
}

extern "C" int tg_linear_recurrence_backward(const tg_recurrence *r) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_backward";
    Shape m;
    int64_t sizes[3];
    if (!r) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    if (const int code = recurrence_shape(fn, *r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    if (const int code = sizes_of(fn, *r, m, sizes)) return code;
    if (m.length > 0 && (!r->inputs || !r->gates || (sizes[0] > 0 && (!r->kept || r->kept_bytes < sizes[0])))) {
        set_error("%s: null pointer, or kept too small", fn);
        return TG_E_ARG;
    }
    if (sizes[2] > 0 && (!r->workspace || r->workspace_bytes < sizes[2])) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)r->workspace_bytes, (long long)sizes[2]);
        return TG_E_WORKSPACE;
    }
    return backward(fn, *r, m);
}

extern "C" int tg_linear_recurrence_step(const void *inputs, const void *gates, const tg_real *state, void *states, tg_real *new_state,
                                         int64_t sequences, int64_t channels, int64_t gate_count, int type, int gate_type, int gate_form,
                                         int input_form, void *stream) {
    using namespace tg;
    const char *fn = "tg_linear_recurrence_step";
    tg_recurrence r = {};
    r.sequences = sequences;
    r.length = 1;
    r.channels = channels;
    r.gate_count = gate_count;
    r.type = type;
    r.gate_type = gate_type;
    r.gate_form = gate_form;
    r.input_form = input_form;
    Shape m;
    if (const int code = recurrence_shape(fn, r, m)) return code;
    if (m.sequences == 0 || m.channels == 0) return 0;
    if (!inputs || !gates || !state || !states || !new_state) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    if (m.sequences * m.channels >= kGridThreads - kStepThreads) {
        set_error("%s: 2^32 channels of sequences or more", fn);
        return TG_E_ARG;
    }
    return by_types(type, gate_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        const auto with = [&](auto v, auto shared) {
            constexpr int V = decltype(v)::value;
            TG_LAUNCH_AS("recurrence_step", (recurrence_step_kernel<T, S, V, decltype(shared)::value>),
                         dim3((unsigned)ceil_div64(m.sequences * m.channels / V, kStepThreads)), dim3(kStepThreads), 0, (hipStream_t)stream, m,
                         (const T *)inputs, (const S *)gates, state, (T *)states, new_state);
            return check_launch(fn);
        };
        using four = std::integral_constant<int, sizeof(real) == 4 ? 4 : 1>;
        using one = std::integral_constant<int, 1>;
        const uintptr_t rows = (uintptr_t)inputs | (uintptr_t)states, wide = (uintptr_t)state | (uintptr_t)new_state;
        const bool whole = (m.shared > 1 ? m.shared : m.channels) % 4 == 0 && rows % (4 * sizeof(T)) == 0 && wide % 16 == 0 &&
                           (m.shared > 1 || (uintptr_t)gates % (4 * sizeof(S)) == 0);
        if (m.shared > 1) return whole ? with(four(), std::true_type()) : with(one(), std::true_type());
        return whole ? with(four(), std::false_type()) : with(one(), std::false_type());
    });
}
