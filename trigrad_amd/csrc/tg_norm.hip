// tg_norm.hip -- group norm with an activation behind it, channels last.
//
//     xh = (x - mean) rstd,  z = weight xh + bias,  y = act(z),  mean and rstd of a sample's positions x (channels / groups)
//     dz = dy act'(z),  dweight = sum dz xh,  dbias = sum dz,  dxh = weight dz,  dx = rstd (dxh - avg dxh - xh avg(dxh xh))
//
// Bound by memory traffic: x in and y out, x and dy in and dx out.  Three ways:
//   token     a sample is one position and its groups are wider than a wave: a workgroup has a group in registers.
//   held      a sample's groups fit the registers of a workgroup: read once, summed, written.  A workgroup has `teams` samples at a
//             time and goes over many, so that the weights' gradients are summed in registers and come to few partial sums.
//   streamed  a sample's rows are split over workgroups: one launch sums them, a small one joins the sums, one reads the rows again
//             (from the last to the first, so that what the first launch read last is still near) and writes.
// A thread's sums are float32, of at most kChain values one after another; its workgroup's threads of a channel (at most 1024, of a row of one access)
// are added in float32 too, or float64 (streamed forward), and workgroups in float64; all in a fixed order.
#include <algorithm>
#include <type_traits>

#include "tg_elements.hpp"

namespace tg {

struct NormShape {
    int64_t samples, positions, channels, groups, width;  // width: channels of a group
    int activation, wide_weights, aligned_weights;         // wide_weights: weight and bias are tg_real whatever x is
    real eps;
};

#ifdef TG_DOUBLE_PRECISION
__device__ __forceinline__ real exp_norm(real z) { return exp(z); }
__device__ __forceinline__ real inverse(real v) { return 1.0 / v; }
__device__ __forceinline__ real inverse_root(real v) { return 1.0 / sqrt(v); }
#else
// 1 / sqrt(v) to one unit; the hardware's takes numbers below the normal ones for 0
__device__ __forceinline__ real inverse_root(real v) { return v < 2.0f * FLT_MIN ? 1.0f / sqrtf(v) : __builtin_amdgcn_rsqf(v); }
// As a power of two of a rounded product, which is half a step of z: what z's own rounding, a step before, costs the exponential too.
__device__ __forceinline__ real exp_norm(real z) { return __builtin_amdgcn_exp2f(z * 1.44269504f); }
__device__ __forceinline__ real inverse(real v) { return __builtin_amdgcn_rcpf(v); }
#endif

// Phi(-|z|) / exp(-z^2 / 2), Phi the normal distribution: a quotient that varies so little that a polynomial of 1 / (1 + 0.3 |z|) has it to
// ten units of 2^-24 of itself wherever the exponential is not 0, three of them the reciprocal's (the coefficients by weighted least squares for
// the smallest relative error).  So the activation falls off with its exponential on the negative side instead of ending in a difference's rounding.
__device__ __forceinline__ real mills(real z) {
#ifdef TG_DOUBLE_PRECISION
    return z * z < 1400.0 ? 0.5 * erfc(fabs(z) * 0.70710678118654752440) / exp(-0.5 * z * z) : 0.0;
#else
    const float t = inverse(fmaf(0.3f, fabsf(z), 1.0f));
    float r = fmaf(0.038425032049417496f, t, -0.16939298808574677f);
    r = fmaf(r, t, 0.22912785410881042f);
    r = fmaf(r, t, -0.07704015076160431f);
    r = fmaf(r, t, 0.14290300011634827f);
    r = fmaf(r, t, 0.09452757239341736f);
    r = fmaf(r, t, 0.12196006625890732f);
    r = fmaf(r, t, 0.11948215216398239f);
    return fmaf(r, t, 7.4919621511071455e-06f);
#endif
}

// act(z); Slope: act'(z)
template <int Kind, bool Slope> __device__ __forceinline__ real activate(real z) {
    if (Kind == TG_ACTIVATION_RELU) {
        if (Slope) return z > 0 ? (real)1 : (real)0;
        return z < 0 ? (real)0 : z;  // NaN stays
    }
    if (Kind == TG_ACTIVATION_SILU) {
        const real s = inverse((real)1 + exp_norm(-z));
        return Slope ? s * fma(z, (real)1 - s, (real)1) : z * s;
    }
    if (Kind == TG_ACTIVATION_GELU) {
        const real e = exp_norm((real)-0.5 * z * z), q = e * mills(z), phi = z < 0 ? q : (real)1 - q;
        return Slope ? fma(z * e, (real)0.39894228040143267794, phi) : z * phi;
    }
    return Slope ? (real)1 : z;
}

template <class Call> __device__ __forceinline__ void by_activation(int kind, Call &&call) {
    if (kind == TG_ACTIVATION_NONE) call(std::integral_constant<int, TG_ACTIVATION_NONE>());
    else if (kind == TG_ACTIVATION_RELU) call(std::integral_constant<int, TG_ACTIVATION_RELU>());
    else if (kind == TG_ACTIVATION_SILU) call(std::integral_constant<int, TG_ACTIVATION_SILU>());
    else call(std::integral_constant<int, TG_ACTIVATION_GELU>());
}

// V successive weights: one access where they are aligned.
template <class S, int V> __device__ __forceinline__ void load_weights_of(const NormShape &m, const S *from, real (&w)[V]) {
    if (m.aligned_weights) {
        const Pack<S, V> in = load_pack<V>(from);
#pragma unroll
        for (int v = 0; v < V; v++) w[v] = in[v];
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) w[v] = (real)from[v];
    }
}
template <class T, int V>
__device__ __forceinline__ void load_weights(const NormShape &m, const void *from, int64_t base, uint32_t at, real missing, real (&w)[V]) {
    if (!from) {
#pragma unroll
        for (int v = 0; v < V; v++) w[v] = missing;
    } else if (sizeof(T) == sizeof(real) || m.wide_weights) {
        load_weights_of(m, (const real *)from + base + at, w);
    } else {
        load_weights_of(m, (const T *)from + base + at, w);
    }
}
template <class T, int V> __device__ __forceinline__ void load_weights(const NormShape &m, const void *from, int64_t at, real missing, real (&w)[V]) {
    load_weights<T, V>(m, from, at, 0, missing, w);
}
// The groups of V successive channels: one division, then steps.
template <int V> __device__ __forceinline__ void groups_of(const NormShape &m, int64_t channel, int (&g)[V]) {
    const uint32_t width = (uint32_t)m.width;
    g[0] = (int)((uint32_t)channel / width);
    uint32_t within = (uint32_t)channel - (uint32_t)g[0] * width;
#pragma unroll
    for (int v = 1; v < V; v++) {
        within++;
        const bool next = within == width;
        g[v] = g[v - 1] + (next ? 1 : 0);
        if (next) within = 0;
    }
}
// mean and rstd (or two averages) of each channel's group
template <int V> __device__ __forceinline__ void load_pairs(const NormShape &m, int64_t n, const int (&g)[V], const real *pairs, real (&a)[V], real (&b)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
        const Pack<real, 2> pair = load_pack<2>(pairs + 2 * (n * m.groups + g[v]));
        a[v] = pair[0];
        b[v] = pair[1];
    }
}
template <class T> __device__ __forceinline__ void store_weight(const NormShape &m, void *to, int64_t at, real w) {
    if (sizeof(T) == sizeof(real) || m.wide_weights) ((real *)to)[at] = w;
    else ((T *)to)[at] = (T)w;
}

// ---- held -------------------------------------------------------------------------------------

// Threads of a workgroup: team (a sample each), row (of the sample's positions), unit (V successive channels) -- the unit fastest.  A slab is a run
// of whole groups.
struct Held {
    int threads, units, rows, teams;
    int unit_groups;   // units of a group
    int slab_groups;   // groups of a slab
    int64_t turns;     // sets of `teams` samples
    int workgroups;    // that go over them
    bool in_wave;      // a group's threads are neighbours in a wave, a power of two of them
};

// Sums of two values over the threads of each group: by neighbours, or through LDS.
__device__ __forceinline__ void sum_groups(const Held &p, int segment, int member, int members, bool active, real &a, real &b, real *shared) {
    if (p.in_wave) {
        a = sum_lanes(a, members);
        b = sum_lanes(b, members);
        return;
    }
    // all of a group's values to LDS, and their sum by every thread of the group (few of them) or by a wave
    real *sums = shared + 2 * p.threads;
    __syncthreads();
    if (active) {
        shared[2 * (segment * members + member)] = a;
        shared[2 * (segment * members + member) + 1] = b;
    }
    __syncthreads();
    if (members <= 8) {
        if (active) {
            const real *from = shared + 2 * segment * members;
            a = from[0];
            b = from[1];
            for (int i = 1; i < members; i++) {
                a += from[2 * i];
                b += from[2 * i + 1];
            }
        }
        return;
    }
    const int segments = p.teams * p.slab_groups, lane = threadIdx.x & (kWave - 1);
    for (int s = threadIdx.x / kWave; s < segments; s += p.threads / kWave) {
        real first = 0, second = 0;
        for (int i = lane; i < members; i += kWave) {
            first += shared[2 * (s * members + i)];
            second += shared[2 * (s * members + i) + 1];
        }
        first = sum_lanes(first, kWave);
        second = sum_lanes(second, kWave);
        if (lane == 0) {
            sums[2 * s] = first;
            sums[2 * s + 1] = second;
        }
    }
    __syncthreads();
    if (active) {
        a = sums[2 * segment];
        b = sums[2 * segment + 1];
    }
}

struct HeldPlace {
    int unit, row, team, group, segment, member, members;
    int64_t channel;
    bool active;
};
template <int V> __device__ __forceinline__ HeldPlace held_place(const NormShape &m, const Held &p, int slab) {
    HeldPlace t;
    const int id = threadIdx.x, line = id / p.units;
    t.unit = id - line * p.units;
    t.team = line / p.rows;
    t.row = line - t.team * p.rows;
    t.active = t.team < p.teams;
    t.group = t.unit / p.unit_groups;
    t.segment = t.team * p.slab_groups + t.group;
    t.member = t.row * p.unit_groups + t.unit - t.group * p.unit_groups;
    t.members = p.rows * p.unit_groups;
    t.channel = (int64_t)slab * p.slab_groups * m.width + (int64_t)t.unit * V;
    // the last slab may have fewer groups
    t.active = t.active && t.channel < m.channels;
    t.group += slab * p.slab_groups;
    return t;
}

// A thread's rows of a turn, from which it goes on by `workgroups` turns.
struct HeldRows {
    int64_t n, base, pitch, n_step, base_step;
    int all;      // rows of the thread where it has a sample: at most K
    int rows;     // 0: none
    bool active;
};
__device__ __forceinline__ HeldRows held_rows(const NormShape &m, const Held &p, const HeldPlace &t, int64_t turn) {
    HeldRows r;
    r.n = turn * p.teams + t.team;
    r.n_step = (int64_t)p.workgroups * p.teams;
    r.base = (r.n * m.positions + t.row) * m.channels + t.channel;
    r.base_step = r.n_step * m.positions * m.channels;
    r.pitch = (int64_t)p.rows * m.channels;
    r.all = t.active ? ((int)m.positions - t.row + p.rows - 1) / p.rows : 0;
    r.active = t.active && r.n < m.samples;
    r.rows = r.active ? r.all : 0;
    return r;
}
__device__ __forceinline__ void next_turn(const NormShape &m, HeldRows &r) {
    r.n += r.n_step;
    r.base += r.base_step;
    r.active = r.active && r.n < m.samples;
    r.rows = r.active ? r.all : 0;
}
template <class T, int V, int K> __device__ __forceinline__ void load_held(const HeldRows &r, const T *x, Pack<T, V> (&in)[K]) {
#pragma unroll
    for (int k = 0; k < K; k++) in[k] = load_pack<V>(x + (k < r.rows ? r.base + r.pitch * k : 0));
}

template <class T, int V, int K>
__global__ __launch_bounds__(1024) void norm_held_forward_kernel(NormShape m, Held p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                 const void *__restrict__ bias, T *__restrict__ y, real *__restrict__ statistics) {
    extern __shared__ real shared[];
    const int slab = (int)(blockIdx.x / (unsigned)p.workgroups), first_turn = (int)(blockIdx.x % (unsigned)p.workgroups);
    const HeldPlace t = held_place<V>(m, p, slab);
    const real per_value = (real)1 / (real)(m.positions * m.width);
    real w[V], b[V];
    load_weights<T, V>(m, weight, t.active ? t.channel : 0, (real)1, w);
    load_weights<T, V>(m, bias, t.active ? t.channel : 0, (real)0, b);
    HeldRows r = held_rows(m, p, t, first_turn);
    for (int64_t turn = first_turn; turn < p.turns; turn += p.workgroups, next_turn(m, r)) {
        const int64_t n = r.n, base = r.base, pitch = r.pitch;
        const int rows = r.rows;
        const bool active = r.active;
        Pack<T, V> in[K];
        load_held(r, x, in);
        real sum = 0, none = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) sum += k < rows ? in[k][v] : (real)0;
        sum_groups(p, t.segment, t.member, t.members, active, sum, none, shared);
        // about the mean of the first sum, again: what its rounding left, and the variance
        const real about = sum * per_value;
        real first = 0, second = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                const real d = k < rows ? in[k][v] - about : (real)0;
                first += d;
                second = fma(d, d, second);
            }
        sum_groups(p, t.segment, t.member, t.members, active, first, second, shared);
        const real rest = first * per_value, mean = about + rest, variance = fma(-rest, rest, second * per_value);
        const real rstd = inverse_root((variance < 0 ? (real)0 : variance) + m.eps);
        if (active && t.member == 0) {
            statistics[2 * (n * m.groups + t.group)] = mean;
            statistics[2 * (n * m.groups + t.group) + 1] = rstd;
        }
        by_activation(m.activation, [&](auto kind) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k >= rows) break;
                real out[V];
#pragma unroll
                for (int v = 0; v < V; v++) out[v] = activate<decltype(kind)::value, false>(fma((in[k][v] - mean) * rstd, w[v], b[v]));
                store_pack<V>(y + base + pitch * k, out);
            }
        });
    }
}

template <class T, int V, int K>
__global__ __launch_bounds__(1024) void norm_held_backward_kernel(NormShape m, Held p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                  const void *__restrict__ bias, const real *__restrict__ statistics,
                                                                  const T *__restrict__ grad_y, T *__restrict__ grad_x, real *__restrict__ partial) {
    extern __shared__ real shared[];
    const int slab = (int)(blockIdx.x / (unsigned)p.workgroups), first_turn = (int)(blockIdx.x % (unsigned)p.workgroups);
    const HeldPlace t = held_place<V>(m, p, slab);
    const real per_value = (real)1 / (real)(m.positions * m.width);
    real w[V], b[V], dw[V], db[V];
    load_weights<T, V>(m, weight, t.active ? t.channel : 0, (real)1, w);
    load_weights<T, V>(m, bias, t.active ? t.channel : 0, (real)0, b);
#pragma unroll
    for (int v = 0; v < V; v++) dw[v] = db[v] = 0;
    HeldRows r = held_rows(m, p, t, first_turn);
    for (int64_t turn = first_turn; turn < p.turns; turn += p.workgroups, next_turn(m, r)) {
        const int64_t base = r.base, pitch = r.pitch;
        const int rows = r.rows;
        Pack<T, V> in[K], dy[K];
        load_held(r, x, in);
        load_held(r, grad_y, dy);
        const Pack<real, 2> of = load_pack<2>(statistics + (r.active ? 2 * (r.n * m.groups + t.group) : 0));
        const real mean = of[0], rstd = of[1];
        real sum = 0, product = 0;
        // dz is computed again where it is used: its 32 bits are not held.  z has the same roundings everywhere, so that at the border of ReLU the
        // output and all gradients agree on the slope.
        by_activation(m.activation, [&](auto kind) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const real hat = (in[k][v] - mean) * rstd;
                    const real dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(hat, w[v], b[v]));
                    if (k < rows) {
                        db[v] += dz;
                        dw[v] = fma(dz, hat, dw[v]);
                        sum = fma(dz, w[v], sum);
                        product = fma(dz * w[v], hat, product);
                    }
                }
        });
        if (grad_x) {
            sum_groups(p, t.segment, t.member, t.members, r.active, sum, product, shared);
            const real c0 = sum * per_value, c1 = product * per_value;
            by_activation(m.activation, [&](auto kind) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    if (k >= rows) break;
                    real out[V];
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const real hat = (in[k][v] - mean) * rstd;
                        const real dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(hat, w[v], b[v]));
                        out[v] = rstd * fma(dz, w[v], fma(hat, -c1, -c0));
                    }
                    store_pack<V>(grad_x + base + pitch * k, out);
                }
            });
        }
    }
    if (!partial) return;
    // sums over the threads that have the same channels
    const int lines = p.teams * p.rows, columns = p.units * V;
    real *at = shared;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; v++)
            if (t.active) at[(threadIdx.x / p.units) * columns + t.unit * V + v] = which ? db[v] : dw[v];
        __syncthreads();
        for (int c = threadIdx.x; c < columns; c += p.threads) {
            const int64_t channel = (int64_t)slab * p.slab_groups * m.width + c;
            if (channel >= m.channels) continue;
            real sum = 0;
            for (int i = 0; i < lines; i++) sum += at[i * columns + c];
            partial[((int64_t)which * p.workgroups + first_turn) * m.channels + channel] = sum;
        }
    }
}

// ---- tokens -------------------------------------------------------------------------------------

// A sample of one position whose groups are wider than a wave: a workgroup has a group of it in registers and goes over many
// samples.  8192 x 8192 in bfloat16: 53 us forward (5.1 TB/s) and 112 backward with its joining (3.6); the held kernels took 103 and 125.  A thread
// has several accesses (forward 53 us, backward 120) or, backward where a workgroup can, one (112): its sums of the weights' gradients take registers.
// With weights in float32 beside 16-bit elements, which are read again for every sample, it is 141 us forward and 113 backward.
struct Token {
    int threads, units;  // units: accesses of a group
    bool single;         // one of them a thread
    int workgroups;      // that go over the samples, for each group
};
// Accesses of a thread where it has several: sixteen elements, or four accesses (more of narrow ones spill registers).
constexpr int token_accesses(int vector) { return std::min((sizeof(real) == 4 ? 16 : 8) / vector, 4); }

// Sums of two values over the workgroup.  The two buffers take turns, so that one barrier is enough.
struct TokenSums {
    real at[2][1024 / kWave][2];
};
__device__ __forceinline__ void sum_token(TokenSums &s, int &buffer, real &a, real &b) {
    a = sum_lanes(a, kWave);
    b = sum_lanes(b, kWave);
    const int waves = blockDim.x / kWave, wave = threadIdx.x / kWave;
    if (waves == 1) return;
    if ((threadIdx.x & (kWave - 1)) == 0) {
        s.at[buffer][wave][0] = a;
        s.at[buffer][wave][1] = b;
    }
    __syncthreads();
    a = b = 0;
    for (int i = 0; i < waves; i++) {
        a += s.at[buffer][i][0];
        b += s.at[buffer][i][1];
    }
    buffer ^= 1;
}

// Of a thread's access k from the group's first channel; that of its first channels where it has no such access.
template <int V> __device__ __forceinline__ uint32_t token_offset(const Token &p, int k, int left) {
    return k * p.threads < left ? (threadIdx.x + k * p.threads) * V : 0;
}

template <class T, int V, int K>
__global__ __launch_bounds__(1024) void norm_token_forward_kernel(NormShape m, Token p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                  const void *__restrict__ bias, T *__restrict__ y, real *__restrict__ statistics) {
    __shared__ TokenSums shared;
    const int64_t group = blockIdx.x / (unsigned)p.workgroups, low = group * m.width;
    const real per_value = (real)1 / (real)m.width;
    const int left = p.units - (int)threadIdx.x;  // accesses k with k * threads < left are the thread's
    int buffer = 0;
    for (int64_t n = blockIdx.x % (unsigned)p.workgroups; n < m.samples; n += p.workgroups) {
        const int64_t base = n * m.channels + low;
        Pack<T, V> in[K];
#pragma unroll
        for (int k = 0; k < K; k++) in[k] = load_pack<V>(x + base + token_offset<V>(p, k, left));
        real sum = 0, none = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) sum += k * p.threads < left ? in[k][v] : (real)0;
        sum_token(shared, buffer, sum, none);
        const real about = sum * per_value;  // as in the held kernels
        real first = 0, second = 0;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                const real d = k * p.threads < left ? in[k][v] - about : (real)0;
                first += d;
                second = fma(d, d, second);
            }
        sum_token(shared, buffer, first, second);
        const real rest = first * per_value, mean = about + rest, variance = fma(-rest, rest, second * per_value);
        const real rstd = inverse_root((variance < 0 ? (real)0 : variance) + m.eps);
        if (threadIdx.x == 0) {
            statistics[2 * (n * m.groups + group)] = mean;
            statistics[2 * (n * m.groups + group) + 1] = rstd;
        }
        by_activation(m.activation, [&](auto kind) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k * p.threads >= left) break;
                const uint32_t at = token_offset<V>(p, k, left);
                real w[V], b[V], out[V];
                load_weights<T, V>(m, weight, low, at, (real)1, w);
                load_weights<T, V>(m, bias, low, at, (real)0, b);
#pragma unroll
                for (int v = 0; v < V; v++) out[v] = activate<decltype(kind)::value, false>(fma((in[k][v] - mean) * rstd, w[v], b[v]));
                store_pack<V>(y + base + at, out);
            }
        });
    }
}

template <class T, int V, int K>
__global__ __launch_bounds__(1024) void norm_token_backward_kernel(NormShape m, Token p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                   const void *__restrict__ bias, const real *__restrict__ statistics,
                                                                   const T *__restrict__ grad_y, T *__restrict__ grad_x, real *__restrict__ partial) {
    __shared__ TokenSums shared;
    const int64_t group = blockIdx.x / (unsigned)p.workgroups, first_sample = blockIdx.x % (unsigned)p.workgroups, low = group * m.width;
    const real per_value = (real)1 / (real)m.width;
    const int left = p.units - (int)threadIdx.x;
    int buffer = 0;
    real dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int v = 0; v < V; v++) dw[k][v] = db[k][v] = 0;
    for (int64_t n = first_sample; n < m.samples; n += p.workgroups) {
        const int64_t base = n * m.channels + low;
        Pack<T, V> in[K], dy[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t at = token_offset<V>(p, k, left);
            in[k] = load_pack<V>(x + base + at);
            dy[k] = load_pack<V>(grad_y + base + at);
        }
        const Pack<real, 2> of = load_pack<2>(statistics + 2 * (n * m.groups + group));
        const real mean = of[0], rstd = of[1];
        real sum = 0, product = 0;
        // dz is computed again where it is used, as in the held kernels
        by_activation(m.activation, [&](auto kind) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k * p.threads >= left) break;
                const uint32_t at = token_offset<V>(p, k, left);
                real w[V], b[V];
                load_weights<T, V>(m, weight, low, at, (real)1, w);
                load_weights<T, V>(m, bias, low, at, (real)0, b);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const real hat = (in[k][v] - mean) * rstd;
                    const real dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(hat, w[v], b[v]));
                    db[k][v] += dz;
                    dw[k][v] = fma(dz, hat, dw[k][v]);
                    sum = fma(dz, w[v], sum);
                    product = fma(dz * w[v], hat, product);
                }
            }
        });
        if (!grad_x) continue;
        sum_token(shared, buffer, sum, product);
        const real c0 = sum * per_value, c1 = product * per_value;
        by_activation(m.activation, [&](auto kind) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (k * p.threads >= left) break;
                const uint32_t at = token_offset<V>(p, k, left);
                real w[V], b[V], out[V];
                load_weights<T, V>(m, weight, low, at, (real)1, w);
                load_weights<T, V>(m, bias, low, at, (real)0, b);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const real hat = (in[k][v] - mean) * rstd;
                    const real dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(hat, w[v], b[v]));
                    out[v] = rstd * fma(dz, w[v], fma(hat, -c1, -c0));
                }
                store_pack<V>(grad_x + base + at, out);
            }
        });
    }
    if (!partial) return;
#pragma unroll
    for (int k = 0; k < K; k++) {
        if (k * p.threads >= left) break;
        const uint32_t at = token_offset<V>(p, k, left);
        store_pack<V>(partial + first_sample * m.channels + low + at, dw[k]);
        store_pack<V>(partial + (p.workgroups + first_sample) * m.channels + low + at, db[k]);
    }
}

// ---- streamed -----------------------------------------------------------------------------------

struct Streamed {
    int units, rows, tiles;  // units of a row that a workgroup has, its rows at a time, workgroups side by side on a row
    int splits;              // workgroups one after another on a sample
    int slots;               // groups that a tile can meet
    int64_t split_rows;
};
constexpr int kNormThreads = 256, kNormAhead = 8;
// Channels of a group that a thread sums alone.  A wave for each group takes 53 us forward where threads take 45, 16 x 64 x 64 x 320 in 32 groups
// in bfloat16, and 133 where they take 26, 700 x 4098 in as many groups in float32.
constexpr int kNarrow = 16;

struct StreamedPlace {
    int unit, row;
    int64_t channel, begin, end;
    bool active;
};
template <int V> __device__ __forceinline__ StreamedPlace streamed_place(const NormShape &m, const Streamed &p, int split, int tile) {
    StreamedPlace t;
    t.row = threadIdx.x / p.units;
    t.unit = threadIdx.x - t.row * p.units;
    t.channel = ((int64_t)tile * p.units + t.unit) * V;
    t.active = t.row < p.rows && t.channel < m.channels;
    t.begin = min(split * p.split_rows, m.positions);
    t.end = min(t.begin + p.split_rows, m.positions);
    return t;
}

// The rows of a workgroup's split, kNormAhead of a thread at a time: call(in[], how many).
template <class T, int V, class Call>
__device__ __forceinline__ void over_rows(const NormShape &m, const Streamed &p, const StreamedPlace &t, const T *x, Call &&call) {
    for (int64_t r = t.begin + t.row; r < t.end; r += (int64_t)kNormAhead * p.rows) {
        const int there = (int)min((int64_t)kNormAhead, (t.end - r + p.rows - 1) / p.rows);
        call(x + r * m.channels + t.channel, there, r);
    }
}

// A tile's sums of two values by channel, summed by group: a thread each where groups are narrow, else a wave.  A group that goes on in the next tile has a sum there too.
// [sample][split][tile][group from the tile's first][2]
template <class R>
__device__ __forceinline__ void group_sums(const NormShape &m, const Streamed &p, int64_t n, int split, int tile, int columns, const R *first,
                                           const R *second, R *partial) {
    const int64_t low = (int64_t)tile * columns, high = min(low + columns, m.channels), g0 = low / m.width, g1 = (high - 1) / m.width;
    const int lanes = m.width <= kNarrow ? 1 : kWave, lane = threadIdx.x & (lanes - 1);
    for (int64_t i = threadIdx.x / lanes; i < 2 * (g1 - g0 + 1); i += kNormThreads / lanes) {
        const int64_t g = g0 + (i >> 1);
        const R *from = i & 1 ? second : first;
        R sum = 0;
        for (int64_t c = max(low, g * m.width) + lane; c < min(high, (g + 1) * m.width); c += lanes) sum += from[c - low];
        if (lanes > 1) sum = sum_lanes(sum, kWave);
        if (lane == 0) partial[((((n * p.splits + split) * p.tiles + tile) * p.slots + g - g0) << 1) + (i & 1)] = sum;
    }
}

// The sum over the splits and tiles of those of a group, by a workgroup; in its first thread.
template <int V, int Threads, class R>
__device__ __forceinline__ void sum_splits(const NormShape &m, const Streamed &p, int64_t n, int64_t g, const R *partial, double &first, double &second) {
    __shared__ double shared[2][Threads / kWave];
    const int64_t columns = (int64_t)p.units * V;
    const int t0 = (int)(g * m.width / columns), t1 = (int)(((g + 1) * m.width - 1) / columns);
    const int64_t slot = g - t0 * columns / m.width;  // in the group's first tile; the others begin within it
    first = second = 0;
    for (int s = threadIdx.x; s < p.splits; s += Threads)
        for (int t = t0; t <= t1; t++) {
            const R *at = partial + (((((n * p.splits + s) * p.tiles + t) * p.slots) + (t == t0 ? slot : 0)) << 1);
            first += at[0];
            second += at[1];
        }
    for (int d = kWave / 2; d > 0; d >>= 1) {
        first += __shfl_xor(first, d);
        second += __shfl_xor(second, d);
    }
    if ((threadIdx.x & (kWave - 1)) == 0) {
        shared[0][threadIdx.x / kWave] = first;
        shared[1][threadIdx.x / kWave] = second;
    }
    __syncthreads();
    for (int i = 1; threadIdx.x == 0 && i < Threads / kWave; i++) {
        first += shared[0][i];
        second += shared[1][i];
    }
}

// What a thread has seen of a channel: how many values (the same for its channels), their mean's distance from the first of them, and their
// squares about the mean.  A batch of rows is summed about its own first row and merged: no value that stands apart is what many others
// are measured from, so it costs no more digits than its own square is of the variance.
template <class T, int V> struct Seen {
    Pack<T, V> first = {};
    real count = 0, mean[V] = {}, squares[V] = {};
};
// `there` rows; the others are the first again, and no distance from it.
template <class T, int V> __device__ __forceinline__ void merge(Seen<T, V> &s, const Pack<T, V> (&in)[kNormAhead], int there) {
    if (s.count == 0) s.first = in[0];
    const real total = s.count + (real)there, per_row = (real)1 / (real)there, share = (real)there / total, both = s.count * share;
#pragma unroll
    for (int v = 0; v < V; v++) {
        real sum = 0, squares = 0;
#pragma unroll
        for (int k = 1; k < kNormAhead; k++) {
            const real d = in[k][v] - in[0][v];
            sum += d;
            squares = fma(d, d, squares);
        }
        const real mean = sum * per_row, apart = (in[0][v] - s.first[v] + mean) - s.mean[v];
        s.squares[v] += fma(apart * apart, both, fma(-sum, mean, squares));
        s.mean[v] = fma(apart, share, s.mean[v]);
    }
    s.count = total;
}

// Sums of x - p and its square by sample, split and group, around the group's first value p: in float32 by thread about means of its own,
// moved to p and joined in float64, where it does not matter which value of the group p is.
// 1920 x 1080 x 32 in bfloat16: 42 us (3.2 TB/s) with 126 registers; the pivot read in front of the rows takes six more and 53 us, sums about p
// in float32 took 43 and lost the variance's digits where p is far from the mean.
template <class T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_sums_kernel(NormShape m, Streamed p, const T *__restrict__ x, double *__restrict__ partial) {
    __shared__ double shared[2][kNormThreads * V];
    const int split = (int)(blockIdx.x % (unsigned)p.splits), tile = (int)(blockIdx.x / (unsigned)p.splits % (unsigned)p.tiles);
    const int64_t n = blockIdx.x / (unsigned)p.splits / (unsigned)p.tiles;
    const StreamedPlace t = streamed_place<V>(m, p, split, tile);
    x += n * m.positions * m.channels;
    Seen<T, V> seen;
    const int64_t pitch = (int64_t)p.rows * m.channels;
    if (t.active)
        over_rows<T, V>(m, p, t, x, [&](const T *from, int there, int64_t) {
            Pack<T, V> in[kNormAhead];
#pragma unroll
            for (int k = 0; k < kNormAhead; k++) in[k] = load_pack<V>(from + (k < there ? pitch * k : 0));
            merge(seen, in, there);
        });
    int g[V];
    groups_of(m, t.active ? t.channel : 0, g);
#pragma unroll
    for (int v = 0; v < V; v++) {
        const double at = (double)seen.first[v] - (double)(real)x[(int64_t)g[v] * m.width] + (double)seen.mean[v], sum = (double)seen.count * at;
        shared[0][threadIdx.x * V + v] = seen.count > 0 ? sum : 0.0;
        shared[1][threadIdx.x * V + v] = seen.count > 0 ? fma(sum, at, (double)seen.squares[v]) : 0.0;
    }
    __syncthreads();
    // sums over the rows by channel: `lines` threads a channel where there are few of them, then one
    const int columns = p.units * V, lines = max(1, min(kNormThreads / 2 / columns, p.rows)), step = lines * columns;
    for (int c = threadIdx.x; p.rows > 1 && c < 2 * step; c += kNormThreads) {
        double *at = shared[c >= step] + (c >= step ? c - step : c), sum = at[0];
        for (int i = (c >= step ? c - step : c) + step; i < p.rows * columns; i += step) sum += shared[c >= step][i];
        at[0] = sum;
    }
    if (p.rows > 1) __syncthreads();
    if (lines > 1) {
        if ((int)threadIdx.x < 2 * columns) {
            double *at = shared[(int)threadIdx.x >= columns] + ((int)threadIdx.x >= columns ? threadIdx.x - columns : threadIdx.x), sum = at[0];
            for (int i = 1; i < lines; i++) sum += at[i * columns];
            at[0] = sum;
        }
        __syncthreads();
    }
    group_sums(m, p, n, split, tile, columns, shared[0], shared[1], partial);
}

// mean and rstd of each group: a workgroup each
template <class T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_statistics_kernel(NormShape m, Streamed p, const T *__restrict__ x, const double *__restrict__ partial,
                                                                       real *__restrict__ statistics) {
    const int64_t id = blockIdx.x, n = id / m.groups, g = id % m.groups;
    double first, second;
    sum_splits<V, kNormThreads>(m, p, n, g, partial, first, second);
    if (threadIdx.x != 0) return;
    const double count = (double)m.positions * (double)m.width, rest = first / count, variance = second / count - rest * rest;
    statistics[2 * id] = (real)((double)(real)x[n * m.positions * m.channels + g * m.width] + rest);
    statistics[2 * id + 1] = (real)(1.0 / sqrt((variance < 0 ? 0.0 : variance) + (double)m.eps));
}

template <class T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormShape m, Streamed p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                  const void *__restrict__ bias, const real *__restrict__ statistics,
                                                                  T *__restrict__ y) {
    const unsigned turned = gridDim.x - 1 - blockIdx.x;
    const int64_t n = turned / (unsigned)p.splits / (unsigned)p.tiles;
    const StreamedPlace t = streamed_place<V>(m, p, (int)(turned % (unsigned)p.splits), (int)(turned / (unsigned)p.splits % (unsigned)p.tiles));
    if (!t.active) return;
    x += n * m.positions * m.channels;
    y += n * m.positions * m.channels;
    real w[V], b[V], mean[V], rstd[V];
    int g[V];
    groups_of(m, t.channel, g);
    load_weights<T, V>(m, weight, t.channel, (real)1, w);
    load_weights<T, V>(m, bias, t.channel, (real)0, b);
    load_pairs(m, n, g, statistics, mean, rstd);
#pragma unroll
    for (int v = 0; v < V; v++) w[v] *= rstd[v];
    const int64_t pitch = (int64_t)p.rows * m.channels;
    by_activation(m.activation, [&](auto kind) {
        over_rows<T, V>(m, p, t, x, [&](const T *from, int there, int64_t r) {
            Pack<T, V> in[kNormAhead];
#pragma unroll
            for (int k = 0; k < kNormAhead; k++) in[k] = load_pack<V>(from + (k < there ? pitch * k : 0));
            T *to = y + r * m.channels + t.channel;
#pragma unroll
            for (int k = 0; k < kNormAhead; k++) {
                if (k >= there) break;
                real out[V];
#pragma unroll
                for (int v = 0; v < V; v++) out[v] = activate<decltype(kind)::value, false>(fma(in[k][v] - mean[v], w[v], b[v]));
                store_pack<V>(to + pitch * k, out);
            }
        });
    });
}

// Sums of dz and dz xh by sample, split and channel, [sample][split][2][channel], and of these times the weight by group.
constexpr int kNormPairs = 4;  // rows of a thread at a time where there are two arrays to read
template <class T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_gradient_sums_kernel(NormShape m, Streamed p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                          const void *__restrict__ bias, const real *__restrict__ statistics,
                                                                          const T *__restrict__ grad_y, real *__restrict__ partial, real *__restrict__ group_partial) {
    __shared__ real shared[2][kNormThreads * V];
    const int split = (int)(blockIdx.x % (unsigned)p.splits), tile = (int)(blockIdx.x / (unsigned)p.splits % (unsigned)p.tiles);
    const int64_t n = blockIdx.x / (unsigned)p.splits / (unsigned)p.tiles;
    const StreamedPlace t = streamed_place<V>(m, p, split, tile);
    real sum[V], product[V];
#pragma unroll
    for (int v = 0; v < V; v++) sum[v] = product[v] = 0;
    if (t.active) {
        real w[V], b[V], mean[V], rstd[V];
        int g[V];
        groups_of(m, t.channel, g);
        load_weights<T, V>(m, weight, t.channel, (real)1, w);
        load_weights<T, V>(m, bias, t.channel, (real)0, b);
        load_pairs(m, n, g, statistics, mean, rstd);
#pragma unroll
        for (int v = 0; v < V; v++) w[v] *= rstd[v];
        const int64_t pitch = (int64_t)p.rows * m.channels;
        by_activation(m.activation, [&](auto kind) {
            for (int64_t r = t.begin + t.row; r < t.end; r += (int64_t)kNormPairs * p.rows) {
                const int there = (int)min((int64_t)kNormPairs, (t.end - r + p.rows - 1) / p.rows);
                const int64_t at = (n * m.positions + r) * m.channels + t.channel;
                Pack<T, V> in[kNormPairs], dy[kNormPairs];
#pragma unroll
                for (int k = 0; k < kNormPairs; k++) {
                    in[k] = load_pack<V>(x + at + (k < there ? pitch * k : 0));
                    dy[k] = load_pack<V>(grad_y + at + (k < there ? pitch * k : 0));
                }
#pragma unroll
                for (int k = 0; k < kNormPairs; k++) {
                    if (k >= there) break;
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const real d = in[k][v] - mean[v], dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(d, w[v], b[v]));
                        sum[v] += dz;
                        product[v] = fma(dz, d, product[v]);
                    }
                }
            }
        });
#pragma unroll
        for (int v = 0; v < V; v++) product[v] *= rstd[v];
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        shared[0][threadIdx.x * V + v] = sum[v];
        shared[1][threadIdx.x * V + v] = product[v];
    }
    __syncthreads();
    const int columns = p.units * V;
    for (int c = threadIdx.x; c < 2 * columns; c += kNormThreads) {
        const int which = c >= columns, column = which ? c - columns : c;
        const int64_t channel = (int64_t)tile * columns + column;
        if (channel >= m.channels) continue;
        real *at = shared[which] + column;
        real total = at[0];
        for (int i = 1; i < p.rows; i++) total += at[i * columns];
        if (partial) partial[((n * p.splits + split) * 2 + which) * m.channels + channel] = total;
        real w[1];
        load_weights<T, 1>(m, weight, channel, (real)1, w);
        at[0] = total * w[0];
    }
    __syncthreads();
    group_sums(m, p, n, split, tile, columns, shared[0], shared[1], group_partial);
}

// Sums of the weights' gradients over the parts, at the given strides: 64 threads a channel.
constexpr int kJoinThreads = 1024, kJoinColumns = 16, kJoinLines = kJoinThreads / kJoinColumns;
template <class T>
__device__ __forceinline__ void join_channel(const NormShape &m, int64_t parts, int64_t stride, int64_t which_stride, int64_t block, const real *partial,
                                             int weight_at, void *grad_weight, void *grad_bias, double (*shared)[kJoinThreads]) {
    const int column = threadIdx.x % kJoinColumns, line = threadIdx.x / kJoinColumns;
    const int64_t channel = block * kJoinColumns + column;
    double sum[2] = {0, 0};
    if (channel < m.channels)
#pragma unroll 8
        for (int64_t i = line; i < parts; i += kJoinLines) {
            sum[0] += partial[i * stride + channel];
            sum[1] += partial[i * stride + which_stride + channel];
        }
    shared[0][threadIdx.x] = sum[0];
    shared[1][threadIdx.x] = sum[1];
    for (int left = kJoinLines / 2; left > 0; left >>= 1) {
        __syncthreads();
        if (line < left) {
            shared[0][threadIdx.x] += shared[0][threadIdx.x + left * kJoinColumns];
            shared[1][threadIdx.x] += shared[1][threadIdx.x + left * kJoinColumns];
        }
    }
    __syncthreads();
    if (line < 2 && channel < m.channels) {
        void *to = line == weight_at ? grad_weight : grad_bias;
        if (to) store_weight<T>(m, to, channel, (real)shared[line][column]);
    }
}

// By group avg dxh and avg(dxh xh), a workgroup each; then the weights' gradients.
template <class T, int V>
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(NormShape m, Streamed p, const real *__restrict__ partial,
                                                                 const real *__restrict__ group_partial, real *__restrict__ averages,
                                                                 int64_t group_blocks, void *__restrict__ grad_weight, void *__restrict__ grad_bias) {
    __shared__ double shared[2][kJoinThreads];
    if (blockIdx.x < group_blocks) {
        const int64_t id = blockIdx.x;
        double sum, product;
        sum_splits<V, kJoinThreads>(m, p, id / m.groups, id % m.groups, group_partial, sum, product);
        const double count = (double)m.positions * (double)m.width;
        if (threadIdx.x == 0) {
            averages[2 * id] = (real)(sum / count);
            averages[2 * id + 1] = (real)(product / count);
        }
    } else {
        join_channel<T>(m, m.samples * p.splits, 2 * m.channels, m.channels, (int64_t)blockIdx.x - group_blocks, partial, 1, grad_weight, grad_bias, shared);
    }
}

template <class T>
__global__ __launch_bounds__(kJoinThreads) void norm_join_held_kernel(NormShape m, int64_t parts, const real *__restrict__ partial,
                                                                      void *__restrict__ grad_weight, void *__restrict__ grad_bias) {
    __shared__ double shared[2][kJoinThreads];
    join_channel<T>(m, parts, m.channels, parts * m.channels, blockIdx.x, partial, 0, grad_weight, grad_bias, shared);
}

template <class T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_gradient_kernel(NormShape m, Streamed p, const T *__restrict__ x, const void *__restrict__ weight,
                                                                     const void *__restrict__ bias, const real *__restrict__ statistics,
                                                                     const real *__restrict__ averages, const T *__restrict__ grad_y,
                                                                     T *__restrict__ grad_x) {
    const unsigned turned = gridDim.x - 1 - blockIdx.x;
    const int64_t n = turned / (unsigned)p.splits / (unsigned)p.tiles;
    const StreamedPlace t = streamed_place<V>(m, p, (int)(turned % (unsigned)p.splits), (int)(turned / (unsigned)p.splits % (unsigned)p.tiles));
    if (!t.active) return;
    real w[V], b[V], mean[V], rstd[V], sum[V], product[V];
    int g[V];
    groups_of(m, t.channel, g);
    load_weights<T, V>(m, weight, t.channel, (real)1, w);
    load_weights<T, V>(m, bias, t.channel, (real)0, b);
    load_pairs(m, n, g, statistics, mean, rstd);
    load_pairs(m, n, g, averages, sum, product);
#pragma unroll
    for (int v = 0; v < V; v++) {
        w[v] *= rstd[v];
        sum[v] *= rstd[v];
        product[v] *= rstd[v] * rstd[v];
    }
    const int64_t pitch = (int64_t)p.rows * m.channels;
    by_activation(m.activation, [&](auto kind) {
        for (int64_t r = t.begin + t.row; r < t.end; r += (int64_t)kNormPairs * p.rows) {
            const int there = (int)min((int64_t)kNormPairs, (t.end - r + p.rows - 1) / p.rows);
            const int64_t at = (n * m.positions + r) * m.channels + t.channel;
            Pack<T, V> in[kNormPairs], dy[kNormPairs];
#pragma unroll
            for (int k = 0; k < kNormPairs; k++) {
                in[k] = load_pack<V>(x + at + (k < there ? pitch * k : 0));
                dy[k] = load_pack<V>(grad_y + at + (k < there ? pitch * k : 0));
            }
#pragma unroll
            for (int k = 0; k < kNormPairs; k++) {
                if (k >= there) break;
                real out[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const real d = in[k][v] - mean[v], dz = dy[k][v] * activate<decltype(kind)::value, true>(fma(d, w[v], b[v]));
                    out[v] = fma(dz, w[v], fma(d, -product[v], -sum[v]));
                }
                store_pack<V>(grad_x + at + pitch * k, out);
            }
        }
    });
}

// ---- host -----------------------------------------------------------------------------------------

static int check_norm(const char *fn, const tg_norm *n, NormShape &m) {
    if (!n) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    const int64_t limit = (int64_t)1 << 40;
    if (n->samples < 0 || n->positions < 0 || n->channels < 1 || n->groups < 1 || n->channels % n->groups != 0 || n->channels >= ((int64_t)1 << 24) ||
        n->samples >= ((int64_t)1 << 31) || (n->positions > 0 && n->samples > limit / n->positions) || n->samples * n->positions > limit / n->channels) {
        set_error("%s: sizes", fn);
        return TG_E_ARG;
    }
    if (!type_known(n->type) || (n->weight_type != n->type && n->weight_type != kRealType)) {
        set_error("%s: types %lld and %lld", fn, (long long)n->type, (long long)n->weight_type);
        return TG_E_ARG;
    }
    if (n->activation < TG_ACTIVATION_NONE || n->activation > TG_ACTIVATION_GELU || !(n->eps >= 0)) {
        set_error("%s: activation %lld, eps %g", fn, (long long)n->activation, n->eps);
        return TG_E_ARG;
    }
    m.samples = n->samples;
    m.positions = n->positions;
    m.channels = n->channels;
    m.groups = n->groups;
    m.width = n->channels / n->groups;
    m.activation = (int)n->activation;
    m.wide_weights = n->weight_type == kRealType;
    const uintptr_t at = (uintptr_t)n->weight | (uintptr_t)n->bias;  // the widest access: eight elements of 32 bits
    m.aligned_weights = at % std::min<uintptr_t>(32, (uintptr_t)(16 / type_bytes(n->type) * type_bytes(n->weight_type))) == 0;
    m.eps = (real)n->eps;
    return 0;
}

// Elements of an access: the most that `widest` bytes hold, two of 16 bits, or one: what divides `run` and is aligned.
static int vector_of(int64_t run, int64_t bytes, std::initializer_list<const void *> pointers, int64_t widest = 16) {
    for (int v : {(int)(widest / bytes), 2}) {
        bool fits = run % v == 0 && (v == 2 ? bytes == 2 : true);
        for (const void *p : pointers) fits = fits && (uintptr_t)p % (uintptr_t)(v * bytes) == 0;
        if (fits) return v;
    }
    return 1;
}
// What a thread of the streamed backward kernels reads at once: 16 bytes, or four elements of 16 bits.  Eight of them took 149 registers for the
// sums and 87 us where four take 92 and 68 (1920 x 1080 x 32 in bfloat16); forward, where there is one array to read, eight are faster (sums 42 us
// to 50, the second reading 51 to 54).
static int64_t gradient_bytes(int64_t element) { return std::min<int64_t>(16, 4 * element); }

// call(T(), integral_constant of the elements of an access), the most of 16-bit ones being Widest.
template <int Widest = 8, class Call> static int by_vector(int64_t type, int vector, Call &&call) {
    const auto with = [&](auto t) {
        using widest = std::integral_constant<int, sizeof(t) == 2 ? Widest : 16 / (int)sizeof(t)>;
        using two = std::integral_constant<int, 2>;
        using one = std::integral_constant<int, 1>;
        if (vector == widest::value) return call(t, widest());
        if (sizeof(t) == 2 && vector == 2) return call(t, std::conditional_t<sizeof(t) == 2, two, one>());
        return call(t, one());
    };
#ifdef TG_DOUBLE_PRECISION
    (void)type;
    return with(double());
#else
    return type == TG_TYPE_F32 ? with(float()) : type == TG_TYPE_F16 ? with(half_t()) : with(bf16_t());
#endif
}

constexpr int kHeldRows = 8;        // accesses of a thread that are held
// Bytes of x up to which one launch of few workgroups beats three of many: 2500 x 32 in float32, 8 us against 14 forward, but 21 against 13
// backward, which reads twice as much.
constexpr int64_t kLittle = 1 << 20, kLittleBackward = 1 << 18;
constexpr int kHeldThreads = 1 << 19;  // of all workgroups together, which go over the samples: the chip's places
constexpr int kChain = 256;            // values that a thread adds one after another, into one channel's sum

constexpr int kTokenThreadsBackward = 1 << 18;  // half as many: each has sums of the weights' gradients to write

// A slab of groups whose rows are 64 bytes or more, if a workgroup can hold it; threads == 0: it cannot.
static Held held_of(const NormShape &m, int vector, int64_t bytes, bool backward) {
    Held p = {};
    const int64_t row = m.width * bytes;
    const bool little = m.samples * m.positions * m.channels * bytes <= (backward ? kLittleBackward : kLittle);  // near enough to be read in narrow columns
    p.slab_groups = little ? 1 : (int)std::min<int64_t>(m.groups, std::max<int64_t>(1, 64 / row));
    // all of a row where that is little: its neighbours are read by the same workgroup
    while (!little && p.slab_groups < m.groups && (int64_t)p.slab_groups * m.width * m.positions <= 1024 * vector / 2) p.slab_groups = (int)std::min<int64_t>(m.groups, p.slab_groups * 2);
    p.unit_groups = (int)(m.width / vector);
    if (m.width / vector > 1024) return p;
    const int64_t units = (int64_t)p.slab_groups * p.unit_groups;
    if (units > 1024) return p;
    p.units = (int)units;
    const int64_t most = 1024 / units;  // rows at a time of the largest workgroup
    if (m.positions > most * kHeldRows) return p;
    // few accesses a thread where there are few positions, more where it takes them
    p.rows = (int)std::min<int64_t>(m.positions, std::max<int64_t>(ceil_div64(m.positions, kHeldRows), std::max<int64_t>(1, 256 / units)));
    if (p.rows > most) p.rows = (int)most;
    const int line = p.rows * p.units;
    p.teams = (int)std::max<int64_t>(1, std::min<int64_t>(m.samples, (line < 256 ? 256 : 1024) / line));
    p.threads = (p.teams * line + kWave - 1) / kWave * kWave;
    p.turns = ceil_div64(m.samples, p.teams);
    p.in_wave = p.rows == 1 && (p.unit_groups & (p.unit_groups - 1)) == 0 && p.unit_groups <= kWave;
    return p;
}
static size_t held_lds(const Held &p, int vector, bool backward) {
    return sizeof(real) * std::max<size_t>(p.in_wave ? 0 : 2 * ((size_t)p.threads + (size_t)p.teams * p.slab_groups), backward ? (size_t)p.threads * vector : 0);
}

// threads == 0: the samples have more positions, their groups fit a wave or no workgroup holds one.
static Token token_of(const NormShape &m, int vector, bool backward) {
    Token p = {};
    const int64_t units = m.width / vector, all = token_accesses(vector);
    if (m.positions != 1 || units <= kWave || units > 1024 * all) return p;
    p.units = (int)units;
    p.single = backward && units <= 1024;
    const int64_t most = p.single ? 1 : all;
    p.threads = (int)(ceil_div64(ceil_div64(units, most), kWave) * kWave);
    const int64_t places = (backward ? kTokenThreadsBackward : kHeldThreads) / p.threads / m.groups;
    p.workgroups = (int)std::min<int64_t>(m.samples, std::max(places, backward ? ceil_div64(m.samples, kChain) : 1));
    return p;
}

static Streamed streamed_of(const NormShape &m, int vector) {
    Streamed p = {};
    const int64_t units = m.channels / vector;
    p.units = (int)std::min<int64_t>(units, kNormThreads);
    p.tiles = (int)ceil_div64(units, p.units);
    p.rows = kNormThreads / p.units;
    // about eight workgroups a CU, of no fewer rows than a thread reads ahead; or two a CU of two rows a thread, where there is less work:
    // 3 x 1961 x 120 in 45 workgroups was 13 to 21 us a launch, in 180 it is 9 to 11
    const auto splits = [&](int64_t rows, int64_t workgroups) {
        return std::max<int64_t>(1, std::min(ceil_div64(m.positions, p.rows * rows), ceil_div64(workgroups, m.samples * p.tiles)));
    };
    p.splits = (int)std::max(std::max(splits(kNormAhead, 2048), splits(2, 512)), ceil_div64(m.positions, (int64_t)p.rows * kChain));
    p.split_rows = ceil_div64(ceil_div64(m.positions, p.splits), p.rows) * p.rows;
    p.splits = (int)ceil_div64(m.positions, p.split_rows);
    p.slots = (int)std::min<int64_t>(m.groups, ((int64_t)p.units * vector - 2 + m.width) / m.width + 1);
    return p;
}

struct NormPlan {
    bool held, token;
    int vector;
    Held h;
    Token t;
    Streamed s;
    int64_t parts, partial, by_group, averages;  // partial sums by channel and by group, averages: reals
    int64_t blocks;
    int threads;
};
static NormPlan plan_of(const NormShape &m, int64_t type, bool backward, bool aligned_only, std::initializer_list<const void *> pointers) {
    NormPlan p = {};
    const int64_t bytes = type_bytes(type);
    p.vector = aligned_only ? vector_of(m.width, bytes, {}) : vector_of(m.width, bytes, pointers);
    p.t = token_of(m, p.vector, backward);
    p.token = p.t.threads > 0;
    if (p.token) {
        p.parts = backward ? p.t.workgroups : 0;
        p.partial = 2 * p.parts * m.channels;
        p.blocks = p.t.workgroups * m.groups;
        p.threads = p.t.threads;
        return p;
    }
    p.h = held_of(m, p.vector, bytes, backward);
    const int64_t slabs = p.h.slab_groups ? ceil_div64(m.groups, p.h.slab_groups) : 0;
    // few workgroups leave most of the chip idle: a sample is then better split
    p.held = p.h.threads > 0 && (p.h.turns * slabs >= 128 || m.samples * m.positions * m.channels * bytes <= (backward ? kLittleBackward : kLittle));
    if (p.held) {
        const int64_t places = std::max<int64_t>(1, kHeldThreads / p.h.threads / slabs), turns = kChain / ceil_div64(m.positions, p.h.rows);
        p.h.workgroups = (int)std::min(p.h.turns, std::max(places, backward ? ceil_div64(p.h.turns, turns) : 1));
        p.parts = backward ? p.h.workgroups : 0;
        p.partial = 2 * p.parts * m.channels;
        p.blocks = p.h.workgroups * slabs;
        p.threads = p.h.threads;
        return p;
    }
    const int64_t widest = backward ? gradient_bytes(bytes) : 16;
    p.vector = aligned_only ? vector_of(m.channels, bytes, {}, widest) : vector_of(m.channels, bytes, pointers, widest);
    p.s = streamed_of(m, p.vector);
    p.parts = m.samples * p.s.splits;
    p.partial = backward ? p.parts * 2 * m.channels : 0;
    p.by_group = p.parts * p.s.tiles * p.s.slots * 2 * (backward ? 1 : (int64_t)(sizeof(double) / sizeof(real)));  // forward: float64
    p.blocks = p.parts * p.s.tiles;
    p.threads = kNormThreads;
    p.averages = backward ? m.samples * m.groups * 2 : 0;
    return p;
}
static int64_t norm_bytes(const NormPlan &p) { return (p.partial + p.by_group + p.averages) * (int64_t)sizeof(real); }

// A grid has fewer than 2^32 threads.
static bool beyond_a_grid(const NormShape &m, const NormPlan &p) {
    const int64_t joins = (p.held || p.token ? 0 : m.samples * m.groups) + ceil_div64(m.channels, kJoinColumns), most = (int64_t)1 << 32;
    return p.blocks >= most / p.threads || joins >= most / kJoinThreads;
}

static int too_many(const char *fn) {
    set_error("%s: too many samples", fn);
    return TG_E_ARG;
}

// Of the workspace, whatever the alignment of the tensors turns out to be.
static int64_t norm_room(const NormShape &m, int64_t type, bool backward) {
    if (m.samples == 0 || m.positions == 0) return 0;
    int64_t most = norm_bytes(plan_of(m, type, backward, true, {}));
    for (int by : {1, 2, 4, 8}) most = std::max(most, norm_bytes(plan_of(m, type, backward, false, {(const void *)(uintptr_t)(16 + by)})));
    return most;
}

}  // namespace tg

extern "C" int tg_group_norm_sizes(const tg_norm *n, int64_t out[2]) {
    using namespace tg;
    NormShape m;
    if (const int code = check_norm("tg_group_norm_sizes", n, m)) return code;
    if (!out) {
        set_error("tg_group_norm_sizes: null pointer");
        return TG_E_ARG;
    }
    out[0] = norm_room(m, n->type, false);
    out[1] = norm_room(m, n->type, true);
    return 0;
}

extern "C" int tg_group_norm_forward(const tg_norm *n) {
    using namespace tg;
    const char *fn = "tg_group_norm_forward";
    NormShape m;
    if (const int code = check_norm(fn, n, m)) return code;
    if (m.samples == 0 || m.positions == 0) return 0;
    if (!n->x || !n->y || !n->statistics) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    const NormPlan p = plan_of(m, n->type, false, false, {n->x, n->y});
    if (beyond_a_grid(m, p)) return too_many(fn);
    if (norm_bytes(p) > 0 && (!n->workspace || n->workspace_bytes < norm_bytes(p))) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)n->workspace_bytes, (long long)norm_bytes(p));
        return TG_E_WORKSPACE;
    }
    hipStream_t stream = (hipStream_t)n->stream;
    return by_vector(n->type, p.vector, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        const T *x = (const T *)n->x;
        if (p.token) {
            TG_LAUNCH_AS("norm_token_forward", (norm_token_forward_kernel<T, V, token_accesses(V)>), dim3((unsigned)p.blocks), dim3((unsigned)p.t.threads), 0, stream, m, p.t, x,
                         n->weight, n->bias, (T *)n->y, n->statistics);
            return check_launch(fn);
        }
        if (p.held) {
            const dim3 grid((unsigned)p.blocks), block((unsigned)p.h.threads);
            const size_t lds = held_lds(p.h, V, false);
            if (m.positions <= p.h.rows)
                TG_LAUNCH_AS("norm_forward", (norm_held_forward_kernel<T, V, 1>), grid, block, lds, stream, m, p.h, x, n->weight, n->bias, (T *)n->y,
                             n->statistics);
            else
                TG_LAUNCH_AS("norm_forward", (norm_held_forward_kernel<T, V, kHeldRows>), grid, block, lds, stream, m, p.h, x, n->weight, n->bias,
                             (T *)n->y, n->statistics);
            return check_launch(fn);
        }
        const dim3 grid((unsigned)p.blocks), block(kNormThreads);
        double *partial = (double *)n->workspace;
        TG_LAUNCH_AS("norm_sums", (norm_sums_kernel<T, V>), grid, block, 0, stream, m, p.s, x, partial);
        TG_LAUNCH_AS("norm_statistics", (norm_statistics_kernel<T, V>), dim3((unsigned)(m.samples * m.groups)), block, 0,
                     stream, m, p.s, x, partial, n->statistics);
        TG_LAUNCH_AS("norm_apply", (norm_apply_kernel<T, V>), grid, block, 0, stream, m, p.s, x, n->weight, n->bias, n->statistics, (T *)n->y);
        return check_launch(fn);
    });
}

namespace tg {
template <class T> __global__ __launch_bounds__(kNormThreads) void norm_no_gradient_kernel(NormShape m, void *grad_weight, void *grad_bias) {
    for (int64_t c = threadIdx.x; c < m.channels; c += kNormThreads) {
        if (grad_weight) store_weight<T>(m, grad_weight, c, (real)0);
        if (grad_bias) store_weight<T>(m, grad_bias, c, (real)0);
    }
}
}  // namespace tg

extern "C" int tg_group_norm_backward(const tg_norm *n) {
    using namespace tg;
    const char *fn = "tg_group_norm_backward";
    NormShape m;
    if (const int code = check_norm(fn, n, m)) return code;
    const bool empty = m.samples == 0 || m.positions == 0, weights = n->grad_weight || n->grad_bias;
    if ((empty || !n->grad_x) && !weights) return 0;
    hipStream_t stream = (hipStream_t)n->stream;
    if (empty)
        return by_vector(n->type, 1, [&](auto t, auto) {
            TG_LAUNCH_AS("norm_no_gradient", (norm_no_gradient_kernel<decltype(t)>), dim3(1), dim3(kNormThreads), 0, stream, m, n->grad_weight, n->grad_bias);
            return check_launch(fn);
        });
    if (!n->x || !n->grad_y || !n->statistics) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    const NormPlan p = plan_of(m, n->type, true, false, {n->x, n->grad_y, n->grad_x});
    if (beyond_a_grid(m, p)) return too_many(fn);
    if (!n->workspace || n->workspace_bytes < norm_bytes(p)) {
        set_error("%s: workspace of %lld bytes, %lld needed", fn, (long long)n->workspace_bytes, (long long)norm_bytes(p));
        return TG_E_WORKSPACE;
    }
    real *partial = (real *)n->workspace;
    const unsigned channel_blocks = (unsigned)ceil_div64(m.channels, kJoinColumns);
    if (p.token || p.held)
        return by_vector(n->type, p.vector, [&](auto t, auto v) {
            using T = decltype(t);
            constexpr int V = decltype(v)::value;
            const T *x = (const T *)n->x, *dy = (const T *)n->grad_y;
            const dim3 grid((unsigned)p.blocks), block((unsigned)(p.token ? p.t.threads : p.h.threads));
            const size_t lds = p.token ? 0 : held_lds(p.h, V, true);
            if (p.token && p.t.single)
                TG_LAUNCH_AS("norm_token_backward", (norm_token_backward_kernel<T, V, 1>), grid, block, lds, stream, m, p.t, x, n->weight, n->bias,
                             n->statistics, dy, (T *)n->grad_x, weights ? partial : nullptr);
            else if (p.token)
                TG_LAUNCH_AS("norm_token_backward", (norm_token_backward_kernel<T, V, token_accesses(V)>), grid, block, lds, stream, m, p.t, x, n->weight,
                             n->bias, n->statistics, dy, (T *)n->grad_x, weights ? partial : nullptr);
            else if (m.positions <= p.h.rows)
                TG_LAUNCH_AS("norm_backward", (norm_held_backward_kernel<T, V, 1>), grid, block, lds, stream, m, p.h, x, n->weight, n->bias, n->statistics,
                             dy, (T *)n->grad_x, weights ? partial : nullptr);
            else
                TG_LAUNCH_AS("norm_backward", (norm_held_backward_kernel<T, V, kHeldRows>), grid, block, lds, stream, m, p.h, x, n->weight, n->bias,
                             n->statistics, dy, (T *)n->grad_x, weights ? partial : nullptr);
            if (weights)
                TG_LAUNCH_AS("norm_join", (norm_join_held_kernel<T>), dim3(channel_blocks), dim3(kJoinThreads), 0, stream, m, p.parts, partial,
                             n->grad_weight, n->grad_bias);
            return check_launch(fn);
        });
    return by_vector<4>(n->type, p.vector, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        const T *x = (const T *)n->x, *dy = (const T *)n->grad_y;
        const dim3 grid((unsigned)p.blocks), block(kNormThreads);
        real *by_group = partial + p.partial, *averages = by_group + p.by_group;
        TG_LAUNCH_AS("norm_gradient_sums", (norm_gradient_sums_kernel<T, V>), grid, block, 0, stream, m, p.s, x, n->weight, n->bias, n->statistics, dy,
                     weights ? partial : nullptr, by_group);
        const int64_t group_blocks = n->grad_x ? m.samples * m.groups : 0;
        TG_LAUNCH_AS("norm_join", (norm_join_kernel<T, V>), dim3((unsigned)group_blocks + (weights ? channel_blocks : 0)), dim3(kJoinThreads), 0, stream, m,
                     p.s, partial, by_group, averages, group_blocks, n->grad_weight, n->grad_bias);
        if (n->grad_x)
            TG_LAUNCH_AS("norm_gradient", (norm_gradient_kernel<T, V>), grid, block, 0, stream, m, p.s, x, n->weight, n->bias, n->statistics, averages, dy,
                         (T *)n->grad_x);
        return check_launch(fn);
    });
}
