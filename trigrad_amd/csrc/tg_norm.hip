// tg_norm.hip -- group norm with an activation behind it, channels last.
//
//     xh = (x - mean) rstd,  z = weight xh + bias,  y = act(z),  mean and rstd of a sample's positions x (channels / groups)
//     dz = dy act'(z),  dweight = sum dz xh,  dbias = sum dz,  dxh = weight dz,  dx = rstd (dxh - avg dxh - xh avg(dxh xh))
#include "tg_elements.hpp"

namespace tg {

struct NormShape {
    int64_t samples, positions, channels, groups, width;  // width: channels of a group
    int activation;
    real eps;
};

// act(z) and act'(z)
__device__ __forceinline__ void activate(int kind, real z, real &y, real &slope) {
    if (kind == TG_ACTIVATION_RELU) {
        y = z < 0 ? (real)0 : z;  // NaN stays
        slope = z > 0 ? (real)1 : (real)0;
    } else if (kind == TG_ACTIVATION_SILU) {
        const real s = (real)1 / ((real)1 + exp(-z));
        y = z * s;
        slope = s * ((real)1 + z * ((real)1 - s));
    } else if (kind == TG_ACTIVATION_GELU) {
        const real phi = (real)0.5 * erfc(z * (real)-0.70710678118654752440);
        y = z * phi;
        slope = phi + z * exp((real)-0.5 * z * z) * (real)0.39894228040143267794;
    } else {
        y = z;
        slope = (real)1;
    }
}

constexpr int kNormThreads = 256;

__device__ __forceinline__ real block_sum(real v, real *shared) {
    __syncthreads();
    shared[threadIdx.x] = v;
    for (int n = kNormThreads / 2; n > 0; n >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < n) shared[threadIdx.x] += shared[threadIdx.x + n];
    }
    __syncthreads();
    return shared[0];
}

// A workgroup for a sample's group.
template <class T, class S>
__global__ __launch_bounds__(kNormThreads) void norm_forward_kernel(NormShape m, const T *__restrict__ x, const S *__restrict__ weight,
                                                                    const S *__restrict__ bias, T *__restrict__ y,
                                                                    real *__restrict__ statistics) {
    __shared__ real shared[kNormThreads];
    const int64_t n = blockIdx.x / m.groups, g = blockIdx.x % m.groups, count = m.positions * m.width;
    const int64_t base = n * m.positions * m.channels + g * m.width;
    const real pivot = (real)x[base];  // sums of differences from it: a mean far from zero takes no digits of the variance
    real sum = 0;
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) sum += (real)x[base + i / m.width * m.channels + i % m.width] - pivot;
    const real mean = pivot + block_sum(sum, shared) / (real)count;
    sum = 0;
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) {
        const real d = (real)x[base + i / m.width * m.channels + i % m.width] - mean;
        sum += d * d;
    }
    const real rstd = (real)1 / sqrt(block_sum(sum, shared) / (real)count + m.eps);
    if (threadIdx.x == 0) {
        statistics[2 * (int64_t)blockIdx.x] = mean;
        statistics[2 * (int64_t)blockIdx.x + 1] = rstd;
    }
    for (int64_t i = threadIdx.x; i < count; i += kNormThreads) {
        const int64_t c = i % m.width, at = base + i / m.width * m.channels + c;
        real z = ((real)x[at] - mean) * rstd, out, slope;
        if (weight) z = z * (real)weight[g * m.width + c];
        if (bias) z = z + (real)bias[g * m.width + c];
        activate(m.activation, z, out, slope);
        y[at] = (T)out;
    }
}

template <class T, class S>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(NormShape m, const T *__restrict__ x, const S *__restrict__ weight,
                                                                     const S *__restrict__ bias, const real *__restrict__ statistics,
                                                                     const T *__restrict__ grad_y, T *__restrict__ grad_x) {
    __shared__ real shared[kNormThreads];
    const int64_t n = blockIdx.x / m.groups, g = blockIdx.x % m.groups, count = m.positions * m.width;
    const int64_t base = n * m.positions * m.channels + g * m.width;
    const real mean = statistics[2 * (int64_t)blockIdx.x], rstd = statistics[2 * (int64_t)blockIdx.x + 1];
    real sum = 0, product = 0;
    for (int pass = 0; pass < 2; pass++) {
        for (int64_t i = threadIdx.x; i < count; i += kNormThreads) {
            const int64_t c = i % m.width, at = base + i / m.width * m.channels + c;
            const real hat = ((real)x[at] - mean) * rstd, w = weight ? (real)weight[g * m.width + c] : (real)1;
            real out, slope;
            activate(m.activation, hat * w + (bias ? (real)bias[g * m.width + c] : (real)0), out, slope);
            const real d = (real)grad_y[at] * slope * w;
            if (pass == 0) {
                sum += d;
                product += d * hat;
            } else {
                grad_x[at] = (T)(rstd * (d - sum - hat * product));
            }
        }
        if (pass == 0) {
            sum = block_sum(sum, shared) / (real)count;
            product = block_sum(product, shared) / (real)count;
        }
    }
}

// A workgroup for a channel.
template <class T, class S>
__global__ __launch_bounds__(kNormThreads) void norm_weights_kernel(NormShape m, const T *__restrict__ x, const S *__restrict__ weight,
                                                                    const S *__restrict__ bias, const real *__restrict__ statistics,
                                                                    const T *__restrict__ grad_y, S *__restrict__ grad_weight,
                                                                    S *__restrict__ grad_bias) {
    __shared__ real shared[kNormThreads];
    const int64_t c = blockIdx.x, g = c / m.width;
    real sum = 0, product = 0;
    for (int64_t i = threadIdx.x; i < m.samples * m.positions; i += kNormThreads) {
        const int64_t n = i / m.positions, at = i * m.channels + c;
        const real hat = ((real)x[at] - statistics[2 * (n * m.groups + g)]) * statistics[2 * (n * m.groups + g) + 1];
        real out, slope;
        activate(m.activation, hat * (weight ? (real)weight[c] : (real)1) + (bias ? (real)bias[c] : (real)0), out, slope);
        sum += (real)grad_y[at] * slope;
        product += (real)grad_y[at] * slope * hat;
    }
    sum = block_sum(sum, shared);
    product = block_sum(product, shared);
    if (threadIdx.x == 0) {
        if (grad_weight) grad_weight[c] = (S)product;
        if (grad_bias) grad_bias[c] = (S)sum;
    }
}

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
    m.eps = (real)n->eps;
    return 0;
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
    out[0] = out[1] = 0;
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
    return by_types(n->type, n->weight_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        TG_LAUNCH_AS("norm_forward", (norm_forward_kernel<T, S>), dim3((unsigned)(m.samples * m.groups)), dim3(kNormThreads), 0,
                     (hipStream_t)n->stream, m, (const T *)n->x, (const S *)n->weight, (const S *)n->bias, (T *)n->y, n->statistics);
        return check_launch(fn);
    });
}

extern "C" int tg_group_norm_backward(const tg_norm *n) {
    using namespace tg;
    const char *fn = "tg_group_norm_backward";
    NormShape m;
    if (const int code = check_norm(fn, n, m)) return code;
    const bool empty = m.samples == 0 || m.positions == 0;
    if ((empty || !n->grad_x) && !n->grad_weight && !n->grad_bias) return 0;
    if (!empty && (!n->x || !n->grad_y || !n->statistics)) {
        set_error("%s: null pointer", fn);
        return TG_E_ARG;
    }
    return by_types(n->type, n->weight_type, [&](auto t, auto s) {
        using T = decltype(t);
        using S = decltype(s);
        hipStream_t stream = (hipStream_t)n->stream;
        if (n->grad_x && !empty)
            TG_LAUNCH_AS("norm_backward", (norm_backward_kernel<T, S>), dim3((unsigned)(m.samples * m.groups)), dim3(kNormThreads), 0, stream, m,
                         (const T *)n->x, (const S *)n->weight, (const S *)n->bias, n->statistics, (const T *)n->grad_y, (T *)n->grad_x);
        if (n->grad_weight || n->grad_bias)
            TG_LAUNCH_AS("norm_weights", (norm_weights_kernel<T, S>), dim3((unsigned)m.channels), dim3(kNormThreads), 0, stream, m,
                         (const T *)n->x, (const S *)n->weight, (const S *)n->bias, n->statistics, (const T *)n->grad_y,
                         (S *)n->grad_weight, (S *)n->grad_bias);
        return check_launch(fn);
    });
}
