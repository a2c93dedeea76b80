// tg_adamw.hip -- one step of AdamW over many tensors, with averages in `real` or in 8 bits.
//
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p (1 - rate decay) - rate / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes an element in float32 (p, g, m, v read, p, m, v written) for about twenty operations; with gradients and copies in
// 16 bits and averages in 8, 16.  Every operation is rounded by itself (no fused multiply-add), so that what an 8-bit value
// becomes does not depend on how a compiler orders them.
//
// The 8-bit averages are m and sqrt(v) (what the step divides by, with half of v's exponents), in units of a block's largest / 448.  With
// b2 = 0.999 an average changes by up to a thousandth of itself in a step, and neighbours in 8 bits are a sixteenth apart: rounded to nearest it
// would stay where it is for good.  So it becomes the upper neighbour with the probability of what lies below.
#include "tg_elements.hpp"

#include <cmath>
#include <type_traits>
#include <vector>

namespace tg {

constexpr int kThreads = 256;
constexpr int kBlock = 256;           // elements of one scale, and of a wave at a time
constexpr int kTurns = 4;             // blocks of a wave
constexpr int kPiece = 4 * kTurns * kBlock;  // elements of a workgroup
constexpr int64_t kMostOfOne = (int64_t)1 << 31;  // elements of one entry of the table

struct Nothing {};
template <class C> constexpr bool kCopies = !std::is_same<C, Nothing>::value;

// A launch's tensors are in its arguments, of which there are 4 KB: no copy of a table has to arrive first, and a graph keeps its own.
template <bool Copies, int Bits> constexpr int kTensors = Bits == 8 ? (Copies ? 58 : 66) : Copies ? 80 : 96;

template <class C, int Bits> struct AdamwLaunch {
    static constexpr int kMost = kTensors<kCopies<C>, Bits>;
    real *p[kMost];
    const void *g[kMost];
    void *m[kMost], *v[kMost];
    C *copy[kCopies<C> ? kMost : 1];
    real *scales[Bits == 8 ? kMost : 1];
    uint32_t size[kMost], piece[kMost];         // piece: the launch's first workgroup of the tensor
    uint32_t place[Bits == 8 ? kMost : 1];      // of the first element, in blocks of all tensors laid end to end
    const float *step, *rate_at;
    const real *grad_scale;
    double rate, decay, left1, left2;  // for what is known on the device alone: 1 - b^t, or log b where t is read there
    real keep, size_of_step, unbias, b1, b1_rest, b2, b2_rest, eps;
    uint32_t noise;
    int count, maximize;
    uint64_t wide[2];  // a bit for each tensor: its parts are aligned for accesses of four elements
};

// What the step multiplies with.
struct AdamwFactors {
    real keep, size_of_step, unbias, scale;
    uint32_t noise;
};
constexpr uint32_t kNoiseOfSeed = 0x85EBCA6Bu;
template <class L> __device__ __forceinline__ AdamwFactors factors_of(const L &a) {
    AdamwFactors f = {a.keep, a.size_of_step, a.unbias, a.grad_scale ? a.grad_scale[0] : (real)1, a.noise};
    if (a.step || a.rate_at) {  // in 64 bits, as the host has it
        const double rate = a.rate_at ? (double)a.rate_at[0] : a.rate;
        f.keep = (real)(1.0 - rate * a.decay);
        const double t = a.step ? (double)a.step[0] : 0.0;
        const double left1 = a.step ? -expm1(t * a.left1) : a.left1, left2 = a.step ? -expm1(t * a.left2) : a.left2;
        f.size_of_step = (real)(rate / left1);
        f.unbias = (real)(1.0 / sqrt(left2));
        f.noise += (uint32_t)(int64_t)t * kNoiseOfSeed;  // the step's number belongs to the seed, so that replays do not all round alike
    }
    if (a.maximize) f.scale = -f.scale;
    return f;
}

// ---- 8 bits -------------------------------------------------------------------------------

#ifndef TG_DOUBLE_PRECISION
constexpr float kLargest8 = 448.0f, kLeastLargest = 0x1p-110f;  // a block whose largest is below becomes zeros

// Products by odd constants and shifts: those of C. Wellons' published search for 32-bit mixers of little bias (2018).  The seed's factor and summand are the
// odd constants of A. Appleby's published finalizer (2011), a place's is the prime next to 2^32 over the golden ratio
// of D. Knuth's multiplicative hashing.
__device__ __forceinline__ uint32_t mixed(uint32_t x) {
    x = (x ^ x >> 16) * 0x7FEB352Du;
    x = (x ^ x >> 15) * 0x846CA68Bu;
    return x ^ x >> 16;
}

// One of the two neighbours of x * unit in 8 bits, as a float.
template <bool Least> __device__ __forceinline__ float neighbour8(float x, float unit, uint32_t noise) {
    const float y = fminf(fabsf(x) * unit, kLargest8);
    // a NaN stays one: the minimum of it and 448 would be 448
    const float normal = __uint_as_float((__float_as_uint(y) + (noise << 4)) & ~0xFFFFFu);
    float small = floorf(y * 512.0f + (float)noise * 0x1p-16f);
    if (Least && y > 0.0f) small = fmaxf(small, 1.0f);
    const float z = y >= 0x1p-6f ? normal : small * 0x1p-9f;
    return x != x ? x : copysignf(z, x);
}

__device__ __forceinline__ float largest_of_wave(float v) {
    v = fmaxf(v, from_lane<kSwapOnes>(v));
    v = fmaxf(v, from_lane<kSwapTwos>(v));
    v = fmaxf(v, from_lane<kMirrorOf8>(v));
    v = fmaxf(v, from_lane<kRotate8>(v));
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ void from8(uint32_t w, float scale, float *x) {
    x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * scale;
    x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale;
    x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale;
    x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale;
}
__device__ __forceinline__ uint32_t to8(const float *x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
}
#endif

// ---- the kernel ---------------------------------------------------------------------------

// Four elements of a block that begins at `at`: neighbours in one access (Wide), or 64 apart for tensors that begin off alignment and ends of tensors,
// zeros behind the end.  All loads are made, in place of those behind the end the last element's, so that none waits for another's result.
template <bool Wide, class T> __device__ __forceinline__ void take4(const T *p, uint32_t at, uint32_t lane, uint32_t size, T *x) {
    if (Wide) {
        const Pack<T, 4> v = load_pack<4>(p + at + 4 * lane);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = v.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = p[min(at + lane + 64 * j, size - 1)];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = at + lane + 64 * j < size ? x[j] : (T)0.0f;
    }
}
template <bool Wide, class T> __device__ __forceinline__ void put4(T *p, uint32_t lane, uint32_t left, const real *x) {
    if (Wide) {
        store_pack<4>(p + 4 * lane, x);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 64 * j < left) p[lane + 64 * j] = (T)x[j];
    }
}

template <class G, class C, int Bits> struct AdamwBlock {  // what a lane has of a block
    G g[4];
    real p[4], m[4], v[4];
    uint32_t m8, v8;
    real scale_m, scale_r;
};

template <bool Wide, class G, class C, int Bits>
__device__ __forceinline__ void load_block(AdamwBlock<G, C, Bits> &b, const AdamwLaunch<C, Bits> &a, int n, uint32_t at, uint32_t lane, uint32_t size) {
    take4<Wide>((const G *)a.g[n], at, lane, size, b.g);
    take4<Wide>(a.p[n], at, lane, size, b.p);
    if constexpr (Bits == 8) {
        const uint8_t *m = (const uint8_t *)a.m[n], *v = (const uint8_t *)a.v[n];
        if (Wide) {
            b.m8 = *(const uint32_t *)(m + at + 4 * lane);
            b.v8 = *(const uint32_t *)(v + at + 4 * lane);
        } else {
            uint8_t m4[4], v4[4];
            take4<false>(m, at, lane, size, m4);
            take4<false>(v, at, lane, size, v4);
            b.m8 = b.v8 = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                b.m8 |= (uint32_t)m4[j] << 8 * j;
                b.v8 |= (uint32_t)v4[j] << 8 * j;
            }
        }
        const uint32_t block = Wide ? at / kBlock : min(at, size - 1) / kBlock;
        b.scale_m = a.scales[n][block * 2];
        b.scale_r = a.scales[n][block * 2 + 1];
    } else {
        take4<Wide>((const real *)a.m[n], at, lane, size, b.m);
        take4<Wide>((const real *)a.v[n], at, lane, size, b.v);
    }
}

template <bool Wide, class G, class C, int Bits>
__device__ __forceinline__ void step_block(AdamwBlock<G, C, Bits> &b, const AdamwLaunch<C, Bits> &a, const AdamwFactors &f, int n, uint32_t at, uint32_t lane,
                                           uint32_t left) {
    real root[4];
#ifndef TG_DOUBLE_PRECISION
    if constexpr (Bits == 8) {
        from8(b.m8, b.scale_m, b.m);
        from8(b.v8, b.scale_r, root);
#pragma unroll
        for (int j = 0; j < 4; j++) b.v[j] = root[j] * root[j];
    }
#endif
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const real g = (real)b.g[j] * f.scale;
        b.m[j] = b.m[j] * a.b1 + g * a.b1_rest;
        b.v[j] = b.v[j] * a.b2 + (g * g) * a.b2_rest;
        root[j] = sqrt(b.v[j]);
        b.p[j] = b.p[j] * f.keep - f.size_of_step * (b.m[j] / (root[j] * f.unbias + a.eps));
    }
    put4<Wide>(a.p[n] + at, lane, left, b.p);
    if constexpr (kCopies<C>) put4<Wide>(a.copy[n] + at, lane, left, b.p);
    if constexpr (Bits == 32) {
        put4<Wide>((real *)a.m[n] + at, lane, left, b.m);
        put4<Wide>((real *)a.v[n] + at, lane, left, b.v);
    }
#ifndef TG_DOUBLE_PRECISION
    if constexpr (Bits == 8) {
        float most_m = 0.0f, most_r = 0.0f;  // what lies behind the tensor's end came as zeros and is zero still
#pragma unroll
        for (int j = 0; j < 4; j++) {
            most_m = fmaxf(most_m, fabsf(b.m[j]));
            most_r = fmaxf(most_r, root[j]);
        }
        most_m = largest_of_wave(most_m);
        most_r = largest_of_wave(most_r);
        const float unit_m = most_m >= kLeastLargest ? 1.0f / most_m * kLargest8 : 0.0f, unit_r = most_r >= kLeastLargest ? 1.0f / most_r * kLargest8 : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t place = a.place[n] * kBlock + at + (Wide ? 4 * lane + j : lane + 64 * j);
            const uint32_t noise = mixed(place * 0x9E3779B1u + f.noise);
            b.m[j] = neighbour8<false>(b.m[j], unit_m, noise & 0xFFFFu);
            root[j] = neighbour8<true>(root[j], unit_r, noise >> 16);
        }
        uint8_t *m = (uint8_t *)a.m[n] + at, *v = (uint8_t *)a.v[n] + at;
        const uint32_t m8 = to8(b.m), v8 = to8(root);
        if (Wide) {
            *(uint32_t *)(m + 4 * lane) = m8;
            *(uint32_t *)(v + 4 * lane) = v8;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (lane + 64 * j < left) {
                    m[lane + 64 * j] = (uint8_t)(m8 >> 8 * j);
                    v[lane + 64 * j] = (uint8_t)(v8 >> 8 * j);
                }
        }
        if (lane == 0) {
            a.scales[n][at / kBlock * 2] = most_m >= kLeastLargest ? most_m * (1.0f / kLargest8) : 0.0f;
            a.scales[n][at / kBlock * 2 + 1] = most_r >= kLeastLargest ? most_r * (1.0f / kLargest8) : 0.0f;
        }
    }
#endif
}

// A wave has four blocks of its workgroup's sixteen, all of which are read before the first is computed on.  12 M elements in float32: 50.6 us, 6.6 TB/s
// where part of them is still in the last-level cache, 69 us and 4.9 TB/s for a whole call; 160 M with gradients and copies in bfloat16 861 us, 5.2 TB/s,
// with averages in 8 bits 501 us, 5.1 TB/s; 320 tensors of 2800 elements 6.8 us a launch of 80.
template <class G, class C, int Bits> __global__ __launch_bounds__(kThreads) void adamw_kernel(const AdamwLaunch<C, Bits> a) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int n = -1;  // the last tensor that begins here or before
    for (int first = 0; first < a.count; first += kWave) {
        const int i = first + (int)lane;
        n += __popcll(__ballot(i < a.count && a.piece[min(i, a.count - 1)] <= blockIdx.x));
    }
    n = __builtin_amdgcn_readfirstlane(n);
    const uint32_t size = a.size[n], begin = (blockIdx.x - a.piece[n]) * (uint32_t)kPiece + wave * kBlock;
    const AdamwFactors f = factors_of(a);
    const bool wide = (a.wide[n >> 6] >> (n & 63) & 1) != 0;
    AdamwBlock<G, C, Bits> b[kTurns];
    if (wide && begin + (kTurns - 1) * 4 * kBlock + kBlock <= size) {
#pragma unroll
        for (int u = 0; u < kTurns; u++) load_block<true>(b[u], a, n, begin + u * 4 * kBlock, lane, size);
#pragma unroll
        for (int u = 0; u < kTurns; u++) step_block<true>(b[u], a, f, n, begin + u * 4 * kBlock, lane, kBlock);
        return;
    }
    if (begin >= size) return;
#pragma unroll
    for (int u = 0; u < kTurns; u++) load_block<false>(b[u], a, n, begin + u * 4 * kBlock, lane, size);
#pragma unroll
    for (int u = 0; u < kTurns; u++) {
        const uint32_t at = begin + u * 4 * kBlock;
        if (at < size) step_block<false>(b[u], a, f, n, at, lane, size - at);
    }
}

// ---- host ---------------------------------------------------------------------------------

struct Entry {
    int64_t tensor, first, size, place;
};

template <class G, class C, int Bits> static int launch(const tg_adamw &c, const std::vector<Entry> &entries) {
    AdamwLaunch<C, Bits> a = {};
    a.step = c.device_step;
    a.rate_at = c.device_rate;
    a.grad_scale = c.grad_scale;
    a.rate = c.rate;
    a.decay = c.decay;
    const double left1 = 1.0 - std::pow(c.beta1, c.step), left2 = 1.0 - std::pow(c.beta2, c.step);
    a.left1 = c.device_step ? std::log(c.beta1) : left1;
    a.left2 = c.device_step ? std::log(c.beta2) : left2;
    a.keep = (real)(1.0 - c.rate * c.decay);
    a.size_of_step = (real)(c.rate / left1);
    a.unbias = (real)(1.0 / std::sqrt(left2));
    a.b1 = (real)c.beta1;
    a.b1_rest = (real)(1.0 - c.beta1);
    a.b2 = (real)c.beta2;
    a.b2_rest = (real)(1.0 - c.beta2);
    a.eps = (real)c.eps;
    a.noise = (uint32_t)c.seed * kNoiseOfSeed + 0xC2B2AE35u;
    a.maximize = c.maximize != 0;
    constexpr int kMost = AdamwLaunch<C, Bits>::kMost;
    static_assert(sizeof(a) <= 4096 && kMost <= 128, "kernel arguments, and a bit of `wide` each");
    int64_t pieces = 0;
    const auto flush = [&]() {
        if (a.count)
            TG_LAUNCH_AS("adamw", (adamw_kernel<G, C, Bits>), dim3((unsigned)pieces), dim3(kThreads), 0, (hipStream_t)c.stream, a);
        a.count = 0;
        a.wide[0] = a.wide[1] = 0;
        pieces = 0;
    };
    for (const Entry &e : entries) {
        const int64_t more = ceil_div64(e.size, kPiece);
        if (a.count == kMost || (pieces + more) >= ((int64_t)1 << 32) / kThreads) flush();
        const int n = a.count++;
        a.p[n] = c.params[e.tensor] + e.first;
        a.g[n] = (const G *)c.grads[e.tensor] + e.first;
        constexpr int64_t kBytes = Bits == 8 ? 1 : sizeof(real);
        a.m[n] = (char *)c.averages[e.tensor] + e.first * kBytes;
        a.v[n] = (char *)c.squares[e.tensor] + e.first * kBytes;
        const auto aligned = [](const void *p, size_t bytes) { return (uintptr_t)p % (4 * bytes) == 0; };
        bool wide = aligned(a.p[n], sizeof(real)) && aligned(a.g[n], sizeof(G)) && aligned(a.m[n], kBytes) && aligned(a.v[n], kBytes);
        if constexpr (kCopies<C>) {
            a.copy[n] = (C *)c.copies[e.tensor] + e.first;
            wide = wide && aligned(a.copy[n], sizeof(C));
        }
        if constexpr (Bits == 8) {
            a.scales[n] = c.scales[e.tensor] + e.first / kBlock * 2;
            a.place[n] = (uint32_t)e.place;
        }
        a.size[n] = (uint32_t)e.size;
        a.piece[n] = (uint32_t)pieces;
        if (wide) a.wide[n >> 6] |= (uint64_t)1 << (n & 63);
        pieces += more;
    }
    flush();
    return check_launch("tg_adamw_step");
}

template <class G, class C> static int by_bits(const tg_adamw &c, const std::vector<Entry> &entries) {
#ifndef TG_DOUBLE_PRECISION
    if (c.bits == 8) return launch<G, C, 8>(c, entries);
#endif
    return launch<G, C, 32>(c, entries);
}

}  // namespace tg

using namespace tg;

static int adamw_call(const tg_adamw *c) {
    const char *fn = "tg_adamw_step";
    const auto refuse = [fn](const char *what) {
        set_error("%s: %s", fn, what);
        return TG_E_ARG;
    };
    if (!c || c->count < 0) return refuse("null pointer or negative count");
    if (c->count == 0) return 0;
    if (!c->params || !c->grads || !c->averages || !c->squares || !c->sizes || !c->grad_types) return refuse("null pointer");
    if (c->bits != 32 && c->bits != 8) return refuse("bits must be 32 or 8");
#ifdef TG_DOUBLE_PRECISION
    if (c->bits == 8) return refuse("averages in 8 bits belong to the float library");
#endif
    if (c->bits == 8 && !c->scales) return refuse("averages in 8 bits need scales");
    if (c->copies && !c->copy_types) return refuse("copies need types");
    if (!(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0) || !(c->eps >= 0.0) || (!c->device_step && !(c->step >= 1.0)))
        return refuse("betas are at least 0 and below 1, eps at least 0, steps count from 1");
    // tensors of the same types in one launch: three types of gradients, and no copy or one of two types
    std::vector<Entry> groups[4][3];
    int64_t place = 0;
    for (int64_t i = 0; i < c->count; i++) {
        const int64_t n = c->sizes[i], copy = c->copies && c->copies[i] ? c->copy_types[i] : -1;
        if (n < 0 || n > (int64_t)1 << 40) return refuse("a tensor's size");
        if (n == 0) continue;
        if (!c->params[i] || !c->grads[i] || !c->averages[i] || !c->squares[i] || (c->bits == 8 && !c->scales[i])) return refuse("null pointer");
        if (!type_known(c->grad_types[i]) || (copy >= 0 && copy != TG_TYPE_F16 && copy != TG_TYPE_BF16)) return refuse("a tensor's type");
#ifdef TG_DOUBLE_PRECISION
        if (copy >= 0) return refuse("copies in 16 bits belong to the float library");
#endif
        auto &group = groups[c->grad_types[i]][copy < 0 ? 0 : copy == TG_TYPE_F16 ? 1 : 2];
        for (int64_t first = 0; first < n; first += kMostOfOne) group.push_back({i, first, std::min(n - first, kMostOfOne), place + first / kBlock});
        place += ceil_div64(n, kBlock);
    }
    for (int64_t type = 0; type < 4; type++)
        for (int copy = 0; copy < 3; copy++) {
            const auto &group = groups[type][copy];
            if (group.empty()) continue;
            int code = 0;
#ifdef TG_DOUBLE_PRECISION
            code = by_bits<double, Nothing>(*c, group);
#else
            const auto with = [&](auto g) {
                using G = decltype(g);
                return copy == 0 ? by_bits<G, Nothing>(*c, group) : copy == 1 ? by_bits<G, half_t>(*c, group) : by_bits<G, bf16_t>(*c, group);
            };
            code = type == TG_TYPE_F32 ? with(float()) : type == TG_TYPE_F16 ? with(half_t()) : with(bf16_t());
#endif
            if (code) return code;
        }
    return 0;
}

extern "C" int tg_adamw_step(const tg_adamw *c) {
    try {
        return adamw_call(c);
    } catch (...) {  // the lists' memory
        set_error("tg_adamw_step: no memory for %lld tensors", (long long)c->count);
        return TG_E_ARG;
    }
}
