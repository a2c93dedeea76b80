// tg_elements.hpp -- tensors of 16, 32 and 64 bits an element as the operators read and write them: a few neighbouring elements in one
// access, computed on in `real` (32 bits, or 64 in the double library) and rounded once, to nearest, where they are stored.
#pragma once
#include "tg_common.hpp"

namespace tg {

using half_t = _Float16;
using bf16_t = __bf16;

// V neighbouring elements.  Powers of two are one access, aligned as such; three are three neighbours that nothing aligns.
template <class T, int V> struct alignas((V & (V - 1)) == 0 ? V * sizeof(T) : sizeof(T)) Pack {
    T v[V];
    __device__ __forceinline__ real operator[](int i) const { return (real)v[i]; }
};

template <int V, class T> __device__ __forceinline__ Pack<T, V> load_pack(const T *p) { return *reinterpret_cast<const Pack<T, V> *>(p); }

template <int V, class T> __device__ __forceinline__ void store_pack(T *p, const real *v) {
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; i++) out.v[i] = (T)v[i];
    *reinterpret_cast<Pack<T, V> *>(p) = out;
}

// The value of another lane of the sixteen, by the data-parallel move's control.
template <int Control> __device__ __forceinline__ float from_lane(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), Control, 0xf, 0xf, true));
}
template <int Control> __device__ __forceinline__ double from_lane(double v) {
    const uint64_t bits = (uint64_t)__double_as_longlong(v);
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, Control, 0xf, 0xf, true);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), Control, 0xf, 0xf, true);
    return __longlong_as_double((long long)((uint64_t)high << 32 | low));
}
constexpr int kRotate8 = 0x128, kMirrorOf8 = 0x141, kSwapOnes = 0xb1, kSwapTwos = 0x4e;

// The sum over `lanes` neighbouring lanes (a power of two, aligned), in each of them.
template <class R> __device__ __forceinline__ R sum_lanes(R v, int lanes) {
    if (lanes >= 2) v += from_lane<kSwapOnes>(v);
    if (lanes >= 4) v += from_lane<kSwapTwos>(v);
    if (lanes >= 8) v += from_lane<kMirrorOf8>(v);
    if (lanes >= 16) v += from_lane<kRotate8>(v);
    if (lanes >= 32) v += __shfl_xor(v, 16);
    if (lanes >= 64) v += __shfl_xor(v, 32);
    return v;
}

inline int64_t type_bytes(int64_t type) { return type == TG_TYPE_F64 ? 8 : type == TG_TYPE_F32 ? 4 : 2; }
#ifdef TG_DOUBLE_PRECISION
constexpr int64_t kRealType = TG_TYPE_F64;
inline bool type_known(int64_t type) { return type == TG_TYPE_F64; }
#else
constexpr int64_t kRealType = TG_TYPE_F32;
inline bool type_known(int64_t type) { return type == TG_TYPE_F32 || type == TG_TYPE_F16 || type == TG_TYPE_BF16; }
#endif

// call(T(), S()) with the element type of a tensor and that of its companion (gates, weights): the same, or tg_real.
template <class Call> int by_types(int64_t type, int64_t second, Call &&call) {
#ifdef TG_DOUBLE_PRECISION
    (void)type;
    (void)second;
    return call(double(), double());
#else
    switch (type) {
        case TG_TYPE_F32: return call(float(), float());
        case TG_TYPE_F16: return second == TG_TYPE_F32 ? call(half_t(), float()) : call(half_t(), half_t());
        default: return second == TG_TYPE_F32 ? call(bf16_t(), float()) : call(bf16_t(), bf16_t());
    }
#endif
}

}  // namespace tg
