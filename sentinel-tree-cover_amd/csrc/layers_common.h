// Shared by the channels-last layer operators (group_norm.hip, linear.hip): element types, unaligned vector access, activations.
#pragma once
#include <cmath>
#include <type_traits>

#include "ttc_internal.h"

namespace layers {

typedef _Float16 f16;
typedef __bf16 bf16;
template <class T, int N> using vec = T __attribute__((ext_vector_type(N)));

// Vector access at the alignment of one element: rows of a channel slice start anywhere.  gfx950 serves a 16-byte global access at any
// address, so these stay single instructions.
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&o)[V]) {
    T t[V];
    __builtin_memcpy(t, p, sizeof t);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)t[i];
}
// the ONE rounding of a result to its type (nearest even; the identity for fp32)
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
    T t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)v[i];
    __builtin_memcpy(p, t, sizeof t);
}

// exp(-v) overflows to +inf for v < -88 and 1 / inf is 0: the limits come out without a branch.  v_rcp_f32 is within 1 ulp.
__device__ __forceinline__ float sigmoidf(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
// 1 - 2 / (1 + e^2v) cancels near 0 (absolute error 1e-7): below 1/2 the odd Taylor series to v^15 (next term 9e-9 of v at 1/2) keeps the
// relative accuracy.  Coefficients: 2^2k (2^2k - 1) B_2k / (2k)!.
__device__ __forceinline__ float tanh_rel(float v) {
    const float t = v * v;
    const float p = v + v * t * (-1.0f / 3 + t * (2.0f / 15 + t * (-17.0f / 315 + t * (62.0f / 2835 + t * (-1382.0f / 155925
                    + t * (21844.0f / 6081075 + t * (-929569.0f / 638512875.0f)))))));
    const float e = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * v));
    return fabsf(v) < 0.5f ? p : e;
}

// h = normal distribution function of -|z|, and e = exp(-z^2 / 2).  h = erfc(x) / 2 with x = |z| / sqrt 2, and erfc(x) = exp(-x^2) t P(t),
// t = 1 / (1 + 0.356 x): P is the degree-9 Chebyshev fit of exp(x^2) erfc(x) / t over t in (0, 1] (0.356 minimises its error; P is halved below):
// with the rounded coefficients within 4e-8 of its value everywhere.  No 1 + erf: the negative tail keeps its relative accuracy.  A quarter of the registers
// of the library's erfc, which set the kernels' occupancy.
__device__ __forceinline__ float normal_tail(float z, float* e) {
    const float az = fabsf(z), t = __builtin_amdgcn_rcpf(1.0f + (0.356f * 0.70710678f) * az);
    const float p = 0.100425743f + t * (0.100426443f + t * (0.094032362f + t * (0.081815816f + t * (0.0595245f + t * (0.061009083f
                    + t * (-0.027474117f + t * (0.08918602f + t * (-0.078777514f + t * 0.01983167f))))))));
    *e = __builtin_amdgcn_exp2f(-0.72134752f * (z * z));        // log2(e) / 2
    return t * p * *e;
}

// act(z) / act'(z) of one element for a fixed activation
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == TTC_ACT_RELU) return z < 0.0f ? 0.0f : z;               // keeps NaN
    if constexpr (ACT == TTC_ACT_SWISH) return z * sigmoidf(z);
    if constexpr (ACT == TTC_ACT_SIGMOID) return sigmoidf(z);
    if constexpr (ACT == TTC_ACT_TANH) return tanh_rel(z);
    if constexpr (ACT == TTC_ACT_GELU) { float e; const float h = normal_tail(z, &e); return z * (z < 0.0f ? h : 1.0f - h); }
    return z;
}
// sigmoid' and tanh' go through e = exp(-|z|), r = 1 / (1 + e): sigmoid' = e r^2 has no 1 - s that cancels for large |z|.  swish' = s (1 + z (1 - s))
// may cancel: it is 1 where that happens.  These slopes are what bounds the 16-bit norm's backward pass (64 lanes a CU and clock, a quarter of
// that for exp and rcp), so every instruction counts.
template <int ACT>
__device__ __forceinline__ float slope_of(float z) {
    if constexpr (ACT == TTC_ACT_RELU) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
    if constexpr (ACT == TTC_ACT_GELU) { float e; const float h = normal_tail(z, &e); return (z < 0.0f ? h : 1.0f - h) + z * 0.39894228f * e; }
    if constexpr (ACT == TTC_ACT_SWISH) { const float s = sigmoidf(z); return s * (1.0f + z * (1.0f - s)); }
    if constexpr (ACT == TTC_ACT_SIGMOID || ACT == TTC_ACT_TANH) {
        const float e = __expf((ACT == TTC_ACT_TANH ? -2.0f : -1.0f) * fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e), er2 = e * r * r;
        return ACT == TTC_ACT_TANH ? 4.0f * er2 : er2;
    }
    return 1.0f;
}
// the same on a vector: ONE uniform branch per vector
template <class F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case TTC_ACT_RELU: f(std::integral_constant<int, TTC_ACT_RELU>{}); break;
        case TTC_ACT_SWISH: f(std::integral_constant<int, TTC_ACT_SWISH>{}); break;
        case TTC_ACT_SIGMOID: f(std::integral_constant<int, TTC_ACT_SIGMOID>{}); break;
        case TTC_ACT_TANH: f(std::integral_constant<int, TTC_ACT_TANH>{}); break;
        case TTC_ACT_GELU: f(std::integral_constant<int, TTC_ACT_GELU>{}); break;
        default: break;
    }
}
template <int V>
__device__ __forceinline__ void act_vec(float (&z)[V], int act) {
    with_act(act, [&](auto k) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = act_of<decltype(k)::value>(z[i]);
    });
}
// d[i] *= act'(z[i])
template <int V>
__device__ __forceinline__ void slope_vec(float (&d)[V], const float (&z)[V], int act) {
    with_act(act, [&](auto k) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] *= slope_of<decltype(k)::value>(z[i]);
    });
}

template <class F>
inline ttc_status with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case TTC_DT_F32: return f(float{});
        case TTC_DT_F16: return f(f16{});
        default: return f(bf16{});
    }
}
inline bool known_dtype(int d) { return d == TTC_DT_F32 || d == TTC_DT_F16 || d == TTC_DT_BF16; }
inline bool known_act(int a) { return a >= TTC_ACT_NONE && a <= TTC_ACT_GELU; }
inline int dtype_bytes(int d) { return d == TTC_DT_F32 ? 4 : 2; }

// Launches go to the context's device whatever the caller's current device is; the caller's is put back.
struct DeviceGuard {
    int prev = -1;
    bool ok;
    explicit DeviceGuard(int dev) {
        ok = hipGetDevice(&prev) == hipSuccess;
        if (ok && prev != dev) ok = hipSetDevice(dev) == hipSuccess;
        else if (ok) prev = -1;
    }
    ~DeviceGuard() { if (prev >= 0) (void)hipSetDevice(prev); }
};

}  // namespace layers
