// Shared by the channels-last layer operators (group_norm.hip, linear.hip): element types, unaligned vector access, activations.
#pragma once
#include <cmath>

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
// 1 - 2 / (1 + e^2v) cancels near 0 (absolute error 1e-7): below 1/2 the odd Taylor series to v^13 (next term 6e-8 of v at 1/2) keeps the
// relative accuracy.  Coefficients: 2^2k (2^2k - 1) B_2k / (2k)!.
__device__ __forceinline__ float tanh_rel(float v) {
    const float t = v * v;
    const float p = v + v * t * (-1.0f / 3 + t * (2.0f / 15 + t * (-17.0f / 315 + t * (62.0f / 2835 + t * (-1382.0f / 155925
                    + t * (21844.0f / 6081075 + t * (-929569.0f / 638512875.0f)))))));
    const float e = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * v));
    return fabsf(v) < 0.5f ? p : e;
}

__device__ __forceinline__ float act_one(float z, int act) {
    switch (act) {
        case TTC_ACT_RELU: return z < 0.0f ? 0.0f : z;               // keeps NaN
        case TTC_ACT_SWISH: return z * sigmoidf(z);
        case TTC_ACT_SIGMOID: return sigmoidf(z);
        case TTC_ACT_TANH: return tanh_rel(z);
        case TTC_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678f);   // erfc, not 1 + erf: no cancellation in the negative tail
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case TTC_ACT_RELU: return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
        case TTC_ACT_SWISH: { const float s = sigmoidf(z); return s + z * s * sigmoidf(-z); }
        case TTC_ACT_SIGMOID: return sigmoidf(z) * sigmoidf(-z);       // not s (1 - s): no cancellation for large z
        case TTC_ACT_TANH: { const float s = sigmoidf(2.0f * z); return 4.0f * s * sigmoidf(-2.0f * z); }   // 1 - tanh^2, same reason
        case TTC_ACT_GELU: return 0.5f * erfcf(z * -0.70710678f) + z * 0.39894228f * __expf(-0.5f * z * z);
        default: return 1.0f;
    }
}
// the same on a vector: one uniform branch per vector
template <int V>
__device__ __forceinline__ void act_vec(float (&z)[V], int act) {
    if (act == TTC_ACT_NONE) return;
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = act_one(z[i], act);
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
