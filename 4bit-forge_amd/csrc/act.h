// Activations of the gated rows and of the int4 product's epilogue, and the 16-bit conversions
// both kernels use.  Everything in f32: a result is rounded once, where it is stored.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include "../../include/forge_hip.h"

namespace forge {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_bits_to_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// round to nearest even (v_cvt_pk_bf16_f32); NaN stays NaN
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    v2 v;
    v[0] = (__bf16)lo;
    v[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// 1 / (1 + e^-v): exp to 2 ulp and a 1-ulp reciprocal are 14 bits finer than the 16-bit results
__device__ __forceinline__ float sigmoid_f32(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-v));
}

// gelu in its tanh form: 0.5 v (1 + tanh(t)) = v * sigmoid(2 t), t = sqrt(2/pi) (v + 0.044715 v^3)
__device__ __forceinline__ float gelu_2t(float v) {
    return 1.5957691216057308f * __builtin_fmaf(0.044715f * v * v, v, v);
}

__device__ __forceinline__ float act_f32(int act, float v) {
    switch (act) {
        case FORGE_ACT_SILU: return v * sigmoid_f32(v);
        // below -10 the value is under 1e-22 of its argument: 0, also where v * v overflows
        case FORGE_ACT_GELU: return v < -10.0f ? 0.0f : v > 10.0f ? v : v * sigmoid_f32(gelu_2t(v));
        case FORGE_ACT_RELU: return v < 0.0f ? 0.0f : v;      // NaN stays NaN
        default: return v;
    }
}

// out = act(v) * times, N values: the activation is looked at once, so that the values' chains overlap
template <int N, typename V>
__device__ __forceinline__ void act_times(int act, const V& v, const V& times, float (&out)[N]) {
    auto all = [&](int fixed) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = act_f32(fixed, v[i]) * times[i];
    };
    switch (act) {
        case FORGE_ACT_SILU: all(FORGE_ACT_SILU); break;
        case FORGE_ACT_GELU: all(FORGE_ACT_GELU); break;
        case FORGE_ACT_RELU: all(FORGE_ACT_RELU); break;
        default: all(FORGE_ACT_NONE);
    }
}

// the same in place, without the product
template <int N>
__device__ __forceinline__ void act_all(int act, float (&v)[N]) {
    auto all = [&](int fixed) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = act_f32(fixed, v[i]);
    };
    switch (act) {
        case FORGE_ACT_SILU: all(FORGE_ACT_SILU); break;
        case FORGE_ACT_GELU: all(FORGE_ACT_GELU); break;
        case FORGE_ACT_RELU: all(FORGE_ACT_RELU); break;
        default: break;
    }
}

// the activation and its derivative
__device__ __forceinline__ void act_grad_f32(int act, float v, float& a, float& da) {
    switch (act) {
        case FORGE_ACT_SILU: {
            const float s = sigmoid_f32(v);
            a = v * s;
            da = s * __builtin_fmaf(v, 1.0f - s, 1.0f);
            break;
        }
        case FORGE_ACT_GELU: {
            if (v < -10.0f || v > 10.0f) {
                a = v < 0.0f ? 0.0f : v;
                da = v < 0.0f ? 0.0f : 1.0f;
                break;
            }
            const float s = sigmoid_f32(gelu_2t(v));
            const float dt = 1.5957691216057308f * __builtin_fmaf(3.0f * 0.044715f * v, v, 1.0f);
            a = v * s;
            da = s * __builtin_fmaf(v * dt, 1.0f - s, 1.0f);
            break;
        }
        case FORGE_ACT_RELU: a = v < 0.0f ? 0.0f : v; da = v > 0.0f ? 1.0f : v <= 0.0f ? 0.0f : v; break;
        default: a = v; da = 1.0f;
    }
}

}  // namespace forge
