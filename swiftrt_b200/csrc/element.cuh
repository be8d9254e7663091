// Element types and activations shared by the kernels: conversions between the stored types and
// fp32 (round to nearest even on the way back) and the activation functions by their enum values.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace srt {

enum : uint32_t { kActSigmoid = 0, kActRelu = 1, kActTanh = 2, kActIdentity = 5, kActGelu = 6, kActGeluTanh = 7, kActSilu = 8 };

__device__ __forceinline__ float apply_activation(uint32_t act, float x)
{
    switch (act) {
    case kActRelu: return x >= 0.0f ? x : 0.0f;
    case kActSigmoid: return 1.0f / (1.0f + expf(-x));
    case kActTanh: return tanhf(x);
    case kActGelu: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f));
    case kActGeluTanh: {
        float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
        return 0.5f * x * (1.0f + tanhf(u));
    }
    case kActSilu: return x / (1.0f + expf(-x));
    default: return x;
    }
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

// The logistic function to a relative error of (6 + 0.61 |a|) 2^-23: the argument -log2(e) a of the power of two is rounded to fp32, which
// counts with its size (4 units at -10, 16 at -40; an exact argument would take four more instructions a gate, and 16-bit results do not
// show it).  The .ftz forms of the two approximations take one instruction each where the others rescale denormals around them: what is
// below 2^-126 is zero.
__device__ __forceinline__ float exp2_ftz(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_ftz(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float logistic(float a)
{
    return reciprocal_ftz(1.0f + exp2_ftz(-kLog2E * a));
}
// The activation of a gate.  For results of 16 bits the logistic function is the one above (ten bits below the result's
// rounding); Float32 takes the exact forms.
template <typename T> __device__ __forceinline__ float gate_activation(uint32_t act, float x)
{
    if constexpr (sizeof(T) == 2) {
        switch (act) {
        case kActSigmoid: return logistic(x);
        case kActSilu: return x * logistic(x);
        default: break;
        }
    }
    return apply_activation(act, x);
}

// its slope at the pre-activation value x
template <typename T> __device__ __forceinline__ float gate_slope(uint32_t act, float x)
{
    switch (act) {
    case kActRelu: return x > 0.0f ? 1.0f : 0.0f;
    case kActSigmoid: {
        const float s = gate_activation<T>(kActSigmoid, x);
        return s * gate_activation<T>(kActSigmoid, -x);
    }
    case kActTanh: {
        const float t = tanhf(x);
        return 1.0f - t * t;
    }
    case kActSilu: {
        const float s = gate_activation<T>(kActSigmoid, x);
        return s * (1.0f + x * gate_activation<T>(kActSigmoid, -x));
    }
    case kActGelu:
        return 0.5f * (1.0f + erff(x * 0.70710678118654752440f)) + x * 0.39894228040143267794f * expf(-0.5f * x * x);
    case kActGeluTanh: {
        const float t = tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x));
        return 0.5f * (1.0f + t) + 0.5f * x * (1.0f - t * t) * 0.7978845608028654f * (1.0f + 3.0f * 0.044715f * x * x);
    }
    default: return 1.0f;
    }
}

// s(a) with 1 - s(a), each to the relative error of logistic(): with e = exp(-a) they are 1 / (1 + e) and
// e / (1 + e), neither of which is the difference of 1 and its neighbour (a gate at 0.9999 keeps its decay 1 - f to full
// precision).  For the pair e is capped at 2^126, so that a closed gate is 2^-126 and not 0 times infinity.
struct Gate { float on, off; };
__device__ __forceinline__ float min_or_nan(float a, float b)
{
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ Gate logistic_pair(float a)
{
    const float e = exp2_ftz(min_or_nan(-kLog2E * a, 126.0f));
    const float on = reciprocal_ftz(1.0f + e);
    return Gate{on, e * on};
}

// activation and slope of VEC values, what they share computed once; the selector is uniform, so the switch is taken once
template <typename T, int VEC> __device__ __forceinline__ void gate_values(uint32_t act, const float (&z)[VEC], float (&a)[VEC], float (&slope)[VEC])
{
    if constexpr (sizeof(T) == 2) {
        if (act == kActSilu) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Gate s = logistic_pair(z[j]);
                a[j] = z[j] * s.on;
                slope[j] = fmaf(a[j], s.off, s.on);                  // s + z s (1 - s), with 1 - s not as a difference
            }
            return;
        }
    }
    switch (act) {
#define SRT_GATE_CASE(A)                                                        \
    case A:                                                                     \
        _Pragma("unroll") for (int j = 0; j < VEC; ++j) {                       \
            a[j] = gate_activation<T>(A, z[j]);                                 \
            slope[j] = gate_slope<T>(A, z[j]);                                  \
        }                                                                       \
        break
    SRT_GATE_CASE(kActSilu);
    SRT_GATE_CASE(kActGelu);
    SRT_GATE_CASE(kActGeluTanh);
    SRT_GATE_CASE(kActRelu);
    SRT_GATE_CASE(kActSigmoid);
    SRT_GATE_CASE(kActTanh);
    SRT_GATE_CASE(kActIdentity);
#undef SRT_GATE_CASE
    default: break;
    }
}

// 32 values of one accumulator row; the selector is uniform, so the switch is taken once
template <typename T> __device__ __forceinline__ void gate_chunk(uint32_t act, float (&v)[32])
{
    switch (act) {
#define SRT_GATE_CASE(A)                                                        \
    case A:                                                                     \
        _Pragma("unroll") for (int j = 0; j < 32; ++j) v[j] = gate_activation<T>(A, v[j]); \
        break
    SRT_GATE_CASE(kActSilu);
    SRT_GATE_CASE(kActGelu);
    SRT_GATE_CASE(kActGeluTanh);
    SRT_GATE_CASE(kActRelu);
    SRT_GATE_CASE(kActSigmoid);
    SRT_GATE_CASE(kActTanh);
#undef SRT_GATE_CASE
    default: break;
    }
}

}  // namespace srt
