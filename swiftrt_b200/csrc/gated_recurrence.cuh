// Gated linear recurrence over time and its backward pass.  Per batch item b and channel d
//     f_t = s(forget_t),   i_t = input ? s(input_t) : 1 - f_t            (s: the logistic function)
//     c_t = f_t c_{t-1} + i_t update_t,   hidden_t = output ? c_t s(output_t) : c_t
// with the state c in fp32.  A step at or behind the item's length leaves the state as it is and its hidden value
// is zero.  Backward, with p_t = dhidden_t s(output_t) and the gradient of the last state added at the last step:
//     dc_t = p_t + f_{t+1} dc_{t+1}
//     dupdate_t = dc_t i_t,      doutput_t = dhidden_t c_t s(output_t) (1 - s(output_t))
//     dforget_t = dc_t (c_{t-1} - [update_t when i = 1 - f]) f_t (1 - f_t),   dinput_t = dc_t update_t i_t (1 - i_t)
//     dinitial  = f_1 dc_1
// The forward pass keeps the state before every 64th step (fp32), from which the backward pass recomputes the
// states in between: 1/16 of the bytes of one 16-bit tensor instead of a second output of 4 bytes per element.
#pragma once
#include "element.cuh"

namespace srt {

constexpr uint32_t kRecurrenceChunk = 64;       // steps between two kept states

struct Strided3 { const void* p; long long b, t, d; };          // element strides; p may be null
struct Strided3W { void* p; long long b, t, d; };

struct RecurrenceParams {
    Strided3 x, f, i, o;                 // update, forget, input, output
    const float* initial; long long initial_b, initial_d;
    const int32_t* lengths;
    Strided3W y;                         // forward: hidden
    float* last; long long last_b, last_d;
    float* states; long long states_b, states_c, states_d;
    // backward only (states is read)
    Strided3 dy;
    const float* dlast; long long dlast_b, dlast_d;
    Strided3W dx, df, di, dout;
    float* dinitial; long long dinitial_b, dinitial_d;
    uint32_t B, T, D;
};

// s(a) and 1 - s(a), each to a relative error of a few 2^-23: both come from e = exp(-|a|), so the small one of the two
// is not the difference of 1 and its neighbour (a gate at 0.9999 keeps its decay 1 - f to full precision).
struct Gate { float on, off; };
__device__ __forceinline__ Gate logistic_pair(float a)
{
    const float e = __expf(-fabsf(a));
    const float big = __fdividef(1.0f, 1.0f + e), small = e * big;
    return a >= 0.0f ? Gate{big, small} : Gate{small, big};          // a NaN is in e already
}

template <typename T> __device__ __forceinline__ float load3(const Strided3& s, uint32_t b, uint32_t t, uint32_t d)
{
    return to_float<T>(static_cast<const T*>(s.p)[b * s.b + t * s.t + d * s.d]);
}
template <typename T> __device__ __forceinline__ void store3(const Strided3W& s, uint32_t b, uint32_t t, uint32_t d, float v)
{
    static_cast<T*>(s.p)[b * s.b + t * s.t + d * s.d] = from_float<T>(v);
}

__device__ __forceinline__ uint32_t live_steps(const RecurrenceParams& p, uint32_t b)
{
    if (p.lengths == nullptr) return p.T;
    const int32_t n = p.lengths[b];
    return n < 0 ? 0u : min(static_cast<uint32_t>(n), p.T);
}

// One thread per channel of one batch item, step after step.
template <typename T>
__global__ void __launch_bounds__(128)
recurrence_steps_kernel(const __grid_constant__ RecurrenceParams p)
{
    const unsigned long long id = blockIdx.x * 128ull + threadIdx.x;
    if (id >= static_cast<unsigned long long>(p.B) * p.D) return;
    const uint32_t b = static_cast<uint32_t>(id / p.D), d = static_cast<uint32_t>(id % p.D);
    const uint32_t n = live_steps(p, b);
    float c = p.initial ? p.initial[b * p.initial_b + d * p.initial_d] : 0.0f;
    for (uint32_t t = 0; t < p.T; ++t) {
        if (p.states && t % kRecurrenceChunk == 0) p.states[b * p.states_b + (t / kRecurrenceChunk) * p.states_c + d * p.states_d] = c;
        float y = 0.0f;
        if (t < n) {
            const Gate f = logistic_pair(load3<T>(p.f, b, t, d));
            const float x = load3<T>(p.x, b, t, d);
            c = fmaf(f.on, c, (p.i.p ? logistic_pair(load3<T>(p.i, b, t, d)).on : f.off) * x);
            y = p.o.p ? c * logistic_pair(load3<T>(p.o, b, t, d)).on : c;
        }
        store3<T>(p.y, b, t, d, y);
    }
    if (p.last) p.last[b * p.last_b + d * p.last_d] = c;
}

// The same for the backward pass: chunk after chunk from the end, the states of a chunk recomputed from its kept one.
template <typename T>
__global__ void __launch_bounds__(128)
recurrence_steps_backward_kernel(const __grid_constant__ RecurrenceParams p)
{
    const unsigned long long id = blockIdx.x * 128ull + threadIdx.x;
    if (id >= static_cast<unsigned long long>(p.B) * p.D) return;
    const uint32_t b = static_cast<uint32_t>(id / p.D), d = static_cast<uint32_t>(id % p.D);
    const uint32_t n = live_steps(p, b);
    float carry = p.dlast ? p.dlast[b * p.dlast_b + d * p.dlast_d] : 0.0f;         // f_{t+1} dc_{t+1}
    for (uint32_t t = p.T; t-- > n;) {
        store3<T>(p.dx, b, t, d, 0.0f);
        store3<T>(p.df, b, t, d, 0.0f);
        if (p.i.p) store3<T>(p.di, b, t, d, 0.0f);
        if (p.o.p) store3<T>(p.dout, b, t, d, 0.0f);
    }
    for (uint32_t chunk = (n + kRecurrenceChunk - 1) / kRecurrenceChunk; chunk-- > 0;) {
        const uint32_t t0 = chunk * kRecurrenceChunk, t1 = min(n, t0 + kRecurrenceChunk);
        float before[kRecurrenceChunk];
        float c = p.states[b * p.states_b + chunk * p.states_c + d * p.states_d];
        for (uint32_t t = t0; t < t1; ++t) {
            before[t - t0] = c;
            const Gate f = logistic_pair(load3<T>(p.f, b, t, d));
            const float x = load3<T>(p.x, b, t, d);
            c = fmaf(f.on, c, (p.i.p ? logistic_pair(load3<T>(p.i, b, t, d)).on : f.off) * x);
        }
        for (uint32_t t = t1; t-- > t0;) {
            const Gate f = logistic_pair(load3<T>(p.f, b, t, d));
            const float x = load3<T>(p.x, b, t, d), dy = load3<T>(p.dy, b, t, d), prev = before[t - t0];
            float dc = carry;
            if (p.o.p) {
                const Gate o = logistic_pair(load3<T>(p.o, b, t, d));
                store3<T>(p.dout, b, t, d, dy * c * o.on * o.off);
                dc = fmaf(dy, o.on, dc);
            } else {
                dc += dy;
            }
            if (p.i.p) {
                const Gate i = logistic_pair(load3<T>(p.i, b, t, d));
                store3<T>(p.dx, b, t, d, dc * i.on);
                store3<T>(p.di, b, t, d, dc * x * i.on * i.off);
                store3<T>(p.df, b, t, d, dc * prev * f.on * f.off);
            } else {
                store3<T>(p.dx, b, t, d, dc * f.off);
                store3<T>(p.df, b, t, d, dc * (prev - x) * f.on * f.off);
            }
            carry = dc * f.on;
            c = prev;
        }
    }
    if (p.dinitial) p.dinitial[b * p.dinitial_b + d * p.dinitial_d] = carry;
}

}  // namespace srt
