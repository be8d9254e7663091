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
#include <type_traits>

#include "element.cuh"
#include "ptx.cuh"

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

// s(a), and s(a) with 1 - s(a), each to a relative error of a few 2^-23.  The pair comes from e = exp(-|a|), so the small one
// of the two is not the difference of 1 and its neighbour (a gate at 0.9999 keeps its decay 1 - f to full precision).  The
// .ftz forms of the two approximations take one instruction each where the others rescale denormals around them: what is
// below 2^-126 counts as closed.
struct Gate { float on, off; };
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
__device__ __forceinline__ Gate logistic_pair(float a)
{
    const float e = exp2_ftz(-kLog2E * fabsf(a));
    const float big = reciprocal_ftz(1.0f + e), small = e * big;
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
            c = fmaf(f.on, c, (p.i.p ? logistic(load3<T>(p.i, b, t, d)) : f.off) * x);
            y = p.o.p ? c * logistic(load3<T>(p.o, b, t, d)) : c;
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
            c = fmaf(f.on, c, (p.i.p ? logistic(load3<T>(p.i, b, t, d)) : f.off) * x);
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

// ------------------------------------------------------------------------------------------ long sequences
// A step is an affine map c -> f c + u, and maps compose: a span of steps is (A, H) with A the product of its f and H its
// result from c = 0.  A CTA takes 64 steps of 64 channels (32 with VEC = 1) at a time: 8 warps of 8 steps, a lane VEC
// neighbouring channels.  Every warp folds its steps into (A, H), the spans are joined in order of time through shared memory, and a second
// pass over the gates, which are still in registers, produces the values: one read and one write of everything.  Where
// batch items and channels alone leave SMs idle, the CTAs of a cluster take neighbouring spans of 64 steps and exchange
// their (A, H) through distributed shared memory, once per 64 x cluster steps.
// While a span is computed, every thread's own elements of the next one are on their way into shared memory (cp.async, read back
// by the thread that asked for them, so no barrier is involved).
constexpr uint32_t kSpanWarps = 8, kSpanSteps = 8, kSpanThreads = 32 * kSpanWarps, kSpanStages = 2;
static_assert(kSpanWarps * kSpanSteps == kRecurrenceChunk, "a CTA's span is what lies between two kept states");

// VEC neighbouring elements as one word
template <typename T, int VEC> struct Lane;
template <> struct Lane<float, 1> {
    using Raw = uint32_t;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = __uint_as_float(r); }
    static __device__ __forceinline__ Raw pack(const float (&v)[1]) { return __float_as_uint(v[0]); }
    static __device__ __forceinline__ Raw infinity() { return 0x7f800000u; }
};
template <> struct Lane<float, 2> {
    using Raw = uint2;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2]) { v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) { return make_uint2(__float_as_uint(v[0]), __float_as_uint(v[1])); }
    static __device__ __forceinline__ Raw infinity() { return make_uint2(0x7f800000u, 0x7f800000u); }
};
template <typename T> struct Lane<T, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = to_float<T>(*reinterpret_cast<T*>(&r)); }
    static __device__ __forceinline__ Raw pack(const float (&v)[1])
    {
        T t = from_float<T>(v[0]);
        return *reinterpret_cast<Raw*>(&t);
    }
    static __device__ __forceinline__ Raw infinity() { return std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u; }
};
template <> struct Lane<__nv_bfloat16, 2> {
    using Raw = uint32_t;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2]) { v[0] = __uint_as_float(r << 16); v[1] = __uint_as_float(r & 0xffff0000u); }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) { return pack2<__nv_bfloat16>(v[0], v[1]); }
    static __device__ __forceinline__ Raw infinity() { return 0x7f807f80u; }
};
template <> struct Lane<__half, 2> {
    using Raw = uint32_t;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2])
    {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&r));
        v[0] = f.x; v[1] = f.y;
    }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) { return pack2<__half>(v[0], v[1]); }
    static __device__ __forceinline__ Raw infinity() { return 0x7c007c00u; }
};

// One tensor as a thread sees it: its elements of 8 consecutive steps, by way of a ring in shared memory where a word is one
// that cp.async can move (4 or 8 bytes), else straight into registers.
template <typename T, int VEC>
struct StepReader {
    using Raw = typename Lane<T, VEC>::Raw;
    static constexpr bool kAsync = sizeof(Raw) >= 4;
    const T* base;
    long long stride;
    uint32_t ring;                       // shared address of this thread's first word; words of a thread are 256 apart
    __device__ __forceinline__ StepReader(const Strided3& s, uint32_t b, uint32_t d, uint32_t ring_base, uint32_t which)
        : base(static_cast<const T*>(s.p) + b * s.b + d * s.d), stride(s.t),
          ring(ring_base + (which * kSpanSteps * kSpanThreads + threadIdx.x) * static_cast<uint32_t>(sizeof(Raw))) {}
    __device__ __forceinline__ void fetch(uint32_t t0, uint32_t live, uint32_t stage_bytes) const
    {
        if constexpr (kAsync) {
            const T* at = base + t0 * stride;
#pragma unroll
            for (uint32_t k = 0; k < kSpanSteps; ++k, at += stride)
                if (k < live)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;"
                                 ::"r"(ring + stage_bytes + k * kSpanThreads * static_cast<uint32_t>(sizeof(Raw))), "l"(at), "n"(sizeof(Raw)) : "memory");
        }
    }
    __device__ __forceinline__ void read(uint32_t t0, uint32_t live, uint32_t stage_bytes, Raw other, Raw (&v)[kSpanSteps]) const
    {
        const T* at = base + t0 * stride;
#pragma unroll
        for (uint32_t k = 0; k < kSpanSteps; ++k, at += stride) {
            v[k] = other;
            if constexpr (kAsync) {
                const uint32_t from = ring + stage_bytes + k * kSpanThreads * static_cast<uint32_t>(sizeof(Raw));
                if (k < live) {
                    if constexpr (sizeof(Raw) == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(*reinterpret_cast<uint32_t*>(&v[k])) : "r"(from) : "memory");
                    else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(reinterpret_cast<uint32_t*>(&v[k])[0]), "=r"(reinterpret_cast<uint32_t*>(&v[k])[1]) : "r"(from) : "memory");
                }
            } else {
                if (k < live) v[k] = *reinterpret_cast<const Raw*>(at);
            }
        }
    }
};
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int VEC> __host__ __device__ constexpr uint32_t span_smem_bytes(uint32_t tensors)
{
    return StepReader<T, VEC>::kAsync ? kSpanStages * tensors * kSpanSteps * kSpanThreads * static_cast<uint32_t>(sizeof(typename Lane<T, VEC>::Raw)) : 0;
}

// a float2 (VEC = 2) or float per lane and quantity, in shared memory of any CTA of the cluster
template <int VEC> struct Span { float a[VEC], h[VEC]; };

template <int VEC> __device__ __forceinline__ void span_to_cta(const Span<VEC>* local, uint32_t rank, const Span<VEC>& s)
{
    const uint32_t at = map_to_cta(smem_u32(local), rank);
    if constexpr (VEC == 2)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(s.a[0]), "f"(s.a[1]), "f"(s.h[0]), "f"(s.h[1]) : "memory");
    else
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(s.a[0]), "f"(s.h[0]) : "memory");
}

template <typename T, bool HAS_I, bool HAS_O, int VEC>
__global__ void __launch_bounds__(kSpanThreads, 3)
recurrence_span_kernel(const __grid_constant__ RecurrenceParams p, uint32_t blocks_d, uint32_t cluster)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    constexpr uint32_t kTensors = 2 + HAS_I + HAS_O, kStageBytes = span_smem_bytes<T, VEC>(kTensors) / kSpanStages;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ alignas(16) Span<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d = ((block % blocks_d) * 32 + lane) * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const StepReader<T, VEC> qf(p.f, b, d, smem_u32(ring), 0), qx(p.x, b, d, smem_u32(ring), 1), qi(p.i, b, d, smem_u32(ring), 2),
        qo(p.o, b, d, smem_u32(ring), 2 + HAS_I);
    // this thread's first step of chunk k, and how many of its 8 belong to the sequence
    auto first_step = [&](uint32_t k) { return (k + rank) * kRecurrenceChunk + warp * kSpanSteps; };
    auto live_from = [&](uint32_t t0) { return on && t0 < n ? n - t0 : 0u; };
    auto fetch = [&](uint32_t k, uint32_t stage_bytes) {
        const uint32_t t0 = first_step(k), live = live_from(t0);
        qf.fetch(t0, live, stage_bytes);
        qx.fetch(t0, live, stage_bytes);
        if constexpr (HAS_I) qi.fetch(t0, live, stage_bytes);
        if constexpr (HAS_O) qo.fetch(t0, live, stage_bytes);
        fetch_commit();
    };

    float state[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) state[j] = p.initial && on ? p.initial[b * p.initial_b + (d + j) * p.initial_d] : 0.0f;

    uint32_t buf = 0;
    if (chunks > 0) fetch(0, 0);
    for (uint32_t first = 0; first < chunks; first += cluster, buf ^= 1) {
        const uint32_t chunk = first + rank, t0 = first_step(first), live = live_from(t0);
        fetch(first + cluster, (buf ^ 1) * kStageBytes);                  // behind the last chunk nothing is live
        fetch_wait<1>();
        // behind the sequence a forget logit of infinity and an update of zero leave the state as it is
        float f[kSpanSteps][VEC], u[kSpanSteps][VEC];
        Span<VEC> mine;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = 0.0f;
        {
            Raw rf[kSpanSteps], rx[kSpanSteps], ri[kSpanSteps];
            qf.read(t0, live, buf * kStageBytes, L::infinity(), rf);
            qx.read(t0, live, buf * kStageBytes, Raw{}, rx);
            if constexpr (HAS_I) qi.read(t0, live, buf * kStageBytes, Raw{}, ri);
#pragma unroll
            for (uint32_t s = 0; s < kSpanSteps; ++s) {
                float vf[VEC], vx[VEC], vi[VEC];
                L::unpack(rf[s], vf);
                L::unpack(rx[s], vx);
                if constexpr (HAS_I) L::unpack(ri[s], vi);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const Gate g = logistic_pair(vf[j]);
                    float in = g.off;
                    if constexpr (HAS_I) in = logistic(vi[j]);
                    f[s][j] = g.on;
                    u[s][j] = in * vx[j];
                    mine.h[j] = fmaf(f[s][j], mine.h[j], u[s][j]);
                    mine.a[j] *= f[s][j];
                }
            }
        }
        in_cta[buf][warp][lane] = mine;
        __syncthreads();
        if (cluster > 1) {
            if (warp == 0) {
                Span<VEC> all = mine;
#pragma unroll
                for (uint32_t w = 1; w < kSpanWarps; ++w) {
                    const Span<VEC> next = in_cta[buf][w][lane];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        all.h[j] = fmaf(next.a[j], all.h[j], next.h[j]);
                        all.a[j] *= next.a[j];
                    }
                }
                for (uint32_t r = 0; r < cluster; ++r) span_to_cta<VEC>(&in_cluster[buf][rank][lane], r, all);
            }
            cluster_arrive_release();
            cluster_wait_acquire();
        }
        // the state before this CTA's span, before this warp's steps, and behind the whole cluster's span
        float c[VEC], begin[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) begin[j] = state[j];
        if (cluster > 1) {
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (r == rank) begin[j] = state[j];
                    state[j] = fmaf(s.a[j], state[j], s.h[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = begin[j];
        for (uint32_t w = 0; w < warp; ++w) {
            const Span<VEC> s = in_cta[buf][w][lane];
#pragma unroll
            for (int j = 0; j < VEC; ++j) c[j] = fmaf(s.a[j], c[j], s.h[j]);
        }
        if (cluster == 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) state[j] = c[j];
            for (uint32_t w = warp; w < kSpanWarps; ++w) {
                const Span<VEC> s = in_cta[buf][w][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) state[j] = fmaf(s.a[j], state[j], s.h[j]);
            }
        }
        if (p.states && warp == 0 && on && chunk < chunks) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.states[b * p.states_b + chunk * p.states_c + (d + j) * p.states_d] = begin[j];
        }
        Raw ro[kSpanSteps];
        if constexpr (HAS_O) qo.read(t0, live, buf * kStageBytes, Raw{}, ro);
        T* at = static_cast<T*>(p.y.p) + b * p.y.b + d * p.y.d + t0 * p.y.t;
        const uint32_t there = on && t0 < p.T ? p.T - t0 : 0;
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s, at += p.y.t) {
            float v[VEC], vo[VEC];
            if constexpr (HAS_O) L::unpack(ro[s], vo);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                c[j] = fmaf(f[s][j], c[j], u[s][j]);
                v[j] = c[j];
                if constexpr (HAS_O) v[j] *= logistic(vo[j]);
            }
            Raw y = L::pack(v);
            if (s >= live) y = Raw{};
            if (s < there) *reinterpret_cast<Raw*>(at) = y;
        }
    }
    if (p.last && rank == 0 && warp == 0 && on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.last[b * p.last_b + (d + j) * p.last_d] = state[j];
    }
}

// Backward: the chunks from the last to the first.  Within a chunk the states come from the kept one as above; the gradient of
// the state runs the other way, e -> f (p + e) per step, with the same product A and E the span's result from e = 0.
template <int VEC> struct SpanBoth { float a[VEC], h[VEC], e[VEC]; };

template <typename T, bool HAS_I, bool HAS_O, int VEC>
__global__ void __launch_bounds__(kSpanThreads, 2)
recurrence_span_backward_kernel(const __grid_constant__ RecurrenceParams p, uint32_t blocks_d, uint32_t cluster)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    constexpr uint32_t kTensors = 3 + HAS_I + HAS_O, kStageBytes = span_smem_bytes<T, VEC>(kTensors) / kSpanStages;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ SpanBoth<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d = ((block % blocks_d) * 32 + lane) * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const StepReader<T, VEC> qf(p.f, b, d, smem_u32(ring), 0), qx(p.x, b, d, smem_u32(ring), 1), qy(p.dy, b, d, smem_u32(ring), 2),
        qi(p.i, b, d, smem_u32(ring), 3), qo(p.o, b, d, smem_u32(ring), 3 + HAS_I);
    // after `done` chunks from the end this CTA has chunk chunks - 1 - done - rank, if that is one
    auto first_step = [&](uint32_t done) { return done + rank < chunks ? (chunks - 1 - done - rank) * kRecurrenceChunk + warp * kSpanSteps : p.T; };
    auto live_from = [&](uint32_t t0) { return on && t0 < n ? n - t0 : 0u; };
    float c[VEC], c_next[VEC];                              // the kept state of the chunk, fetched one chunk ahead
    auto fetch = [&](uint32_t done, uint32_t stage_bytes) {
        const uint32_t t0 = first_step(done), live = live_from(t0);
        qf.fetch(t0, live, stage_bytes);
        qx.fetch(t0, live, stage_bytes);
        qy.fetch(t0, live, stage_bytes);
        if constexpr (HAS_I) qi.fetch(t0, live, stage_bytes);
        if constexpr (HAS_O) qo.fetch(t0, live, stage_bytes);
        fetch_commit();
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            c_next[j] = done + rank < chunks && on ? p.states[b * p.states_b + (chunks - 1 - done - rank) * p.states_c + (d + j) * p.states_d] : 0.0f;
    };

    float carry[VEC];                                       // f_{t+1} dc_{t+1} behind what is left
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = p.dlast && on ? p.dlast[b * p.dlast_b + (d + j) * p.dlast_d] : 0.0f;

    uint32_t buf = 0;
    if (chunks > 0) fetch(0, 0);
    for (uint32_t done = 0; done < chunks; done += cluster, buf ^= 1) {
        const uint32_t t0 = first_step(done), live = live_from(t0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = c_next[j];
        fetch(done + cluster, (buf ^ 1) * kStageBytes);
        fetch_wait<1>();
        Raw rf[kSpanSteps], rx[kSpanSteps], ri[kSpanSteps], ro[kSpanSteps], ry[kSpanSteps];
        qf.read(t0, live, buf * kStageBytes, L::infinity(), rf);          // 1 - f = 0 where nothing is live
        qx.read(t0, live, buf * kStageBytes, Raw{}, rx);
        qy.read(t0, live, buf * kStageBytes, Raw{}, ry);
        if constexpr (HAS_I) qi.read(t0, live, buf * kStageBytes, Raw{}, ri);
        if constexpr (HAS_O) qo.read(t0, live, buf * kStageBytes, Raw{}, ro);
        float f[kSpanSteps][VEC], off[kSpanSteps][VEC], dp[kSpanSteps][VEC];
        SpanBoth<VEC> mine;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = mine.e[j] = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            float vf[VEC], vx[VEC], vi[VEC], vo[VEC];
            L::unpack(rf[s], vf);
            L::unpack(rx[s], vx);
            L::unpack(ry[s], dp[s]);
            if constexpr (HAS_I) L::unpack(ri[s], vi);
            if constexpr (HAS_O) L::unpack(ro[s], vo);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Gate g = logistic_pair(vf[j]);
                f[s][j] = g.on;
                off[s][j] = g.off;
                float in = g.off;
                if constexpr (HAS_I) in = logistic(vi[j]);
                mine.h[j] = fmaf(f[s][j], mine.h[j], in * vx[j]);
                mine.a[j] *= f[s][j];
                if constexpr (HAS_O) dp[s][j] *= logistic(vo[j]);
            }
        }
#pragma unroll
        for (int s = kSpanSteps - 1; s >= 0; --s)
#pragma unroll
            for (int j = 0; j < VEC; ++j) mine.e[j] = f[s][j] * (dp[s][j] + mine.e[j]);
        in_cta[buf][warp][lane] = mine;
        __syncthreads();
        if (cluster > 1) {
            if (warp == 0) {
                Span<VEC> all;
#pragma unroll
                for (int j = 0; j < VEC; ++j) all.a[j] = 1.0f, all.h[j] = 0.0f;
#pragma unroll
                for (int w = kSpanWarps - 1; w >= 0; --w) {
                    const SpanBoth<VEC>& s = in_cta[buf][w][lane];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        all.h[j] = fmaf(s.a[j], all.h[j], s.e[j]);
                        all.a[j] *= s.a[j];
                    }
                }
                for (uint32_t r = 0; r < cluster; ++r) span_to_cta<VEC>(&in_cluster[buf][rank][lane], r, all);
            }
            cluster_arrive_release();
            cluster_wait_acquire();
        }
        float e[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = carry[j];
        if (cluster > 1) {
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (r == rank) e[j] = carry[j];
                    carry[j] = fmaf(s.a[j], carry[j], s.h[j]);
                }
            }
        }
        for (uint32_t w = kSpanWarps - 1; w > warp; --w) {
            const SpanBoth<VEC>& s = in_cta[buf][w][lane];
#pragma unroll
            for (int j = 0; j < VEC; ++j) e[j] = fmaf(s.a[j], e[j], s.e[j]);
        }
        if (cluster == 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) carry[j] = e[j];
            for (int w = warp; w >= 0; --w) {
                const SpanBoth<VEC>& s = in_cta[buf][w][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) carry[j] = fmaf(s.a[j], carry[j], s.e[j]);
            }
        }
        for (uint32_t w = 0; w < warp; ++w) {
            const SpanBoth<VEC>& s = in_cta[buf][w][lane];
#pragma unroll
            for (int j = 0; j < VEC; ++j) c[j] = fmaf(s.a[j], c[j], s.h[j]);
        }
        float before[kSpanSteps][VEC];
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            float vx[VEC], vi[VEC];
            L::unpack(rx[s], vx);
            if constexpr (HAS_I) L::unpack(ri[s], vi);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                before[s][j] = c[j];
                float in = off[s][j];
                if constexpr (HAS_I) in = logistic(vi[j]);
                c[j] = fmaf(f[s][j], c[j], in * vx[j]);
            }
        }
        const uint32_t there = on && t0 < p.T ? p.T - t0 : 0;
        const long long top = t0 + kSpanSteps - 1;
        T* ax = static_cast<T*>(p.dx.p) + b * p.dx.b + d * p.dx.d + top * p.dx.t;
        T* af = static_cast<T*>(p.df.p) + b * p.df.b + d * p.df.d + top * p.df.t;
        T* ai = static_cast<T*>(p.di.p) + b * p.di.b + d * p.di.d + top * p.di.t;
        T* ao = static_cast<T*>(p.dout.p) + b * p.dout.b + d * p.dout.d + top * p.dout.t;
#pragma unroll
        for (int s = kSpanSteps - 1; s >= 0; --s, ax -= p.dx.t, af -= p.df.t, ai -= p.di.t, ao -= p.dout.t) {
            float vx[VEC], vi[VEC], vo[VEC], vy[VEC], dx[VEC], df[VEC], di[VEC], dout[VEC];
            L::unpack(rx[s], vx);
            if constexpr (HAS_I) L::unpack(ri[s], vi);
            if constexpr (HAS_O) {
                L::unpack(ro[s], vo);
                L::unpack(ry[s], vy);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float dc = dp[s][j] + e[j];
                const float slope = dc * (f[s][j] * off[s][j]);
                if constexpr (HAS_I) {
                    const Gate in = logistic_pair(vi[j]);
                    dx[j] = dc * in.on;
                    di[j] = dx[j] * vx[j] * in.off;
                    df[j] = slope * before[s][j];
                } else {
                    dx[j] = dc * off[s][j];
                    df[j] = slope * (before[s][j] - vx[j]);
                }
                if constexpr (HAS_O) {
                    const Gate out = logistic_pair(vo[j]);
                    dout[j] = vy[j] * c[j] * out.on * out.off;
                }
                e[j] = f[s][j] * dc;
                c[j] = before[s][j];
            }
            Raw wx = L::pack(dx), wf = L::pack(df), wi{}, wo{};
            if constexpr (HAS_I) wi = L::pack(di);
            if constexpr (HAS_O) wo = L::pack(dout);
            if (static_cast<uint32_t>(s) >= live) wx = wf = wi = wo = Raw{};
            if (static_cast<uint32_t>(s) < there) {
                *reinterpret_cast<Raw*>(ax) = wx;
                *reinterpret_cast<Raw*>(af) = wf;
                if constexpr (HAS_I) *reinterpret_cast<Raw*>(ai) = wi;
                if constexpr (HAS_O) *reinterpret_cast<Raw*>(ao) = wo;
            }
        }
    }
    if (p.dinitial && rank == 0 && warp == 0 && on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.dinitial[b * p.dinitial_b + (d + j) * p.dinitial_d] = carry[j];
    }
}

}  // namespace srt
