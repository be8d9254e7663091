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

// ------------------------------------------------------------------------------------------ long sequences
// A step is an affine map c -> f c + u, and maps compose: a span of steps is (A, H) with A the product of its f and H its
// result from c = 0.  A CTA takes 64 steps of 64 channels (32 with VEC = 1) at a time: 8 warps of 8 steps, a lane VEC
// neighbouring channels.  Every warp folds its steps into (A, H), the spans are joined in order of time through shared memory, and a second
// pass over the gates, which are still in registers, produces the values: one read and one write of everything.  Where
// batch items and channels alone leave SMs idle, the CTAs of a cluster take neighbouring spans of 64 steps and exchange
// their (A, H) through distributed shared memory, once per 64 x cluster steps.
constexpr uint32_t kSpanWarps = 8, kSpanSteps = 8;
static_assert(kSpanWarps * kSpanSteps == kRecurrenceChunk, "a CTA's span is what lies between two kept states");

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> load_pack(const Strided3& s, long long base, uint32_t t, bool live)
{
    Pack<T, VEC> v;
    if (live) {
        v = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(s.p) + base + t * s.t);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] = from_float<T>(0.0f);
    }
    return v;
}
template <typename T, int VEC> __device__ __forceinline__ void store_pack(const Strided3W& s, long long base, uint32_t t, const Pack<T, VEC>& v)
{
    *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(s.p) + base + t * s.t) = v;
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
__global__ void __launch_bounds__(256, 3)
recurrence_span_kernel(const __grid_constant__ RecurrenceParams p, uint32_t blocks_d, uint32_t cluster)
{
    __shared__ alignas(16) Span<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d = ((block % blocks_d) * 32 + lane) * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const long long bx = b * p.x.b + d * p.x.d, bf = b * p.f.b + d * p.f.d, bi = b * p.i.b + d * p.i.d, bo = b * p.o.b + d * p.o.d;
    const long long by = b * p.y.b + d * p.y.d;

    float state[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) state[j] = p.initial && on ? p.initial[b * p.initial_b + (d + j) * p.initial_d] : 0.0f;

    uint32_t buf = 0;
    for (uint32_t first = 0; first < chunks; first += cluster, buf ^= 1) {
        const uint32_t chunk = first + rank, t0 = chunk * kRecurrenceChunk + warp * kSpanSteps;
        Pack<T, VEC> rx[kSpanSteps], rf[kSpanSteps], ri[HAS_I ? kSpanSteps : 1], ro[HAS_O ? kSpanSteps : 1];
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            const bool live = on && t0 + s < n;
            rf[s] = load_pack<T, VEC>(p.f, bf, t0 + s, live);
            rx[s] = load_pack<T, VEC>(p.x, bx, t0 + s, live);
            if constexpr (HAS_I) ri[s] = load_pack<T, VEC>(p.i, bi, t0 + s, live);
            if constexpr (HAS_O) ro[s] = load_pack<T, VEC>(p.o, bo, t0 + s, live);
        }
        float f[kSpanSteps][VEC], u[kSpanSteps][VEC];
        Span<VEC> mine;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Gate g = logistic_pair(to_float<T>(rf[s].v[j]));
                const float in = HAS_I ? logistic_pair(to_float<T>(ri[HAS_I ? s : 0].v[j])).on : g.off;
                const bool live = t0 + s < n;
                f[s][j] = live ? g.on : 1.0f;                              // behind the sequence: the state stays
                u[s][j] = live ? in * to_float<T>(rx[s].v[j]) : 0.0f;
                mine.h[j] = fmaf(f[s][j], mine.h[j], u[s][j]);
                mine.a[j] *= f[s][j];
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
        for (int j = 0; j < VEC; ++j) c[j] = begin[j] = state[j];
        if (cluster > 1) {
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (r == rank) begin[j] = state[j];
                    state[j] = fmaf(s.a[j], state[j], s.h[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) c[j] = begin[j];
        }
#pragma unroll
        for (uint32_t w = 0; w < kSpanWarps; ++w) {
            if (cluster > 1 && w >= warp) break;
            const Span<VEC> s = in_cta[buf][w][lane];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (cluster == 1) state[j] = fmaf(s.a[j], state[j], s.h[j]);
                if (w < warp) c[j] = fmaf(s.a[j], c[j], s.h[j]);
            }
        }
        if (p.states && warp == 0 && on && chunk < chunks) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.states[b * p.states_b + chunk * p.states_c + (d + j) * p.states_d] = begin[j];
        }
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            Pack<T, VEC> y;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                c[j] = fmaf(f[s][j], c[j], u[s][j]);
                float v = c[j];
                if constexpr (HAS_O) v *= logistic_pair(to_float<T>(ro[s].v[j])).on;
                y.v[j] = from_float<T>(t0 + s < n ? v : 0.0f);
            }
            if (on && t0 + s < p.T) store_pack<T, VEC>(p.y, by, t0 + s, y);
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
__global__ void __launch_bounds__(256, 2)
recurrence_span_backward_kernel(const __grid_constant__ RecurrenceParams p, uint32_t blocks_d, uint32_t cluster)
{
    __shared__ SpanBoth<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d = ((block % blocks_d) * 32 + lane) * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const long long bx = b * p.x.b + d * p.x.d, bf = b * p.f.b + d * p.f.d, bi = b * p.i.b + d * p.i.d, bo = b * p.o.b + d * p.o.d;
    const long long by = b * p.dy.b + d * p.dy.d, gx = b * p.dx.b + d * p.dx.d, gf = b * p.df.b + d * p.df.d;
    const long long gi = b * p.di.b + d * p.di.d, go = b * p.dout.b + d * p.dout.d;

    float carry[VEC];                                       // f_{t+1} dc_{t+1} behind what is left
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = p.dlast && on ? p.dlast[b * p.dlast_b + (d + j) * p.dlast_d] : 0.0f;

    uint32_t buf = 0;
    for (uint32_t done = 0; done < chunks; done += cluster, buf ^= 1) {
        const bool mine_exists = done + rank < chunks;
        const uint32_t chunk = mine_exists ? chunks - 1 - done - rank : 0;
        const uint32_t t0 = chunk * kRecurrenceChunk + warp * kSpanSteps;
        const uint32_t end = mine_exists ? n : 0;           // no step of a chunk that is not there is live
        Pack<T, VEC> rx[kSpanSteps], rf[kSpanSteps], ri[HAS_I ? kSpanSteps : 1], ro[HAS_O ? kSpanSteps : 1], ry[kSpanSteps];
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            const bool live = on && t0 + s < end;
            rf[s] = load_pack<T, VEC>(p.f, bf, t0 + s, live);
            rx[s] = load_pack<T, VEC>(p.x, bx, t0 + s, live);
            ry[s] = load_pack<T, VEC>(p.dy, by, t0 + s, live);
            if constexpr (HAS_I) ri[s] = load_pack<T, VEC>(p.i, bi, t0 + s, live);
            if constexpr (HAS_O) ro[s] = load_pack<T, VEC>(p.o, bo, t0 + s, live);
        }
        float c[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            c[j] = mine_exists && on ? p.states[b * p.states_b + chunk * p.states_c + (d + j) * p.states_d] : 0.0f;

        float f[kSpanSteps][VEC], off[kSpanSteps][VEC], dp[kSpanSteps][VEC];
        SpanBoth<VEC> mine;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = mine.e[j] = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const Gate g = logistic_pair(to_float<T>(rf[s].v[j]));
                const bool live = t0 + s < end;
                f[s][j] = live ? g.on : 1.0f;
                off[s][j] = live ? g.off : 0.0f;
                const float in = HAS_I ? logistic_pair(to_float<T>(ri[HAS_I ? s : 0].v[j])).on : off[s][j];
                mine.h[j] = fmaf(f[s][j], mine.h[j], in * to_float<T>(rx[s].v[j]));       // x is 0 where nothing is live
                mine.a[j] *= f[s][j];
                dp[s][j] = to_float<T>(ry[s].v[j]);
                if constexpr (HAS_O) dp[s][j] *= logistic_pair(to_float<T>(ro[s].v[j])).on;
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
        float e[VEC], begin[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) begin[j] = carry[j];
        if (cluster > 1) {
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (r == rank) begin[j] = carry[j];
                    carry[j] = fmaf(s.a[j], carry[j], s.h[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = begin[j];
#pragma unroll
        for (int w = kSpanWarps - 1; w >= 0; --w) {
            const SpanBoth<VEC>& s = in_cta[buf][w][lane];
            const SpanBoth<VEC>& q = in_cta[buf][kSpanWarps - 1 - w][lane];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (cluster == 1) carry[j] = fmaf(s.a[j], carry[j], s.e[j]);
                if (w > static_cast<int>(warp)) e[j] = fmaf(s.a[j], e[j], s.e[j]);
                if (kSpanWarps - 1 - w < warp) c[j] = fmaf(q.a[j], c[j], q.h[j]);
            }
        }
        float before[kSpanSteps][VEC];
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                before[s][j] = c[j];
                const float in = HAS_I ? logistic_pair(to_float<T>(ri[HAS_I ? s : 0].v[j])).on : off[s][j];
                c[j] = fmaf(f[s][j], c[j], in * to_float<T>(rx[s].v[j]));
            }
#pragma unroll
        for (int s = kSpanSteps - 1; s >= 0; --s) {
            Pack<T, VEC> vx, vf, vi, vo;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float dc = dp[s][j] + e[j], x = to_float<T>(rx[s].v[j]);
                const bool live = t0 + s < end;
                float dx, df, di = 0.0f, dout = 0.0f;
                if constexpr (HAS_I) {
                    const Gate in = logistic_pair(to_float<T>(ri[s].v[j]));
                    dx = dc * in.on;
                    di = dc * x * in.on * in.off;
                    df = dc * before[s][j] * f[s][j] * off[s][j];
                } else {
                    dx = dc * off[s][j];
                    df = dc * (before[s][j] - x) * f[s][j] * off[s][j];
                }
                if constexpr (HAS_O) {
                    const Gate out = logistic_pair(to_float<T>(ro[s].v[j]));
                    dout = to_float<T>(ry[s].v[j]) * c[j] * out.on * out.off;
                }
                e[j] = live ? f[s][j] * dc : e[j];
                c[j] = before[s][j];
                vx.v[j] = from_float<T>(live ? dx : 0.0f);
                vf.v[j] = from_float<T>(live ? df : 0.0f);
                vi.v[j] = from_float<T>(live ? di : 0.0f);
                vo.v[j] = from_float<T>(live ? dout : 0.0f);
            }
            if (on && mine_exists && t0 + s < p.T) {
                store_pack<T, VEC>(p.dx, gx, t0 + s, vx);
                store_pack<T, VEC>(p.df, gf, t0 + s, vf);
                if constexpr (HAS_I) store_pack<T, VEC>(p.di, gi, t0 + s, vi);
                if constexpr (HAS_O) store_pack<T, VEC>(p.dout, go, t0 + s, vo);
            }
        }
    }
    if (p.dinitial && rank == 0 && warp == 0 && on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.dinitial[b * p.dinitial_b + (d + j) * p.dinitial_d] = carry[j];
    }
}

}  // namespace srt
