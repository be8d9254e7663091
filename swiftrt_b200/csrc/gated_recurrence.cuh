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
#include <cuda.h>

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
    uint32_t* status;                    // the device's status word, and the limit of a wait in SM cycles (TMA loads only)
    unsigned long long wait_cycles;
};

// Two neighbouring channels at a time where VEC is 2 (one instruction for both products or sums)
template <int VEC> __device__ __forceinline__ void mul_to(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC])
{
    if constexpr (VEC == 2) {
        asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
    } else {
        d[0] = a[0] * b[0];
    }
}
template <int VEC> __device__ __forceinline__ void add_to(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC])
{
    if constexpr (VEC == 2) {
        asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
    } else {
        d[0] = a[0] + b[0];
    }
}
template <int VEC> __device__ __forceinline__ void fma_to(float (&d)[VEC], const float (&a)[VEC], const float (&b)[VEC], const float (&c)[VEC])
{
    if constexpr (VEC == 2) {
        asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\t"
            "mov.b64 {%0, %1}, x;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(c[0]), "f"(c[1]));
    } else {
        d[0] = fmaf(a[0], b[0], c[0]);
    }
}
template <int VEC> __device__ __forceinline__ void logistic_to(float (&on)[VEC], const float (&a)[VEC])
{
    float e[VEC], k[VEC], one[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) k[j] = -kLog2E, one[j] = 1.0f;
    mul_to<VEC>(e, a, k);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = exp2_ftz(e[j]);
    add_to<VEC>(e, e, one);
#pragma unroll
    for (int j = 0; j < VEC; ++j) on[j] = reciprocal_ftz(e[j]);
}
template <int VEC> __device__ __forceinline__ void logistic_pair_to(float (&on)[VEC], float (&off)[VEC], const float (&a)[VEC])
{
    float e[VEC], k[VEC], one[VEC], sum[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) k[j] = -kLog2E, one[j] = 1.0f;
    mul_to<VEC>(e, a, k);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = exp2_ftz(min_or_nan(e[j], 126.0f));
    add_to<VEC>(sum, e, one);
#pragma unroll
    for (int j = 0; j < VEC; ++j) on[j] = reciprocal_ftz(sum[j]);
    mul_to<VEC>(off, e, on);
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

// Up to this many steps one thread walks a channel of one batch item, step after step: a launch is all that such a call costs (16 tokens of
// 2048 channels 5.3 us a call, most of it on the host).
constexpr uint32_t kFewSteps = 8;
static_assert(kFewSteps <= kRecurrenceChunk, "the state before the first step is the only one kept");

template <typename T>
__global__ void __launch_bounds__(128)
recurrence_steps_kernel(const __grid_constant__ RecurrenceParams p)
{
    const unsigned long long id = blockIdx.x * 128ull + threadIdx.x;
    if (id >= static_cast<unsigned long long>(p.B) * p.D) return;
    const uint32_t b = static_cast<uint32_t>(id / p.D), d = static_cast<uint32_t>(id % p.D);
    const uint32_t n = live_steps(p, b);
    float c = p.initial ? p.initial[b * p.initial_b + d * p.initial_d] : 0.0f;
    if (p.states && p.T > 0) p.states[b * p.states_b + d * p.states_d] = c;
    for (uint32_t t = 0; t < p.T; ++t) {
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

// The same for the backward pass: the states are recomputed from the kept one, then the steps are walked from the last.
template <typename T>
__global__ void __launch_bounds__(128)
recurrence_steps_backward_kernel(const __grid_constant__ RecurrenceParams p)
{
    const unsigned long long id = blockIdx.x * 128ull + threadIdx.x;
    if (id >= static_cast<unsigned long long>(p.B) * p.D) return;
    const uint32_t b = static_cast<uint32_t>(id / p.D), d = static_cast<uint32_t>(id % p.D);
    const uint32_t n = min(live_steps(p, b), kFewSteps);
    float carry = p.dlast ? p.dlast[b * p.dlast_b + d * p.dlast_d] : 0.0f;         // f_{t+1} dc_{t+1}
    for (uint32_t t = p.T; t-- > n;) {
        store3<T>(p.dx, b, t, d, 0.0f);
        store3<T>(p.df, b, t, d, 0.0f);
        if (p.i.p) store3<T>(p.di, b, t, d, 0.0f);
        if (p.o.p) store3<T>(p.dout, b, t, d, 0.0f);
    }
    float before[kFewSteps];
    float c = n > 0 ? p.states[b * p.states_b + d * p.states_d] : 0.0f;
    for (uint32_t t = 0; t < n; ++t) {
        before[t] = c;
        const Gate f = logistic_pair(load3<T>(p.f, b, t, d));
        const float x = load3<T>(p.x, b, t, d);
        c = fmaf(f.on, c, (p.i.p ? logistic(load3<T>(p.i, b, t, d)) : f.off) * x);
    }
    for (uint32_t t = n; t-- > 0;) {
        const Gate f = logistic_pair(load3<T>(p.f, b, t, d));
        const float x = load3<T>(p.x, b, t, d), dy = load3<T>(p.dy, b, t, d), prev = before[t];
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
    if (p.dinitial) p.dinitial[b * p.dinitial_b + d * p.dinitial_d] = carry;
}

// ------------------------------------------------------------------------------------------ long sequences
// A step is an affine map c -> f c + u, and maps compose: a span of steps is (A, H) with A the product of its f and H its
// result from c = 0.  A CTA takes 64 steps of 32 VEC channels at a time: 8 warps of 8 steps, a lane VEC neighbouring
// channels.  Every warp folds its steps into (A, H), the spans are joined in order of time through shared memory, and a second
// pass over the gates, which are still in registers, produces the values: one read and one write of everything.  Where
// batch items and channels alone leave SMs idle, the CTAs of a cluster take neighbouring spans of 64 steps and exchange
// their (A, H) through distributed shared memory, once per 64 x cluster steps.
//
// How the elements travel (SRC):
//   kFromTiles   TMA: one thread asks for a [64 steps x 128 bytes] box of every tensor, two spans ahead, and every warp stores its
//                [8 x 128 bytes] of the results the same way: no addresses, bounds or predicates per element.  Needs 16-byte aligned rows.
//   kFromWords   cp.async of 4 bytes (a Float32, two 16-bit elements), by the thread that will use them (no barrier), one span ahead.
//   kFromMemory  plain loads: 16-bit elements at odd offsets.
//
// HBM is the bound of what has to move (4 to 9 values an element), the kernels come within 0.74 (forward) and 0.67 (backward) of a
// copy's rate: 8 x 2048 x 4096 bf16 with an output gate 111 us (4.9 TB/s) and 216 us (4.4 TB/s).  Two to three CTAs of eight warps an SM leave
// the scheduler without a ready warp half of the time; the unit for exponentials is 55 % busy, issue slots 50 %.  One reciprocal shared by several gates
// (the product of their denominators) took 7 of that unit's instructions instead of 12 and 17 % more time: the multiplications it costs
// lie on the same chains.  A single sequence (8191 x 4096) 74 us; 1530 fp16 channels with all gates, whose rows start on 4 bytes and go
// through the second path, 33 / 70 us at 5 x 777 steps, 1536 in tiles 25 / 44 us.
constexpr uint32_t kSpanWarps = 8, kSpanSteps = 8, kSpanThreads = 32 * kSpanWarps, kSpanStages = 2;
static_assert(kSpanWarps * kSpanSteps == kRecurrenceChunk, "a CTA's span is what lies between two kept states");
enum : int { kFromMemory = 0, kFromWords = 1, kFromTiles = 2 };

// tensor maps of a kFromTiles launch: forget, update, input, output, outGrad; results
struct RecurrenceMaps { CUtensorMap f, x, i, o, dy, y, dx, df, di, dout; };
struct NoMaps { uint32_t unused; };
template <int SRC> struct MapsOf { using type = NoMaps; };
template <> struct MapsOf<kFromTiles> { using type = RecurrenceMaps; };

// VEC neighbouring elements as one word
template <typename T, int VEC> struct Lane;
template <> struct Lane<float, 1> {
    using Raw = uint32_t;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = __uint_as_float(r); }
    static __device__ __forceinline__ Raw pack(const float (&v)[1]) { return __float_as_uint(v[0]); }
    static __device__ __forceinline__ Raw infinity() { return 0x7f800000u; }
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

template <typename Raw> __device__ __forceinline__ Raw shared_word(uint32_t at)
{
    Raw r;
    if constexpr (sizeof(Raw) == 2) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(at) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
    return r;
}
template <typename Raw> __device__ __forceinline__ void store_shared_word(uint32_t at, Raw r)
{
    if constexpr (sizeof(Raw) == 2) asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(r) : "memory");
    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(r) : "memory");
}

template <typename T, int VEC> struct SpanTile {
    using Raw = typename Lane<T, VEC>::Raw;
    static constexpr uint32_t kRow = 32 * static_cast<uint32_t>(sizeof(Raw)), kBytes = kRecurrenceChunk * kRow;      // one tensor's span in shared memory
    static constexpr uint32_t kWarpBytes = kSpanSteps * kRow;
};

// One tensor as a thread sees it: its elements of 8 consecutive steps.
template <typename T, int VEC, int SRC>
struct StepReader {
    using Raw = typename Lane<T, VEC>::Raw;
    using Tile = SpanTile<T, VEC>;
    const T* base;
    long long stride;
    uint32_t at;                         // shared address of this thread's element of its first step, stage 0
    __device__ __forceinline__ StepReader(const Strided3& s, uint32_t b, uint32_t d, uint32_t ring, uint32_t which)
        : base(static_cast<const T*>(s.p) + b * s.b + d * s.d), stride(s.t),
          at(ring + which * Tile::kBytes + (threadIdx.x >> 5) * Tile::kWarpBytes + (threadIdx.x & 31) * static_cast<uint32_t>(sizeof(Raw))) {}
    __device__ __forceinline__ void fetch(uint32_t t0, uint32_t live, uint32_t stage_bytes) const
    {
        const T* from = base + t0 * stride;
#pragma unroll
        for (uint32_t k = 0; k < kSpanSteps; ++k, from += stride)
            if (k < live) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at + stage_bytes + k * Tile::kRow), "l"(from), "n"(sizeof(Raw)) : "memory");
    }
    // step k again, from the stage (behind the sequence: whatever is there)
    __device__ __forceinline__ Raw again(uint32_t k, uint32_t stage_bytes, const Raw (&kept)[kSpanSteps]) const
    {
        if constexpr (SRC == kFromMemory) return kept[k];
        else return shared_word<Raw>(at + stage_bytes + k * Tile::kRow);
    }
    // steps at or behind `live` read as `other`; whole: none of them is (uniform over the warp)
    __device__ __forceinline__ void read(uint32_t t0, uint32_t live, bool whole, uint32_t stage_bytes, Raw other, Raw (&v)[kSpanSteps]) const
    {
        if constexpr (SRC == kFromMemory) {
            const T* from = base + t0 * stride;
#pragma unroll
            for (uint32_t k = 0; k < kSpanSteps; ++k, from += stride) v[k] = k < live ? *reinterpret_cast<const Raw*>(from) : other;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < kSpanSteps; ++k) v[k] = shared_word<Raw>(at + stage_bytes + k * Tile::kRow);
            if (!whole) {
#pragma unroll
                for (uint32_t k = 0; k < kSpanSteps; ++k)
                    if (k >= live) v[k] = other;
            }
        }
    }
};
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int VEC, int SRC> __host__ __device__ constexpr uint32_t span_stage_bytes(uint32_t tensors)
{
    return SRC == kFromMemory ? 0 : tensors * SpanTile<T, VEC>::kBytes;
}
template <typename T, int VEC, int SRC> __host__ __device__ constexpr uint32_t span_smem_bytes(uint32_t tensors, uint32_t results)
{
    return kSpanStages * span_stage_bytes<T, VEC, SRC>(tensors) + (SRC == kFromTiles ? results * SpanTile<T, VEC>::kBytes + 128 : 0);
}

// Where a warp's results of 8 steps go.
template <typename T, int VEC, bool TILE>
struct StepWriter {
    using Raw = typename Lane<T, VEC>::Raw;
    using Tile = SpanTile<T, VEC>;
    T* to;
    long long stride;
    uint32_t at;
    __device__ __forceinline__ StepWriter(const Strided3W& s, uint32_t b, uint32_t d, uint32_t t0, uint32_t staging, uint32_t which)
        : to(static_cast<T*>(s.p) + b * s.b + d * s.d + t0 * s.t), stride(s.t),
          at(staging + which * Tile::kBytes + (threadIdx.x >> 5) * Tile::kWarpBytes + (threadIdx.x & 31) * static_cast<uint32_t>(sizeof(Raw))) {}
    // `there`: how many of the 8 steps exist
    __device__ __forceinline__ void put(uint32_t k, uint32_t there, Raw v) const
    {
        if constexpr (TILE) store_shared_word<Raw>(at + k * Tile::kRow, v);
        else if (k < there) *reinterpret_cast<Raw*>(to + k * stride) = v;
    }
};

// zeros in up to 8 steps from t0
template <typename T, int VEC> __device__ __forceinline__ void write_zeros(const Strided3W& s, uint32_t b, uint32_t d, uint32_t t0, uint32_t there)
{
    using Raw = typename Lane<T, VEC>::Raw;
    T* to = static_cast<T*>(s.p) + b * s.b + d * s.d + t0 * s.t;
#pragma unroll
    for (uint32_t k = 0; k < kSpanSteps; ++k)
        if (k < there) *reinterpret_cast<Raw*>(to + k * s.t) = Raw{};
}

// a float2 (VEC = 2) or float per lane and quantity, in shared memory of any CTA of the cluster
template <int VEC> struct Span { float a[VEC], h[VEC]; };

// `s` to the same place in the shared memory of CTA `rank`, counted there on its barrier: no fence and no barrier of the whole
// cluster, which would wait for the results' stores as well
template <int VEC> __device__ __forceinline__ void span_to_cta(const Span<VEC>* local, uint32_t bar, uint32_t rank, const Span<VEC>& s)
{
    const uint32_t at = map_to_cta(smem_u32(local), rank), done = map_to_cta(bar, rank);
    if constexpr (VEC == 2)
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                     ::"r"(at), "r"(__float_as_uint(s.a[0])), "r"(__float_as_uint(s.a[1])), "r"(__float_as_uint(s.h[0])), "r"(__float_as_uint(s.h[1])), "r"(done) : "memory");
    else
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                     ::"r"(at), "r"(__float_as_uint(s.a[0])), "r"(__float_as_uint(s.h[0])), "r"(done) : "memory");
}

// Bounded waits on a pair of barriers: for the tiles of a stage, or for the spans of the cluster's CTAs.  A wait that runs over the limit is noted in the status word (the result of the launch is
// invalid then); the thread still waits, up to kDrainLimitCycles longer, for what is on its way before it goes on.
constexpr uint64_t kDrainLimitCycles = 4000000000ull;
struct PhaseWaits {
    uint32_t bars;                       // two mbarriers
    uint32_t* status;
    uint64_t limit;
    uint32_t phases = 0;                 // bit s: parity of the next wait on barrier s
    bool dead = false;
    __device__ __forceinline__ void wait(uint32_t stage)
    {
        const uint32_t parity = (phases >> stage) & 1;
        phases ^= 1u << stage;
        if (dead || mbar_test_wait(bars + 8 * stage, parity)) return;
        const uint64_t t0 = sm_clock();
        while (!mbar_try_wait(bars + 8 * stage, parity) && !dead) dead = sm_clock() - t0 > limit + kDrainLimitCycles;
        if (sm_clock() - t0 > limit) atomicOr(status, 1u);
    }
};

template <typename T, bool HAS_I, bool HAS_O, int VEC, int SRC>
__global__ void __launch_bounds__(kSpanThreads, 3)
recurrence_span_kernel(const __grid_constant__ RecurrenceParams p, const __grid_constant__ typename MapsOf<SRC>::type maps, uint32_t blocks_d, uint32_t cluster)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    using Tile = SpanTile<T, VEC>;
    constexpr uint32_t kTensors = 2 + HAS_I + HAS_O, kStageBytes = span_stage_bytes<T, VEC, SRC>(kTensors);
    extern __shared__ __align__(128) uint8_t dynamic_smem[];
    __shared__ alignas(16) Span<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    __shared__ alignas(8) uint64_t full[kSpanStages], arrived[2];
    const uint32_t ring = SRC == kFromTiles ? (smem_u32(dynamic_smem) + 127u) & ~127u : smem_u32(dynamic_smem);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d0 = (block % blocks_d) * 32 * VEC, d = d0 + lane * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const StepReader<T, VEC, SRC> qf(p.f, b, d, ring, 0), qx(p.x, b, d, ring, 1), qi(p.i, b, d, ring, 2), qo(p.o, b, d, ring, 2 + HAS_I);
    PhaseWaits waits{smem_u32(full), p.status, p.wait_cycles}, arrivals{smem_u32(arrived), p.status, p.wait_cycles};
    // this thread's first step of chunk k, and how many of its 8 belong to the sequence
    auto first_step = [&](uint32_t k) { return (k + rank) * kRecurrenceChunk + warp * kSpanSteps; };
    auto live_from = [&](uint32_t t0) { return t0 < n ? n - t0 : 0u; };
    auto fetch = [&](uint32_t k, uint32_t stage) {
        if constexpr (SRC == kFromTiles) {
            const uint32_t t = (k + rank) * kRecurrenceChunk;
            if (threadIdx.x == 0 && t < n) {                    // (t < n <= T keeps k below chunks)
                const uint32_t bar = smem_u32(&full[stage]), to = ring + stage * kStageBytes;
                mbar_arrive_expect_tx(bar, kStageBytes);
                tma_load_3d(to, &maps.f, bar, d0, t, b);
                tma_load_3d(to + Tile::kBytes, &maps.x, bar, d0, t, b);
                if constexpr (HAS_I) tma_load_3d(to + 2 * Tile::kBytes, &maps.i, bar, d0, t, b);
                if constexpr (HAS_O) tma_load_3d(to + (2 + HAS_I) * Tile::kBytes, &maps.o, bar, d0, t, b);
            }
        } else if constexpr (SRC == kFromWords) {
            const uint32_t t0 = first_step(k), live = on ? live_from(t0) : 0;
            qf.fetch(t0, live, stage * kStageBytes);
            qx.fetch(t0, live, stage * kStageBytes);
            if constexpr (HAS_I) qi.fetch(t0, live, stage * kStageBytes);
            if constexpr (HAS_O) qo.fetch(t0, live, stage * kStageBytes);
            fetch_commit();
        }
    };
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&arrived[i]), 1);
        }
        fence_mbar_init();
    }
    if (cluster > 1) {
        cluster_arrive_release();                                 // before anyone sends to a barrier
        cluster_wait_acquire();
    } else {
        __syncthreads();
    }
    fetch(0, 0);
    if constexpr (SRC == kFromTiles) fetch(cluster, 1);

    float state[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) state[j] = p.initial && on ? p.initial[b * p.initial_b + (d + j) * p.initial_d] : 0.0f;

    uint32_t buf = 0, first = 0;
    for (; first * kRecurrenceChunk < n; first += cluster, buf ^= 1) {
        const uint32_t chunk = first + rank, t0 = first_step(first), live = live_from(t0);
        const bool whole = live >= kSpanSteps;
        if constexpr (SRC == kFromWords) {
            fetch(first + cluster, buf ^ 1);                      // behind the last chunk nothing is live
            fetch_wait<1>();
        }
        if constexpr (SRC == kFromTiles) {
            if (chunk * kRecurrenceChunk < n) waits.wait(buf);
        }
        // behind the sequence a forget logit of infinity and an update of zero leave the state as it is
        float f[kSpanSteps][VEC], u[kSpanSteps][VEC];
        Span<VEC> mine;
        Raw ro[kSpanSteps];
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = 0.0f;
        {
            Raw rf[kSpanSteps], rx[kSpanSteps], ri[kSpanSteps];
            const uint32_t mem_live = SRC == kFromMemory && !on ? 0 : live;
            qf.read(t0, mem_live, whole, buf * kStageBytes, L::infinity(), rf);
            qx.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, rx);
            if constexpr (HAS_I) qi.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, ri);
            if constexpr (HAS_O) qo.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, ro);
#pragma unroll
            for (uint32_t s = 0; s < kSpanSteps; ++s) {
                float vf[VEC], vx[VEC], in[VEC];
                L::unpack(rf[s], vf);
                L::unpack(rx[s], vx);
                logistic_pair_to<VEC>(f[s], in, vf);
                if constexpr (HAS_I) {
                    float vi[VEC];
                    L::unpack(ri[s], vi);
                    logistic_to<VEC>(in, vi);
                }
                mul_to<VEC>(u[s], in, vx);
                fma_to<VEC>(mine.h, f[s], mine.h, u[s]);
                mul_to<VEC>(mine.a, mine.a, f[s]);
            }
        }
        in_cta[buf][warp][lane] = mine;
        __syncthreads();
        if constexpr (SRC == kFromTiles) fetch(first + 2 * cluster, buf);         // everyone has read this stage
        // this CTA's spans in order: `whole_span` all of them, `ahead` those before this warp's
        Span<VEC> whole_span, ahead;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            whole_span.a[j] = ahead.a[j] = 1.0f;
            whole_span.h[j] = ahead.h[j] = 0.0f;
        }
#pragma unroll
        for (uint32_t w = 0; w < kSpanWarps; ++w) {
            const Span<VEC> s = in_cta[buf][w][lane];
            if (w == warp) ahead = whole_span;
            fma_to<VEC>(whole_span.h, s.a, whole_span.h, s.h);
            mul_to<VEC>(whole_span.a, whole_span.a, s.a);
        }
        // the state before this CTA's span, before this warp's steps, and behind the whole cluster's span
        float c[VEC], begin[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) begin[j] = state[j];
        if (cluster > 1) {
            if (warp == 0) {
                if (lane == 0) mbar_arrive_expect_tx(smem_u32(&arrived[buf]), cluster * 32 * static_cast<uint32_t>(sizeof(Span<VEC>)));
                for (uint32_t r = 0; r < cluster; ++r) span_to_cta<VEC>(&in_cluster[buf][rank][lane], smem_u32(&arrived[buf]), r, whole_span);
            }
            arrivals.wait(buf);
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (r == rank) begin[j] = state[j];
                fma_to<VEC>(state, s.a, state, s.h);
            }
        } else {
            fma_to<VEC>(state, whole_span.a, state, whole_span.h);
        }
        fma_to<VEC>(c, ahead.a, begin, ahead.h);
        if (p.states && warp == 0 && on && chunk < chunks) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.states[b * p.states_b + chunk * p.states_c + (d + j) * p.states_d] = begin[j];
        }
        const uint32_t there = on && t0 < p.T ? p.T - t0 : 0;
        const StepWriter<T, VEC, SRC == kFromTiles> out(p.y, b, d, t0, ring + kSpanStages * kStageBytes, 0);
        if constexpr (SRC == kFromTiles) {
            if (lane == 0) bulk_wait_group_read<0>();             // the last span's results have left the staging rows
            __syncwarp();
        }
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            float v[VEC];
            fma_to<VEC>(c, f[s], c, u[s]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = c[j];
            if constexpr (HAS_O) {
                float vo[VEC];
                L::unpack(ro[s], vo);
                logistic_to<VEC>(vo, vo);
                mul_to<VEC>(v, v, vo);
            }
            Raw y = L::pack(v);
            if (!whole && s >= live) y = Raw{};
            out.put(s, there, y);
        }
        if constexpr (SRC == kFromTiles) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && t0 < p.T) {                          // steps and channels that do not exist are not written
                tma_store_3d(&maps.y, ring + kSpanStages * kStageBytes + warp * Tile::kWarpBytes, d0, t0, b);
                bulk_commit_group();
            }
        }
    }
    for (; first + rank < chunks; first += cluster) {             // nothing but padding
        const uint32_t t0 = first_step(first);
        if (on && t0 < p.T) write_zeros<T, VEC>(p.y, b, d, t0, p.T - t0);
        if (p.states && warp == 0 && on) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.states[b * p.states_b + (first + rank) * p.states_c + (d + j) * p.states_d] = state[j];
        }
    }
    if constexpr (SRC == kFromTiles) {
        if (lane == 0) bulk_wait_group<0>();
    }
    if (cluster > 1 && p.last && p.last == p.initial) {                   // a state advanced in place: the other CTAs have read it
        cluster_arrive_release();
        cluster_wait_acquire();
    }
    if (p.last && rank == 0 && warp == 0 && on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.last[b * p.last_b + (d + j) * p.last_d] = state[j];
    }
}

// Backward: the chunks from the last to the first.  Within a chunk the states come from the kept one as above; the gradient of
// the state runs the other way, e -> f (p + e) per step, with the same product A and E the span's result from e = 0.
template <int VEC> struct SpanBoth { float a[VEC], h[VEC], e[VEC]; };

template <typename T, bool HAS_I, bool HAS_O, int VEC, int SRC>
__global__ void __launch_bounds__(kSpanThreads, 2)
recurrence_span_backward_kernel(const __grid_constant__ RecurrenceParams p, const __grid_constant__ typename MapsOf<SRC>::type maps, uint32_t blocks_d, uint32_t cluster)
{
    using L = Lane<T, VEC>;
    using Raw = typename L::Raw;
    using Tile = SpanTile<T, VEC>;
    constexpr uint32_t kTensors = 3 + HAS_I + HAS_O, kStageBytes = span_stage_bytes<T, VEC, SRC>(kTensors);
    constexpr bool kTileStores = SRC == kFromTiles;
    extern __shared__ __align__(128) uint8_t dynamic_smem[];
    __shared__ SpanBoth<VEC> in_cta[2][kSpanWarps][32];
    __shared__ alignas(16) Span<VEC> in_cluster[2][8][32];
    __shared__ alignas(8) uint64_t full[kSpanStages], arrived[2];
    const uint32_t ring = SRC == kFromTiles ? (smem_u32(dynamic_smem) + 127u) & ~127u : smem_u32(dynamic_smem);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster > 1 ? cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / cluster;
    const uint32_t b = block / blocks_d, d0 = (block % blocks_d) * 32 * VEC, d = d0 + lane * VEC;
    const bool on = d < p.D;
    const uint32_t n = live_steps(p, b);
    const uint32_t chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const StepReader<T, VEC, SRC> qf(p.f, b, d, ring, 0), qx(p.x, b, d, ring, 1), qy(p.dy, b, d, ring, 2), qi(p.i, b, d, ring, 3), qo(p.o, b, d, ring, 3 + HAS_I);
    PhaseWaits waits{smem_u32(full), p.status, p.wait_cycles}, arrivals{smem_u32(arrived), p.status, p.wait_cycles};
    // after `done` chunks from the end this CTA has chunk chunks - 1 - done - rank, if that is one
    auto chunk_start = [&](uint32_t done) { return done + rank < chunks ? (chunks - 1 - done - rank) * kRecurrenceChunk : p.T; };
    auto live_from = [&](uint32_t t0) { return t0 < n ? n - t0 : 0u; };
    float c[VEC], c_next[VEC];                              // the kept state of the chunk, fetched one chunk ahead
    auto fetch_state = [&](uint32_t done) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            c_next[j] = done + rank < chunks && on ? p.states[b * p.states_b + (chunks - 1 - done - rank) * p.states_c + (d + j) * p.states_d] : 0.0f;
    };
    auto fetch = [&](uint32_t done, uint32_t stage) {
        if constexpr (SRC == kFromTiles) {
            const uint32_t t = chunk_start(done);
            if (threadIdx.x == 0 && t < n) {
                const uint32_t bar = smem_u32(&full[stage]), to = ring + stage * kStageBytes;
                mbar_arrive_expect_tx(bar, kStageBytes);
                tma_load_3d(to, &maps.f, bar, d0, t, b);
                tma_load_3d(to + Tile::kBytes, &maps.x, bar, d0, t, b);
                tma_load_3d(to + 2 * Tile::kBytes, &maps.dy, bar, d0, t, b);
                if constexpr (HAS_I) tma_load_3d(to + 3 * Tile::kBytes, &maps.i, bar, d0, t, b);
                if constexpr (HAS_O) tma_load_3d(to + (3 + HAS_I) * Tile::kBytes, &maps.o, bar, d0, t, b);
            }
        } else if constexpr (SRC == kFromWords) {
            const uint32_t t0 = chunk_start(done) + warp * kSpanSteps, live = on ? live_from(t0) : 0;
            qf.fetch(t0, live, stage * kStageBytes);
            qx.fetch(t0, live, stage * kStageBytes);
            qy.fetch(t0, live, stage * kStageBytes);
            if constexpr (HAS_I) qi.fetch(t0, live, stage * kStageBytes);
            if constexpr (HAS_O) qo.fetch(t0, live, stage * kStageBytes);
            fetch_commit();
        }
    };
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&arrived[i]), 1);
        }
        fence_mbar_init();
    }
    if (cluster > 1) {
        cluster_arrive_release();                                 // before anyone sends to a barrier
        cluster_wait_acquire();
    } else {
        __syncthreads();
    }
    // the groups of spans behind the sequence
    const uint32_t live_chunks = (n + kRecurrenceChunk - 1) / kRecurrenceChunk, dead = (chunks - live_chunks) / cluster * cluster;
    fetch(dead, 0);
    if constexpr (SRC == kFromTiles) fetch(dead + cluster, 1);
    fetch_state(dead);
    if (on) {
        for (uint32_t done = 0; done < dead; done += cluster) {
            const uint32_t t0 = chunk_start(done) + warp * kSpanSteps;
            if (t0 >= p.T) continue;
            write_zeros<T, VEC>(p.dx, b, d, t0, p.T - t0);
            write_zeros<T, VEC>(p.df, b, d, t0, p.T - t0);
            if constexpr (HAS_I) write_zeros<T, VEC>(p.di, b, d, t0, p.T - t0);
            if constexpr (HAS_O) write_zeros<T, VEC>(p.dout, b, d, t0, p.T - t0);
        }
    }

    float carry[VEC];                                       // f_{t+1} dc_{t+1} behind what is left
#pragma unroll
    for (int j = 0; j < VEC; ++j) carry[j] = p.dlast && on ? p.dlast[b * p.dlast_b + (d + j) * p.dlast_d] : 0.0f;

    uint32_t buf = 0;
    for (uint32_t done = dead; done < chunks; done += cluster, buf ^= 1) {
        const uint32_t start = chunk_start(done), t0 = start + warp * kSpanSteps, live = live_from(t0);
        const bool whole = live >= kSpanSteps;
        const uint32_t stage = buf * kStageBytes;
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = c_next[j];
        fetch_state(done + cluster);
        if constexpr (SRC == kFromWords) {
            fetch(done + cluster, buf ^ 1);
            fetch_wait<1>();
        }
        if constexpr (SRC == kFromTiles) {
            if (start < n) waits.wait(buf);
        }
        Raw rf[kSpanSteps], rx[kSpanSteps], ri[kSpanSteps], ro[kSpanSteps], ry[kSpanSteps];
        const uint32_t mem_live = SRC == kFromMemory && !on ? 0 : live;
        qf.read(t0, mem_live, whole, buf * kStageBytes, L::infinity(), rf);       // 1 - f = 0 where nothing is live
        qx.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, rx);
        qy.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, ry);
        if constexpr (HAS_I) qi.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, ri);
        if constexpr (HAS_O) qo.read(t0, mem_live, whole, buf * kStageBytes, Raw{}, ro);
        float f[kSpanSteps][VEC], off[kSpanSteps][VEC], dp[kSpanSteps][VEC];
        SpanBoth<VEC> mine;
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine.a[j] = 1.0f, mine.h[j] = mine.e[j] = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            float vf[VEC], vx[VEC], in[VEC];
            L::unpack(rf[s], vf);
            L::unpack(rx[s], vx);
            L::unpack(ry[s], dp[s]);
            logistic_pair_to<VEC>(f[s], off[s], vf);
            if constexpr (HAS_I) {
                float vi[VEC];
                L::unpack(ri[s], vi);
                logistic_to<VEC>(in, vi);
                mul_to<VEC>(in, in, vx);
            } else {
                mul_to<VEC>(in, off[s], vx);
            }
            fma_to<VEC>(mine.h, f[s], mine.h, in);
            mul_to<VEC>(mine.a, mine.a, f[s]);
            if constexpr (HAS_O) {
                float vo[VEC];
                L::unpack(ro[s], vo);
                logistic_to<VEC>(vo, vo);
                mul_to<VEC>(dp[s], dp[s], vo);
            }
        }
#pragma unroll
        for (int s = kSpanSteps - 1; s >= 0; --s) {
            add_to<VEC>(mine.e, dp[s], mine.e);
            mul_to<VEC>(mine.e, f[s], mine.e);
        }
        in_cta[buf][warp][lane] = mine;
        if constexpr (kTileStores) {
            if (lane == 0) bulk_wait_group_read<0>();             // the results of the last span have left the other stage
        }
        __syncthreads();
        // everyone is done with the other stage: this one is read again below, so that its elements need no registers meanwhile
        if constexpr (SRC == kFromTiles) {
            if (done > dead) fetch(done + cluster, buf ^ 1);
        }
        // this CTA's spans from the end: `whole_span` all of them, `behind` those after this warp's; and the state before this warp's
        Span<VEC> whole_span, behind;
        float e[VEC], fore[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            whole_span.a[j] = behind.a[j] = 1.0f;
            whole_span.h[j] = behind.h[j] = 0.0f;
            fore[j] = c[j];
        }
#pragma unroll
        for (uint32_t k = 0; k < kSpanWarps; ++k) {
            const uint32_t w = kSpanWarps - 1 - k;
            const SpanBoth<VEC>& back = in_cta[buf][w][lane];
            const SpanBoth<VEC>& forth = in_cta[buf][k][lane];
            if (w == warp) behind = whole_span;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (k == warp) c[j] = fore[j];
            fma_to<VEC>(whole_span.h, back.a, whole_span.h, back.e);
            mul_to<VEC>(whole_span.a, whole_span.a, back.a);
            if (k + 1 < kSpanWarps) fma_to<VEC>(fore, forth.a, fore, forth.h);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = carry[j];
        if (cluster > 1) {
            if (warp == 0) {
                if (lane == 0) mbar_arrive_expect_tx(smem_u32(&arrived[buf]), cluster * 32 * static_cast<uint32_t>(sizeof(Span<VEC>)));
                for (uint32_t r = 0; r < cluster; ++r) span_to_cta<VEC>(&in_cluster[buf][rank][lane], smem_u32(&arrived[buf]), r, whole_span);
            }
            arrivals.wait(buf);
            for (uint32_t r = 0; r < cluster; ++r) {
                const Span<VEC> s = in_cluster[buf][r][lane];
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (r == rank) e[j] = carry[j];
                fma_to<VEC>(carry, s.a, carry, s.h);
            }
        } else {
            fma_to<VEC>(carry, whole_span.a, carry, whole_span.h);
        }
        fma_to<VEC>(e, behind.a, e, behind.h);
        const uint32_t there = on && t0 < p.T ? p.T - t0 : 0;
        // with tiles every gradient takes its operand's place in the stage, which this thread alone reads and for the last time before
        const uint32_t tiles = ring + stage;
        const StepWriter<T, VEC, kTileStores> out_f(p.df, b, d, t0, tiles, 0), out_x(p.dx, b, d, t0, tiles, 1), out_i(p.di, b, d, t0, tiles, 3),
            out_o(p.dout, b, d, t0, tiles, 3 + HAS_I);
        // the states, and the output gate's gradient, which needs nothing else: its operands make room for the states
        float before[kSpanSteps][VEC];
#pragma unroll
        for (uint32_t s = 0; s < kSpanSteps; ++s) {
            float vx[VEC], in[VEC];
            const bool dead = !whole && s >= live;
            Raw wx = qx.again(s, stage, rx);
            if (dead) wx = Raw{};
            L::unpack(wx, vx);
            if constexpr (HAS_I) {
                float vi[VEC];
                Raw wi = qi.again(s, stage, ri);
                if (dead) wi = Raw{};
                L::unpack(wi, vi);
                logistic_to<VEC>(in, vi);
                mul_to<VEC>(in, in, vx);
            } else {
                mul_to<VEC>(in, off[s], vx);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) before[s][j] = c[j];
            fma_to<VEC>(c, f[s], c, in);
            if constexpr (HAS_O) {
                float vo[VEC], dout[VEC], closed[VEC];
                L::unpack(qo.again(s, stage, ro), vo);
                L::unpack(qy.again(s, stage, ry), dout);
                logistic_pair_to<VEC>(vo, closed, vo);
                mul_to<VEC>(dout, dout, c);
                mul_to<VEC>(dout, dout, vo);
                mul_to<VEC>(dout, dout, closed);
                Raw wo = L::pack(dout);
                if (dead) wo = Raw{};
                out_o.put(s, there, wo);
            }
        }
#pragma unroll
        for (int s = kSpanSteps - 1; s >= 0; --s) {
            float vx[VEC], dx[VEC], df[VEC], di[VEC], dc[VEC], slope[VEC];
            const bool dead = !whole && static_cast<uint32_t>(s) >= live;
            L::unpack(qx.again(s, stage, rx), vx);
            add_to<VEC>(dc, dp[s], e);
            mul_to<VEC>(slope, f[s], off[s]);
            mul_to<VEC>(slope, slope, dc);
            if constexpr (HAS_I) {
                float vi[VEC], in[VEC], closed[VEC];
                L::unpack(qi.again(s, stage, ri), vi);
                logistic_pair_to<VEC>(in, closed, vi);
                mul_to<VEC>(dx, dc, in);
                mul_to<VEC>(di, dx, vx);
                mul_to<VEC>(di, di, closed);
                mul_to<VEC>(df, slope, before[s]);
            } else {
                mul_to<VEC>(dx, dc, off[s]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) df[j] = before[s][j] - vx[j];
                mul_to<VEC>(df, df, slope);
            }
            mul_to<VEC>(e, f[s], dc);
            Raw wx = L::pack(dx), wf = L::pack(df), wi{};
            if constexpr (HAS_I) wi = L::pack(di);
            if (dead) wx = wf = wi = Raw{};
            out_x.put(s, there, wx);
            out_f.put(s, there, wf);
            if constexpr (HAS_I) out_i.put(s, there, wi);
        }
        if constexpr (kTileStores) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && t0 < p.T) {
                const uint32_t from = tiles + warp * Tile::kWarpBytes;
                tma_store_3d(&maps.df, from, d0, t0, b);
                tma_store_3d(&maps.dx, from + Tile::kBytes, d0, t0, b);
                if constexpr (HAS_I) tma_store_3d(&maps.di, from + 3 * Tile::kBytes, d0, t0, b);
                if constexpr (HAS_O) tma_store_3d(&maps.dout, from + (3 + HAS_I) * Tile::kBytes, d0, t0, b);
                bulk_commit_group();
            }
        }
    }
    if constexpr (kTileStores) {
        if (lane == 0) bulk_wait_group<0>();
    }
    if (p.dinitial && rank == 0 && warp == 0 && on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.dinitial[b * p.dinitial_b + (d + j) * p.dinitial_d] = carry[j];
    }
}

}  // namespace srt
