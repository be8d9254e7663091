// The elementwise passes of a gated Dense layer, y = act(g) * u with g = x . Wg + bg and u = x . Wu + bu:
//   gate_forward_kernel    y from g and u, for products that do not run on the fused kernel
//   add_kernel             the sum of two products
//   gate_backward_kernel   dg = dy u act'(g), du = dy act(g), and their column sums (the bias gradients)
// Both are bound by HBM (2 reads and 1 write, 3 reads and 2 writes per element).
#pragma once
#include "element.cuh"
#include "ptx.cuh"

namespace srt {

struct View2 { const void* p; long long m, n; };        // element strides
struct View2W { void* p; long long m, n; };

struct GateForwardParams {
    View2 g, u;
    View2W y;
    uint32_t M, N, act;
};

template <typename T>
__global__ void __launch_bounds__(256)
gate_forward_kernel(const __grid_constant__ GateForwardParams p)
{
    const unsigned long long total = static_cast<unsigned long long>(p.M) * p.N;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t m = static_cast<uint32_t>(i / p.N), n = static_cast<uint32_t>(i % p.N);
        const float g = to_float<T>(static_cast<const T*>(p.g.p)[m * p.g.m + n * p.g.n]);
        const float u = to_float<T>(static_cast<const T*>(p.u.p)[m * p.u.m + n * p.u.n]);
        static_cast<T*>(p.y.p)[m * p.y.m + n * p.y.n] = from_float<T>(gate_activation<T>(p.act, g) * u);
    }
}

// y = g + u (which may be y): the sum of two products that could not share a launch
template <typename T>
__global__ void __launch_bounds__(256)
add_kernel(const __grid_constant__ GateForwardParams p)
{
    const unsigned long long total = static_cast<unsigned long long>(p.M) * p.N;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t m = static_cast<uint32_t>(i / p.N), n = static_cast<uint32_t>(i % p.N);
        const float g = to_float<T>(static_cast<const T*>(p.g.p)[m * p.g.m + n * p.g.n]);
        const float u = to_float<T>(static_cast<const T*>(p.u.p)[m * p.u.m + n * p.u.n]);
        static_cast<T*>(p.y.p)[m * p.y.m + n * p.y.n] = from_float<T>(g + u);
    }
}

struct GateBackwardParams {
    View2 dy, g, u;
    View2W dg, du;
    void* sum_g; long long sum_g_n;          // bias gradients, may be null
    void* sum_u; long long sum_u_n;
    uint32_t M, N, act;
};

// A CTA owns 8 VEC columns: a warp's lanes are 8 column groups by 4 rows, its 8 warps 32 rows.  With CLUSTER the CTAs of a cluster
// (grid y, 2 .. 8 of them) walk the same columns at interleaved groups of 32 rows; each leaves its column sums in its shared memory, and
// behind a barrier of the cluster the first CTA adds them in rank order: no scratch memory, no atomics.  Up to 32 rows are one CTA's,
// which needs no cluster.  The unrounded fp32 values are summed.
// Reading three and writing two values an element bounds it: 3999 x 8200 bf16 82 us (4.0 TB/s) from a cold cache, without the sums 64 us (5.2 TB/s).
// Gates of four values at a time and three CTAs an SM took a tenth off.  Sums sent with st.async instead saved another tenth; that is not
// done: launches with clusters of one CTA, which sent to itself, are among the suspects of an illegal access.
template <typename T, int VEC, bool CLUSTER>
__global__ void __launch_bounds__(256, 3)
gate_backward_kernel(const __grid_constant__ GateBackwardParams p)
{
    constexpr uint32_t kCols = 8 * VEC;
    __shared__ float sums[2][8][kCols];
    __shared__ float total[2][kCols];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t col = (blockIdx.x * 8 + (lane & 7)) * VEC;
    float sg[VEC], su[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) sg[j] = su[j] = 0.0f;
    if (col < p.N) {
        const uint32_t step = gridDim.y * 32;
        for (uint32_t r0 = blockIdx.y * 32 + warp * 4 + (lane >> 3); r0 < p.M; r0 += 2 * step) {
            __align__(16) T dy[2][VEC], g[2][VEC], u[2][VEC];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const long long r = static_cast<long long>(r0) + k * static_cast<long long>(step);
                if (r >= p.M) continue;
                const T* a = static_cast<const T*>(p.dy.p) + r * p.dy.m + col * p.dy.n;
                const T* b = static_cast<const T*>(p.g.p) + r * p.g.m + col * p.g.n;
                const T* c = static_cast<const T*>(p.u.p) + r * p.u.m + col * p.u.n;
                if constexpr (VEC > 1) {
                    *reinterpret_cast<uint4*>(dy[k]) = *reinterpret_cast<const uint4*>(a);
                    *reinterpret_cast<uint4*>(g[k]) = *reinterpret_cast<const uint4*>(b);
                    *reinterpret_cast<uint4*>(u[k]) = *reinterpret_cast<const uint4*>(c);
                } else {
                    dy[k][0] = *a; g[k][0] = *b; u[k][0] = *c;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const long long r = static_cast<long long>(r0) + k * static_cast<long long>(step);
                if (r >= p.M) continue;
                __align__(16) T dg[VEC], du[VEC];
                constexpr int kPart = VEC < 4 ? VEC : 4;                      // registers for four values at a time
#pragma unroll
                for (int i = 0; i < VEC; i += kPart) {
                    float z[kPart], value[kPart], slope[kPart];
#pragma unroll
                    for (int j = 0; j < kPart; ++j) z[j] = to_float<T>(g[k][i + j]);
                    gate_values<T, kPart>(p.act, z, value, slope);
#pragma unroll
                    for (int j = 0; j < kPart; ++j) {
                        const float d = to_float<T>(dy[k][i + j]);
                        const float vg = d * to_float<T>(u[k][i + j]) * slope[j], vu = d * value[j];
                        dg[i + j] = from_float<T>(vg);
                        du[i + j] = from_float<T>(vu);
                        sg[i + j] += vg;
                        su[i + j] += vu;
                    }
                }
                T* a = static_cast<T*>(p.dg.p) + r * p.dg.m + col * p.dg.n;
                T* b = static_cast<T*>(p.du.p) + r * p.du.m + col * p.du.n;
                if constexpr (VEC > 1) {
                    *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(dg);
                    *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(du);
                } else {
                    *a = dg[0]; *b = du[0];
                }
            }
        }
    }
    if (p.sum_g == nullptr && p.sum_u == nullptr) return;               // uniform over the grid
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        sg[j] += __shfl_xor_sync(0xffffffffu, sg[j], 8);
        su[j] += __shfl_xor_sync(0xffffffffu, su[j], 8);
        sg[j] += __shfl_xor_sync(0xffffffffu, sg[j], 16);
        su[j] += __shfl_xor_sync(0xffffffffu, su[j], 16);
        if (lane < 8) {
            sums[0][warp][lane * VEC + j] = sg[j];
            sums[1][warp][lane * VEC + j] = su[j];
        }
    }
    __syncthreads();
    const uint32_t which = threadIdx.x / kCols, c = threadIdx.x % kCols;
    float s = 0.0f;
    if (which < 2) {
        s = sums[which][0][c];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += sums[which][w][c];
    }
    uint32_t rank = 0;
    if constexpr (CLUSTER) {
        rank = cluster_ctarank();
        if (which < 2) total[which][c] = s;
        cluster_arrive_release();
        cluster_wait_acquire();
        if (rank == 0 && which < 2)
            for (uint32_t r = 1; r < gridDim.y; ++r) s += __uint_as_float(ld_shared_remote_u32(smem_u32(&total[which][c]), r));
    }
    const uint32_t n = blockIdx.x * kCols + c;
    if (rank == 0 && which < 2 && n < p.N) {
        if (which == 0 && p.sum_g) static_cast<T*>(p.sum_g)[n * p.sum_g_n] = from_float<T>(s);
        if (which == 1 && p.sum_u) static_cast<T*>(p.sum_u)[n * p.sum_u_n] = from_float<T>(s);
    }
    if constexpr (CLUSTER) {                                             // a CTA's sums are read until here
        cluster_arrive_release();
        cluster_wait_acquire();
    }
}

}  // namespace srt
