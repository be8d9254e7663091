// Products of a few rows with a wide weight: y = act(x . W + b), or act(x . W0 + b0) * (x . W1 + b1), for M = 1 .. some tens of
// rows.  Every weight is read once and used M times, so the reading of the weights bounds it; the kernel streams them
// straight from global memory into the registers of warp-wide MMAs (m16n8k16, fp32 accumulators): the weight is the MMA's
// 16-row operand (16 columns of W), eight rows of x its 8-column operand, and within a k-step k may be permuted freely as
// long as both operands agree, so each weight format is loaded 16 bytes at a time in whatever order it is stored:
//
//   Int4   word (j, n) of the packed weight: rows 8 j .. 8 j + 7 of column n.  Lane (g, t) of a warp takes 4 columns (16 bytes)
//          of word row t: 32 columns x 32 rows per load.  Two nibbles at a time become the 16-bit floats 128 + q (bf16) or
//          1024 + q (fp16) by one AND-OR; subtracting 128 + z (1024 + z) is exact, so the MMA multiplies the integers
//          q - z and the group's scale is applied to its fp32 sum, once per group: no weight is ever rounded.
//   Rows   16-bit elements, columns contiguous ([K x N] as Dense keeps it): lane (g, t) takes 8 columns of rows 4 t .. 4 t + 3;
//          neighbouring rows are paired by byte permutes.
//   Cols   16-bit elements, K contiguous: lane (g, t) takes 8 k of columns g, g + 8, g + 16, g + 24, pairs as they are.
//
// A CTA's warps are warps_n column tiles by the other warps as parts of K, a cluster splits K further; the fp32 partial sums
// are added in the order of the parts (shared memory, then distributed shared memory): one launch, no workspace, and the same bits every time.
// Whole batches run without a bounds check: lanes beyond the last column or row read the last one's and their sums are dropped.
#pragma once
#include <type_traits>

#include "element.cuh"
#include "ptx.cuh"

namespace srt {

struct FewRowsWeight {
    const void* w; long long ld;                  // Int4: int32 words, ld words between word rows; Rows / Cols: ld elements between rows / columns
    const void* scales; long long scales_ld;
    const uint8_t* zeros; long long zeros_ld;     // may be null: 8
    uint32_t vec;                                 // 16-byte loads are aligned
    const void* bias; long long bias_n;           // may be null
    void* keep; long long keep_m, keep_n;         // receives x . W + b; may be null
};

struct FewRowsParams {
    FewRowsWeight w[2];
    const void* x; long long x_m, x_k;
    uint32_t x_vec;                               // rows of x are 16-byte aligned and contiguous
    void* out; long long o_m, o_n;
    uint32_t M, N, K, group, act;
    uint32_t warps_n, k_per_warp;                 // column tiles per CTA; rows of W per warp (a multiple of the batch)
};

constexpr uint32_t kFewRowsMaxWarps = 8;

template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// `count` (4 or 8) consecutive 16-bit elements as words, from address at + i * stride while i < live; zeros behind that
template <uint32_t COUNT>
__device__ __forceinline__ void gather_words(const void* at, long long stride, uint32_t live, uint32_t (&w)[COUNT / 2])
{
    const unsigned short* bits = static_cast<const unsigned short*>(at);
#pragma unroll
    for (uint32_t i = 0; i < COUNT / 2; ++i) w[i] = 0;
#pragma unroll
    for (uint32_t i = 0; i < COUNT; ++i)
        if (i < live) w[i >> 1] |= static_cast<uint32_t>(__ldg(bits + static_cast<long long>(i) * stride)) << (16 * (i & 1));
}

// Weight words pass through once: they are not kept in L1.
__device__ __forceinline__ uint4 load_stream(const void* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// One lane's view of x: its rows of the NT row tiles.
template <typename T, int NT>
struct FewRowsX {
    const T* row[NT];
    long long x_k;
    uint32_t live[NT];                            // 0: no such row
    uint32_t K;
    __device__ __forceinline__ FewRowsX(const FewRowsParams& p, uint32_t m0, uint32_t g) : x_k(p.x_k), K(p.K)
    {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint32_t m = m0 + 8 * j + g;
            live[j] = m < p.M;
            row[j] = static_cast<const T*>(p.x) + static_cast<long long>(min(m, p.M - 1)) * p.x_m;
        }
    }
    // COUNT (4 or 8) elements from column k on; FULL: they exist and are aligned
    template <uint32_t COUNT, bool FULL> __device__ __forceinline__ void load(uint32_t j, uint32_t k, uint32_t (&w)[COUNT / 2]) const
    {
        if constexpr (FULL) {
            if constexpr (COUNT == 8) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(row[j] + k));
                w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            } else {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(row[j] + k));
                w[0] = v.x; w[1] = v.y;
            }
        } else {
            gather_words<COUNT>(row[j] + static_cast<long long>(k) * x_k, x_k, live[j] && k < K ? K - k : 0, w);
        }
    }
};

// ------------------------------------------------------------------------------------------ 4-bit weights
// GPB: scale groups in a batch of 128 rows (4, 2, or 1 for groups of 128 and more).
template <typename T, int GPB>
struct Int4Format {
    static constexpr uint32_t kCols = 32, kTiles = 2, kBatch = 128;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 4 * g + 2 * tile + half; }

    struct Batch {
        uint32_t word[4][4];
        uint2 scale[GPB];
        uint32_t zero[GPB];
    };
    // this lane's part of a weight
    struct Source {
        const uint32_t* words; long long step;         // word row t of the first batch, and 32 rows further
        const unsigned short* scales; const uint8_t* zeros;
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t t)
        {
            const uint32_t n = n0 + 4 * g < p.N ? n0 + 4 * g : 0;
            words = static_cast<const uint32_t*>(w.w) + static_cast<long long>(t) * w.ld + n;
            step = 4 * w.ld;
            scales = static_cast<const unsigned short*>(w.scales) + n;
            zeros = w.zeros ? w.zeros + n : nullptr;
        }
    };

    template <bool FULL>
    static __device__ __forceinline__ void load(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t n0, uint32_t k, uint32_t g, uint32_t t, Batch& b)
    {
        const uint32_t live = n0 + 4 * g < p.N ? p.N - n0 - 4 * g : 0;             // columns of this lane that exist (FULL: 4 or none)
        const uint32_t* at = src.words + static_cast<long long>(k >> 3) * w.ld;
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s, at += src.step) {
            if constexpr (FULL) {
                const uint4 v = load_stream(at);
                b.word[s][0] = v.x; b.word[s][1] = v.y; b.word[s][2] = v.z; b.word[s][3] = v.w;
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) b.word[s][j] = j < live && k + 32 * s + 8 * t < p.K ? __ldg(at + j) : 0u;
            }
        }
#pragma unroll
        for (uint32_t s = 0; s < GPB; ++s) {
            const uint32_t row = k + (128 / GPB) * s;
            const long long group = row / p.group;
            if constexpr (FULL) {
                b.scale[s] = __ldg(reinterpret_cast<const uint2*>(src.scales + group * w.scales_ld));
                b.zero[s] = src.zeros ? __ldg(reinterpret_cast<const uint32_t*>(src.zeros + group * w.zeros_ld)) : 0x08080808u;
            } else {
                const uint32_t there = row < p.K ? live : 0;
                uint32_t bits[2];
                gather_words<4>(src.scales + group * w.scales_ld, 1, there, bits);
                b.scale[s] = make_uint2(bits[0], bits[1]);
                b.zero[s] = 0x08080808u;
                if (src.zeros) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        if (j < there) b.zero[s] = (b.zero[s] & ~(255u << (8 * j))) | static_cast<uint32_t>(__ldg(src.zeros + group * w.zeros_ld + j)) << (8 * j);
                }
            }
        }
    }

    // pair s of a word's nibbles, rows s and s + 4 of its eight, as the integers q - z in two 16-bit floats
    static __device__ __forceinline__ uint32_t integers(uint32_t word, uint32_t s, uint32_t magic_zero)
    {
        constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;
        uint32_t v = ((word >> (4 * s)) & 0x000f000fu) | kMagic;
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<const __half2*>(&magic_zero));
            return *reinterpret_cast<const uint32_t*>(&d);
        } else {
            const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&magic_zero));
            return *reinterpret_cast<const uint32_t*>(&d);
        }
    }

    template <int NT, bool FULL>
    static __device__ __forceinline__ void compute(const Batch& b, const FewRowsParams& p, const FewRowsX<T, NT>& x, uint32_t k, uint32_t t, float (&acc)[kTiles][NT][4])
    {
        constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x6400u : 0x4300u;
        constexpr uint32_t kStepsPerGroup = 4 / GPB;
#pragma unroll
        for (uint32_t grp = 0; grp < GPB; ++grp) {
            uint32_t mz[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) mz[j] = (kMagic | ((b.zero[grp] >> (8 * j)) & 15u)) * 0x10001u;
            float sum[kTiles][NT][4];
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                for (uint32_t j = 0; j < NT; ++j)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) sum[i][j][c] = 0.0f;
#pragma unroll
            for (uint32_t s = grp * kStepsPerGroup; s < (grp + 1) * kStepsPerGroup; ++s) {
                uint32_t xw[NT][4];
#pragma unroll
                for (uint32_t j = 0; j < NT; ++j) {
                    uint32_t v[4];
                    x.template load<8, FULL>(j, k + 32 * s + 8 * t, v);
                    xw[j][0] = __byte_perm(v[0], v[2], 0x5410);        // rows 0 and 4 of this lane's eight
                    xw[j][1] = __byte_perm(v[0], v[2], 0x7632);        // 1 and 5
                    xw[j][2] = __byte_perm(v[1], v[3], 0x5410);        // 2 and 6
                    xw[j][3] = __byte_perm(v[1], v[3], 0x7632);        // 3 and 7
                }
#pragma unroll
                for (uint32_t i = 0; i < kTiles; ++i) {
                    uint32_t a[2][4];
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) a[h][q] = integers(b.word[s][2 * i + h], q, mz[2 * i + h]);
#pragma unroll
                    for (uint32_t j = 0; j < NT; ++j) {
                        mma_16x8x16<T>(sum[i][j], a[0][0], a[1][0], a[0][1], a[1][1], xw[j][0], xw[j][1]);
                        mma_16x8x16<T>(sum[i][j], a[0][2], a[1][2], a[0][3], a[1][3], xw[j][2], xw[j][3]);
                    }
                }
            }
            const uint32_t sb[2] = {b.scale[grp].x, b.scale[grp].y};
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                const T* pair = reinterpret_cast<const T*>(&sb[i]);
                const float s0 = to_float<T>(pair[0]), s1 = to_float<T>(pair[1]);
#pragma unroll
                for (uint32_t j = 0; j < NT; ++j) {
                    acc[i][j][0] = fmaf(s0, sum[i][j][0], acc[i][j][0]);
                    acc[i][j][1] = fmaf(s0, sum[i][j][1], acc[i][j][1]);
                    acc[i][j][2] = fmaf(s1, sum[i][j][2], acc[i][j][2]);
                    acc[i][j][3] = fmaf(s1, sum[i][j][3], acc[i][j][3]);
                }
            }
        }
    }
};

// ------------------------------------------------------------------------------------------ 16-bit weights
template <typename T>
struct RowsFormat {
    static constexpr uint32_t kCols = 64, kTiles = 4, kBatch = 16;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 8 * g + 2 * tile + half; }
    struct Batch { uint32_t word[4][4]; };             // rows 4 t + r: 8 columns
    struct Source {
        const T* at;
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t t)
            : at(static_cast<const T*>(w.w) + static_cast<long long>(4 * t) * w.ld + (n0 + 8 * g < p.N ? n0 + 8 * g : 0)) {}
    };
    template <bool FULL>
    static __device__ __forceinline__ void load(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t n0, uint32_t k, uint32_t g, uint32_t t, Batch& b)
    {
        const T* at = src.at + static_cast<long long>(k) * w.ld;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r, at += w.ld) {
            if constexpr (FULL) {
                const uint4 v = load_stream(at);
                b.word[r][0] = v.x; b.word[r][1] = v.y; b.word[r][2] = v.z; b.word[r][3] = v.w;
            } else {
                gather_words<8>(at, 1, k + 4 * t + r < p.K && n0 + 8 * g < p.N ? p.N - n0 - 8 * g : 0, b.word[r]);
            }
        }
    }
    template <int NT, bool FULL>
    static __device__ __forceinline__ void compute(const Batch& b, const FewRowsParams&, const FewRowsX<T, NT>& x, uint32_t k, uint32_t t, float (&acc)[kTiles][NT][4])
    {
        uint32_t xw[NT][2];
#pragma unroll
        for (uint32_t j = 0; j < NT; ++j) x.template load<4, FULL>(j, k + 4 * t, xw[j]);
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
            const uint32_t a0 = __byte_perm(b.word[0][i], b.word[1][i], 0x5410), a1 = __byte_perm(b.word[0][i], b.word[1][i], 0x7632);
            const uint32_t a2 = __byte_perm(b.word[2][i], b.word[3][i], 0x5410), a3 = __byte_perm(b.word[2][i], b.word[3][i], 0x7632);
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) mma_16x8x16<T>(acc[i][j], a0, a1, a2, a3, xw[j][0], xw[j][1]);
        }
    }
};

template <typename T>
struct ColsFormat {
    static constexpr uint32_t kCols = 32, kTiles = 2, kBatch = 32;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 16 * tile + 8 * half + g; }
    struct Batch { uint32_t word[4][4]; };             // column g + 8 c: 8 k
    struct Source {
        const T* at[4];
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t t)
        {
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c)
                at[c] = static_cast<const T*>(w.w) + static_cast<long long>(min(n0 + 8 * c + g, p.N - 1)) * w.ld + 8 * t;
        }
    };
    template <bool FULL>
    static __device__ __forceinline__ void load(const FewRowsParams& p, const FewRowsWeight&, const Source& src, uint32_t n0, uint32_t k, uint32_t g, uint32_t t, Batch& b)
    {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            if constexpr (FULL) {
                const uint4 v = load_stream(src.at[c] + k);
                b.word[c][0] = v.x; b.word[c][1] = v.y; b.word[c][2] = v.z; b.word[c][3] = v.w;
            } else {
                gather_words<8>(src.at[c] + k, 1, n0 + 8 * c + g < p.N && k + 8 * t < p.K ? p.K - k - 8 * t : 0, b.word[c]);
            }
        }
    }
    template <int NT, bool FULL>
    static __device__ __forceinline__ void compute(const Batch& b, const FewRowsParams&, const FewRowsX<T, NT>& x, uint32_t k, uint32_t t, float (&acc)[kTiles][NT][4])
    {
        uint32_t xw[NT][4];
#pragma unroll
        for (uint32_t j = 0; j < NT; ++j) x.template load<8, FULL>(j, k + 8 * t, xw[j]);
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) {
                mma_16x8x16<T>(acc[i][j], b.word[2 * i][0], b.word[2 * i + 1][0], b.word[2 * i][1], b.word[2 * i + 1][1], xw[j][0], xw[j][1]);
                mma_16x8x16<T>(acc[i][j], b.word[2 * i][2], b.word[2 * i + 1][2], b.word[2 * i][3], b.word[2 * i + 1][3], xw[j][2], xw[j][3]);
            }
    }
};

// ------------------------------------------------------------------------------------------ the kernel
// NW: weights (2: gated).  NT: tiles of 8 rows of x per CTA; grid z walks further rows.  Grid x: column tiles, grid y = the
// cluster: parts of K.
template <typename T, typename Format, int NW, int NT>
__global__ void __launch_bounds__(32 * kFewRowsMaxWarps)
few_rows_kernel(const __grid_constant__ FewRowsParams p)
{
    constexpr uint32_t kCols = Format::kCols, kTiles = Format::kTiles, kPitch = kCols + 1;
    __shared__ float red[NW][kFewRowsMaxWarps][8][kPitch];      // [weight][warp][row of x][column]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t wn = warp % p.warps_n, wk = warp / p.warps_n, parts = (blockDim.x >> 5) / p.warps_n;
    const uint32_t n0 = (blockIdx.x * p.warps_n + wn) * kCols, m0 = blockIdx.z * (8 * NT);
    const uint32_t k0 = (blockIdx.y * parts + wk) * p.k_per_warp, k1 = min(p.K, k0 + p.k_per_warp);

    float acc[NW][kTiles][NT][4];
#pragma unroll
    for (uint32_t w = 0; w < NW; ++w)
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j)
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) acc[w][i][j][c] = 0.0f;

    if (k0 < k1 && n0 < p.N) {
        const FewRowsX<T, NT> x(p, m0, g);
        const typename Format::Source src[2] = {{p, p.w[0], n0, g, t}, {p, p.w[NW - 1], n0, g, t}};
        const bool aligned = p.x_vec && p.w[0].vec && p.w[NW - 1].vec;
        const uint32_t whole = aligned ? k0 + (k1 - k0) / Format::kBatch * Format::kBatch : k0;
        typename Format::Batch one[NW], two[NW];
        auto load = [&](uint32_t k, typename Format::Batch (&b)[NW]) {
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) Format::template load<true>(p, p.w[w], src[w], n0, k, g, t, b[w]);
        };
        auto compute = [&](uint32_t k, const typename Format::Batch (&b)[NW]) {
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) Format::template compute<NT, true>(b[w], p, x, k, t, acc[w]);
        };
        if (k0 < whole) load(k0, one);
        for (uint32_t k = k0; k < whole; k += 2 * Format::kBatch) {                // the next batch is in flight under this one
            const uint32_t k_two = k + Format::kBatch, k_next = k_two + Format::kBatch;
            if (k_two < whole) load(k_two, two);
            compute(k, one);
            if (k_two < whole) {
                if (k_next < whole) load(k_next, one);
                compute(k_two, two);
            }
        }
        for (uint32_t k = whole; k < k1; k += Format::kBatch)
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) {
                Format::template load<false>(p, p.w[w], src[w], n0, k, g, t, one[w]);
                Format::template compute<NT, false>(one[w], p, x, k, t, acc[w]);
            }
    }

    const bool split = gridDim.y > 1;
#pragma unroll
    for (uint32_t j = 0; j < NT; ++j) {
        if (j > 0) __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < NW; ++w)
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) red[w][warp][2 * t + (c & 1)][Format::column(g, i, c >> 1)] = acc[w][i][j][c];
        __syncthreads();
        // the parts of K inside the CTA in order; with a cluster, the sums wait in the place of the first for those of the other CTAs
        const uint32_t items = p.warps_n * 8 * kCols, rows = min(8u, p.M - min(p.M, m0 + 8 * j));
        if (split) {
            for (uint32_t id = threadIdx.x; id < items; id += blockDim.x) {
                const uint32_t col = id % kCols, row = id / kCols % 8, tile = id / (8 * kCols);
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) {
                    float s = red[w][tile][row][col];
                    for (uint32_t q = 1; q < parts; ++q) s += red[w][q * p.warps_n + tile][row][col];
                    red[w][tile][row][col] = s;
                }
            }
            cluster_arrive_release();
            cluster_wait_acquire();
        }
        if (blockIdx.y == 0) {
            for (uint32_t id = threadIdx.x; id < items; id += blockDim.x) {
                const uint32_t col = id % kCols, row = id / kCols % 8, tile = id / (8 * kCols);
                const uint32_t m = m0 + 8 * j + row, n = (blockIdx.x * p.warps_n + tile) * kCols + col;
                if (row >= rows || n >= p.N) continue;
                float v[NW];
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) {
                    v[w] = red[w][tile][row][col];
                    if (split)
                        for (uint32_t r = 1; r < gridDim.y; ++r) v[w] += __uint_as_float(ld_shared_remote_u32(smem_u32(&red[w][tile][row][col]), r));
                    else
                        for (uint32_t q = 1; q < parts; ++q) v[w] += red[w][q * p.warps_n + tile][row][col];
                    if (p.w[w].bias) v[w] += to_float<T>(static_cast<const T*>(p.w[w].bias)[n * p.w[w].bias_n]);
                    if (p.w[w].keep) static_cast<T*>(p.w[w].keep)[m * p.w[w].keep_m + n * p.w[w].keep_n] = from_float<T>(v[w]);
                }
                float y = gate_activation<T>(p.act, v[0]);
                if constexpr (NW == 2) y *= v[1];
                static_cast<T*>(p.out)[m * p.o_m + n * p.o_n] = from_float<T>(y);
            }
        }
        if (split) {                                             // the sums are read by the first CTA until here
            cluster_arrive_release();
            cluster_wait_acquire();
        }
    }
}

// ------------------------------------------------------------------------------------------ making 4-bit weights
struct Int4QuantizeParams {
    const void* w; long long w_k, w_n;
    uint32_t* words; long long words_ld;
    void* scales; long long scales_ld;
    uint8_t* zeros; long long zeros_ld;           // null: symmetric
    uint32_t K, N, group;
};

// One thread per (group, column).  Symmetric: s = max |w| / 7 and q = round(w / s) + 8; with zero points: s = (max - min) / 15 over the
// group's values and 0, z = round(-min / s), q = round(w / s) + z; clamped to 0 .. 15, ties to even, everything in fp32 with s as stored.
// A group of zeros has s = 0; one with a value that is not finite has s = NaN.
template <typename T>
__global__ void __launch_bounds__(128)
int4_quantize_kernel(const __grid_constant__ Int4QuantizeParams p)
{
    const uint32_t n = blockIdx.x * 128 + threadIdx.x, k0 = blockIdx.y * p.group, k1 = min(p.K, k0 + p.group);
    if (n >= p.N) return;
    const T* w = static_cast<const T*>(p.w) + n * p.w_n;
    float lo = 0.0f, hi = 0.0f;
    bool finite = true;
    for (uint32_t k = k0; k < k1; ++k) {
        const float v = to_float<T>(w[k * p.w_k]);
        finite = finite && fabsf(v) <= 3.402823466e38f;
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    const T stored = from_float<T>(finite ? (p.zeros ? __fdiv_rn(hi - lo, 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f)) : __int_as_float(0x7fffffff));
    const float s = to_float<T>(stored);
    const bool some = s > 0.0f;
    float z = 8.0f;
    if (p.zeros && some) z = fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f);
    static_cast<T*>(p.scales)[static_cast<long long>(blockIdx.y) * p.scales_ld + n] = stored;
    if (p.zeros) p.zeros[static_cast<long long>(blockIdx.y) * p.zeros_ld + n] = static_cast<uint8_t>(z);
    for (uint32_t k = k0; k < k1; k += 8) {
        uint32_t word = 0;
        for (uint32_t j = 0; j < 8; ++j) {
            float q = z;
            if (some && k + j < k1) q = fminf(fmaxf(rintf(__fdiv_rn(to_float<T>(w[(k + j) * p.w_k]), s)) + z, 0.0f), 15.0f);
            word |= static_cast<uint32_t>(q) << (4 * j);
        }
        p.words[static_cast<long long>(k >> 3) * p.words_ld + n] = word;
    }
}

struct Int4DequantizeParams {
    FewRowsWeight w;
    void* out; long long o_k, o_n;
    uint32_t K, N, group;
};

template <typename T>
__global__ void __launch_bounds__(128)
int4_dequantize_kernel(const __grid_constant__ Int4DequantizeParams p)
{
    const uint32_t n = blockIdx.x * 128 + threadIdx.x;
    if (n >= p.N) return;
    for (uint32_t word_row = blockIdx.y; word_row * 8 < p.K; word_row += gridDim.y) {
        const uint32_t word = static_cast<const uint32_t*>(p.w.w)[static_cast<long long>(word_row) * p.w.ld + n];
        const long long group = word_row * 8 / p.group;
        const float s = to_float<T>(static_cast<const T*>(p.w.scales)[group * p.w.scales_ld + n]);
        const int32_t z = p.w.zeros ? p.w.zeros[group * p.w.zeros_ld + n] & 15 : 8;
        for (uint32_t j = 0; j < 8 && word_row * 8 + j < p.K; ++j)
            static_cast<T*>(p.out)[static_cast<long long>(word_row * 8 + j) * p.o_k + n * p.o_n] =
                from_float<T>(static_cast<float>(static_cast<int32_t>((word >> (4 * j)) & 15u) - z) * s);
    }
}

}  // namespace srt
