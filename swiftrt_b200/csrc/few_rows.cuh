// Products of a few rows with a wide weight: y = act(x . W + b), or act(x . W0 + b0) * (x . W1 + b1), for M = 1 .. some tens of
// rows.  Every weight is read once and used M times, so the reading of the weights bounds it.  The multiplying is done by
// warp-wide MMAs (m16n8k16, fp32 accumulators): the weight is the MMA's 16-row operand (16 columns of W), eight rows of x its
// 8-column operand.  Within a k-step k may be permuted freely as long as both operands agree, so every weight format is taken 16
// bytes at a time in whatever order it is stored:
//
//   Int4   word (j, n) of the packed weight: rows 8 j .. 8 j + 7 of column n.  Lane (g, t) of a warp takes 4 columns (16 bytes)
//          of one word row: 32 columns x 32 rows per step.  Two nibbles at a time become the 16-bit floats 128 + q (bf16) or
//          1024 + q (fp16) by one AND-OR (as published by Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run", 2022); subtracting 128 + z (1024 + z) is exact, so the MMA multiplies the integers
//          q - z and the group's scale is applied to its fp32 sum, once per group: no weight is ever rounded.
//   Rows   16-bit elements, columns contiguous ([K x N] as Dense keeps it): lane (g, t) takes 8 columns of four rows;
//          neighbouring rows are paired by byte permutes.
//   Cols   16-bit elements, K contiguous: lane (g, t) takes 8 k of columns g, g + 8, g + 16, g + 24, pairs as they are.
//
// Two kernels.  few_rows_tiles_kernel takes weights whose rows start on 16 bytes: TMA boxes of 128 bytes by 16 KG or 32 rows go through
// a ring of 16 KB stages per weight, x lies in shared memory from the start.  few_rows_kernel takes any view with guarded loads.
// In both, the fp32 partial sums of the parts of K are added in their order (shared memory, then the distributed shared memory of a
// cluster): one launch, no workspace, and the same bits every time.
//
// One token: 4096 x 2 x 16384 bf16 43 us (6.2 TB/s, 0.95 of a copy); 4096 x 16384 in 4 bits 14.3 us (2.4 TB/s), 4096 x 2 x 16384 in 4 bits,
// four tokens, 26.4 us (2.6 TB/s).  In 4 bits about 4 us are start and finish, and then three instructions for every two weights
// bind next to the loads (issue slots 47 %, half-rate integer units 42 % busy).
#pragma once
#include <cuda.h>

#include <type_traits>

#include "element.cuh"
#include "fast_div.cuh"
#include "few_rows_plan.h"
#include "ptx.cuh"

namespace srt {

struct FewRowsWeight {
    const void* w; long long ld;                  // Int4: int32 words, ld words between word rows; Rows / Cols: ld elements between rows / columns
    const void* scales; long long scales_ld;
    const uint8_t* zeros; long long zeros_ld;     // may be null: 8
    uint32_t vec;                                 // rows on 16 bytes (scales on 8, zero points on 4)
    const void* bias; long long bias_n;           // may be null
    void* keep; long long keep_m, keep_n;         // receives x . W + b; may be null
};

struct FewRowsParams {
    FewRowsWeight w[2];
    const void* x; long long x_m, x_k;
    uint32_t x_vec;                               // rows of x are 16-byte aligned and contiguous
    void* out; long long o_m, o_n;
    uint32_t M, N, K, group, act;
    FastDiv by_group;
    uint32_t k_per_part;                          // rows of W per warp (few_rows_kernel) or CTA (few_rows_tiles_kernel)
    uint32_t column_groups;                       // few_rows_tiles_kernel: column tiles of a CTA
    uint32_t stages, x_pitch;                     // its ring, and bytes between rows of x in shared memory
    uint32_t* status;
    unsigned long long wait_cycles;
};
struct FewRowsMaps { CUtensorMap w[2]; };

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

// COUNT consecutive 16-bit elements as words, from address at + i * stride while i < live; zeros behind that
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
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[4])
{
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds_word(uint32_t at)
{
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
    return w;
}

// ------------------------------------------------------------------------------------------ weight formats
// A format says what a lane loads of one unit (kUnit rows of W: kChunks times 16 bytes of the weight, eight or four elements of every row
// of x), how a unit lies in a stage of the ring, and how it enters the MMAs.  kWarpRows: rows of W of a warp's 2 KB of a stage.
// Stages are swizzled: the 16-byte chunk c of a 128-byte row r lies at chunk c ^ (r mod 8).  The rows (Int4, Rows) or chunks (Cols) that the
// four t of a load take are two apart, so that the eight lanes of a quarter warp read eight different chunks: no bank conflicts.
template <typename T, int GPB>            // GPB: scale groups in 128 rows (4, 2, or 1 for groups of 128 and more)
struct Int4Format {
    static constexpr FewRowsFormat kFormat = kInt4Weights;
    static constexpr uint32_t kCols = kFormat.cols, kTiles = 2, kUnit = 32, kChunks = 1, kXWords = 4, kWarpRows = kFormat.warp_rows, kUnits = 4;
    static constexpr bool kGroups = kFormat.grouped;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 4 * g + 2 * tile + half; }

    struct Group { uint32_t scale[2], zero; };
    struct Offsets { uint32_t v[4]; };             // the zero points as the floats that the nibbles' magic makes of them
    // this lane's part of a weight in memory
    struct Source {
        const uint32_t* words;                     // word row t
        const unsigned short* scales; const uint8_t* zeros;
        uint32_t live;                             // columns of this lane that exist
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t t)
        {
            const uint32_t n = n0 + 4 * g < p.N ? n0 + 4 * g : 0;
            live = n0 + 4 * g < p.N ? p.N - n0 - 4 * g : 0;
            words = static_cast<const uint32_t*>(w.w) + static_cast<long long>(t) * w.ld + n;
            scales = static_cast<const unsigned short*>(w.scales) + n;
            zeros = w.zeros ? w.zeros + n : nullptr;
        }
    };
    // aligned; rows behind the last read the last one's group
    static __device__ __forceinline__ void load_group(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t k, Group& gr)
    {
        const long long group = fast_div(min(k, p.K - 1), p.by_group);
        if (src.live >= 4) {
            const uint2 s = __ldg(reinterpret_cast<const uint2*>(src.scales + group * w.scales_ld));
            gr.scale[0] = s.x; gr.scale[1] = s.y;
            gr.zero = src.zeros ? __ldg(reinterpret_cast<const uint32_t*>(src.zeros + group * w.zeros_ld)) : 0x08080808u;
        } else {
            gather_group(p, w, src, min(k, p.K - 1), gr);             // the last columns
        }
    }
    // the same, and a unit's words, where anything may be unaligned or missing
    static __device__ __forceinline__ void gather_group(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t k, Group& gr)
    {
        const long long group = k / p.group;
        gather_words<4>(src.scales + group * w.scales_ld, 1, src.live, gr.scale);
        gr.zero = 0x08080808u;
        if (src.zeros) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (j < src.live) gr.zero = (gr.zero & ~(255u << (8 * j))) | static_cast<uint32_t>(__ldg(src.zeros + group * w.zeros_ld + j)) << (8 * j);
        }
    }
    static __device__ __forceinline__ void gather_unit(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t k, uint32_t t, uint32_t (&words)[kChunks][4])
    {
        const uint32_t* at = src.words + static_cast<long long>(k >> 3) * w.ld;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) words[0][j] = j < src.live && k + 8 * t < p.K ? __ldg(at + j) : 0u;
    }
    static __device__ __forceinline__ void gather_x(const void* row, long long stride, uint32_t k, uint32_t live, uint32_t t, uint32_t (&x)[kXWords])
    {
        gather_words<8>(static_cast<const T*>(row) + static_cast<long long>(k + 8 * t) * stride, stride, live > 8 * t ? live - 8 * t : 0, x);
        arrange(x);
    }
    // eight elements of x in the order of the weight's pairs: rows 0 and 4, 1 and 5, 2 and 6, 3 and 7
    static __device__ __forceinline__ void arrange(uint32_t (&x)[4])
    {
        const uint32_t a = x[0], b = x[1], c = x[2], d = x[3];
        x[0] = __byte_perm(a, c, 0x5410);
        x[1] = __byte_perm(a, c, 0x7632);
        x[2] = __byte_perm(b, d, 0x5410);
        x[3] = __byte_perm(b, d, 0x7632);
    }
    // unit u of a warp's part of a stage (16 word rows of 128 bytes), and x from its first row's elements on
    // (groups of 32 rows: a unit has to be 4 neighbouring word rows, and two lanes of a quarter warp share a bank)
    static __device__ __forceinline__ uint32_t word_row(uint32_t u, uint32_t t) { return GPB == 4 ? 4 * u + t : 8 * (u >> 1) + 2 * t + (u & 1); }
    static __device__ __forceinline__ void stage_unit(uint32_t at, uint32_t, uint32_t u, uint32_t g, uint32_t t, uint32_t (&words)[kChunks][4])
    {
        const uint32_t r = word_row(u, t);
        lds_words(at + r * 128 + ((g ^ (r & 7)) << 4), words[0]);
    }
    static __device__ __forceinline__ void stage_x(uint32_t at, uint32_t u, uint32_t t, uint32_t (&x)[kXWords]) { lds_words(at + 16 * word_row(u, t), x); }

    static __device__ __forceinline__ Offsets offsets(const Group& gr)
    {
        constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x6400u : 0x4300u;
        Offsets o;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) o.v[j] = (kMagic | ((gr.zero >> (8 * j)) & 15u)) * 0x10001u;
        return o;
    }
    // pair s of a word's nibbles, rows s and s + 4 of its eight, as the integers q - z in two 16-bit floats
    static __device__ __forceinline__ uint32_t integers(uint32_t word, uint32_t s, uint32_t magic_zero)
    {
        constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;
        uint32_t v;                                    // (word & mask) | magic as the one instruction that it is
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(word >> (4 * s)), "r"(0x000f000fu), "r"(kMagic));
        if constexpr (std::is_same<T, __half>::value) {
            const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<const __half2*>(&magic_zero));
            return *reinterpret_cast<const uint32_t*>(&d);
        } else {
            const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&magic_zero));
            return *reinterpret_cast<const uint32_t*>(&d);
        }
    }
    template <int NT>
    static __device__ __forceinline__ void multiply(const uint32_t (&words)[kChunks][4], const Offsets& o, const uint32_t (&x)[NT][kXWords], float (&sum)[kTiles][NT][4])
    {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
            uint32_t a[2][4];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) a[h][q] = integers(words[0][2 * i + h], q, o.v[2 * i + h]);
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) {
                mma_16x8x16<T>(sum[i][j], a[0][0], a[1][0], a[0][1], a[1][1], x[j][0], x[j][1]);
                mma_16x8x16<T>(sum[i][j], a[0][2], a[1][2], a[0][3], a[1][3], x[j][2], x[j][3]);
            }
        }
    }
    template <int NT>
    static __device__ __forceinline__ void close_group(const Group& gr, float (&sum)[kTiles][NT][4], float (&acc)[kTiles][NT][4])
    {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
            const T* pair = reinterpret_cast<const T*>(&gr.scale[i]);
            const float s0 = to_float<T>(pair[0]), s1 = to_float<T>(pair[1]);
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) {
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) {
                    acc[i][j][c] = fmaf(c < 2 ? s0 : s1, sum[i][j][c], acc[i][j][c]);
                    sum[i][j][c] = 0.0f;
                }
            }
        }
    }
    static constexpr uint32_t kGroupUnits = 4 / GPB;
};

// 16-bit weights have no groups: their MMAs add into the result at once.
struct NoGroup { uint32_t unused; };

template <typename T>
struct RowsFormat {
    static constexpr FewRowsFormat kFormat = kRowWeights;
    static constexpr uint32_t kCols = kFormat.cols, kTiles = 4, kUnit = 16, kChunks = 4, kXWords = 2, kWarpRows = kFormat.warp_rows, kUnits = 1, kGroupUnits = 1;
    static constexpr bool kGroups = kFormat.grouped;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 8 * g + 2 * tile + half; }
    static __device__ __forceinline__ uint32_t row(uint32_t c, uint32_t t) { return 8 * (c >> 1) + 2 * t + (c & 1); }
    using Group = NoGroup;
    using Offsets = NoGroup;
    struct Source {
        const T* at;
        uint32_t live;
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t)
            : at(static_cast<const T*>(w.w) + (n0 + 8 * g < p.N ? n0 + 8 * g : 0)), live(n0 + 8 * g < p.N ? p.N - n0 - 8 * g : 0) {}
    };
    static __device__ __forceinline__ void gather_unit(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t k, uint32_t t, uint32_t (&words)[kChunks][4])
    {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) gather_words<8>(src.at + static_cast<long long>(k + row(c, t)) * w.ld, 1, k + row(c, t) < p.K ? src.live : 0, words[c]);
    }
    static __device__ __forceinline__ void gather_x(const void* x_row, long long stride, uint32_t k, uint32_t live, uint32_t t, uint32_t (&x)[kXWords])
    {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t from = 8 * h + 2 * t;
            uint32_t w[1];
            gather_words<2>(static_cast<const T*>(x_row) + static_cast<long long>(k + from) * stride, stride, live > from ? live - from : 0, w);
            x[h] = w[0];
        }
    }
    static __device__ __forceinline__ void stage_unit(uint32_t at, uint32_t, uint32_t, uint32_t g, uint32_t t, uint32_t (&words)[kChunks][4])
    {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) lds_words(at + row(c, t) * 128 + ((g ^ (row(c, t) & 7)) << 4), words[c]);
    }
    static __device__ __forceinline__ void stage_x(uint32_t at, uint32_t, uint32_t t, uint32_t (&x)[kXWords])
    {
        x[0] = lds_word(at + 4 * t);
        x[1] = lds_word(at + 16 + 4 * t);
    }
    template <int NT>
    static __device__ __forceinline__ void multiply(const uint32_t (&words)[kChunks][4], const Offsets&, const uint32_t (&x)[NT][kXWords], float (&acc)[kTiles][NT][4])
    {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) {
            const uint32_t a0 = __byte_perm(words[0][i], words[1][i], 0x5410), a1 = __byte_perm(words[0][i], words[1][i], 0x7632);
            const uint32_t a2 = __byte_perm(words[2][i], words[3][i], 0x5410), a3 = __byte_perm(words[2][i], words[3][i], 0x7632);
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) mma_16x8x16<T>(acc[i][j], a0, a1, a2, a3, x[j][0], x[j][1]);
        }
    }
};

template <typename T>
struct ColsFormat {
    static constexpr FewRowsFormat kFormat = kColumnWeights;
    static constexpr uint32_t kCols = kFormat.cols, kTiles = 2, kUnit = 32, kChunks = 4, kXWords = 4, kWarpRows = kFormat.warp_rows, kUnits = 1, kGroupUnits = 1;
    static constexpr bool kGroups = kFormat.grouped;
    static __device__ __forceinline__ uint32_t column(uint32_t g, uint32_t tile, uint32_t half) { return 16 * tile + 8 * half + g; }
    using Group = NoGroup;
    using Offsets = NoGroup;
    struct Source {
        const T* at;                                   // column n0 + g
        uint32_t live;                                 // of columns n0 + g + 8 c
        __device__ __forceinline__ Source(const FewRowsParams& p, const FewRowsWeight& w, uint32_t n0, uint32_t g, uint32_t)
        {
            live = n0 + g < p.N ? min(4u, (p.N - n0 - g + 7) / 8) : 0;
            at = static_cast<const T*>(w.w) + static_cast<long long>(min(n0 + g, p.N - 1)) * w.ld;
        }
    };
    static __device__ __forceinline__ void gather_unit(const FewRowsParams& p, const FewRowsWeight& w, const Source& src, uint32_t k, uint32_t t, uint32_t (&words)[kChunks][4])
    {
        const uint32_t from = k + 8 * t;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) gather_words<8>(src.at + static_cast<long long>(8 * c) * w.ld + from, 1, c < src.live && from < p.K ? p.K - from : 0, words[c]);
    }
    static __device__ __forceinline__ void gather_x(const void* row, long long stride, uint32_t k, uint32_t live, uint32_t t, uint32_t (&x)[kXWords])
    {
        gather_words<8>(static_cast<const T*>(row) + static_cast<long long>(k + 8 * t) * stride, stride, live > 8 * t ? live - 8 * t : 0, x);
    }
    // a box holds 64 k of 32 columns: two warps' parts, `odd` says which
    static __device__ __forceinline__ void stage_unit(uint32_t at, uint32_t odd, uint32_t, uint32_t g, uint32_t t, uint32_t (&words)[kChunks][4])
    {
        at -= odd * 2048;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) lds_words(at + (g + 8 * c) * 128 + (((2 * t + odd) ^ g) << 4), words[c]);
    }
    static __device__ __forceinline__ void stage_x(uint32_t at, uint32_t, uint32_t t, uint32_t (&x)[kXWords]) { lds_words(at + 32 * t, x); }
    template <int NT>
    static __device__ __forceinline__ void multiply(const uint32_t (&words)[kChunks][4], const Offsets&, const uint32_t (&x)[NT][kXWords], float (&acc)[kTiles][NT][4])
    {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) {
                mma_16x8x16<T>(acc[i][j], words[2 * i][0], words[2 * i + 1][0], words[2 * i][1], words[2 * i + 1][1], x[j][0], x[j][1]);
                mma_16x8x16<T>(acc[i][j], words[2 * i][2], words[2 * i + 1][2], words[2 * i][3], words[2 * i + 1][3], x[j][2], x[j][3]);
            }
    }
};

template <int NW, int TILES, int NT> __device__ __forceinline__ void clear(float (&v)[NW][TILES][NT][4])
{
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[w][i][j][c] = 0.0f;
}

// ------------------------------------------------------------------------------------------ sums and results
// The warps' sums to the result, for both kernels: warp `slot` holds part slot / groups of column tile slot mod groups (of this CTA's
// `groups`); red: room for few_rows_sum_bytes.  All threads of the CTA call it; `mine`: this thread holds sums.
template <typename T, typename Format, int NW, int NT>
__device__ __forceinline__ void few_rows_finish(const FewRowsParams& p, float* red, uint32_t slot, bool mine, uint32_t groups, uint32_t tile0, uint32_t m0,
                                                const float (&acc)[NW][Format::kTiles][NT][4])
{
    constexpr uint32_t kCols = Format::kCols, kPitch = kCols + 1;
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, parts = kFewRowsWarps / groups;
    auto place = [&](uint32_t w, uint32_t s, uint32_t row, uint32_t col) { return ((w * kFewRowsWarps + s) * (8 * NT) + row) * kPitch + col; };
    const bool split = gridDim.y > 1;
    __syncthreads();
    if (mine) {
#pragma unroll
        for (uint32_t w = 0; w < NW; ++w)
#pragma unroll
            for (uint32_t i = 0; i < Format::kTiles; ++i)
#pragma unroll
                for (uint32_t j = 0; j < NT; ++j)
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) red[place(w, slot, 8 * j + 2 * t + (c & 1), Format::column(g, i, c >> 1))] = acc[w][i][j][c];
    }
    __syncthreads();
    const uint32_t rows = min(8u * NT, p.M - m0), items = groups * rows * kCols;
    // with a cluster, the sum of a CTA's parts takes the place of the first, and every CTA finishes its share of the results
    uint32_t first = threadIdx.x, end = items;
    if (split) {
        if (parts > 1) {
            for (uint32_t id = threadIdx.x; id < items; id += blockDim.x) {
                const uint32_t col = id % kCols, row = id / kCols % rows, tile = id / (rows * kCols);
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w) {
                    float s = red[place(w, tile, row, col)];
                    for (uint32_t q = 1; q < parts; ++q) s += red[place(w, q * groups + tile, row, col)];
                    red[place(w, tile, row, col)] = s;
                }
            }
        }
        cluster_arrive_release();
        cluster_wait_acquire();
        const uint32_t share = (items + gridDim.y - 1) / gridDim.y;
        first += blockIdx.y * share;
        end = min(items, (blockIdx.y + 1) * share);
    }
    for (uint32_t id = first; id < end; id += blockDim.x) {
        const uint32_t col = id % kCols, row = id / kCols % rows, tile = id / (rows * kCols);
        const uint32_t m = m0 + row, n = (tile0 + tile) * kCols + col;
        if (n >= p.N) continue;
        float v[NW];
#pragma unroll
        for (uint32_t w = 0; w < NW; ++w) {
            const float* at = &red[place(w, tile, row, col)];
            if (split) {
                float part[8];
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) part[r] = r < gridDim.y ? __uint_as_float(ld_shared_remote_u32(smem_u32(at), r)) : 0.0f;
                v[w] = part[0];
#pragma unroll
                for (uint32_t r = 1; r < 8; ++r) v[w] += part[r];
            } else {
                v[w] = *at;
                for (uint32_t q = 1; q < parts; ++q) v[w] += red[place(w, q * groups + tile, row, col)];
            }
            if (p.w[w].bias) v[w] += to_float<T>(static_cast<const T*>(p.w[w].bias)[n * p.w[w].bias_n]);
            if (p.w[w].keep) static_cast<T*>(p.w[w].keep)[m * p.w[w].keep_m + n * p.w[w].keep_n] = from_float<T>(v[w]);
        }
        float y = gate_activation<T>(p.act, v[0]);
        if constexpr (NW == 2) y *= v[1];
        static_cast<T*>(p.out)[m * p.o_m + n * p.o_n] = from_float<T>(y);
    }
    if (split) {                                                 // a CTA's sums are read by the others until here
        cluster_arrive_release();
        cluster_wait_acquire();
    }
}

// ------------------------------------------------------------------------------------------ any view
// NW: weights (2: gated).  NT: tiles of 8 rows of x per CTA; grid z walks further rows.  Grid x: column tiles, grid y = the
// cluster: parts of K beyond the eight warps.
template <typename T, typename Format, int NW, int NT>
__global__ void __launch_bounds__(32 * kFewRowsWarps)
few_rows_kernel(const __grid_constant__ FewRowsParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t n0 = blockIdx.x * Format::kCols, m0 = blockIdx.z * (8 * NT);
    const uint32_t k0 = (blockIdx.y * kFewRowsWarps + warp) * p.k_per_part, k1 = min(p.K, k0 + p.k_per_part);
    float acc[NW][Format::kTiles][NT][4];
    clear(acc);
    if (k0 < k1) {
        const typename Format::Source src[2] = {{p, p.w[0], n0, g, t}, {p, p.w[NW - 1], n0, g, t}};
        for (uint32_t k = k0; k < k1; k += Format::kUnit) {
            uint32_t words[NW][Format::kChunks][4], x[NT][Format::kXWords];
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) Format::gather_unit(p, p.w[w], src[w], k, t, words[w]);
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) {
                const uint32_t m = m0 + 8 * j + g;
                Format::gather_x(static_cast<const T*>(p.x) + static_cast<long long>(min(m, p.M - 1)) * p.x_m, p.x_k, k, m < p.M ? p.K - k : 0, t, x[j]);
            }
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) {
                if constexpr (Format::kGroups) {
                    typename Format::Group group;
                    Format::gather_group(p, p.w[w], src[w], k, group);
                    float sum[1][Format::kTiles][NT][4];
                    clear(sum);
                    Format::template multiply<NT>(words[w], Format::offsets(group), x, sum[0]);
                    Format::template close_group<NT>(group, sum[0], acc[w]);
                } else {
                    Format::template multiply<NT>(words[w], NoGroup{}, x, acc[w]);
                }
            }
        }
    }
    few_rows_finish<T, Format, NW, NT>(p, reinterpret_cast<float*>(smem), warp, true, 1, blockIdx.x, m0, acc);
}

// ------------------------------------------------------------------------------------------ aligned weights
// Warps 0 .. 7 multiply: warp w takes column tile w mod CG and part w / CG (of KG = 8 / CG) of every stage's rows.  Warp 8 asks for the
// stages: per weight 16 KB, CG tiles of 128-byte rows.  CG is 8 for wide weights (the rows of a stage are then a kilobyte of memory each)
// and smaller where column tiles are few.
template <typename T, typename Format, int NW, int NT>
__global__ void __launch_bounds__(kFewRowsTileThreads)
few_rows_tiles_kernel(const __grid_constant__ FewRowsParams p, const __grid_constant__ FewRowsMaps maps)
{
    extern __shared__ uint8_t dynamic_smem[];
    __shared__ __align__(8) uint64_t full_bar[kFewRowsMaxStages], empty_bar[kFewRowsMaxStages];
    __shared__ volatile uint32_t never_set;
    const uint32_t ring = (smem_u32(dynamic_smem) + 1023u) & ~1023u;                // the swizzle repeats every 1024 bytes
    const uint32_t xs = ring + p.stages * NW * kFewRowsStageBytes;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t groups = p.column_groups, parts = kFewRowsWarps / groups, stage_rows = parts * Format::kWarpRows;
    const uint32_t tile0 = blockIdx.x * groups, m0 = blockIdx.z * (8 * NT);
    const uint32_t k0 = blockIdx.y * p.k_per_part, k1 = min(p.K, k0 + p.k_per_part);
    const uint32_t rounds = k0 < k1 ? (k1 - k0 + stage_rows - 1) / stage_rows : 0;
    if (threadIdx.x == 0) {
        never_set = 0;
        for (uint32_t s = 0; s < p.stages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), kFewRowsWarps);
        }
        fence_mbar_init();
        for (uint32_t w = 0; w < NW; ++w) prefetch_tensormap(&maps.w[w]);
    }
    __syncthreads();

    float acc[NW][Format::kTiles][NT][4];
    clear(acc);
    // a wait over the limit is noted (the result is invalid then) and goes on, so that nothing is left in flight
    auto wait = [&](uint64_t& bar, uint32_t parity) {
        if (mbar_wait(smem_u32(&bar), parity, &never_set, p.wait_cycles)) return true;
        atomicOr(p.status, 1u);
        return mbar_wait(smem_u32(&bar), parity, &never_set, 4000000000ull);
    };
    if (warp == kFewRowsWarps) {
        if (elect_one()) {
            for (uint32_t r = 0; r < rounds; ++r) {
                const uint32_t s = r % p.stages, bar = smem_u32(&full_bar[s]);
                if (r >= p.stages && !wait(empty_bar[s], (r / p.stages - 1) & 1)) break;
                mbar_arrive_expect_tx(bar, NW * kFewRowsStageBytes);
                const uint32_t k = k0 + r * stage_rows;
                for (uint32_t w = 0; w < NW; ++w) {
                    const uint32_t to = ring + (s * NW + w) * kFewRowsStageBytes;
                    for (uint32_t c = 0; c < groups; ++c) {
                        const int32_t n = static_cast<int32_t>((tile0 + c) * Format::kCols);
                        if constexpr (std::is_same<Format, ColsFormat<T>>::value) {
                            for (uint32_t b = 0; b < parts / 2; ++b)
                                tma_load_3d(to + (c * parts + 2 * b) * 2048, &maps.w[w], bar, static_cast<int32_t>(k + 64 * b), n, 0);
                        } else {
                            tma_load_3d(to + c * parts * 2048, &maps.w[w], bar, n, static_cast<int32_t>(Format::kGroups ? k / 8 : k), 0);
                        }
                    }
                }
            }
        }
        __syncwarp();
    }
    // x of this CTA's rows of W, zeros behind them (the producer's first stages are on their way meanwhile)
    const uint32_t x_rows = min(8u * NT, p.M - m0), x_words = rounds * stage_rows / 8;
    if (warp < kFewRowsWarps) {
        const uint32_t total = x_rows * x_words;
        for (uint32_t base = threadIdx.x; base < total; base += 4 * 32 * kFewRowsWarps) {
            uint32_t v[4][4], to[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {                                     // four loads in flight
                const uint32_t id = base + u * 32 * kFewRowsWarps;
                if (id >= total) break;
                const uint32_t row = id / x_words, word = id - row * x_words, k = k0 + word * 8;
                const T* at = static_cast<const T*>(p.x) + static_cast<long long>(m0 + row) * p.x_m + static_cast<long long>(k) * p.x_k;
                to[u] = xs + row * p.x_pitch + word * 16;
                if (p.x_vec && k + 8 <= p.K) {
                    const uint4 q = __ldg(reinterpret_cast<const uint4*>(at));
                    v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
                } else {
                    gather_words<8>(at, p.x_k, k < p.K ? p.K - k : 0, v[u]);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                if (base + u * 32 * kFewRowsWarps >= total) break;
                if constexpr (Format::kGroups) Format::arrange(v[u]);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to[u]), "r"(v[u][0]), "r"(v[u][1]), "r"(v[u][2]), "r"(v[u][3]) : "memory");
            }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");                              // the eight multiplying warps
        const uint32_t group_of = warp % groups, part = warp / groups;
        const uint32_t n0 = (tile0 + group_of) * Format::kCols;
        const typename Format::Source src[2] = {{p, p.w[0], n0, g, t}, {p, p.w[NW - 1], n0, g, t}};
        uint32_t x_at[NT];
#pragma unroll
        for (uint32_t j = 0; j < NT; ++j) x_at[j] = xs + min(8 * j + g, x_rows - 1) * p.x_pitch + part * Format::kWarpRows * 2;
        const uint32_t mine = (group_of * parts + part) * 2048, odd = part & 1;
        constexpr uint32_t kGroupsPerStage = Format::kUnits / Format::kGroupUnits;
        typename Format::Group next[NW][kGroupsPerStage];
        if constexpr (Format::kGroups) {
            if (rounds > 0) {
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w)
#pragma unroll
                    for (uint32_t q = 0; q < kGroupsPerStage; ++q)
                        Format::load_group(p, p.w[w], src[w], k0 + part * Format::kWarpRows + q * Format::kGroupUnits * Format::kUnit, next[w][q]);
            }
        }
        uint32_t s = 0, phase = 0;
        for (uint32_t r = 0; r < rounds; ++r) {
            typename Format::Group group[NW][kGroupsPerStage];
            if constexpr (Format::kGroups) {
                // the groups of the next stage are fetched under this one
#pragma unroll
                for (uint32_t w = 0; w < NW; ++w)
#pragma unroll
                    for (uint32_t q = 0; q < kGroupsPerStage; ++q) {
                        group[w][q] = next[w][q];
                        Format::load_group(p, p.w[w], src[w], k0 + (r + 1) * stage_rows + part * Format::kWarpRows + q * Format::kGroupUnits * Format::kUnit, next[w][q]);
                    }
            }
            if (!wait(full_bar[s], phase)) break;
            const uint32_t at = ring + s * NW * kFewRowsStageBytes + mine;
#pragma unroll
            for (uint32_t q = 0; q < kGroupsPerStage; ++q) {
                typename Format::Offsets off[NW];
                float sum[NW][Format::kTiles][NT][4];
                if constexpr (Format::kGroups) {
                    clear(sum);
#pragma unroll
                    for (uint32_t w = 0; w < NW; ++w) off[w] = Format::offsets(group[w][q]);
                }
#pragma unroll
                for (uint32_t v = 0; v < Format::kGroupUnits; ++v) {
                    const uint32_t u = q * Format::kGroupUnits + v;
                    uint32_t words[NW][Format::kChunks][4], x[NT][Format::kXWords];
#pragma unroll
                    for (uint32_t w = 0; w < NW; ++w) Format::stage_unit(at + w * kFewRowsStageBytes, odd, u, g, t, words[w]);
#pragma unroll
                    for (uint32_t j = 0; j < NT; ++j) {
                        // (Cols: the two warps of a box take its even and its odd 16-byte chunks)
                        uint32_t from = x_at[j];
                        if constexpr (std::is_same<Format, ColsFormat<T>>::value) from -= odd * 48;
                        Format::stage_x(from, u, t, x[j]);
                    }
#pragma unroll
                    for (uint32_t w = 0; w < NW; ++w) {
                        if constexpr (Format::kGroups) Format::template multiply<NT>(words[w], off[w], x, sum[w]);
                        else Format::template multiply<NT>(words[w], off[w], x, acc[w]);
                    }
                }
                if constexpr (Format::kGroups) {
#pragma unroll
                    for (uint32_t w = 0; w < NW; ++w) Format::template close_group<NT>(group[w][q], sum[w], acc[w]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) x_at[j] += stage_rows * 2;
            if (++s == p.stages) { s = 0; phase ^= 1; }
        }
    }
    few_rows_finish<T, Format, NW, NT>(p, reinterpret_cast<float*>(dynamic_smem + (ring - smem_u32(dynamic_smem))), warp, warp < kFewRowsWarps, groups, tile0, m0, acc);
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
    // (the range of finite BFloat16 values may exceed fp32's: the halves are subtracted then)
    const float range = hi - lo <= 3.402823466e38f ? __fdiv_rn(hi - lo, 15.0f) : __fdiv_rn(0.5f * hi - 0.5f * lo, 7.5f);
    const T stored = from_float<T>(finite ? (p.zeros ? range : __fdiv_rn(fmaxf(hi, -lo), 7.0f)) : __int_as_float(0x7fffffff));
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
