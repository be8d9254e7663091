// How a product of a few rows runs on few_rows_tiles_kernel (few_rows.cuh): column tiles and CTAs of a launch, the ring and the
// shared memory that it asks for.  Host arithmetic only, without a device.
#pragma once
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace srt {

// A CTA of few_rows_tiles_kernel: eight multiplying warps and one that asks for the stages, 16 KB per weight and stage.
constexpr uint32_t kFewRowsWarps = 8, kFewRowsTileThreads = 32 * (kFewRowsWarps + 1), kFewRowsStageBytes = 16384, kFewRowsMaxStages = 6;
// dynamic shared memory that the kernels are allowed (1 KB of the 227 is left for barriers)
constexpr uint32_t kFewRowsSharedLimit = 226 * 1024;

// What the plan needs to know of a weight format.
struct FewRowsFormat {
    uint32_t cols;                       // columns of a tile
    uint32_t warp_rows;                  // rows of W in a warp's 2 KB of a stage
    uint32_t max_column_groups;
    bool grouped;                        // 4-bit weights with group scales
};
constexpr FewRowsFormat kInt4Weights = {32, 128, 8, true}, kRowWeights = {64, 16, 8, false}, kColumnWeights = {32, 32, 2, false};

// the fp32 sums of all warps (rows of an odd pitch, without bank conflicts); nw weights, 8 nt rows of x
constexpr uint32_t few_rows_sum_bytes(const FewRowsFormat& f, uint32_t nw, uint32_t nt) { return nw * kFewRowsWarps * 8 * nt * (f.cols + 1) * 4; }

// Dynamic shared memory of a launch: the ring, whose place the sums take when it is done with, x behind it, and room to align them.
constexpr uint64_t few_rows_tiles_smem(const FewRowsFormat& f, uint32_t nw, uint32_t nt, uint32_t stages, uint64_t x_bytes)
{
    const uint64_t ring = static_cast<uint64_t>(stages) * nw * kFewRowsStageBytes, sums = (few_rows_sum_bytes(f, nw, nt) + 127) / 128 * 128;
    return 1024 + (ring > sums ? ring : sums) + x_bytes;
}

// groups = 0: x of these rows fits beside no stage
struct RowsPlan {
    double cost = 1e300;                 // estimate of its time in microseconds
    uint32_t groups = 0, cluster = 0, stages = 0, k_per_part = 0, x_pitch = 0, smem = 0;
};

// The choice of column tiles to a CTA and CTAs to a cluster by what it costs: rounds of CTAs and what they stream, x to bring in before
// the first product, the exchange of a cluster, SMs with one CTA's eight warps only, and the places that clusters of 4 and 8 leave
// free.  The constants are fitted to the times of all choices at 9 shapes of 4-bit and 6 of 16-bit weights and 1 .. 48 rows; the choice is
// on average 4 % slower than the best one.  One row, 4096 x 16384 in 4 bits, tiles x cluster: 8 x 4 17.0, 4 x 2 17.0, 2 x 1 16.4 us; 8 x 2
// 21.3, 8 x 8 22.5 us.  17 rows, 8192 x 1024: 2 x 8 in rows of 8 13.3, in rows of 32 19.6 us.
// most: CTAs that an SM's registers hold
inline RowsPlan plan_few_rows(const FewRowsFormat& f, uint32_t nw, uint32_t nt, uint32_t M, uint32_t N, uint32_t K, uint32_t most)
{
    RowsPlan best;
    const uint32_t row_blocks = (M + 8 * nt - 1) / (8 * nt), tiles = (N + f.cols - 1) / f.cols;
    const uint32_t x_rows = M < 8 * nt ? M : 8 * nt, stage_bytes = nw * kFewRowsStageBytes;
    for (uint32_t c = 1; c <= 8; c *= 2)
        for (uint32_t g = f.max_column_groups; g >= 1; g /= 2) {
            const uint32_t stage_rows = 8 / g * f.warp_rows, rounds = ((K + stage_rows - 1) / stage_rows + c - 1) / c;
            const uint64_t x_pitch = ((uint64_t)rounds * stage_rows * 2 + 127) / 128 * 128 + 16;      // rows of x start four banks apart
            const uint64_t x_bytes = x_rows * x_pitch;
            // as many CTAs to an SM as leave each three stages beside x
            uint32_t per_sm = most, stages = 0;
            for (; per_sm >= 1; --per_sm) {
                const uint64_t room = (224u / per_sm - 2) * 1024u - 1024u;
                stages = x_bytes < room ? (uint32_t)((room - x_bytes) / stage_bytes) : 0;
                if (stages >= 3 || stages >= rounds || per_sm == 1) break;
            }
            if (stages > kFewRowsMaxStages) stages = kFewRowsMaxStages;
            if (stages > rounds) stages = rounds;
            if (stages == 0) continue;
            const uint64_t smem = few_rows_tiles_smem(f, nw, nt, stages, x_bytes);
            if (smem > kFewRowsSharedLimit) continue;                                    // (beside much of x a ring may be shorter than the sums)
            const uint32_t at_once = per_sm > 2 ? 2 : per_sm;
            const double places = 148.0 * at_once * (c == 8 ? 0.45 : c == 4 ? 0.93 : 1.0), full = (double)((tiles + g - 1) / g) * row_blocks * c / places;
            const double waves = std::ceil(full), stream = rounds * stage_bytes * places / 5.5e6 * (at_once == 1 && f.grouped ? 1.4 : 1.0);  // a round at 5.5 TB/s
            double cost = waves * (7.3 + (f.grouped ? 0.6 * rounds : 0.0)) + stream * (0.15 * waves + 0.85 * (full > 0.25 ? full : 0.25)) + x_bytes / 1024.0 * 0.04 +
                          0.1 * nw * nt;
            if (c > 1) cost += 1.0 + 0.3 * c;
            if (cost < best.cost) {
                best.cost = cost;
                best.groups = g; best.cluster = c; best.stages = stages;
                best.k_per_part = rounds * stage_rows; best.x_pitch = (uint32_t)x_pitch; best.smem = (uint32_t)smem;
            }
        }
    return best;
}

// Which of the plans of 8, 16 and 32 rows to a CTA runs a product: the cheapest; kFewRowsElsewhere where the caller has another way that takes `limit`
// microseconds and none is faster or fits; kFewRowsAnyView, the kernel without tiles, where none fits and there is no other way
// (`limit` is infinite).
enum : int { kFewRowsAnyView = -1, kFewRowsElsewhere = -2 };
inline int choose_few_rows(const RowsPlan (&plan)[3], double limit)
{
    int which = plan[1].cost < plan[0].cost ? 1 : 0;
    if (plan[2].cost < plan[which].cost) which = 2;
    if (plan[which].groups == 0) return std::isinf(limit) ? kFewRowsAnyView : kFewRowsElsewhere;
    return plan[which].cost > limit ? kFewRowsElsewhere : which;
}

}  // namespace srt
