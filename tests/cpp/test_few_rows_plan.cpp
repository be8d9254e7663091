// Host check of the plans of few-row products (few_rows_plan.h): over a grid of rows, reductions and columns, every plan of every
// kernel asks for no more shared memory than the kernels are allowed, holds what it is meant to hold, and covers K.
#include <cstdio>
#include <initializer_list>

#include "few_rows_plan.h"

using namespace srt;

static long g_failures = 0, g_plans = 0;

static void expect(bool ok, const char* what, const char* format, uint32_t nw, uint32_t nt, uint32_t M, uint32_t K, uint32_t N, uint32_t most, const RowsPlan& p)
{
    if (ok) return;
    if (++g_failures <= 20)
        printf("%s: %s, %u weights, %u rows a CTA, %u x %u x %u, %u CTAs an SM: groups %u cluster %u stages %u, %u bytes\n", what, format, nw, 8 * nt, M, K, N, most,
               p.groups, p.cluster, p.stages, p.smem);
}

int main()
{
    struct Kernel { const char* name; FewRowsFormat f; uint32_t nw, nt; };
    const Kernel kernels[] = {{"4-bit", kInt4Weights, 1, 1}, {"4-bit", kInt4Weights, 1, 2}, {"4-bit", kInt4Weights, 1, 4}, {"4-bit", kInt4Weights, 2, 1},
                              {"4-bit", kInt4Weights, 2, 2}, {"rows", kRowWeights, 2, 1}, {"rows", kRowWeights, 2, 2}, {"columns", kColumnWeights, 2, 1},
                              {"columns", kColumnWeights, 2, 2}};
    for (const Kernel& k : kernels) {
        // the kernel without tiles holds its sums only
        if (few_rows_sum_bytes(k.f, k.nw, k.nt) > kFewRowsSharedLimit) ++g_failures, printf("the sums of %s do not fit\n", k.name);
        for (uint32_t M : {1, 2, 7, 8, 9, 12, 13, 15, 16, 17, 24, 25, 31, 32, 33, 40, 48, 63, 64, 70, 100, 128, 200, 256, 509, 512})
            for (uint32_t K : {64, 100, 129, 256, 500, 1024, 1111, 2048, 2500, 3200, 4096, 5000, 6144, 6400, 7168, 8192, 8200, 10240, 11008, 12288, 14336, 16384, 20000, 24576,
                               24816, 28672, 32768, 50000, 65536, 100000, 110000, 131072})
                for (uint32_t N : {64, 100, 512, 1001, 2048, 4096, 5000, 8192, 12288, 14336, 16384, 24576, 28672, 30976, 40408, 65536, 128256, 262144})
                    for (uint32_t most = 1; most <= 3; ++most) {
                        const RowsPlan p = plan_few_rows(k.f, k.nw, k.nt, M, N, K, most);
                        const auto check = [&](bool ok, const char* what) { expect(ok, what, k.name, k.nw, k.nt, M, K, N, most, p); };
                        const uint32_t x_rows = M < 8 * k.nt ? M : 8 * k.nt;
                        // a row of x of an eighth of K and one stage: a plan is missing only where these or the sums exceed the limit
                        if (p.groups == 0) {
                            check(p.cost >= 1e300, "no plan has a cost");
                            const uint64_t x_min = (uint64_t)x_rows * ((K / 8 + 8 * k.f.warp_rows) * 2 + 256);
                            check(few_rows_tiles_smem(k.f, k.nw, k.nt, 1, x_min) + 4096 > kFewRowsSharedLimit, "no plan for a small product");
                            continue;
                        }
                        ++g_plans;
                        const uint32_t stage_rows = 8 / p.groups * k.f.warp_rows, ring = p.stages * k.nw * kFewRowsStageBytes;
                        check(p.smem <= kFewRowsSharedLimit, "more shared memory than allowed");
                        check(p.smem >= 1024 + ring + x_rows * p.x_pitch && p.smem >= 1024 + few_rows_sum_bytes(k.f, k.nw, k.nt) + x_rows * p.x_pitch, "less than ring, sums and x");
                        check(p.x_pitch >= 2 * p.k_per_part && p.x_pitch % 16 == 0, "rows of x overlap");
                        check(p.stages >= 1 && p.stages <= kFewRowsMaxStages && p.cluster >= 1 && p.cluster <= 8 && p.groups <= k.f.max_column_groups, "a launch that the kernel does not know");
                        check(p.k_per_part % stage_rows == 0 && (uint64_t)p.k_per_part * p.cluster >= K, "K is not covered");
                    }
    }
    // which of three plans runs: no plan leads to the kernel that takes any view unless the caller has another way
    const auto chosen = [](double a, double b, double c, double limit) {
        RowsPlan plan[3];
        const double cost[3] = {a, b, c};
        for (int i = 0; i < 3; ++i)
            if (cost[i] > 0) plan[i].cost = cost[i], plan[i].groups = 1;
        return choose_few_rows(plan, limit);
    };
    const bool choices = chosen(3, 0, 0, HUGE_VAL) == 0 && chosen(3, 2, 0, HUGE_VAL) == 1 && chosen(3, 2, 1, 1e299) == 2 && chosen(0, 0, 1, HUGE_VAL) == 2 &&
                         chosen(3, 2, 4, 1.5) == kFewRowsElsewhere && chosen(0, 0, 0, 1.5) == kFewRowsElsewhere && chosen(0, 0, 0, 1e299) == kFewRowsElsewhere &&
                         chosen(0, 0, 0, HUGE_VAL) == kFewRowsAnyView;
    const RowsPlan none[3] = {plan_few_rows(kInt4Weights, 1, 1, 8, 4096, 131072, 3), plan_few_rows(kInt4Weights, 1, 2, 8, 4096, 131072, 3), RowsPlan{}};
    if (!choices || choose_few_rows(none, HUGE_VAL) != kFewRowsAnyView) ++g_failures, printf("a wrong choice\n");
    printf("%ld plans, %ld failures\n", g_plans, g_failures);
    return g_failures != 0 || g_plans == 0;
}
