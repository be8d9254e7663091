// C ABI of the products with 4-bit weights: argument checks, the shape of a launch, and the making of such weights.
// Declarations are in include/srt_matmul_api.h.
#include "srt_matmul_api.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "few_rows.cuh"
#include "host_common.h"

namespace {

using namespace srt;
using namespace srt::host;

cudaError_t check_weight(const char* op, const char* what, const srtInt4Matrix* w, bool empty_ok)
{
    if (!w) return fail(cudaErrorInvalidValue, "%s: %s: missing", op, what);
    if (w->type != real16F && w->type != real16BF)
        return fail(cudaErrorNotSupported, "%s: %s: scales are Float16 or BFloat16", op, what);
    if (w->rows > 0x7fffff00ull || w->cols > 0x7fffff00ull) return fail(cudaErrorInvalidValue, "%s: %s: dimension exceeds the supported range", op, what);
    const uint32_t g = w->groupSize;
    if (g != 32 && g != 64 && (g == 0 || g % 128 != 0))
        return fail(cudaErrorInvalidValue, "%s: %s: groups are 32, 64 or a multiple of 128 rows, got %u", op, what, g);
    const bool some = w->rows != 0 && w->cols != 0;
    if (some && (!w->packed || !w->scales)) return fail(cudaErrorInvalidValue, "%s: %s: null packed or scales", op, what);
    if (!some && !empty_ok) return fail(cudaErrorInvalidValue, "%s: %s has no elements", op, what);
    if (some && (w->packedStride < (int64_t)w->cols || w->scalesStride < (int64_t)w->cols || (w->zeros && w->zerosStride < (int64_t)w->cols)))
        return fail(cudaErrorInvalidValue, "%s: %s: a stride is smaller than a row", op, what);
    return cudaSuccess;
}

cudaError_t check_matrix(const char* op, const char* what, const void* ptr, const srtTensorDescriptor* d, srtDataType type, bool written, uint64_t& rows,
                         uint64_t& cols, long long& sm, long long& sn)
{
    if (!d || !d->shape || !d->strides) return fail(cudaErrorInvalidValue, "%s: %s: missing descriptor", op, what);
    if (d->rank != 2) return fail(cudaErrorInvalidValue, "%s: %s must have rank 2", op, what);
    if (d->type != type) return fail(cudaErrorInvalidValue, "%s: %s must have the type of the weight's scales", op, what);
    rows = d->shape[0]; cols = d->shape[1];
    sm = (long long)d->strides[0]; sn = (long long)d->strides[1];
    if (rows > 0x7fffff00ull || cols > 0x7fffff00ull) return fail(cudaErrorInvalidValue, "%s: %s: dimension exceeds the supported range", op, what);
    if (!ptr && rows * cols != 0) return fail(cudaErrorInvalidValue, "%s: %s is null", op, what);
    if (written && rows * cols != 0 && ((rows > 1 && sm == 0) || (cols > 1 && sn == 0))) return fail(cudaErrorInvalidValue, "%s: %s must not repeat elements (zero stride)", op, what);
    return cudaSuccess;
}

FewRowsWeight weight_arg(const srtInt4Matrix* w)
{
    FewRowsWeight f;
    memset(&f, 0, sizeof f);
    f.w = w->packed; f.ld = w->packedStride;
    f.scales = w->scales; f.scales_ld = w->scalesStride;
    f.zeros = w->zeros; f.zeros_ld = w->zerosStride;
    // rows of words on 16 bytes, and four columns' scales on 8 and zero points on 4
    auto rows_on = [&](const void* ptr, int64_t stride, int64_t bytes, uint64_t rows, uintptr_t to) {
        return reinterpret_cast<uintptr_t>(ptr) % to == 0 && (rows <= 1 || stride * bytes % (int64_t)to == 0);
    };
    const uint64_t groups = (w->rows + w->groupSize - 1) / w->groupSize;
    f.vec = rows_on(w->packed, w->packedStride, 4, (w->rows + 7) / 8, 16) && rows_on(w->scales, w->scalesStride, 2, groups, 8) &&
            (!w->zeros || rows_on(w->zeros, w->zerosStride, 1, groups, 4));
    return f;
}

template <typename T, typename Format> constexpr bool kByColumns = std::is_same<Format, ColsFormat<T>>::value;

// the weight's tensor map, as the boxes of a stage (see few_rows_tiles_kernel)
template <typename T, typename Format>
bool encode_weight(EncodeTiledFn encode, const FewRowsParams& p, const FewRowsWeight& w, uint32_t parts, CUtensorMap* map)
{
    const bool int4 = Format::kGroups;
    const cuuint64_t elem = int4 ? 4 : 2, rows = int4 ? (p.K + 7) / 8 : p.K;
    cuuint64_t dims[3] = {p.N, rows, 1};
    cuuint32_t box[3] = {(cuuint32_t)(128 / elem), 16 * parts, 1}, unit[3] = {1, 1, 1};
    if (kByColumns<T, Format>) { dims[0] = p.K; dims[1] = p.N; box[1] = 32; }
    const cuuint64_t ld = dims[1] == 1 ? (dims[0] * elem + 15) / 16 * 16 : (cuuint64_t)w.ld * elem;
    const cuuint64_t strides[2] = {ld, ld * dims[1]};
    if (reinterpret_cast<uintptr_t>(w.w) % 16 != 0 || ld % 16 != 0 || ld < dims[0] * elem || strides[1] >= (1ull << 40)) return false;
    const CUtensorMapDataType type = int4 ? CU_TENSOR_MAP_DATA_TYPE_INT32 : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 3, const_cast<void*>(w.w), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Kernel, typename... Args>
cudaError_t launch_rows_kernel(Kernel kernel, std::atomic<uint64_t>& ready, dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t stream, const Args&... args)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {            // once per kernel and device
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewRowsSharedLimit)) != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = grid.y;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = launch_status(cudaLaunchKernelEx(&cfg, kernel, args...));
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}

template <typename T, typename Format, int NW, int NT>
cudaError_t plan_rows(const FewRowsParams& p, RowsPlan& plan)
{
    static std::atomic<uint32_t> by_registers{0};                            // CTAs that an SM's registers hold
    uint32_t most = by_registers.load(std::memory_order_relaxed);
    if (most == 0) {
        cudaFuncAttributes attributes;
        const cudaError_t e = cudaFuncGetAttributes(&attributes, few_rows_tiles_kernel<T, Format, NW, NT>);
        if (e != cudaSuccess) return e;
        most = 65536u / (((uint32_t)attributes.numRegs + 7) / 8 * 8 * kFewRowsTileThreads);
        most = most > 3 ? 3 : most < 1 ? 1 : most;
        by_registers.store(most, std::memory_order_relaxed);
    }
    plan = plan_few_rows(Format::kFormat, NW, NT, p.M, p.N, p.K, most);
    return cudaSuccess;
}

template <typename T, typename Format, int NW, int NT>
cudaError_t launch_tiles(FewRowsParams& p, const RowsPlan& plan, EncodeTiledFn encode, bool& done, cudaStream_t stream)
{
    const uint32_t row_blocks = (p.M + 8 * NT - 1) / (8 * NT), tiles = (p.N + Format::kCols - 1) / Format::kCols, parts = 8 / plan.groups;
    p.column_groups = plan.groups;
    p.stages = plan.stages;
    p.k_per_part = plan.k_per_part;
    p.x_pitch = plan.x_pitch;
    FewRowsMaps maps;
    done = row_blocks <= 65535 && encode_weight<T, Format>(encode, p, p.w[0], parts, &maps.w[0]) && encode_weight<T, Format>(encode, p, p.w[NW - 1], parts, &maps.w[1]);
    if (!done) return cudaSuccess;
    static std::atomic<uint64_t> ready{0};
    return launch_rows_kernel(few_rows_tiles_kernel<T, Format, NW, NT>, ready, dim3((tiles + plan.groups - 1) / plan.groups, plan.cluster, row_blocks), kFewRowsTileThreads,
                              plan.smem, stream, p, maps);
}

template <typename T, typename Format, int NW, int NT>
cudaError_t launch_any(FewRowsParams& p, cudaStream_t stream)
{
    const uint32_t row_blocks = (p.M + 8 * NT - 1) / (8 * NT), tiles = (p.N + Format::kCols - 1) / Format::kCols;
    if (row_blocks > 65535) return fail(cudaErrorInvalidValue, "too many rows for a product of a few rows: %u", p.M);
    const uint32_t units = (p.K + Format::kUnit - 1) / Format::kUnit;
    uint32_t cluster = 1;
    while (cluster < 8 && (uint64_t)tiles * row_blocks * cluster * 2 <= 2 * 148 && kFewRowsWarps * cluster * 2 <= units) cluster *= 2;
    p.k_per_part = (units + kFewRowsWarps * cluster - 1) / (kFewRowsWarps * cluster) * Format::kUnit;
    static std::atomic<uint64_t> ready{0};
    return launch_rows_kernel(few_rows_kernel<T, Format, NW, NT>, ready, dim3(tiles, cluster, row_blocks), 32 * kFewRowsWarps, few_rows_sum_bytes(Format::kFormat, NW, NT), stream, p);
}

// Eight, 16 or 32 rows of x to a CTA, whichever is estimated to be fastest: more rows read the weights fewer times, fewer rows have
// less of x to bring in and more CTAs to an SM (two weights' sums of 32 rows do not fit into registers).
// cudaErrorNotSupported, without text, where the caller's other way, of `limit` microseconds, is to be taken (see choose_few_rows).
template <typename T, typename Format, int NW>
cudaError_t launch_few_rows(FewRowsParams& p, double limit, int device, cudaStream_t stream)
{
    if (p.w[0].vec && p.w[NW - 1].vec) {
        TileServices services;
        cudaError_t e = tile_services(device, services);
        if (e != cudaSuccess) return e;
        p.status = services.status;
        p.wait_cycles = services.wait_cycles;
        RowsPlan plan[3];
        if ((e = plan_rows<T, Format, NW, 1>(p, plan[0])) != cudaSuccess) return e;
        if (p.M > 8 && (e = plan_rows<T, Format, NW, 2>(p, plan[1])) != cudaSuccess) return e;
        if constexpr (NW == 1)
            if (p.M > 16 && (e = plan_rows<T, Format, NW, 4>(p, plan[2])) != cudaSuccess) return e;
        bool done = false;
        const int which = choose_few_rows(plan, limit);
        if (which == kFewRowsElsewhere) return cudaErrorNotSupported;
        if (which == 0) e = launch_tiles<T, Format, NW, 1>(p, plan[0], services.encode, done, stream);
        else if (which == 1) e = launch_tiles<T, Format, NW, 2>(p, plan[1], services.encode, done, stream);
        if constexpr (NW == 1)
            if (which == 2) e = launch_tiles<T, Format, NW, 4>(p, plan[2], services.encode, done, stream);
        if (done || e != cudaSuccess) return e;
    }
    return p.M <= 8 ? launch_any<T, Format, NW, 1>(p, stream) : launch_any<T, Format, NW, 2>(p, stream);
}

template <typename T, int NW>
cudaError_t launch_int4(FewRowsParams& p, int device, cudaStream_t stream)
{
    if (p.group == 32) return launch_few_rows<T, Int4Format<T, 4>, NW>(p, HUGE_VAL, device, stream);
    if (p.group == 64) return launch_few_rows<T, Int4Format<T, 2>, NW>(p, HUGE_VAL, device, stream);
    return launch_few_rows<T, Int4Format<T, 1>, NW>(p, HUGE_VAL, device, stream);
}

cudaError_t run_int4(const char* op, const void* x, const srtTensorDescriptor* xDesc, const srtInt4Matrix* w0, const srtInt4Matrix* w1, const void* bias0,
                     const srtTensorDescriptor* bias0Desc, const void* bias1, const srtTensorDescriptor* bias1Desc, srtActivationType activation,
                     void* out, const srtTensorDescriptor* outDesc, cudaStream_t stream)
{
    cudaError_t e = check_weight(op, w1 ? "wGate" : "weight", w0, true);
    if (e != cudaSuccess) return e;
    if (w1) {
        if ((e = check_weight(op, "wUp", w1, true)) != cudaSuccess) return e;
        if (w1->type != w0->type || w1->rows != w0->rows || w1->cols != w0->cols || w1->groupSize != w0->groupSize)
            return fail(cudaErrorInvalidValue, "%s: wGate and wUp must have one type, shape and group size", op);
    }
    const srtDataType type = w0->type;
    uint64_t M, K, m2, N;
    FewRowsParams p;
    memset(&p, 0, sizeof p);
    if ((e = check_matrix(op, "x", x, xDesc, type, false, M, K, p.x_m, p.x_k)) != cudaSuccess ||
        (e = check_matrix(op, "out", out, outDesc, type, true, m2, N, p.o_m, p.o_n)) != cudaSuccess)
        return e;
    if (K != w0->rows) return fail(cudaErrorInvalidValue, "%s: inner dimensions must be equal (%llu vs %llu)", op, (unsigned long long)K, (unsigned long long)w0->rows);
    if (m2 != M || N != w0->cols)
        return fail(cudaErrorInvalidValue, "%s: out must be [%llu x %llu]", op, (unsigned long long)M, (unsigned long long)w0->cols);
    if (K == 0) return fail(cudaErrorInvalidValue, "%s: a weight without rows", op);
    p.w[0] = weight_arg(w0);
    p.w[1] = w1 ? weight_arg(w1) : p.w[0];
    const void* bias[2] = {bias0, bias1};
    const srtTensorDescriptor* bd[2] = {bias0Desc, bias1Desc};
    for (int i = 0; i < 2; ++i) {
        if (!bias[i]) continue;
        if (!bd[i] || !bd[i]->shape || !bd[i]->strides || bd[i]->rank != 1 || bd[i]->shape[0] != N || bd[i]->type != type)
            return fail(cudaErrorInvalidValue, "%s: a bias must be rank 1 with %llu elements of x's type", op, (unsigned long long)N);
        p.w[i].bias = bias[i];
        p.w[i].bias_n = (long long)bd[i]->strides[0];
    }
    switch ((int)activation) {
    case srtActivationSigmoid: case srtActivationRelu: case srtActivationTanh: case srtActivationIdentity:
    case srtActivationGelu: case srtActivationGeluTanh: case srtActivationSilu: break;
    case srtActivationClippedRelu: case srtActivationElu:
        return fail(cudaErrorNotSupported, "%s: clippedRelu and elu need coefficients that this entry point does not carry", op);
    default: return fail(cudaErrorInvalidValue, "%s: unknown activation %d", op, (int)activation);
    }
    g_error[0] = 0;
    if (M == 0 || N == 0) return cudaSuccess;
    p.x = x; p.out = out;
    p.x_vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && p.x_k == 1 && (M == 1 || p.x_m % 8 == 0);
    p.M = (uint32_t)M; p.N = (uint32_t)N; p.K = (uint32_t)K;
    p.group = w0->groupSize;
    p.by_group = make_fast_div(p.group);
    p.act = (uint32_t)activation;
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    const int device = scope.device;
    if (type == real16F) return w1 ? launch_int4<__half, 2>(p, device, stream) : launch_int4<__half, 1>(p, device, stream);
    return w1 ? launch_int4<__nv_bfloat16, 2>(p, device, stream) : launch_int4<__nv_bfloat16, 1>(p, device, stream);
}

template <typename T>
cudaError_t launch_gated_rows(FewRowsParams& p, bool k_contiguous, double limit, int device, cudaStream_t stream)
{
    return k_contiguous ? launch_few_rows<T, ColsFormat<T>, 2>(p, limit, device, stream) : launch_few_rows<T, RowsFormat<T>, 2>(p, limit, device, stream);
}

}  // namespace

namespace srt {
namespace host {

// the gated product of a few rows with 16-bit weights (srtMatmulGated)
cudaError_t gated_few_rows(srtDataType type, const FewRowsParams& params, bool k_contiguous, double limit, int device, cudaStream_t stream)
{
    FewRowsParams p = params;
    return type == real16F ? launch_gated_rows<__half>(p, k_contiguous, limit, device, stream) : launch_gated_rows<__nv_bfloat16>(p, k_contiguous, limit, device, stream);
}

}  // namespace host
}  // namespace srt

extern "C" {

cudaError_t srtMatmulInt4(const void* x, const srtTensorDescriptor* xDesc, const srtInt4Matrix* weight, const void* bias, const srtTensorDescriptor* biasDesc,
                          srtActivationType activation, void* out, const srtTensorDescriptor* outDesc, cudaStream_t stream)
{
    return run_int4("srtMatmulInt4", x, xDesc, weight, nullptr, bias, biasDesc, nullptr, nullptr, activation, out, outDesc, stream);
}

cudaError_t srtMatmulGatedInt4(const void* x, const srtTensorDescriptor* xDesc, const srtInt4Matrix* wGate, const srtInt4Matrix* wUp, const void* biasGate,
                               const srtTensorDescriptor* biasGateDesc, const void* biasUp, const srtTensorDescriptor* biasUpDesc,
                               srtActivationType activation, void* out, const srtTensorDescriptor* outDesc, cudaStream_t stream)
{
    if (!wUp) return fail(cudaErrorInvalidValue, "srtMatmulGatedInt4: wUp: missing");
    return run_int4("srtMatmulGatedInt4", x, xDesc, wGate, wUp, biasGate, biasGateDesc, biasUp, biasUpDesc, activation, out, outDesc, stream);
}

cudaError_t srtQuantizeInt4(const void* w, const srtTensorDescriptor* wDesc, const srtInt4Matrix* weight, cudaStream_t stream)
{
    const char* const op = "srtQuantizeInt4";
    cudaError_t e = check_weight(op, "weight", weight, true);
    if (e != cudaSuccess) return e;
    Int4QuantizeParams p;
    uint64_t K, N;
    if ((e = check_matrix(op, "w", w, wDesc, weight->type, false, K, N, p.w_k, p.w_n)) != cudaSuccess) return e;
    if (K != weight->rows || N != weight->cols)
        return fail(cudaErrorInvalidValue, "%s: w must be [%llu x %llu]", op, (unsigned long long)weight->rows, (unsigned long long)weight->cols);
    g_error[0] = 0;
    if (K == 0 || N == 0) return cudaSuccess;
    const uint64_t groups = (K + weight->groupSize - 1) / weight->groupSize;
    if (groups > 65535) return fail(cudaErrorInvalidValue, "%s: %llu groups exceed the supported range", op, (unsigned long long)groups);
    p.w = w;
    p.words = reinterpret_cast<uint32_t*>(const_cast<int32_t*>(weight->packed)); p.words_ld = weight->packedStride;
    p.scales = const_cast<void*>(weight->scales); p.scales_ld = weight->scalesStride;
    p.zeros = const_cast<uint8_t*>(weight->zeros); p.zeros_ld = weight->zerosStride;
    p.K = (uint32_t)K; p.N = (uint32_t)N; p.group = weight->groupSize;
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    const dim3 grid((p.N + 127) / 128, (unsigned)groups, 1);
    if (weight->type == real16F) int4_quantize_kernel<__half><<<grid, 128, 0, stream>>>(p);
    else                         int4_quantize_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    e = cudaGetLastError();
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}

cudaError_t srtDequantizeInt4(const srtInt4Matrix* weight, void* out, const srtTensorDescriptor* outDesc, cudaStream_t stream)
{
    const char* const op = "srtDequantizeInt4";
    cudaError_t e = check_weight(op, "weight", weight, true);
    if (e != cudaSuccess) return e;
    Int4DequantizeParams p;
    uint64_t K, N;
    if ((e = check_matrix(op, "out", out, outDesc, weight->type, true, K, N, p.o_k, p.o_n)) != cudaSuccess) return e;
    if (K != weight->rows || N != weight->cols)
        return fail(cudaErrorInvalidValue, "%s: out must be [%llu x %llu]", op, (unsigned long long)weight->rows, (unsigned long long)weight->cols);
    g_error[0] = 0;
    if (K == 0 || N == 0) return cudaSuccess;
    p.w = weight_arg(weight);
    p.out = out;
    p.K = (uint32_t)K; p.N = (uint32_t)N; p.group = weight->groupSize;
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    const uint32_t word_rows = (p.K + 7) / 8;
    const dim3 grid((p.N + 127) / 128, word_rows < 65535 ? word_rows : 65535, 1);
    if (weight->type == real16F) int4_dequantize_kernel<__half><<<grid, 128, 0, stream>>>(p);
    else                         int4_dequantize_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    e = cudaGetLastError();
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}

}  // extern "C"
