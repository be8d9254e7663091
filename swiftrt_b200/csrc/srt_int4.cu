// C ABI of the products with 4-bit weights: argument checks, the shape of a launch, and the making of such weights.
// Declarations are in include/srt_matmul_api.h.
#include "srt_matmul_api.h"

#include <cuda_runtime.h>

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
    // four columns at a time: 16 bytes of words, 8 of scales, 4 of zero points
    f.vec = w->cols % 4 == 0 && w->packedStride % 4 == 0 && w->scalesStride % 4 == 0 && reinterpret_cast<uintptr_t>(w->packed) % 16 == 0 &&
            reinterpret_cast<uintptr_t>(w->scales) % 8 == 0 && (!w->zeros || (w->zerosStride % 4 == 0 && reinterpret_cast<uintptr_t>(w->zeros) % 4 == 0));
    return f;
}

template <typename T, typename Format, int NW, int NT>
cudaError_t launch_few_rows(FewRowsParams& p, cudaStream_t stream)
{
    const uint32_t batches = (p.K + Format::kBatch - 1) / Format::kBatch, row_blocks = (p.M + 8 * NT - 1) / (8 * NT);
    const uint32_t tiles = (p.N + Format::kCols - 1) / Format::kCols;
    if (row_blocks > 65535) return fail(cudaErrorInvalidValue, "too many rows for a product of a few rows: %u", p.M);
    p.warps_n = 1;
    // Four warps to a column tile where there are tiles for every SM, else eight, and parts of K beyond them (a cluster) while the
    // CTAs do not fill the device twice and a warp still has a batch of its own.
    const uint32_t warps = (uint64_t)tiles * row_blocks >= 2 * 148 ? 4 : 8;
    uint32_t parts = 1;
    while (parts < 8 && (uint64_t)tiles * row_blocks * parts * 2 <= 2 * 148 && warps * parts * 2 <= batches) parts *= 2;
    const uint32_t workers = warps / p.warps_n * parts;
    p.k_per_warp = (batches + workers - 1) / workers * Format::kBatch;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3((tiles + p.warps_n - 1) / p.warps_n, parts, row_blocks);
    cfg.blockDim = dim3(32 * warps, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = parts;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, few_rows_kernel<T, Format, NW, NT>, p);
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}

template <typename T, int GPB, int NW>
cudaError_t launch_int4_rows(FewRowsParams& p, cudaStream_t stream)
{
    if (p.M <= 8) return launch_few_rows<T, Int4Format<T, GPB>, NW, 1>(p, stream);
    // (two weights' sums of 32 rows do not fit into registers)
    if (p.M <= 16 || NW == 2) return launch_few_rows<T, Int4Format<T, GPB>, NW, 2>(p, stream);
    return launch_few_rows<T, Int4Format<T, GPB>, 1, 4>(p, stream);
}

template <typename T, int NW>
cudaError_t launch_int4_groups(FewRowsParams& p, cudaStream_t stream)
{
    if (p.group == 32) return launch_int4_rows<T, 4, NW>(p, stream);
    if (p.group == 64) return launch_int4_rows<T, 2, NW>(p, stream);
    return launch_int4_rows<T, 1, NW>(p, stream);
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
    p.act = (uint32_t)activation;
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    if (type == real16F) return w1 ? launch_int4_groups<__half, 2>(p, stream) : launch_int4_groups<__half, 1>(p, stream);
    return w1 ? launch_int4_groups<__nv_bfloat16, 2>(p, stream) : launch_int4_groups<__nv_bfloat16, 1>(p, stream);
}

template <typename T>
cudaError_t launch_gated_rows(FewRowsParams& p, bool k_contiguous, cudaStream_t stream)
{
    if (k_contiguous) return p.M <= 8 ? launch_few_rows<T, ColsFormat<T>, 2, 1>(p, stream) : launch_few_rows<T, ColsFormat<T>, 2, 2>(p, stream);
    return p.M <= 8 ? launch_few_rows<T, RowsFormat<T>, 2, 1>(p, stream) : launch_few_rows<T, RowsFormat<T>, 2, 2>(p, stream);
}

}  // namespace

namespace srt {
namespace host {

// the gated product of a few rows with 16-bit weights (srtMatmulGated)
cudaError_t gated_few_rows(srtDataType type, const FewRowsParams& params, bool k_contiguous, cudaStream_t stream)
{
    FewRowsParams p = params;
    return type == real16F ? launch_gated_rows<__half>(p, k_contiguous, stream) : launch_gated_rows<__nv_bfloat16>(p, k_contiguous, stream);
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
