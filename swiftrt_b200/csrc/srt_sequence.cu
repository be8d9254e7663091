// C ABI of the recurrence over whole sequences: argument checks and launches.  Declarations are in
// include/srt_matmul_api.h.
#include "srt_matmul_api.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "gated_recurrence.cuh"
#include "host_common.h"

namespace {

using namespace srt;
using namespace srt::host;

struct Shape3 { uint64_t B, T, D; };

// rank 3 [batch x steps x channels], or rank 2 [batch x channels] for one step
cudaError_t shape3(const char* op, const char* what, const srtTensorDescriptor* d, Shape3& s, long long (&strides)[3])
{
    if (!d || !d->shape || !d->strides) return fail(cudaErrorInvalidValue, "%s: %s: missing descriptor", op, what);
    if (d->rank != 2 && d->rank != 3) return fail(cudaErrorInvalidValue, "%s: %s must have rank 3, or rank 2 for one step", op, what);
    const uint32_t last = d->rank - 1;
    s.B = d->shape[0];
    s.T = d->rank == 3 ? d->shape[1] : 1;
    s.D = d->shape[last];
    strides[0] = (long long)d->strides[0];
    strides[1] = d->rank == 3 ? (long long)d->strides[1] : 0;
    strides[2] = (long long)d->strides[last];
    return cudaSuccess;
}

cudaError_t sequence_arg(const char* op, const char* what, const void* ptr, const srtTensorDescriptor* d, srtDataType type, const Shape3& want,
                         bool written, long long (&strides)[3])
{
    Shape3 s;
    cudaError_t e = shape3(op, what, d, s, strides);
    if (e != cudaSuccess) return e;
    if (d->type != type) return fail(cudaErrorInvalidValue, "%s: %s must have the element type of update", op, what);
    if (s.B != want.B || s.T != want.T || s.D != want.D)
        return fail(cudaErrorInvalidValue, "%s: %s must be [%llu x %llu x %llu] like update", op, what, (unsigned long long)want.B,
                    (unsigned long long)want.T, (unsigned long long)want.D);
    if (!ptr && s.B * s.T * s.D != 0) return fail(cudaErrorInvalidValue, "%s: %s is null", op, what);
    if (written && s.B * s.T * s.D != 0 && ((s.B > 1 && strides[0] == 0) || (s.T > 1 && strides[1] == 0) || (s.D > 1 && strides[2] == 0)))
        return fail(cudaErrorInvalidValue, "%s: %s must not repeat elements (zero stride)", op, what);
    return cudaSuccess;
}

cudaError_t read_arg(const char* op, const char* what, const void* ptr, const srtTensorDescriptor* d, srtDataType type, const Shape3& want, Strided3& out)
{
    long long st[3];
    cudaError_t e = sequence_arg(op, what, ptr, d, type, want, false, st);
    if (e == cudaSuccess) out = Strided3{ptr, st[0], st[1], st[2]};
    return e;
}

cudaError_t write_arg(const char* op, const char* what, void* ptr, const srtTensorDescriptor* d, srtDataType type, const Shape3& want, Strided3W& out)
{
    long long st[3];
    cudaError_t e = sequence_arg(op, what, ptr, d, type, want, true, st);
    if (e == cudaSuccess) out = Strided3W{ptr, st[0], st[1], st[2]};
    return e;
}

// a Float32 state [batch x channels]
cudaError_t state_arg(const char* op, const char* what, const srtTensorDescriptor* d, const Shape3& want, bool written, long long& sb, long long& sd)
{
    if (!d || !d->shape || !d->strides) return fail(cudaErrorInvalidValue, "%s: %s: missing descriptor", op, what);
    if (d->type != real32F || d->rank != 2 || d->shape[0] != want.B || d->shape[1] != want.D)
        return fail(cudaErrorInvalidValue, "%s: %s must be Float32 [%llu x %llu]", op, what, (unsigned long long)want.B, (unsigned long long)want.D);
    sb = (long long)d->strides[0];
    sd = (long long)d->strides[1];
    if (written && ((want.B > 1 && sb == 0) || (want.D > 1 && sd == 0)))
        return fail(cudaErrorInvalidValue, "%s: %s must not repeat elements (zero stride)", op, what);
    return cudaSuccess;
}

cudaError_t states_arg(const char* op, const srtTensorDescriptor* d, const Shape3& want, bool written, RecurrenceParams& p)
{
    const uint64_t chunks = (want.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    if (!d || !d->shape || !d->strides) return fail(cudaErrorInvalidValue, "%s: states: missing descriptor", op);
    if (d->type != real32F || d->rank != 3 || d->shape[0] != want.B || d->shape[1] != chunks || d->shape[2] != want.D)
        return fail(cudaErrorInvalidValue, "%s: states must be Float32 [%llu x %llu x %llu]", op, (unsigned long long)want.B,
                    (unsigned long long)chunks, (unsigned long long)want.D);
    p.states_b = (long long)d->strides[0];
    p.states_c = (long long)d->strides[1];
    p.states_d = (long long)d->strides[2];
    if (written && ((want.B > 1 && p.states_b == 0) || (chunks > 1 && p.states_c == 0) || (want.D > 1 && p.states_d == 0)))
        return fail(cudaErrorInvalidValue, "%s: states must not repeat elements (zero stride)", op);
    return cudaSuccess;
}

// type and extents of the call, from `update`
cudaError_t recurrence_shape(const char* op, const srtTensorDescriptor* updateDesc, Shape3& s, RecurrenceParams& p)
{
    long long st[3];
    cudaError_t e = shape3(op, "update", updateDesc, s, st);
    if (e != cudaSuccess) return e;
    if (elem_size(updateDesc->type) == 0)
        return fail(cudaErrorNotSupported, "%s: element type %d is not computed by this library", op, (int)updateDesc->type);
    if (s.B > 65535 || s.T > 0x7fffffffull || s.D > 0x7fffffffull)
        return fail(cudaErrorInvalidValue, "%s: dimension exceeds the supported range", op);
    memset(&p, 0, sizeof p);
    p.B = (uint32_t)s.B;
    p.T = (uint32_t)s.T;
    p.D = (uint32_t)s.D;
    return cudaSuccess;
}

template <typename Kernel, typename Maps>
cudaError_t launch_spans_kernel(Kernel kernel, const Maps& maps, std::atomic<uint64_t>* ready, uint32_t smem, const RecurrenceParams& p, uint32_t channels,
                                cudaStream_t stream)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready->load(std::memory_order_acquire) & bit)) {            // once per kernel and device
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return e;
        ready->fetch_or(bit, std::memory_order_release);
    }
    const uint32_t blocks_d = (p.D + channels - 1) / channels, chunks = (p.T + kRecurrenceChunk - 1) / kRecurrenceChunk;
    const uint64_t blocks = (uint64_t)p.B * blocks_d;
    // Spans of one item and channel block side by side while their CTAs find a place at once, three to an SM less what clusters
    // leave free: a CTA alone on its SM waits for its own latencies.  Forward / backward in us of 2048 steps, bf16, with 1, 2, 4
    // and 8 CTAs a cluster: 40 blocks 42/76 29/47 21/33 17/34; 55 blocks 41/78 29/47 21/37 23/39; 104 blocks 44/78 37/64 29/58
    // 38/68; 130 blocks 43/80 39/64 39/70 45/79; 222 blocks 62/111 52/105 62/117 71/129; 256 blocks forward 63 79 76 86.
    uint32_t cluster = 1;
    while (cluster < 8 && cluster < chunks && blocks * cluster * 2 <= 148 * 3 - 28 * (cluster - 1)) cluster *= 2;
    if (blocks * cluster > 0x7fffffffull) return fail(cudaErrorInvalidValue, "too many channels for one call");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3((unsigned)(blocks * cluster), 1, 1);
    cfg.blockDim = dim3(kSpanThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launch_status(cudaLaunchKernelEx(&cfg, kernel, p, maps, blocks_d, cluster));
}

template <typename T, bool HAS_I, bool HAS_O, int VEC, int SRC>
cudaError_t launch_spans(const RecurrenceParams& p, const typename MapsOf<SRC>::type& maps, bool backward, cudaStream_t stream)
{
    static std::atomic<uint64_t> ready[2];
    constexpr uint32_t kInputs = 2 + HAS_I + HAS_O;
    return backward ? launch_spans_kernel(recurrence_span_backward_kernel<T, HAS_I, HAS_O, VEC, SRC>, maps, &ready[1],
                                          span_smem_bytes<T, VEC, SRC>(kInputs + 1, 0), p, 32 * VEC, stream)
                    : launch_spans_kernel(recurrence_span_kernel<T, HAS_I, HAS_O, VEC, SRC>, maps, &ready[0],
                                          span_smem_bytes<T, VEC, SRC>(kInputs, 1), p, 32 * VEC, stream);
}

template <typename T, int VEC, int SRC>
cudaError_t launch_spans_gates(const RecurrenceParams& p, const typename MapsOf<SRC>::type& maps, bool backward, cudaStream_t stream)
{
    if (p.i.p) return p.o.p ? launch_spans<T, true, true, VEC, SRC>(p, maps, backward, stream) : launch_spans<T, true, false, VEC, SRC>(p, maps, backward, stream);
    return p.o.p ? launch_spans<T, false, true, VEC, SRC>(p, maps, backward, stream) : launch_spans<T, false, false, VEC, SRC>(p, maps, backward, stream);
}

template <typename T> constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
template <> constexpr CUtensorMapDataType kMapType<__half> = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
template <> constexpr CUtensorMapDataType kMapType<__nv_bfloat16> = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;

// Tensor maps of every tensor of the call, boxes of 128 bytes of channels by 64 steps (inputs) or 8 steps (results); false when one
// cannot have it: rows that do not start on 16 bytes, channels apart from each other, repeated or overlapping rows; or channels
// that end inside 16 bytes, which the boxes of the results would write whole.
template <typename T>
bool encode_maps(const RecurrenceParams& p, EncodeTiledFn encode, RecurrenceMaps& maps)
{
    auto one = [&](const void* ptr, long long b, long long t, long long d, uint32_t steps, CUtensorMap* map) {
        if (!ptr) return true;
        const long long elem = sizeof(T);
        if (p.D * elem % 16 != 0) return false;
        if (p.T == 1) t = (long long)(p.D + 7) / 8 * 8;
        if (p.B == 1) b = t;
        if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0 || (d != 1 && p.D > 1) || t < (long long)p.D || b <= 0 || t * elem % 16 != 0 || b * elem % 16 != 0 ||
            t * elem >= (1ll << 40) || b * elem >= (1ll << 40))
            return false;
        const cuuint64_t dims[3] = {p.D, p.T, p.B}, strides[2] = {(cuuint64_t)(t * elem), (cuuint64_t)(b * elem)};
        const cuuint32_t box[3] = {(cuuint32_t)(128 / elem), steps, 1}, unit[3] = {1, 1, 1};
        return encode(map, kMapType<T>, 3, const_cast<void*>(ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    auto in = [&](const Strided3& s, CUtensorMap* map) { return one(s.p, s.b, s.t, s.d, kRecurrenceChunk, map); };
    auto out = [&](const Strided3W& s, CUtensorMap* map) { return one(s.p, s.b, s.t, s.d, kSpanSteps, map); };
    return in(p.f, &maps.f) && in(p.x, &maps.x) && in(p.i, &maps.i) && in(p.o, &maps.o) && in(p.dy, &maps.dy) && out(p.y, &maps.y) && out(p.dx, &maps.dx) &&
           out(p.df, &maps.df) && out(p.di, &maps.di) && out(p.dout, &maps.dout);
}

template <typename T>
cudaError_t launch_recurrence(RecurrenceParams& p, bool backward, int device, cudaStream_t stream)
{
    cudaError_t e;
    if (p.T <= kFewSteps) {
        const unsigned long long threads = (unsigned long long)p.B * p.D;
        const unsigned blocks = (unsigned)((threads + 127) / 128);
        if (backward) recurrence_steps_backward_kernel<T><<<blocks, 128, 0, stream>>>(p);
        else          recurrence_steps_kernel<T><<<blocks, 128, 0, stream>>>(p);
        e = cudaGetLastError();
    } else {
        TileServices services;
        if ((e = tile_services(device, services)) != cudaSuccess) return e;
        p.status = services.status;
        p.wait_cycles = services.wait_cycles;
        RecurrenceMaps maps;
        memset(&maps, 0, sizeof maps);
        // two 16-bit channels per access where every tensor has them side by side and aligned (Float32 gains more from twice the CTAs: 3 x 1025 x
        // 1002, all gates, 25 / 54 us one by one, 35 / 66 in pairs; 8 x 2048 x 2046 144 / 266 and 173 / 243)
        bool pairs = sizeof(T) == 2 && p.D % 2 == 0;
        auto look = [&](const void* ptr, long long b, long long t, long long d) {
            pairs = pairs && (!ptr || (reinterpret_cast<uintptr_t>(ptr) % (2 * sizeof(T)) == 0 && d == 1 && b % 2 == 0 && t % 2 == 0));
        };
        for (const Strided3* s : {&p.x, &p.f, &p.i, &p.o, &p.dy}) look(s->p, s->b, s->t, s->d);
        for (const Strided3W* s : {&p.y, &p.dx, &p.df, &p.di, &p.dout}) look(s->p, s->b, s->t, s->d);
        constexpr int kPair = sizeof(T) == 2 ? 2 : 1;
        if (encode_maps<T>(p, services.encode, maps)) e = launch_spans_gates<T, kPair, kFromTiles>(p, maps, backward, stream);
        else if (pairs || sizeof(T) == 4) e = launch_spans_gates<T, kPair, kFromWords>(p, NoMaps{}, backward, stream);
        else {
            if constexpr (sizeof(T) == 2) e = launch_spans_gates<T, 1, kFromMemory>(p, NoMaps{}, backward, stream);
        }
    }
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}

cudaError_t launch_recurrence_type(srtDataType type, RecurrenceParams& p, bool backward, int device, cudaStream_t stream)
{
    switch (type) {
    case real32F: return launch_recurrence<float>(p, backward, device, stream);
    case real16F: return launch_recurrence<__half>(p, backward, device, stream);
    default: return launch_recurrence<__nv_bfloat16>(p, backward, device, stream);
    }
}

}  // namespace

extern "C" {

cudaError_t srtGatedRecurrence(const void* update, const srtTensorDescriptor* updateDesc, const void* forget, const srtTensorDescriptor* forgetDesc,
                               const void* input, const srtTensorDescriptor* inputDesc, const void* output, const srtTensorDescriptor* outputDesc,
                               const void* initial, const srtTensorDescriptor* initialDesc, const int32_t* lengths,
                               void* hidden, const srtTensorDescriptor* hiddenDesc, void* last, const srtTensorDescriptor* lastDesc,
                               void* states, const srtTensorDescriptor* statesDesc, cudaStream_t stream)
{
    const char* const op = "srtGatedRecurrence";
    RecurrenceParams p;
    Shape3 s;
    cudaError_t e = recurrence_shape(op, updateDesc, s, p);
    if (e != cudaSuccess) return e;
    const srtDataType type = updateDesc->type;
    if ((e = read_arg(op, "update", update, updateDesc, type, s, p.x)) != cudaSuccess) return e;
    if ((e = read_arg(op, "forget", forget, forgetDesc, type, s, p.f)) != cudaSuccess) return e;
    if (input && (e = read_arg(op, "input", input, inputDesc, type, s, p.i)) != cudaSuccess) return e;
    if (output && (e = read_arg(op, "output", output, outputDesc, type, s, p.o)) != cudaSuccess) return e;
    if ((e = write_arg(op, "hidden", hidden, hiddenDesc, type, s, p.y)) != cudaSuccess) return e;
    if (initial && (e = state_arg(op, "initial", initialDesc, s, false, p.initial_b, p.initial_d)) != cudaSuccess) return e;
    if (last && (e = state_arg(op, "last", lastDesc, s, true, p.last_b, p.last_d)) != cudaSuccess) return e;
    if (states && (e = states_arg(op, statesDesc, s, true, p)) != cudaSuccess) return e;
    g_error[0] = 0;
    if (s.B == 0 || s.D == 0 || (s.T == 0 && !last)) return cudaSuccess;
    p.initial = static_cast<const float*>(initial);
    p.lengths = lengths;
    p.last = static_cast<float*>(last);
    p.states = static_cast<float*>(states);
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    return launch_recurrence_type(type, p, false, scope.device, stream);
}

cudaError_t srtGatedRecurrenceBackward(const void* outGrad, const srtTensorDescriptor* outGradDesc, const void* lastGrad, const srtTensorDescriptor* lastGradDesc,
                                       const void* update, const srtTensorDescriptor* updateDesc, const void* forget, const srtTensorDescriptor* forgetDesc,
                                       const void* input, const srtTensorDescriptor* inputDesc, const void* output, const srtTensorDescriptor* outputDesc,
                                       const void* states, const srtTensorDescriptor* statesDesc, const int32_t* lengths,
                                       void* dUpdate, const srtTensorDescriptor* dUpdateDesc, void* dForget, const srtTensorDescriptor* dForgetDesc,
                                       void* dInput, const srtTensorDescriptor* dInputDesc, void* dOutput, const srtTensorDescriptor* dOutputDesc,
                                       void* dInitial, const srtTensorDescriptor* dInitialDesc, cudaStream_t stream)
{
    const char* const op = "srtGatedRecurrenceBackward";
    RecurrenceParams p;
    Shape3 s;
    cudaError_t e = recurrence_shape(op, updateDesc, s, p);
    if (e != cudaSuccess) return e;
    const srtDataType type = updateDesc->type;
    if ((e = read_arg(op, "outGrad", outGrad, outGradDesc, type, s, p.dy)) != cudaSuccess) return e;
    if ((e = read_arg(op, "update", update, updateDesc, type, s, p.x)) != cudaSuccess) return e;
    if ((e = read_arg(op, "forget", forget, forgetDesc, type, s, p.f)) != cudaSuccess) return e;
    if (input && (e = read_arg(op, "input", input, inputDesc, type, s, p.i)) != cudaSuccess) return e;
    if (output && (e = read_arg(op, "output", output, outputDesc, type, s, p.o)) != cudaSuccess) return e;
    if ((e = write_arg(op, "dUpdate", dUpdate, dUpdateDesc, type, s, p.dx)) != cudaSuccess) return e;
    if ((e = write_arg(op, "dForget", dForget, dForgetDesc, type, s, p.df)) != cudaSuccess) return e;
    if (input && (e = write_arg(op, "dInput", dInput, dInputDesc, type, s, p.di)) != cudaSuccess) return e;
    if (output && (e = write_arg(op, "dOutput", dOutput, dOutputDesc, type, s, p.dout)) != cudaSuccess) return e;
    if (lastGrad && (e = state_arg(op, "lastGrad", lastGradDesc, s, false, p.dlast_b, p.dlast_d)) != cudaSuccess) return e;
    if (dInitial && (e = state_arg(op, "dInitial", dInitialDesc, s, true, p.dinitial_b, p.dinitial_d)) != cudaSuccess) return e;
    if (!states && s.B * s.T * s.D != 0) return fail(cudaErrorInvalidValue, "%s: states is null: the forward pass has to keep them", op);
    if ((e = states_arg(op, statesDesc, s, false, p)) != cudaSuccess) return e;
    g_error[0] = 0;
    if (s.B == 0 || s.D == 0 || (s.T == 0 && !dInitial)) return cudaSuccess;
    p.dlast = static_cast<const float*>(lastGrad);
    p.lengths = lengths;
    p.states = static_cast<float*>(const_cast<void*>(states));
    p.dinitial = static_cast<float*>(dInitial);
    DeviceScope scope(stream);
    if (scope.status != cudaSuccess) return scope.status;
    return launch_recurrence_type(type, p, true, scope.device, stream);
}

}  // extern "C"
