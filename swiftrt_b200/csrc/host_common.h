// What the translation units of the library share on the host side: the calling thread's error
// text, the launch counter, the device a call works on and element sizes.
#pragma once
#include "srt_matmul_api.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

namespace srt { struct FewRowsParams; }

// internal to the library: none of this is part of its dynamic symbols
namespace srt __attribute__((visibility("hidden"))) {
namespace host {

inline thread_local char g_error[512] = "";
inline std::atomic<uint64_t> g_launches{0};

inline cudaError_t fail(cudaError_t code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return code;
}

// What a launch returned, as the call's status.  A refused launch is also the runtime's last error, where the next kernel of anyone
// who asks for that would find it: it is taken away and becomes the call's text.
inline cudaError_t launch_status(cudaError_t e)
{
    if (e == cudaSuccess) return e;
    (void)cudaGetLastError();
    return fail(e, "a kernel could not be launched: %s", cudaGetErrorString(e));
}

// ------------------------------------------------------------------ the device of a call
// Every entry point that takes a stream works on THAT stream's device, whatever device is current
// on the calling thread: the reference's queues never select a device before they enqueue
// (Sources/SwiftRTCore/platform/cuda/functions/CudaMath.swift:117-125 launches on `stream` with no
// device call; nothing calls CudaQueue.selectDevice, cuda/device/CudaQueue.swift:77).  The scope
// resolves the stream's device, makes it current for the duration of the call when it differs and
// restores the caller's device afterwards; per-device state (workspaces, kernel attributes, the
// status word, the static scratch) is keyed by `device`.  The legacy and per-thread default
// streams belong to whatever device is current.  While a stream is being captured the runtime
// refuses the device query (and a refused call would invalidate the capture), so a capturing
// stream is taken to belong to the current device: capture with the stream's device current.
struct DeviceScope {
    int device = -1;
    int previous = -1;
    cudaError_t status = cudaSuccess;
    explicit DeviceScope(cudaStream_t stream)
    {
        int cur = 0;
        status = cudaGetDevice(&cur);
        if (status != cudaSuccess) return;
        int dev = cur;
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        if (stream != nullptr && stream != cudaStreamLegacy && stream != cudaStreamPerThread &&
            cudaStreamIsCapturing(stream, &cap) == cudaSuccess && cap == cudaStreamCaptureStatusNone) {
            status = cudaStreamGetDevice(stream, &dev);
            if (status != cudaSuccess) {
                fail(status, "cannot resolve the device of the stream: %s", cudaGetErrorString(status));
                return;
            }
        }
        device = dev;
        if (dev != cur) {
            status = cudaSetDevice(dev);
            if (status == cudaSuccess) previous = cur;
        }
    }
    ~DeviceScope()
    {
        if (previous >= 0) cudaSetDevice(previous);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

inline uint32_t elem_size(srtDataType t)
{
    switch (t) {
    case real32F: return 4;
    case real16F: case real16BF: return 2;
    default: return 0;
    }
}

// What kernels with TMA loads need from the host: the driver's tensor-map encoder, the status word of the device (which is current)
// and the limit of a wait in SM cycles.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
struct TileServices {
    EncodeTiledFn encode;
    uint32_t* status;
    unsigned long long wait_cycles;
};
cudaError_t tile_services(int device, TileServices& out);

cudaError_t gated_few_rows(srtDataType type, const FewRowsParams& params, bool k_contiguous, double limit, int device, cudaStream_t stream);

}  // namespace host
}  // namespace srt
