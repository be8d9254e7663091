// What becomes of a refused launch (launch_status of host_common.h), with a runtime of its own that only keeps a last error.
#include <cstdio>
#include <cstring>

#include "host_common.h"

static cudaError_t g_last = cudaSuccess;
extern "C" cudaError_t cudaGetLastError()
{
    const cudaError_t e = g_last;
    g_last = cudaSuccess;
    return e;
}
extern "C" const char* cudaGetErrorString(cudaError_t) { return "refused here"; }

int main()
{
    using namespace srt::host;
    // what a refused launch does in the runtime
    g_last = cudaErrorInvalidValue;
    const bool code = launch_status(cudaErrorInvalidValue) == cudaErrorInvalidValue;
    const bool text = strstr(g_error, "refused here") != nullptr, cleared = g_last == cudaSuccess;
    // a good one touches neither the text nor an error that someone else left
    g_error[0] = 0;
    g_last = cudaErrorInvalidConfiguration;
    const bool good = launch_status(cudaSuccess) == cudaSuccess && g_error[0] == 0 && g_last == cudaErrorInvalidConfiguration;
    printf("code %d text %d cleared %d good %d\n", code, text, cleared, good);
    return !(code && text && cleared && good);
}
