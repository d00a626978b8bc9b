// Device calls of the HIP runtime on host memory, kernels left out, for tests of error paths without a GPU
// (preloaded before the real runtime). fake_hip_fail_at(n): the nth launch from here on fails.
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <stdlib.h>
#include <string.h>

static long launches = 0, fail_at = -1;
static hipError_t last = hipSuccess;

extern "C" {
long fake_hip_launches() { return launches; }
void fake_hip_fail_at(long n) { fail_at = launches + n; }

hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_t *p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void **p, const void *) { return *p = calloc(1, 1 << 20), hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) { return (*p = calloc(1, n)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void *p) { return hipFree(p); }
hipError_t hipMemset(void *p, int v, size_t n) { return memset(p, v, n), hipSuccess; }
hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind) { return memcpy(d, s, n), hipSuccess; }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind k, hipStream_t) { return hipMemcpy(d, s, n, k); }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { return *s = (hipStream_t)calloc(1, 64), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
// a kernel's call is pushed, popped by its stub and launched; without the real runtime nothing is kept
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *n, hipStream_t *s) {
    return *g = *b = dim3(1), *n = 0, *s = nullptr, hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) {
    return last = ++launches == fail_at ? hipErrorLaunchFailure : hipSuccess;
}
hipError_t hipGetLastError() {
    const hipError_t e = last;
    last = hipSuccess;
    return e;
}
}
