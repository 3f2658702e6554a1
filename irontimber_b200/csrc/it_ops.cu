// Device facts of the operators that take a stream instead of a context.
#include "it_ops.cuh"
#include "it_ops_sites.h"
#include <mutex>

int it_ops_current(void* stream, const char* who, it_ops_device* out) {
    static std::mutex lock;
    static it_ops_device known[64];
    static bool have[64] = {};
    int dev = 0;
    IT_CUDA(cudaGetDevice(&dev));
    IT_CHECK_ARG(dev < 64, "%s: device %d", who, dev);
    std::lock_guard<std::mutex> hold(lock);
    if (!have[dev]) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        IT_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &cap));
        if (cap != cudaStreamCaptureStatusNone) return it_fail(IT_ESTATE, "%s: the first call on a device cannot be recorded", who);
        it_ops_device d; d.device = dev;
        int major = 0;
        IT_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
        if (major != 10) return it_fail(IT_ESTATE, "%s: device %d is not sm_100a, which this library is built for", who, dev);
        IT_CUDA(cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev));
        IT_CUDA(cudaHostAlloc((void**)&d.status_host, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        *d.status_host = 0;
        const cudaError_t e = cudaHostGetDevicePointer((void**)&d.status_dev, d.status_host, 0);
        if (e != cudaSuccess) { cudaFreeHost(d.status_host); return it_fail(IT_ECUDA, "%s: %s", who, cudaGetErrorString(e)); }
        known[dev] = d; have[dev] = true;
    }
    *out = known[dev];
    // A wait that ran out in an earlier call: said once, by the next call.
    volatile int* status = out->status_host;
    if (*status) { const int site = *status; *status = 0; return it_fail(IT_ETIMEOUT, "%s: a wait of an earlier call on this device ran out (site %d); %s", who, site, it_ops_after_timeout(site)); }
    return IT_OK;
}
