// qgru_seq.cu - status messages of the sequence operators, which have no handle to keep them.
#include "qgru_seq.cuh"

#include <pthread.h>

#include <cstdarg>
#include <cstdio>

namespace qgru {
namespace seq {
namespace {
thread_local char message[256] = "";
}

int fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(message, sizeof message, fmt, ap);
    va_end(ap);
    return status;
}
int cuda_fail(cudaError_t e, const char *where) {
    cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? QGRU_ERR_NOMEM : QGRU_ERR_CUDA, "%s: %s", where, cudaGetErrorString(e));
}

namespace {
struct Flag {
    volatile int *host = nullptr;
    int *device = nullptr;
};
constexpr int MAX_DEVICES = 64;
Flag flags[MAX_DEVICES];                 // made by the first call on a device, kept until the process ends
pthread_mutex_t flags_lock = PTHREAD_MUTEX_INITIALIZER;

cudaError_t make_flag(Flag *f) {
    // (allowed while another stream or this one is being captured: nothing of it is part of the graph)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    void *p = nullptr, *d = nullptr;
    e = cudaHostAlloc(&p, 64, cudaHostAllocMapped);
    if (e == cudaSuccess) {
        *static_cast<int *>(p) = 0;
        if ((e = cudaHostGetDevicePointer(&d, p, 0)) != cudaSuccess) cudaFreeHost(p);
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaSuccess) {
        f->device = static_cast<int *>(d);
        f->host = static_cast<volatile int *>(p);
    }
    return e;
}
}  // namespace

int expiry_flag(int device, int **flag) {
    if (device < 0 || device >= MAX_DEVICES) return fail(QGRU_ERR_BAD_ARG, "device %d", device);
    pthread_mutex_lock(&flags_lock);
    Flag &f = flags[device];
    const cudaError_t e = f.host ? cudaSuccess : make_flag(&f);
    const bool expired = f.host && *f.host;
    if (expired) *f.host = 0;
    *flag = f.device;
    pthread_mutex_unlock(&flags_lock);
    if (e != cudaSuccess) return cuda_fail(e, "cudaHostAlloc");
    return expired ? fail(QGRU_ERR_TIMEOUT, "a wait inside a kernel of an earlier call has run out: its results are not to be used") : QGRU_OK;
}

}  // namespace seq
}  // namespace qgru

extern "C" const char *qgru_seq_last_error(void) { return qgru::seq::message; }
