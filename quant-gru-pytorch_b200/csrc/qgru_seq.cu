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
    long long times = 0;                 // that it was found set
};
constexpr int MAX_DEVICES = 64;
Flag flags[MAX_DEVICES];                 // made by the first call on a device, kept until the process ends
pthread_mutex_t flags_lock = PTHREAD_MUTEX_INITIALIZER;
thread_local long long told[MAX_DEVICES];        // of them, that this thread knows of, plus one; 0 before its first call

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

int check_expiry(int device) {
    if (device < 0 || device >= MAX_DEVICES) return QGRU_OK;         // (no device: the call says so)
    pthread_mutex_lock(&flags_lock);
    Flag &f = flags[device];
    if (!told[device]) told[device] = f.times + 1;                   // what was before a thread's first call is not its own
    if (f.host && *f.host) {
        *f.host = 0;
        ++f.times;
    }
    const bool news = told[device] <= f.times;
    told[device] = f.times + 1;
    pthread_mutex_unlock(&flags_lock);
    return news ? fail(QGRU_ERR_TIMEOUT, "a wait inside a kernel of an earlier call has run out: its results are not to be used") : QGRU_OK;
}

int expiry_flag(int device, int **flag) {
    if (device < 0 || device >= MAX_DEVICES) return fail(QGRU_ERR_BAD_ARG, "device %d", device);
    pthread_mutex_lock(&flags_lock);
    Flag &f = flags[device];
    const cudaError_t e = f.host ? cudaSuccess : make_flag(&f);
    *flag = f.device;
    pthread_mutex_unlock(&flags_lock);
    return e != cudaSuccess ? cuda_fail(e, "cudaHostAlloc") : QGRU_OK;
}

}  // namespace seq
}  // namespace qgru

using namespace qgru;

extern "C" {

const char *qgru_seq_last_error(void) { return seq::message; }
int qgru_seq_check(int device) { return seq::check_expiry(device); }
int qgru_seq_test_expire(int device) {
    const seq::OnDevice on(device);
    SEQ_CK(on.error());
    int *flag = nullptr;
    if (const int rc = seq::expiry_flag(device, &flag)) return rc;
    *seq::flags[device].host = 1;
    return QGRU_OK;
}

}  // extern "C"
