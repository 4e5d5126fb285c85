// qgru_seq.cu - status messages of the sequence operators, which have no handle to keep them.
#include "qgru_seq.cuh"

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

}  // namespace seq
}  // namespace qgru

extern "C" const char *qgru_seq_last_error(void) { return qgru::seq::message; }
