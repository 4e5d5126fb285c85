// qgru_seq.cuh - what the sequence operators beside the GRU share: linear attention with a decay for each head
// (qgru_attn*.cu) and the root-mean-square norm (qgru_norm.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qgru.h"

namespace qgru {
namespace seq {

// ---- status and message of a call without a handle (qgru_seq.cu)
int fail(int status, const char *fmt, ...);
int cuda_fail(cudaError_t e, const char *where);

// QGRU_ERR_TIMEOUT, once for each thread that makes these calls, where a wait inside a kernel of an earlier call on the device has run out.
int check_expiry(int device);
// Where a kernel on the (current) device says so: a word of host memory, so that the next call knows without waiting.
int expiry_flag(int device, int **flag);

// Work goes to the device that the caller names; the thread's current device is put back when the call ends.  (Set even where it
// is the current one: a thread that has not used the device yet has no context, which tensor maps are encoded in.)
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if ((err_ = cudaGetDevice(&before_)) == cudaSuccess && (err_ = cudaSetDevice(device)) == cudaSuccess) moved_ = before_ != device;
    }
    ~OnDevice() {
        if (moved_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    cudaError_t error() const { return err_; }

  private:
    int before_ = 0;
    bool moved_ = false;
    cudaError_t err_;
};

#define SEQ_CK(expr)                                                     \
    do {                                                                 \
        const cudaError_t e_ = (expr);                                   \
        if (e_ != cudaSuccess) return ::qgru::seq::cuda_fail(e_, #expr); \
    } while (0)

// ---- element types
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ float load_f(const void *p, long long i, int bf16) {
    return bf16 ? to_f(static_cast<const __nv_bfloat16 *>(p)[i]) : static_cast<const float *>(p)[i];
}
__device__ __forceinline__ void store_f(void *p, long long i, int bf16, float v) {
    if (bf16)
        static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<float *>(p)[i] = v;
}

}  // namespace seq
}  // namespace qgru
