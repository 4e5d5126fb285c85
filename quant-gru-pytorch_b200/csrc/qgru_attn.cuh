// qgru_attn.cuh - linear attention with a decay for each head: what its kernels share.
//
// A sequence is cut into chunks of C tokens.  With G_t the running sum of the decays' logarithms from the chunk's start (base 2
// here) and S0 the state before the chunk
//     out_t = scale (2^G_t q_t S0 + sum_{s<=t} 2^(G_t - G_s) (q_t.k_s) v_s),    S' = 2^G_C S0 + sum_s 2^(G_C - G_s) k_s^T v_s
// so that one pass ("state pass") walks the chunks and leaves the state before each of them, and another takes every chunk by
// itself.  The gradient of the states obeys the same recurrence from the end, with q for k, dout for v and scale 2^G_t as
// weight, and is left behind each chunk by the same pass.
#pragma once
#include "qgru_seq.cuh"

namespace qgru {
namespace attn {

constexpr int MAX_D = 256;
constexpr float LOG2E = 1.4426950408889634f, LOG2E_REST = 1.92596303e-8f;
struct Cut {               // of a sequence of T tokens into chunks, and of the chunks into segments that run side by side
    int chunk = 0, chunks = 0, segments = 0, per = 0;
    size_t states = 0;     // bytes of the states before the chunks
    size_t seg = 0;        // bytes of the segments' own last states and decays, 0 for one segment
    size_t through = 0;    // bytes of the products of the states before the chunks with their gradients, where a pass leaves them
};

__device__ __forceinline__ int valid_tokens(const qgru_attention &a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
}

// Decays are summed up in 64-bit integers, base 2, in units of 2^-38: exact sums (a token's own rounding is 2^-38, 128 of them make 5e-10)
// that depend on no order.  A decay below 2^-160 is zero to any fp32 sum and one above 2^128 infinite, so the
// clamps keep -inf, +inf and a chunk's sum in range (128 * 160 < 2^14.4, 2^52.4 units); a NaN is a value beyond all sums, which makes
// every sum from it on NaN.
constexpr float UNITS = 0x1p38f;
constexpr long long NAN_UNITS = 1ll << 54;
__device__ __forceinline__ long long decay_units(float x) {
    const float hi = x * LOG2E;                                                       // x log2(e) as two floats
    if (!(hi > -160.f)) return hi == hi ? (long long)(-160.f * UNITS) : NAN_UNITS;
    if (hi > 128.f) return (long long)(128.f * UNITS);
    const float lo = fmaf(x, LOG2E, -hi) + x * LOG2E_REST;
    return __float2ll_rn(hi * UNITS) + __float2ll_rn(lo * UNITS);
}
__device__ __forceinline__ long long decay_units(const qgru_attention &a, long long at) { return decay_units(seq::load_f(a.decay.p, at, a.decay_bf16)); }
// A running sum as two floats, so that the difference of two of them is as exact as a float of its size, however large the sums are:
// G_t - G_s = (hi_t - hi_s) + (lo_t - lo_s), rounded once, 2^-24 of the difference.  (A difference of 20 is off by 1.2e-6 then, and so is
// its power of two, which is 1e-6 itself.)
__device__ __forceinline__ float2 two_floats(long long x) {
    if (x > NAN_UNITS / 2) return make_float2(__int_as_float(0x7fffffff), 0.f);
    const float hi = __ll2float_rn(x);
    return make_float2(hi * (1.f / UNITS), __ll2float_rn(x - __float2ll_rn(hi)) * (1.f / UNITS));
}
__device__ __forceinline__ float exp2_diff(float2 t, float2 s) { return exp2f((t.x - s.x) + (t.y - s.y)); }
__device__ __forceinline__ float exp2_of(float2 t) { return exp2f(t.x + t.y); }

// Running sums over N tokens (N / 32 warps, thread i has token i of them): the sum up to and with the thread's own.
template <int N, class T>
__device__ __forceinline__ T running_sum(T g, T *warp_sums, int tid) {
    const int lane = tid & 31;
    for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, g, o);
        if (lane >= o) g += u;
    }
    if (lane == 31) warp_sums[tid >> 5] = g;
    return g;
}

// ---- kernels for every size and type (qgru_attn.cu): fp32, products by warp-level tensor instructions on two tf32 values an operand
Cut generic_cut(const qgru_attention &a, int sms);
int generic_forward(const qgru_attention &a, const Cut &c, cudaStream_t st);
int generic_backward(const qgru_attention &a, const Cut &c, cudaStream_t st);
size_t group_bytes(const qgru_attention &a);
int sum_groups(const qgru_attention &a, const float *dq, const float *dk, cudaStream_t st);
int scan_segments(const qgru_attention &a, const Cut &c, bool reverse, char *seg, cudaStream_t st);

inline size_t a256(size_t n) { return (n + 255) & ~size_t(255); }
inline size_t state_elems(const qgru_attention &a) { return (size_t)a.B * a.H * a.Dk * a.Dv; }

}  // namespace attn
}  // namespace qgru
