// qgru_norm.cu - root-mean-square norm with the residual's addition, its output in the element type or in 8 bits, and its gradient.
//
//     h = x + residual (rounded: the stream),  y = h w r,  r = 1 / sqrt(mean(h^2) + eps)
//     dh = r (dy w - n mean(dy w n)) + (gradient of the stream),  n = h r;   dw = sum over rows of dy n
//
// Bytes bound all of them: each tensor is read or written once, with a row in registers between its sum and its output.
// TPR threads have a row, each E elements of it in vectors of V neighbours; a warp each up to 1024 columns, a CTA above.
// 51200 x 1024 bf16 with residual, 420 MB: 67 us (6.3 TB/s).  In 8 bits with a scale a row, 367 MB: 76 us (4.8 TB/s): the row's
// phases (loads, sum, maximum, rounding, stores) follow one another; 101 us with a conversion instruction for every element.  4096 x
// 8192: 41 us (6.5 TB/s).  One row: 3 us, the launch.
#include <algorithm>
#include <type_traits>

#include "qgru_seq.cuh"

namespace qgru {
namespace norm {
namespace {

using bf16 = __nv_bfloat16;
constexpr int MOST = 32;        // elements of a row per thread; half of it in the largest CTA, whose threads have 64 registers
constexpr int MAX_COLS = 1024 * MOST / 2;
constexpr int WARPS_PER_CTA = 8;

enum Output { PLAIN, ROW8, GIVEN8 };

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// Sum or maximum over the TPR threads of a row; all get it.
template <int TPR, class F>
__device__ __forceinline__ float over_row(float x, float *part, F f) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
    if constexpr (TPR > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
        __syncthreads();
        x = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) x = f(x, part[w]);
    }
    return x;
}
template <int TPR>
__device__ __forceinline__ double max_over_row(double x, double *part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmax(x, __shfl_xor_sync(0xffffffffu, x, o));
    if constexpr (TPR > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
        __syncthreads();
        x = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) x = fmax(x, part[w]);
    }
    return x;
}

template <int V, class W>
__device__ __forceinline__ void load_weights(float (&w)[V], const void *p, int at) {
    const Vec<W, V> u = *reinterpret_cast<const Vec<W, V> *>(static_cast<const W *>(p) + at);
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = seq::to_f(u.v[i]);
}

template <class T, class W, int V, int TPR, int E, Output Out>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 32 * WARPS_PER_CTA) k_norm(const __grid_constant__ qgru_norm n) {
    constexpr int N = E / V;
    __shared__ float part[TPR / 32];
    __shared__ double part_d[TPR / 32];
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x & 31;
    const long long row = TPR > 32 ? blockIdx.x : (long long)blockIdx.x * WARPS_PER_CTA + (threadIdx.x >> 5);
    if (row >= n.rows) return;                       // (whole warps: a row wider than a warp has a CTA)
    const T *x = static_cast<const T *>(n.x) + row * n.x_stride;
    const T *r = n.residual ? static_cast<const T *>(n.residual) + row * n.residual_stride : nullptr;
    float h[N][V];
    float sum = 0.f;
    if (r) {
        T *to = static_cast<T *>(n.h_out) + row * n.h_stride;
        Vec<T, V> u[N], w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at < n.cols) {
                u[i] = *reinterpret_cast<const Vec<T, V> *>(x + at);
                w[i] = *reinterpret_cast<const Vec<T, V> *>(r + at);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // the stream is what is stored, so the norm is of the rounded sum, as its backward sees it
                const T s = seq::from_f<T>(seq::to_f(u[i].v[j]) + seq::to_f(w[i].v[j]));
                u[i].v[j] = s;
                h[i][j] = at < n.cols ? seq::to_f(s) : 0.f;
            }
            if (at < n.cols) *reinterpret_cast<Vec<T, V> *>(to + at) = u[i];
        }
    } else {
        Vec<T, V> u[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at < n.cols) u[i] = *reinterpret_cast<const Vec<T, V> *>(x + at);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) h[i][j] = (i * TPR + t) * V < n.cols ? seq::to_f(u[i].v[j]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    sum = over_row<TPR>(sum, part, [](float p, float q) { return p + q; });
    const float rstd = 1.f / sqrtf(sum / (float)n.cols + n.eps);
    if (n.rstd && t == 0) n.rstd[row] = rstd;
    if constexpr (Out == PLAIN) {
        T *y = static_cast<T *>(n.y) + row * n.y_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            float w[V];
            load_weights<V, W>(w, n.weight, at);
            Vec<T, V> u;
#pragma unroll
            for (int j = 0; j < V; ++j) u.v[j] = seq::from_f<T>(h[i][j] * rstd * w[j]);
            *reinterpret_cast<Vec<T, V> *>(y + at) = u;
        }
    } else if constexpr (Out == GIVEN8) {
        uint8_t *q = static_cast<uint8_t *>(n.q8) + row * n.cols;
        const float lo = (float)(n.q8_lo - n.q8_zero_point), hi = (float)(n.q8_hi - n.q8_zero_point);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            float w[V];
            load_weights<V, W>(w, n.weight, at);
            Vec<uint8_t, V> u;
#pragma unroll
            for (int j = 0; j < V; ++j) u.v[j] = (uint8_t)(__float2int_rn(fminf(fmaxf(rintf(h[i][j] * rstd * w[j] / n.q8_scale), lo), hi)) + n.q8_zero_point);
            *reinterpret_cast<Vec<uint8_t, V> *>(q + at) = u;
        }
    } else {
        // y / max|y| is h w / max|h w|: the root mean square drops out of q.  A quotient within 1e-4 of a border between two
        // steps (its fp32 rounding is below 3e-5) is decided by 64 bits, where h w is exact.
        constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;      // two bf16 factors have an exact fp32 product
        float hw[N][V];
        float top = 0.f, bad = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            float w[V] = {};
            if (at < n.cols) load_weights<V, W>(w, n.weight, at);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                hw[i][j] = h[i][j] * w[j];
                top = fmaxf(top, fabsf(hw[i][j]));
                bad = fmaf(hw[i][j], 0.f, bad);      // (fmaxf drops NaN)
            }
        }
        top = over_row<TPR>(bad != 0.f ? INFINITY : top, part, [](float p, float q) { return fmaxf(p, q); });
        uint8_t *q = static_cast<uint8_t *>(n.q8) + row * n.cols;
        if (!(top > 0.f && top < INFINITY)) {
            if (t == 0) n.scales[row] = top > 0.f ? NAN : 0.f;
            for (int at = t; at < n.cols; at += TPR) q[at] = 0;
            return;
        }
        double exact_top = (double)top;
        if constexpr (!EXACT) {
            double d = 0.0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = (i * TPR + t) * V;
                if (at >= n.cols) continue;
                float w[V];
                load_weights<V, W>(w, n.weight, at);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (fabsf(hw[i][j]) == top) d = fmax(d, fabs((double)h[i][j] * (double)w[j]));
            }
            exact_top = max_over_row<TPR>(d, part_d);
        }
        if (t == 0) n.scales[row] = top * rstd / 127.f;
        const float steps = 127.f / top;
        const bool plain_range = top > 1e-30f && top < 1e30f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            // rounded by adding 1.5 * 2^23, which leaves the integer in the low bits
            Vec<int8_t, V> u;
            float off = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = hw[i][j] * steps, r = __fadd_rn(p, 12582912.f);
                u.v[j] = (int8_t)__float_as_int(r);
                off = fmaxf(off, fabsf(p - __fadd_rn(r, -12582912.f)));
            }
            if (!plain_range || off > 0.5f - 1e-4f) {
                float w[V];
                if constexpr (!EXACT) load_weights<V, W>(w, n.weight, at);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const double exact = EXACT ? (double)hw[i][j] : (double)h[i][j] * (double)w[j];
                    u.v[j] = (int8_t)__double2int_rn(exact * 127.0 / exact_top);
                }
            }
            *reinterpret_cast<Vec<int8_t, V> *>(q + at) = u;
        }
    }
}

struct Backward {
    const void *h, *dy, *dh;
    void *dx;
    long long h_stride, dy_stride, dh_stride, dx_stride;
    float *parts;                   // [CTAs][cols], or null
};

__device__ __forceinline__ void cp_async16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// Rows in turn; a thread keeps the weights of its E columns and the sums of dw, which leave once a CTA.  Whole vectors of the next rows
// (three of bf16, one of fp32; with sixteen elements a thread one and none) are on their way into shared memory, where each thread reads
// back what it has fetched itself; single elements come straight from memory.  51200 x 1024 bf16 with the stream's gradient, 420 MB: 155 us with a warp a row and no row
// ahead, 123 us with one row ahead in registers, 74 us so (5.7 TB/s).
constexpr int AHEAD_BYTES = 192;                     // of shared memory a thread
template <class T, class W, int V, int TPR, int E>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 32 * WARPS_PER_CTA) k_norm_backward(const __grid_constant__ qgru_norm n, const Backward g) {
    constexpr int N = E / V, ROWS = TPR > 32 ? 1 : WARPS_PER_CTA;
    constexpr int STAGES = V > 1 ? AHEAD_BYTES / (3 * E * (int)sizeof(T)) : 1;
    __shared__ float part[2][TPR / 32];
    extern __shared__ uint4 smem[];                  // [STAGES][3 N][threads], then [ROWS][cols] sums where a row is a warp's
    float *dw_part = reinterpret_cast<float *>(smem);
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x & 31, mine = TPR > 32 ? 0 : threadIdx.x >> 5;
    float dw[N][V], w[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int at = (i * TPR + t) * V + j;
            dw[i][j] = 0.f;
            w[i][j] = at < n.cols ? seq::to_f(static_cast<const W *>(n.weight)[at]) : 0.f;
        }
    const long long step = (long long)gridDim.x * ROWS;
    const auto place = [&](int stage, int which, int i) { return smem + ((stage * 3 + which) * N + i) * blockDim.x + threadIdx.x; };
    const auto row_of = [&](const void *p, long long row, long long stride) { return static_cast<const T *>(p) + row * stride; };
    const auto fetch = [&](long long row, int stage) {
        if constexpr (V > 1) {
            if (row < n.rows) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int at = (i * TPR + t) * V;
                    if (at >= n.cols) continue;
                    cp_async16(place(stage, 0, i), row_of(g.h, row, g.h_stride) + at);
                    cp_async16(place(stage, 1, i), row_of(g.dy, row, g.dy_stride) + at);
                    if (g.dh) cp_async16(place(stage, 2, i), row_of(g.dh, row, g.dh_stride) + at);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    long long row = (long long)blockIdx.x * ROWS + mine;
    for (int k = 0; k < STAGES - 1; ++k) fetch(row + k * step, k);
    int stage = 0;
    for (int buf = 0; row < n.rows; row += step, buf ^= 1) {
        const float rstd = n.rstd[row];
        float x[N][V], y[N][V], d[N][V], sum = 0.f;
        if constexpr (V > 1) {
            fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            Vec<T, V> u, v, s;
#pragma unroll
            for (int j = 0; j < V; ++j) u.v[j] = v.v[j] = s.v[j] = seq::from_f<T>(0.f);
            if (at < n.cols) {
                if constexpr (V > 1) {
                    u = *reinterpret_cast<const Vec<T, V> *>(place(stage, 0, i));
                    v = *reinterpret_cast<const Vec<T, V> *>(place(stage, 1, i));
                    if (g.dh) s = *reinterpret_cast<const Vec<T, V> *>(place(stage, 2, i));
                } else {
                    u.v[0] = row_of(g.h, row, g.h_stride)[at];
                    v.v[0] = row_of(g.dy, row, g.dy_stride)[at];
                    if (g.dh) s.v[0] = row_of(g.dh, row, g.dh_stride)[at];
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[i][j] = seq::to_f(u.v[j]) * rstd;
                const float dy = seq::to_f(v.v[j]);
                dw[i][j] = fmaf(dy, x[i][j], dw[i][j]);
                y[i][j] = dy * w[i][j];
                sum = fmaf(y[i][j], x[i][j], sum);
                d[i][j] = seq::to_f(s.v[j]);
            }
        }
        if (++stage == STAGES) stage = 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if constexpr (TPR > 32) {
            if ((threadIdx.x & 31) == 0) part[buf][threadIdx.x >> 5] = sum;
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < TPR / 32; ++k) sum += part[buf][k];
        }
        sum /= (float)n.cols;
        T *dx = static_cast<T *>(g.dx) + row * g.dx_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            Vec<T, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) o.v[j] = seq::from_f<T>(fmaf(rstd, fmaf(-sum, x[i][j], y[i][j]), d[i][j]));
            if (at < n.cols) *reinterpret_cast<Vec<T, V> *>(dx + at) = o;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (!g.parts) return;
    float *to = g.parts + (long long)blockIdx.x * n.cols;
    if constexpr (TPR > 32) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if ((i * TPR + t) * V < n.cols) to[(i * TPR + t) * V + j] = dw[i][j];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if ((i * TPR + t) * V < n.cols) dw_part[mine * n.cols + (i * TPR + t) * V + j] = dw[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < n.cols; c += blockDim.x) {
            float x = 0.f;
            for (int r = 0; r < ROWS; ++r) x += dw_part[r * n.cols + c];
            to[c] = x;
        }
    }
}

// dw: the CTAs' sums, 32 columns a CTA, 32 warps that take every 32nd CTA's, in a fixed order.  Memory's latency bounds it: 2 to 9 us.
template <class W>
__global__ void __launch_bounds__(1024) k_sum_parts(const float *parts, int count, int cols, W *dw) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float x = 0.f;
    if (c < cols) {
#pragma unroll 4
        for (int p = warp; p < count; p += 32) x += parts[(long long)p * cols + c];
    }
    part[warp][lane] = x;
    __syncthreads();
    if (warp == 0 && c < cols) {
        for (int w = 1; w < 32; ++w) x += part[w][lane];
        dw[c] = seq::from_f<W>(x);
    }
}

template <class F>
int by_width(int cols, F f) {
    const auto with = [&](auto tpr, auto e) -> int { return f(tpr, e); };
    using std::integral_constant;
    if (cols <= 32 * MOST / 4) return with(integral_constant<int, 32>(), integral_constant<int, MOST / 4>());
    if (cols <= 32 * MOST / 2) return with(integral_constant<int, 32>(), integral_constant<int, MOST / 2>());
    if (cols <= 32 * MOST) return with(integral_constant<int, 32>(), integral_constant<int, MOST>());
    if (cols <= 128 * MOST) return with(integral_constant<int, 128>(), integral_constant<int, MOST>());
    if (cols <= 256 * MOST) return with(integral_constant<int, 256>(), integral_constant<int, MOST>());
    return with(integral_constant<int, 1024>(), integral_constant<int, MOST / 2>());
}
// whether vectors of `v` elements of `size` bytes fit all rows of a tensor
bool fits(const void *p, long long stride, int v, int size, long long rows) {
    return !p || (reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && (rows <= 1 || stride % v == 0));
}

template <class T, class W, int V, Output Out>
int forward(const qgru_norm &n, cudaStream_t st) {
    return by_width(n.cols, [&](auto tpr, auto e) -> int {
        constexpr int TPR = tpr.value, E = e.value;
        constexpr int per = TPR > 32 ? 1 : WARPS_PER_CTA;
        k_norm<T, W, V, TPR, E, Out><<<(unsigned)((n.rows + per - 1) / per), TPR > 32 ? TPR : 32 * per, 0, st>>>(n);
        SEQ_CK(cudaGetLastError());
        return QGRU_OK;
    });
}
template <class T, class W, int V>
int forward(const qgru_norm &n, cudaStream_t st) {
    return !n.q8 ? forward<T, W, V, PLAIN>(n, st) : n.q8_scale > 0.f ? forward<T, W, V, GIVEN8>(n, st) : forward<T, W, V, ROW8>(n, st);
}
template <class T, class W>
int forward(const qgru_norm &n, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool wide = n.cols % V == 0 && fits(n.x, n.x_stride, V, sizeof(T), n.rows) && fits(n.residual, n.residual_stride, V, sizeof(T), n.rows) &&
                      fits(n.h_out, n.h_stride, V, sizeof(T), n.rows) && fits(n.y, n.y_stride, V, sizeof(T), n.rows) && fits(n.weight, 0, V, sizeof(W), 1) &&
                      fits(n.q8, n.cols, V, 1, n.rows);
    return wide ? forward<T, W, V>(n, st) : forward<T, W, 1>(n, st);
}

// Threads of a row of the backward: eight columns each, up to 1024 (sixteen each above 8192 columns), and CTAs: 1024 threads an SM, whose
// rows and next rows in flight are what its latency takes.
int threads_of_row(int cols) {
    int t = 32;
    while (t < 1024 && t * 8 < cols) t *= 2;
    return t;
}
int ctas(int sms, long long rows, int cols) {
    const int t = threads_of_row(cols);
    const long long units = t == 32 ? (rows + WARPS_PER_CTA - 1) / WARPS_PER_CTA : rows;
    const int per_sm = 1024 / (t == 32 ? 32 * WARPS_PER_CTA : t);
    return (int)std::max<long long>(1, std::min<long long>(units, (long long)sms * per_sm));
}
template <class T, class W, int V>
int backward(const qgru_norm &n, const Backward &g, int grid, cudaStream_t st) {
    using std::integral_constant;
    const auto run = [&](auto tpr, auto e) -> int {
        constexpr int TPR = tpr.value, E = e.value;
        constexpr int threads = TPR > 32 ? TPR : 32 * WARPS_PER_CTA;
        const size_t sums = TPR == 32 && g.parts ? sizeof(float) * WARPS_PER_CTA * n.cols : 0, ahead = V > 1 ? (size_t)AHEAD_BYTES * threads : 0;
        const size_t bytes = std::max(sums, ahead);
        const auto kernel = k_norm_backward<T, W, V, TPR, E>;
        if (bytes > 40 * 1024) SEQ_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        kernel<<<grid, threads, bytes, st>>>(n, g);
        SEQ_CK(cudaGetLastError());
        return QGRU_OK;
    };
    const integral_constant<int, 8> e;
    switch (threads_of_row(n.cols)) {
        case 32: return run(integral_constant<int, 32>(), e);
        case 64: return run(integral_constant<int, 64>(), e);
        case 128: return run(integral_constant<int, 128>(), e);
        case 256: return run(integral_constant<int, 256>(), e);
        case 512: return run(integral_constant<int, 512>(), e);
        default: return n.cols <= 8192 ? run(integral_constant<int, 1024>(), e) : run(integral_constant<int, 1024>(), integral_constant<int, 16>());
    }
}
template <class T, class W>
int backward(const qgru_norm &n, const Backward &g, int grid, W *dw, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool wide = n.cols % V == 0 && fits(g.h, g.h_stride, V, sizeof(T), n.rows) && fits(g.dy, g.dy_stride, V, sizeof(T), n.rows) &&
                      fits(g.dh, g.dh_stride, V, sizeof(T), n.rows) && fits(g.dx, g.dx_stride, V, sizeof(T), n.rows) && fits(n.weight, 0, V, sizeof(W), 1);
    if (const int rc = wide ? backward<T, W, V>(n, g, grid, st) : backward<T, W, 1>(n, g, grid, st)) return rc;
    if (dw) {
        k_sum_parts<W><<<(n.cols + 31) / 32, 1024, 0, st>>>(g.parts, grid, n.cols, dw);
        SEQ_CK(cudaGetLastError());
    }
    return QGRU_OK;
}

int check(const qgru_norm *n) {
    using seq::fail;
    if (!n) return fail(QGRU_ERR_BAD_ARG, "null argument block");
    if (n->rows < 0 || n->cols < 1) return fail(QGRU_ERR_BAD_ARG, "rows must not be negative and cols must be positive");
    if (n->cols > MAX_COLS) return fail(QGRU_ERR_UNSUPPORTED, "at most %d columns, got %d", MAX_COLS, n->cols);
    if (n->rows > 2147483647ll) return fail(QGRU_ERR_UNSUPPORTED, "at most 2^31 - 1 rows");
    return QGRU_OK;
}

}  // namespace
}  // namespace norm
}  // namespace qgru

using namespace qgru;

extern "C" {

int qgru_norm_forward(const qgru_norm *n, void *stream) {
    if (const int rc = norm::check(n)) return rc;
    if (n->rows == 0) return QGRU_OK;
    if (!n->x || !n->weight || (n->residual && !n->h_out)) return seq::fail(QGRU_ERR_BAD_ARG, "null tensor");
    if (!n->y == !n->q8) return seq::fail(QGRU_ERR_BAD_ARG, "one of y and q8 is written");
    if (n->q8 && !(n->q8_scale > 0.f) && !n->scales) return seq::fail(QGRU_ERR_BAD_ARG, "scales is null");
    if (n->q8 && n->q8_scale > 0.f && (n->q8_lo > n->q8_hi || n->q8_lo < -128 || n->q8_hi > 255 || n->q8_hi - n->q8_lo > 255 || (n->q8_lo < 0 && n->q8_hi > 127)))
        return seq::fail(QGRU_ERR_BAD_ARG, "%d .. %d is no range of 8 bits", n->q8_lo, n->q8_hi);
    if (const int rc = seq::check_expiry(n->device)) return rc;
    const seq::OnDevice on(n->device);
    SEQ_CK(on.error());
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    using b = __nv_bfloat16;
    return n->bf16 ? (n->weight_bf16 ? norm::forward<b, b>(*n, st) : norm::forward<b, float>(*n, st))
                   : (n->weight_bf16 ? norm::forward<float, b>(*n, st) : norm::forward<float, float>(*n, st));
}

size_t qgru_norm_workspace(int device, long long rows, int cols) {
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return sizeof(float) * (size_t)norm::ctas(sms, rows, cols) * (size_t)cols;
}

int qgru_norm_backward(const qgru_norm *n, const void *h, long long h_stride, const void *dy, long long dy_stride, const void *dh, long long dh_stride, void *dx,
                       long long dx_stride, void *dweight, void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = norm::check(n)) return rc;
    if (const int rc = seq::check_expiry(n->device)) return rc;
    const seq::OnDevice on(n->device);
    SEQ_CK(on.error());
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n->rows == 0) {
        if (dweight) SEQ_CK(cudaMemsetAsync(dweight, 0, (size_t)n->cols * (n->weight_bf16 ? 2 : 4), st));
        return QGRU_OK;
    }
    if (!h || !dy || !dx || !n->weight || !n->rstd) return seq::fail(QGRU_ERR_BAD_ARG, "null tensor");
    int sms = 0;
    SEQ_CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, n->device));
    const int grid = norm::ctas(sms, n->rows, n->cols);
    const size_t need = sizeof(float) * (size_t)grid * (size_t)n->cols;
    if (dweight && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return seq::fail(QGRU_ERR_BAD_ARG, "workspace needs %zu bytes aligned to 16, got %zu", need, workspace_bytes);
    const norm::Backward g{h, dy, dh, dx, h_stride, dy_stride, dh_stride, dx_stride, dweight ? static_cast<float *>(workspace) : nullptr};
    using b = __nv_bfloat16;
    if (n->weight_bf16) {
        b *dw = static_cast<b *>(dweight);
        return n->bf16 ? norm::backward<b, b>(*n, g, grid, dw, st) : norm::backward<float, b>(*n, g, grid, dw, st);
    }
    float *dw = static_cast<float *>(dweight);
    return n->bf16 ? norm::backward<b, float>(*n, g, grid, dw, st) : norm::backward<float, float>(*n, g, grid, dw, st);
}

}  // extern "C"
