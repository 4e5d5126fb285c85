// qgru_norm.cu - root-mean-square norm with the residual's addition, its output in the element type or in 8 bits, and its gradient.
//
//     h = x + residual (rounded: the stream),  y = h w r,  r = 1 / sqrt(mean(h^2) + eps)
//     dh = r (dy w - n mean(dy w n)) + (gradient of the stream),  n = h r;   dw = sum over rows of dy n
//
// Bytes bound all of them: each tensor is read or written once, with a row in registers between its sum and its output.
// TPR threads have a row, each N vectors of V neighbouring elements; a warp each up to 1024 columns, a CTA above.
#include <algorithm>
#include <type_traits>

#include "qgru_seq.cuh"

namespace qgru {
namespace norm {
namespace {

using bf16 = __nv_bfloat16;
constexpr int MOST = 32;        // elements of a row per thread; half of it in the largest CTA, whose threads have 64 registers
template <int TPR>
constexpr int MOST_OF = TPR == 1024 ? MOST / 2 : MOST;
constexpr int MAX_COLS = 1024 * MOST_OF<1024>;
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

template <class T, class W, int V, int TPR, Output Out>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 32 * WARPS_PER_CTA) k_norm(const __grid_constant__ qgru_norm n) {
    constexpr int N = MOST_OF<TPR> / V;
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
        float top = 0.f, bad = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            float w[V];
            load_weights<V, W>(w, n.weight, at);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = fabsf(h[i][j] * w[j]);
                top = fmaxf(top, p);
                if (!isfinite(p)) bad = 1.f;         // (fmaxf drops NaN)
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
        if constexpr (sizeof(T) == 4 || sizeof(W) == 4) {     // two bf16 factors have an exact product
            double d = 0.0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = (i * TPR + t) * V;
                if (at >= n.cols) continue;
                float w[V];
                load_weights<V, W>(w, n.weight, at);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (fabsf(h[i][j] * w[j]) == top) d = fmax(d, fabs((double)h[i][j] * (double)w[j]));
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
            float w[V];
            load_weights<V, W>(w, n.weight, at);
            Vec<int8_t, V> u;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = h[i][j] * w[j] * steps;
                float k = rintf(p);
                if (!plain_range || 0.5f - fabsf(p - k) < 1e-4f) k = (float)rint((double)h[i][j] * (double)w[j] * 127.0 / exact_top);
                u.v[j] = (int8_t)__float2int_rn(k);
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

// Rows in turn; a thread keeps the sums of dw of its columns, which leave once a CTA.
template <class T, class W, int V, int TPR>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 32 * WARPS_PER_CTA) k_norm_backward(const __grid_constant__ qgru_norm n, const Backward g) {
    constexpr int N = MOST_OF<TPR> / V, ROWS = TPR > 32 ? 1 : WARPS_PER_CTA;
    __shared__ float part[TPR / 32];
    extern __shared__ float dw_part[];               // [ROWS][cols] where a row is a warp's
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x & 31, mine = TPR > 32 ? 0 : threadIdx.x >> 5;
    float dw[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = 0.f;
    for (long long row = (long long)blockIdx.x * ROWS + mine; row < n.rows; row += (long long)gridDim.x * ROWS) {
        const T *h = static_cast<const T *>(g.h) + row * g.h_stride, *dy = static_cast<const T *>(g.dy) + row * g.dy_stride;
        Vec<T, V> u[N], v[N], s[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            u[i] = *reinterpret_cast<const Vec<T, V> *>(h + at);
            v[i] = *reinterpret_cast<const Vec<T, V> *>(dy + at);
            if (g.dh) s[i] = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(g.dh) + row * g.dh_stride + at);
        }
        const float rstd = n.rstd[row];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            float w[V];
            load_weights<V, W>(w, n.weight, at);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = seq::to_f(u[i].v[j]) * rstd, y = seq::to_f(v[i].v[j]);
                sum = fmaf(y * w[j], x, sum);
                dw[i][j] = fmaf(y, x, dw[i][j]);
            }
        }
        sum = over_row<TPR>(sum, part, [](float p, float q) { return p + q; }) / (float)n.cols;
        T *dx = static_cast<T *>(g.dx) + row * g.dx_stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * TPR + t) * V;
            if (at >= n.cols) continue;
            float w[V];
            load_weights<V, W>(w, n.weight, at);
            Vec<T, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = seq::to_f(u[i].v[j]) * rstd;
                float d = rstd * (seq::to_f(v[i].v[j]) * w[j] - x * sum);
                if (g.dh) d += seq::to_f(s[i].v[j]);
                o.v[j] = seq::from_f<T>(d);
            }
            *reinterpret_cast<Vec<T, V> *>(dx + at) = o;
        }
    }
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

// dw: the CTAs' sums, 32 columns a CTA, eight warps that take every eighth CTA's, in a fixed order.
template <class W>
__global__ void __launch_bounds__(256) k_sum_parts(const float *parts, int count, int cols, W *dw) {
    __shared__ float part[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float x = 0.f;
    if (c < cols)
        for (int p = warp; p < count; p += 8) x += parts[(long long)p * cols + c];
    part[warp][lane] = x;
    __syncthreads();
    if (warp == 0 && c < cols) {
        for (int w = 1; w < 8; ++w) x += part[w][lane];
        dw[c] = seq::from_f<W>(x);
    }
}

template <class F>
int by_width(int cols, F f) {
    if (cols <= 32 * MOST) return f(std::integral_constant<int, 32>());
    if (cols <= 128 * MOST) return f(std::integral_constant<int, 128>());
    if (cols <= 256 * MOST) return f(std::integral_constant<int, 256>());
    return f(std::integral_constant<int, 1024>());
}
// whether vectors of `v` elements of `size` bytes fit all rows of a tensor
bool fits(const void *p, long long stride, int v, int size, long long rows) {
    return !p || (reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && (rows <= 1 || stride % v == 0));
}

template <class T, class W, int V, Output Out>
int forward(const qgru_norm &n, cudaStream_t st) {
    return by_width(n.cols, [&](auto tpr) -> int {
        constexpr int TPR = tpr.value;
        constexpr int per = TPR > 32 ? 1 : WARPS_PER_CTA;
        k_norm<T, W, V, TPR, Out><<<(unsigned)((n.rows + per - 1) / per), TPR > 32 ? TPR : 32 * per, 0, st>>>(n);
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

// CTAs of the backward: what is resident at once, each with its sums of dw at the end.
int ctas(int sms, long long rows, int cols) {
    const bool warps = cols <= 32 * MOST;
    const long long units = warps ? (rows + WARPS_PER_CTA - 1) / WARPS_PER_CTA : rows;
    const int per_sm = warps ? 2 : cols <= 128 * MOST ? 4 : cols <= 256 * MOST ? 2 : 1;
    return (int)std::max<long long>(1, std::min<long long>(units, (long long)sms * per_sm));
}
template <class T, class W, int V>
int backward(const qgru_norm &n, const Backward &g, int grid, cudaStream_t st) {
    return by_width(n.cols, [&](auto tpr) -> int {
        constexpr int TPR = tpr.value;
        const size_t bytes = TPR == 32 && g.parts ? sizeof(float) * WARPS_PER_CTA * n.cols : 0;
        k_norm_backward<T, W, V, TPR><<<grid, TPR > 32 ? TPR : 32 * WARPS_PER_CTA, bytes, st>>>(n, g);
        SEQ_CK(cudaGetLastError());
        return QGRU_OK;
    });
}
template <class T, class W>
int backward(const qgru_norm &n, const Backward &g, int grid, W *dw, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool wide = n.cols % V == 0 && fits(g.h, g.h_stride, V, sizeof(T), n.rows) && fits(g.dy, g.dy_stride, V, sizeof(T), n.rows) &&
                      fits(g.dh, g.dh_stride, V, sizeof(T), n.rows) && fits(g.dx, g.dx_stride, V, sizeof(T), n.rows) && fits(n.weight, 0, V, sizeof(W), 1);
    if (const int rc = wide ? backward<T, W, V>(n, g, grid, st) : backward<T, W, 1>(n, g, grid, st)) return rc;
    if (dw) {
        k_sum_parts<W><<<(n.cols + 31) / 32, 256, 0, st>>>(g.parts, grid, n.cols, dw);
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
