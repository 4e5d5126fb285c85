// qgru_attn.cu - linear attention: the entry points, the kernels for every size and type, and the single-token form.
//
// The kernels here compute in fp32 whatever the inputs' type, 64 tokens a chunk and 64 x 64 tiles, by warp-level tensor instructions;
// they serve fp32 tensors and head sizes above 128, which the tcgen05 kernels (qgru_attn_fwd.cu, qgru_attn_tc.cu) do not take: fp32
// operands as three bf16 parts would be three times the shared memory, and the gradients' six tiles fill it with one.
#include <algorithm>
#include <type_traits>

#include "qgru_attn.cuh"
#include "qgru_attn_tc.cuh"

namespace qgru {
namespace attn {
namespace {

constexpr int C = 64, THREADS = 256;
constexpr int TILE = 64 * 64;                   // floats
using bf16 = __nv_bfloat16;

// A 64 x 64 tile in shared memory: rows of sixteen 16-byte chunks, chunk c of row r at c ^ f(r), so that eight rows' neighbouring four
// values, and four rows' neighbouring eight, lie in different banks: the operands of the products below either way.
__device__ __forceinline__ int idx(int r, int c) { return r * 64 + ((((c >> 2) ^ (2 * r) ^ (r >> 3)) & 15) << 2) + (c & 3); }

// 64 x 64 sums of 32 / NT warps: 16 rows and 8 NT columns a warp, lane (g, t) = (lane / 4, lane % 4) has rows g and g + 8 and columns 2 t
// and 2 t + 1 of each eight.
template <int NT>
struct Sums {
    float v[NT][4];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = 0.f;
    }
};
using Acc = Sums<4>;
// x as two tf32 values (11 significant bits): the nearest one, and of the rest, which has twelve bits at the most, all but the last.  (By
// hand: the conversion instruction is three times the work.)  The nearest one of the largest floats is infinite, and an infinity less
// itself is NaN; Finite: the first is finite always, the second may be the infinity or the NaN.
constexpr float MOST = 0x1.ffdffep+127f;          // the largest that is rounded to a finite one
template <bool Finite>
__device__ __forceinline__ void two_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(Finite ? fminf(fmaxf(x, -MOST), MOST) : x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// acc += sum over k = 8 from .. 8 to - 1 of A(m, k) B(k, n).  ARows: A's tile has k as its rows, else m; BRows: B's tile has k as its rows,
// else n.  fp32 by warp-level tensor instructions: each operand is the sum of two tf32 values (off by 2^-23 of it at the most), and of the
// four products the one of the two small parts is left out (2^-22 of the product at the most).  Operands below 2^-114 keep 11 bits.
// Where a lane's value of eight K lies in a tile for K = 0 .. 7 (bytes), and for K = 8 s .. 8 s + 7 after it: the swizzle is a change of bits
// that both depend on.  line: the row or column that is not K; up: 0 or 4 of the eight.
template <bool KRows>
__device__ __forceinline__ uint32_t first_at(int line, int t, int up) { return (uint32_t)idx(KRows ? t + up : line, KRows ? line : t + up) * 4; }
template <bool KRows>
__device__ __forceinline__ float value_at(const float *tile, uint32_t first, int s) {
    const uint32_t at = KRows ? (first ^ (uint32_t)(s << 4)) + (uint32_t)(s << 11) : first ^ (uint32_t)(s << 5);
    return *reinterpret_cast<const float *>(reinterpret_cast<const char *>(tile) + at);
}
template <bool ARows, bool BRows, bool Finite, int NT>
__device__ __forceinline__ void eight(Sums<NT> &c, const float *A, const float *B, const uint32_t (&pa)[4], const uint32_t (&pb)[NT][2], int s) {
    uint32_t ah[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) two_tf32<Finite>(value_at<ARows>(A, pa[i], s), ah[i], al[i]);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        uint32_t bh[2], bl[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) two_tf32<Finite>(value_at<BRows>(B, pb[j][i], s), bh[i], bl[i]);
        // (the tensor cores cut off what a sum cannot hold: eight K stay there, longer sums are rounded to nearest)
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        mma(t, al, bh);
        mma(t, ah, bl);
        mma(t, ah, bh);
#pragma unroll
        for (int i = 0; i < 4; ++i) c.v[j][i] += t[i];
    }
}
// Look: a sum that is not finite is taken again with first parts that are, so that the largest floats have results and infinities stay
// infinities.  32 x 200 tokens of 8 heads of 64: outputs 32.4 us and gradients 87, where first parts that are finite from the start make it 34.3
// and 92 (32.0 and 84.5 with neither).  The state pass, whose sums stay in their registers from chunk to chunk, has none to spare for the
// sums as they were (31.9 us), and finite parts from the start (25.7; 24.7 with neither).
template <bool ARows, bool BRows, bool Look = true, int NT>
__device__ __forceinline__ void multiply(Sums<NT> &c, const float *A, const float *B, int from, int to, int tid) {
    const int lane = tid & 31, g = lane >> 2, t = lane & 3, m = (tid >> 5 & 3) * 16 + g, n = (tid >> 7) * (8 * NT) + g;
    uint32_t pa[4], pb[NT][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) pa[i] = first_at<ARows>(m + (i & 1) * 8, t, (i >> 1) * 4);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) pb[j][i] = first_at<BRows>(n + 8 * j, t, 4 * i);
    const Sums<NT> before = c;
#pragma unroll 2
    for (int s = from; s < to; ++s) eight<ARows, BRows, !Look>(c, A, B, pa, pb, s);
    if constexpr (!Look) return;
    float odd = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd = fmaf(c.v[j][i], 0.f, odd);
    if (__any_sync(0xffffffffu, !(odd == 0.f))) {
        c = before;
#pragma unroll 1
        for (int s = from; s < to; ++s) eight<ARows, BRows, true>(c, A, B, pa, pb, s);
    }
}
template <int NT, class F>
__device__ __forceinline__ void each(Sums<NT> &c, int tid, F f) {
    const int lane = tid & 31, m = (tid >> 5 & 3) * 16 + (lane >> 2), n = (tid >> 7) * (8 * NT) + (lane & 3) * 2;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) f(m + (i >> 1) * 8, n + j * 8 + (i & 1), c.v[j][i]);
}
__device__ __forceinline__ int eights(int n) { return (min(n, 64) + 7) >> 3; }
// Every row of the sums times a factor, in place; the rows' products with a tile's: [8 / NT][64], a warp's columns each.
template <int NT, class F>
__device__ __forceinline__ void scale_rows(Sums<NT> &c, const float *X, float *dots, F factor, int tid) {
    const int lane = tid & 31, m = (tid >> 5 & 3) * 16 + (lane >> 2), n = (tid >> 7) * (8 * NT) + (lane & 3) * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = m + 8 * h;
        const float w = factor(row);
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c.v[j][2 * h + i] *= w;
                x = fmaf(c.v[j][2 * h + i], X[idx(row, n + j * 8 + i)], x);
            }
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if ((lane & 3) == 0) dots[(tid >> 7) * 64 + row] += x;
    }
}

// A thread's share of a 64 x 64 tile: four neighbouring columns at four places.  64 tokens x 64 columns of a tensor, zeros outside; four
// columns a load where rows and strides allow it.
struct Four {
    float4 v[4];
    template <class T>
    __device__ __forceinline__ void load(const qgru_seq_tensor &x, long long base, int t0, int tokens, int d0, int d, int tid) {
        const T *p = static_cast<const T *>(x.p) + base;
        const bool wide = ((x.ts | x.bs | x.hs | d) & 3) == 0 && reinterpret_cast<uintptr_t>(x.p) % (4 * sizeof(T)) == 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (tid >> 4) + 16 * i, c = (tid & 15) * 4;
            float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < tokens && d0 + c < d) {
                const T *q = p + (long long)(t0 + r) * x.ts + d0 + c;
                if (wide) {
                    if constexpr (sizeof(T) == 4) {
                        u = *reinterpret_cast<const float4 *>(q);
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2 *>(q);
                        u = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
                    }
                } else {
                    u.x = seq::to_f(q[0]);
                    if (d0 + c + 1 < d) u.y = seq::to_f(q[1]);
                    if (d0 + c + 2 < d) u.z = seq::to_f(q[2]);
                    if (d0 + c + 3 < d) u.w = seq::to_f(q[3]);
                }
            }
            v[i] = u;
        }
    }
    __device__ __forceinline__ void store(float *to, int tid) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4 *>(to + idx((tid >> 4) + 16 * i, (tid & 15) * 4)) = v[i];
    }
    // whether one of them is infinite or NaN
    __device__ __forceinline__ bool odd() const {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x = fmaf(v[i].x, 0.f, fmaf(v[i].y, 0.f, fmaf(v[i].z, 0.f, fmaf(v[i].w, 0.f, x))));
        return !(x == 0.f);
    }
};
template <class T>
__device__ __forceinline__ void load_tile(float *to, const qgru_seq_tensor &x, long long base, int t0, int tokens, int d0, int d, int tid) {
    Four f;
    f.load<T>(x, base, t0, tokens, d0, d, tid);
    f.store(to, tid);
}
__device__ __forceinline__ void load_state(float *to, const float *S, int i0, int j0, const qgru_attention &a, int tid) {
#pragma unroll
    for (int e = tid; e < TILE / 4; e += THREADS) {
        const int r = e >> 4, c = (e & 15) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + r < a.Dk && j0 + c < a.Dv) {
            const float *q = S + (long long)(i0 + r) * a.Dv + j0 + c;
            if (a.Dv % 4 == 0) {
                v = *reinterpret_cast<const float4 *>(q);
            } else {
                v.x = q[0];
                if (j0 + c + 1 < a.Dv) v.y = q[1];
                if (j0 + c + 2 < a.Dv) v.z = q[2];
                if (j0 + c + 3 < a.Dv) v.w = q[3];
            }
        }
        *reinterpret_cast<float4 *>(to + idx(r, c)) = v;
    }
}
__device__ __forceinline__ long long at(const qgru_seq_tensor &x, int b, int h) { return b * x.bs + h * x.hs; }

// G of a chunk by the first 64 threads, others pass
__device__ __forceinline__ void sum_decays(float2 *G, long long *sums, long long g, int tid) {
    if (tid < C) g = running_sum<C>(g, sums, tid);
    __syncthreads();
    if (tid < C) G[tid] = two_floats(g + (tid >= 32 ? sums[0] : 0));
    __syncthreads();
}

// The chunk's running sums G[0 .. 63] (tokens behind the sequence add nothing).
__device__ __forceinline__ void load_decays(float2 *G, long long *sums, const qgru_attention &a, int b, int h, int t0, int tokens, int tid) {
    sum_decays(G, sums, tid < tokens ? decay_units(a, at(a.decay, b, h) + (long long)(t0 + tid) * a.decay.ts) : 0, tid);
}

struct Pass {                      // a state pass
    qgru_seq_tensor k, v;
    int k_share;                   // heads that share one of k
    const float *first;            // the state it starts from, or null
    float *last;                   // where the last one goes, or null
    float *states;                 // before each chunk (in the pass's order)
    bool own_sums;                 // instead: each segment's sum, from zero
    float *seg_state, *seg_log;    // [segments][B H][Dk][Dv], [segments][B H]
    int segments, per, chunks;
};

// grid: (B H, tiles of the state, segments).  Order of chunks: forward, or from the last one back (Reverse), where the weight of a
// token is scale 2^G_t instead of 2^(G_C - G_t).
// S' = 2^G_C S + (w k)^T v: a 64 x 64 tile of the state in registers, one product a chunk.  Every tile of the state reads k or v anew, and
// the chunks follow one another: a chunk's latency bounds it (32 x 200 tokens of 8 heads of 64, fp32: 25 us, 6 us a chunk).
template <class T, bool Reverse>
__global__ void __launch_bounds__(THREADS) k_states(const __grid_constant__ qgru_attention a, const Pass p) {
    __shared__ alignas(16) float K[TILE], V[TILE];
    __shared__ float2 G[C];
    __shared__ float W[C];
    __shared__ long long g_sums[2];
    const int tid = threadIdx.x, bh = blockIdx.x, b = bh / a.H, h = bh % a.H;
    const int nj = (a.Dv + 63) / 64, i0 = (int)blockIdx.y / nj * 64, j0 = (int)blockIdx.y % nj * 64;
    const int n = valid_tokens(a, b), seg = blockIdx.z;
    const long long kb = at(p.k, b, h / p.k_share), vb = at(p.v, b, h), tile = (long long)bh * a.Dk * a.Dv;
    const bool own_sums = p.own_sums;
    Acc S;
    S.zero();
    const long long size = (long long)gridDim.x * a.Dk * a.Dv;
    const auto inside = [&](int i, int j) { return i0 + i < a.Dk && j0 + j < a.Dv; };
    const auto place = [&](int i, int j) { return (long long)(i0 + i) * a.Dv + j0 + j; };
    const float *first = p.segments > 1 ? p.seg_state + seg * size : p.first;
    if (!own_sums && first) each(S, tid, [&](int i, int j, float &s) { s = inside(i, j) ? first[tile + place(i, j)] : 0.f; });
    double all = 0.0;
    const int c_end = min((seg + 1) * p.per, p.chunks);
    const auto chunk_of = [&](int c) { return Reverse ? p.chunks - 1 - c : c; };
    const auto tokens_of = [&](int c) { return c < c_end ? min(max(n - chunk_of(c) * C, 0), C) : 0; };
    // (four neighbouring columns a load; the next chunk's are on their way while one is worked on)
    Four k4, v4;
    long long g = 0;
    const auto load = [&](int c) {
        const int tokens = tokens_of(c), t0 = chunk_of(c) * C;
        k4.template load<T>(p.k, kb, t0, tokens, i0, a.Dk, tid);
        v4.template load<T>(p.v, vb, t0, tokens, j0, a.Dv, tid);
        g = tid < tokens ? decay_units(a, at(a.decay, b, h) + (long long)(t0 + tid) * a.decay.ts) : 0;
    };
    if (seg * p.per < c_end) load(seg * p.per);
    for (int c = seg * p.per; c < c_end; ++c) {
        const int chunk = chunk_of(c), tokens = tokens_of(c);
        if (!own_sums) each(S, tid, [&](int i, int j, float &s) { if (inside(i, j)) p.states[chunk * size + tile + place(i, j)] = s; });
        __syncthreads();
        if (tokens) {
            k4.store(K, tid);
            v4.store(V, tid);
        }
        sum_decays(G, g_sums, g, tid);
        if (c + 1 < c_end) load(c + 1);
        if (tokens == 0) continue;
        const float2 end = G[C - 1];
        if (tid < C) W[tid] = Reverse ? a.scale * exp2_of(G[tid]) : exp2_diff(end, G[tid]);
        __syncthreads();
        for (int e = tid; e < TILE; e += THREADS) K[e] *= W[e >> 6];
        __syncthreads();
        const float whole = exp2_of(end);
        all += (double)end.x + (double)end.y;
        each(S, tid, [&](int, int, float &s) { s *= whole; });
        multiply<true, true, false>(S, K, V, 0, eights(tokens), tid);
    }
    if (own_sums) {
        each(S, tid, [&](int i, int j, float &s) { if (inside(i, j)) p.seg_state[seg * size + tile + place(i, j)] = s; });
        if (blockIdx.y == 0 && tid == 0) p.seg_log[seg * gridDim.x + bh] = (float)all;
    } else if (p.last && seg == p.segments - 1) {
        each(S, tid, [&](int i, int j, float &s) { if (inside(i, j)) p.last[tile + place(i, j)] = s; });
    }
}

// The segments' own sums become the states that they start from.  A thread per element; eight segments' sums are in flight.  Memory's
// latency bounds it: a state of 4 heads of 128 x 128 over 37 segments, 10 MB, in 6 us.
__global__ void __launch_bounds__(128) k_scan_segments(float *seg_state, const float *seg_log, const float *first, int segments, long long size, int per_head) {
    constexpr int AHEAD = 8;
    const long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= size) return;
    const int heads = (int)(size / per_head), bh = (int)(e / per_head);
    float s = first ? first[e] : 0.f;
    for (int g0 = 0; g0 < segments; g0 += AHEAD) {
        float own[AHEAD], log[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int g = min(g0 + j, segments - 1);
            own[j] = seg_state[g * size + e];
            log[j] = seg_log[g * heads + bh];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (g0 + j >= segments) break;
            seg_state[(g0 + j) * size + e] = s;
            s = fmaf(exp2f(log[j]), s, own[j]);
        }
    }
}

// grid: chunks x B H, the heads of one chunk beside each other (their tokens lie together).  out = 2^G_t q S + P v, 64 columns of the
// output at a time over 64 of the head's; the tiles pass through shared memory one after another, so a CTA waits for each: 37 x 127
// tokens of 5 heads of 40 x 72, fp32, ragged: 23 us.  Up to 64 x 64 of fp32 the kernels further down fetch all tiles at once instead.
template <class T>
__global__ void __launch_bounds__(THREADS) k_outputs(const __grid_constant__ qgru_attention a, const float *states) {
    extern __shared__ float4 smem4[];
    float *X = reinterpret_cast<float *>(smem4), *Y = X + TILE, *P = Y + TILE;
    __shared__ float2 G[C];
    __shared__ long long g_sums[2];
    const int tid = threadIdx.x, heads = a.B * a.H, chunk = blockIdx.x / heads, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H, t0 = chunk * C;
    const int all = min(a.T - t0, C), tokens = min(max(valid_tokens(a, b) - t0, 0), C);
    T *out = static_cast<T *>(a.out.p) + at(a.out, b, h) + t0 * a.out.ts;
    if (tokens == 0) {
        for (int e = tid; e < all * a.Dv; e += THREADS) out[(e / a.Dv) * a.out.ts + e % a.Dv] = seq::from_f<T>(0.f);
        return;
    }
    const int hk = h / (a.H / a.Hk);
    const bool carried = chunk > 0 || a.state0;
    const long long qb = at(a.q, b, hk), kb = at(a.k, b, hk), vb = at(a.v, b, h);
    const float *S = states + chunk * (long long)heads * a.Dk * a.Dv + (long long)bh * a.Dk * a.Dv;
    load_decays(G, g_sums, a, b, h, t0, tokens, tid);
    // the pairs of a warp's 16 rows end in their columns
    const int up_to = (tid >> 5 & 3) * 2 + 2;
    Acc c;
    c.zero();
    for (int d = 0; d < a.Dk; d += 64) {
        load_tile<T>(X, a.q, qb, t0, tokens, d, a.Dk, tid);
        load_tile<T>(Y, a.k, kb, t0, tokens, d, a.Dk, tid);
        __syncthreads();
        multiply<false, false>(c, X, Y, 0, eights(a.Dk - d), tid);
        __syncthreads();
    }
    each(c, tid, [&](int t, int s, float &x) { P[idx(t, s)] = s <= t ? a.scale * exp2_diff(G[t], G[s]) * x : 0.f; });
    for (int j = 0; j < a.Dv; j += 64) {
        c.zero();
        for (int d = 0; d < a.Dk && carried; d += 64) {
            load_tile<T>(X, a.q, qb, t0, tokens, d, a.Dk, tid);
            load_state(Y, S, d, j, a, tid);
            __syncthreads();
            multiply<false, true>(c, X, Y, 0, eights(a.Dk - d), tid);
            __syncthreads();
        }
        each(c, tid, [&](int t, int, float &x) { x *= a.scale * exp2_of(G[t]); });
        Four v4;
        v4.load<T>(a.v, vb, t0, tokens, j, a.Dv, tid);
        v4.store(Y, tid);
        // A later token's infinity or NaN is none of an earlier one's business, and zero times it is NaN.  (Each thread looks at what it
        // has loaded itself: the tile is not whole before the barrier.)
        if (__syncthreads_or(v4.odd())) {
            each(c, tid, [&](int t, int n, float &x) {
                for (int s = 0; s <= t; ++s) x = fmaf(P[idx(t, s)], Y[idx(s, n)], x);
            });
        } else {
            multiply<false, true>(c, P, Y, 0, min(eights(tokens), up_to), tid);
        }
        __syncthreads();
        each(c, tid, [&](int t, int n, float &x) {
            if (t < all && j + n < a.Dv) out[t * a.out.ts + j + n] = seq::from_f<T>(t < tokens ? x : 0.f);
        });
    }
}

// grid: chunks x B H.  dq, dk: where the type's elements go, or fp32 sums of every head [T][B][H][Dk] (heads that share q and k).
// Nine products of 64 x 64 tiles for each pair of them, tiles one after another: shared memory and its barriers bound it.
template <class T>
__global__ void __launch_bounds__(THREADS) k_gradients(const __grid_constant__ qgru_attention a, const float *states, const float *dstates, float *dq_heads,
                                                       float *dk_heads) {
    extern __shared__ float4 smem4[];
    float *X = reinterpret_cast<float *>(smem4), *Y = X + TILE, *P = Y + TILE, *E = P + TILE;
    __shared__ float2 G[C];
    __shared__ long long g_sums[2];
    __shared__ float dG[3][C], kE[2][C];     // what a change of the decays' sum up to token t brings; k_s's share behind the chunk
    const int tid = threadIdx.x, heads = a.B * a.H, chunk = blockIdx.x / heads, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H, t0 = chunk * C;
    const int all = min(a.T - t0, C), tokens = min(max(valid_tokens(a, b) - t0, 0), C);
    const int hk = h / (a.H / a.Hk);
    const long long qb = at(a.q, b, hk), kb = at(a.k, b, hk), vb = at(a.v, b, h), ob = at(a.dout, b, h);
    const auto put_qk = [&](const qgru_seq_tensor &x, float *heads, int t, int d, float v) {
        if (heads)
            heads[(((long long)(t0 + t) * a.B + b) * a.H + h) * a.Dk + d] = v;
        else
            static_cast<T *>(x.p)[at(x, b, h) + (t0 + t) * x.ts + d] = seq::from_f<T>(v);
    };
    T *dv = static_cast<T *>(a.dv.p) + at(a.dv, b, h) + t0 * a.dv.ts;
    const long long gb = at(a.ddecay, b, h) + t0 * a.ddecay.ts;
    if (tokens == 0) {
        for (int e = tid; e < all * a.Dk; e += THREADS) {
            put_qk(a.dq, dq_heads, e / a.Dk, e % a.Dk, 0.f);
            put_qk(a.dk, dk_heads, e / a.Dk, e % a.Dk, 0.f);
        }
        for (int e = tid; e < all * a.Dv; e += THREADS) dv[(e / a.Dv) * a.dv.ts + e % a.Dv] = seq::from_f<T>(0.f);
        if (tid < all) seq::store_f(a.ddecay.p, gb + tid * a.ddecay.ts, a.decay_bf16, 0.f);
        return;
    }
    const long long tile = chunk * (long long)heads * a.Dk * a.Dv + (long long)bh * a.Dk * a.Dv;
    const float *S = states + tile, *dS = dstates + tile;
    load_decays(G, g_sums, a, b, h, t0, tokens, tid);
    if (tid < C) kE[0][tid] = kE[1][tid] = dG[0][tid] = dG[1][tid] = dG[2][tid] = 0.f;
    // the pairs of a warp's 16 rows end in their columns, or begin there
    const int diagonal = (tid >> 5 & 3) * 2, last = eights(tokens);
    Acc c, e2;
    c.zero();
    e2.zero();
    for (int d = 0; d < a.Dk; d += 64) {
        load_tile<T>(X, a.q, qb, t0, tokens, d, a.Dk, tid);
        load_tile<T>(Y, a.k, kb, t0, tokens, d, a.Dk, tid);
        __syncthreads();
        multiply<false, false>(c, X, Y, 0, eights(a.Dk - d), tid);
        __syncthreads();
    }
    for (int d = 0; d < a.Dv; d += 64) {
        load_tile<T>(X, a.dout, ob, t0, tokens, d, a.Dv, tid);
        load_tile<T>(Y, a.v, vb, t0, tokens, d, a.Dv, tid);
        __syncthreads();
        multiply<false, false>(e2, X, Y, 0, eights(a.Dv - d), tid);
        __syncthreads();
    }
    {
        const int lane = tid & 31, t0 = (tid >> 5 & 3) * 16 + (lane >> 2), s0 = (tid >> 7) * 32 + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + (i >> 1) * 8, s = s0 + j * 8 + (i & 1);
                const float w = s <= t ? a.scale * exp2_diff(G[t], G[s]) : 0.f, ov = e2.v[j][i];
                const float p = s <= t ? w * c.v[j][i] : 0.f, e = s <= t ? w * ov : 0.f;
                P[idx(t, s)] = p;
                E[idx(t, s)] = e;
                X[idx(t, s)] = s < t ? p * ov : 0.f;
            }
    }
    __syncthreads();
    // every pair (t, s), s < t: a change of G_t adds, one of G_s takes away
    if (tid < C) {
        double r = 0.0;
        for (int s = 0; s < C; ++s) r += (double)X[idx(tid, s)] - (double)X[idx(s, tid)];
        dG[2][tid] = (float)r;
    }
    __syncthreads();
    const float2 end = G[C - 1];
    for (int i = 0; i < a.Dk; i += 64) {
        // dq = E k + scale 2^G_t dout S^T
        c.zero();
        for (int j = 0; j < a.Dv; j += 64) {
            load_tile<T>(X, a.dout, ob, t0, tokens, j, a.Dv, tid);
            load_state(Y, S, i, j, a, tid);
            __syncthreads();
            multiply<false, false>(c, X, Y, 0, eights(a.Dv - j), tid);
            __syncthreads();
        }
        load_tile<T>(X, a.q, qb, t0, tokens, i, a.Dk, tid);
        load_tile<T>(Y, a.k, kb, t0, tokens, i, a.Dk, tid);
        __syncthreads();
        scale_rows(c, X, dG[0], [&](int t) { return a.scale * exp2_of(G[t]); }, tid);
        multiply<false, true>(c, E, Y, 0, min(diagonal + 2, last), tid);
        each(c, tid, [&](int t, int d, float &x) { if (t < all && i + d < a.Dk) put_qk(a.dq, dq_heads, t, i + d, t < tokens ? x : 0.f); });
        __syncthreads();
        // dk = E^T q + 2^(G_C - G_s) v dS^T
        c.zero();
        for (int j = 0; j < a.Dv; j += 64) {
            load_tile<T>(X, a.v, vb, t0, tokens, j, a.Dv, tid);
            load_state(Y, dS, i, j, a, tid);
            __syncthreads();
            multiply<false, false>(c, X, Y, 0, eights(a.Dv - j), tid);
            __syncthreads();
        }
        load_tile<T>(X, a.q, qb, t0, tokens, i, a.Dk, tid);
        load_tile<T>(Y, a.k, kb, t0, tokens, i, a.Dk, tid);
        __syncthreads();
        scale_rows(c, Y, kE[0], [&](int s) { return exp2_diff(end, G[s]); }, tid);
        multiply<true, true>(c, E, X, diagonal, last, tid);
        each(c, tid, [&](int s, int d, float &x) { if (s < all && i + d < a.Dk) put_qk(a.dk, dk_heads, s, i + d, s < tokens ? x : 0.f); });
        __syncthreads();
    }
    for (int j = 0; j < a.Dv; j += 64) {
        // dv = P^T dout + 2^(G_C - G_s) k dS
        c.zero();
        for (int i = 0; i < a.Dk; i += 64) {
            load_tile<T>(X, a.k, kb, t0, tokens, i, a.Dk, tid);
            load_state(Y, dS, i, j, a, tid);
            __syncthreads();
            multiply<false, true>(c, X, Y, 0, eights(a.Dk - i), tid);
            __syncthreads();
        }
        each(c, tid, [&](int s, int, float &x) { x *= exp2_diff(end, G[s]); });
        load_tile<T>(X, a.dout, ob, t0, tokens, j, a.Dv, tid);
        __syncthreads();
        multiply<true, true>(c, P, X, diagonal, last, tid);
        each(c, tid, [&](int s, int d, float &x) { if (s < all && j + d < a.Dv) dv[s * a.dv.ts + j + d] = seq::from_f<T>(s < tokens ? x : 0.f); });
        __syncthreads();
    }
    // The state before the chunk reaches everything behind it through all of the chunk's decays.
    double through = 0.0;
    for (int e = tid; e < a.Dk * a.Dv; e += THREADS) through += (double)S[e] * (double)dS[e];
    for (int o = 16; o; o >>= 1) through += __shfl_xor_sync(0xffffffffu, through, o);
    double *sum_of = reinterpret_cast<double *>(smem4);
    if ((tid & 31) == 0) sum_of[tid >> 5] = through;
    __syncthreads();
    if (tid == 0) {
        through = 0.0;
        for (int w = 0; w < THREADS / 32; ++w) through += sum_of[w];
        through *= (double)exp2_of(end);
        for (int s = 0; s < tokens; ++s) through += (double)kE[0][s] + (double)kE[1][s];
        // from the end: sum over u >= t of dG_u, the shares of k_s for s < t, and what passes through
        double acc = 0.0;
        for (int t = tokens - 1; t >= 0; --t) {
            acc += (double)dG[0][t] + (double)dG[1][t] + (double)dG[2][t];
            through -= (double)kE[0][t] + (double)kE[1][t];
            X[64 + t] = (float)(acc + through);
        }
    }
    __syncthreads();
    if (tid < all) seq::store_f(a.ddecay.p, gb + tid * a.ddecay.ts, a.decay_bf16, tid < tokens ? X[64 + tid] : 0.f);
}

// ------------------------------------------------------------------------------------- fp32, head sizes up to 64
// Every chunk's tiles are fetched at once, asynchronously, into a tile each; then nothing waits for memory.  What bounds these is the
// issue of mma.sync and of the operands' splits (two tf32 values for each, three products, rounded to nearest every eight K).
// 32 x 200 ragged tokens of 8 heads of 64: outputs 32 us; gradients 87 us so, with sixteen warps, 16 x 16 sums a warp, and 118 us tile
// after tile, with eight warps, three CTAs an SM.
constexpr int ALL = 512, NT2 = 2;

__device__ __forceinline__ void cp_float4(float *to, const float *from, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_float(float *to, const float *from, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(on ? 4 : 0) : "memory");
}
// `rows` rows of d floats, ld apart; zeros around them
template <int N>
__device__ __forceinline__ void fetch(float *to, const float *p, long long ld, int rows, int d, int tid) {
    if (d % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
        for (int e = tid; e < TILE / 4; e += N) {
            const int r = e >> 4, c = (e & 15) * 4;
            const bool on = r < rows && c < d;
            cp_float4(to + idx(r, c), on ? p + r * ld + c : p, on);
        }
    } else {
        for (int e = tid; e < TILE; e += N) {
            const int r = e >> 6, c = e & 63;
            const bool on = r < rows && c < d;
            cp_float(to + idx(r, c), on ? p + r * ld + c : p, on);
        }
    }
}
__device__ __forceinline__ const float *token(const qgru_seq_tensor &x, long long base, int t0) { return static_cast<const float *>(x.p) + base + (long long)t0 * x.ts; }
__device__ __forceinline__ void cp_all() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__global__ void __launch_bounds__(THREADS, 2) k_outputs_small(const __grid_constant__ qgru_attention a, const float *states) {
    extern __shared__ float4 smem4[];
    float *Q = reinterpret_cast<float *>(smem4), *K = Q + TILE, *V = K + TILE, *S = V + TILE, *P = S + TILE;
    __shared__ float2 G[C];
    __shared__ long long g_sums[2];
    const int tid = threadIdx.x, heads = a.B * a.H, chunk = blockIdx.x / heads, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H, t0 = chunk * C;
    const int all = min(a.T - t0, C), tokens = min(max(valid_tokens(a, b) - t0, 0), C);
    float *out = static_cast<float *>(a.out.p) + at(a.out, b, h) + t0 * a.out.ts;
    if (tokens == 0) {
        for (int e = tid; e < all * a.Dv; e += THREADS) out[(e / a.Dv) * a.out.ts + e % a.Dv] = 0.f;
        return;
    }
    const int hk = h / (a.H / a.Hk);
    const bool carried = chunk > 0 || a.state0;
    fetch<THREADS>(Q, token(a.q, at(a.q, b, hk), t0), a.q.ts, tokens, a.Dk, tid);
    fetch<THREADS>(K, token(a.k, at(a.k, b, hk), t0), a.k.ts, tokens, a.Dk, tid);
    fetch<THREADS>(V, token(a.v, at(a.v, b, h), t0), a.v.ts, tokens, a.Dv, tid);
    if (carried) fetch<THREADS>(S, states + chunk * (long long)heads * a.Dk * a.Dv + (long long)bh * a.Dk * a.Dv, a.Dv, a.Dk, a.Dv, tid);
    const long long g = tid < tokens ? decay_units(a, at(a.decay, b, h) + (long long)(t0 + tid) * a.decay.ts) : 0;
    cp_all();
    sum_decays(G, g_sums, g, tid);
    const int up_to = min((tid >> 5 & 3) * 2 + 2, eights(tokens));       // the pairs of a warp's 16 rows end in their columns
    Acc c;
    c.zero();
    multiply<false, false>(c, Q, K, 0, eights(a.Dk), tid);
    each(c, tid, [&](int t, int s, float &x) { P[idx(t, s)] = s <= t ? a.scale * exp2_diff(G[t], G[s]) * x : 0.f; });
    // A later token's infinity or NaN is none of an earlier one's business, and zero times it is NaN.
    int odd = 0;
    for (int e = tid; e < TILE; e += THREADS) odd |= !isfinite(V[e]);
    c.zero();
    if (carried) {
        multiply<false, true>(c, Q, S, 0, eights(a.Dk), tid);
        each(c, tid, [&](int t, int, float &x) { x *= a.scale * exp2_of(G[t]); });
    }
    if (__syncthreads_or(odd)) {
        each(c, tid, [&](int t, int n, float &x) {
            for (int s = 0; s <= t; ++s) x = fmaf(P[idx(t, s)], V[idx(s, n)], x);
        });
    } else {
        multiply<false, true>(c, P, V, 0, up_to, tid);
    }
    each(c, tid, [&](int t, int n, float &x) {
        if (t < all && n < a.Dv) out[t * a.out.ts + n] = t < tokens ? x : 0.f;
    });
}

__global__ void __launch_bounds__(ALL, 1) k_gradients_small(const __grid_constant__ qgru_attention a, const float *states, const float *dstates, float *dq_heads, float *dk_heads) {
    extern __shared__ float4 smem4[];
    float *Q = reinterpret_cast<float *>(smem4), *K = Q + TILE, *V = K + TILE, *O = V + TILE, *S = O + TILE, *dS = S + TILE, *P = dS + TILE, *E = P + TILE;
    __shared__ float2 G[C];
    __shared__ long long g_sums[2];
    __shared__ double sums[2], totals[2], through_of[ALL / 32];
    __shared__ float rows[4][C], columns[4][C], q_dots[4][C], k_dots[4][C];
    const int tid = threadIdx.x, lane = tid & 31, heads = a.B * a.H, chunk = blockIdx.x / heads, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H, t0 = chunk * C;
    const int all = min(a.T - t0, C), tokens = min(max(valid_tokens(a, b) - t0, 0), C);
    const int hk = h / (a.H / a.Hk);
    const auto put_qk = [&](const qgru_seq_tensor &x, float *heads_sums, int t, int d, float v) {
        if (heads_sums)
            heads_sums[(((long long)(t0 + t) * a.B + b) * a.H + h) * a.Dk + d] = v;
        else
            static_cast<float *>(x.p)[at(x, b, h) + (t0 + t) * x.ts + d] = v;
    };
    float *dv = static_cast<float *>(a.dv.p) + at(a.dv, b, h) + t0 * a.dv.ts;
    const long long gb = at(a.ddecay, b, h) + t0 * a.ddecay.ts;
    if (tokens == 0) {
        for (int e = tid; e < all * a.Dk; e += ALL) {
            put_qk(a.dq, dq_heads, e / a.Dk, e % a.Dk, 0.f);
            put_qk(a.dk, dk_heads, e / a.Dk, e % a.Dk, 0.f);
        }
        for (int e = tid; e < all * a.Dv; e += ALL) dv[(e / a.Dv) * a.dv.ts + e % a.Dv] = 0.f;
        if (tid < all) seq::store_f(a.ddecay.p, gb + tid * a.ddecay.ts, a.decay_bf16, 0.f);
        return;
    }
    const long long tile = chunk * (long long)heads * a.Dk * a.Dv + (long long)bh * a.Dk * a.Dv;
    fetch<ALL>(Q, token(a.q, at(a.q, b, hk), t0), a.q.ts, tokens, a.Dk, tid);
    fetch<ALL>(K, token(a.k, at(a.k, b, hk), t0), a.k.ts, tokens, a.Dk, tid);
    fetch<ALL>(V, token(a.v, at(a.v, b, h), t0), a.v.ts, tokens, a.Dv, tid);
    fetch<ALL>(O, token(a.dout, at(a.dout, b, h), t0), a.dout.ts, tokens, a.Dv, tid);
    fetch<ALL>(S, states + tile, a.Dv, a.Dk, a.Dv, tid);
    fetch<ALL>(dS, dstates + tile, a.Dv, a.Dk, a.Dv, tid);
    const long long g = tid < tokens ? decay_units(a, at(a.decay, b, h) + (long long)(t0 + tid) * a.decay.ts) : 0;
    if (tid < 4 * C) q_dots[0][tid] = k_dots[0][tid] = 0.f;
    cp_all();
    sum_decays(G, g_sums, g, tid);
    const float2 end = G[C - 1];
    const int ek = eights(a.Dk), ev = eights(a.Dv), last = eights(tokens), diagonal = (tid >> 5 & 3) * 2;
    Sums<NT2> c, e;
    c.zero();
    e.zero();
    multiply<false, false>(c, Q, K, 0, ek, tid);
    multiply<false, false>(e, O, V, 0, ev, tid);
    {
        const int m = (tid >> 5 & 3) * 16 + (lane >> 2), n = (tid >> 7) * (8 * NT2) + (lane & 3) * 2;
        float row[2] = {0.f, 0.f}, column[NT2][2];
#pragma unroll
        for (int j = 0; j < NT2; ++j) {
            column[j][0] = column[j][1] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = m + (i >> 1) * 8, s = n + j * 8 + (i & 1);
                const bool on = s <= t;
                const float w = on ? a.scale * exp2_diff(G[t], G[s]) : 0.f, p = on ? w * c.v[j][i] : 0.f;
                P[idx(t, s)] = p;
                E[idx(t, s)] = on ? w * e.v[j][i] : 0.f;
                // every pair, s < t: a change of G_t adds, one of G_s takes away
                const float x = s < t ? p * e.v[j][i] : 0.f;
                row[i >> 1] += x;
                column[j][i & 1] += x;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            row[i] += __shfl_xor_sync(0xffffffffu, row[i], 1);
            row[i] += __shfl_xor_sync(0xffffffffu, row[i], 2);
            if ((lane & 3) == 0) rows[tid >> 7][m + 8 * i] = row[i];
#pragma unroll
            for (int j = 0; j < NT2; ++j) {
                float x = column[j][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (lane < 4) columns[tid >> 5 & 3][n + 8 * j + i] = x;
            }
        }
    }
    {
        double x = 0.0;
        for (int i = tid; i < TILE; i += ALL) x += (double)S[i] * (double)dS[i];       // (the same order in both)
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (lane == 0) through_of[tid >> 5] = x;
    }
    __syncthreads();
    // dq = E k + scale 2^G_t dout S^T
    c.zero();
    multiply<false, false>(c, O, S, 0, ev, tid);
    scale_rows(c, Q, q_dots[0], [&](int t) { return a.scale * exp2_of(G[t]); }, tid);
    multiply<false, true>(c, E, K, 0, min(diagonal + 2, last), tid);
    each(c, tid, [&](int t, int d, float &x) { if (t < all && d < a.Dk) put_qk(a.dq, dq_heads, t, d, t < tokens ? x : 0.f); });
    // dk = E^T q + 2^(G_C - G_s) v dS^T
    c.zero();
    multiply<false, false>(c, V, dS, 0, ev, tid);
    scale_rows(c, K, k_dots[0], [&](int s) { return exp2_diff(end, G[s]); }, tid);
    multiply<true, true>(c, E, Q, diagonal, last, tid);
    each(c, tid, [&](int s, int d, float &x) { if (s < all && d < a.Dk) put_qk(a.dk, dk_heads, s, d, s < tokens ? x : 0.f); });
    // dv = P^T dout + 2^(G_C - G_s) k dS
    c.zero();
    multiply<false, true>(c, K, dS, 0, ek, tid);
    each(c, tid, [&](int s, int, float &x) { x *= exp2_diff(end, G[s]); });
    multiply<true, true>(c, P, O, diagonal, last, tid);
    each(c, tid, [&](int s, int d, float &x) { if (s < all && d < a.Dv) dv[s * a.dv.ts + d] = s < tokens ? x : 0.f; });
    __syncthreads();
    // the decays' gradient: sum over u >= t of dG_u, the shares of k_s for s < t, and what passes from the state before the chunk to that behind it
    double own = 0.0, before = 0.0;
    if (tid < C) {
        double kd = 0.0;
        for (int w = 0; w < 4; ++w) {
            own += (double)rows[w][tid] - (double)columns[w][tid] + (double)q_dots[w][tid];
            kd += (double)k_dots[w][tid];
        }
        before = running_sum<C>(kd - own, sums, tid) - (kd - own);
        for (int o = 16; o; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
        if (lane == 0) totals[tid >> 5] = own;
    }
    __syncthreads();
    if (tid < all) {
        double through = 0.0;
        for (int w = 0; w < ALL / 32; ++w) through += through_of[w];
        const double x = before + (tid >= 32 ? sums[0] : 0.0) + totals[0] + totals[1] + through * (double)exp2_of(end);
        seq::store_f(a.ddecay.p, gb + tid * a.ddecay.ts, a.decay_bf16, tid < tokens ? (float)x : 0.f);
    }
}

// dq and dk of heads that share q and k: the sum over each group, one rounding.  V neighbouring elements a thread.  Bytes bound it: 6400
// tokens, 8 heads of 64 summed in pairs, fp32, 39 MB in 9.5 us (4.1 TB/s, the sums come out of L2).
template <class T, int V>
__global__ void k_sum_groups(const __grid_constant__ qgru_attention a, const float *dq, const float *dk) {
    const int g = a.H / a.Hk, per_head = a.Dk / V;
    const long long n = (long long)a.T * a.B * a.Hk * per_head;
    const qgru_seq_tensor to = blockIdx.y ? a.dk : a.dq;
    const float *from = blockIdx.y ? dk : dq;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (long long)gridDim.x * blockDim.x) {
        const long long head = e / per_head, tb = head / a.Hk;
        const int d = (int)(e - head * per_head) * V, hk = (int)(head - tb * a.Hk);
        const float *p = from + (tb * a.H + (long long)hk * g) * a.Dk + d;
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = 0.f;
        for (int i = 0; i < g; ++i) {
            if constexpr (V == 4) {
                const float4 u = *reinterpret_cast<const float4 *>(p + (long long)i * a.Dk);
                s[0] += u.x;
                s[1] += u.y;
                s[2] += u.z;
                s[3] += u.w;
            } else {
                s[0] += p[(long long)i * a.Dk];
            }
        }
        T *q = static_cast<T *>(to.p) + tb / a.B * to.ts + tb % a.B * to.bs + hk * to.hs + d;
#pragma unroll
        for (int j = 0; j < V; ++j) q[j] = seq::from_f<T>(s[j]);
    }
}

template <class F>
int with_smem(F *kernel, size_t bytes) {
    SEQ_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return QGRU_OK;
}

template <class T, bool Reverse>
int run_states(const qgru_attention &a, const Cut &c, float *states, char *seg, cudaStream_t st) {
    Pass p{};
    p.k = Reverse ? a.q : a.k;
    p.v = Reverse ? a.dout : a.v;
    p.k_share = a.H / a.Hk;
    p.first = Reverse ? a.dstate : a.state0;
    p.last = Reverse ? a.dstate0 : a.state;
    p.segments = c.segments;
    p.per = c.per;
    p.chunks = c.chunks;
    const dim3 grid(a.B * a.H, (unsigned)((a.Dk + 63) / 64 * ((a.Dv + 63) / 64)), c.segments);
    if (c.segments > 1) {
        p.seg_state = reinterpret_cast<float *>(seg);
        p.seg_log = p.seg_state + c.segments * state_elems(a);
        p.own_sums = true;
        k_states<T, Reverse><<<grid, THREADS, 0, st>>>(a, p);
        SEQ_CK(cudaGetLastError());
        if (const int rc = scan_segments(a, c, Reverse, seg, st)) return rc;
    }
    p.states = states;
    p.own_sums = false;
    k_states<T, Reverse><<<grid, THREADS, 0, st>>>(a, p);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

template <class T>
int forward(const qgru_attention &a, const Cut &c, cudaStream_t st) {
    float *states = static_cast<float *>(a.keep ? a.states : a.workspace);
    char *seg = static_cast<char *>(a.workspace) + (a.keep ? 0 : a256(c.states));
    if (const int rc = run_states<T, false>(a, c, states, seg, st)) return rc;
    if (c.chunks == 0) return QGRU_OK;
    if (std::is_same<T, float>::value && a.Dk <= 64 && a.Dv <= 64) {
        constexpr size_t bytes = 5 * TILE * sizeof(float);
        if (const int rc = with_smem(k_outputs_small, bytes)) return rc;
        k_outputs_small<<<c.chunks * a.B * a.H, THREADS, bytes, st>>>(a, states);
        SEQ_CK(cudaGetLastError());
        return QGRU_OK;
    }
    constexpr size_t bytes = 3 * TILE * sizeof(float);
    if (const int rc = with_smem(k_outputs<T>, bytes)) return rc;
    k_outputs<T><<<c.chunks * a.B * a.H, THREADS, bytes, st>>>(a, states);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

template <class T>
int backward(const qgru_attention &a, const Cut &c, cudaStream_t st) {
    char *ws = static_cast<char *>(a.workspace);
    float *dstates = reinterpret_cast<float *>(ws);
    ws += a256(c.states);
    char *seg = ws;
    ws += a256(c.seg);
    if (const int rc = run_states<T, true>(a, c, dstates, seg, st)) return rc;
    if (c.chunks == 0) return QGRU_OK;
    float *dq = nullptr, *dk = nullptr;
    if (a.H != a.Hk) {
        dq = reinterpret_cast<float *>(ws);
        dk = dq + group_bytes(a) / 8;
    }
    const float *states = static_cast<const float *>(a.states);
    if (std::is_same<T, float>::value && a.Dk <= 64 && a.Dv <= 64) {
        constexpr size_t bytes = 8 * TILE * sizeof(float);
        if (const int rc = with_smem(k_gradients_small, bytes)) return rc;
        k_gradients_small<<<c.chunks * a.B * a.H, ALL, bytes, st>>>(a, states, dstates, dq, dk);
    } else {
        constexpr size_t bytes = 4 * TILE * sizeof(float);
        if (const int rc = with_smem(k_gradients<T>, bytes)) return rc;
        k_gradients<T><<<c.chunks * a.B * a.H, THREADS, bytes, st>>>(a, states, dstates, dq, dk);
    }
    SEQ_CK(cudaGetLastError());
    return dq ? sum_groups(a, dq, dk, st) : QGRU_OK;
}

// ------------------------------------------------------------------------------------ single tokens
// One CTA per (row, head, 128 columns of the state): a lane has V neighbouring columns of a state row, W lanes a row and 256 / W rows at
// a time, U of them in flight.  Bytes bound it: the state, read and written once.  256 rows of 16 states of 128 x 128, 541 MB: 83 us, 6.5
// TB/s.  One row of 4 states of 64 x 64: 2.8 us, the launch.
template <class T, int V>
__global__ void __launch_bounds__(256) k_step(const __grid_constant__ qgru_attention a, long long state_bs, long long state_hs, int W) {
    constexpr int U = 8;
    __shared__ float qs[MAX_D], ks[MAX_D], part[256 * V];
    const int tid = threadIdx.x, b = blockIdx.x / a.H, h = blockIdx.x % a.H, hk = h / (a.H / a.Hk);
    const int lane = tid % W, group = tid / W, groups = 256 / W, j = blockIdx.y * 32 * V + lane * V;
    const bool on = j < a.Dv;
    float *S = a.state + b * state_bs + h * state_hs + j;
    float s[U][V];
    const auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
            if (!on || r >= a.Dk) continue;
            if constexpr (V == 4)
                *reinterpret_cast<float4 *>(s[u]) = *reinterpret_cast<const float4 *>(S + (long long)r * a.Dv);
            else
                s[u][0] = S[(long long)r * a.Dv];
        }
    };
    fetch(group);
    const T *q = static_cast<const T *>(a.q.p) + at(a.q, b, hk), *k = static_cast<const T *>(a.k.p) + at(a.k, b, hk);
    for (int d = tid; d < a.Dk; d += 256) {
        qs[d] = seq::to_f(q[d]);
        ks[d] = seq::to_f(k[d]);
    }
    const float g = seq::load_f(a.decay.p, at(a.decay, b, h), a.decay_bf16), keep = expf(g);
    float v[V], o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] = on ? seq::to_f(static_cast<const T *>(a.v.p)[at(a.v, b, h) + j + i]) : 0.f;
        o[i] = 0.f;
    }
    __syncthreads();
    for (int r0 = group; r0 < a.Dk; r0 += U * groups) {
        if (r0 != group) fetch(r0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
            if (!on || r >= a.Dk) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[u][i] = fmaf(ks[r], v[i], keep * s[u][i]);
                o[i] = fmaf(qs[r], s[u][i], o[i]);
            }
            if constexpr (V == 4)
                *reinterpret_cast<float4 *>(S + (long long)r * a.Dv) = *reinterpret_cast<const float4 *>(s[u]);
            else
                S[(long long)r * a.Dv] = s[u][0];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part[tid * V + i] = o[i];
    __syncthreads();
    for (int c = tid; c < W * V; c += 256) {
        float x = 0.f;
        for (int g2 = 0; g2 < groups; ++g2) x += part[g2 * W * V + c];
        const int col = blockIdx.y * 32 * V + c;
        if (col < a.Dv) static_cast<T *>(a.out.p)[at(a.out, b, h) + col] = seq::from_f<T>(a.scale * x);
    }
}

template <class T>
int step(const qgru_attention &a, long long bs, long long hs, cudaStream_t st) {
    const bool wide = a.Dv % 4 == 0 && bs % 4 == 0 && hs % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
    const int V = wide ? 4 : 1, vectors = (a.Dv + V - 1) / V;
    int W = 1;
    while (W < vectors && W < 32) W *= 2;
    const dim3 grid(a.B * a.H, (a.Dv + 32 * V - 1) / (32 * V));
    if (wide)
        k_step<T, 4><<<grid, 256, 0, st>>>(a, bs, hs, W);
    else
        k_step<T, 1><<<grid, 256, 0, st>>>(a, bs, hs, W);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

}  // namespace

size_t group_bytes(const qgru_attention &a) { return a.H == a.Hk ? 0 : 2 * sizeof(float) * (size_t)a.T * a.B * a.H * a.Dk; }

int sum_groups(const qgru_attention &a, const float *dq, const float *dk, cudaStream_t st) {
    const bool wide = a.Dk % 4 == 0;
    const long long n = (long long)a.T * a.B * a.Hk * a.Dk / (wide ? 4 : 1);
    const dim3 grid((unsigned)std::min<long long>((n + 255) / 256, 4096), 2);
    const auto run = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(a, dq, dk); };
    a.bf16 ? (wide ? run(k_sum_groups<bf16, 4>) : run(k_sum_groups<bf16, 1>)) : (wide ? run(k_sum_groups<float, 4>) : run(k_sum_groups<float, 1>));
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

int scan_segments(const qgru_attention &a, const Cut &c, bool reverse, char *seg, cudaStream_t st) {
    float *s = reinterpret_cast<float *>(seg);
    const long long n = (long long)state_elems(a);
    k_scan_segments<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(s, s + c.segments * n, reverse ? a.dstate : a.state0, c.segments, n, a.Dk * a.Dv);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

// Segments: where the heads alone leave half of two CTAs an SM idle, of two chunks at the least (each token's k and v are read once more
// for it).
Cut generic_cut(const qgru_attention &a, int sms) {
    Cut c;
    c.chunk = C;
    c.chunks = (a.T + C - 1) / C;
    const long long units = (long long)a.B * a.H * ((a.Dk + 63) / 64) * ((a.Dv + 63) / 64);
    c.segments = (int)std::max<long long>(1, std::min<long long>(c.chunks / 2, 2 * sms / std::max<long long>(units, 1)));
    c.per = std::max(1, (c.chunks + c.segments - 1) / c.segments);
    c.segments = std::max(1, (c.chunks + c.per - 1) / c.per);
    c.states = sizeof(float) * c.chunks * state_elems(a);
    c.seg = c.segments > 1 ? sizeof(float) * c.segments * (state_elems(a) + (size_t)a.B * a.H) : 0;
    return c;
}
int generic_forward(const qgru_attention &a, const Cut &c, cudaStream_t st) { return a.bf16 ? forward<bf16>(a, c, st) : forward<float>(a, c, st); }
int generic_backward(const qgru_attention &a, const Cut &c, cudaStream_t st) { return a.bf16 ? backward<bf16>(a, c, st) : backward<float>(a, c, st); }

namespace {

int check(const qgru_attention *a) {
    using seq::fail;
    if (!a) return fail(QGRU_ERR_BAD_ARG, "null argument block");
    if (a->T < 0 || a->B < 0 || a->H < 1 || a->Hk < 1 || a->Dk < 1 || a->Dv < 1) return fail(QGRU_ERR_BAD_ARG, "sizes must be positive (T and B may be 0)");
    if (a->H % a->Hk) return fail(QGRU_ERR_BAD_ARG, "%d heads cannot share %d heads of q and k", a->H, a->Hk);
    if (a->Dk > MAX_D || a->Dv > MAX_D) return fail(QGRU_ERR_UNSUPPORTED, "head sizes are at most %d, got %d and %d", MAX_D, a->Dk, a->Dv);
    if (a->T > 1 << 30 || (long long)a->B * a->H > 2147483647ll || (long long)a->B * a->H * ((a->T + 63) / 64) > 2147483647ll)
        return fail(QGRU_ERR_UNSUPPORTED, "at most 2^30 tokens, and 2^31 chunks of 64 tokens over all sequences and heads");
    return QGRU_OK;
}

int cut(const qgru_attention &a, Cut *c, int *sms) {
    SEQ_CK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, a.device));
    *c = tc_takes(a) ? tc_cut(a, *sms) : generic_cut(a, *sms);
    return QGRU_OK;
}

}  // namespace
}  // namespace attn
}  // namespace qgru

using namespace qgru;

extern "C" {

int qgru_attention_sizes(const qgru_attention *a, size_t *states_bytes, size_t *forward_workspace, size_t *backward_workspace) {
    if (const int rc = attn::check(a)) return rc;
    attn::Cut c;
    int sms = 0;
    if (const int rc = attn::cut(*a, &c, &sms)) return rc;
    const bool walks = attn::tc_takes(*a) && attn::walk_takes(*a, false);
    if (states_bytes) *states_bytes = a->keep ? attn::a256(c.states) : 0;
    if (forward_workspace) *forward_workspace = attn::a256(c.seg) + (a->keep || walks ? 0 : attn::a256(c.states));
    if (backward_workspace) *backward_workspace = attn::a256(c.states) + attn::a256(c.seg) + attn::a256(c.through) + attn::group_bytes(*a);
    return QGRU_OK;
}

static int attention_run(const qgru_attention *a, bool backward, void *stream) {
    if (const int rc = attn::check(a)) return rc;
    if (a->B == 0) return QGRU_OK;
    if (backward && !a->keep) return seq::fail(QGRU_ERR_BAD_ARG, "the forward has not kept its states");
    size_t states = 0, fwd = 0, bwd = 0;
    if (const int rc = qgru_attention_sizes(a, &states, &fwd, &bwd)) return rc;
    const size_t ws = backward ? bwd : fwd;
    if (a->T > 0 && (!a->q.p || !a->k.p || !a->v.p || !a->decay.p)) return seq::fail(QGRU_ERR_BAD_ARG, "null input");
    if (a->T > 0 && (backward ? !a->dout.p || !a->dq.p || !a->dk.p || !a->dv.p || !a->ddecay.p : !a->out.p)) return seq::fail(QGRU_ERR_BAD_ARG, "null output or gradient");
    if ((states && !a->states) || a->states_bytes < states) return seq::fail(QGRU_ERR_BAD_ARG, "states needs %zu bytes, got %zu", states, a->states_bytes);
    if ((ws && !a->workspace) || a->workspace_bytes < ws) return seq::fail(QGRU_ERR_BAD_ARG, "workspace needs %zu bytes, got %zu", ws, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->states) | reinterpret_cast<uintptr_t>(a->workspace)) % 256) return seq::fail(QGRU_ERR_BAD_ARG, "states and workspace must be aligned to 256 bytes");
    if (const int rc = seq::check_expiry(a->device)) return rc;
    const seq::OnDevice on(a->device);
    SEQ_CK(on.error());
    attn::Cut c;
    int sms = 0;
    if (const int rc = attn::cut(*a, &c, &sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (attn::tc_takes(*a)) {
        int *flag = nullptr;
        if (const int rc = seq::expiry_flag(a->device, &flag)) return rc;
        return backward ? attn::tc_backward(*a, c, flag, sms, st) : attn::tc_forward(*a, c, flag, sms, st);
    }
    return backward ? attn::generic_backward(*a, c, st) : attn::generic_forward(*a, c, st);
}

int qgru_attention_forward(const qgru_attention *a, void *stream) { return attention_run(a, false, stream); }
int qgru_attention_backward(const qgru_attention *a, void *stream) { return attention_run(a, true, stream); }

int qgru_attention_step(const qgru_attention *a, long long state_bs, long long state_hs, void *stream) {
    if (const int rc = attn::check(a)) return rc;
    if (a->B == 0) return QGRU_OK;
    if (!a->q.p || !a->k.p || !a->v.p || !a->decay.p || !a->out.p || !a->state) return seq::fail(QGRU_ERR_BAD_ARG, "null tensor");
    if (a->T != 1 || a->lengths) return seq::fail(QGRU_ERR_BAD_ARG, "a step takes one token of every sequence");
    if (const int rc = seq::check_expiry(a->device)) return rc;
    const seq::OnDevice on(a->device);
    SEQ_CK(on.error());
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->bf16 ? attn::step<__nv_bfloat16>(*a, state_bs, state_hs, st) : attn::step<float>(*a, state_bs, state_hs, st);
}

}  // extern "C"
