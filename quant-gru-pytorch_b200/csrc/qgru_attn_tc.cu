// qgru_attn_tc.cu - linear attention on the tensor cores: the gradients, and the state pass and outputs of tensors that TMA does not take
// (rows or strides that are no multiple of 16 bytes, strides of 0).  bf16, head sizes up to 128 (padded to 64 or 128), chunks of 128 tokens.
//
// Outputs and gradients take every chunk by itself, from the states that a pass over the chunks has left.  Rounded to 16 bits (two
// bf16 parts, 2^-16 of the value) on the way are the weights of the pairs of tokens (P, E), and the state before a chunk and its gradient
// behind it where they are factors of a product.  The states themselves are fp32: their products take k scaled by the decays as three bf16 parts (24 bits).
#include <algorithm>
#include <type_traits>

#include "qgru_attn.cuh"
#include "qgru_attn_tc.cuh"
#include "qgru_tc.cuh"

namespace qgru {
namespace attn {
namespace {

using namespace tile;
constexpr int THREADS = 256;

// Rows t0 .. t0 + 127 of a tensor (zeros from `tokens` on and behind its columns) as a tile of D columns, element by element.
template <int D, int N = THREADS>
__device__ __forceinline__ void load_rows(uint32_t tile, const qgru_seq_tensor &x, long long base, int t0, int tokens, int d, int tid) {
    const bf16 *p = static_cast<const bf16 *>(x.p) + base + (long long)t0 * x.ts;
    constexpr int PER_ROW = D / 8;
#pragma unroll
    for (int i = 0; i < C * PER_ROW / N; ++i) {
        const int e = i * N + tid, r = e / PER_ROW, c = e % PER_ROW;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d0 = c * 8 + 2 * j;
            const uint32_t u0 = r < tokens && d0 < d ? __bfloat16_as_ushort(p[r * x.ts + d0]) : 0u;
            const uint32_t u1 = r < tokens && d0 + 1 < d ? __bfloat16_as_ushort(p[r * x.ts + d0 + 1]) : 0u;
            w[j] = u0 | u1 << 16;
        }
        sts16(tile + (c >> 3) * PANEL + chunk_at(r, c & 7), w[0], w[1], w[2], w[3]);
    }
}
// `Bytes` of a state as it is kept before each chunk.
template <int Bytes, int N = THREADS>
__device__ __forceinline__ void load_state(uint32_t to, const bf16 *S, int tid) {
#pragma unroll
    for (int i = 0; i < Bytes / 16 / N; ++i) cp_async(to + (i * N + tid) * 16, S + (i * N + tid) * 8, 16);
}
struct Shared {                 // behind the tiles
    float2 G[C];                // running sums of the decays, base 2
    float f[C];                 // factors of a token
    long long g_sums[4];
    double sums[4];
    uint64_t bar[6];
    uint32_t tmem;
    int failed;
};

__device__ __forceinline__ long long load_decay(const qgru_attention &a, int b, int h, int t0, int tokens, int tid) {
    return tid < tokens ? decay_units(a, at(a.decay, b, h) + (long long)(t0 + tid) * a.decay.ts) : 0;
}
// G of the chunk from the threads' decays (the first 128; two __syncthreads).
__device__ __forceinline__ void sum_decays(Shared &s, long long g, int tid) {
    if (tid < C) g = running_sum<C>(g, s.g_sums, tid);
    __syncthreads();
    if (tid < C) {
        for (int w = 0; w < tid >> 5; ++w) g += s.g_sums[w];
        s.G[tid] = two_floats(g);
    }
    __syncthreads();
}
__device__ __forceinline__ void begin(Shared &s, uint32_t columns, int tid) {
    if (tid == 0) {
        for (int i = 0; i < 6; ++i) tc::mbar_init(&s.bar[i], 1);
        s.failed = 0;
        tc::fence_barrier_init();
    }
    if (tid < 32) tc::tmem_alloc(&s.tmem, columns);
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
}
// Every warp's wait for products: false once one has run out (all warps of the CTA then leave at the next common point).
__device__ __forceinline__ void await(Shared &s, int bar, uint32_t parity) {
    if (!tc::mbar_wait(&s.bar[bar], parity, WAIT_BUDGET)) s.failed = 1;
    tc::tc_fence_after_sync();
}
__device__ __forceinline__ void end(Shared &s, uint32_t columns, int *flag, int tid) {
    tc::tc_fence_before_sync();
    __syncthreads();
    if (s.failed) {            // copies and products may be under way: a millisecond is far more than they take
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) {
        }
        if (tid == 0) *flag = 1;
    }
    if (tid < 32) tc::tmem_dealloc(s.tmem, columns);
}
__device__ __forceinline__ unsigned char *tiles_of(unsigned char *raw) {
    return reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
}

// ------------------------------------------------------------------------------------- state pass
struct Pass {
    qgru_seq_tensor k, v;
    int k_share;
    const float *first;
    float *last;
    bf16 *states;                  // before each chunk in the pass's order, [chunks][B H][2 parts][DV / 8][DK][8]
    bool own_sums;                 // instead: each segment's sum, from zero
    const bf16 *other;             // from the end: the forward's states, and where their products with these go
    float *through;
    float *seg_state, *seg_log;
    int segments, per, chunks;
    int *flag;
};
template <int DK, int DV>
constexpr int STATES_TILES = DK / 64 * PANEL + 2 * (DV / 64) * PANEL + 3 * (DK / 64) * PANEL;

// grid (B H, segments).  S' = 2^G_C S + (w k)^T v: lane i of tensor memory is row i of the state, whose fp32 sums stay in
// registers, half a row a thread.  While the products of a chunk run, the next one's tokens are read and the state before this one
// leaves.  With DK = 64 lanes 64 .. 127 repeat the first 64 (M is 128) and are not read.  One chunk's chain of load, split, product and
// conversion bounds it, eight in turn: 16 x 1000 tokens of 8 heads of 60, 63 us.
template <int DK, int DV, bool Reverse>
__global__ void __launch_bounds__(THREADS) k_states_tc(const __grid_constant__ qgru_attention a, const __grid_constant__ Pass p) {
    extern __shared__ unsigned char raw[];
    unsigned char *tiles = tiles_of(raw);
    Shared &s = *reinterpret_cast<Shared *>(tiles + STATES_TILES<DK, DV>);
    constexpr int KT = DK / 64 * PANEL, VT = DV / 64 * PANEL, HALF = DV / 2;
    const uint32_t k_raw = tc::smem_u32(tiles), v_raw = k_raw + KT, parts = v_raw + 2 * VT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bh = blockIdx.x, b = bh / a.H, h = bh % a.H, seg = blockIdx.y;
    const int n = valid_tokens(a, b), row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * HALF;
    const bool mine = (warp & 3) * 32 < DK;
    const long long kb = at(p.k, b, h / p.k_share), vb = at(p.v, b, h), dense = (long long)bh * a.Dk * a.Dv, dense_all = (long long)gridDim.x * a.Dk * a.Dv;
    const bool own_sums = p.own_sums;
    float S[HALF];
    const float *first = own_sums ? nullptr : p.segments > 1 ? p.seg_state + seg * dense_all : p.first;
#pragma unroll
    for (int i = 0; i < HALF; ++i) S[i] = first && row < a.Dk && c0 + i < a.Dv ? first[dense + (long long)row * a.Dv + c0 + i] : 0.f;
    begin(s, DV == 64 ? 64 : 128, tid);
    const uint32_t U = lane_base(s.tmem, warp) + c0;
    // the chunks with tokens, in the pass's order
    int c = seg * p.per;
    const int c_end = min((seg + 1) * p.per, p.chunks), used = (n + C - 1) / C;
    const auto chunk_of = [&](int i) { return Reverse ? p.chunks - 1 - i : i; };
    const auto leave = [&](int chunk) {            // the state before the chunk
        if (own_sums || !mine) return;
        uint4 *to = reinterpret_cast<uint4 *>(p.states + ((long long)chunk * gridDim.x + bh) * (2 * DK * DV) + (c0 * DK + row * 8));
#pragma unroll
        for (int i = 0; i < HALF; i += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 x = make_float2(S[i + 2 * j], S[i + 2 * j + 1]);
                hi[j] = pack_part(x);
                lo[j] = pack(rest(x, hi[j]));
            }
            to[i / 8 * DK] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            to[DK * DV / 8 + i / 8 * DK] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    };
    const auto fetch = [&](int i) {
        const int t0 = chunk_of(i) * C, tokens = min(max(n - t0, 0), C);
        load_rows<DK>(k_raw, p.k, kb, t0, tokens, a.Dk, tid);
        load_rows<DV>(v_raw + (i & 1) * VT, p.v, vb, t0, tokens, a.Dv, tid);
    };
    if (Reverse) {                                 // those behind the sequence: nothing reads the state there
        c = max(c, p.chunks - used);
    }
    const int stop = Reverse ? c_end : min(c_end, used);
    double all = 0.0;
    long long g = 0;
    uint32_t phase = 0;
    if (c < stop) {
        fetch(c);
        g = load_decay(a, b, h, chunk_of(c) * C, min(n - chunk_of(c) * C, C), tid);
    }
    for (; c < stop; ++c) {
        const int chunk = chunk_of(c);
        sum_decays(s, g, tid);
        const float2 last = s.G[C - 1];
        if (tid < C) s.f[tid] = Reverse ? a.scale * exp2_of(s.G[tid]) : exp2_diff(last, s.G[tid]);
        __syncthreads();
        // w k as the sum of three bf16 values; the parts lie as k does
#pragma unroll 2
        for (int i = 0; i < C * DK / 8 / THREADS; ++i) {
            const int e = i * THREADS + tid, r = e / (DK / 8), ch = e % (DK / 8);
            const uint32_t off = (ch >> 3) * PANEL + chunk_at(r, ch & 7);
            const uint4 q = lds16(k_raw + off);
            const uint32_t in[4] = {q.x, q.y, q.z, q.w};
            const float w = s.f[r];
            uint32_t o[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 x = make_float2(low(in[j]) * w, high(in[j]) * w);
#pragma unroll
                for (int t = 0; t < 3; ++t) {
                    o[t][j] = t < 2 ? pack_part(x) : pack(x);
                    if (t < 2) x = rest(x, o[t][j]);
                }
            }
#pragma unroll
            for (int t = 0; t < 3; ++t) sts16(parts + t * KT + off, o[t][0], o[t][1], o[t][2], o[t][3]);
        }
        fence_async();
        tc::tc_fence_before_sync();
        __syncthreads();
        if (tid < 32) {
            const uint32_t leader = elect();
            tc::tc_fence_after_sync();
            const Operand v{v_raw + (uint32_t)(c & 1) * VT, PANEL};
            for (int t = 2; t >= 0; --t) {
                const Operand k{parts + (uint32_t)t * KT, DK == 64 ? 0 : PANEL};
                product<true, true, DV, C>(leader, s.tmem, k, v, t != 2);
            }
            commit(leader, &s.bar[0]);
        }
        if (c + 1 < stop) {
            fetch(c + 1);
            g = load_decay(a, b, h, chunk_of(c + 1) * C, min(n - chunk_of(c + 1) * C, C), tid);
        }
        leave(chunk);
        if (Reverse && !own_sums) {
            const long long head = (long long)chunk * gridDim.x + bh;
            float sum = 0.f;
            if (mine) {
                const uint4 *o = reinterpret_cast<const uint4 *>(p.other + head * (2 * DK * DV) + (c0 * DK + row * 8));
                float2 x = both(0.f);
#pragma unroll
                for (int i = 0; i < HALF; i += 8) {
                    const float2 u[4] = {make_float2(S[i], S[i + 1]), make_float2(S[i + 2], S[i + 3]), make_float2(S[i + 4], S[i + 5]), make_float2(S[i + 6], S[i + 7])};
                    x = dot8(o[DK * DV / 8 + i / 8 * DK], u, x);
                    x = dot8(o[i / 8 * DK], u, x);
                }
                sum = x.x + x.y;
            }
            for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
            if (lane == 0) p.through[head * THROUGH + warp] = sum;
        }
        const float whole = exp2_of(last);
        all += (double)last.x + (double)last.y;
        await(s, 0, phase);
        phase ^= 1;
        if (mine) {
            float u[HALF];
            tmem_load(U, u);
#pragma unroll
            for (int i = 0; i < HALF; ++i) S[i] = fmaf(whole, S[i], u[i]);
        }
        tc::tc_fence_before_sync();
        __syncthreads();
        if (s.failed) break;
    }
    float *to = own_sums ? p.seg_state + seg * dense_all : p.last && seg == p.segments - 1 ? p.last : nullptr;
    if (to) {
#pragma unroll
        for (int i = 0; i < HALF; ++i)
            if (row < a.Dk && c0 + i < a.Dv) to[dense + (long long)row * a.Dv + c0 + i] = S[i];
    }
    if (own_sums && tid == 0) p.seg_log[seg * gridDim.x + bh] = (float)all;
    end(s, DV == 64 ? 64 : 128, p.flag, tid);
}

// ------------------------------------------------------------------------------------- outputs
template <int DK, int DV>
constexpr int OUTPUTS_TILES = 2 * (DK / 64) * PANEL + DV / 64 * PANEL;

// grid: chunks x B H, the heads of one chunk beside each other.  Two threads a token, each half of the pairs' weights and half of the
// output's columns.  The state lies where k was once q k^T is there.  Two CTAs an SM cover each other's waits; the element loads of what
// TMA does not take bound it: 16 x 1000 tokens of 8 heads of 60, 119 us (64, by TMA, in k_walk: 34 with the states).
template <int DK, int DV>
__global__ void __launch_bounds__(THREADS, 2) k_outputs_tc(const __grid_constant__ qgru_attention a, const bf16 *states, int *flag) {
    extern __shared__ unsigned char raw[];
    unsigned char *tiles = tiles_of(raw);
    Shared &s = *reinterpret_cast<Shared *>(tiles + OUTPUTS_TILES<DK, DV>);
    constexpr int KT = DK / 64 * PANEL, HALF = DV / 2;
    const uint32_t q_t = tc::smem_u32(tiles), k_t = q_t + KT, v_t = k_t + KT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, heads = a.B * a.H, chunk = blockIdx.x / heads, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H;
    const int t0 = chunk * C, all = min(a.T - t0, C), tokens = min(max(valid_tokens(a, b) - t0, 0), C);
    const int block = warp & 3, row = block * 32 + lane, half = warp >> 2, c0 = half * HALF;
    bf16 *out = static_cast<bf16 *>(a.out.p) + at(a.out, b, h) + (long long)(t0 + row) * a.out.ts;
    const bool vec_out = a.Dv % 8 == 0 && (a.out.ts | a.out.bs | a.out.hs) % 8 == 0 && reinterpret_cast<uintptr_t>(a.out.p) % 16 == 0;
    float o[HALF];
    if (tokens == 0) {
#pragma unroll
        for (int i = 0; i < HALF; ++i) o[i] = 0.f;
        if (row < all) store_row(out, o, c0, a.Dv, vec_out);
        return;
    }
    const int hk = h / (a.H / a.Hk);
    const bool carried = chunk > 0 || a.state0;
    const bf16 *S = states + ((long long)chunk * heads + bh) * (2 * DK * DV);
    load_rows<DK>(q_t, a.q, at(a.q, b, hk), t0, tokens, a.Dk, tid);
    load_rows<DK>(k_t, a.k, at(a.k, b, hk), t0, tokens, a.Dk, tid);
    load_rows<DV>(v_t, a.v, at(a.v, b, h), t0, tokens, a.Dv, tid);
    const long long g = load_decay(a, b, h, t0, tokens, tid);
    begin(s, 256, tid);
    const uint32_t base = lane_base(s.tmem, warp);
    fence_async();
    sum_decays(s, g, tid);
    if (tid < 32) {
        const uint32_t leader = elect();
        tc::tc_fence_after_sync();
        product<false, false, C, DK>(leader, s.tmem, Operand{q_t, PANEL}, Operand{k_t, PANEL}, false);
        commit(leader, &s.bar[0]);
    }
    // Blocks of 32 x 32 pairs.  Below the diagonal 2^(G_t - G_s) is a product of two factors, both at most 1: from s to the end of
    // its block and from there to t.
    if (tid < C) s.f[tid] = ex2_diff(s.G[tid | 31], s.G[tid]);
    await(s, 0, 0);
    __syncthreads();
    if (carried) {
        load_state<DK * DV * 2>(k_t, S, tid);
        cp_commit();
    }
    const float2 G = s.G[row];
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
        const int sb = half * 2 + jb;                   // block of s
        uint32_t P[32];                                 // of each sixteen columns the large parts, then the small ones, in their place
        if (sb > block) {
#pragma unroll
            for (int i = 0; i < 32; ++i) P[i] = 0u;
        } else {
            float x[32];
            tmem_load(base + sb * 32, x);
            if (sb < block) {
                const float r = a.scale * ex2_diff(G, s.G[sb * 32 + 31]);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] *= r * s.f[sb * 32 + i];
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float w = a.scale * ex2_diff(G, s.G[sb * 32 + i]);
                    x[i] = i <= lane ? x[i] * w : 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const int at = (i & 16) + (i & 15) / 2;
                const float2 v = make_float2(x[i], x[i + 1]);
                P[at] = pack_part(v);
                P[at + 8] = pack(rest(v, P[at]));
            }
        }
        tmem_store(base + sb * 32, P);
    }
    tc::tmem_st_wait();
    cp_wait<0>();
    fence_async();
    tc::tc_fence_before_sync();
    __syncthreads();                                    // the pairs' weights and the state are there
    if (carried && tid < 32) {
        const uint32_t leader = elect();
        tc::tc_fence_after_sync();
        product_state<true, DV, DK, DK>(leader, s.tmem + 128, Operand{q_t, PANEL}, k_t, false);
        commit(leader, &s.bar[1]);
    }
    if (carried) {
        await(s, 1, 0);
        load_state<DK * DV * 2>(k_t, S + DK * DV, tid);      // its small part, where the large one was (no room for both beside a second CTA)
        cp_commit();
        cp_wait<0>();
        fence_async();
        tc::tc_fence_before_sync();
        __syncthreads();
        if (tid < 32) {
            const uint32_t leader = elect();
            tc::tc_fence_after_sync();
            product_state<true, DV, DK, DK>(leader, s.tmem + 128, Operand{q_t, PANEL}, k_t, true);
            commit(leader, &s.bar[3]);
        }
        await(s, 3, 0);
        tmem_load(base + 128 + c0, o);
        const float r = a.scale * ex2(G.x + G.y);
#pragma unroll
        for (int i = 0; i < HALF; ++i) o[i] *= r;
    } else {
#pragma unroll
        for (int i = 0; i < HALF; ++i) o[i] = 0.f;
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    if (tid < 32) {
        const uint32_t leader = elect();
        tc::tc_fence_after_sync();
        product_ts<true, DV, C>(leader, s.tmem + 128, s.tmem, Operand{v_t, PANEL}, false);
        commit(leader, &s.bar[2]);
    }
    await(s, 2, 0);
    float x[HALF];
    tmem_load(base + 128 + c0, x);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < HALF; ++i) odd |= !isfinite(x[i]);
    if (odd && row < tokens) {
        // A later token's infinity or NaN is none of an earlier one's business, and zero times it is NaN: the sums again, over the
        // tokens up to this one.
        const bf16 *q = static_cast<const bf16 *>(a.q.p) + at(a.q, b, hk) + (long long)(t0 + row) * a.q.ts;
        const bf16 *k = static_cast<const bf16 *>(a.k.p) + at(a.k, b, hk) + (long long)t0 * a.k.ts;
        const bf16 *v = static_cast<const bf16 *>(a.v.p) + at(a.v, b, h) + (long long)t0 * a.v.ts + c0;
#pragma unroll
        for (int i = 0; i < HALF; ++i) x[i] = 0.f;
        for (int t = 0; t <= row; ++t) {
            float w = 0.f;
            for (int d = 0; d < a.Dk; ++d) w = fmaf(seq::to_f(q[d]), seq::to_f(k[t * a.k.ts + d]), w);
            w *= a.scale * ex2_diff(G, s.G[t]);
#pragma unroll
            for (int i = 0; i < HALF; ++i)
                if (c0 + i < a.Dv) x[i] = fmaf(w, seq::to_f(v[t * a.v.ts + i]), x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < HALF; ++i) o[i] = row < tokens ? o[i] + x[i] : 0.f;
    if (row < all) store_row(out, o, c0, a.Dv, vec_out);
    end(s, 256, flag, tid);
}

// ------------------------------------------------------------------------------------- gradients
constexpr int GRAD_THREADS = 512;
struct Item {
    int index, b, h, t0, all, tokens;
};
struct Gradients {
    CUtensorMap q, k, v, o, dq, dk, dv;  // where TMA takes the tensors
    const bf16 *states, *dstates;
    const float *through;                // products of the two, THROUGH parts each
    float *dq_heads, *dk_heads;          // [T][B][H][Dk] where heads share q and k, else null
    int items;                           // chunks of all heads
    int *flag;
};
// Shared memory: q, k, v, dout; the two parts of a state (X, Y: first that of the gradient behind the chunk, then the one before it); the
// large part of E and the small one, which takes the place of X where a state is as large as it.
template <int DK, int DV>
struct Tiles {
    static constexpr int KT = DK / 64 * PANEL, VT = DV / 64 * PANEL, ST = DK * DV * 2, ET = 2 * PANEL;
    static constexpr bool SHARED = ST >= ET;
    static constexpr int K = KT, V = 2 * KT, O = V + VT, X = O + VT, Y = X + ST, E = Y + ST, E2 = SHARED ? X : E + ET, ALL = SHARED ? E + ET : E2 + ET;
    // where the results become rows of bf16 when all products are done
    static constexpr int DQ = DV == 128 ? X : E, DKEYS = DV == 128 ? Y : E2, DVALUES = DV == 128 ? E : X;
    static_assert(DV == 128 ? KT <= ST && VT <= ET : KT <= ET && VT <= 2 * ST, "the results fit");
};

// Sum over the lanes of a warp for each of 32 columns: lane i gets column i's.
__device__ __forceinline__ float sum_columns(float (&m)[32], int lane) {
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const float give = up ? m[i] : m[i + w], keep = up ? m[i + w] : m[i];
            m[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
        }
    }
    return m[0];
}
// sum of a row's Cols values, from column c0 on, times those of a tile
template <int Cols>
__device__ __forceinline__ float dot_row(uint32_t tile, int row, int c0, const float (&v)[Cols]) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < Cols; i += 8) {
        const int c = (c0 + i) / 8;
        const uint4 u = lds16(tile + (c >> 3) * PANEL + chunk_at(row, c & 7));
        const uint32_t in[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x = fmaf(v[i + 2 * j], low(in[j]), x);
            x = fmaf(v[i + 2 * j + 1], high(in[j]), x);
        }
    }
    return x;
}
// The sums of a row times a factor, back into tensor memory for the products that add to them; their product with the tile's row.
template <int Cols>
__device__ __forceinline__ float scale_sums(uint32_t taddr, float w, uint32_t tile, int row, int c0, bool dot) {
    float v[Cols];
    tmem_load(taddr, v);
    uint32_t r[Cols];
#pragma unroll
    for (int i = 0; i < Cols; ++i) {
        v[i] *= w;
        r[i] = __float_as_uint(v[i]);
    }
    tmem_store(taddr, r);
    return dot ? dot_row(tile, row, c0, v) : 0.f;
}

// A row's Cols values from column c0 on, as bf16, into a tile; and the tile's rows below `rows` into a tensor, whole lines at a time.
template <int Cols>
__device__ __forceinline__ void put_row(uint32_t tile, int row, int c0, const float (&v)[Cols]) {
#pragma unroll
    for (int i = 0; i < Cols; i += 8) {
        const int c = (c0 + i) / 8;
        sts16(tile + (c >> 3) * PANEL + chunk_at(row, c & 7), pack(v[i], v[i + 1]), pack(v[i + 2], v[i + 3]), pack(v[i + 4], v[i + 5]), pack(v[i + 6], v[i + 7]));
    }
}
template <int D, bool Zeros>
__device__ __forceinline__ void copy_out(uint32_t tile, const qgru_seq_tensor &x, long long base, int t0, int rows, int d, int tid) {
    bf16 *p = static_cast<bf16 *>(x.p) + base + (long long)t0 * x.ts;
    const bool vec = d % 8 == 0 && (x.ts | x.bs | x.hs) % 8 == 0 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0;
    constexpr int PER_ROW = D / 8;
#pragma unroll
    for (int i = 0; i < C * PER_ROW / GRAD_THREADS; ++i) {
        const int e = i * GRAD_THREADS + tid, r = e / PER_ROW, c = e % PER_ROW;
        if (r >= rows || c * 8 >= d) continue;
        const uint4 v = Zeros ? make_uint4(0u, 0u, 0u, 0u) : lds16(tile + (c >> 3) * PANEL + chunk_at(r, c & 7));
        bf16 *to = p + (long long)r * x.ts + c * 8;
        if (vec) {
            *reinterpret_cast<uint4 *>(to) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c * 8 + j < d) to[j] = __ushort_as_bfloat16((unsigned short)(w[j / 2] >> (j & 1) * 16));
        }
    }
}

// A CTA an SM, which takes chunk after chunk of all heads.  Pairs lie as [s][t] here, lane s of tensor memory.  Four blocks of 128 columns of it:
//   0  k q^T, then P^T in two parts     1  v dout^T, then dq     2  dk     3  dv
// Four threads a row, a quarter of the columns each.  P^T is the operand of dv from tensor memory, E^T that of dk (K in its columns) and
// of dq (K in its rows) from shared memory.  P, E and the states are two bf16 parts each: 16 bits of a factor, so that a result is the
// type's rounding of a sum that is nearly exact.  With one part, as much lost as by that rounding, the kernel took 92 us where it takes 100
// (16 x 1000 tokens of 8 heads of 128; bytes alone would take 56, 363 MB).
// The next chunk's tiles are fetched while this one's results leave (both by TMA), its decays are summed up beside this one's products,
// those of the state's gradient run beside the pairs, and the state before the chunk comes after them into the same place.  What bounds
// it is the chain of products, pairs and conversions between tensor memory and operands, and what of the loads it does not cover: 224 KB of
// operands leave no room for a second CTA or for tiles fetched earlier.  Heads of 64: 74 us; of 60, by the threads' own loads: 172.
template <int DK, int DV, bool Tma>
__global__ void __launch_bounds__(GRAD_THREADS) k_gradients_tc(const __grid_constant__ qgru_attention a, const __grid_constant__ Gradients p) {
    extern __shared__ unsigned char raw[];
    unsigned char *tiles = tiles_of(raw);
    using L = Tiles<DK, DV>;
    Shared &s = *reinterpret_cast<Shared *>(tiles + L::ALL);
    constexpr int KT = L::KT, VT = L::VT, ST = L::ST, KQ = DK / 4, VQ = DV / 4;
    const uint32_t q_t = tc::smem_u32(tiles), k_t = q_t + L::K, v_t = q_t + L::V, o_t = q_t + L::O, X_t = q_t + L::X, Y_t = q_t + L::Y, E_t = q_t + L::E, E2_t = q_t + L::E2;
    const uint32_t dq_t = q_t + L::DQ, dk_t = q_t + L::DKEYS, dv_t = q_t + L::DVALUES;
    // once v has been used, its tile holds sums by token
    float *t_sums = reinterpret_cast<float *>(tiles + 2 * KT);          // [4][128] over s of a block's lanes, for each t
    float *s_sums = t_sums + 4 * C, *q_dots = s_sums + 4 * C, *k_dots = q_dots + 4 * C;     // [4][128] each
    double *totals = reinterpret_cast<double *>(k_dots + 4 * C);        // [4]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, heads = a.B * a.H, share = a.H / a.Hk;
    const int block = warp & 3, row = block * 32 + lane, part = warp >> 2;
    const auto put_heads = [&](float *sums, const Item &x, const float (&v)[KQ]) {        // heads that share q and k: fp32, added up afterwards
        if (row >= x.all) return;
        const int c0 = part * KQ;
        float *to = sums + (((long long)(x.t0 + row) * a.B + x.b) * a.H + x.h) * a.Dk + c0;
#pragma unroll
        for (int i = 0; i < KQ; i += 4) {
            if (a.Dk % 4 == 0) {
                if (c0 + i < a.Dk) *reinterpret_cast<float4 *>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c0 + i + e < a.Dk) to[i + e] = v[i + e];
            }
        }
    };
    // The CTA's next chunk with tokens; those before it, behind the ends of their sequences, get zeros.
    const auto next_of = [&](long long index) {
        Item x{};
        for (; index < p.items; index += gridDim.x) {
            x.index = (int)index;
            x.b = x.index % heads / a.H;
            x.h = x.index % heads % a.H;
            x.t0 = x.index / heads * C;
            x.all = min(a.T - x.t0, C);
            x.tokens = min(max(valid_tokens(a, x.b) - x.t0, 0), C);
            if (x.tokens) return x;
            if (p.dq_heads) {
                const float z[KQ] = {};
                put_heads(p.dq_heads, x, z);
                put_heads(p.dk_heads, x, z);
            } else {
                copy_out<DK, true>(0, a.dq, at(a.dq, x.b, x.h), x.t0, x.all, a.Dk, tid);
                copy_out<DK, true>(0, a.dk, at(a.dk, x.b, x.h), x.t0, x.all, a.Dk, tid);
            }
            copy_out<DV, true>(0, a.dv, at(a.dv, x.b, x.h), x.t0, x.all, a.Dv, tid);
            if (tid < x.all) seq::store_f(a.ddecay.p, at(a.ddecay, x.b, x.h) + (long long)(x.t0 + tid) * a.ddecay.ts, a.decay_bf16, 0.f);
        }
        return x;                       // (no tokens)
    };
    // Tiles by TMA, by one thread: keys and queries; values and the output's gradient; the states.
    const auto fetch_qk = [&](const Item &x) {
        tc::mbar_expect_tx(&s.bar[4], 2 * KT + 2 * VT);
        for (int i = 0; i < DK / 64; ++i) {
            tma_load_4d(k_t + i * PANEL, &p.k, &s.bar[4], i * 64, x.t0, x.h / share, x.b);
            tma_load_4d(q_t + i * PANEL, &p.q, &s.bar[4], i * 64, x.t0, x.h / share, x.b);
        }
    };
    const auto fetch_vo = [&](const Item &x) {
        for (int i = 0; i < DV / 64; ++i) {
            tma_load_4d(v_t + i * PANEL, &p.v, &s.bar[4], i * 64, x.t0, x.h, x.b);
            tma_load_4d(o_t + i * PANEL, &p.o, &s.bar[4], i * 64, x.t0, x.h, x.b);
        }
    };
    // both parts of a state
    const auto fetch_state = [&](const bf16 *states, const Item &x) {
        tc::mbar_expect_tx(&s.bar[5], 2 * ST);
        bulk_load(X_t, states + (long long)x.index * (2 * DK * DV), 2 * ST, &s.bar[5]);
    };
    Item x = next_of(blockIdx.x);
    // The decays of a chunk are the second four warps': read early, summed up while the first four sum up the last chunk's gradient.
    const int token = tid - C;
    const bool decays = tid >= C && tid < 2 * C;
    const auto decay_of = [&](const Item &x) {
        return decays && token < x.tokens ? seq::load_f(a.decay.p, at(a.decay, x.b, x.h) + (long long)(x.t0 + token) * a.decay.ts, a.decay_bf16) : 0.f;
    };
    const auto put_decays = [&](long long g) {
        if (!decays) return;
        for (int w = 0; w < token >> 5; ++w) g += s.g_sums[w];
        s.G[token] = two_floats(g);
    };
    long long g = 0;
    {
        const float decay = decay_of(x);
        if (decays) g = running_sum<C>(decay_units(decay), s.g_sums, token);
    }
    begin(s, 512, tid);
    if constexpr (Tma) {
        if (tid == 0 && x.tokens) {
            fetch_qk(x);
            fetch_vo(x);
        }
    }
    put_decays(g);
    const uint32_t tm = s.tmem, base = lane_base(tm, warp);
    const Operand q{q_t, PANEL}, k{k_t, PANEL}, v{v_t, PANEL}, o{o_t, PANEL}, E{E_t, PANEL}, E2{E2_t, PANEL};
    for (uint32_t turn = 0; x.tokens; turn ^= 1) {
        const int b = x.b, h = x.h, hk = h / share, t0 = x.t0, all = x.all, tokens = x.tokens;
        if constexpr (!Tma) {
            load_rows<DK, GRAD_THREADS>(q_t, a.q, at(a.q, b, hk), t0, tokens, a.Dk, tid);
            load_rows<DK, GRAD_THREADS>(k_t, a.k, at(a.k, b, hk), t0, tokens, a.Dk, tid);
            load_rows<DV, GRAD_THREADS>(v_t, a.v, at(a.v, b, h), t0, tokens, a.Dv, tid);
            load_rows<DV, GRAD_THREADS>(o_t, a.dout, at(a.dout, b, h), t0, tokens, a.Dv, tid);
            load_state<2 * ST, GRAD_THREADS>(X_t, p.dstates + (long long)x.index * (2 * DK * DV), tid);
            cp_commit();
        }
        if constexpr (Tma) {
            await(s, 4, turn);
            if (tokens < C) {               // what lies behind the sequence was fetched too
                for (int e = tid; e < (C - tokens) * 8; e += GRAD_THREADS) {
                    const int r = tokens + e / 8, at16 = r * 128 + e % 8 * 16;
                    for (int i = 0; i < (2 * KT + 2 * VT) / PANEL; ++i) sts16(q_t + i * PANEL + at16, 0u, 0u, 0u, 0u);
                }
            }
        } else {
            cp_wait<0>();
        }
        fence_async();
        __syncthreads();
        if (tid < 32) {
            const uint32_t leader = elect();
            tc::tc_fence_after_sync();
            product<false, false, C, DK>(leader, tm, k, q, false);
            product<false, false, C, DV>(leader, tm + 128, v, o, false);
            commit(leader, &s.bar[0]);
        }
        if constexpr (Tma) {
            if (tid == 0) {
                stores_read();             // the tiles of the states and of E were the last chunk's outputs
                fetch_state(p.dstates, x);
            }
        }
        // from the start of t's block of 32 to t
        if (tid < C) s.f[tid] = tid < 32 ? ex2(s.G[tid].x + s.G[tid].y) : ex2_diff(s.G[tid], s.G[(tid & ~31) - 1]);
        const Item next = next_of((long long)x.index + gridDim.x);
        const float decay = decay_of(next);
        __syncthreads();
        if (warp == 3) {                      // (no pairs of its own)
            const uint32_t leader = elect();
            if constexpr (Tma) await(s, 5, 0);
            tc::tc_fence_after_sync();
            product_state<false, DK, DV, DK>(leader, tm + 256, v, Y_t, false);
            product_state<false, DK, DV, DK>(leader, tm + 256, v, X_t, true);
            product_state<true, DV, DK, DK>(leader, tm + 384, k, Y_t, false);
            product_state<true, DV, DK, DK>(leader, tm + 384, k, X_t, true);
            commit(leader, &s.bar[1]);
            if constexpr (Tma) {
                await(s, 1, turn);            // the state before the chunk in the same place
                if (lane == 0) fetch_state(p.states, x);
            }
            __syncwarp();
        }
        await(s, 0, turn);
        const float2 G = s.G[row], last = s.G[C - 1];
        // the pairs: blocks of 32 x 32, t from s on
        float s_sum = 0.f, t_sum = 0.f;
        uint32_t small[16];                   // of E, until there is room for it
        if (part < block) {
            const uint32_t zeros[32] = {};
#pragma unroll
            for (int i = 0; i < 16; ++i) small[i] = 0u;
            tmem_store(base + part * 32, zeros);
#pragma unroll
            for (int i = 0; i < 4; ++i) sts16(E_t + (part >> 1) * PANEL + chunk_at(row, (part & 1) * 4 + i), 0u, 0u, 0u, 0u);
        } else {
            float m[32];
            float2 sum = both(0.f);
            const float2 r = both(a.scale * (part > block ? ex2_diff(s.G[part * 32 - 1], G) : 1.f));
#pragma unroll
            for (int t0 = 0; t0 < 32; t0 += 16) {
                float2 x[8], y[8];
                int32_t u[2][16];
                tc::tmem_ld16(base + part * 32 + t0, u[0]);
                tc::tmem_ld16(base + 128 + part * 32 + t0, u[1]);
                tc::tmem_ld_wait();
                uint32_t e[8], P[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = make_float2(__int_as_float(u[0][2 * i]), __int_as_float(u[0][2 * i + 1]));
                    y[i] = make_float2(__int_as_float(u[1][2 * i]), __int_as_float(u[1][2 * i + 1]));
                    const int t = t0 + 2 * i;
                    float2 w;
                    if (part > block) {
                        w = __fmul2_rn(r, *reinterpret_cast<const float2 *>(&s.f[part * 32 + t]));
                    } else {
                        const float4 g2 = *reinterpret_cast<const float4 *>(&s.G[part * 32 + t]);
                        w = __fmul2_rn(r, make_float2(ex2_diff(make_float2(g2.x, g2.y), G), ex2_diff(make_float2(g2.z, g2.w), G)));
                        // (not by a factor of 0: what it would hide may be infinite)
                        if (t < lane) x[i].x = y[i].x = 0.f, w.x = 0.f;
                        if (t + 1 < lane) x[i].y = y[i].y = 0.f, w.y = 0.f;
                    }
                    const float2 pv = __fmul2_rn(w, x[i]);
                    float2 mv = __fmul2_rn(pv, y[i]);
                    if (part == block) {            // a pair of a token with itself moves with no decay
                        if (t == lane) mv.x = 0.f;
                        if (t + 1 == lane) mv.y = 0.f;
                    }
                    sum = __fadd2_rn(sum, mv);
                    m[t] = mv.x;
                    m[t + 1] = mv.y;
                    P[i] = pack_part(pv);
                    P[8 + i] = pack(rest(pv, P[i]));
                    const float2 ev = __fmul2_rn(w, y[i]);
                    e[i] = pack_part(ev);
                    small[t / 2] = pack(rest(ev, e[i]));
                }
                tmem_st16(base + part * 32 + t0, P);          // (in the place of k q^T, which no other warp reads)
                sts16(E_t + (part >> 1) * PANEL + chunk_at(row, (part & 1) * 4 + t0 / 8), e[0], e[1], e[2], e[3]);
                sts16(E_t + (part >> 1) * PANEL + chunk_at(row, (part & 1) * 4 + t0 / 8 + 1), e[4], e[5], e[6], e[7]);
            }
            s_sum = sum.x + sum.y;
            t_sum = sum_columns(m, lane);
        }
        const auto put_small = [&] {
#pragma unroll
            for (int i = 0; i < 4; ++i) sts16(E2_t + (part >> 1) * PANEL + chunk_at(row, (part & 1) * 4 + i), small[4 * i], small[4 * i + 1], small[4 * i + 2], small[4 * i + 3]);
        };
        if constexpr (!L::SHARED) put_small();
        await(s, 1, turn);
        if constexpr (!Tma) {
            load_state<2 * ST, GRAD_THREADS>(X_t, p.states + (long long)x.index * (2 * DK * DV), tid);
            cp_commit();
        }
        if (part >= block) t_sums[block * C + part * 32 + lane] = t_sum;
        s_sums[part * C + row] = s_sum;
        const float to_end = ex2_diff(last, G), from_start = a.scale * ex2(G.x + G.y);
        k_dots[part * C + row] = scale_sums<KQ>(base + 256 + part * KQ, to_end, k_t, row, part * KQ, true);
        scale_sums<VQ>(base + 384 + part * VQ, to_end, 0, 0, 0, false);
        if constexpr (!Tma) cp_wait<0>();
        fence_async();
        tc::tmem_st_wait();
        tc::tc_fence_before_sync();
        __syncthreads();                                  // the pairs' sums have been read, P^T, E^T and the scaled sums are there
        if (tid < 32) {
            const uint32_t leader = elect();
            if constexpr (Tma) await(s, 5, 1);
            tc::tc_fence_after_sync();
            product_state<false, DK, DV, DK>(leader, tm + 128, o, Y_t, false);
            product_state<false, DK, DV, DK>(leader, tm + 128, o, X_t, true);
            commit(leader, &s.bar[2]);
            product<false, true, DK, C>(leader, tm + 256, E, q, true);
            product_ts<true, DV, C>(leader, tm + 384, tm, o, true);
        }
        if (decays) g = running_sum<C>(decay_units(decay), s.g_sums, token);
        await(s, 2, turn);
        q_dots[part * C + row] = scale_sums<KQ>(base + 128 + part * KQ, from_start, q_t, row, part * KQ, true);
        if constexpr (L::SHARED) put_small();
        fence_async();
        tc::tmem_st_wait();
        tc::tc_fence_before_sync();
        __syncthreads();
        if (tid < 32) {
            const uint32_t leader = elect();
            tc::tc_fence_after_sync();
            product<true, true, DK, C>(leader, tm + 128, E2, k, true);
            product<true, true, DK, C>(leader, tm + 128, E, k, true);
            product<false, true, DK, C>(leader, tm + 256, E2, q, true);
            commit(leader, &s.bar[3]);
        }
        put_decays(g);                        // (every thread has read the last chunk's)
        // the decays' gradient: from each token on, every pair across it, and what passes from the state before the chunk to that behind it
        if (tid < C) {
            float t_sum = 0.f;
            for (int w = 0; w <= tid >> 5; ++w) t_sum += t_sums[w * C + tid];
            double own = (double)t_sum, kd = 0.0;
            for (int w = 0; w < 4; ++w) {
                own += (double)q_dots[w * C + tid] - (double)s_sums[w * C + tid];
                kd += (double)k_dots[w * C + tid];
            }
            double sum = running_sum<C>(kd - own, s.sums, tid) - (kd - own);
            for (int i = 16; i; i >>= 1) own += __shfl_xor_sync(0xffffffffu, own, i);
            if (lane == 0) totals[warp] = own;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int w = 0; w < tid >> 5; ++w) sum += s.sums[w];
            double through = 0.0;
            for (int w = 0; w < THROUGH; ++w) through += (double)p.through[(long long)x.index * THROUGH + w];
            sum += totals[0] + totals[1] + totals[2] + totals[3] + through * (double)exp2_of(last);
            if (tid < all) seq::store_f(a.ddecay.p, at(a.ddecay, b, h) + (long long)(t0 + tid) * a.ddecay.ts, a.decay_bf16, tid < tokens ? (float)sum : 0.f);
        }
        // The next chunk's tiles come as soon as nothing reads the ones that they replace.
        const bool live = row < tokens;
        await(s, 3, turn);
        if constexpr (Tma) {
            if (tid == 0 && next.tokens) fetch_qk(next);
        }
        // Out by way of tiles: a thread's part of a row on its own would be a store of 16 bytes in each of 32 lines.
        {
            float r[KQ];
            tmem_load(base + 128 + part * KQ, r);
#pragma unroll
            for (int i = 0; i < KQ; ++i) r[i] = live ? r[i] : 0.f;
            p.dq_heads ? put_heads(p.dq_heads, x, r) : put_row(dq_t, row, part * KQ, r);
            tmem_load(base + 256 + part * KQ, r);
#pragma unroll
            for (int i = 0; i < KQ; ++i) r[i] = live ? r[i] : 0.f;
            p.dk_heads ? put_heads(p.dk_heads, x, r) : put_row(dk_t, row, part * KQ, r);
        }
        {
            float r[VQ];
            tmem_load(base + 384 + part * VQ, r);
#pragma unroll
            for (int i = 0; i < VQ; ++i) r[i] = live ? r[i] : 0.f;
            put_row(dv_t, row, part * VQ, r);
        }
        fence_async();                                    // (the sums in v's tile come before what TMA writes there)
        tc::tc_fence_before_sync();
        if (__syncthreads_or(s.failed)) break;
        if constexpr (Tma) {
            if (tid == 0) {
                if (next.tokens) fetch_vo(next);
                for (int i = 0; i < DK / 64 && !p.dq_heads; ++i) {
                    tma_store_4d(&p.dq, dq_t + i * PANEL, i * 64, t0, h, b);
                    tma_store_4d(&p.dk, dk_t + i * PANEL, i * 64, t0, h, b);
                }
                for (int i = 0; i < DV / 64; ++i) tma_store_4d(&p.dv, dv_t + i * PANEL, i * 64, t0, h, b);
                stores_commit();
            }
        } else {
            if (!p.dq_heads) {
                copy_out<DK, false>(dq_t, a.dq, at(a.dq, b, h), t0, all, a.Dk, tid);
                copy_out<DK, false>(dk_t, a.dk, at(a.dk, b, h), t0, all, a.Dk, tid);
            }
            copy_out<DV, false>(dv_t, a.dv, at(a.dv, b, h), t0, all, a.Dv, tid);
            __syncthreads();
        }
        x = next;
    }
    if (Tma && tid == 0) stores_read();
    end(s, 512, p.flag, tid);
}

// ------------------------------------------------------------------------------------- launches
template <class F>
int with_smem(F *kernel, int tiles, int *bytes) {
    *bytes = tiles + 1024 + (int)sizeof(Shared);
    SEQ_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, *bytes));
    return QGRU_OK;
}

template <int DK, int DV, bool Reverse>
int run_states(const qgru_attention &a, const Cut &c, bf16 *states, char *seg, float *through, int *flag, cudaStream_t st) {
    Pass p{};
    p.other = static_cast<const bf16 *>(a.states);
    p.through = through;
    p.k = Reverse ? a.q : a.k;
    p.v = Reverse ? a.dout : a.v;
    p.k_share = a.H / a.Hk;
    p.first = Reverse ? a.dstate : a.state0;
    p.last = Reverse ? a.dstate0 : a.state;
    p.segments = c.segments;
    p.per = c.per;
    p.chunks = c.chunks;
    p.flag = flag;
    p.states = states;
    const auto kernel = k_states_tc<DK, DV, Reverse>;
    int bytes = 0;
    if (const int rc = with_smem(kernel, STATES_TILES<DK, DV>, &bytes)) return rc;
    const dim3 grid(a.B * a.H, c.segments);
    if (c.segments > 1) {
        p.seg_state = reinterpret_cast<float *>(seg);
        p.seg_log = p.seg_state + c.segments * state_elems(a);
        p.own_sums = true;
        kernel<<<grid, THREADS, bytes, st>>>(a, p);
        SEQ_CK(cudaGetLastError());
        if (const int rc = scan_segments(a, c, Reverse, seg, st)) return rc;
        p.own_sums = false;
    }
    kernel<<<grid, THREADS, bytes, st>>>(a, p);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

template <int DK, int DV>
int forward(const qgru_attention &a, const Cut &c, int *flag, cudaStream_t st) {
    bf16 *states = static_cast<bf16 *>(a.keep ? a.states : a.workspace);
    char *seg = static_cast<char *>(a.workspace) + (a.keep ? 0 : a256(c.states));
    if (const int rc = run_states<DK, DV, false>(a, c, states, seg, nullptr, flag, st)) return rc;
    if (c.chunks == 0) return QGRU_OK;
    int bytes = 0;
    if (const int rc = with_smem(k_outputs_tc<DK, DV>, OUTPUTS_TILES<DK, DV>, &bytes)) return rc;
    k_outputs_tc<DK, DV><<<c.chunks * a.B * a.H, THREADS, bytes, st>>>(a, states, flag);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}
template <int DK, int DV, bool Tma>
int backward(const qgru_attention &a, const Cut &c, int *flag, int sms, cudaStream_t st) {
    char *ws = static_cast<char *>(a.workspace);
    bf16 *dstates = reinterpret_cast<bf16 *>(ws);
    ws += a256(c.states);
    char *seg = ws;
    ws += a256(c.seg);
    float *through = reinterpret_cast<float *>(ws);
    ws += a256(c.through);
    if (const int rc = walk_takes(a, true) ? walk(a, c, true, dstates, seg, through, flag, sms, st) : run_states<DK, DV, true>(a, c, dstates, seg, through, flag, st)) return rc;
    if (c.chunks == 0) return QGRU_OK;
    Gradients g{};
    g.states = static_cast<const bf16 *>(a.states);
    g.dstates = dstates;
    g.through = through;
    g.flag = flag;
    g.items = c.chunks * a.B * a.H;
    if (Tma) {
        if (!head_map(&g.q, a.q, a.T, a.B, a.Hk, a.Dk) || !head_map(&g.k, a.k, a.T, a.B, a.Hk, a.Dk) || !head_map(&g.v, a.v, a.T, a.B, a.H, a.Dv) ||
            !head_map(&g.o, a.dout, a.T, a.B, a.H, a.Dv) || !head_map(&g.dv, a.dv, a.T, a.B, a.H, a.Dv) ||
            (a.H == a.Hk && (!head_map(&g.dq, a.dq, a.T, a.B, a.H, a.Dk) || !head_map(&g.dk, a.dk, a.T, a.B, a.H, a.Dk))))
            return seq::fail(QGRU_ERR_CUDA, "cuTensorMapEncodeTiled");
    }
    if (a.H != a.Hk) {
        g.dq_heads = reinterpret_cast<float *>(ws);
        g.dk_heads = g.dq_heads + group_bytes(a) / 8;
    }
    int bytes = 0;
    if (const int rc = with_smem(k_gradients_tc<DK, DV, Tma>, Tiles<DK, DV>::ALL, &bytes)) return rc;
    k_gradients_tc<DK, DV, Tma><<<std::min(g.items, sms), GRAD_THREADS, bytes, st>>>(a, g);
    SEQ_CK(cudaGetLastError());
    return g.dq_heads ? sum_groups(a, g.dq_heads, g.dk_heads, st) : QGRU_OK;
}

template <class F>
int by_size(const qgru_attention &a, F f) {
    const std::integral_constant<int, 64> small;
    const std::integral_constant<int, 128> large;
    return a.Dk <= 64 ? (a.Dv <= 64 ? f(small, small) : f(small, large)) : (a.Dv <= 64 ? f(large, small) : f(large, large));
}

}  // namespace

bool tc_takes(const qgru_attention &a) { return a.bf16 && a.Dk <= 128 && a.Dv <= 128; }

// Segments: one CTA of the state pass per SM (or two, with the smaller tiles) where the heads alone do not give that many; of two
// chunks at the least.
Cut tc_cut(const qgru_attention &a, int sms) {
    Cut c;
    c.chunk = C;
    c.chunks = (a.T + C - 1) / C;
    const long long units = std::max<long long>((long long)a.B * a.H, 1);
    c.segments = (int)std::max<long long>(1, std::min<long long>(c.chunks / 2, sms / units));
    c.per = std::max(1, (c.chunks + c.segments - 1) / c.segments);
    c.segments = std::max(1, (c.chunks + c.per - 1) / c.per);
    c.states = 2 * sizeof(bf16) * (size_t)c.chunks * a.B * a.H * (a.Dk <= 64 ? 64 : 128) * (a.Dv <= 64 ? 64 : 128);
    c.seg = c.segments > 1 ? sizeof(float) * c.segments * (state_elems(a) + (size_t)a.B * a.H) : 0;
    c.through = sizeof(float) * THROUGH * c.chunks * (size_t)a.B * a.H;
    return c;
}
int tc_forward(const qgru_attention &a, const Cut &c, int *flag, int sms, cudaStream_t st) {
    if (walk_takes(a, false)) return walk(a, c, false, a.keep ? a.states : nullptr, static_cast<char *>(a.workspace), nullptr, flag, sms, st);
    return by_size(a, [&](auto dk, auto dv) -> int { return forward<dk.value, dv.value>(a, c, flag, st); });
}
int tc_backward(const qgru_attention &a, const Cut &c, int *flag, int sms, cudaStream_t st) {
    const bool tma = fetchable(a.q, a.T, a.B, a.Hk, a.Dk) && fetchable(a.k, a.T, a.B, a.Hk, a.Dk) && fetchable(a.v, a.T, a.B, a.H, a.Dv) && fetchable(a.dout, a.T, a.B, a.H, a.Dv) &&
                     fetchable(a.dv, a.T, a.B, a.H, a.Dv) && (a.H != a.Hk || (fetchable(a.dq, a.T, a.B, a.H, a.Dk) && fetchable(a.dk, a.T, a.B, a.H, a.Dk)));
    return by_size(a, [&](auto dk, auto dv) -> int {
        return tma ? backward<dk.value, dv.value, true>(a, c, flag, sms, st) : backward<dk.value, dv.value, false>(a, c, flag, sms, st);
    });
}

}  // namespace attn
}  // namespace qgru
