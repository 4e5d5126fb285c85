// qgru_attn_fwd.cu - linear attention over the chunks of a sequence in turn, on the tensor cores, every token read once: the outputs and
// the state, or the states alone (also from the end, for the gradient of the states).
//
// A CTA per SM walks through (sequence and head, segment) after another, chunk by chunk of 128 tokens.  Five warpgroups work on
// different chunks at the same time and hand them on through barriers in shared memory:
//   K  takes k times the decays to the chunk's end apart into three bf16 parts (24 bits), 64 tokens at a time
//   S  keeps the state in fp32 registers: S' = 2^G_C S + (w k)^T v, and puts it, as two bf16 parts (16 bits), beside q
//   P  weighs the pairs of tokens: q k^T out of tensor memory, times 2^(G_t - G_s), into it again as two bf16 parts, the operand of P v
//   O  out = 2^G_t q S + P v: out of tensor memory, into the output
//   X  a warp issues the products, one fetches tiles by TMA, two sum the decays up
// In the order of the products the chunk's part of the state comes first, since the next chunk's outputs wait for it.
//
// What is rounded on the way: P, and the state where it is a factor, to 16 bits (two bf16 parts each); the output once, to bf16, in the end.
//
// What bounds it: the products, one after the other, not the bytes.  64 x 1000 tokens of 16 heads of 64, 524 MB: 188 us, 2.8 TB/s, 5900
// cycles a chunk and SM.  The warp that issues the products waits for no role: every operand is there when it comes to it (of a chunk's
// 5900 cycles K works 3000, P 4300, O 1900, S 600).  Its 56 products take 100 cycles each, with five roles on the same shared and tensor
// memory; alone they take 32 to 64.  P as one part would be eight products fewer, 175 us, and a rounding more in every output.  The roles
// share one instruction cache, so their loops stay rolled.  16 x 1000 tokens of 8 heads of 128: 65 us with the outputs and kept states, 46
// from the end without outputs.  One phrase of 24 tokens, 4 heads of 64: 9 us, the latency of the roles one after another.
#include <algorithm>
#include <type_traits>

#include "qgru_attn_tc.cuh"

namespace qgru {
namespace attn {
namespace {

using namespace tile;
constexpr int WG = 128, THREADS = 5 * WG;
// 640 threads start with 96 registers each; the warpgroups share the 480 of five threads by the columns of a state that a thread has.
constexpr int REGS = 96;
template <int N>
struct Regs {
    static constexpr int S = N == 128 ? 168 : N == 64 ? 128 : 104, P = 96, O = N == 128 ? 112 : 120, K = N == 128 ? 64 : 80, X = N == 128 ? 40 : 56;
    static_assert(S + P + O + K + X <= 5 * REGS, "the shares add up to what the block starts with");
};
template <int R>
__device__ __forceinline__ void take_registers() {
    if constexpr (R > REGS)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
constexpr int SLOTS = 4;                    // chunks whose decays are known at once

struct Slot {
    float hi[C], lo[C];                     // running sums, base 2, each as two floats
    float to_block[C];                      // 2^(G at the end of s's block of 32 - G_s)
    float weight[C];                        // of k: 2^(G_C - G_s), or from the end scale 2^G_t
    float from_start[C];                    // scale 2^G_t
    float whole;
    float pad[3];
    __device__ __forceinline__ float2 G(int t) const { return make_float2(hi[t], lo[t]); }
};

template <int DK, int DV, bool Outputs, bool Reverse>
struct Plan {
    static constexpr int KT = DK / 64 * PANEL, VT = DV / 64 * PANEL, STAGE = (Outputs ? 2 : 1) * KT + VT;
    static constexpr int PART = DK / 64 * PANEL / 2, PARTS = 3 * PART;            // 64 tokens
    static constexpr int STATE = DK * DV * 2, STATES = Outputs ? 2 * STATE : 0;
    static constexpr int NB = DK == 128 && (DV == 128 || !Outputs) ? 1 : 2;       // buffers of parts
    // from the end: a ring of pieces of the forward's states, each of so many eights of columns
    static constexpr int PIECE = 16384, PIECES = 2 * STATE / PIECE, EIGHTS = PIECE / (DK * 16), RING = Reverse ? 2 * PIECE : 0;
    static constexpr int ROOM = 213000 - NB * PARTS - STATES - RING;
    static constexpr int NS = ROOM / STAGE >= 3 ? 3 : ROOM / STAGE >= 2 ? 2 : 1;  // stages of tiles
    static constexpr int NQ = DV == 64 && NS > 1 ? 2 : 1;                         // buffers of q k^T
    static constexpr int TILES = NS * STAGE + NB * PARTS + STATES + RING;
    // columns of tensor memory
    static constexpr uint32_t INTER = NQ * 128, INTRA = INTER + DV, U = Outputs ? INTRA + DV : 0, COLUMNS = Outputs ? 512 : DV;
    static_assert(!Outputs || U + DV <= 512, "tensor memory");
    static_assert(NS >= 1 && TILES <= 213000, "shared memory");
};

struct Ctl {
    uint64_t k_full[3], k_empty[3], q_full[3], q_empty[3], v_full[3], v_empty[3], parts_full[2], parts_empty[2], pairs_full[2], p_full[2], g_full[SLOTS], g_empty[SLOTS];
    uint64_t u_full, u_empty, s_full, o_empty, ring_full[2], ring_empty[2];
    uint32_t tmem;
    volatile int failed;
};

struct Args {
    CUtensorMap q, k, v;                    // [B][heads][T][D]
    const float *first;                     // the state it starts from, or null
    float *last;                            // where the last one goes, or null
    bf16 *states;                           // before each chunk in the pass's order, [chunks][B H][2 parts][DV / 8][DK][8], or null
    const bf16 *other;                      // from the end: the forward's states, and where their products with these go
    float *through;
    float *seg_state, *seg_log;
    int own_sums;                           // states alone: each segment's sum, from zero, and nothing else
    int segments, per, chunks, items, share;
    int *flag;
};

// A (sequence, head, segment) and its chunks with tokens, in the pass's order.
template <bool Reverse>
struct Item {
    int bh, b, h, seg, n, begin, stop, end;
    __device__ __forceinline__ Item(const qgru_attention &a, const Args &p, int item) {
        const int heads = a.B * a.H;
        seg = item / heads;
        bh = item % heads;
        b = bh / a.H;
        h = bh % a.H;
        n = valid_tokens(a, b);
        const int used = (n + C - 1) / C;
        begin = seg * p.per;
        end = min(begin + p.per, p.chunks);
        if (Reverse) begin = min(max(begin, p.chunks - used), end);
        stop = Reverse ? end : max(begin, min(end, used));
    }
    static __device__ __forceinline__ int chunk(const Args &p, int c) { return Reverse ? p.chunks - 1 - c : c; }
    __device__ __forceinline__ int tokens(int chunk) const { return min(n - chunk * C, C); }
};

// A wait is one instruction that sleeps until the phase is over, most of the time: code and instructions of twenty warps that poll would
// cost the others more than anything else here (the SM's instruction cache holds about what one step of all of them takes).
__device__ __forceinline__ bool over(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(100000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait(Ctl &s, uint64_t &bar, uint32_t parity) {
    const uint32_t at = tc::smem_u32(&bar);
    if (over(at, parity)) return true;
    const long long t0 = clock64();
    while (!over(at, parity)) {
        if (s.failed) return false;
        if (clock64() - t0 > WAIT_BUDGET) {
            s.failed = 1;
            return false;
        }
    }
    return true;
}
// for a whole warp: all its lanes or none go on
__device__ __forceinline__ bool wait_warp(Ctl &s, uint64_t &bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(s, bar, parity)); }
// A ring of N: the buffer and the parity of step i; `free`: of the wait for it to be empty.
template <int N>
struct At {
    int buf;
    uint32_t full, free;
    __device__ __forceinline__ explicit At(int i) : buf(i % N), full((uint32_t)(i / N) & 1u), free(full ^ 1u) {}
};
template <int DK, int DV, bool Outputs, bool Reverse>
struct Roles {
    using L = Plan<DK, DV, Outputs, Reverse>;
    const qgru_attention &a;
    const Args &p;
    Ctl &s;
    Slot *slots;
    uint32_t tiles;                         // stages, then the parts, then the state
    int tid;                                // in the warpgroup

    __device__ __forceinline__ uint32_t k_tile(int st) const { return tiles + st * L::STAGE; }
    __device__ __forceinline__ uint32_t v_tile(int st) const { return tiles + st * L::STAGE + L::KT; }
    __device__ __forceinline__ uint32_t q_tile(int st) const { return tiles + st * L::STAGE + L::KT + L::VT; }
    __device__ __forceinline__ uint32_t parts(int b) const { return tiles + L::NS * L::STAGE + b * L::PARTS; }
    __device__ __forceinline__ uint32_t state(int part) const { return tiles + L::NS * L::STAGE + L::NB * L::PARTS + part * L::STATE; }
    __device__ __forceinline__ uint32_t ring(int b) const { return tiles + L::NS * L::STAGE + L::NB * L::PARTS + L::STATES + b * L::PIECE; }
    // f(item, its chunk in the pass's order, running number of the chunk) until it says that a wait has run out
    template <class F>
    __device__ __forceinline__ bool each(F f) const {
        int i = 0;
        for (int it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item<Reverse> w(a, p, it);
            for (int c = w.begin; c < w.stop; ++c, ++i)
                if (!f(w, Item<Reverse>::chunk(p, c), i)) return false;
        }
        return true;
    }

    // ---- X, warp 0: products.  Those that add to the same sums follow one another as they are issued; others need not, so the pairs of a chunk
    // wait until P v of the chunk whose weights they overwrite is done.
    __device__ __forceinline__ bool pairs(uint32_t leader, int i) const {
        const At<L::NS> st(i);
        if (i >= L::NQ) {
            const At<L::NS> before(i - L::NQ);
            if (!wait(s, s.v_empty[before.buf], before.full)) return false;
        }
        if (!wait(s, s.k_full[st.buf], st.full) || !wait(s, s.q_full[st.buf], st.full)) return false;
        tc::tc_fence_after_sync();
        product<false, false, C, DK>(leader, s.tmem + (i % L::NQ) * 128, Operand{q_tile(st.buf), PANEL}, Operand{k_tile(st.buf), PANEL}, false);
        commit(leader, &s.pairs_full[i % L::NQ]);
        commit(leader, &s.k_empty[st.buf]);
        return true;
    }
    __device__ __forceinline__ void issue() const {
        const uint32_t leader = elect();
        int steps = 0;
        for (int it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item<Reverse> w(a, p, it);
            steps += w.stop - w.begin;
        }
        if (Outputs && L::NQ == 2 && steps && !pairs(leader, 0)) return;
        for (int i = 0; i < steps; ++i) {
            const At<L::NS> st(i);
            const At<1> one(i);
            if (Outputs && L::NQ == 1 && !pairs(leader, i)) return;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                const At<L::NB> pb(2 * i + half);
                if (!wait(s, s.parts_full[pb.buf], pb.full)) return;
                if (half == 0 && (!wait(s, s.v_full[st.buf], st.full) || !wait(s, s.u_empty, one.free))) return;
                tc::tc_fence_after_sync();
                const Operand v{v_tile(st.buf) + half * (PANEL / 2), PANEL};
                // the small parts first
#pragma unroll 1
                for (int t = 2; t >= 0; --t) {
                    const Operand k{parts(pb.buf) + t * L::PART, DK == 64 ? 0 : PANEL / 2};      // (64 lanes: the rest repeats them)
                    product<true, true, DV, 64>(leader, s.tmem + L::U, k, v, half || t != 2);
                }
                commit(leader, &s.parts_empty[pb.buf]);
            }
            if (L::NB == 1) commit(leader, &s.u_full);
            if constexpr (Outputs) {
                if (!wait(s, s.s_full, one.full) || !wait(s, s.o_empty, one.free)) return;
                tc::tc_fence_after_sync();
                const Operand q{q_tile(st.buf), PANEL};
#pragma unroll 1
                for (int part = 1; part >= 0; --part) product<false, true, DV, DK>(leader, s.tmem + L::INTER, q, Operand{state(part), DK * 128}, part == 0);
                commit(leader, &s.q_empty[st.buf]);
                if (L::NQ == 2 && i + 1 < steps && !pairs(leader, i + 1)) return;
                const At<L::NQ> qb(i);
                if (!wait(s, s.p_full[qb.buf], qb.full)) return;
                tc::tc_fence_after_sync();
                product_ts<true, DV, C>(leader, s.tmem + L::INTRA, s.tmem + qb.buf * 128, Operand{v_tile(st.buf), PANEL}, false);
            }
            commit(leader, &s.v_empty[st.buf]);
        }
    }
    // ---- X, warp 1: tiles
    __device__ __forceinline__ void fetch() const {
        const auto load = [&](uint32_t to, const CUtensorMap *map, uint64_t *bar, int panels, int t, int h, int b) {
            tc::mbar_expect_tx(bar, panels * PANEL);
            for (int i = 0; i < panels; ++i) tma_load_4d(to + i * PANEL, map, bar, i * 64, t, h, b);
        };
        each([&](const Item<Reverse> &w, int chunk, int i) {
            const At<L::NS> st(i);
            // (k is there after the v that was in this stage before it: K waits for v of short chunks alone, and a phase of v_full that is
            // two ahead of the barrier's would look like one that is over)
            if (!wait(s, s.k_empty[st.buf], st.free) || !wait(s, s.v_full[st.buf], st.free)) return false;
            load(k_tile(st.buf), &p.k, &s.k_full[st.buf], DK / 64, chunk * C, w.h / p.share, w.b);
            if constexpr (Outputs) {
                if (!wait(s, s.q_empty[st.buf], st.free)) return false;
                load(q_tile(st.buf), &p.q, &s.q_full[st.buf], DK / 64, chunk * C, w.h / p.share, w.b);
            }
            if (!wait(s, s.v_empty[st.buf], st.free)) return false;
            load(v_tile(st.buf), &p.v, &s.v_full[st.buf], DV / 64, chunk * C, w.h, w.b);
            return true;
        });
    }
    // ---- From the end, a warp of P (which has nothing to weigh there): the forward's states, piece after piece
    __device__ __forceinline__ void fetch_states() const {
        each([&](const Item<Reverse> &w, int chunk, int i) {
            const bf16 *from = p.other + ((long long)chunk * a.B * a.H + w.bh) * (2 * DK * DV);
            for (int piece = 0; piece < L::PIECES; ++piece) {
                const At<2> o(i * L::PIECES + piece);
                if (!wait(s, s.ring_empty[o.buf], o.free)) return false;
                tc::mbar_expect_tx(&s.ring_full[o.buf], L::PIECE);
                bulk_load(ring(o.buf), from + piece * (L::PIECE / 2), L::PIECE, &s.ring_full[o.buf]);
            }
            return true;
        });
    }
    // ---- X, warps 2 and 3, every second chunk each: decays, four neighbouring tokens a lane
    __device__ __forceinline__ void decays() const {
        const int lane = tid & 31;
        each([&](const Item<Reverse> &w, int chunk, int i) {
            if ((i & 1) != ((tid >> 5) & 1)) return true;
            const At<SLOTS> at(i);
            const int tokens = w.tokens(chunk);
            const long long base = w.b * a.decay.bs + w.h * a.decay.hs + (long long)chunk * C * a.decay.ts;
            float f[4];
            long long g[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = 0.f;
                if (4 * lane + j < tokens) {
                    if (a.decay_bf16)
                        f[j] = seq::to_f(static_cast<const bf16 *>(a.decay.p)[base + (4 * lane + j) * a.decay.ts]);
                    else
                        f[j] = static_cast<const float *>(a.decay.p)[base + (4 * lane + j) * a.decay.ts];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = sum += decay_units(f[j]);
            long long before = sum;
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += u;
            }
            before = __shfl_up_sync(0xffffffffu, before, 1);
            if (lane == 0) before = 0;
            if (!wait_warp(s, s.g_empty[at.buf], at.free)) return false;
            Slot &to = slots[at.buf];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 G = two_floats(before + g[j]);
                to.hi[4 * lane + j] = G.x;
                to.lo[4 * lane + j] = G.y;
            }
            __syncwarp();
            const float2 end = to.G(C - 1);
#pragma unroll 1
            for (int t = lane; t < C; t += 32) {
                const float2 G = to.G(t);
                const float start = a.scale * exp2_of(G);
                to.to_block[t] = ex2_diff(to.G(t | 31), G);
                to.weight[t] = Reverse ? start : exp2_diff(end, G);
                to.from_start[t] = start;
            }
            if (lane == 0) to.whole = exp2_of(end);
            tc::mbar_arrive(&s.g_full[at.buf]);
            return true;
        });
    }
    // ---- K
    __device__ __forceinline__ void split() const {
        each([&](const Item<Reverse> &w, int chunk, int i) {
            const At<L::NS> st(i);
            const At<SLOTS> at(i);
            const int tokens = w.tokens(chunk);
            if (!wait_warp(s, s.g_full[at.buf], at.full) || !wait_warp(s, s.k_full[st.buf], st.full)) return false;
            if (tokens < C) {              // what lies behind the sequence was fetched too: v must not bring infinities or NaN into the sums
                if (!wait_warp(s, s.v_full[st.buf], st.full)) return false;
                for (int e = tid; e < (C - tokens) * (DV / 8); e += WG) {
                    const int r = tokens + e / (DV / 8), c = e % (DV / 8);
                    sts16(v_tile(st.buf) + (c >> 3) * PANEL + r * 128 + (c & 7) * 16, 0u, 0u, 0u, 0u);
                }
            }
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                const At<L::NB> pb(2 * i + half);
                if (!wait_warp(s, s.parts_empty[pb.buf], pb.free)) return false;
                const uint32_t from = k_tile(st.buf) + half * (PANEL / 2), to = parts(pb.buf);
#pragma unroll 1
                for (int j = 0; j < 64 * DK / 8 / WG; ++j) {
                    const int e = j * WG + tid, r = e / (DK / 8), ch = e % (DK / 8);
                    const uint32_t off = chunk_at(r, ch & 7);
                    const uint4 u = lds16(from + (ch >> 3) * PANEL + off);
                    uint32_t in[4] = {u.x, u.y, u.z, u.w};
                    if (half * 64 + r >= tokens) in[0] = in[1] = in[2] = in[3] = 0u;
                    const float f = slots[at.buf].weight[half * 64 + r];
                    uint32_t o[3][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float2 x = __fmul2_rn(unpack(in[q]), both(f));
#pragma unroll
                        for (int t = 0; t < 3; ++t) {
                            o[t][q] = t < 2 ? pack_part(x) : pack(x);
                            if (t < 2) x = rest(x, o[t][q]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < 3; ++t) sts16(to + t * L::PART + (ch >> 3) * (PANEL / 2) + off, o[t][0], o[t][1], o[t][2], o[t][3]);
                }
                fence_async();
                tc::mbar_arrive(&s.parts_full[pb.buf]);
            }
            tc::mbar_arrive(&s.k_empty[st.buf]);
            tc::mbar_arrive(&s.g_empty[at.buf]);
            return true;
        });
    }
    // ---- S.  Lane i of tensor memory is row i; with 64 rows the upper lanes repeat them and take the second half of the columns.
    __device__ __forceinline__ void states() const {
        constexpr int N = DK == 64 ? DV / 2 : DV;
        const int row = DK == 64 ? tid & 63 : tid, c0 = DK == 64 ? (tid >> 6) * N : 0;
        const uint32_t U = lane_base(s.tmem, tid >> 5) + L::U + c0;
        const long long dense_all = (long long)a.B * a.H * a.Dk * a.Dv;
        float2 S[N / 2];
        int i = 0;
        for (int it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item<Reverse> w(a, p, it);
            const long long dense = (long long)w.bh * a.Dk * a.Dv + (long long)row * a.Dv + c0;
            const float *first = p.own_sums ? nullptr : p.segments > 1 ? p.seg_state + w.seg * dense_all : p.first;
            if (first && row >= a.Dk) first = nullptr;
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (first && c0 + j < a.Dv) x = *reinterpret_cast<const float4 *>(first + dense + j);      // (head sizes here are multiples of 8)
                S[j / 2] = make_float2(x.x, x.y);
                S[j / 2 + 1] = make_float2(x.z, x.w);
            }
            double all = 0.0;
            for (int c = w.begin; c < w.stop; ++c, ++i) {
                const At<SLOTS> at(i);
                uint4 *keep = p.states && !p.own_sums ? reinterpret_cast<uint4 *>(p.states + ((long long)Item<Reverse>::chunk(p, c) * a.B * a.H + w.bh) * (2 * DK * DV) + (c0 * DK + row * 8)) : nullptr;
                if (Reverse && !p.own_sums) {
                    const long long head = (long long)Item<Reverse>::chunk(p, c) * a.B * a.H + w.bh;
                    float2 x = both(0.f);
#pragma unroll
                    for (int e = 0; e < 2 * N / 8; ++e) {
                        // eights of columns of the two parts; with 64 rows a piece holds both halves of them, the lanes' own and the others'
                        const int part = e / (N / 8), j = e % (N / 8), at8 = part * (DV / 8) + (DK == 64 ? 0 : j), piece = at8 / L::EIGHTS;
                        const bool first = at8 % L::EIGHTS == 0 && (DK != 64 || j == 0);
                        const bool last = DK == 64 ? j == N / 8 - 1 && (part + 1) * (DV / 8) % L::EIGHTS == 0 : at8 % L::EIGHTS == L::EIGHTS - 1;
                        const At<2> o(i * L::PIECES + piece);
                        if (first && !wait_warp(s, s.ring_full[o.buf], o.full)) return;
                        x = dot8(lds16(ring(o.buf) + (uint32_t)((part * (DV / 8) + c0 / 8 + j) % L::EIGHTS * DK + row) * 16), &S[j * 4], x);
                        if (last) {
                            fence_async();         // (ordinary reads, and the bulk copy that follows into the same place, are ordered by this alone)
                            tc::mbar_arrive(&s.ring_empty[o.buf]);
                        }
                    }
                    float sum = x.x + x.y;
                    for (int e = 16; e; e >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, e);
                    if ((tid & 31) == 0) {
                        p.through[head * THROUGH + (tid >> 5)] = sum;
                        p.through[head * THROUGH + 4 + (tid >> 5)] = 0.f;
                    }
                }
                if constexpr (Outputs)
                    if (i && !wait_warp(s, s.q_empty[At<L::NS>(i - 1).buf], At<L::NS>(i - 1).full)) return;      // q S of the chunk before is done
#pragma unroll
                for (int j = 0; j < N; j += 8) {
                    if (!Outputs && !keep) break;
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        hi[e] = pack_part(S[j / 2 + e]);
                        lo[e] = pack(rest(S[j / 2 + e], hi[e]));
                    }
                    if (keep) {
                        keep[j / 8 * DK] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        keep[DK * DV / 8 + j / 8 * DK] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                    if constexpr (Outputs) {
                        const uint32_t off = (uint32_t)((c0 + j) >> 6) * (DK * 128) + chunk_at(row, ((c0 + j) >> 3) & 7);
                        sts16(state(0) + off, hi[0], hi[1], hi[2], hi[3]);
                        sts16(state(1) + off, lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                if constexpr (Outputs) {
                    fence_async();
                    tc::mbar_arrive(&s.s_full);
                }
                if (!wait_warp(s, s.g_full[at.buf], at.full)) return;
                const float2 whole = both(slots[at.buf].whole);
                all += (double)slots[at.buf].hi[C - 1] + (double)slots[at.buf].lo[C - 1];
                tc::mbar_arrive(&s.g_empty[at.buf]);
                // the products with the second half of k are done, and so all: of two buffers that half's says it
                if (!wait_warp(s, L::NB == 1 ? s.u_full : s.parts_empty[1], (uint32_t)i & 1u)) return;
                tc::tc_fence_after_sync();
#pragma unroll
                for (int j = 0; j < N; j += 32) {
                    float2 u[2][8];
                    int32_t r[2][16];
                    tc::tmem_ld16(U + j, r[0]);
                    tc::tmem_ld16(U + j + 16, r[1]);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        u[e / 8][e % 8] = make_float2(__int_as_float(r[e / 8][e % 8 * 2]), __int_as_float(r[e / 8][e % 8 * 2 + 1]));
                        S[j / 2 + e] = __ffma2_rn(whole, S[j / 2 + e], u[e / 8][e % 8]);
                    }
                }
                tc::tc_fence_before_sync();
                tc::mbar_arrive(&s.u_empty);
            }
            float *to = p.own_sums ? p.seg_state + w.seg * dense_all : p.last && w.seg == p.segments - 1 ? p.last : nullptr;
            if (to && row < a.Dk) {
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    if (c0 + j < a.Dv) *reinterpret_cast<float4 *>(to + dense + j) = make_float4(S[j / 2].x, S[j / 2].y, S[j / 2 + 1].x, S[j / 2 + 1].y);
                }
            }
            if (p.own_sums && tid == 0) p.seg_log[w.seg * (a.B * a.H) + w.bh] = (float)all;
        }
    }
    // ---- P.  Blocks of 32 x 32 pairs; below the diagonal 2^(G_t - G_s) is a product of two factors, both at most 1: from s to the end
    // of its block and from there to t.
    __device__ __forceinline__ void weights() const {
        const int warp = tid >> 5, lane = tid & 31;
        each([&](const Item<Reverse> &, int, int i) {
            const At<SLOTS> at(i);
            const At<L::NQ> qb(i);
            if (!wait_warp(s, s.g_full[at.buf], at.full)) return false;
            const Slot &g = slots[at.buf];
            const float2 G = g.G(tid);
            const uint32_t from = lane_base(s.tmem, warp) + qb.buf * 128;
            if (!wait_warp(s, s.pairs_full[qb.buf], qb.full)) return false;
            tc::tc_fence_after_sync();
#pragma unroll 1
            for (int s0 = 0; s0 < C; s0 += 16) {
                const int sb = s0 >> 5;
                uint32_t P[16];
                if (sb > warp) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) P[j] = 0u;
                } else {
                    float2 x[8];
                    tmem_load(from + s0, x);
                    if (sb < warp) {
                        const float2 r = both(a.scale * ex2_diff(G, g.G(s0 | 31)));
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = __fmul2_rn(x[j], __fmul2_rn(r, *reinterpret_cast<const float2 *>(&g.to_block[s0 + 2 * j])));
                    } else {
                        const int last = lane - (s0 & 31);
                        const float2 minus = both(-1.f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 d = __fadd2_rn(__ffma2_rn(*reinterpret_cast<const float2 *>(&g.hi[s0 + 2 * j]), minus, both(G.x)),
                                                        __ffma2_rn(*reinterpret_cast<const float2 *>(&g.lo[s0 + 2 * j]), minus, both(G.y)));
                            const float2 v = __fmul2_rn(x[j], __fmul2_rn(both(a.scale), make_float2(ex2(d.x), ex2(d.y))));
                            x[j] = make_float2(2 * j <= last ? v.x : 0.f, 2 * j + 1 <= last ? v.y : 0.f);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        P[j] = pack_part(x[j]);
                        P[8 + j] = pack(rest(x[j], P[j]));
                    }
                }
                tmem_st16(from + s0, P);
            }
            tc::tmem_st_wait();
            tc::tc_fence_before_sync();
            tc::mbar_arrive(&s.p_full[qb.buf]);
            tc::mbar_arrive(&s.g_empty[at.buf]);
            return true;
        });
    }
    // ---- O
    __device__ __forceinline__ void outputs() const {
        const int warp = tid >> 5, row = tid;
        const uint32_t from = lane_base(s.tmem, warp);
        int i = 0;
        for (int it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item<Reverse> w(a, p, it);
            bf16 *out = static_cast<bf16 *>(a.out.p) + at(a.out, w.b, w.h) + (long long)row * a.out.ts;
            for (int c = w.begin; c < w.stop; ++c, ++i) {
                const At<L::NS> done(i);
                const At<SLOTS> g(i);
                const int t0 = c * C, all = min(a.T - t0, C), tokens = w.tokens(c);
                if (!wait_warp(s, s.g_full[g.buf], g.full) || !wait_warp(s, s.v_empty[done.buf], done.full)) return;      // P v, the last with v, is done
                tc::tc_fence_after_sync();
                const float r = slots[g.buf].from_start[row];
                bf16 *to = out + (long long)t0 * a.out.ts;
                uint32_t odd_groups = 0;
#pragma unroll 1
                for (int j = 0; j < DV; j += 16) {
                    int32_t u[2][16];
                    tc::tmem_ld16(from + L::INTRA + j, u[0]);
                    tc::tmem_ld16(from + L::INTER + j, u[1]);
                    tc::tmem_ld_wait();
                    float2 odd = both(0.f);
                    uint32_t y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 intra = make_float2(__int_as_float(u[0][2 * e]), __int_as_float(u[0][2 * e + 1]));
                        odd = __ffma2_rn(intra, both(0.f), odd);
                        y[e] = pack(__ffma2_rn(make_float2(__int_as_float(u[1][2 * e]), __int_as_float(u[1][2 * e + 1])), both(r), intra));
                    }
                    if (row < tokens) {
                        if (!(odd.x + odd.y == 0.f)) odd_groups |= 1u << (j / 16);      // NaN: not all of P v are finite
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = 0u;
                    }
                    if (row < all) {
                        if (j < a.Dv) *reinterpret_cast<uint4 *>(to + j) = make_uint4(y[0], y[1], y[2], y[3]);
                        if (j + 8 < a.Dv) *reinterpret_cast<uint4 *>(to + j + 8) = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                }
                if (__any_sync(0xffffffffu, odd_groups)) again(odd_groups, from + L::INTER, r, w.b, w.h, t0, row, to, slots[g.buf]);
                tc::tc_fence_before_sync();
                tc::mbar_arrive(&s.o_empty);
                tc::mbar_arrive(&s.g_empty[g.buf]);
            }
            for (int c = w.stop; c < w.end; ++c)               // behind the sequence
                if (c * C + row < a.T)
                    for (int j = 0; j < a.Dv; j += 8) *reinterpret_cast<uint4 *>(out + (long long)c * C * a.out.ts + j) = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    // A later token's infinity or NaN is none of an earlier one's business, and zero times it is NaN: the sums again, over the tokens up
    // to this one, for the groups of sixteen columns that a lane has found odd.
    __device__ __noinline__ void again(uint32_t groups, uint32_t inter, float r, int b, int h, int t0, int row, bf16 *to, const Slot &g) const {
        const bf16 *q = static_cast<const bf16 *>(a.q.p) + at(a.q, b, h / p.share) + (long long)(t0 + row) * a.q.ts;
        const bf16 *k = static_cast<const bf16 *>(a.k.p) + at(a.k, b, h / p.share) + (long long)t0 * a.k.ts;
        const bf16 *v = static_cast<const bf16 *>(a.v.p) + at(a.v, b, h) + (long long)t0 * a.v.ts;
        for (int j = 0; j < DV; j += 16) {
            float x[16];
            tmem_load(inter + j, x);
            if (groups >> (j / 16) & 1) {
                for (int e = 0; e < 16; ++e) x[e] *= r;
                for (int t = 0; t <= row; ++t) {
                    float f = 0.f;
                    for (int d = 0; d < a.Dk; ++d) f = fmaf(seq::to_f(q[d]), seq::to_f(k[t * a.k.ts + d]), f);
                    f *= a.scale * ex2_diff(g.G(row), g.G(t));
                    for (int e = 0; e < 16; ++e)
                        if (j + e < a.Dv) x[e] = fmaf(f, seq::to_f(v[t * a.v.ts + j + e]), x[e]);
                }
                for (int e = 0; e < 16; ++e)
                    if (j + e < a.Dv) to[j + e] = __float2bfloat16_rn(x[e]);
            }
            __syncwarp();
        }
    }
};

template <int DK, int DV, bool Outputs, bool Reverse>
__global__ void __launch_bounds__(THREADS, 1) k_walk(const __grid_constant__ qgru_attention a, const __grid_constant__ Args p) {
    using L = Plan<DK, DV, Outputs, Reverse>;
    extern __shared__ unsigned char raw[];
    unsigned char *tiles = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    Slot *slots = reinterpret_cast<Slot *>(tiles + L::TILES);
    Ctl &s = *reinterpret_cast<Ctl *>(slots + SLOTS);
    using G = Regs<DK == 64 ? DV / 2 : DV>;
    const int tid = threadIdx.x, wg = tid / WG;
    if (tid == 0) {
        constexpr int readers = (Outputs ? 4 : 2) * WG;
        for (int i = 0; i < 3; ++i) {
            tc::mbar_init(&s.k_full[i], 1);
            tc::mbar_init(&s.k_empty[i], WG + (Outputs ? 1 : 0));
            tc::mbar_init(&s.q_full[i], 1);
            tc::mbar_init(&s.q_empty[i], 1);
            tc::mbar_init(&s.v_full[i], 1);
            tc::mbar_init(&s.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&s.parts_full[i], WG);
            tc::mbar_init(&s.parts_empty[i], 1);
            tc::mbar_init(&s.pairs_full[i], 1);
            tc::mbar_init(&s.p_full[i], WG);
            tc::mbar_init(&s.ring_full[i], 1);
            tc::mbar_init(&s.ring_empty[i], WG);
        }
        for (int i = 0; i < SLOTS; ++i) {
            tc::mbar_init(&s.g_full[i], 32);
            tc::mbar_init(&s.g_empty[i], readers);
        }
        tc::mbar_init(&s.u_full, 1);
        tc::mbar_init(&s.u_empty, WG);
        tc::mbar_init(&s.s_full, WG);
        tc::mbar_init(&s.o_empty, WG);
        s.failed = 0;
        tc::fence_barrier_init();
        tc::tma_prefetch_desc(&p.k);
        tc::tma_prefetch_desc(&p.v);
        if (Outputs) tc::tma_prefetch_desc(&p.q);
    }
    if (tid < 32) tc::tmem_alloc(&s.tmem, L::COLUMNS);
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const Roles<DK, DV, Outputs, Reverse> r{a, p, s, slots, tc::smem_u32(tiles), tid % WG};
    if (wg == 0) {
        take_registers<G::X>();
        const int warp = tid >> 5;
        if (warp == 0) {
            r.issue();
        } else if (warp == 1) {
            if (tid == 32) r.fetch();
        } else {
            r.decays();
        }
        __syncwarp();
    } else if (wg == 1) {
        take_registers<G::K>();
        r.split();
    } else if (wg == 2) {
        take_registers<G::S>();
        r.states();
    } else if (wg == 3) {
        take_registers<G::P>();
        if constexpr (Outputs) r.weights();
        if (Reverse && !p.own_sums && tid == 3 * WG) r.fetch_states();
        __syncwarp();
    } else {
        take_registers<G::O>();
        if constexpr (Outputs) r.outputs();
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    if (s.failed) {            // copies and products may be under way: a millisecond is far more than they take
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) {
        }
        if (tid == 0) *p.flag = 1;
    }
    if (tid < 32) tc::tmem_dealloc(s.tmem, L::COLUMNS);
}

// ------------------------------------------------------------------------------------- launches
template <int DK, int DV, bool Outputs, bool Reverse>
int launch(const qgru_attention &a, const Args &p, int sms, cudaStream_t st) {
    const auto kernel = k_walk<DK, DV, Outputs, Reverse>;
    constexpr int bytes = Plan<DK, DV, Outputs, Reverse>::TILES + 1024 + SLOTS * (int)sizeof(Slot) + (int)sizeof(Ctl);
    static_assert(bytes <= 232448, "shared memory");
    SEQ_CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    kernel<<<std::min(p.items, sms), THREADS, bytes, st>>>(a, p);
    SEQ_CK(cudaGetLastError());
    return QGRU_OK;
}

template <int DK, int DV, bool Reverse>
int run(const qgru_attention &a, const Cut &c, bf16 *states, char *seg, float *through, int *flag, int sms, cudaStream_t st) {
    Args p{};
    p.other = static_cast<const bf16 *>(a.states);
    p.through = through;
    const qgru_seq_tensor &k = Reverse ? a.q : a.k, &v = Reverse ? a.dout : a.v;
    if (a.T > 0 && (!head_map(&p.k, k, a.T, a.B, a.Hk, a.Dk) || !head_map(&p.v, v, a.T, a.B, a.H, a.Dv) || !head_map(&p.q, a.q, a.T, a.B, a.Hk, a.Dk)))
        return seq::fail(QGRU_ERR_CUDA, "cuTensorMapEncodeTiled");
    p.first = Reverse ? a.dstate : a.state0;
    p.last = Reverse ? a.dstate0 : a.state;
    p.states = states;
    p.segments = c.segments;
    p.per = c.per;
    p.chunks = c.chunks;
    p.share = a.H / a.Hk;
    p.items = a.B * a.H * c.segments;
    p.flag = flag;
    if (c.segments > 1) {
        p.seg_state = reinterpret_cast<float *>(seg);
        p.seg_log = p.seg_state + c.segments * state_elems(a);
        p.own_sums = 1;
        if (const int rc = launch<DK, DV, false, Reverse>(a, p, sms, st)) return rc;
        if (const int rc = scan_segments(a, c, Reverse, seg, st)) return rc;
        p.own_sums = 0;
    }
    return launch<DK, DV, !Reverse, Reverse>(a, p, sms, st);
}

}  // namespace

bool head_map(CUtensorMap *map, const qgru_seq_tensor &x, int T, int B, int heads, int d) {
    const EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)T, (cuuint64_t)heads, (cuuint64_t)B};
    // (the stride of a dimension of one is nobody's)
    const auto bytes = [](long long s, int n) { return n > 1 ? (cuuint64_t)s * 2 : (cuuint64_t)256; };
    const cuuint64_t strides[3] = {bytes(x.ts, T), bytes(x.hs, heads), bytes(x.bs, B)};
    const cuuint32_t box[4] = {64, C, 1, 1}, step[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, x.p, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool fetchable(const qgru_seq_tensor &x, int T, int B, int heads, int d) {
    const auto ok = [](long long s, int n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };       // (a stride of 0 is not for TMA)
    return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && d % 8 == 0 && ok(x.ts, T) && ok(x.bs, B) && ok(x.hs, heads);
}


// Whether the tensors can be fetched by TMA and written in vectors: rows and strides of a multiple of 16 bytes.
bool walk_takes(const qgru_attention &a, bool reverse) {
    const auto dense = [](const float *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (reverse) return fetchable(a.q, a.T, a.B, a.Hk, a.Dk) && fetchable(a.dout, a.T, a.B, a.H, a.Dv) && dense(a.dstate) && dense(a.dstate0);
    return fetchable(a.q, a.T, a.B, a.Hk, a.Dk) && fetchable(a.k, a.T, a.B, a.Hk, a.Dk) && fetchable(a.v, a.T, a.B, a.H, a.Dv) &&
           fetchable(a.out, a.T, a.B, a.H, a.Dv) && dense(a.state0) && dense(a.state);
}
int walk(const qgru_attention &a, const Cut &c, bool reverse, void *states, char *seg, float *through, int *flag, int sms, cudaStream_t st) {
    using std::integral_constant;
    const auto with = [&](auto dk, auto dv) -> int {
        bf16 *to = static_cast<bf16 *>(states);
        return reverse ? run<dk.value, dv.value, true>(a, c, to, seg, through, flag, sms, st) : run<dk.value, dv.value, false>(a, c, to, seg, through, flag, sms, st);
    };
    const integral_constant<int, 64> small;
    const integral_constant<int, 128> large;
    return a.Dk <= 64 ? (a.Dv <= 64 ? with(small, small) : with(small, large)) : (a.Dv <= 64 ? with(large, small) : with(large, large));
}

}  // namespace attn
}  // namespace qgru
