// qgru_attn_tc.cuh - linear attention on the tensor cores (qgru_attn_fwd.cu, qgru_attn_tc.cu): tiles, products, values.
//
// All products are tcgen05.mma kind::f16 with fp32 sums in tensor memory and bf16 operands in shared memory as rows of 128 bytes
// with the 128-byte swizzle.  Such a tile [rows][64 columns] is an operand with its columns as K (K-major) and one with its
// rows as K (MN-major), so that no operand is transposed anywhere.
#pragma once
#include "qgru_attn.cuh"
#include "qgru_tc.cuh"

namespace qgru {
namespace attn {

bool tc_takes(const qgru_attention &a);
Cut tc_cut(const qgru_attention &a, int sms);
// flag: where a kernel says that a wait of its own has run out
int tc_forward(const qgru_attention &a, const Cut &c, int *flag, int sms, cudaStream_t st);
int tc_backward(const qgru_attention &a, const Cut &c, int *flag, int sms, cudaStream_t st);
// Tensor map of a tensor's heads ([B][heads][T][D], boxes of 128 tokens x 64 columns); fetchable: whether TMA takes a tensor (rows and strides multiples of 16 bytes, no stride of 0)
bool head_map(CUtensorMap *map, const qgru_seq_tensor &x, int T, int B, int heads, int d);
bool fetchable(const qgru_seq_tensor &x, int T, int B, int heads, int d);
// A walk through the chunks (qgru_attn_fwd.cu): forward with the outputs, or from the end with the gradient of the states alone
bool walk_takes(const qgru_attention &a, bool reverse);
int walk(const qgru_attention &a, const Cut &c, bool reverse, void *states, char *seg, float *through, int *flag, int sms, cudaStream_t st);
// The pass from the end meets every state's gradient in fp32: it multiplies it with the state, as it was kept, and leaves the sum in
// THROUGH parts a chunk and head (the sums of its warps).  A state is kept as 32 bits, the two bf16 parts (16 of its bits) that the
// products take it in: [chunk][B H][part][DV / 8][DK][8], so that the threads of a warp, a row each, read and write whole lines (row by row,
// with 16 bytes of 32 lines an instruction, the two passes took 86 and 66 us where they take 65 and 58, and 46 with the
// states on their way through shared memory; 16 x 1000 tokens of 8 heads of 128).
constexpr int THROUGH = 8;

namespace tile {

constexpr int C = 128;                                 // tokens of a chunk
constexpr int PANEL = C * 128;                          // bytes of 64 columns of a tile of 128 rows
constexpr long long WAIT_BUDGET = 2000000000ll;         // about a second of SM clocks
using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------- operands and products
constexpr uint32_t DESC_HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);     // groups of eight rows 1024 bytes apart, 128-byte swizzle

struct Operand {                        // a tile, `panel` bytes from 64 columns to the next
    uint32_t at;
    int panel;
};
// Low word of the descriptor, and what K = 16 j .. 16 j + 15 adds to it (16-byte units; addresses below 2^18 never carry out of the
// field).  K in the columns: 32 bytes a step, four steps a panel.  K in the rows: 2048 bytes (sixteen rows) a step, and the
// descriptor's leading distance is that between panels.
template <bool KRows>
__device__ __forceinline__ uint32_t desc_lo(const Operand &o) {
    return ((o.at & 0x3FFFFu) >> 4) | (KRows ? (uint32_t)o.panel >> 4 << 16 : 1u << 16);
}
template <bool KRows>
__device__ __forceinline__ uint32_t desc_step(const Operand &o, int j) {
    return KRows ? j * (2048 >> 4) : (j >> 2) * (o.panel >> 4) + (j & 3) * (32 >> 4);
}
// D fp32, A and B bf16, M = 128
__host__ __device__ constexpr uint32_t idesc(int N, bool a_rows, bool b_rows) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_rows ? 1u : 0u) << 15) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Products and their commits are issued by one lane of a warp that stays together: operands of tcgen05.mma are warp-uniform
// registers, and in a branch of one thread every one of them costs a move from an ordinary register (about 110 cycles an
// instruction then, 128 x 64 x 16).
__device__ __forceinline__ uint32_t elect() {
    uint32_t r;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(r));
    return r;
}
template <uint32_t B_HI = DESC_HI>
__device__ __forceinline__ void mma(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        ".reg .b64 da, db;\n"
        "mov.b64 da, {%1, %5};\n"
        "mov.b64 db, {%2, %7};\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 e, %6, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(id), "r"(accumulate), "n"(DESC_HI), "r"(leader), "n"(B_HI)
        : "memory");
}
// A from tensor memory: lane i is row i, a column holds two neighbouring K, sixteen K are eight columns
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        ".reg .b64 db;\n"
        "mov.b64 db, {%2, %5};\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 e, %6, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(id), "r"(accumulate), "n"(DESC_HI), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t *bar) {
    asm volatile(
        "{\n"
        ".reg .pred e;\n"
        "setp.ne.b32 e, %1, 0;\n"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(tc::smem_u32(bar)),
        "r"(leader)
        : "memory");
}
// (Loops over 64 K, four instructions each: warps that do different things share one small instruction cache.)
template <bool ARows, bool BRows, int N, int K>
__device__ __forceinline__ void product(uint32_t leader, uint32_t d, const Operand &a, const Operand &b, bool add) {
    uint32_t a0 = desc_lo<ARows>(a), b0 = desc_lo<BRows>(b), more = add;
#pragma unroll 1
    for (int p = 0; p < K / 64; ++p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mma(leader, d, a0 + desc_step<ARows>(a, j), b0 + desc_step<BRows>(b, j), idesc(N, ARows, BRows), j ? 1u : more);
        a0 += desc_step<ARows>(a, 4);
        b0 += desc_step<BRows>(b, 4);
        more = 1;
    }
}
// B a part of a state as it is kept, [columns / 8][Rows][8] without a swizzle: groups of eight rows are 128 bytes apart, neighbouring
// eights of columns 16 Rows.  K in the columns (N in the rows), or the other way: the descriptor's leading distance is K's then, its stride N's.
template <bool BRows, int N, int K, int Rows>
__device__ __forceinline__ void product_state(uint32_t leader, uint32_t d, const Operand &a, uint32_t b, bool add) {
    constexpr uint32_t HI = (uint32_t)(BRows ? Rows : 128 >> 4) | (1u << 14), STEP = BRows ? 256 >> 4 : 2 * Rows;
    uint32_t a0 = desc_lo<false>(a), b0 = ((b & 0x3FFFFu) >> 4) | (uint32_t)(BRows ? 128 >> 4 : Rows) << 16, more = add;
#pragma unroll 1
    for (int p = 0; p < K / 64; ++p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) mma<HI>(leader, d, a0 + desc_step<false>(a, j), b0 + j * STEP, idesc(N, false, BRows), j ? 1u : more);
        a0 += desc_step<false>(a, 4);
        b0 += 4 * STEP;
        more = 1;
    }
}
// A as two parts: of each sixteen columns the first eight hold sixteen K of the large part, the others those of the small one, where their
// sixteen fp32 values were before.
template <bool BRows, int N, int K>
__device__ __forceinline__ void product_ts(uint32_t leader, uint32_t d, uint32_t a, const Operand &b, bool add) {
    uint32_t b0 = desc_lo<BRows>(b), more = add;
#pragma unroll 1
    for (int p = 0; p < K / 64; ++p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mma_ts(leader, d, a + j * 16 + 8, b0 + desc_step<BRows>(b, j), idesc(N, false, BRows), j ? 1u : more);
            mma_ts(leader, d, a + j * 16, b0 + desc_step<BRows>(b, j), idesc(N, false, BRows), 1u);
        }
        a += 64;
        b0 += desc_step<BRows>(b, 4);
        more = 1;
    }
}

__device__ __forceinline__ uint32_t lane_base(uint32_t tmem, int warp) { return tmem + ((uint32_t)((warp & 3) * 32) << 16); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                 "r"(v[14]), "r"(v[15])
                 : "memory");
}
// Cols / 16 groups of sixteen columns
template <int Cols>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[Cols]) {
    int32_t r[Cols / 16][16];
#pragma unroll
    for (int i = 0; i < Cols / 16; ++i) tc::tmem_ld16(taddr + i * 16, r[i]);
    tc::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < Cols; ++i) v[i] = __int_as_float(r[i / 16][i % 16]);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, float2 (&v)[8]) {
    int32_t r[16];
    tc::tmem_ld16(taddr, r);
    tc::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = make_float2(__int_as_float(r[2 * i]), __int_as_float(r[2 * i + 1]));
}
template <int Cols>
__device__ __forceinline__ void tmem_store(uint32_t taddr, const uint32_t (&v)[Cols]) {
#pragma unroll
    for (int i = 0; i < Cols / 16; ++i) {
        uint32_t r[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = v[i * 16 + j];
        tmem_st16(taddr + i * 16, r);
    }
}

// ------------------------------------------------------------------------------------- values
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack(float2 x) { return pack(x.x, x.y); }
// The first of several parts: the largest finite value for an infinity, so that what is left of it is the infinity and not NaN
__device__ __forceinline__ uint32_t pack_part(float2 x) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
    return r;
}
__device__ __forceinline__ float2 unpack(uint32_t x) { return make_float2(low(x), high(x)); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// Eight values, packed, times eight of a state's
__device__ __forceinline__ float2 dot8(const uint4 &u, const float2 *s, float2 sum) {
    sum = __ffma2_rn(unpack(u.x), s[0], sum);
    sum = __ffma2_rn(unpack(u.y), s[1], sum);
    sum = __ffma2_rn(unpack(u.z), s[2], sum);
    return __ffma2_rn(unpack(u.w), s[3], sum);
}
// x minus what its first part keeps (exact)
__device__ __forceinline__ float2 rest(float2 x, uint32_t packed) { return __ffma2_rn(unpack(packed), make_float2(-1.f, -1.f), x); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float ex2_diff(float2 t, float2 s) { return ex2((t.x - s.x) + (t.y - s.y)); }

// 16-byte chunk c (of eight columns) of row r of a panel
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ void bulk_load(uint32_t to, const void *from, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t to, const CUtensorMap *map, uint64_t *bar, int x, int t, int h, int b) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(to),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(x), "r"(t), "r"(h), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap *map, uint32_t from, int x, int t, int h, int b) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(from),
                 "r"(x), "r"(t), "r"(h), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }       // their tiles are free
__device__ __forceinline__ void cp_async(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int Left>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(Left) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ long long at(const qgru_seq_tensor &x, int b, int h) { return b * x.bs + h * x.hs; }

// A thread's Cols neighbouring columns, from `c0` on, of a row of bf16.
template <int Cols>
__device__ __forceinline__ void store_row(bf16 *row, const float (&v)[Cols], int c0, int d, bool vec) {
#pragma unroll
    for (int i = 0; i < Cols; i += 8) {
        if (vec) {
            if (c0 + i < d) *reinterpret_cast<uint4 *>(row + c0 + i) = make_uint4(pack(v[i], v[i + 1]), pack(v[i + 2], v[i + 3]), pack(v[i + 4], v[i + 5]), pack(v[i + 6], v[i + 7]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + i + j < d) row[c0 + i + j] = __float2bfloat16_rn(v[i + j]);
        }
    }
}

}  // namespace tile
}  // namespace attn
}  // namespace qgru
