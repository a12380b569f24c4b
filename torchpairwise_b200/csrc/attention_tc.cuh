// What the tensor-core attention kernels share: tcgen05 wrappers for 16-bit operands, tiles of [tokens, features] in shared memory
// and their descriptors, and the exponential.
//
// A tile of 128 tokens lies in shared memory as one or two blocks of 64 features (128 tokens x 128 bytes, 128-byte swizzle), 16 KB each,
// as TMA writes it.  The same bytes serve a product that contracts the features (K-major operand) and one that contracts the tokens
// (MN-major operand).
#pragma once
#include "attention.cuh"
#include "packed_f32x2.cuh"
#include "tcgen05.cuh"

namespace tpw {
namespace {

constexpr int TILE = 128;                  // tokens per tile
constexpr uint32_t BLOCK_BYTES = 16384;    // 128 tokens x 64 features

template <typename T> struct Narrow;
template <> struct Narrow<__nv_bfloat16> {
    static constexpr uint32_t kFormat = 1;   // of the instruction descriptor
    static constexpr float kLift = 0.f;      // probabilities are formed times 2^kLift: bfloat16 has the exponents of float32
    static constexpr float kSlack = 40.f;    // and may exceed 1 by 2^kSlack
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ uint32_t rest(float lo, float hi) {   // of what pack makes of them
        const uint32_t w = pack(lo, hi);
        return pack(lo - __uint_as_float(w << 16), hi - __uint_as_float(w & 0xffff0000u));
    }
};
template <> struct Narrow<__half> {
    static constexpr uint32_t kFormat = 0;
    static constexpr float kLift = 6.f;      // and half precision loses digits below 2^-14: see attention_forward.cu
    static constexpr float kSlack = 8.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ uint32_t rest(float lo, float hi) {
        const float2 w = __half22float2(__floats2half2_rn(lo, hi));
        return pack(lo - w.x, hi - w.y);
    }
};

// The lane that issues for its warp.  The whole warp runs through the issuing code and the instructions themselves are predicated: their operands
// then live in uniform registers.  Under a branch on the lane the compiler moves every operand there anew, 80 to 125 clocks per MMA.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// D[tmem] (+)= A[smem] B[smem] and D[tmem] (+)= A[tmem] B[smem]; operands of one 16-bit type, fp32 accumulate, K = 16
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t leader, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(leader)
        : "memory");
}
// fp32 accumulators (bits [4,6) = 1), A and B formats in [7,10) and [10,13), bit 16: B is MN-major, N >> 3 in [17,23), M >> 4 in [24,29)
__device__ __forceinline__ uint32_t instruction(uint32_t format, uint32_t n, bool b_mn) {
    return (1u << 4) | (format << 7) | (format << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
}
// MN-major 16-bit tile, 128-byte swizzle: groups of eight tokens 1024 bytes apart, blocks of 64 features BLOCK_BYTES apart
__device__ __forceinline__ uint64_t make_smem_desc_tokens(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(BLOCK_BYTES >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// start of the k-th 16 features of a K-major tile, in units of 16 bytes
__device__ __forceinline__ uint64_t feature_step(int k) { return (uint64_t)((k >> 2) * (BLOCK_BYTES >> 4) + (k & 3) * 2); }
// D = X Y^T over 16 * steps features, at most 64 * BLOCKS; X, Y tiles
template <int BLOCKS> __device__ __forceinline__ void product_features(uint32_t leader, uint32_t d, uint32_t x, uint32_t y, uint32_t idesc, int steps) {
    const uint64_t a = make_smem_desc(x), b = make_smem_desc(y);
#pragma unroll
    for (int k = 0; k < 4 * BLOCKS; ++k)
        if (k < steps) mma_ss(leader, d, a + feature_step(k), b + feature_step(k), idesc, k != 0);
}
// D (+)= P Y over the tokens [16 FROM, 16 TO) of a tile; P in tensor memory, 16 tokens to 8 columns, its second half `gap` columns behind the
// first's start
template <int FROM = 0, int TO = TILE / 16>
__device__ __forceinline__ void product_tokens(uint32_t leader, uint32_t d, uint32_t p, uint32_t gap, uint32_t y, uint32_t idesc, bool accumulate) {
    const uint64_t b = make_smem_desc_tokens(y);
#pragma unroll
    for (int k = FROM; k < TO; ++k)
        mma_ts(leader, d, p + (k < 4 ? 8 * k : gap + 8 * (k - 4)), b + (uint64_t)k * (2048 >> 4), idesc, accumulate || k != 0);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
// 16 lanes x 64 columns, spread like an mma accumulator: thread 4 g + t has, of the i-th eight columns, 2 t and 2 t + 1 of lane g (registers
// 4 i, 4 i + 1) and of lane g + 8 (4 i + 2, 4 i + 3)
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// 16 lanes x 32 columns: thread 4 g + t has column t of the i-th four, of lane g (register 2 i) and of lane g + 8 (2 i + 1)
__device__ __forceinline__ void tmem_st_16x128(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}
// tile of 128 tokens, BLOCKS blocks of 64 features
template <int BLOCKS>
__device__ __forceinline__ void load_tokens(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int token, int head, int batch) {
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) tma_load_4d(dst + c * BLOCK_BYTES, map, bar, 64 * c, token, head, batch);
}
// Tokens [from, 128) of a tile set to zero by one warp, visible to the tensor cores: what lies there belongs to no key, and 0 times it
// need not be 0.
template <int BLOCKS> __device__ __forceinline__ void clear_tokens(unsigned char *tile, int from, int lane) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = 0; c < BLOCKS; ++c)
        for (int at = from * 8 + lane; at < TILE * 8; at += 32) *reinterpret_cast<uint4 *>(tile + c * BLOCK_BYTES + at * 16) = zero;
    fence_proxy_async_smem();
    __syncwarp();
}

// Registers per thread of a warpgroup.  A block of 384 threads is launched with 168 each, 64512: two warpgroups at 208 and one at 88.
constexpr int kTcThreads = 384;
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }

// Persistent CTAs: a CTA that is done takes over a block of the grid that has not been launched yet (cluster launch control), instead of
// ending and leaving the SM to set up the next one: launch, barriers, tensor memory and first loads are 7 us a block here.  The TMA lane
// asks; the others learn the answer from a ring of two, and say when they have read it.
struct BlockQueue {
    uint64_t *answered, *read;   // [2] each
    uint32_t response;           // shared-memory address of two times 16 bytes, 16-byte aligned
    __device__ __forceinline__ void init(uint32_t readers) const {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&answered[i], 1);
            mbar_init(&read[i], readers);
        }
    }
    // The TMA lane, when it has issued the loads of its n-th block: asked for earlier, a block would wait behind a long one while other SMs
    // run dry ([4, 1500 x 2111, 16, 64] with ragged lengths, asked for at a block's start: 105 us instead of 74).  False after a
    // wait that gave up.
    template <typename W> __device__ __forceinline__ bool ask(uint32_t n, W wait) const {
        const uint32_t s = n & 1;
        if (n >= 2 && !wait(&read[s], (n >> 1 & 1) ^ 1)) return false;
        mbar_expect_tx(&answered[s], 16);
        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(response + 16 * s),
                     "r"(smem_u32(&answered[s]))
                     : "memory");
        if (wait(&answered[s], n >> 1 & 1)) return true;
        mbar_wait_bounded(&answered[s], n >> 1 & 1);   // it arrives before the CTA ends
        return false;
    }
    __device__ __forceinline__ bool answer(uint32_t s, unsigned &block) const {
        uint32_t got;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
            "ld.shared.b128 r, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "mov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, r;\n\t}"
            : "=r"(got), "=r"(block)
            : "r"(response + 16 * s)
            : "memory");
        return got != 0;
    }
    // A reading warp (or lane): the n-th block after the first; false: there is none.  `one`: the lane that says it has read.
    template <bool WARP, typename W> __device__ __forceinline__ bool next(uint32_t n, unsigned &block, bool one, W wait) const {
        const uint32_t s = n & 1;
        if (!wait(&answered[s], n >> 1 & 1)) return false;
        const bool got = answer(s, block);
        fence_proxy_async_smem();   // read before the next answer is written there
        if (WARP) __syncwarp();
        if (one) mbar_arrive(&read[s]);
        return got;
    }
};

// 32 rows of a warp on their way to global memory: a lane has a row and puts it down in pieces of 16 bytes, the warp then stores whole
// rows.  Straight from a row per lane every store would touch 32 half sectors.
template <int PIECES> struct RowStage {
    uint4 *at;   // the warp's own 32 * PIECES pieces of shared memory, no longer in use
    static __device__ __forceinline__ int place(int row, int piece) {
        return row * PIECES + (piece ^ (PIECES >= 8 ? row & 7 : (row * PIECES / 8) & (PIECES - 1)));
    }
    __device__ __forceinline__ void put(int lane, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const { at[place(lane, piece)] = make_uint4(a, b, c, d); }
    // rows below `valid`, pieces below `width`; row_bytes apart
    __device__ __forceinline__ void store(unsigned char *to, long long row_bytes, int lane, int valid, int width) const {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int row = (32 * k + lane) / PIECES, piece = lane % PIECES;
            if (row < valid && piece < width) *reinterpret_cast<uint4 *>(to + row * row_bytes + piece * 16) = at[place(row, piece)];
        }
        __syncwarp();
    }
};

// 32 rows of 64 features on their way from a warp to global memory: a lane puts its row down in pieces of 16 bytes (128-byte swizzle), then the copy
// engine takes the block, clipped to the tensor, while the warp goes on.  Plain stores held the warp up for 2 us a block when all
// SMs wrote at once.  The 4 KB are 1024-byte aligned and the warp's own.
struct RowBlock {
    unsigned char *at;
    __device__ __forceinline__ void put(int lane, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
        *reinterpret_cast<uint4 *>(at + swz128(lane, piece)) = make_uint4(a, b, c, d);
    }
    // before the next block is put down: the last one has been read
    static __device__ __forceinline__ void reuse(int lane) {
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
    }
    __device__ __forceinline__ void send(int lane, const CUtensorMap *map, int feature, int token, int head, int batch) const {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(reinterpret_cast<uint64_t>(map)),
                         "r"(feature), "r"(token), "r"(head), "r"(batch), "r"(smem_u32(at))
                         : "memory");
            tma_store_commit();
        }
    }
};

// n / d for n < 2^31 by a multiplication; prepared on the host
struct Divider {
    uint32_t d, mul, shift;
};
inline Divider divider(long long d) {
    Divider r = {(uint32_t)d, 0, 0};
    while ((1ll << r.shift) < d) ++r.shift;
    r.mul = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - (uint64_t)d)) / (uint64_t)d + 1);
    return r;
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const Divider &by) { return (__umulhi(n, by.mul) + n) >> by.shift; }
__device__ __forceinline__ uint32_t operator%(uint32_t n, const Divider &by) { return n - (n / by) * by.d; }

__device__ __forceinline__ float exp2_fast(float x) {   // 2 units of the last place; 0 below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// NaN if any operand is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^z of a pair on the FMA pipes: 2^n 2^f with n the nearest whole number and f in [-1/2, 1/2], where the polynomial (relative minimax fit of
// degree 4, by the exchange algorithm) is good to 2.6e-6.  Below 2^-126 it stays there: beside a row's largest term that is zero.  NaN
// gives 2^128 - 2^104, infinity in 16 bits.
// The special-function units make 16 exponentials a clock and SM; the gradient walks take a quarter of theirs from here ([2, 4096, 16, 64]
// 599 -> 556 us, with half of them 584).
__device__ __forceinline__ f32x2 exp2_polynomial(f32x2 z) {
    float z0, z1;
    unpack2(z, z0, z1);
    z = pack2(max3_nan(z0, -126.f, -126.f), max3_nan(z1, -126.f, -126.f));
    const f32x2 magic = pack2(12582912.f, 12582912.f);   // 1.5 * 2^23: a sum with it ends in the nearest whole number
    const f32x2 n = add2(z, magic), f = sub2(z, sub2(n, magic));
    f32x2 p = pack2(0.009570102207362652f, 0.009570102207362652f);
    p = fma2(p, f, pack2(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, f, pack2(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, f, pack2(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, pack2(0.9999992847442627f, 0.9999992847442627f));
    float p0, p1, n0, n1;
    unpack2(p, p0, p1);
    unpack2(n, n0, n1);
    return pack2(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(n0) << 23)), __uint_as_float(__float_as_uint(p1) + (__float_as_uint(n1) << 23)));
}
__device__ __forceinline__ f32x2 exp2_pair(f32x2 z) {
    float z0, z1;
    unpack2(z, z0, z1);
    return pack2(exp2_fast(z0), exp2_fast(z1));
}
} // namespace
} // namespace tpw
