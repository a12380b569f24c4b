// Attention of few query rows over a cache of quantised keys and values: one or a few new tokens against long sequences.
//
// Bound by HBM (4-bit codes with their steps and zeros: 160 bytes for a key and value of 128 features), closely followed by the instructions that unpack
// them.  So the codes go into the products as they are: as the low bits of half-precision numbers they are whole multiples of 2^-24,
// exactly, and masks are all the unpacking there is.
//   scores   K q^T, m16n8k16, 16 keys by 8 query rows: sum_g step_jg (sum_d c_jd q_d) + zero_jg a_g, a_g = sum_d q_d over the group.  The second
//            term is a product of its own, bfloat16: words of the cache, step and zero, are the operand, beside 0 (or M a_g, below) and a_g in four parts,
//            32 bits (two parts left 2^-17 of every term: log-sums of keys far from zero were off by 1e-5).  A row of q is lifted by a power of two to half
//            precision's upper end.
//   output   V^T P^T, 16 features by 8 rows: the steps go into the probabilities, y_jg = p_j step_jg, formed in 32 bits and rounded to half precision
//            once: sum_j y_jg (c_jd - M) + p_j (zero_jg + M step_jg), M the middle code, so that a rounding counts by how far a value is from its group's
//            middle.  The second term stays in 32 bits; M sum_j y_jg comes from a product with ones, and is taken off every second stage: tensor cores cut sums
//            off at 24 digits, which over 65536 keys attended to evenly cost 12 times a float16 rounding (35 times in 8 bits; 51.7 -> 52.6 us with it).
// Steps of one head may be any numbers from 2^-100 to 2^97, and half precision has 40 powers of two: a row of queries has a norm for every group,
// a power of two that brings the largest y_jg that it met to [4, 8).  So what a row loses (2^-27 of its largest share) depends neither on other groups, nor on
// other rows, nor on tokens that it gives no weight.  Norms move where references do, or where a step is far above those met.
// With keys along M a product has 8 rows of queries; rows along M would leave half of every product empty for up to 8 heads that share a key.
//
// Tensor-core sums truncate, so they are kept small: those of scores are of codes less M, or begin at -M a_g, with zero_jg + M step_jg in the second term.  (Not
// for 4-bit groups of 32 and 16-bit queries: 32 codes below 16 add up to little, and the beginnings would cost 16 registers of the 168 that three CTAs an SM
// leave, 51.3 -> 49.7 us without.)  Float32 queries: q and y as two half-precision parts each, what those leave is below 2^-23;
// codes less M as numbers, since the products of 4-bit codes below 2^-20 are lined up as if they were 2^-14 and lose 6 digits (errors of results 6e-6 -> 6e-7, no time; 16-bit queries
// keep those products, log-sums are good to 1e-6 of themselves), and the products of 16 keys with values go to sums in registers.
//
// All stages of keys (64 or 128) of all sequences and heads form one line that the CTAs, three on an SM, take equal shares of, whatever the lengths: a
// share ends and begins anywhere in a sequence.  What a CTA has of a head that others have parts of goes to scratch, and a second kernel, whose launch
// overlaps this one, weighs the parts together in their order.  In a CTA four warps take 16 keys or 32 of a stage each, with a running reference, sum and
// output of their own; bulk copies bring the stages into a ring, across the ends of heads.
//
// Measured bfloat16, 4 bits: [16, 1 x 16384, 32/8, 128] ragged, groups of 32, 185 MB in 52 us (3.6 TB/s), of which copies alone take 31;
// [64, 1 x 4096, 32/8, 128], one group, 158 MB in 46 us.  Norms by row and group cost 4 and 1 us of that against one power of two for all steps of a warp, which
// leaves groups beside a loud one, and tokens beside a loud token, without digits: 1.5 us the look at them at the beginning of a head, the rest products in 32 bits.
// Where tokens' values differ by factors of e (a normal deviation of their logarithm by 1 or 2) and scores by 20 the look is needed more often: 54 to 58 us and 44 to 46.
#pragma once
#include "attention_tc.cuh"
#include "cache.cuh"
#include "packed_f32x2.cuh"

namespace tpw {
namespace {

constexpr int kFewWarps = 4, kFewThreads = 128;
constexpr int kFewSlack = 8;          // probabilities may exceed their reference by 2^8
constexpr int kFewHighest = 110;      // norms go from 2^-110 to 2^110: p * norm * step never leaves the range of 32 bits on its way

struct CacheFewParams {
    CacheAttnParams a;
    int rows, row_blocks;            // group * Nq, and blocks of them
    int whole;                       // a CTA for each head and block of rows, no joining
    Divider by_nq, by_blocks;
    int q_vector;                    // rows of queries in 16-byte pieces
    float *part_out;                 // [CTA][2][rows of a block][features of a row in storage]: of a head begun by another CTA, of one that this CTA begins
    float2 *part_stats;              // [CTA][2][rows of a block]: reference (a power of 2) and sum
};

template <int BITS, int W, int NG, int NT, int PARTS> struct CacheFew {
    static constexpr int KEYS = BITS == 4 ? 128 : 64, OWN = KEYS / kFewWarps, SUB = OWN / 16;   // of a stage; a warp's of them, and blocks of 16
    static constexpr uint32_t ROW = W * 4 * BITS, CODES = KEYS * ROW, SCALES = KEYS * NG * 4, STAGE = 2 * (CODES + SCALES), DP = 32 * W, ROWS = 8 * NT;
    static constexpr int PER_SM = NT == 1 ? 3 : 2;
    static constexpr uint32_t NP = NG == 3 ? 4 : NG;   // words that a key's groups take
    static constexpr uint32_t STATS = kFewWarps * 8 * 8, PREPARED = kFewWarps * SUB * 16 * NP * 8, NORMS = kFewWarps * NT * 8 * NP * 4,
                              QUERIES = PARTS * NT * W * 512, SUMS = NT * (W + 1) * 32;
    static constexpr uint32_t ROOM = (NT == 1 ? 75776 : 112640) - STATS - PREPARED - NORMS - QUERIES - SUMS - 320;
    static constexpr int kStages = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
    static_assert(kStages >= 2, "a ring of two stages at least");
    static_assert(kFewWarps * 8 * DP * 4 <= STAGE, "the warps' 8 rows of results fit a stage");
    static constexpr uint32_t OFF_STATS = kStages * STAGE, OFF_PREPARED = OFF_STATS + STATS, OFF_NORMS = OFF_PREPARED + PREPARED, OFF_QUERIES = OFF_NORMS + NORMS, OFF_SUMS = OFF_QUERIES + QUERIES,
                              OFF_BAR = OFF_SUMS + SUMS, OFF_FLAG = OFF_BAR + 16 * kStages, ALLOC = OFF_FLAG + 16;
};

// D += A B, and D = C + A B where C stays
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_bf16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) { return Narrow<__half>::pack(lo, hi); }
__device__ __forceinline__ uint32_t half2_rest(float lo, float hi) { return Narrow<__half>::rest(lo, hi); }
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e < 1 ? 1 : e > 254 ? 254 : e) << 23); }   // 2^(e - 127)
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// N 32-bit words that lie together, in the widest pieces that their number allows
template <int N> __device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[k];
            w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const uint2 v = reinterpret_cast<const uint2 *>(p)[k];
            w[2 * k] = v.x; w[2 * k + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = reinterpret_cast<const uint32_t *>(p)[k];
    }
}

// N floats, likewise
template <uint32_t N> __device__ __forceinline__ void store_words(float *p, const float (&x)[N]) {
    if constexpr (N == 4) *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else if constexpr (N == 2) *reinterpret_cast<float2 *>(p) = make_float2(x[0], x[1]);
    else p[0] = x[0];
}
// N pairs of floats
template <int N> __device__ __forceinline__ void load_pairs(f32x2 (&x)[N], const float *p) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            const ulonglong2 v = reinterpret_cast<const ulonglong2 *>(p)[k];
            x[2 * k] = v.x; x[2 * k + 1] = v.y;
        }
    } else x[0] = *reinterpret_cast<const f32x2 *>(p);
}

// Two codes that masks left in halves as numbers, less the middle; `upper`: 16 times the codes of 4 bits
template <int BITS> __device__ __forceinline__ uint32_t numbers_of(uint32_t codes, bool upper) {
    constexpr float MIDDLE = BITS == 4 ? 8.f : 128.f;
    const uint32_t c = codes | 0x64006400u;   // 1024 and that
    const __half2 v = *reinterpret_cast<const __half2 *>(&c);
    const __half2 r = BITS == 4 && upper ? __hfma2(v, __float2half2_rn(0.0625f), __float2half2_rn(-64.f - MIDDLE)) : __hsub2(v, __float2half2_rn(1024.f + MIDDLE));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// 8 features of a row of queries in 32 bits, `n` of which there are
__device__ __forceinline__ void load_query(float (&x)[8], const CacheFewParams &F, long long at, int n) {
    const CacheAttnParams &P = F.a;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.f;
    if (n <= 0) return;
    if (P.dtype == TPW_F32) {
        const float *p = static_cast<const float *>(P.q) + at;
        if (F.q_vector) {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) x[k] = p[k];
        return;
    }
    const uint16_t *p = static_cast<const uint16_t *>(P.q) + at;
    alignas(16) uint16_t v[8] = {};
    if (F.q_vector) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
    else
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) v[k] = p[k];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = P.dtype == TPW_F16 ? __half2float(__ushort_as_half(v[k])) : __uint_as_float((uint32_t)v[k] << 16);
}
// 4 features of a row of results, `n` of which there are
__device__ __forceinline__ void store_out(const CacheAttnParams &P, long long at, const float (&x)[4], int n) {
    if (n <= 0) return;
    const bool vector = P.c.D % 4 == 0;
    if (P.dtype == TPW_F32) {
        float *p = static_cast<float *>(P.out) + at;
        if (vector) *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < n) p[k] = x[k];
        return;
    }
    uint16_t *p = static_cast<uint16_t *>(P.out) + at;
    const uint32_t a = P.dtype == TPW_F16 ? half2_of(x[0], x[1]) : Narrow<__nv_bfloat16>::pack(x[0], x[1]);
    const uint32_t b = P.dtype == TPW_F16 ? half2_of(x[2], x[3]) : Narrow<__nv_bfloat16>::pack(x[2], x[3]);
    if (vector) *reinterpret_cast<uint2 *>(p) = make_uint2(a, b);
    else {
        const uint16_t e[4] = {(uint16_t)a, (uint16_t)(a >> 16), (uint16_t)b, (uint16_t)(b >> 16)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) p[k] = e[k];
    }
}

// four features of row r from the weighed sums of values and of probabilities
__device__ __forceinline__ void finish(const CacheFewParams &F, int b, int hk, int r, int d, float (&v)[4], float reference, float sum) {
    const CacheAttnParams &P = F.a;
    const int over = (unsigned)r / F.by_nq, i = r - over * (int)P.Nq, h = (int)(hk * P.group) + over;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] *= inv;
        // A group of zeros has a step all the same, 2^-100, and M steps do not go without a rest, up to 2^-12 of them: below 2^-104 there is nothing else
        if (fabsf(v[e]) < 4.930380657631324e-32f) v[e] = 0.f;
    }
    if (d == 0 && P.lse) P.lse[(b * P.Hq + h) * P.Nq + i] = sum == 0.f ? -INFINITY : (reference + log2f(sum)) * 0.69314718055994531f;
    store_out(P, ((b * P.Nq + i) * P.Hq + h) * P.c.D + d, v, P.c.D - d);
}

// Of 16 keys, the one in slot s of a product (a row of K, a column of P).  In this order the rows that lanes of a quarter warp read lie in different
// banks for keys, and two by two for values.
__device__ __forceinline__ int key_of_slot(int s) {
    const int t = (s >> 1) & 3;
    return (s & 8) + ((s & 1) ? 4 + (t ^ 1) : t);
}
__device__ __forceinline__ int slot_of_key(int k) { return (k & 8) + ((k & 4) ? 2 * ((k & 3) ^ 1) + 1 : 2 * (k & 3)); }

// The keys of a sequence that any row sees, and their stages
template <int KEYS> struct Stages {
    int first, end, begin, count;
    __device__ __forceinline__ Stages(const CacheAttnParams &P, int b) {
        const CacheSeen see(P, b);
        first = see.lo(0);
        end = see.hi((int)P.Nq - 1);
        begin = first & ~63;
        count = end > first ? (end - begin + KEYS - 1) / KEYS : 0;
    }
    // of those, the keys that a block of rows sees: the stages stay, others are neither fetched nor looked at
    __device__ __forceinline__ void narrow(const CacheFewParams &F, int b, int row0, int rows) {
        const int nq = (int)F.a.Nq, last = (row0 + rows < F.rows ? row0 + rows : F.rows) - 1, i0 = row0 - (int)((unsigned)row0 / F.by_nq) * nq, i1 = i0 + last - row0;
        if (i1 >= nq) return;   // rows of two heads
        const CacheSeen see(F.a, b);
        first = see.lo(i0);
        end = see.hi(i1);
    }
};
// The line of all stages: sequences one after the other, a sequence's items (heads, and blocks of rows of each) one after the other, an item's
// stages in order.  An item with stages stands on the line for kFewExtra more, which come first: what beginning and ending it costs, 4 to 5 us beside
// 1.6 us a stage ([64, 1 x 4096] 55.6 us with 1, 47 with 3, 44 with 4 and what came meanwhile).
// Found by the whole CTA (128 threads): how long the line is, and the sequence that place `at` (or item `item` of sequence `of`) lies in.
constexpr int kFewExtra = 4;
struct Line {
    unsigned total, before;   // places in all; in sequences before `b`
    int b;
    // the first place of a CTA's share
    __device__ __forceinline__ unsigned start(unsigned share, unsigned shares) const { return total / shares * share + total % shares * share / shares; }
};
template <int KEYS> __device__ __forceinline__ Line line_of(const CacheFewParams &F, int share, int shares, int of, unsigned (&room)[kFewWarps + 2]) {
    const CacheAttnParams &P = F.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = (int)P.c.B, per = (B + kFewThreads - 1) / kFewThreads;
    const unsigned items = (unsigned)P.c.H * F.row_blocks;
    const int b0 = tid * per < B ? tid * per : B, b1 = b0 + per < B ? b0 + per : B;
    auto places = [&](int b) {
        const int n = Stages<KEYS>(P, b).count;
        return n > 0 ? (n + kFewExtra) * items : 0u;
    };
    unsigned mine = 0, last = 0;
    for (int b = b0; b < b1; ++b) mine += last = places(b);
    unsigned up = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += x;
    }
    if (lane == 31) room[warp] = up;
    __syncthreads();
    Line r = {0, 0, 0};
    unsigned before = up - mine;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
        if (w < warp) before += room[w];
        r.total += room[w];
    }
    const unsigned at = of < 0 ? r.start(share, shares) : 0;
    if (of < 0 ? before <= at && at < before + mine : b0 <= of && of < b1)
        for (int b = b0; b < b1; ++b) {
            const unsigned n = per == 1 ? last : places(b);
            if (of < 0 ? at < before + n : b == of) {
                room[kFewWarps] = b;
                room[kFewWarps + 1] = before;
                break;
            }
            before += n;
        }
    __syncthreads();
    r.b = (int)room[kFewWarps];
    r.before = room[kFewWarps + 1];
    return r;
}

template <int BITS, int W, int NG, int NT, int PARTS>
__global__ void __launch_bounds__(kFewThreads, CacheFew<BITS, W, NG, NT, PARTS>::PER_SM) cache_few_kernel(const CacheFewParams F) {
    typedef CacheFew<BITS, W, NG, NT, PARTS> L;
    const CacheAttnParams &P = F.a;
    constexpr int DP = 32 * W, ROWS = 8 * NT, SUB = L::SUB, KEYS = L::KEYS;
    constexpr bool WIDE = PARTS == 2;
    constexpr float MIDDLE = BITS == 4 ? 8.f : 128.f;
    constexpr bool SMALL = WIDE || NG == 1 || BITS == 8;   // sums of scores are less M a_g
    constexpr int ZEROS = NG > 2 && SMALL ? 2 : 1;                 // products that zeros take
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned room[kFewWarps + 2];
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_FLAG);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int nq = (int)P.Nq, items = (int)P.c.H * F.row_blocks;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *empty = full + L::kStages;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], kFewWarps); }
        *abort_flag = 0;
        mbar_init_fence();
    }
    // what came before has ended; the join may be set up meanwhile
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // this CTA's share: `total` stages from stage `stage` of item `item` of sequence b on
    int b, item, stage, total;
    if (F.whole) {
        b = (int)(blockIdx.x / items);
        item = (int)(blockIdx.x % items);
        stage = 0;
        total = Stages<KEYS>(P, b).count;
        __syncthreads();
    } else {
        const Line line = line_of<KEYS>(F, (int)blockIdx.x, (int)gridDim.x, -1, room);
        unsigned at = line.start(blockIdx.x, gridDim.x), to = line.start(blockIdx.x + 1, gridDim.x);
        if (at == to) return;
        b = line.b;
        unsigned n = Stages<KEYS>(P, b).count, inside = (at - line.before) % (n + kFewExtra);
        item = (int)((at - line.before) / (n + kFewExtra));
        stage = inside > kFewExtra ? (int)inside - kFewExtra : 0;
        // stages of the share: places that stand for one
        total = 0;
        for (int of = b, i = item; at < to;) {
            const unsigned places = n + kFewExtra - inside < to - at ? n + kFewExtra - inside : to - at, extra = inside < kFewExtra ? kFewExtra - inside : 0;
            total += places > extra ? (int)(places - extra) : 0;
            at += places;
            inside = 0;
            if (at < to && ++i == items) {
                i = 0;
                do n = Stages<KEYS>(P, ++of).count;
                while (n == 0);
            }
        }
        if (total == 0) return;
    }
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (23 << 16) | site);
    };

    // Warp 0 also issues the copies, as many stages ahead as the ring has room for: a lane each for the codes and scales of keys and values.
    int ahead_b = b, ahead_item = item, ahead_left = 0, ahead_key = 0, ahead_first = 0, ahead_end = 0, issued = 0;
    uint32_t issued_slot = 0, issued_phase = 1, slot = 0, phase = 0;   // of the next stage to be issued; of the next to be used
    const uint32_t copy_bytes = lane & 2 ? NG * 4 : L::ROW, copy_to = smem_u32(smem) + (lane & 2 ? 2 * L::CODES + (lane & 1) * L::SCALES : (lane & 1) * L::CODES);
    const unsigned char *copy_base = lane & 2 ? reinterpret_cast<const unsigned char *>(P.c.scales[lane & 1]) : P.c.codes[lane & 1], *copy_from = nullptr;
    bool ok = true;
    auto ahead_of = [&](int skip) {   // the next item's stages but for the first `skip`
        const int head = (int)((unsigned)ahead_item / F.by_blocks);
        Stages<KEYS> S(P, ahead_b);
        ahead_left = S.count - skip;
        ahead_key = S.begin + skip * KEYS;
        S.narrow(F, ahead_b, (ahead_item - head * F.row_blocks) * ROWS, ROWS);
        ahead_first = S.first;
        ahead_end = S.end;
        copy_from = copy_base + (((long long)ahead_b * P.c.H + head) * P.c.capacity + ahead_key) * copy_bytes;
    };
    auto fill = [&](int limit) {
        limit = limit < total ? limit : total;
        while (issued < limit && ok) {
            const uint32_t st = issued_slot;
            if (issued >= L::kStages && !(ok = __all_sync(0xffffffffu, wait_or_abort(&empty[st], issued_phase, abort_flag)))) {
                give_up(1);
                return;
            }
            if (++issued_slot == L::kStages) {
                issued_slot = 0;
                issued_phase ^= 1;
            }
            // the capacity and a stage's first key are multiples of 64
            const bool some = ahead_key < ahead_end && ahead_key + KEYS > ahead_first;
            const uint32_t n = (uint32_t)((int)P.c.capacity - ahead_key < KEYS ? (int)P.c.capacity - ahead_key : KEYS);
            if (lane == 0) {
                if (some) mbar_expect_tx(&full[st], n * 2 * (L::ROW + NG * 4));
                else mbar_arrive(&full[st]);
            }
            __syncwarp();
            if (some && lane < 4) bulk_load(copy_to + st * L::STAGE, copy_from, n * copy_bytes, &full[st]);
            ++issued;
            ahead_key += KEYS;
            copy_from += KEYS * copy_bytes;
            if (--ahead_left == 0 && issued < total) {
                if (++ahead_item == items) {
                    ahead_item = 0;
                    do ++ahead_b;
                    while (Stages<KEYS>(P, ahead_b).count == 0);
                }
                ahead_of(0);
            }
        }
    };
    // one stage for now: the queries are not to wait behind what all CTAs ask for
    if (warp == 0 && total > 0) {
        ahead_of(stage);
        fill(1);
    }

    float2 *stats = reinterpret_cast<float2 *>(smem + L::OFF_STATS);
    uint32_t *queries = reinterpret_cast<uint32_t *>(smem + L::OFF_QUERIES);   // [part][block][w][lane][4]
    float *query_sums = reinterpret_cast<float *>(smem + L::OFF_SUMS);         // [block][w and, last, the factor of scores][row]
    // a warp's own: of every 16 keys [slot][group] steps, then middles of values (zero + M step); of every row its norms
    constexpr int NP = L::NP;
    float *prepared = reinterpret_cast<float *>(smem + L::OFF_PREPARED) + warp * SUB * 32 * NP;
    float *norms = reinterpret_cast<float *>(smem + L::OFF_NORMS) + warp * NT * 8 * NP;
    const int slot0 = key_of_slot(g), value0 = t, value1 = 4 + (t ^ 1);   // and 8 more
    int used = 0;

    do {
        Stages<KEYS> S(P, b);
        const CacheSeen see(P, b);
        const int hk = (unsigned)item / F.by_blocks, row0 = (item - hk * F.row_blocks) * ROWS, stage0 = stage;
        S.narrow(F, b, row0, ROWS);
        const int stages = S.count - stage < total - used ? S.count - stage : total - used;
        // Queries as operands, a warp making those of every fourth block of 32 features: row g of a block, features 32 w + 8 t + (0 .. 7), in the order
        // in which masks leave the codes of a key.  Row r is query r % nq of head hk * group + r / nq.
#pragma unroll 1
        for (int unit = warp; unit < NT * W; unit += kFewWarps) {
            const int x = unit / W, w = unit % W, r = row0 + 8 * x + g;
            const bool valid = r < F.rows;
            const int h = valid ? (unsigned)r / F.by_nq : 0;
            const long long row = b * P.q_s[0] + (valid ? r - h * nq : 0) * P.q_s[1] + (hk * P.group + h) * P.q_s[2] + 8 * t;
            float y[8] = {}, top = 0.f;
#pragma unroll
            for (int v = 0; v < W; ++v) {
                float z[8];
                load_query(z, F, row + 32 * v, valid ? P.c.D - (32 * v + 8 * t) : 0);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    top = fmaxf(top, fabsf(z[n]));
                    if (v == w) y[n] = z[n];
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // into [2^14, 2^15)
            int lift = 14 + 127 - (int)(__float_as_uint(top) >> 23);
            lift = top == 0.f ? 0 : lift > 100 ? 100 : lift < -100 ? -100 : lift;
            const float by = power_of_two(127 + lift);
            float sum = 0.f;
            uint32_t parts[PARTS][4];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int n = BITS == 4 ? 2 * k + e : 4 * k + e;
                    const float s = BITS == 4 && e && !WIDE ? 0.0625f : 1.f, y0 = y[n] * by, y1 = y[n + (BITS == 4 ? 4 : 2)] * by;
                    const float h0 = __half2float(__float2half_rn(y0)), h1 = __half2float(__float2half_rn(y1));
                    parts[0][2 * k + e] = half2_of(h0 * s, h1 * s);
                    sum += h0 + h1;
                    if constexpr (WIDE) {
                        const float r0 = __half2float(__float2half_rn(y0 - h0)), r1 = __half2float(__float2half_rn(y1 - h1));
                        parts[1][2 * k + e] = half2_of(r0 * s, r1 * s);
                        sum += r0 + r1;
                    }
                }
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
                *reinterpret_cast<uint4 *>(queries + ((part * NT * W + unit) * 32 + lane) * 4) = make_uint4(parts[part][0], parts[part][1], parts[part][2], parts[part][3]);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t == 0) {
                query_sums[(x * (W + 1) + w) * 8 + g] = WIDE ? sum : sum * 5.9604644775390625e-8f;   // 2^-24, the unit of codes
                if (w == 0) query_sums[(x * (W + 1) + W) * 8 + g] = fmaxf(P.scale_log2 * power_of_two(127 + (WIDE ? 0 : 24) - lift), 1.17549435e-38f);
            }
        }
        __syncthreads();
        if (warp == 0 && used == 0) fill(L::kStages);
        uint32_t q[PARTS][NT][W][2][2], qz[NT][ZEROS][2];
        float start[NT][NG][4], factor[NT][2];   // -M a_g (SMALL, where codes are not less M already); raw scores times the factor are powers of 2
        int all_lo = S.first, all_hi = S.end;   // keys that all rows see
        auto sees = [&](int x, int e, int &lo, int &hi) {   // those of a row
            const int mine = row0 + 8 * x + 2 * t + e, i = mine < F.rows ? (unsigned)mine % F.by_nq : 0;
            lo = mine < F.rows ? see.lo(i) : 0;
            hi = mine < F.rows ? see.hi(i) : 1 << 30;
        };
        float m[NT][2], l[NT][2], o[NT][2 * W][4];   // rows 2 t, 2 t + 1 of every block: reference (a power of 2), sums
        float ones[NT][4];                       // sums of y: of group g, rows 2 t, 2 t + 1
        f32x2 middles[NT][NP];                   // sums of p (zero + M step) over this lane's keys: of a row two groups to a word, one after the other (one group: the two rows)
        uint32_t limits[(NG + 1) / 2];           // the highest steps, as bits, that need no look at the norms; two groups in a word
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const float *sums = query_sums + x * (W + 1) * 8;
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(queries + ((part * NT * W + x * W + w) * 32 + lane) * 4);
                    q[part][x][w][0][0] = v.x; q[part][x][w][0][1] = v.y;
                    q[part][x][w][1][0] = v.z; q[part][x][w][1][1] = v.w;
                }
            // a of row g in four bfloat16 parts, beside M times it, as the K of a product has room for them: four lanes' pairs, twice.  One group: a part to a
            // lane.  Two: a group and part to a lane, twice.  More: a group to a lane, and two parts in a word where M is not wanted, else two products.
            float own = 0.f, a[4];
            if (NG > 1) own = (t & (NG == 2 ? 1 : 3)) < NG ? sums[(NG == 2 ? t & 1 : t) * 8 + g] : 0.f;
            else
#pragma unroll
                for (int w = 0; w < W; ++w) own += sums[w * 8 + g];
#pragma unroll
            for (int part = 0; part < 4; ++part) {
                a[part] = __uint_as_float(Narrow<__nv_bfloat16>::pack(0.f, own) & 0xffff0000u);
                own -= a[part];
            }
            auto word = [&](float part) { return Narrow<__nv_bfloat16>::pack(SMALL ? part * MIDDLE : 0.f, part); };
            if constexpr (NG == 1) {
                qz[x][0][0] = word(t == 0 ? a[0] : t == 1 ? a[1] : t == 2 ? a[2] : a[3]);
                qz[x][0][1] = 0;
            } else if constexpr (NG == 2) {
                qz[x][0][0] = word(t < 2 ? a[0] : a[1]);
                qz[x][0][1] = word(t < 2 ? a[2] : a[3]);
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (ZEROS == 1) qz[x][0][k] = Narrow<__nv_bfloat16>::pack(a[2 * k], a[2 * k + 1]);
                    else {
                        qz[x][k][0] = word(a[2 * k]);
                        qz[x][k][1] = word(a[2 * k + 1]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 2 * t + e;
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    float a = 0.f;
                    if (NG > 1) a = sums[k * 8 + row];
                    else
#pragma unroll
                        for (int w = 0; w < W; ++w) a += sums[w * 8 + row];
                    start[x][k][e] = start[x][k][2 + e] = SMALL && !WIDE ? -MIDDLE * a : 0.f;
                }
                factor[x][e] = sums[W * 8 + row];
                int lo, hi;
                sees(x, e, lo, hi);
                all_lo = max(all_lo, lo);
                all_hi = min(all_hi, hi);
                m[x][e] = -INFINITY;
                l[x][e] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < 2 * W; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) ones[x][e] = 0.f;
#pragma unroll
            for (int k = 0; k < NP; ++k) middles[x][k] = 0;
        }
#pragma unroll
        for (int k = 0; k < (NG + 1) / 2; ++k) limits[k] = 0xffffffffu;
        for (int k = lane; k < NT * 8 * NP; k += 32) norms[k] = power_of_two(127 + kFewHighest);
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);
        uint32_t st = slot;
        for (int u = 0; u < stages; ++u, ++used) {
            st = slot;
            if (ok && !(ok = __all_sync(0xffffffffu, wait_or_abort(&full[st], phase, abort_flag)))) give_up(2);
            if (++slot == L::kStages) {
                slot = 0;
                phase ^= 1;
            }
            const int j0 = S.begin + (stage0 + u) * KEYS + L::OWN * warp;
            if (ok && j0 < S.end && j0 + 16 * SUB > S.first) {
                const unsigned char *k_at = smem + st * L::STAGE + L::OWN * warp * L::ROW, *v_at = k_at + L::CODES;
                const unsigned char *ks_at = smem + st * L::STAGE + 2 * L::CODES + L::OWN * warp * NG * 4, *vs_at = ks_at + L::SCALES;
                float p[SUB][NT][4];
#pragma unroll
                for (int h = 0; h < SUB; ++h) {
                    uint32_t kw[2][W * BITS / 4], ks[2][NG], kz[2];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int key = 16 * h + 8 * s + slot0;
                        load_words(kw[s], k_at + key * L::ROW + t * (W * BITS));
                        load_words(ks[s], ks_at + key * NG * 4);
                        kz[s] = reinterpret_cast<const uint32_t *>(ks_at)[key * NG + (NG == 1 ? 0 : NG == 2 ? t & 1 : t < NG ? t : 0)];
                        if (NG == 3 && t == 3) kz[s] = 0;
                        if (NG > 2 && ZEROS == 1) kz[s] = __byte_perm(kz[s], kz[s], 0x3232);   // the zero twice
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        mma_bf16_new(p[h][x], kz[0], kz[1], kz[0], kz[1], qz[x][0][0], qz[x][0][1]);
                        if constexpr (ZEROS == 2) mma_bf16(p[h][x], kz[0], kz[1], kz[0], kz[1], qz[x][1][0], qz[x][1][1]);
                    }
                    float acc[NT][4];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t a[4];
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                if constexpr (BITS == 4) {
                                    const uint32_t c = kw[s][w] >> (8 * k);
                                    a[s] = c & 0x000f000fu;
                                    a[2 + s] = c & 0x00f000f0u;
                                } else {
                                    const uint32_t c = kw[s][2 * w + k];
                                    a[s] = c & 0x00ff00ffu;
                                    a[2 + s] = (c >> 8) & 0x00ff00ffu;
                                }
                                if constexpr (WIDE) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e) a[2 * e + s] = numbers_of<BITS>(a[2 * e + s], e);
                                }
                            }
#pragma unroll
                            for (int x = 0; x < NT; ++x)
#pragma unroll
                                for (int part = 0; part < PARTS; ++part) {
                                    if (k == 0 && part == 0 && (NG > 1 || w == 0))
                                        mma_f16_from(acc[x], start[x][NG > 1 ? w : 0], a[0], a[1], a[2], a[3], q[part][x][w][k][0], q[part][x][w][k][1]);
                                    else mma_f16(acc[x], a[0], a[1], a[2], a[3], q[part][x][w][k][0], q[part][x][w][k][1]);
                                }
                        }
                        if (NG > 1 || w == W - 1)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const float step = step_of(ks[s][NG > 1 ? w : 0]);
#pragma unroll
                                for (int x = 0; x < NT; ++x)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) p[h][x][2 * s + e] = fmaf(step, acc[x][2 * s + e], p[h][x][2 * s + e]);
                            }
                    }
                }
                // steps and zeros of values, a lane to a key
                uint32_t vs[NG];
                load_words(vs, vs_at + (lane % (16 * SUB)) * NG * 4);
                // keys that some row does not see; steps and zeros of those that none sees need not be numbers
                if (j0 < all_lo || j0 + 16 * SUB > all_hi) {
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            int lo, hi;
                            sees(x, e, lo, hi);
#pragma unroll
                            for (int h = 0; h < SUB; ++h)
#pragma unroll
                                for (int s = 0; s < 2; ++s) {
                                    const int j = j0 + 16 * h + 8 * s + slot0;
                                    if (j < lo || j >= hi || j >= S.end) p[h][x][2 * s + e] = -INFINITY;
                                }
                        }
                    const int j = j0 + lane % (16 * SUB);
                    if (j < S.first || j >= S.end)
#pragma unroll
                        for (int k = 0; k < NG; ++k) vs[k] = 0;
                }
                // References move, norms are looked at and sums are scaled, only where a score has left its reference behind or a step what norms allow
                bool loud = false, moves = false;
#pragma unroll
                for (int k = 0; k < (NG + 1) / 2; ++k) {
                    const uint32_t steps = __byte_perm(vs[2 * k], 2 * k + 1 < NG ? vs[2 * k + 1 < NG ? 2 * k + 1 : 0] : 0u, 0x5410);
                    loud = loud || max_halves(steps, limits[k]) != limits[k];
                }
                float high[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        high[x][e] = fmaxf(p[0][x][e], p[0][x][2 + e]);
                        if constexpr (SUB == 2) high[x][e] = fmaxf(high[x][e], fmaxf(p[1][x][e], p[1][x][2 + e]));
                        high[x][e] *= factor[x][e];
                        moves = moves || high[x][e] > m[x][e] + kFewSlack;
                    }
                moves = __any_sync(0xffffffffu, moves || loud);
                float up[NT][2];   // of references
                if (moves) {
                    loud = __any_sync(0xffffffffu, loud);
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = high[x][e];
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            float now = fmaxf(top, m[x][e]);
                            // Steps are large beside what norms allow, which reckon with scores like the highest.  Where one token takes the weight and has small
                            // values all others would be: the reference comes down to these keys' scores, so far that the sum of probabilities stays below about 2^24.
                            if (loud) {   // (of the whole warp: so are the exchanges)
                                float sum = l[x][e];
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1) sum = fmaxf(sum, __shfl_xor_sync(0xffffffffu, sum, d));
                                const int room = 24 + 127 - (int)(__float_as_uint(sum) >> 23);
                                if (top > -INFINITY) now = fmaxf(top, m[x][e] - (room < 0 ? 0.f : room > 24 ? 24.f : (float)room));
                            }
                            up[x][e] = now == m[x][e] ? 0.f : now - m[x][e];
                            m[x][e] = now;
                            l[x][e] *= exp2_fast(-up[x][e]);
                        }
                }
                __syncwarp();   // what the last keys left is read
                if (lane < 16 * SUB) {
                    float *to = prepared + ((lane >> 4) * 32 + slot_of_key(lane & 15)) * NP;
                    alignas(16) float step[NP] = {}, middle[NP] = {};
#pragma unroll
                    for (int k = 0; k < NG; ++k) {
                        step[k] = step_of(vs[k]);
                        middle[k] = fmaf(step[k], MIDDLE, zero_of(vs[k]));
                    }
                    store_words(to, step);
                    store_words(to + 16 * NP, middle);
                }
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float shift = m[x][e] == -INFINITY ? 0.f : -m[x][e];
#pragma unroll
                        for (int h = 0; h < SUB; ++h)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                p[h][x][2 * s + e] = exp2_fast(fmaf(p[h][x][2 * s + e], factor[x][e], shift));
                                l[x][e] += p[h][x][2 * s + e];
                            }
                    }
                __syncwarp();
                if (moves) {
                    uint32_t allowed[NG];
#pragma unroll
                    for (int k = 0; k < NG; ++k) allowed[k] = 0xffff;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        float top[2][NG] = {}, *norm = norms + (8 * x + 2 * t) * NP;
                        int was[2][NG];
#pragma unroll
                        for (int h = 0; h < SUB; ++h)
#pragma unroll
                            for (int s = 0; s < 2; ++s)
#pragma unroll
                                for (int k = 0; k < NG; ++k) {
                                    const float step = prepared[(h * 32 + g + 8 * s) * NP + k];
#pragma unroll
                                    for (int e = 0; e < 2; ++e) top[e][k] = fmaxf(top[e][k], fabsf(p[h][x][2 * s + e] * step));
                                }
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int k = 0; k < NG; ++k) was[e][k] = (int)(__float_as_uint(norm[e * NP + k]) >> 23) - 127;
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int k = 0; k < NG; ++k) top[e][k] = fmaxf(top[e][k], __shfl_xor_sync(0xffffffffu, top[e][k], d));
                        __syncwarp();   // norms are read
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float by = exp2_fast(-up[x][e]);
                            if constexpr (NP == 1) middles[x][0] = mul2(middles[x][0], e ? pack2(1.f, by) : pack2(by, 1.f));
                            else {
#pragma unroll
                                for (int k = 0; k < NP / 2; ++k) middles[x][e * (NP / 2) + k] = mul2(middles[x][e * (NP / 2) + k], pack2(by, by));
                            }
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                // up or down with the reference; down so far that the largest y of these keys is below 8
                                const int high = min(was[e][k] + (int)floorf(fminf(up[x][e], 1024.f)), kFewHighest), now = max(min(high, 129 - (int)(__float_as_uint(top[e][k]) >> 23)), -kFewHighest);
                                if (g == 0) norm[e * NP + k] = power_of_two(127 + now);
                                // steps below 2^6 over the norm: y stays below 2^14, and twice that where scores near 2^24 are a unit off
                                if (m[x][e] > -INFINITY) allowed[k] = min(allowed[k], (uint32_t)((133 - now) << 7) - 1);
                                const float scale = by * power_of_two(127 + now - was[e][k]);
                                if (g == k) ones[x][e] *= scale;
#pragma unroll
                                for (int n = 0; n < 2 * W; ++n)
                                    if (NG == 1 || n / 2 == k) {
                                        o[x][n][e] *= scale;
                                        o[x][n][2 + e] *= scale;
                                    }
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < NG; ++k) allowed[k] = __reduce_min_sync(0xffffffffu, allowed[k]);
#pragma unroll
                    for (int k = 0; k < (NG + 1) / 2; ++k) limits[k] = allowed[2 * k] | (2 * k + 1 < NG ? allowed[2 * k + 1 < NG ? 2 * k + 1 : 0] : 0xffffu) << 16;
                    __syncwarp();
                }
                f32x2 norm[NT][NP];   // laid out as the middles
#pragma unroll
                for (int x = 0; x < NT; ++x) load_pairs(norm[x], norms + (8 * x + 2 * t) * NP);
#pragma unroll
                for (int h = 0; h < SUB; ++h) {
                    constexpr int UNITS = BITS == 4 ? 2 * W : 4 * W;   // bytes of a lane's codes of a value
                    uint32_t vw[4][(UNITS + 3) / 4];                   // of slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const unsigned char *at = v_at + (16 * h + 8 * (s >> 1) + ((s & 1) ? value1 : value0)) * L::ROW + g * UNITS;
                        if constexpr (UNITS % 4 == 0) load_words(vw[s], at);
                        else {
                            vw[s][0] = *reinterpret_cast<const uint16_t *>(at) | (uint32_t)*reinterpret_cast<const uint16_t *>(at + 2) << 16;
                            vw[s][1] = *reinterpret_cast<const uint16_t *>(at + 4);
                        }
                    }
                    // y as operands, slots 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 of row g, of every group: rounded, and what that left
                    uint32_t y[NG][PARTS][NT][2];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const float *steps = prepared + (h * 32 + g + 8 * s) * NP;
                        auto narrow = [&](int k, int x, float y0, float y1) {
                            y[k][0][x][s] = transposed(half2_of(y0, y1));
                            if constexpr (WIDE) y[k][1][x][s] = transposed(half2_rest(y0, y1));
                        };
                        if constexpr (NP == 1) {
                            const f32x2 step = pack2(steps[0], steps[0]), middle = pack2(steps[16], steps[16]);
#pragma unroll
                            for (int x = 0; x < NT; ++x) {
                                const f32x2 both = pack2(p[h][x][2 * s], p[h][x][2 * s + 1]);
                                middles[x][0] = fma2(both, middle, middles[x][0]);
                                float y0, y1;
                                unpack2(mul2(mul2(both, norm[x][0]), step), y0, y1);
                                narrow(0, x, y0, y1);
                            }
                        } else {
                            f32x2 step[NP / 2], middle[NP / 2];
                            load_pairs(step, steps);
                            load_pairs(middle, steps + 16 * NP);
#pragma unroll
                            for (int x = 0; x < NT; ++x) {
                                const f32x2 p0 = pack2(p[h][x][2 * s], p[h][x][2 * s]), p1 = pack2(p[h][x][2 * s + 1], p[h][x][2 * s + 1]);
#pragma unroll
                                for (int k = 0; k < NP / 2; ++k) {
                                    middles[x][k] = fma2(p0, middle[k], middles[x][k]);
                                    middles[x][NP / 2 + k] = fma2(p1, middle[k], middles[x][NP / 2 + k]);
                                    float a0, a1, b0, b1;
                                    unpack2(mul2(mul2(p0, norm[x][k]), step[k]), a0, a1);
                                    unpack2(mul2(mul2(p1, norm[x][NP / 2 + k]), step[k]), b0, b1);
                                    narrow(2 * k, x, a0, b0);
                                    if (2 * k + 1 < NG) narrow(2 * k + 1 < NG ? 2 * k + 1 : 0, x, a1, b1);
                                }
                            }
                        }
                    }
                    if constexpr (!WIDE) {
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const uint32_t one = g == k ? 0x3c003c00u : 0u;   // 1 in row k
#pragma unroll
                            for (int x = 0; x < NT; ++x) mma_f16(ones[x], one, 0u, one, 0u, y[k][0][x][0], y[k][0][x][1]);
                        }
                    }
#pragma unroll
                    for (int w = 0; w < W; ++w) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {   // features 32 w + 4 g + 2 k and one more
                            uint32_t a[4];
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                if constexpr (BITS == 4) {
                                    const uint32_t c = __byte_perm(vw[2 * s][w / 2], vw[2 * s + 1][w / 2], w % 2 ? 0x7632 : 0x5410) >> (8 * k);
                                    a[2 * s] = c & 0x000f000fu;
                                    a[2 * s + 1] = c & 0x00f000f0u;
                                } else {
                                    const uint32_t c = __byte_perm(vw[2 * s][w], vw[2 * s + 1][w], k ? 0x7632 : 0x5410);
                                    a[2 * s] = c & 0x00ff00ffu;
                                    a[2 * s + 1] = (c >> 8) & 0x00ff00ffu;
                                }
                                if constexpr (WIDE) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e) a[2 * s + e] = numbers_of<BITS>(a[2 * s + e], e);
                                }
                            }
#pragma unroll
                            for (int x = 0; x < NT; ++x) {
                                if constexpr (!WIDE) {
                                    mma_f16(o[x][2 * w + k], a[0], a[1], a[2], a[3], y[NG > 1 ? w : 0][0][x][0], y[NG > 1 ? w : 0][0][x][1]);
                                } else {
                                    float sum[4] = {};
#pragma unroll
                                    for (int part = 0; part < PARTS; ++part) mma_f16(sum, a[0], a[1], a[2], a[3], y[NG > 1 ? w : 0][part][x][0], y[NG > 1 ? w : 0][part][x][1]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[x][2 * w + k][e] += sum[e];
                                }
                            }
                        }
                    }
                }
            }
            // M sums of y leave the outputs every second stage, before sums that grow by M with every key have lost what even attention leaves of their differences
            if constexpr (!WIDE) {
                if (u % 2) {
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
#pragma unroll
                            for (int k = 0; k < NG; ++k) {
                                const float less = __shfl_sync(0xffffffffu, ones[x][e], 4 * k + t) * (MIDDLE * -5.9604644775390625e-8f);   // 2^-24, as codes
#pragma unroll
                                for (int n = 0; n < 2 * W; ++n)
                                    if (NG == 1 || n / 2 == k) {
                                        o[x][n][e] += less;
                                        o[x][n][2 + e] += BITS == 4 ? 16.f * less : less;
                                    }
                            }
                            ones[x][e] = 0.f;
                        }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            // A stage late, so that the other warps are done with what is filled anew.  The last stage's room is where the warps' outputs meet: it is
            // filled after that.
            if (warp == 0 && u + 1 < stages) fill(used + L::kStages);
        }
        // The warps' outputs meet, 8 rows at a time, each in the room of its last stage beside references and sums.  A thread weighs four features of a
        // row together.
        const uint32_t share_at = st * L::STAGE;
        float *share = reinterpret_cast<float *>(smem + share_at + warp * 8 * DP * 4);
        constexpr float UNIT = WIDE ? 1.f : 16777216.f, UNIT_UPPER = BITS == 4 && !WIDE ? 1048576.f : UNIT;   // codes as half-precision numbers
        const bool all = stages == S.count;
        const long long part = ((long long)blockIdx.x * 2 + (stage0 == 0 ? 1 : 0)) * ROWS;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], d);
                float back[NG], middle[NG];   // one over the norms; sums of p (zero + M step) less M sums of y
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    float lo, hi;
                    unpack2(middles[x][NP == 1 ? 0 : e * (NP / 2) + k / 2], lo, hi);
                    middle[k] = (NP == 1 ? e : k % 2) ? hi : lo;
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) middle[k] += __shfl_xor_sync(0xffffffffu, middle[k], d);
                    back[k] = power_of_two(254 - (int)(__float_as_uint(norms[(8 * x + 2 * t + e) * NP + k]) >> 23));
                }
                if constexpr (!WIDE) {
#pragma unroll
                    for (int k = 0; k < NG; ++k) middle[k] = fmaf(__shfl_sync(0xffffffffu, ones[x][e], 4 * k + t) * -MIDDLE, back[k], middle[k]);
                }
                const int row = 2 * t + e;
                if (row0 + 8 * x + row >= F.rows) continue;
                if (g == 0) stats[warp * 8 + row] = make_float2(m[x][e], l[x][e]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float z = middle[NG > 1 ? w : 0], by = back[NG > 1 ? w : 0];
                    float4 v;
                    v.x = fmaf(o[x][2 * w][e] * UNIT, by, z);
                    v.y = fmaf(o[x][2 * w][2 + e] * UNIT_UPPER, by, z);
                    v.z = fmaf(o[x][2 * w + 1][e] * UNIT, by, z);
                    v.w = fmaf(o[x][2 * w + 1][2 + e] * UNIT_UPPER, by, z);
                    *reinterpret_cast<float4 *>(share + row * DP + 32 * w + 4 * g) = v;
                }
            }
            __syncthreads();
            for (int at = threadIdx.x; at < 8 * DP / 4; at += kFewThreads) {
                const int row = at / (DP / 4), d = at % (DP / 4) * 4, r = row0 + 8 * x + row;
                if (r >= F.rows || !ok) break;
                float2 s[kFewWarps];
                float top = -INFINITY, sum = 0.f, v[4] = {};
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) {
                    s[w] = stats[w * 8 + row];
                    top = fmaxf(top, s[w].x);
                }
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) {
                    if (s[w].y == 0.f) continue;   // saw nothing; what stands beside it need not be a number
                    const float by = s[w].x == -INFINITY ? s[w].y : exp2_fast(s[w].x - top);   // a sum with no reference is NaN
                    const float4 z = *reinterpret_cast<const float4 *>(smem + share_at + ((w * 8 + row) * DP + d) * 4);
                    sum = fmaf(by, s[w].y, sum);
                    v[0] = fmaf(by, z.x, v[0]);
                    v[1] = fmaf(by, z.y, v[1]);
                    v[2] = fmaf(by, z.z, v[2]);
                    v[3] = fmaf(by, z.w, v[3]);
                }
                if (all) finish(F, b, hk, r, d, v, top, sum);
                else {
                    if (d == 0) F.part_stats[part + 8 * x + row] = make_float2(top, sum);
                    *reinterpret_cast<float4 *>(F.part_out + (part + 8 * x + row) * DP + d) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            fence_proxy_async_smem();   // read and written by threads before copies write there
            fill(used + L::kStages);
        }
        stage = 0;
        if (++item == items) {
            item = 0;
            do ++b;
            while (used < total && Stages<KEYS>(P, b).count == 0);
        }
    } while (used < total);
    if (threadIdx.x == 0 && *abort_flag)   // what was issued arrives before the CTA ends
        for (uint32_t u = first_of_last_uses(issued, L::kStages); u < (uint32_t)issued; ++u) mbar_wait_bounded(&full[u % L::kStages], parity_of_use(u, L::kStages));
}

// Items that several CTAs have parts of, and those that have no keys.  A lane has four features of a row, and four parts on their way at a time.  A CTA to an
// item, a warp to a row; where items are few and their parts many (gridDim.y rows) a CTA to a row, whose warps share the parts.
template <int BITS, int W, int NG, int NT, int PARTS> __global__ void __launch_bounds__(kFewThreads) cache_join_kernel(const CacheFewParams F, int shares) {
    typedef CacheFew<BITS, W, NG, NT, PARTS> L;
    const CacheAttnParams &P = F.a;
    constexpr int DP = 32 * W, ROWS = 8 * NT;
    __shared__ unsigned room[kFewWarps + 2];
    __shared__ float met[kFewWarps][6][32];
    const int items = (int)P.c.H * F.row_blocks, of = (int)(blockIdx.x / items), item = (int)(blockIdx.x % items), hk = item / F.row_blocks, row0 = item % F.row_blocks * ROWS;
    const int n = Stages<L::KEYS>(P, of).count, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 4 * lane;
    const Line line = line_of<L::KEYS>(F, 0, shares, of, room);
    const unsigned at = line.before + (unsigned)item * (n + kFewExtra) + kFewExtra;
    // the CTA that has a place of the line; where places are fewer than CTAs some have none
    auto owner = [&](unsigned place) { return (int)(((unsigned long long)(place + 1) * shares - 1) / line.total); };
    auto none = [&](int c) { return line.total < (unsigned)shares && line.start(c, shares) == line.start(c + 1, shares); };
    const int first = n > 0 ? owner(at) : 0, last = n > 0 ? owner(at + n - 1) : -1;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // of every CTA: what comes after this kernel comes after both
    if (first == last) return;   // written already
    // parts from, from + by, ... of a row: the highest reference, the weighed sums
    auto gather = [&](int row, int from, int by, float &top, float &sum, float (&v)[4]) {
        top = -INFINITY;
        sum = v[0] = v[1] = v[2] = v[3] = 0.f;
        for (int c0 = from; c0 <= last; c0 += 4 * by) {
            float2 s[4];
            float4 z[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = c0 + u * by;
                const bool has = c <= last && !none(c);
                const long long place = ((long long)c * 2 + (c == first ? 1 : 0)) * ROWS + row;
                s[u] = has ? F.part_stats[place] : make_float2(-INFINITY, 0.f);
                z[u] = has && d < DP ? *reinterpret_cast<const float4 *>(F.part_out + place * DP + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float now = top;
#pragma unroll
            for (int u = 0; u < 4; ++u) now = fmaxf(now, s[u].x);
            const float old = now == top ? 1.f : exp2_fast(top - now);
            sum *= old;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= old;
            top = now;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (s[u].y == 0.f) continue;
                const float w = s[u].x == -INFINITY ? s[u].y : exp2_fast(s[u].x - top);   // a sum with no reference is NaN
                sum = fmaf(w, s[u].y, sum);
                v[0] = fmaf(w, z[u].x, v[0]);
                v[1] = fmaf(w, z[u].y, v[1]);
                v[2] = fmaf(w, z[u].z, v[2]);
                v[3] = fmaf(w, z[u].w, v[3]);
            }
        }
    };
    float top, sum, v[4];
    if (gridDim.y == 1) {
        for (int row = warp; row < ROWS && row0 + row < F.rows; row += kFewWarps) {
            gather(row, first, 1, top, sum, v);
            if (d < P.c.D) finish(F, of, hk, row0 + row, d, v, top, sum);
        }
        return;
    }
    const int row = blockIdx.y;
    if (row0 + row >= F.rows) return;
    gather(row, first + warp, kFewWarps, top, sum, v);
    const float mine[6] = {v[0], v[1], v[2], v[3], top, sum};
#pragma unroll
    for (int k = 0; k < 6; ++k) met[warp][k][lane] = mine[k];
    __syncthreads();
    if (warp > 0 || d >= P.c.D) return;
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) all = fmaxf(all, met[w][4][lane]);
    sum = v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
        const float s = met[w][5][lane], t = met[w][4][lane];
        if (s == 0.f) continue;
        const float by = t == -INFINITY ? s : exp2_fast(t - all);
        sum = fmaf(by, s, sum);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(by, met[w][k][lane], v[k]);
    }
    finish(F, of, hk, row0 + row, d, v, all, sum);
}

template <int BITS, int W, int NG, int NT, int PARTS> int launch_few(CacheFewParams F, void *scratch, long long *bytes, cudaStream_t s) {
    typedef CacheFew<BITS, W, NG, NT, PARTS> L;
    const CacheAttnParams &P = F.a;
    F.row_blocks = (int)((F.rows + L::ROWS - 1) / L::ROWS);
    F.by_nq = divider(P.Nq);
    F.by_blocks = divider(F.row_blocks);
    const long long items = P.c.B * P.c.H * F.row_blocks, seen = P.window > 0 && P.window + P.Nq < P.c.capacity ? P.window + P.Nq : P.c.capacity;
    const long long longest = (seen + L::KEYS - 1) / L::KEYS, slots = (long long)L::PER_SM * sm_count();
    // A CTA for an item where none can have more than 512 keys, about what a second kernel costs.  Else shares of at least 256 keys.
    F.whole = longest * L::KEYS <= 512;
    const long long least = items * longest * L::KEYS / 256, ctas = F.whole ? items : least < slots ? least : slots;
    if (bytes) {
        *bytes = F.whole ? 0 : ctas * 2 * L::ROWS * (4 * L::DP + 8);
        return TPW_OK;
    }
    TPW_CHECK_ARG(items * (longest + kFewExtra) < (1LL << 31), "tpw_cache_attention: more than 2^31 stages of work");
    F.part_out = static_cast<float *>(scratch);
    F.part_stats = reinterpret_cast<float2 *>(F.part_out + (F.whole ? 0 : ctas * 2 * L::ROWS * L::DP));
    constexpr auto *kern = &cache_few_kernel<BITS, W, NG, NT, PARTS>;
    if (const int e = allow_shared_memory<kern>((int)L::ALLOC)) return e;
    // Either kernel is launched while the one before it still runs, and waits for that one's end where it first reads what others write.
    cudaLaunchAttribute overlap = {};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3(kFewThreads);
    config.dynamicSmemBytes = L::ALLOC;
    config.stream = s;
    config.attrs = &overlap;
    config.numAttrs = 1;
    TPW_CUDA_OK(cudaLaunchKernelEx(&config, kern, F));
    TPW_LAUNCH_OK("cache_few_kernel");
    if (F.whole) return TPW_OK;
    config.gridDim = dim3((unsigned)items, ctas > 4 * items ? (unsigned)(F.rows < (int)L::ROWS ? F.rows : L::ROWS) : 1);
    config.dynamicSmemBytes = 0;
    TPW_CUDA_OK(cudaLaunchKernelEx(&config, &cache_join_kernel<BITS, W, NG, NT, PARTS>, F, (int)ctas));
    TPW_LAUNCH_OK("cache_join_kernel");
    return TPW_OK;
}
template <int BITS, int W, int NG> int launch_rows(const CacheFewParams &F, void *scratch, long long *bytes, cudaStream_t s) {
    if (F.a.dtype == TPW_F32) return launch_few<BITS, W, NG, 1, 2>(F, scratch, bytes, s);
    // 16 rows at a time unpack the codes half as often, by 8 warps an SM instead of 12, and pay for a last block that is half empty.  Measured 8 / 16 at a time, bfloat16, us:
    // [8, 12345, 8, 128] through a window of 4096, 4 bits, groups of 32, 16 rows 30.7 / 30.2, 40 rows 55 / 65, 80 rows 97 / 96, 128 rows 147 / 140; one group 26 / 24, 46 / 51, 79 / 74,
    // 119 / 107; [2, 16384, 8, 128] 22 / 25, 37 / 41, 63 / 64, 91 / 92; [4, 8000, 8, 64] in 8 bits 19 / 17, 35 / 38, 59 / 53, 87 / 77; [1, 1000, 8, 128] 12 / 18, 13 / 18, 16 / 21, 18 / 22.
    return F.rows <= 80 ? launch_few<BITS, W, NG, 1, 1>(F, scratch, bytes, s) : launch_few<BITS, W, NG, 2, 1>(F, scratch, bytes, s);
}
// with `bytes` only says how much scratch the call wants
template <int BITS> int launch_width(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s) {
    CacheFewParams F = {};
    F.a = P;
    F.rows = (int)(P.group * P.Nq);
    const long long piece = P.dtype == TPW_F32 ? 4 : 8;
    F.q_vector = P.c.D % 8 == 0 && aligned16(P.q) && P.q_s[0] % piece == 0 && P.q_s[1] % piece == 0 && P.q_s[2] % piece == 0;
    const bool one = P.c.groups == 1;
    if (P.c.width == 2) return one ? launch_rows<BITS, 2, 1>(F, scratch, bytes, s) : launch_rows<BITS, 2, 2>(F, scratch, bytes, s);
    if (P.c.width == 3) return one ? launch_rows<BITS, 3, 1>(F, scratch, bytes, s) : launch_rows<BITS, 3, 3>(F, scratch, bytes, s);
    return one ? launch_rows<BITS, 4, 1>(F, scratch, bytes, s) : launch_rows<BITS, 4, 4>(F, scratch, bytes, s);
}

} // namespace
} // namespace tpw
