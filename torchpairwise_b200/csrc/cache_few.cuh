// Attention of few query rows over a cache of quantised keys and values: one or a few new tokens against long sequences.
//
// Bound by HBM (4-bit codes with their steps and zeros: 160 bytes for a key and value of 128 features), closely followed by the instructions that unpack
// them.  So the codes go into the products as they are: as the low bits of half-precision numbers they are whole multiples of 2^-24,
// exactly, and masks are all the unpacking there is.
//   scores   K q^T, m16n8k16, 16 keys by 8 query rows: sum_g step_jg (sum_d c_jd q_d) + zero_jg (sum_d q_d).  A row of q is lifted by a
//            power of two to half precision's upper end; the sums begin at minus half the code range times sum_d q_d, so that they stay small.
//   output   V^T P^T, 16 features by 8 rows: the steps go into the probabilities, (p_j step_jg) c_jd, the zeros into a sum beside it.
// With keys along M a product has 8 rows of queries; rows along M would leave half of every product empty for up to 8 heads that share a key.
//
// Float32 queries: q and p step as two half-precision parts each, 22 bits; codes of values less half their range, and the products of 16 keys go
// to sums in registers, because tensor-core sums truncate.
//
// A CTA is a warp that issues bulk copies into a ring of 128-key stages, and four warps with 32 keys of a stage each and a running reference, sum
// and output of their own.  The CTAs of a cluster take equal shares of a sequence's keys, whatever its length, and join through
// distributed shared memory: no second launch, the same order every time.
#pragma once
#include "attention_tc.cuh"
#include "cache.cuh"

namespace tpw {
namespace {

constexpr int kCacheStage = 128;     // keys
constexpr int kCacheWarps = 4;       // that compute
constexpr int kCacheThreads = 32 * (kCacheWarps + 1);
constexpr int kLift = 6;             // probabilities times steps are lifted by 2^6 beside 2^8 that they may exceed their reference by: below 2^16,
constexpr float kSlack = 8.f;        // and normal half-precision numbers down to 2^-20 of it

struct CacheFewParams {
    CacheAttnParams a;
    int rows, row_blocks;            // group * Nq, and blocks of them
    int splits;                      // CTAs of a cluster
};

// NG: groups of a row; W: features / 32; NT: blocks of 8 query rows; PARTS: half-precision parts of queries and probabilities
template <int BITS, int W, int NG, int NT> struct CacheFewSmem {
    static constexpr uint32_t ROW = W * 4 * BITS, CODES = kCacheStage * ROW, SCALES = kCacheStage * NG * 4, STAGE = 2 * (CODES + SCALES);
    static constexpr int kStages = 106496 / STAGE < 6 ? 106496 / STAGE : 6;
    static constexpr uint32_t RING = kStages * STAGE, DP = 32 * W, ROWS = 8 * NT;
    // when the keys are done: the warps' shares and statistics, then the CTA's
    static constexpr uint32_t OFF_STATS = kCacheWarps * ROWS * DP * 4, OFF_RESULT = OFF_STATS + kCacheWarps * ROWS * 8, OFF_RESULT_STATS = OFF_RESULT + ROWS * DP * 4,
                              SHARES = OFF_RESULT_STATS + ROWS * 8;
    static constexpr uint32_t OFF_BAR = RING > SHARES ? RING : SHARES, OFF_FLAG = OFF_BAR + 16 * kStages, ALLOC = OFF_FLAG + 16;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) { return Narrow<__half>::pack(lo, hi); }
__device__ __forceinline__ uint32_t half2_rest(float lo, float hi) { return Narrow<__half>::rest(lo, hi); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
    float4 r;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(at) : "memory");
    return r;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t at) {
    float2 r;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(at) : "memory");
    return r;
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

// the n-th feature of a row of queries, in 32 bits
__device__ __forceinline__ float query(const CacheAttnParams &P, long long row, int n) {
    if (P.dtype == TPW_F32) return static_cast<const float *>(P.q)[row + n];
    if (P.dtype == TPW_F16) return __half2float(static_cast<const __half *>(P.q)[row + n]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(P.q)[row + n]);
}

// Of 16 keys, the one in slot s of a product (a row of K, a column of P).  In this order the rows that lanes of a quarter warp read lie in different
// banks for keys, and two by two for values.
__device__ __forceinline__ int key_of_slot(int s) {
    const int t = (s >> 1) & 3;
    return (s & 8) + ((s & 1) ? 4 + (t ^ 1) : t);
}

template <int BITS, int W, int NG, int NT, int PARTS>
__global__ void __launch_bounds__(kCacheThreads, 2) cache_few_kernel(const CacheFewParams F) {
    typedef CacheFewSmem<BITS, W, NG, NT> L;
    const CacheAttnParams &P = F.a;
    constexpr int DP = 32 * W, ROWS = 8 * NT;
    constexpr bool CENTRED = PARTS == 2;
    constexpr float MIDDLE = BITS == 4 ? 8.f : 128.f;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *empty = full + L::kStages;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_FLAG);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)(blockIdx.x % F.splits);
    const unsigned item = blockIdx.x / F.splits;
    const int block = (int)(item % F.row_blocks), bh = (int)(item / F.row_blocks), hk = (int)(bh % P.c.H), b = (int)(bh / P.c.H);
    const int nq = (int)P.Nq, row0 = block * ROWS;
    const CacheSeen see(P, b);
    // keys that any row sees, and this CTA's stages of them
    const int first = see.lo(0), end = see.hi(nq - 1), begin = first & ~63;
    const int all = end > first ? (end - begin + kCacheStage - 1) / kCacheStage : 0;
    const int u0 = (int)((long long)all * rank / F.splits), u1 = (int)((long long)all * (rank + 1) / F.splits), stages = u1 - u0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], kCacheWarps); }
        *abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (23 << 16) | site);
    };

    float m[NT][2], l[NT][2], o[NT][2 * W][4], zeros[NT][NG][2];   // of rows 2 t, 2 t + 1 of every block: reference (a power of 2), sums
    int top_step = 0;                                              // largest exponent of a step of a value so far, as in its bits
    if (warp == kCacheWarps) {
        if (lane == 0) {
            uint32_t issued = 0;
            const long long place0 = (long long)bh * P.c.capacity;
            for (int u = 0; u < stages; ++u) {
                const uint32_t st = u % L::kStages;
                if (u >= L::kStages && !wait_or_abort(&empty[st], parity_of_use(u, L::kStages) ^ 1, abort_flag)) {
                    give_up(1);
                    break;
                }
                // capacity and the stage's first key are multiples of 64
                const long long j = begin + (long long)(u0 + u) * kCacheStage;
                const uint32_t n = (uint32_t)(P.c.capacity - j < kCacheStage ? P.c.capacity - j : kCacheStage), to = smem_u32(smem) + st * L::STAGE;
                mbar_expect_tx(&full[st], n * 2 * (L::ROW + NG * 4));
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    bulk_load(to + w * L::CODES, P.c.codes[w] + (place0 + j) * L::ROW, n * L::ROW, &full[st]);
                    bulk_load(to + 2 * L::CODES + w * L::SCALES, P.c.scales[w] + (place0 + j) * NG, n * NG * 4, &full[st]);
                }
                issued = u + 1;
            }
            if (*abort_flag)   // what was issued arrives before the CTA ends
                for (uint32_t u = first_of_last_uses(issued, L::kStages); u < issued; ++u) mbar_wait_bounded(&full[u % L::kStages], parity_of_use(u, L::kStages));
        }
    } else {
        // Queries as operands: row g of a block, features 32 w + 8 t + (0 .. 7), in the order in which masks leave the codes of a key.  Row r is
        // query r % nq of head hk * group + r / nq.
        uint32_t q[PARTS][NT][W][2][2];
        float start[NT][NG][2], factor[NT][2];   // -MIDDLE 2^-24 sum_d q_d; scores of 2^: factor times the raw ones
        int lo[NT][2], hi[NT][2];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const int r = row0 + 8 * x + g;
            const bool valid = r < F.rows;
            const long long row = b * P.q_s[0] + (valid ? r % nq : 0) * P.q_s[1] + (hk * P.group + (valid ? r / nq : 0)) * P.q_s[2];
            auto feature = [&](int d) { return valid && d < P.c.D ? query(P, row, d) : 0.f; };
            float top = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int n = 0; n < 8; ++n) top = fmaxf(top, fabsf(feature(32 * w + 8 * t + n)));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // into [2^14, 2^15)
            int lift = 14 + 127 - (int)(__float_as_uint(top) >> 23);
            lift = top == 0.f ? 0 : lift > 100 ? 100 : lift < -100 ? -100 : lift;
            const float by = __uint_as_float((uint32_t)(127 + lift) << 23);
            float sums[NG] = {};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float y[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    y[n] = feature(32 * w + 8 * t + n) * by;
                    const float high = __half2float(__float2half_rn(y[n]));
                    sums[NG > 1 ? w : 0] += PARTS == 1 ? high : high + __half2float(__float2half_rn(y[n] - high));
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int n = BITS == 4 ? 2 * k + e : 4 * k + e;
                        const float s = BITS == 4 && e ? 0.0625f : 1.f, y0 = y[n], y1 = y[n + (BITS == 4 ? 4 : 2)];
                        q[0][x][w][k][e] = half2_of(y0 * s, y1 * s);
                        if constexpr (PARTS == 2) {
                            const float h0 = __half2float(__float2half_rn(y0)), h1 = __half2float(__float2half_rn(y1));
                            q[1][x][w][k][e] = half2_of((y0 - h0) * s, (y1 - h1) * s);
                        }
                    }
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], 1);
                sums[k] += __shfl_xor_sync(0xffffffffu, sums[k], 2);
            }
            const float f = P.scale_log2 * __uint_as_float((uint32_t)(127 + 24 - lift) << 23);
#pragma unroll
            for (int e = 0; e < 2; ++e) {   // of row 2 t + e, which lanes 4 (2 t + e) have
                const int from = 4 * (2 * t + e), mine = row0 + 8 * x + 2 * t + e;
#pragma unroll
                for (int k = 0; k < NG; ++k) start[x][k][e] = -MIDDLE * 5.9604644775390625e-8f * __shfl_sync(0xffffffffu, sums[k], from);
                factor[x][e] = fmaxf(__shfl_sync(0xffffffffu, f, from), 1.17549435e-38f);
                lo[x][e] = mine < F.rows ? see.lo(mine % nq) : 0;
                hi[x][e] = mine < F.rows ? see.hi(mine % nq) : 1 << 30;
                m[x][e] = -INFINITY;
                l[x][e] = 0.f;
#pragma unroll
                for (int k = 0; k < NG; ++k) zeros[x][k][e] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < 2 * W; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
        }
        float step_by = 0.f;   // 2^kLift over the power of two in top_step
        const int slot0 = key_of_slot(g), value0 = t, value1 = 4 + (t ^ 1);   // and 8 more
        for (int u = 0; u < stages; ++u) {
            const uint32_t st = u % L::kStages;
            const bool ok = __all_sync(0xffffffffu, wait_or_abort(&full[st], parity_of_use(u, L::kStages), abort_flag));
            if (!ok) {
                give_up(2);
                break;
            }
            const int j0 = begin + (u0 + u) * kCacheStage + 32 * warp;
            if (j0 < end && j0 + 32 > first) {
                const unsigned char *k_at = smem + st * L::STAGE + 32 * warp * L::ROW, *v_at = k_at + L::CODES;
                const unsigned char *ks_at = smem + st * L::STAGE + 2 * L::CODES + 32 * warp * NG * 4, *vs_at = ks_at + L::SCALES;
                float p[2][NT][4];
                uint32_t vs[2][2][NG];   // [16 keys][slots g, g + 8][group]
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t kw[2][W * BITS / 4], ks[2][NG];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int key = 16 * h + 8 * s + slot0;
                        load_words(kw[s], k_at + key * L::ROW + t * (W * BITS));
                        load_words(ks[s], ks_at + key * NG * 4);
                        load_words(vs[h][s], vs_at + key * NG * 4);
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[h][x][e] = 0.f;
                    float acc[NT][4];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if (NG > 1 || w == 0)
#pragma unroll
                            for (int x = 0; x < NT; ++x)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[x][e] = start[x][NG > 1 ? w : 0][e & 1];
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
                            }
#pragma unroll
                            for (int x = 0; x < NT; ++x)
#pragma unroll
                                for (int part = 0; part < PARTS; ++part) mma_f16(acc[x], a[0], a[1], a[2], a[3], q[part][x][w][k][0], q[part][x][w][k][1]);
                        }
                        if (NG > 1 || w == W - 1)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const uint32_t sc = ks[s][NG > 1 ? w : 0];
                                const float step = step_of(sc), shift = fmaf(zero_of(sc), -1.f / MIDDLE, -step);
#pragma unroll
                                for (int x = 0; x < NT; ++x)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        p[h][x][2 * s + e] = fmaf(shift, start[x][NG > 1 ? w : 0][e], fmaf(step, acc[x][2 * s + e], p[h][x][2 * s + e]));
                            }
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[h][x][e] *= factor[x][e & 1];
                }
                // keys that some row does not see; steps and zeros of those that none sees need not be numbers
                bool edge = j0 < first || j0 + 32 > end;
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) edge = edge || j0 < lo[x][e] || j0 + 32 > hi[x][e];
                if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const int j = j0 + 16 * h + 8 * s + slot0;
#pragma unroll
                            for (int x = 0; x < NT; ++x)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    if (j < lo[x][e] || j >= hi[x][e] || j >= end) p[h][x][2 * s + e] = -INFINITY;
#pragma unroll
                            for (int k = 0; k < NG; ++k)
                                if (j < first || j >= end) vs[h][s][k] = 0;
                        }
                }
                // the reference moves, and sums are scaled, only where a score or a step has left it behind
                int high_step = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int k = 0; k < NG; ++k) high_step = max(high_step, (int)(vs[h][s][k] & 0xffffu));
                bool moves = high_step >> 7 > top_step;
                float high[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        high[x][e] = fmaxf(fmaxf(p[0][x][e], p[0][x][2 + e]), fmaxf(p[1][x][e], p[1][x][2 + e]));
                        moves = moves || high[x][e] > m[x][e] + kSlack;
                    }
                if (__any_sync(0xffffffffu, moves)) {
                    const int now = max(__reduce_max_sync(0xffffffffu, high_step >> 7), top_step);
                    const float by_step = now > top_step && now - top_step < 127 ? __uint_as_float((uint32_t)(127 + top_step - now) << 23) : now > top_step ? 0.f : 1.f;
                    top_step = now;
                    step_by = __uint_as_float((uint32_t)(254 + kLift - (now > 7 ? now : 7)) << 23);
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = high[x][e];
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            top = fmaxf(top, m[x][e]);
                            const float by = top == m[x][e] ? 1.f : exp2_fast(m[x][e] - top);
                            m[x][e] = top;
                            l[x][e] *= by;
#pragma unroll
                            for (int k = 0; k < NG; ++k) zeros[x][k][e] *= by;
#pragma unroll
                            for (int n = 0; n < 2 * W; ++n) {
                                o[x][n][e] *= by * by_step;
                                o[x][n][2 + e] *= by * by_step;
                            }
                        }
                }
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float shift = m[x][e] == -INFINITY ? 0.f : m[x][e];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                p[h][x][2 * s + e] = exp2_fast(p[h][x][2 * s + e] - shift);
                                l[x][e] += p[h][x][2 * s + e];
                            }
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
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
                    uint32_t y[PARTS][NT][2];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if (NG > 1 || w == 0)
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const uint32_t sc = vs[h][s][NG > 1 ? w : 0];
                                const float step = step_of(sc) * step_by, zero = CENTRED ? fmaf(step_of(sc), MIDDLE, zero_of(sc)) : zero_of(sc);
#pragma unroll
                                for (int x = 0; x < NT; ++x) {
                                    const float p0 = p[h][x][2 * s], p1 = p[h][x][2 * s + 1];
                                    zeros[x][NG > 1 ? w : 0][0] = fmaf(p0, zero, zeros[x][NG > 1 ? w : 0][0]);
                                    zeros[x][NG > 1 ? w : 0][1] = fmaf(p1, zero, zeros[x][NG > 1 ? w : 0][1]);
                                    y[0][x][s] = transposed(half2_of(p0 * step, p1 * step));
                                    if constexpr (PARTS == 2) y[1][x][s] = transposed(half2_rest(p0 * step, p1 * step));
                                }
                            }
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
                                if constexpr (CENTRED)   // codes less the middle, as numbers
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const uint32_t c = a[2 * s + e] | 0x64006400u;   // 1024 + code, for the upper 4 bits 1024 + 16 code
                                        const __half2 v = *reinterpret_cast<const __half2 *>(&c);
                                        const __half2 r = BITS == 4 && e ? __hfma2(v, __float2half2_rn(0.0625f), __float2half2_rn(-64.f - MIDDLE)) : __hsub2(v, __float2half2_rn(1024.f + MIDDLE));
                                        a[2 * s + e] = *reinterpret_cast<const uint32_t *>(&r);
                                    }
                            }
#pragma unroll
                            for (int x = 0; x < NT; ++x) {
                                if constexpr (PARTS == 1) {
                                    mma_f16(o[x][2 * w + k], a[0], a[1], a[2], a[3], y[0][x][0], y[0][x][1]);
                                } else {
                                    float sum[4] = {};
#pragma unroll
                                    for (int part = 0; part < PARTS; ++part) mma_f16(sum, a[0], a[1], a[2], a[3], y[part][x][0], y[part][x][1]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[x][2 * w + k][e] += sum[e];
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
    }
    __syncthreads();
    // The warps' shares meet in the ring: [warp][row][feature] outputs, [warp][row] reference and sum
    const bool failed = *abort_flag != 0;
    float *share = reinterpret_cast<float *>(smem), *result = reinterpret_cast<float *>(smem + L::OFF_RESULT);
    float2 *stats = reinterpret_cast<float2 *>(smem + L::OFF_STATS), *result_stats = reinterpret_cast<float2 *>(smem + L::OFF_RESULT_STATS);
    if (warp < kCacheWarps) {
        const int power = (top_step > 7 ? top_step : 7) - 127 - kLift + (CENTRED ? 0 : 24);
        // as two factors: their exponents stay within 32 bits' range
        const float unit = ldexpf(1.f, power / 2), unit2 = ldexpf(1.f, power - power / 2), upper = BITS == 4 && !CENTRED ? 0.0625f : 1.f;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], d);
#pragma unroll
                    for (int k = 0; k < NG; ++k) zeros[x][k][e] += __shfl_xor_sync(0xffffffffu, zeros[x][k][e], d);
                }
                const int row = 8 * x + 2 * t + e;
                if (g == 0) stats[warp * ROWS + row] = make_float2(m[x][e], l[x][e]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float z = zeros[x][NG > 1 ? w : 0][e];
                    float4 v;
                    v.x = fmaf(o[x][2 * w][e] * unit, unit2, z);
                    v.y = fmaf(o[x][2 * w][2 + e] * unit, unit2 * upper, z);
                    v.z = fmaf(o[x][2 * w + 1][e] * unit, unit2, z);
                    v.w = fmaf(o[x][2 * w + 1][2 + e] * unit, unit2 * upper, z);
                    *reinterpret_cast<float4 *>(share + (warp * ROWS + row) * DP + 32 * w + 4 * g) = v;
                }
            }
    }
    __syncthreads();
    auto weight = [](float mine, float top) { return mine == -INFINITY ? 0.f : exp2_fast(mine - top); };   // NaN of a NaN
    for (int at = threadIdx.x; at < ROWS * DP / 4; at += kCacheThreads) {
        const int row = at / (DP / 4), d = at % (DP / 4) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kCacheWarps; ++w) top = fmaxf(top, stats[w * ROWS + row].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kCacheWarps; ++w) {
            const float2 s = stats[w * ROWS + row];
            if (s.y == 0.f) continue;   // saw nothing; what stands beside it need not be a number
            const float by = s.x == -INFINITY ? s.y : weight(s.x, top);   // a sum with no reference is NaN
            sum = fmaf(by, s.y, sum);
            const float4 z = *reinterpret_cast<const float4 *>(share + (w * ROWS + row) * DP + d);
            v.x = fmaf(by, z.x, v.x);
            v.y = fmaf(by, z.y, v.y);
            v.z = fmaf(by, z.z, v.z);
            v.w = fmaf(by, z.w, v.w);
        }
        *reinterpret_cast<float4 *>(result + row * DP + d) = v;
        if (d == 0) result_stats[row] = make_float2(top, sum);
    }
    if (F.splits > 1) cluster_sync();
    else __syncthreads();
    // the CTAs' results meet: a CTA finishes every splits-th row
    for (int at = threadIdx.x; at < ROWS * DP / 4; at += kCacheThreads) {
        const int row = at / (DP / 4), d = at % (DP / 4) * 4, r = row0 + row;
        if (row % F.splits != rank || r >= F.rows || d >= P.c.D || failed) continue;
        float top = -INFINITY, sum = 0.f;
        for (int s = 0; s < F.splits; ++s) top = fmaxf(top, ld_cluster2(cluster_addr(result_stats + row, s)).x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < F.splits; ++s) {
            const float2 z = ld_cluster2(cluster_addr(result_stats + row, s));
            if (z.y == 0.f) continue;
            const float by = z.x == -INFINITY ? z.y : weight(z.x, top);
            sum = fmaf(by, z.y, sum);
            const float4 y = ld_cluster4(cluster_addr(result + row * DP + d, s));
            v.x = fmaf(by, y.x, v.x);
            v.y = fmaf(by, y.y, v.y);
            v.z = fmaf(by, y.z, v.z);
            v.w = fmaf(by, y.w, v.w);
        }
        const int i = r % nq, h = (int)(hk * P.group) + r / nq, n = P.c.D - d;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float out[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
        const long long to = ((b * P.Nq + i) * P.Hq + h) * P.c.D + d;
        if (d == 0 && P.lse) P.lse[(b * P.Hq + h) * P.Nq + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
        if (P.dtype == TPW_F32) {
            float *dst = static_cast<float *>(P.out) + to;
            if (P.c.D % 4 == 0) *reinterpret_cast<float4 *>(dst) = make_float4(out[0], out[1], out[2], out[3]);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < n) dst[e] = out[e];
        } else {
            const uint32_t a = P.dtype == TPW_F16 ? half2_of(out[0], out[1]) : Narrow<__nv_bfloat16>::pack(out[0], out[1]);
            const uint32_t c = P.dtype == TPW_F16 ? half2_of(out[2], out[3]) : Narrow<__nv_bfloat16>::pack(out[2], out[3]);
            uint16_t *dst = static_cast<uint16_t *>(P.out) + to;
            if (P.c.D % 4 == 0) *reinterpret_cast<uint2 *>(dst) = make_uint2(a, c);
            else {
                const uint16_t e[4] = {(uint16_t)a, (uint16_t)(a >> 16), (uint16_t)c, (uint16_t)(c >> 16)};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < n) dst[k] = e[k];
            }
        }
    }
    if (F.splits > 1) cluster_sync();   // the others have read
}

template <int BITS, int W, int NG, int NT, int PARTS> int launch_few(const CacheFewParams &F, cudaStream_t s) {
    typedef CacheFewSmem<BITS, W, NG, NT> L;
    constexpr auto *kern = &cache_few_kernel<BITS, W, NG, NT, PARTS>;
    if (const int e = allow_shared_memory<kern>((int)L::ALLOC)) return e;
    const long long blocks = F.a.c.B * F.a.c.H * F.row_blocks * F.splits;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_cache_attention: more than 2^31 blocks of work");
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)blocks);
    config.blockDim = dim3(kCacheThreads);
    config.dynamicSmemBytes = L::ALLOC;
    config.stream = s;
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim = {(unsigned)F.splits, 1, 1};
    config.attrs = &cluster;
    config.numAttrs = F.splits > 1 ? 1 : 0;
    TPW_CUDA_OK(cudaLaunchKernelEx(&config, kern, F));
    TPW_LAUNCH_OK("cache_few_kernel");
    return TPW_OK;
}
template <int BITS, int W, int NG> int launch_rows(const CacheFewParams &F, cudaStream_t s) {
    if (F.a.dtype == TPW_F32) return launch_few<BITS, W, NG, 1, 2>(F, s);
    return F.rows <= 8 ? launch_few<BITS, W, NG, 1, 1>(F, s) : launch_few<BITS, W, NG, 2, 1>(F, s);
}
template <int BITS> int launch_width(const CacheFewParams &F, cudaStream_t s) {
    const bool one = F.a.c.groups == 1;
    if (F.a.c.width == 2) return one ? launch_rows<BITS, 2, 1>(F, s) : launch_rows<BITS, 2, 2>(F, s);
    if (F.a.c.width == 3) return one ? launch_rows<BITS, 3, 1>(F, s) : launch_rows<BITS, 3, 3>(F, s);
    return one ? launch_rows<BITS, 4, 1>(F, s) : launch_rows<BITS, 4, 4>(F, s);
}

} // namespace
} // namespace tpw
