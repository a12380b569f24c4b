// Gradients of attention on the tensor cores (16-bit types, up to 128 features).
//
// p_ij = exp(s_ij - lse_i) is formed anew from the forward's lse; ds_ij = p_ij (dO_i . v_j - delta_i).
//   keys walk    (dk, dv): a CTA holds 128 keys of one key head and walks over the query tiles of every head that shares it.
//                S^T = K Q^T and dP^T = V dO^T, a key row per thread pair; dV += P^T dO, dK += dS^T Q with P^T and dS^T in tensor memory.
//   queries walk (dq): a CTA holds 128 queries of one head and walks over the key tiles.  S = Q K^T, dP = dO V^T, dQ += dS K.
// Every gradient element is summed by one CTA in a fixed order: no atomics, the same bits each time.  That costs S and dP twice, 7 products
// of 128 x 128 x D per pair of tiles where 5 would do with 32-bit atomics into dq, whose order changes results.
//
// Bound by the tensor cores: 4 products (2048 clocks at D = 128) in the keys walk, 3 (1536) in the queries walk, with 16384
// exponentials (1024 clocks of the special-function units) beside either.  The elementwise work of one half of an
// iteration runs while the tensor cores do the other half: the keys walk forms P^T(i) during dK(i-1) and dP(i), dS^T(i) during dV(i) and
// S(i+1); tensor memory is full (S, dP, dV, dK of 128 columns each), so it cannot look further ahead.  The queries walk has room for
// two dP and gives S back as soon as it is read, so its S and dP are always one tile ahead.
//
// Two warpgroups share a tile's 128 rows: each has half of the columns, and writes its half of P or dS over the columns it read.
//
// Measured with the row terms' kernel (attention_rows.cu), bfloat16 [2, 4096, 16/4, 128] 730 us = 940 TFLOP/s on the five products that are asked for, 1320 on the
// seven; causal [1, 4096, 32/8, 128] the tensor cores are busy 66 % of the time.  [2, 4096, 16, 64] 575 us.  Both walks in one launch; CTAs that take over further blocks, as in the
// forward, were slower (1520 -> 1575 us causal [1, 8192, 32/8, 128]): the accumulators leave no tensor memory to overlap two blocks in.
#include "attention_tc.cuh"

namespace tpw {
namespace {

struct BackwardParams {
    AttnParams a;
    float scale_log2, scale;
    int q_tiles;
    unsigned key_blocks;   // blocks of the keys walk, before those of the queries walk
};

// Half precision: probabilities are lifted by 2^12 and gradients of scores by another power of two (attention_rows.cu), both undone in
// the epilogue; the largest of either is then 2^12 and 2^15.  factor: of the query heads [h, h + heads) of key head hk.
template <typename T> struct Lift {
    static constexpr bool kNeeded = false;
    static __device__ __forceinline__ float factor(const AttnParams &, int, int, int, int) { return 1.f; }
};
template <> struct Lift<__half> {
    static constexpr bool kNeeded = true;
    static __device__ __forceinline__ float factor(const AttnParams &P, int b, int h, int heads, int hk) {
        const unsigned *rows = P.row_max + 2 * (b * P.Hq + h);
        unsigned top = 0, more = 0;
        for (int g = 0; g < heads; ++g) {
            top = max(top, rows[2 * g]);
            more = max(more, rows[2 * g + 1]);
        }
        const float most = 2.f * sqrtf(__uint_as_float(top)) * sqrtf(__uint_as_float(P.row_max[2 * P.B * P.Hq + b * P.Hk + hk])) + __uint_as_float(more);
        if (!(most > 0.f) || !(most < INFINITY)) return 1.f;
        const float e = floorf(3.f - log2f(most));
        return exp2f(e < -100.f ? -100.f : e > 100.f ? 100.f : e);
    }
};

// Shared memory of either walk: the CTA's own two tiles, then rings of walked tiles, each with its full and empty barriers.
template <int BLOCKS> struct KeysSmem {
    static constexpr int kStages = BLOCKS == 2 ? 2 : 4;                        // of queries and of gradients
    static constexpr uint32_t TILE_BYTES = BLOCKS * BLOCK_BYTES;
    static constexpr uint32_t OFF_Q = 2 * TILE_BYTES, OFF_G = OFF_Q + kStages * TILE_BYTES;
    static constexpr uint32_t OFF_ROWS = OFF_G + kStages * TILE_BYTES;         // lse, delta of a query tile per stage
    static constexpr uint32_t OFF_BAR = OFF_ROWS + kStages * 2 * TILE * 4;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + 8 * (4 * kStages + 7);
    static constexpr uint32_t ALLOC = OFF_TMEM + 16 + 1024;
    static_assert(ALLOC <= 232448, "exceeds the dynamic shared memory of one CTA");
};
template <int BLOCKS> struct QueriesSmem {
    // a V tile is free again once dP has read it, a K tile only after dQ
    static constexpr int kKeys = BLOCKS == 2 ? 3 : 4, kValues = BLOCKS == 2 ? 2 : 3;
    static constexpr uint32_t TILE_BYTES = BLOCKS * BLOCK_BYTES;
    static constexpr uint32_t OFF_K = 2 * TILE_BYTES, OFF_V = OFF_K + kKeys * TILE_BYTES;
    static constexpr uint32_t OFF_BAR = OFF_V + kValues * TILE_BYTES;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + 8 * (2 * (kKeys + kValues) + 9);
    static constexpr uint32_t ALLOC = OFF_TMEM + 16 + 1024;
    static_assert(ALLOC <= 232448, "exceeds the dynamic shared memory of one CTA");
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}

// 64 columns of a thread's row: ds = p (dp - delta) in place of p, times `lift`
template <bool LIFT>
__device__ __forceinline__ f32x2 score_gradient(f32x2 p, f32x2 dp, f32x2 minus_delta, f32x2 lift) {
    f32x2 d = add2(dp, minus_delta);
    if (LIFT) d = mul2(d, lift);
    return mul2(p, d);
}

// A warp's 32 rows of an accumulator to global memory, this warpgroup's half of the columns, through shared memory that is no longer in use.
// A lane whose row is not to `keep` (nothing is seen from there, or nobody sees it) writes zeros, although its sums are 0 times what need not be
// finite; rows from `valid` on are not there.
template <typename T, int BLOCKS>
__device__ __forceinline__ void store_half(T *rows, long long row_stride, uint32_t acc, unsigned char *smem, int warp, int lane, int half, float by, bool keep, int valid, int D) {
    const RowStage<4 * BLOCKS> stage = {reinterpret_cast<uint4 *>(smem) + warp * 128 * BLOCKS};
    const int first = half * 32 * BLOCKS;
#pragma unroll 1
    for (int g = 0; g < BLOCKS; ++g) {
        uint32_t o[32];
        tmem_ld32(acc + first + 32 * g, o);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = keep ? Narrow<T>::pack(__uint_as_float(o[8 * k + 2 * e]) * by, __uint_as_float(o[8 * k + 2 * e + 1]) * by) : 0u;
            stage.put(lane, 4 * g + k, w[0], w[1], w[2], w[3]);
        }
    }
    stage.store(reinterpret_cast<unsigned char *>(rows + first), row_stride * 2, lane, valid, (D - first) / 8);
}

template <typename T, int BLOCKS>
__device__ __forceinline__ void keys_walk(const CUtensorMap &map_q, const CUtensorMap &map_k, const CUtensorMap &map_v, const CUtensorMap &map_g,
                                   const BackwardParams &F, unsigned block) {
    typedef KeysSmem<BLOCKS> L;
    typedef Narrow<T> N;
    const AttnParams &P = F.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *g_full = q_full + L::kStages, *q_empty = g_full + L::kStages,
             *g_empty = q_empty + L::kStages, *kv_full = g_empty + L::kStages, *s_full = kv_full + 1, *dp_full = s_full + 1, *p_ready = dp_full + 1, *ds_ready = p_ready + 1,
             *acc_full = ds_ready + 1, *drained = acc_full + 1;
    uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(smem + L::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_TMEM + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned heads = (unsigned)(P.B * P.Hk);
    const int row0 = (int)(block / heads) * TILE;   // a causal call's first keys are seen by most queries
    const long long bh = block % heads;
    const int hk = (int)(bh % P.Hk), b = (int)(bh / P.Hk);
    const Seen see(P, b);
    const int last = (row0 + TILE < see.length ? row0 + TILE : see.length) - 1;
    const int i_lo = see.qlo(row0), i_hi = last < row0 ? 0 : see.qhi(last);
    const int begin = i_lo / TILE, per_head = i_hi > i_lo ? (i_hi + TILE - 1) / TILE - begin : 0;
    const int total = per_head * (int)P.group;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) { mbar_init(&q_full[i], 1); mbar_init(&g_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&g_empty[i], 1); }
        mbar_init(kv_full, 1);
        mbar_init(s_full, 1);
        mbar_init(dp_full, 1);
        mbar_init(p_ready, 8);
        mbar_init(ds_ready, 8);
        mbar_init(acc_full, 1);
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_descriptor(&map_q);
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
        tma_prefetch_descriptor(&map_g);
    }
    if (warp == 9) tmem_alloc(tmem_ptr, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (17 << 16) | site);
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag));
        if (!ok) give_up(site);
        return ok;
    };
    const uint32_t k_at = smem_u32(smem), v_at = k_at + L::TILE_BYTES, q_ring = smem_u32(smem + L::OFF_Q), g_ring = smem_u32(smem + L::OFF_G),
                   rows_at = smem_u32(smem + L::OFF_ROWS);
    const uint32_t S = tmem, DP = tmem + TILE, DV = tmem + 2 * TILE, DK = tmem + 3 * TILE;

    if (warp >= 8) registers_down();
    if (warp == 8) {
        if (lane == 0 && total > 0) {
            uint32_t issued_q = 0, issued_g = 0;
            mbar_expect_tx(kv_full, 2 * L::TILE_BYTES);
            load_tokens<BLOCKS>(k_at, &map_k, kv_full, row0, hk, b);
            load_tokens<BLOCKS>(v_at, &map_v, kv_full, row0, hk, b);
            auto load = [&](uint64_t *full, uint64_t *empty, uint32_t ring, const CUtensorMap *map, bool terms, uint32_t u, uint32_t &issued) {
                const uint32_t st = u % L::kStages;
                if (u >= L::kStages && !wait_or_abort(&empty[st], parity_of_use(u, L::kStages) ^ 1, abort_flag)) {
                    give_up(1);
                    return false;
                }
                const int h = hk * (int)P.group + u / per_head, i0 = (begin + u % per_head) * TILE;
                mbar_expect_tx(&full[st], L::TILE_BYTES + (terms ? 2 * TILE * 4 : 0));
                load_tokens<BLOCKS>(ring + st * L::TILE_BYTES, map, &full[st], i0, h, b);
                if (terms) {
                    const long long from = (b * P.Hq + h) * P.Nqp + i0;
                    bulk_load(rows_at + st * 2 * TILE * 4, static_cast<const float *>(P.row_lse) + from, TILE * 4, &full[st]);
                    bulk_load(rows_at + (2 * st + 1) * TILE * 4, static_cast<const float *>(P.row_delta) + from, TILE * 4, &full[st]);
                }
                issued = u + 1;
                return true;
            };
            // A gradient tile is free after dV, a query tile only after dK: the gradients are fetched first.  The row terms come with the queries: the
            // row warps read delta until they arrive at ds_ready, for which dK waits and dV does not.
            for (int u = 0; u < total; ++u)
                if (!load(g_full, g_empty, g_ring, &map_g, false, u, issued_g) || !load(q_full, q_empty, q_ring, &map_q, true, u, issued_q)) break;
            if (!wait_for_releases(q_empty, issued_q, L::kStages, abort_flag) || !wait_for_releases(g_empty, issued_g, L::kStages, abort_flag)) give_up(2);
            if (*abort_flag) {   // what was issued arrives before the CTA ends
                mbar_wait_bounded(kv_full, 0);
                for (uint32_t u = first_of_last_uses(issued_q, L::kStages); u < issued_q; ++u) mbar_wait_bounded(&q_full[u % L::kStages], parity_of_use(u, L::kStages));
                for (uint32_t u = first_of_last_uses(issued_g, L::kStages); u < issued_g; ++u) mbar_wait_bounded(&g_full[u % L::kStages], parity_of_use(u, L::kStages));
            }
        }
    } else if (warp == 9) {
        const int steps = (int)(P.D + 15) / 16;
        const uint32_t idesc_s = instruction(N::kFormat, TILE, false), idesc_d = instruction(N::kFormat, 16 * steps, true);
        const uint32_t leader = elect_lane();
        bool ok = total == 0 || warp_wait(kv_full, 0, 3);
        // S^T or dP^T of use u, once its tile has arrived
        auto first = [&](uint64_t *arrives, int u, uint32_t d, uint32_t own, uint32_t ring, uint64_t *done, int site) {
            const uint32_t st = u % L::kStages;
            if (!warp_wait(&arrives[st], parity_of_use(u, L::kStages), site)) return false;
            tc_fence_after();
            product_features<BLOCKS>(leader, d, own, ring + st * L::TILE_BYTES, idesc_s, steps);
            commit_by(leader, done);
            return true;
        };
        if (total > 0 && ok) ok = first(q_full, 0, S, k_at, q_ring, s_full, 4) && first(g_full, 0, DP, v_at, g_ring, dp_full, 5);
        for (int u = 0; u < total && ok; ++u) {
            const uint32_t st = u % L::kStages;
            if (!(ok = warp_wait(p_ready, u & 1, 6))) break;
            tc_fence_after();
            product_tokens(leader, DV, S, 64, g_ring + st * L::TILE_BYTES, idesc_d, u > 0);
            commit_by(leader, &g_empty[st]);
            if (u + 1 < total && !(ok = first(q_full, u + 1, S, k_at, q_ring, s_full, 4))) break;
            if (!(ok = warp_wait(ds_ready, u & 1, 7))) break;
            tc_fence_after();
            product_tokens(leader, DK, DP, 64, q_ring + st * L::TILE_BYTES, idesc_d, u > 0);
            commit_by(leader, &q_empty[st]);
            if (u + 1 < total && !(ok = first(g_full, u + 1, DP, v_at, g_ring, dp_full, 5))) break;
        }
        if (ok && total > 0) commit_by(leader, acc_full);
        __syncwarp();
    } else if (warp < 8) {
        // ---- 32 key rows and 64 query columns per warp ----
        // Loads of 16 lanes x 256 bits spread them like an mma accumulator: thread 4 g + t has rows g, g + 8, g + 16, g + 24 and of every
        // eight columns 2 t and 2 t + 1.  It needs 16 of the columns' lse and delta; with a row per thread it would be all 64, 16 bytes
        // at a time to every lane, 1300 shared-memory wavefronts per tile beside operands that the MMAs read at the full rate.
        registers_up();
        const int half = warp >> 2, g = lane >> 2, t = lane & 3;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, upper = 16u << 16;
        const uint32_t s_at = S + lanes + 64 * half, dp_at = DP + lanes + 64 * half;
        // query tiles from all_lo on, and below all_hi, are seen by every key of the tile; keys beyond the length are not stored
        const int all_lo = see.qlo(row0 + TILE - 1), all_hi = see.window ? row0 - see.off + see.window : 0x7fffffff;
        const float c = F.scale_log2, lift = Lift<T>::factor(P, b, hk * (int)P.group, (int)P.group, hk);
        const f32x2 c2 = pack2(c, c), lift2 = pack2(lift, lift);
        // index 2 i + r of a half's 16 pairs: columns 8 i + 2 t and the next, row g + 8 r (and 16 in the upper half)
        auto hide = [&](f32x2 (&p)[2][16], int i0) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int j = row0 + (warp & 3) * 32 + 16 * hh + 8 * r + g, lo = see.qlo(j), hi = see.window ? see.qhi(j) : 0x7fffffff;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = i0 + 64 * half + 8 * i + 2 * t;
                        float p0, p1;
                        unpack2(p[hh][2 * i + r], p0, p1);
                        p[hh][2 * i + r] = pack2(at >= lo && at < hi ? p0 : 0.f, at + 1 >= lo && at + 1 < hi ? p1 : 0.f);
                    }
                }
        };
        auto hand_over = [&](const f32x2 (&p)[2][16], uint32_t at, uint64_t *bar) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float p0, p1;
                    unpack2(p[hh][e], p0, p1);
                    w[e] = N::pack(p0, p1);
                }
                tmem_st_16x128(at + hh * upper, w);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        bool ok = true;
        for (int u = 0; u < total; ++u) {
            const uint32_t st = u % L::kStages;
            const float *rows = reinterpret_cast<const float *>(smem + L::OFF_ROWS + st * 2 * TILE * 4) + 64 * half + 2 * t;
            const int i0 = (begin + u % per_head) * TILE;
            if (!(ok = warp_wait(s_full, u & 1, 8) && warp_wait(&q_full[st], parity_of_use(u, L::kStages), 9))) break;
            tc_fence_after();
            uint32_t x[2][32];
            tmem_ld_16x256(s_at, x[0]);
            tmem_ld_16x256(s_at + upper, x[1]);
            tmem_ld_wait();
            const bool masked = i0 < all_lo || i0 + TILE > all_hi;
            f32x2 p[2][16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x2 minus_lse = *reinterpret_cast<const f32x2 *>(rows + 8 * i);
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t *pair = &x[hh][4 * i + 2 * r];
                        const f32x2 z = fma2(pack2(__uint_as_float(pair[0]), __uint_as_float(pair[1])), c2, minus_lse);
                        p[hh][2 * i + r] = 2 * hh + r == 1 ? exp2_polynomial(z) : exp2_pair(z);
                    }
            }
            if (masked) hide(p, i0);
            hand_over(p, s_at, p_ready);
            if (!(ok = warp_wait(dp_full, u & 1, 10))) break;
            tc_fence_after();
            tmem_ld_16x256(dp_at, x[0]);
            tmem_ld_16x256(dp_at + upper, x[1]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const f32x2 minus_delta = *reinterpret_cast<const f32x2 *>(rows + TILE + 8 * i);
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t *pair = &x[hh][4 * i + 2 * r];
                        p[hh][2 * i + r] = score_gradient<Lift<T>::kNeeded>(p[hh][2 * i + r], pack2(__uint_as_float(pair[0]), __uint_as_float(pair[1])),
                                                                           minus_delta, lift2);
                    }
            }
            if (masked) hide(p, i0);   // 0 times what need not be finite
            hand_over(p, dp_at, ds_ready);
        }
        if (ok && total > 0) {
            ok = warp_wait(acc_full, 0, 12);
            tc_fence_after();
        }
        if (ok) {
            const int row = row0 + (warp & 3) * 32, j = row + lane, valid = (int)P.Nk - row;
            const bool keep = total > 0 && see.qlo(j) < see.qhi(j);
            const long long to = ((b * P.Nk + row) * P.Hk + hk) * P.D;
            const float down = Lift<T>::kNeeded ? 0.000244140625f : 1.f;   // 2^-12
            store_half<T, BLOCKS>(static_cast<T *>(P.dv) + to, P.Hk * P.D, DV + lanes, smem, warp, lane, half, down, keep, valid, (int)P.D);
            store_half<T, BLOCKS>(static_cast<T *>(P.dk) + to, P.Hk * P.D, DK + lanes, smem, warp, lane, half, F.scale * down / lift, keep, valid, (int)P.D);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        if (*abort_flag) {   // the commits behind all MMAs were waited for, or one more is waited for here
            commit_by(elect_lane(), drained);   // of the lane that issued them
            mbar_wait_bounded(drained, 0);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int BLOCKS>
__device__ __forceinline__ void queries_walk(const CUtensorMap &map_q, const CUtensorMap &map_k, const CUtensorMap &map_v, const CUtensorMap &map_g,
                                   const BackwardParams &F, unsigned block) {
    typedef QueriesSmem<BLOCKS> L;
    typedef Narrow<T> N;
    const AttnParams &P = F.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *k_empty = k_full + L::kKeys, *v_full = k_empty + L::kKeys,
             *v_empty = v_full + L::kValues, *own_full = v_empty + L::kValues, *s_full = own_full + 1,
             *s_read = s_full + 1, *dp_full = s_read + 1, *ds_ready = dp_full + 2, *acc_full = ds_ready + 2, *drained = acc_full + 1;
    uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(smem + L::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_TMEM + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned heads = (unsigned)(P.B * P.Hq);
    const int row0 = (F.q_tiles - 1 - (int)(block / heads)) * TILE;   // a causal call's longest rows first
    const long long bh = block % heads;
    const int h = (int)(bh % P.Hq), b = (int)(bh / P.Hq), hk = h / (int)P.group;
    const Seen see(P, b);
    const int nq = (int)P.Nq, last = (row0 + TILE < nq ? row0 + TILE : nq) - 1;
    const int begin = see.lo(row0) / TILE, end = (see.hi(last) + TILE - 1) / TILE;
    const int total = end > begin ? end - begin : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kKeys; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < L::kValues; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        mbar_init(own_full, 1);
        mbar_init(s_full, 1);
        mbar_init(s_read, 8);
        mbar_init(&dp_full[0], 1);
        mbar_init(&dp_full[1], 1);
        mbar_init(&ds_ready[0], 8);
        mbar_init(&ds_ready[1], 8);
        mbar_init(acc_full, 1);
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_descriptor(&map_q);
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
        tma_prefetch_descriptor(&map_g);
    }
    if (warp == 9) tmem_alloc(tmem_ptr, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (18 << 16) | site);
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag));
        if (!ok) give_up(site);
        return ok;
    };
    const uint32_t q_at = smem_u32(smem), g_at = q_at + L::TILE_BYTES, keys = smem_u32(smem + L::OFF_K), values = smem_u32(smem + L::OFF_V);
    const uint32_t S = tmem, DP = tmem + TILE, DQ = tmem + 3 * TILE;

    if (warp >= 8) registers_down();
    if (warp == 8) {
        if (lane == 0 && total > 0) {
            uint32_t issued_k = 0, issued_v = 0;
            mbar_expect_tx(own_full, 2 * L::TILE_BYTES);
            load_tokens<BLOCKS>(q_at, &map_q, own_full, row0, h, b);
            load_tokens<BLOCKS>(g_at, &map_g, own_full, row0, h, b);
            for (int u = 0; u < total; ++u) {
                const uint32_t sk = u % L::kKeys, sv = u % L::kValues;
                if (u >= L::kKeys && !wait_or_abort(&k_empty[sk], parity_of_use(u, L::kKeys) ^ 1, abort_flag)) {
                    give_up(1);
                    break;
                }
                mbar_expect_tx(&k_full[sk], L::TILE_BYTES);
                load_tokens<BLOCKS>(keys + sk * L::TILE_BYTES, &map_k, &k_full[sk], (begin + u) * TILE, hk, b);
                issued_k = u + 1;
                if (u >= L::kValues && !wait_or_abort(&v_empty[sv], parity_of_use(u, L::kValues) ^ 1, abort_flag)) {
                    give_up(1);
                    break;
                }
                mbar_expect_tx(&v_full[sv], L::TILE_BYTES);
                load_tokens<BLOCKS>(values + sv * L::TILE_BYTES, &map_v, &v_full[sv], (begin + u) * TILE, hk, b);
                issued_v = u + 1;
            }
            if (!wait_for_releases(k_empty, issued_k, L::kKeys, abort_flag) || !wait_for_releases(v_empty, issued_v, L::kValues, abort_flag)) give_up(2);
            if (*abort_flag) {   // what was issued arrives before the CTA ends
                mbar_wait_bounded(own_full, 0);
                for (uint32_t u = first_of_last_uses(issued_k, L::kKeys); u < issued_k; ++u) mbar_wait_bounded(&k_full[u % L::kKeys], parity_of_use(u, L::kKeys));
                for (uint32_t u = first_of_last_uses(issued_v, L::kValues); u < issued_v; ++u) mbar_wait_bounded(&v_full[u % L::kValues], parity_of_use(u, L::kValues));
            }
        }
    } else if (warp == 9) {
        const int steps = (int)(P.D + 15) / 16;
        const uint32_t idesc_s = instruction(N::kFormat, TILE, false), idesc_d = instruction(N::kFormat, 16 * steps, true);
        const uint32_t leader = elect_lane();
        bool ok = total == 0 || warp_wait(own_full, 0, 3);
        auto first = [&](int u) {   // S and dP of key tile u
            const uint32_t sk = u % L::kKeys, sv = u % L::kValues;
            if (!warp_wait(&k_full[sk], parity_of_use(u, L::kKeys), 4)) return false;
            tc_fence_after();
            const int beyond = see.length - (begin + u) * TILE;
            if (beyond < TILE && (int)P.Nk > see.length) clear_tokens<BLOCKS>(smem + L::OFF_K + sk * L::TILE_BYTES, beyond, lane);
            product_features<BLOCKS>(leader, S, q_at, keys + sk * L::TILE_BYTES, idesc_s, steps);
            commit_by(leader, s_full);
            if (!warp_wait(&v_full[sv], parity_of_use(u, L::kValues), 10)) return false;
            tc_fence_after();
            product_features<BLOCKS>(leader, DP + (u & 1) * TILE, g_at, values + sv * L::TILE_BYTES, idesc_s, steps);
            commit_by(leader, &dp_full[u & 1]);
            commit_by(leader, &v_empty[sv]);
            return true;
        };
        if (total > 0 && ok) ok = first(0);
        for (int u = 0; u < total && ok; ++u) {
            if (u + 1 < total) {
                if (!(ok = warp_wait(s_read, u & 1, 5))) break;
                tc_fence_after();
                if (!(ok = first(u + 1))) break;
            }
            // S and dP of the next tile are already under way, so its gradients may be ready before this warp has seen that this tile's are: a barrier
            // each for even and odd tiles, or the wait would miss a phase and never end
            if (!(ok = warp_wait(&ds_ready[u & 1], (u >> 1) & 1, 6))) break;
            tc_fence_after();
            product_tokens(leader, DQ, DP + (u & 1) * TILE, 64, keys + (u % L::kKeys) * L::TILE_BYTES, idesc_d, u > 0);
            commit_by(leader, &k_empty[u % L::kKeys]);
        }
        if (ok && total > 0) commit_by(leader, acc_full);
        __syncwarp();
    } else if (warp < 8) {
        // ---- a query row and 64 key columns per thread ----
        registers_up();
        const int half = warp >> 2, i = row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int lo = see.lo(i), hi = i < nq ? see.hi(i) : 0;
        const int all_lo = see.lo(last), all_hi = see.hi(row0);   // seen by every query of the tile
        const float c = F.scale_log2, lift = Lift<T>::factor(P, b, h, 1, hk);
        const float lse = static_cast<const float *>(P.row_lse)[bh * P.Nqp + i], delta = static_cast<const float *>(P.row_delta)[bh * P.Nqp + i];
        const f32x2 c2 = pack2(c, c), lift2 = pack2(lift, lift), minus_lse = pack2(lse, lse), minus_delta = pack2(delta, delta);
        bool ok = true;
        for (int u = 0; u < total; ++u) {
            const int j0 = (begin + u) * TILE;
            const uint32_t s_at = S + lanes + 64 * half, dp_at = DP + (u & 1) * TILE + lanes + 64 * half;
            const bool masked = j0 < all_lo || j0 + TILE > all_hi;
            if (!(ok = warp_wait(s_full, u & 1, 7))) break;
            tc_fence_after();
            uint32_t x[2][32];
            tmem_ld32(s_at, x[0]);
            tmem_ld32(s_at + 32, x[1]);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_read);
            f32x2 p[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const uint32_t *pair = &x[e >> 4][2 * (e & 15)];
                const f32x2 z = fma2(pack2(__uint_as_float(pair[0]), __uint_as_float(pair[1])), c2, minus_lse);
                p[e] = e % 4 == 1 ? exp2_polynomial(z) : exp2_pair(z);
            }
            if (!(ok = warp_wait(&dp_full[u & 1], (u >> 1) & 1, 8))) break;
            tc_fence_after();
            tmem_ld32(dp_at, x[0]);
            tmem_ld32(dp_at + 32, x[1]);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const uint32_t *pair = &x[e >> 4][2 * (e & 15)];
                p[e] = score_gradient<Lift<T>::kNeeded>(p[e], pack2(__uint_as_float(pair[0]), __uint_as_float(pair[1])), minus_delta, lift2);
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const int j = j0 + 64 * half + 2 * e;
                    float d0, d1;
                    unpack2(p[e], d0, d1);
                    p[e] = pack2(j >= lo && j < hi ? d0 : 0.f, j + 1 >= lo && j + 1 < hi ? d1 : 0.f);
                }
            }
            uint32_t w[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                float d0, d1;
                unpack2(p[e], d0, d1);
                w[e] = N::pack(d0, d1);
            }
            tmem_st32(dp_at, w);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ds_ready[u & 1]);
        }
        if (ok && total > 0) {
            ok = warp_wait(acc_full, 0, 9);
            tc_fence_after();
        }
        if (ok) {
            const float down = Lift<T>::kNeeded ? 0.000244140625f : 1.f;   // 2^-12
            const int row = i - lane;
            T *rows = static_cast<T *>(P.dq) + ((b * P.Nq + row) * P.Hq + h) * P.D;
            store_half<T, BLOCKS>(rows, P.Hq * P.D, DQ + lanes, smem, warp, lane, half, F.scale * down / lift, total > 0 && lo < hi, nq - row, (int)P.D);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        if (*abort_flag) {
            commit_by(elect_lane(), drained);   // of the lane that issued them
            mbar_wait_bounded(drained, 0);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Both walks in one launch: the queries walk fills the SMs that the keys walk's last blocks leave, and a small problem is through in the time
// of the longer one.
template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_backward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ CUtensorMap map_g, const BackwardParams F) {
    if (blockIdx.x < F.key_blocks) keys_walk<T, BLOCKS>(map_q, map_k, map_v, map_g, F, blockIdx.x);
    else queries_walk<T, BLOCKS>(map_q, map_k, map_v, map_g, F, blockIdx.x - F.key_blocks);
}

template <typename T, int BLOCKS> int launch(const AttnParams &P, cudaStream_t s) {
    BackwardParams F = {};
    F.a = P;
    F.a.status = device_status_ptr();
    F.scale = (float)P.scale;
    F.scale_log2 = (float)(P.scale * 1.4426950408889634074);
    CUtensorMap q, k, v, g;
    int e = make_tensor_map_heads(&q, P.q, P.D, P.Nq, P.Hq, P.B, 2 * P.q_s[1], 2 * P.q_s[2], 2 * P.q_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&k, P.k, P.D, P.Nk, P.Hk, P.B, 2 * P.k_s[1], 2 * P.k_s[2], 2 * P.k_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&v, P.v, P.D, P.Nk, P.Hk, P.B, 2 * P.v_s[1], 2 * P.v_s[2], 2 * P.v_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&g, P.dout, P.D, P.Nq, P.Hq, P.B, 2 * P.do_s[1], 2 * P.do_s[2], 2 * P.do_s[0], TILE);
    if (e != TPW_OK) return e;
    F.q_tiles = (int)((P.Nq + TILE - 1) / TILE);
    const long long keys = P.dk ? (P.Nk + TILE - 1) / TILE * P.B * P.Hk : 0, queries = P.dq ? F.q_tiles * P.B * P.Hq : 0;
    TPW_CHECK_ARG(keys + queries < (1LL << 31), "attention: more than 2^31 blocks of work");
    F.key_blocks = (unsigned)keys;
    constexpr auto *kern = &attention_backward_kernel<T, BLOCKS>;
    constexpr uint32_t smem = KeysSmem<BLOCKS>::ALLOC > QueriesSmem<BLOCKS>::ALLOC ? KeysSmem<BLOCKS>::ALLOC : QueriesSmem<BLOCKS>::ALLOC;
    e = allow_shared_memory<kern>((int)smem);
    if (e != TPW_OK) return e;
    kern<<<(unsigned)(keys + queries), kTcThreads, smem, s>>>(q, k, v, g, F);
    TPW_LAUNCH_OK("attention_backward_kernel");
    return TPW_OK;
}

} // namespace

bool attn_tc_backward_fits(int dtype, const AttnParams &P) {
    if (!attn_tc_fits(dtype, P) || !aligned16(P.dout) || !aligned16(P.dq) || !aligned16(P.dk) || !aligned16(P.dv)) return false;
    for (int i = 0; i < 3; ++i)
        if (P.do_s[i] % 8 != 0 || P.do_s[i] <= 0 || P.do_s[i] >= (1LL << 38)) return false;
    return true;
}

int attn_tc_backward(int dtype, const AttnParams &P, cudaStream_t s) {
    if (dtype == TPW_F16) return P.D <= 64 ? launch<__half, 1>(P, s) : launch<__half, 2>(P, s);
    return P.D <= 64 ? launch<__nv_bfloat16, 1>(P, s) : launch<__nv_bfloat16, 2>(P, s);
}

} // namespace tpw
