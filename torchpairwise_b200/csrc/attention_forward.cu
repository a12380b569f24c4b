// Attention forward on the tensor cores (16-bit types, up to 128 features).
//
// out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i) in one pass over the keys with a running reference m_i of every row.
// A CTA works on 256 queries of one head as two tiles of 128, each with a warpgroup of its own whose thread t owns row t; one more
// warp issues TMA, one the MMAs.  Tensor memory holds, for each tile, the 128 x 128 scores and the output accumulators.  Per key tile: S = Q K^T
// (both operands in shared memory), the row's thread reads its 128 scores, forms the probabilities, and writes them, rounded to
// the inputs' type, over the scores; O += P V takes them from there.  While one tile's threads form probabilities the tensor cores work for the other.
//
// Bound: per pair of tiles 4 products of 128 x 128 x D, 2048 tensor-core clocks at D = 128, and 32768 exponentials, 2048 clocks of
// the four special-function units: both pipes would be full at once.
//
// The reference m_i is the first tile's maximum and moves only when a later score exceeds it by more than a factor 2^40 (the accumulators must
// then be read, scaled and written back): probabilities above 1 do no harm in fp32 sums and bfloat16.  So a tile's probabilities do not
// wait for its maximum, which is taken beside them; a tile that moves the reference forms them again.  Half precision ends at 2^16: there the
// factor is 2^8, and all are lifted by 2^6, so that they lose digits only below 2^-20 of the row's largest.
// O += P V starts when three quarters of P are there.
//
// Measured [2, 4096, 16/4, 128] bfloat16 256 us, 1070 TFLOP/s; 64 features 228 us, 600 TFLOP/s.  The tensor cores are busy 60 % of the time (64
// features: 33 %), the special-function units 59 % (66 %), so the bound is a row warp's own chain of steps: reading, 96 probabilities,
// handing over.  Tried and no faster: a quarter of the exponentials as polynomials on the FMA pipes (266 us), two warps to a row, which have to
// agree on its reference (300 us), probabilities beside the scores where 64 features leave room (229 us).
#include "attention_tc.cuh"

namespace tpw {
namespace {

struct ForwardParams {
    AttnParams a;
    float scale_log2;
    int tiles;                    // of 256 queries
    int splits, tiles_per_split;  // ranges of key tiles
    Divider by_splits, by_heads, by_hq, by_group;   // splits, B * Hq, Hq, Hq / Hk
    float *part_out, *part_lse;   // splits > 1
};

template <int BLOCKS> struct ForwardSmem {
    static constexpr int kSlots = BLOCKS == 2 ? 4 : 6;
    static constexpr uint32_t TILE_BYTES = BLOCKS * BLOCK_BYTES;
    static constexpr uint32_t OFF_RING = 2 * TILE_BYTES;
    static constexpr uint32_t OFF_STAGE = OFF_RING + kSlots * TILE_BYTES;   // 4 KB a warp: 32 rows of 64 features
    static constexpr uint32_t OFF_QUEUE = OFF_STAGE + 8 * 4096;
    static constexpr uint32_t OFF_BAR = OFF_QUEUE + 32;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + 8 * (2 * kSlots + 17);
    static constexpr uint32_t ALLOC = OFF_TMEM + 16 + 1024;
    static_assert(ALLOC <= 232448, "exceeds the dynamic shared memory of one CTA");
};

// One block of the grid: 256 queries of a head, a range of keys, and the key tiles [lo, hi) that either query tile sees
struct ForwardBlock {
    Seen see;
    int split, row0, h, b, hk, lo[2], hi[2], begin, end;
    // a causal call's longest rows first, all heads of them together
    __device__ __forceinline__ ForwardBlock(const ForwardParams &F, unsigned block) : ForwardBlock(F, block, block / F.by_splits) {}
    __device__ __forceinline__ ForwardBlock(const ForwardParams &F, unsigned block, unsigned item) : ForwardBlock(F, block - item * F.splits, item / F.by_heads, item % F.by_heads) {}
    __device__ __forceinline__ ForwardBlock(const ForwardParams &F, unsigned range, unsigned place, unsigned bh)
        : see(F.a, bh / F.by_hq), split((int)range), row0((F.tiles - 1 - (int)place) * 2 * TILE), h((int)(bh % F.by_hq)), b((int)(bh / F.by_hq)), hk((int)((unsigned)h / F.by_group)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int first = row0 + s * TILE, last = (first + TILE < see.nq ? first + TILE : see.nq) - 1;
            lo[s] = see.lo(first) / TILE;
            hi[s] = first < see.nq ? (see.hi(last) + TILE - 1) / TILE : 0;
            if (F.splits > 1) {
                const int from = split * F.tiles_per_split, to = from + F.tiles_per_split;
                lo[s] = lo[s] > from ? lo[s] : from;
                hi[s] = hi[s] < to ? hi[s] : to;
            }
            if (hi[s] <= lo[s]) lo[s] = hi[s] = 0;
        }
        const bool some0 = hi[0] > 0, some1 = hi[1] > 0;
        begin = some0 && (!some1 || lo[0] < lo[1]) ? lo[0] : lo[1];
        end = hi[0] > hi[1] ? hi[0] : hi[1];
    }
};

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_rest,
                         const ForwardParams F) {
    typedef ForwardSmem<BLOCKS> L;
    typedef Narrow<T> N;
    const AttnParams &P = F.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *empty = full + L::kSlots, *q_full = empty + L::kSlots, *q_empty = q_full + 1,
             *s_full = q_empty + 1, *p_most = s_full + 2, *p_full = p_most + 2, *o_full = p_full + 2, *o_empty = o_full + 2, *drained = o_empty + 2;
    const BlockQueue queue = {drained + 1, drained + 3, smem_u32(smem + L::OFF_QUEUE)};
    uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(smem + L::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_TMEM + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kSlots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(drained, 1);
        for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_most[s], 4); mbar_init(&p_full[s], 4); mbar_init(&o_full[s], 1); mbar_init(&o_empty[s], 4); }
        queue.init(10);   // the TMA lane, the MMA warp and eight warps of rows
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_descriptor(&map_q);
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
    }
    if (warp == 9) tmem_alloc(tmem_ptr, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (16 << 16) | site);
    };
    // a wait of a whole warp, with the same answer in every lane
    auto warp_wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag));
        if (!ok) give_up(site);
        return ok;
    };
    const uint32_t ring = smem_u32(smem + L::OFF_RING), q_at = smem_u32(smem);
    unsigned block = blockIdx.x;

    if (warp >= 8) registers_down();
    if (warp == 8) {
        if (lane == 0) {
            // uses of the ring (K and V tiles in turn) and of the query tiles by all blocks so far
            uint32_t used = 0, q_used = 0;
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
                ok = wait_or_abort(bar, parity, abort_flag);
                if (!ok) give_up(site);
                return ok;
            };
            for (uint32_t n = 0; ok; ++n) {
                const ForwardBlock W(F, block);
                if (W.end > W.begin) {
                    if (q_used > 0 && !wait(q_empty, (q_used & 1) ^ 1, 1)) break;
                    mbar_expect_tx(q_full, 2 * L::TILE_BYTES);
                    load_tokens<BLOCKS>(q_at, &map_q, q_full, W.row0, W.h, W.b);
                    load_tokens<BLOCKS>(q_at + L::TILE_BYTES, &map_q, q_full, W.row0 + TILE, W.h, W.b);
                    ++q_used;
                }
                for (int u = 0; u < 2 * (W.end - W.begin); ++u, ++used) {
                    const uint32_t slot = used % L::kSlots;
                    if (used >= L::kSlots && !wait(&empty[slot], parity_of_use(used, L::kSlots) ^ 1, 1)) break;
                    mbar_expect_tx(&full[slot], L::TILE_BYTES);
                    load_tokens<BLOCKS>(ring + slot * L::TILE_BYTES, u & 1 ? &map_v : &map_k, &full[slot], (W.begin + u / 2) * TILE, W.hk, W.b);
                }
                auto waits = [&](uint64_t *bar, uint32_t parity) { return wait(bar, parity, 11); };
                if (!ok || !queue.ask(n, waits) || !queue.next<false>(n, block, true, waits)) break;
            }
            // the commits that release the last uses have arrived before the CTA ends
            if (ok && (!wait_for_releases(empty, used, L::kSlots, abort_flag) || (q_used > 0 && !wait_or_abort(q_empty, (q_used & 1) ^ 1, abort_flag)))) give_up(2);
            if (*abort_flag) {   // what was issued arrives before the CTA ends
                if (q_used > 0) mbar_wait_bounded(q_full, (q_used & 1) ^ 1);
                for (uint32_t u = first_of_last_uses(used, L::kSlots); u < used; ++u) mbar_wait_bounded(&full[u % L::kSlots], parity_of_use(u, L::kSlots));
            }
        }
    } else if (warp == 9) {
        const int steps = (int)(P.D + 15) / 16;
        const uint32_t idesc_s = instruction(N::kFormat, TILE, false), idesc_o = instruction(N::kFormat, 16 * steps, true);
        const uint32_t leader = elect_lane();
        uint32_t used = 0, q_used = 0, done[2] = {0, 0}, finished[2] = {0, 0};   // products and blocks of either tile
        bool ok = true;
        auto arrived = [&](uint32_t u) {
            if (!warp_wait(&full[u % L::kSlots], parity_of_use(u, L::kSlots), 4)) return false;
            tc_fence_after();
            return true;
        };
        auto scores = [&](int s, uint32_t u) {
            product_features<BLOCKS>(leader, tmem + s * TILE, q_at + s * L::TILE_BYTES, ring + (u % L::kSlots) * L::TILE_BYTES, idesc_s, steps);
            commit_by(leader, &s_full[s]);
        };
        auto release = [&](uint32_t u) { commit_by(leader, &empty[u % L::kSlots]); };
        for (uint32_t n = 0; ok; ++n) {
            const ForwardBlock W(F, block);
            if (W.end > W.begin) {
                if (!(ok = warp_wait(q_full, q_used & 1, 3))) break;
                ++q_used;
                if (!(ok = arrived(used))) break;
                for (int s = 0; s < 2; ++s)
                    if (W.lo[s] <= W.begin && W.begin < W.hi[s]) scores(s, used);
                release(used);
                if (W.end == W.begin + 1) commit_by(leader, q_empty);
            }
            bool fresh[2] = {true, true};   // the output accumulators hold another block's sums
            for (int t = W.begin; t < W.end && ok; ++t, used += 2) {
                const uint32_t u = used + 1;   // of V; the next K is u + 1
                if (!(ok = arrived(u))) break;
                const int beyond = W.see.length - t * TILE;
                if (beyond < TILE && (int)P.Nk > W.see.length) clear_tokens<BLOCKS>(smem + L::OFF_RING + (u % L::kSlots) * L::TILE_BYTES, beyond, lane);
                if (t + 1 < W.end && !(ok = arrived(u + 1))) break;
                for (int s = 0; s < 2 && ok; ++s) {
                    if (W.lo[s] <= t && t < W.hi[s]) {
                        const uint32_t v_at = ring + (u % L::kSlots) * L::TILE_BYTES;
                        if (fresh[s] && finished[s] > 0 && !(ok = warp_wait(&o_empty[s], (finished[s] & 1) ^ 1, 12))) break;
                        if (!(ok = warp_wait(&p_most[s], done[s] & 1, 5))) break;
                        tc_fence_after();
                        product_tokens<0, 6>(leader, tmem + (2 + s) * TILE, tmem + s * TILE, 32, v_at, idesc_o, !fresh[s]);
                        if (!(ok = warp_wait(&p_full[s], done[s] & 1, 9))) break;
                        tc_fence_after();
                        product_tokens<6, 8>(leader, tmem + (2 + s) * TILE, tmem + s * TILE, 32, v_at, idesc_o, true);
                        commit_by(leader, &o_full[s]);
                        fresh[s] = false;
                        ++done[s];
                    }
                    if (W.lo[s] <= t + 1 && t + 1 < W.hi[s]) scores(s, u + 1);
                }
                if (!ok) break;
                release(u);
                if (t + 1 < W.end) release(u + 1);
                if (t + 2 == W.end) commit_by(leader, q_empty);
            }
            for (int s = 0; s < 2; ++s)
                if (W.hi[s] > W.lo[s]) ++finished[s];
            if (!ok || !queue.next<true>(n, block, lane == 0, [&](uint64_t *bar, uint32_t parity) { return ok = warp_wait(bar, parity, 11); })) break;
        }
        __syncwarp();
    } else if (warp < 8) {
        // ---- a query row per thread ----
        registers_up();
        const int s = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + s * TILE, o_at = tmem + lanes + (2 + s) * TILE;
        const RowBlock rows = {smem + L::OFF_STAGE + warp * 4096};
        const float c = F.scale_log2;
        const long long all_rows = P.B * P.Hq * P.Nq;
        uint32_t done = 0;   // scores of this tile by all blocks so far
        bool ok = true;
        for (uint32_t turn = 0; ok; ++turn) {
            int lo, hi, all_lo, all_hi, t_first, t_end;   // [lo, hi) of this row; [all_lo, all_hi) every row of the tile sees
            {
                const ForwardBlock W(F, block);
                const int first = W.row0 + s * TILE, last = (first + TILE < W.see.nq ? first + TILE : W.see.nq) - 1, i = first + (warp & 3) * 32 + lane;
                lo = W.see.lo(i);
                hi = i < W.see.nq ? W.see.hi(i) : 0;
                all_lo = W.see.lo(last);
                all_hi = W.see.hi(first);
                t_first = s ? W.lo[1] : W.lo[0];
                t_end = s ? W.hi[1] : W.hi[0];
            }
            float m = -INFINITY, l = 0.f;
            int n = 0;
#pragma unroll 1
            for (int t = t_first; t < t_end; ++t, ++n, ++done) {
                if (!(ok = warp_wait(&s_full[s], done & 1, 6))) break;
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int g = 0; g < 4; ++g) tmem_ld32(s_at + 32 * g, x[g]);
                tmem_ld_wait();
                const int j0 = t * TILE;
                if (j0 < all_lo || j0 + TILE > all_hi) {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int j = j0 + 32 * g + e;
                            if (j < lo || j >= hi) x[g][e] = 0xff800000u;
                        }
                }
                auto highest = [&]() {   // NaN for a score that is NaN or +inf: inf - inf makes the row NaN from there on
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
#pragma unroll
                        for (int g = 0; g < 4; ++g) tops[g] = max3_nan(tops[g], __uint_as_float(x[g][e]), __uint_as_float(x[g][e + 1]));
                    const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
                    return top < INFINITY ? top : NAN;
                };
                f32x2 sum, shift2;
                auto form = [&](int g) {   // 32 keys' probabilities
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const f32x2 z = fma2(pack2(__uint_as_float(x[g][2 * e]), __uint_as_float(x[g][2 * e + 1])), pack2(c, c), shift2);
                        const f32x2 y = exp2_pair(z);
                        sum = add2(sum, y);
                        float y0, y1;
                        unpack2(y, y0, y1);
                        p[e] = N::pack(y0, y1);
                    }
                    tmem_st16(s_at + 16 * g, p);
                };
                auto hand_over = [&](uint64_t *bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                if (n == 0) m = highest();
#pragma unroll 1
                for (int pass = 0;; ++pass) {
                    const float shift = m == -INFINITY ? 0.f : N::kLift - m * c;
                    shift2 = pack2(shift, shift);
                    sum = pack2(0.f, 0.f);
#pragma unroll
                    for (int g = 0; g < 3; ++g) form(g);
                    const float top = highest();
                    const bool moves = m == -INFINITY ? top != -INFINITY : !((top - m) * c <= N::kSlack);
                    if (pass > 0 || !__any_sync(0xffffffffu, moves)) break;
                    const bool scales = moves && m != -INFINITY;   // so far only zeros were added otherwise
                    const float by = scales ? exp2_fast((m - top) * c) : 1.f;
                    l *= by;
                    if (moves) m = top;
                    if (n == 0 || !__any_sync(0xffffffffu, scales)) continue;
                    if (!(ok = warp_wait(&o_full[s], (done & 1) ^ 1, 7))) break;
                    tc_fence_after();
                    for (int g = 0; g < 2 * BLOCKS; ++g) {
                        uint32_t o[32];
                        tmem_ld32(o_at + 32 * g, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                        tmem_st32(o_at + 32 * g, o);
                    }
                }
                if (!ok) break;
                // the first 96 keys' probabilities start the product while the last ones are formed
                hand_over(&p_most[s]);
                form(3);
                hand_over(&p_full[s]);
                float s0, s1;
                unpack2(sum, s0, s1);
                l += s0 + s1;
            }
            if (ok && n > 0) {
                ok = warp_wait(&o_full[s], (done & 1) ^ 1, 8);
                tc_fence_after();
            }
            if (!ok) break;
            const ForwardBlock W(F, block);
            const int nq = W.see.nq, i = W.row0 + s * TILE + (warp & 3) * 32 + lane;
            if (m == -INFINITY) l = 0.f;   // nothing seen
            const float by = l == 0.f ? 0.f : 1.f / l;
            const float lse = l == 0.f ? -INFINITY : (m * c - N::kLift + log2f(l)) * 0.69314718055994531f;
            const long long bh = W.b * P.Hq + W.h, flat = bh * P.Nq + i;
            if (i < nq && F.splits > 1) F.part_lse[W.split * all_rows + flat] = lse;
            else if (i < nq && P.lse) static_cast<float *>(P.lse)[flat] = lse;
            const bool empty = n == 0 || l == 0.f;
            const int row = i - lane;
            float *part = F.part_out + (W.split * all_rows + flat) * P.D;
#pragma unroll 1
            for (int g = 0; g < BLOCKS; ++g) {   // 64 features at a time
                uint32_t o[2][32];   // whatever lies there where nothing was seen
                tmem_ld32(o_at + 64 * g, o[0]);
                tmem_ld32(o_at + 64 * g + 32, o[1]);
                tmem_ld_wait();
                if (g == BLOCKS - 1 && n > 0) {   // the accumulators are read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[s]);
                }
                if (F.splits > 1) {   // nothing seen: the joining kernel does not look at it
#pragma unroll
                    for (int e = 0; e < 64; e += 4) {
                        float4 w;
                        w.x = empty ? 0.f : __uint_as_float(o[e >> 5][e & 31]) * by;
                        w.y = empty ? 0.f : __uint_as_float(o[e >> 5][(e & 31) + 1]) * by;
                        w.z = empty ? 0.f : __uint_as_float(o[e >> 5][(e & 31) + 2]) * by;
                        w.w = empty ? 0.f : __uint_as_float(o[e >> 5][(e & 31) + 3]) * by;
                        if (n > 0 && i < nq && 64 * g + e < (int)P.D) *reinterpret_cast<float4 *>(part + 64 * g + e) = w;
                    }
                    continue;
                }
#pragma unroll 1
                for (int what = 0; what < (P.rest ? 2 : 1); ++what) {   // the result, and what rounding took from it
                    RowBlock::reuse(lane);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t *pair = &o[k >> 2][8 * (k & 3) + 2 * e];
                            const float a0 = empty ? 0.f : __uint_as_float(pair[0]) * by, a1 = empty ? 0.f : __uint_as_float(pair[1]) * by;
                            w[e] = what ? N::rest(a0, a1) : N::pack(a0, a1);
                        }
                        rows.put(lane, k, w[0], w[1], w[2], w[3]);
                    }
                    if (row < nq) rows.send(lane, what ? &map_rest : &map_out, 64 * g, row, W.h, W.b);
                }
            }
            if (!queue.next<true>(turn, block, lane == 0, [&](uint64_t *bar, uint32_t parity) { return ok = warp_wait(bar, parity, 11); })) break;
        }
        RowBlock::reuse(lane);   // the copy engine has read the last block before the CTA ends
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        // all MMAs are over: the commits behind them were waited for, or, after a wait that gave up, one more is waited for here
        if (*abort_flag) {
            commit_by(elect_lane(), drained);   // of the lane that issued them
            mbar_wait_bounded(drained, 0);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int BLOCKS> int launch(const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    typedef ForwardSmem<BLOCKS> L;
    ForwardParams F = {};
    F.a = P;
    F.a.status = device_status_ptr();
    F.scale_log2 = (float)(P.scale * 1.4426950408889634074);
    F.tiles = (int)((P.Nq + 2 * TILE - 1) / (2 * TILE));
    F.splits = splits.count;
    F.tiles_per_split = splits.keys / TILE;
    F.part_out = splits.out;
    F.part_lse = splits.lse;
    F.by_splits = divider(F.splits);
    F.by_heads = divider(P.B * P.Hq);
    F.by_hq = divider(P.Hq);
    F.by_group = divider(P.group);
    CUtensorMap q, k, v, out, rest;
    int e = make_tensor_map_heads(&q, P.q, P.D, P.Nq, P.Hq, P.B, 2 * P.q_s[1], 2 * P.q_s[2], 2 * P.q_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&k, P.k, P.D, P.Nk, P.Hk, P.B, 2 * P.k_s[1], 2 * P.k_s[2], 2 * P.k_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&v, P.v, P.D, P.Nk, P.Hk, P.B, 2 * P.v_s[1], 2 * P.v_s[2], 2 * P.v_s[0], TILE);
    if (e == TPW_OK) e = make_tensor_map_heads(&out, P.out, P.D, P.Nq, P.Hq, P.B, 2 * P.Hq * P.D, 2 * P.D, 2 * P.Nq * P.Hq * P.D, 32);
    if (e != TPW_OK) return e;
    rest = out;
    if (P.rest) e = make_tensor_map_heads(&rest, P.rest, P.D, P.Nq, P.Hq, P.B, 2 * P.Hq * P.D, 2 * P.D, 2 * P.Nq * P.Hq * P.D, 32);
    if (e != TPW_OK) return e;
    const long long blocks = F.tiles * P.B * P.Hq * F.splits;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    constexpr auto *kern = &attention_forward_kernel<T, BLOCKS>;
    if (const int e = allow_shared_memory<kern>((int)L::ALLOC)) return e;
    kern<<<(unsigned)blocks, kTcThreads, L::ALLOC, s>>>(q, k, v, out, rest, F);
    TPW_LAUNCH_OK("attention_forward_kernel");
    return TPW_OK;
}

} // namespace

// Rows must start on 16-byte boundaries (TMA, 16-byte stores), and tensors must not be empty.
bool attn_tc_fits(int dtype, const AttnParams &P) {
    if (dtype != TPW_F16 && dtype != TPW_BF16) return false;
    if (tma_disabled() || P.D % 8 != 0 || P.D > 128 || P.Nk == 0) return false;
    auto fits = [](const void *p, const long long (&st)[3]) {
        for (int i = 0; i < 3; ++i)
            if (st[i] % 8 != 0 || st[i] <= 0 || st[i] >= (1LL << 38)) return false;
        return aligned16(p);
    };
    return fits(P.q, P.q_s) && fits(P.k, P.k_s) && fits(P.v, P.v_s) && aligned16(P.out) && aligned16(P.rest);
}

// Ranges of keys for calls whose query tiles are fewer than two CTAs per SM: about three CTAs per SM, so that ragged sequences even
// out, with at least four key tiles each, below which writing and joining the parts costs more than the keys.  bfloat16 [2, 256 x 16384, 32/8,
// 128], lengths 16384 and 1638: 64 CTAs without ranges 260 us, with them 92 and 13 for the join.
AttnSplits attn_tc_splits(const AttnParams &P) {
    AttnSplits r;
    const long long blocks = (P.Nq + 2 * TILE - 1) / (2 * TILE) * P.B * P.Hq, sms = sm_count(), key_tiles = (P.Nk + TILE - 1) / TILE;
    if (blocks >= 2 * sms || key_tiles < 8) return r;
    long long want = (3 * sms + blocks / 2) / blocks;
    if (want > key_tiles / 4) want = key_tiles / 4;
    const long long per = (key_tiles + want - 1) / want;
    r.keys = (int)(per * TILE);
    r.count = (int)((key_tiles + per - 1) / per);
    return r;
}

int attn_tc_forward(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    if (dtype == TPW_F16) return P.D <= 64 ? launch<__half, 1>(P, splits, s) : launch<__half, 2>(P, splits, s);
    return P.D <= 64 ? launch<__nv_bfloat16, 1>(P, splits, s) : launch<__nv_bfloat16, 2>(P, splits, s);
}

} // namespace tpw
