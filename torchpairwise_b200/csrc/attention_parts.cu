// Attention and its gradients in float32 up to 64 features on the 16-bit tensor cores, at float32 accuracy.
//
// Every operand x is the sum of three bfloat16 numbers, h + m + l, each the rounded remainder of those before it: 24 digits and float32's
// exponents.  A product is h h' + (h m' + m h') + (m m' + h l' + l h'), six MMAs; what is left out is below 2^-25 of |x y|.  The tensor cores
// add with truncation, so the small products come first, the large ones last, into an accumulator that starts at zero, over at most 64
// features or 64 tokens; from there a tile's sum moves to a register sum rounded to nearest.
//
// One pass writes the parts of the inputs (attention_parts_kernel): 4 bytes read, 6 written an element, and what lies beyond a sequence's length as zeros.
// Probabilities and gradients of scores are taken apart in registers and go to tensor memory as three operands of 32 columns.
//
// Bound by the tensor cores: 6 x 2 products forward and 6 x 7 backward per 128 x 64 pairs.  An MMA of 128 x 64 x 16 takes 48 clocks where both operands come from
// shared memory (six kilobytes at 128 a clock) and 32 where the left one lies in tensor memory, so 1920 forward and 6900 backward.
// Measured [4, 1024, 8, 64]: parts 11 us, forward 48 us, 1070 TFLOP/s of 16-bit products (179 of float32), the tensor cores busy 63 % of the time; backward 185 us,
// 975 (162), 54 %, what is left being the start of each CTA (216 KB to fetch, 2.5 us) and uneven ends.  The same products as three of tf32: attention_f32.cu.
#include "attention_tc.cuh"

namespace tpw {
namespace {

constexpr int KEYS = 64;                      // tokens of a walked tile
constexpr uint32_t OWN_PART = BLOCK_BYTES;    // a part of 128 tokens, 64 features
constexpr uint32_t WALK_PART = BLOCK_BYTES / 2;
constexpr uint32_t PART_COLUMNS = KEYS / 2;   // of a 128 x 64 operand in tensor memory
typedef Narrow<__nv_bfloat16> Part;

struct PartsParams {
    AttnParams a;
    float scale_log2, scale;
    int tiles;             // of 256 queries forward, 128 backward
    unsigned key_blocks;   // backward: blocks of the keys walk, before those of the queries walk
};

// ---- the inputs' parts ----
struct PartsSource {
    const float *src;
    long long s[3];
    unsigned tokens, heads, pieces;   // pieces of 8 features in all
    bool keys;
    uint4 *dst;                       // [3][B, tokens, heads, features rounded up to 8]
};
struct PartsSources {
    PartsSource at[4];
    const int *key_lengths;
    int D, width;   // pieces a row
};

__device__ __forceinline__ void apart(float a, float b, uint32_t &h, uint32_t &m, uint32_t &l) {
    h = Part::pack(a, b);
    f32x2 r = sub2(pack2(a, b), pack2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)));
    float r0, r1;
    unpack2(r, r0, r1);
    m = Part::pack(r0, r1);
    r = sub2(r, pack2(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)));
    unpack2(r, r0, r1);
    l = Part::pack(r0, r1);
}

__global__ void __launch_bounds__(256) attention_parts_kernel(const __grid_constant__ PartsSources S) {
    const PartsSource &X = S.at[blockIdx.y];
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at >= X.pieces) return;
    const unsigned w = at % S.width, row = at / S.width, h = row % X.heads, bn = row / X.heads, n = bn % X.tokens, b = bn / X.tokens;
    float x[8] = {};
    if (!X.keys || !S.key_lengths || (int)n < S.key_lengths[b]) {
        const float *from = X.src + b * X.s[0] + n * X.s[1] + h * X.s[2] + 8 * w;
        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(from);
        if ((int)(8 * w + 4) < S.D) *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(from + 4);
    }
    uint32_t parts[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) apart(x[2 * e], x[2 * e + 1], parts[0][e], parts[1][e], parts[2][e]);
#pragma unroll
    for (int p = 0; p < 3; ++p) X.dst[(size_t)p * X.pieces + at] = make_uint4(parts[p][0], parts[p][1], parts[p][2], parts[p][3]);
}

// ---- products of parts ----
// the pairs of parts, small products first
__device__ __forceinline__ constexpr int left_part(int i) { return i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0; }
__device__ __forceinline__ constexpr int right_part(int i) { return i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0; }

// D = X Y^T over 64 features (zeros beyond D); X 128 tokens, Y 64.  Fixed counts and addresses that are the same in every lane: the MMAs are
// issued back to back (a count that depends on D: backward 196 -> 187 us at 64 features).
__device__ __forceinline__ void parts_along_features(uint32_t leader, uint32_t d, uint32_t x, uint32_t y, uint32_t idesc) {
    x = __shfl_sync(0xffffffffu, x, 0), y = __shfl_sync(0xffffffffu, y, 0), d = __shfl_sync(0xffffffffu, d, 0);
    const uint64_t a = make_smem_desc(x), b = make_smem_desc(y);
#pragma unroll
    for (int i = 0; i < 6; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            mma_ss(leader, d, a + left_part(i) * (OWN_PART >> 4) + feature_step(k), b + right_part(i) * (WALK_PART >> 4) + feature_step(k), idesc, i + k != 0);
}
// D = P Y over 64 tokens; P in tensor memory
__device__ __forceinline__ void parts_along_tokens(uint32_t leader, uint32_t d, uint32_t p, uint32_t y, uint32_t idesc) {
    p = __shfl_sync(0xffffffffu, p, 0), y = __shfl_sync(0xffffffffu, y, 0), d = __shfl_sync(0xffffffffu, d, 0);
    const uint64_t b = make_smem_desc_tokens(y);
#pragma unroll
    for (int i = 0; i < 6; ++i)
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)
            mma_ts(leader, d, p + left_part(i) * PART_COLUMNS + 8 * k, b + right_part(i) * (WALK_PART >> 4) + k * (2048 >> 4), idesc, i + k != 0);
}
__device__ __forceinline__ uint32_t instruction_parts(uint32_t n, bool b_mn) { return instruction(Part::kFormat, n, b_mn); }

// 64 numbers of a thread's row to tensor memory, in three parts
__device__ __forceinline__ void put_parts(uint32_t at, const float (&p)[KEYS]) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t h[16], m[16], l[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) apart(p[32 * g + 2 * e], p[32 * g + 2 * e + 1], h[e], m[e], l[e]);
        tmem_st16(at + 16 * g, h);
        tmem_st16(at + PART_COLUMNS + 16 * g, m);
        tmem_st16(at + 2 * PART_COLUMNS + 16 * g, l);
    }
}
// acc += a tile's sums
__device__ __forceinline__ void add_tile(f32x2 (&acc)[32], uint32_t at) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t o[32];
        tmem_ld32(at + 32 * g, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[16 * g + e] = add2(acc[16 * g + e], pack2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])));
    }
}
template <int TOKENS> __device__ __forceinline__ void load_parts(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int token, int head, int batch, int batches) {
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int t = 0; t < TOKENS; t += KEYS) tma_load_4d(dst + (p * TOKENS + t) * 128, map, bar, 0, token + t, head, p * batches + batch);
}
// a warp's 32 rows, a row per thread, through 8 KB of shared memory that is no longer in use
__device__ __forceinline__ void store_rows(float *to, long long row_stride, unsigned char *smem, const f32x2 (&acc)[32], float by, bool keep, int lane, int valid, int D) {
    const RowStage<16> stage = {reinterpret_cast<uint4 *>(smem)};
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        float x[4];
        unpack2(acc[2 * k], x[0], x[1]);
        unpack2(acc[2 * k + 1], x[2], x[3]);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = keep ? __float_as_uint(x[e] * by) : 0u;
        stage.put(lane, k, w[0], w[1], w[2], w[3]);
    }
    stage.store(reinterpret_cast<unsigned char *>(to), row_stride * 4, lane, valid, D / 4);
}

// ---- forward ----
// A CTA has two tiles of 128 queries, a row to a thread of either warpgroup, and a warp each that issues its MMAs; the key tiles come once for both,
// through a ring.  While one tile's threads form probabilities the tensor cores work for the other, and the next scores are formed while these are worked on.
// (A CTA per query tile, two to an SM, with room for one K and one V each, waited for them: 60 us where this takes 48, [4, 1024, 8, 64].)
struct ForwardPartsSmem {
    static constexpr int kSlots = 5;
    static constexpr uint32_t TILE_BYTES = 3 * WALK_PART;
    static constexpr uint32_t OFF_RING = 6 * OWN_PART;
    static constexpr uint32_t OFF_BAR = OFF_RING + kSlots * TILE_BYTES;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + 8 * (2 * kSlots + 11);
    static constexpr uint32_t ALLOC = OFF_TMEM + 16 + 1024;
    static_assert(ALLOC <= 232448, "exceeds the dynamic shared memory of one CTA");
};

__global__ void __launch_bounds__(kTcThreads, 1)
attention_forward_parts_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PartsParams F) {
    typedef ForwardPartsSmem L;
    const AttnParams &P = F.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *empty = full + L::kSlots, *q_full = empty + L::kSlots, *s_full = q_full + 1, *o_full = s_full + 2,
             *s_read = o_full + 2, *p_full = s_read + 2, *drained = p_full + 2;   // two of each: the query tiles'
    uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(smem + L::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_TMEM + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned heads = (unsigned)(P.B * P.Hq), bh = blockIdx.x % heads;
    const int row0 = (F.tiles - 1 - (int)(blockIdx.x / heads)) * 2 * TILE;   // a causal call's longest rows first
    const int h = (int)(bh % (unsigned)P.Hq), b = (int)(bh / (unsigned)P.Hq), hk = h / (int)P.group;
    const Seen see(P, b);
    const int nq = (int)P.Nq;
    // key tiles [lo, hi) of query tile s, the same in every lane
    auto range = [&](int s, int &lo, int &hi) {
        const int first = row0 + s * TILE, last = (first + TILE < nq ? first + TILE : nq) - 1;
        lo = see.lo(first) / KEYS;
        hi = first < nq ? (see.hi(last) + KEYS - 1) / KEYS : 0;
        if (hi <= lo) lo = hi = 0;
        lo = __shfl_sync(0xffffffffu, lo, 0);
        hi = __shfl_sync(0xffffffffu, hi, 0);
    };
    int lo0, hi0, lo1, hi1;
    range(0, lo0, hi0);
    range(1, lo1, hi1);
    const int begin = hi0 > 0 && (hi1 == 0 || lo0 < lo1) ? lo0 : lo1, end = hi0 > hi1 ? hi0 : hi1, total = end - begin;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kSlots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 2); }
        mbar_init(q_full, 1);
        for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&o_full[s], 1); mbar_init(&s_read[s], 4); mbar_init(&p_full[s], 4); mbar_init(&drained[s], 1); }
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
        if (P.status) atomicCAS(P.status, 0, (22 << 16) | site);
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag));
        if (!ok) give_up(site);
        return ok;
    };
    const uint32_t q_at = smem_u32(smem), ring = smem_u32(smem + L::OFF_RING);
    // of query tile s: scores, the probabilities' parts, the sums of a key tile
    auto at_of = [&](int s, uint32_t &S, uint32_t &Pr, uint32_t &O) {
        S = tmem + s * 256;
        Pr = S + KEYS;
        O = Pr + 3 * PART_COLUMNS;
    };

    if (warp >= 8) registers_down();
    if (warp == 8) {
        if (lane == 0 && total > 0) {
            uint32_t used = 0;
            mbar_expect_tx(q_full, 6 * OWN_PART);
            load_parts<TILE>(q_at, &map_q, q_full, row0, h, b, (int)P.B);
            load_parts<TILE>(q_at + 3 * OWN_PART, &map_q, q_full, row0 + TILE, h, b, (int)P.B);
            for (uint32_t u = 0; u < 2u * total; ++u) {   // K and V in turn
                const uint32_t slot = u % L::kSlots;
                if (u >= L::kSlots && !wait_or_abort(&empty[slot], parity_of_use(u, L::kSlots) ^ 1, abort_flag)) {
                    give_up(1);
                    break;
                }
                mbar_expect_tx(&full[slot], L::TILE_BYTES);
                load_parts<KEYS>(ring + slot * L::TILE_BYTES, u & 1 ? &map_v : &map_k, &full[slot], (begin + (int)(u / 2)) * KEYS, hk, b, (int)P.B);
                used = u + 1;
            }
            if (!wait_for_releases(empty, used, L::kSlots, abort_flag)) give_up(2);
            if (*abort_flag) {   // what was issued arrives before the CTA ends
                mbar_wait_bounded(q_full, 0);
                for (uint32_t u = first_of_last_uses(used, L::kSlots); u < used; ++u) mbar_wait_bounded(&full[u % L::kSlots], parity_of_use(u, L::kSlots));
            }
        }
    } else if (warp == 9 || warp == 10) {
        const int s = warp - 9, lo = s ? lo1 : lo0, hi = s ? hi1 : hi0;
        const uint32_t idesc_s = instruction_parts(KEYS, false), idesc_o = instruction_parts(KEYS, true);
        const uint32_t leader = elect_lane();
        uint32_t S, Pr, O, done = 0;
        at_of(s, S, Pr, O);
        bool ok = total == 0 || warp_wait(q_full, 0, 3);
        auto mine = [&](int t) { return lo <= t && t < hi; };
        auto scores = [&](int t) {
            const uint32_t u = 2 * (t - begin), slot = u % L::kSlots;
            if (!warp_wait(&full[slot], parity_of_use(u, L::kSlots), 4)) return false;
            tc_fence_after();
            if (mine(t)) {
                parts_along_features(leader, S, q_at + s * 3 * OWN_PART, ring + slot * L::TILE_BYTES, idesc_s);
                commit_by(leader, &s_full[s]);
            }
            commit_by(leader, &empty[slot]);
            return true;
        };
        if (total > 0 && ok) ok = scores(begin);
        for (int t = begin; t < end && ok; ++t) {
            if (t + 1 < end) {
                if (mine(t) && mine(t + 1) && !(ok = warp_wait(&s_read[s], done & 1, 5))) break;
                tc_fence_after();
                if (!(ok = scores(t + 1))) break;
            }
            const uint32_t u = 2 * (t - begin) + 1, slot = u % L::kSlots;
            if (!(ok = warp_wait(&full[slot], parity_of_use(u, L::kSlots), 6))) break;
            if (mine(t)) {
                if (!(ok = warp_wait(&p_full[s], done & 1, 7))) break;
                tc_fence_after();
                parts_along_tokens(leader, O, Pr, ring + slot * L::TILE_BYTES, idesc_o);
                commit_by(leader, &o_full[s]);
                ++done;
            }
            commit_by(leader, &empty[slot]);
        }
        __syncwarp();
    } else if (warp < 8) {
        registers_up();
        const int s = warp >> 2, first = row0 + s * TILE, last = (first + TILE < nq ? first + TILE : nq) - 1, t_first = s ? lo1 : lo0, mine = (s ? hi1 : hi0) - t_first;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int i = first + (warp & 3) * 32 + lane, lo = see.lo(i), hi = i < nq ? see.hi(i) : 0;
        const int all_lo = see.lo(last), all_hi = see.hi(first);   // seen by every row of the tile; rows beyond Nq are not stored
        const float c = F.scale_log2;
        uint32_t S, Pr, O;
        at_of(s, S, Pr, O);
        float m = -INFINITY, l = 0.f, shift = 0.f;
        f32x2 acc[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[e] = pack2(0.f, 0.f);
        bool ok = true;
        for (int u = 0; u < mine; ++u) {
            const int j0 = (t_first + u) * KEYS;
            if (!(ok = warp_wait(&s_full[s], u & 1, 8))) break;
            tc_fence_after();
            float p[KEYS];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t x[32];
                tmem_ld32(S + lanes + 32 * g, x);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) p[32 * g + e] = __uint_as_float(x[e]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_read[s]);
            if (j0 < all_lo || j0 + KEYS > all_hi) {
#pragma unroll
                for (int e = 0; e < KEYS; ++e)
                    if (j0 + e < lo || j0 + e >= hi) p[e] = -INFINITY;
            }
            float tops[4] = {m, -INFINITY, -INFINITY, -INFINITY};   // NaN for a score that is NaN; +inf makes the row NaN: inf - inf
#pragma unroll
            for (int e = 0; e < KEYS; e += 8)
#pragma unroll
                for (int g = 0; g < 4; ++g) tops[g] = max3_nan(tops[g], p[e + 2 * g], p[e + 2 * g + 1]);
            const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
            // Sums are relative to 2^-shift, so what they are scaled by is the quotient of two such powers: exactly 1 while the maximum stays.  (With m c formed
            // anew in a fused multiply-add it was off by the rounding of top c in every tile, all to one side.)
            const float before = shift;
            shift = top == -INFINITY ? 0.f : __fmul_rn(-top, c);
            const float by = m == -INFINITY ? 1.f : exp2_fast(shift - before);   // nothing seen before: sums are zero
            m = top;
            f32x2 sum = pack2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < KEYS; e += 2) {
                const f32x2 y = exp2_pair(fma2(pack2(p[e], p[e + 1]), pack2(c, c), pack2(shift, shift)));
                sum = add2(sum, y);
                unpack2(y, p[e], p[e + 1]);
            }
            float s0, s1;
            unpack2(sum, s0, s1);
            l = l * by + (s0 + s1);
            if (u > 0) {   // the last tile's product is over
                if (!(ok = warp_wait(&o_full[s], (u & 1) ^ 1, 9))) break;
                tc_fence_after();
            }
            put_parts(Pr + lanes, p);
            if (u > 0) add_tile(acc, O + lanes);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[s]);
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[e] = mul2(acc[e], pack2(by, by));
        }
        if (ok && mine > 0) {
            ok = warp_wait(&o_full[s], (mine & 1) ^ 1, 10);
            tc_fence_after();
        } else if (ok && total > 0) {
            ok = warp_wait(q_full, 0, 11);   // its queries are not on their way any more where the zeros go through
        }
        if (ok) {
            if (mine > 0) add_tile(acc, O + lanes);
            const float lse = l == 0.f ? -INFINITY : (log2f(l) - shift) * 0.69314718055994531f;
            if (i < nq && P.lse) static_cast<float *>(P.lse)[bh * P.Nq + i] = lse;
            const int row = i - lane;
            // through the tile's own queries, which no product reads any more
            store_rows(static_cast<float *>(P.out) + ((b * P.Nq + row) * P.Hq + h) * P.D, P.Hq * P.D, smem + s * 3 * OWN_PART + (warp & 3) * 8192, acc, l == 0.f ? 0.f : 1.f / l,
                       l != 0.f, lane, nq - row, (int)P.D);
        }
    }
    tc_fence_before();
    __syncthreads();
    if ((warp == 9 || warp == 10) && *abort_flag) {   // the commits behind all MMAs were waited for, or one more of each issuing lane is waited for here
        commit_by(elect_lane(), &drained[warp - 9]);
        mbar_wait_bounded(&drained[warp - 9], 0);
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- gradients ----
// Two walks as for 16-bit types, each gradient element summed by one CTA in a fixed order.
//   keys walk: 128 keys of a key head, their rows' threads in two warpgroups.  The first forms P^T and sums dV, the second forms dS^T and sums dK, which
//   costs the exponentials twice (512 clocks of the special-function units beside 3840 of the tensor cores) and spares an exchange.
//   queries walk: 128 queries of a head; the warpgroups take the key tiles in turn and add their sums at the end.
// Own and walked parts are 216 KB; twice as many features would not fit.
struct BackwardPartsSmem {
    static constexpr int kX = 3, kY = 2;   // walked tiles of Q or K, which are free after the last product, and of dO or V
    static constexpr uint32_t TILE_BYTES = 3 * WALK_PART;
    static constexpr uint32_t OFF_X = 6 * OWN_PART, OFF_Y = OFF_X + kX * TILE_BYTES;
    static constexpr uint32_t OFF_ROWS = OFF_Y + kY * TILE_BYTES;   // keys walk: lse, delta of a query tile, with its Q
    static constexpr uint32_t OFF_BAR = OFF_ROWS + kX * 2 * KEYS * 4;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + 8 * 26;
    static constexpr uint32_t ALLOC = OFF_TMEM + 16 + 1024;
    static_assert(ALLOC <= 232448, "exceeds the dynamic shared memory of one CTA");
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void take_row(uint32_t at, float (&x)[KEYS]) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t r[32];
        tmem_ld32(at + 32 * g, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[32 * g + e] = __uint_as_float(r[e]);
    }
}
__device__ __forceinline__ void hide(float (&x)[KEYS], int first, int lo, int hi) {
#pragma unroll
    for (int e = 0; e < KEYS; ++e)
        if (first + e < lo || first + e >= hi) x[e] = 0.f;
}

// Barriers of either walk.  A wait for a use of a barrier comes after the one before is known to be over: what both warpgroups pass or
// arrive at, each at its own pace, has a barrier for the even tiles and one for the odd ones.
struct BackwardBarriers {
    uint64_t *own, *x_full, *x_empty, *y_full, *y_empty, *s_full, *dp_full, *s_read, *p_ready, *ds_ready, *sum_full, *sum_read, *all_full, *drained;
    __device__ __forceinline__ explicit BackwardBarriers(uint64_t *at)
        : own(at), x_full(at + 1), x_empty(at + 4), y_full(at + 7), y_empty(at + 9), s_full(at + 11), dp_full(at + 13), s_read(at + 15), p_ready(at + 17), ds_ready(at + 18),
          sum_full(at + 20), sum_read(at + 22), all_full(at + 23), drained(at + 24) {}
    template <bool OF_KEYS> __device__ __forceinline__ void init() const {
        auto init = [](uint64_t *at, int n, int count) {
            for (int i = 0; i < n; ++i) mbar_init(at + i, count);
        };
        init(own, 7, 1);                        // and x_full, x_empty
        init(y_full, 2, 1);
        init(y_empty, 2, OF_KEYS ? 2 : 1);      // keys walk: dP and dV read it
        init(s_full, 4, 1);                     // and dp_full
        init(s_read, 2, 8);
        init(p_ready, 3, 4);                    // and ds_ready
        init(sum_full, 2, 1);
        init(sum_read, 1, 4);
        init(all_full, 1, 2);
        init(drained, 2, 1);
    }
};

template <bool OF_KEYS>
__device__ __forceinline__ void walk(const CUtensorMap &map_q, const CUtensorMap &map_k, const CUtensorMap &map_v, const CUtensorMap &map_g, const PartsParams &F, unsigned block) {
    typedef BackwardPartsSmem L;
    const AttnParams &P = F.a;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const BackwardBarriers bar(reinterpret_cast<uint64_t *>(smem + L::OFF_BAR));
    uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(smem + L::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_TMEM + 4);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned per = (unsigned)(OF_KEYS ? P.Hk : P.Hq), heads = (unsigned)P.B * per, bh = block % heads;
    const int tile = (int)(block / heads), row0 = (OF_KEYS ? tile : F.tiles - 1 - tile) * TILE;   // a causal call's longest rows first
    const int h0 = (int)(bh % per), b = (int)(bh / per), hk = OF_KEYS ? h0 : h0 / (int)P.group, batches = (int)P.B;
    const Seen see(P, b);
    const int nq = (int)P.Nq, rows = OF_KEYS ? see.length : nq, last = (row0 + TILE < rows ? row0 + TILE : rows) - 1;
    const int first = last < row0 ? 0 : OF_KEYS ? see.qlo(row0) : see.lo(row0), end = last < row0 ? 0 : OF_KEYS ? see.qhi(last) : see.hi(last);
    const int begin = first / KEYS, per_head = end > first ? (end + KEYS - 1) / KEYS - begin : 0, total = __shfl_sync(0xffffffffu, OF_KEYS ? per_head * (int)P.group : per_head, 0);

    if (threadIdx.x == 0) {
        bar.init<OF_KEYS>();
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
        if (P.status) atomicCAS(P.status, 0, ((OF_KEYS ? 20 : 21) << 16) | site);
    };
    auto warp_wait = [&](uint64_t *at, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait_or_abort(at, parity, abort_flag));
        if (!ok) give_up(site);
        return ok;
    };
    const uint32_t own_x = smem_u32(smem), own_y = own_x + 3 * OWN_PART, ring_x = smem_u32(smem + L::OFF_X), ring_y = smem_u32(smem + L::OFF_Y);
    // scores of two tiles; keys walk: dP of one, parts of P and dS, sums dV, dK; queries walk: dP of two, parts of two dS, sums dQ
    const uint32_t S = tmem, DP = tmem + 2 * KEYS, LEFT = DP + (OF_KEYS ? 1 : 2) * KEYS, RIGHT = LEFT + 3 * PART_COLUMNS, SUM = RIGHT + 3 * PART_COLUMNS;

    if (warp >= 8) registers_down();
    if (warp == 8) {
        if (lane == 0 && total > 0) {
            uint32_t issued_x = 0, issued_y = 0;
            mbar_expect_tx(bar.own, 6 * OWN_PART);
            load_parts<TILE>(own_x, OF_KEYS ? &map_k : &map_q, bar.own, row0, h0, b, batches);
            load_parts<TILE>(own_y, OF_KEYS ? &map_v : &map_g, bar.own, row0, h0, b, batches);
            auto free = [&](uint64_t *empty, uint32_t u, uint32_t stages) {
                if (u < stages || wait_or_abort(&empty[u % stages], parity_of_use(u, stages) ^ 1, abort_flag)) return true;
                give_up(1);
                return false;
            };
            const uint32_t rows_at = smem_u32(smem + L::OFF_ROWS);
            for (int u = 0; u < total; ++u) {
                const int h = OF_KEYS ? hk * (int)P.group + u / per_head : hk, t0 = (begin + (OF_KEYS ? u % per_head : u)) * KEYS;
                const uint32_t sx = u % L::kX, sy = u % L::kY;
                if (!free(bar.x_empty, u, L::kX)) break;
                mbar_expect_tx(&bar.x_full[sx], L::TILE_BYTES + (OF_KEYS ? 2 * KEYS * 4 : 0));
                load_parts<KEYS>(ring_x + sx * L::TILE_BYTES, OF_KEYS ? &map_q : &map_k, &bar.x_full[sx], t0, h, b, batches);
                if (OF_KEYS) {
                    const long long terms = (b * P.Hq + h) * P.Nqp + t0;
                    bulk_load(rows_at + sx * 2 * KEYS * 4, static_cast<const float *>(P.row_lse) + terms, KEYS * 4, &bar.x_full[sx]);
                    bulk_load(rows_at + (2 * sx + 1) * KEYS * 4, static_cast<const float *>(P.row_delta) + terms, KEYS * 4, &bar.x_full[sx]);
                }
                issued_x = u + 1;
                if (!free(bar.y_empty, u, L::kY)) break;
                mbar_expect_tx(&bar.y_full[sy], L::TILE_BYTES);
                load_parts<KEYS>(ring_y + sy * L::TILE_BYTES, OF_KEYS ? &map_g : &map_v, &bar.y_full[sy], t0, h, b, batches);
                issued_y = u + 1;
            }
            if (!wait_for_releases(bar.x_empty, issued_x, L::kX, abort_flag) || !wait_for_releases(bar.y_empty, issued_y, L::kY, abort_flag)) give_up(2);
            if (*abort_flag) {   // what was issued arrives before the CTA ends
                mbar_wait_bounded(bar.own, 0);
                for (uint32_t u = first_of_last_uses(issued_x, L::kX); u < issued_x; ++u) mbar_wait_bounded(&bar.x_full[u % L::kX], parity_of_use(u, L::kX));
                for (uint32_t u = first_of_last_uses(issued_y, L::kY); u < issued_y; ++u) mbar_wait_bounded(&bar.y_full[u % L::kY], parity_of_use(u, L::kY));
            }
        }
    } else if (warp == 9 || warp == 10) {
        // Two warps issue, each the products of one chain: a wait and a commit cost the issuing warp 100 to 200 clocks, in which the other's MMAs
        // run.
        const uint32_t idesc_s = instruction_parts(KEYS, false), idesc_d = instruction_parts(KEYS, true);
        const uint32_t leader = elect_lane();
        bool ok = total == 0 || warp_wait(bar.own, 0, 3);
        auto arrived = [&](uint64_t *full, uint32_t u, uint32_t stages, int site) {
            if (!warp_wait(&full[u % stages], parity_of_use(u, stages), site)) return false;
            tc_fence_after();
            return true;
        };
        auto from_x = [&](int u) {   // scores
            if (!arrived(bar.x_full, u, L::kX, 4)) return false;
            parts_along_features(leader, S + (u & 1) * KEYS, own_x, ring_x + (u % L::kX) * L::TILE_BYTES, idesc_s);
            commit_by(leader, &bar.s_full[u & 1]);
            return true;
        };
        auto from_y = [&](int u) {   // dP
            if (!arrived(bar.y_full, u, L::kY, 5)) return false;
            parts_along_features(leader, DP + (OF_KEYS ? 0 : (u & 1) * KEYS), own_y, ring_y + (u % L::kY) * L::TILE_BYTES, idesc_s);
            commit_by(leader, &bar.dp_full[OF_KEYS ? 0 : u & 1]);
            commit_by(leader, &bar.y_empty[u % L::kY]);
            return true;
        };
        auto sums = [&](uint32_t to, uint32_t parts, uint32_t tile, uint64_t *full, uint64_t *empty) {
            tc_fence_after();
            parts_along_tokens(leader, to, parts, tile, idesc_d);
            commit_by(leader, full);
            commit_by(leader, empty);
        };
        if (OF_KEYS && warp == 9) {   // S, dV
            if (total > 0 && ok) ok = from_x(0);
            for (int u = 0; u < total && ok; ++u) {
                if (u + 1 < total) {
                    if (u > 0 && !(ok = warp_wait(&bar.s_read[(u - 1) & 1], ((u - 1) >> 1) & 1, 6))) break;
                    if (!(ok = from_x(u + 1))) break;
                }
                if (!(ok = warp_wait(bar.p_ready, u & 1, 7))) break;
                if (!(ok = arrived(bar.y_full, u, L::kY, 12))) break;   // P is made of the scores: it says nothing of dO
                sums(SUM, LEFT, ring_y + (u % L::kY) * L::TILE_BYTES, &bar.sum_full[0], &bar.y_empty[u % L::kY]);
            }
        } else if (OF_KEYS) {   // dP, dK
            if (total > 0 && ok) ok = from_y(0);
            for (int u = 0; u < total && ok; ++u) {
                if (!(ok = warp_wait(bar.ds_ready, u & 1, 8))) break;
                tc_fence_after();
                if (u + 1 < total && !(ok = from_y(u + 1))) break;
                sums(SUM + KEYS, RIGHT, ring_x + (u % L::kX) * L::TILE_BYTES, &bar.sum_full[1], &bar.x_empty[u % L::kX]);
            }
        } else if (warp == 9) {   // S, dQ
            if (total > 0 && ok) ok = from_x(0);
            for (int u = 0; u < total && ok; ++u) {
                if (u + 1 < total && !(ok = from_x(u + 1))) break;   // tile u - 1's gradients are there, so its scores have been read
                if (!(ok = warp_wait(&bar.ds_ready[u & 1], (u >> 1) & 1, 6))) break;
                if (u > 0 && !(ok = warp_wait(bar.sum_read, (u & 1) ^ 1, 7))) break;
                sums(SUM, u & 1 ? RIGHT : LEFT, ring_x + (u % L::kX) * L::TILE_BYTES, &bar.sum_full[u & 1], &bar.x_empty[u % L::kX]);
            }
        } else {   // dP
            for (int u = 0; u < total && ok; ++u) {
                if (u > 1 && !(ok = warp_wait(&bar.ds_ready[u & 1], ((u - 2) >> 1) & 1, 8))) break;
                tc_fence_after();
                ok = from_y(u);
            }
        }
        if (ok && total > 0) commit_by(leader, bar.all_full);
        __syncwarp();
    } else if (warp < 8) {
        registers_up();
        const int group = warp >> 2, i = row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float c = F.scale_log2;
        f32x2 acc[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[e] = pack2(0.f, 0.f);
        bool ok = true;
        if constexpr (OF_KEYS) {
            // rows: keys, columns: queries; those beyond Nq have p = exp(-inf)
            const int lo = see.qlo(i), hi = see.window ? see.qhi(i) : 0x7fffffff;
            const int all_lo = see.qlo(row0 + TILE - 1), all_hi = see.window ? row0 - see.off + see.window : 0x7fffffff;
            uint64_t *const ready = group ? bar.ds_ready : bar.p_ready, *const sums = &bar.sum_full[group];
            const uint32_t parts_at = (group ? RIGHT : LEFT) + lanes, sums_at = SUM + group * KEYS + lanes;
            for (int u = 0; u < total; ++u) {
                const uint32_t st = u % L::kX;
                const float4 *lse = reinterpret_cast<const float4 *>(smem + L::OFF_ROWS + st * 2 * KEYS * 4), *delta = lse + KEYS / 4;
                const int i0 = (begin + u % per_head) * KEYS;
                const bool masked = i0 < all_lo || i0 + KEYS > all_hi;
                if (!(ok = warp_wait(&bar.s_full[u & 1], (u >> 1) & 1, 9) && warp_wait(&bar.x_full[st], parity_of_use(u, L::kX), 10))) break;
                tc_fence_after();
                float p[KEYS];
                take_row(S + (u & 1) * KEYS + lanes, p);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.s_read[u & 1]);
#pragma unroll
                for (int e = 0; e < KEYS; e += 4) {
                    const float4 t = lse[e / 4];
                    unpack2(exp2_pair(fma2(pack2(p[e], p[e + 1]), pack2(c, c), pack2(-t.x, -t.y))), p[e], p[e + 1]);
                    unpack2(exp2_pair(fma2(pack2(p[e + 2], p[e + 3]), pack2(c, c), pack2(-t.z, -t.w))), p[e + 2], p[e + 3]);
                }
                if (group) {
                    if (!(ok = warp_wait(&bar.dp_full[0], u & 1, 11))) break;
                    tc_fence_after();
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t x[32];
                        tmem_ld32(DP + lanes + 32 * g, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 t = delta[8 * g + e / 4];
                            p[32 * g + e] *= __uint_as_float(x[e]) - t.x;
                            p[32 * g + e + 1] *= __uint_as_float(x[e + 1]) - t.y;
                            p[32 * g + e + 2] *= __uint_as_float(x[e + 2]) - t.z;
                            p[32 * g + e + 3] *= __uint_as_float(x[e + 3]) - t.w;
                        }
                    }
                }
                if (masked) hide(p, i0, lo, hi);
                if (u > 0) {   // the last tile's product is over
                    if (!(ok = warp_wait(sums, (u & 1) ^ 1, 13))) break;
                    tc_fence_after();
                }
                put_parts(parts_at, p);
                if (u > 0) add_tile(acc, sums_at);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ready);
            }
            // both sums are over before shared memory serves the stores
            if (ok && total > 0) {
                ok = warp_wait(bar.all_full, 0, 14);
                tc_fence_after();
            }
            if (ok) {
                if (total > 0) add_tile(acc, sums_at);
                const int row = i - lane;
                float *to = static_cast<float *>(group ? P.dk : P.dv) + ((b * P.Nk + row) * P.Hk + hk) * P.D;
                store_rows(to, P.Hk * P.D, smem + warp * 8192, acc, group ? F.scale : 1.f, total > 0 && lo < see.qhi(i), lane, (int)P.Nk - row, (int)P.D);
            }
        } else {
            const int lo = see.lo(i), hi = i < nq ? see.hi(i) : 0;
            const int all_lo = see.lo(last), all_hi = see.hi(row0);   // seen by every query of the tile; those beyond Nq have p = exp(-inf)
            const float lse = static_cast<const float *>(P.row_lse)[bh * P.Nqp + i], delta = static_cast<const float *>(P.row_delta)[bh * P.Nqp + i];
            const uint32_t parts_at = (group ? RIGHT : LEFT) + lanes;
            for (int u = group; u < total; u += 2) {
                const int j0 = (begin + u) * KEYS;
                if (!(ok = warp_wait(&bar.s_full[group], (u >> 1) & 1, 9) && warp_wait(&bar.dp_full[group], (u >> 1) & 1, 11))) break;
                tc_fence_after();
                float p[KEYS];
                take_row(S + group * KEYS + lanes, p);
#pragma unroll
                for (int e = 0; e < KEYS; e += 2) unpack2(exp2_pair(fma2(pack2(p[e], p[e + 1]), pack2(c, c), pack2(-lse, -lse))), p[e], p[e + 1]);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint32_t x[32];
                    tmem_ld32(DP + group * KEYS + lanes + 32 * g, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) p[32 * g + e] *= __uint_as_float(x[e]) - delta;
                }
                if (j0 < all_lo || j0 + KEYS > all_hi) hide(p, j0, lo, hi);
                put_parts(parts_at, p);   // this warpgroup has seen the product over the last ones
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.ds_ready[group]);
                if (!(ok = warp_wait(&bar.sum_full[group], (u >> 1) & 1, 10))) break;
                tc_fence_after();
                add_tile(acc, SUM + lanes);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar.sum_read);
            }
            // the last product is over before shared memory serves the stores; the second warpgroup's sums come through it
            if (ok && total > 0) ok = warp_wait(bar.all_full, 0, 14);
            if (group) {
                float *mine = reinterpret_cast<float *>(smem + 4 * 8192) + (warp & 3) * 32 + lane;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float a0, a1;
                    unpack2(acc[e], a0, a1);
                    mine[(2 * e) * TILE] = a0;
                    mine[(2 * e + 1) * TILE] = a1;
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!group && ok && !*abort_flag) {
                const float *other = reinterpret_cast<const float *>(smem + 4 * 8192) + warp * 32 + lane;
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[e] = add2(acc[e], pack2(other[(2 * e) * TILE], other[(2 * e + 1) * TILE]));
                const int row = i - lane;
                store_rows(static_cast<float *>(P.dq) + ((b * P.Nq + row) * P.Hq + h0) * P.D, P.Hq * P.D, smem + warp * 8192, acc, F.scale, total > 0 && lo < hi, lane, nq - row, (int)P.D);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if ((warp == 9 || warp == 10) && *abort_flag) {   // the commits behind all MMAs were waited for, or one more of each issuing lane is waited for here
        commit_by(elect_lane(), &bar.drained[warp - 9]);
        mbar_wait_bounded(&bar.drained[warp - 9], 0);
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

__global__ void __launch_bounds__(kTcThreads, 1)
attention_backward_parts_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                const __grid_constant__ CUtensorMap map_g, const PartsParams F) {
    if (blockIdx.x < F.key_blocks) walk<true>(map_q, map_k, map_v, map_g, F, blockIdx.x);
    else walk<false>(map_q, map_k, map_v, map_g, F, blockIdx.x - F.key_blocks);
}

long long row_features(const AttnParams &P) { return (P.D + 7) / 8 * 8; }

// parts of `count` tensors (q, k, v and, backward, dO) into scratch, with their maps
int make_parts(const AttnParams &P, int count, void *scratch, CUtensorMap *maps, cudaStream_t s) {
    PartsSources S = {};
    S.key_lengths = P.key_lengths;
    S.D = (int)P.D;
    S.width = (int)(row_features(P) / 8);
    const void *from[4] = {P.q, P.k, P.v, P.dout};
    const long long *strides[4] = {P.q_s, P.k_s, P.v_s, P.do_s};
    uint4 *to = static_cast<uint4 *>(scratch);
    long long most = 0;
    for (int i = 0; i < count; ++i) {
        const bool keys = i == 1 || i == 2;
        const long long tokens = keys ? P.Nk : P.Nq, heads = keys ? P.Hk : P.Hq, pieces = P.B * tokens * heads * S.width, D = row_features(P);
        S.at[i] = {static_cast<const float *>(from[i]), {strides[i][0], strides[i][1], strides[i][2]}, (unsigned)tokens, (unsigned)heads, (unsigned)pieces, keys, to};
        if (const int e = make_tensor_map_heads(&maps[i], to, D, tokens, heads, 3 * P.B, 2 * heads * D, 2 * D, 2 * tokens * heads * D, KEYS)) return e;
        to += 3 * pieces;
        most = most > pieces ? most : pieces;
    }
    attention_parts_kernel<<<dim3((unsigned)((most + 255) / 256), count), 256, 0, s>>>(S);
    TPW_LAUNCH_OK("attention_parts_kernel");
    return TPW_OK;
}

PartsParams parts_params(const AttnParams &P) {
    PartsParams F = {};
    F.a = P;
    F.a.status = device_status_ptr();
    F.scale = (float)P.scale;
    F.scale_log2 = (float)(P.scale * 1.4426950408889634074);
    F.tiles = (int)((P.Nq + TILE - 1) / TILE);
    return F;
}

} // namespace

// Against the tf32 products, all kernels of a call, forward and backward: [4, 1024, 8, 64] 200 and 637 -> 58 and 199 us, causal [1, 4096, 8, 64] 369 and 1263 ->
// 161 and 339, [32, 128, 12, 64] 46 and 145 -> 41 and 101.  64 tokens ([16, 64, 12, 64] 10 and 30 -> 13 and 39 us) leave tiles of 128 rows half empty, and
// forward the parts cost what they save at [8, 77, 8, 64] (11.4 -> 12.6; backward 31 -> 19).  A forward call of few rows goes by ranges of keys
// (attn_f32_splits), which this kernel has not.
static bool parts_fit(int dtype, const AttnParams &P, long long tokens) {
    const long long limit = 1LL << 34;   // numbers of 16-byte pieces stay below 2^31
    return P.D <= 64 && P.Nq >= tokens && P.Nk >= tokens && !tma_disabled() && P.B * P.Nq * P.Hq * row_features(P) < limit && P.B * P.Nk * P.Hk * row_features(P) < limit &&
           3 * P.B * P.Hq < (1LL << 31) && attn_f32_fits(dtype, P);
}
bool attn_parts_fits(int dtype, const AttnParams &P) { return parts_fit(dtype, P, 96) && attn_f32_splits(P).count == 1; }
bool attn_parts_backward_fits(int dtype, const AttnParams &P) { return parts_fit(dtype, P, 65) && attn_f32_backward_fits(dtype, P); }
long long attn_parts_bytes(const AttnParams &P, bool backward) {
    return 6 * row_features(P) * P.B * ((backward ? 2 : 1) * P.Nq * P.Hq + 2 * P.Nk * P.Hk);
}
int attn_parts_forward(const AttnParams &P, void *scratch, cudaStream_t s) {
    CUtensorMap maps[4];
    if (const int e = make_parts(P, 3, scratch, maps, s)) return e;
    PartsParams F = parts_params(P);
    F.tiles = (int)((P.Nq + 2 * TILE - 1) / (2 * TILE));
    const long long blocks = F.tiles * P.B * P.Hq;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    constexpr auto *kern = &attention_forward_parts_kernel;
    if (const int e = allow_shared_memory<kern>((int)ForwardPartsSmem::ALLOC)) return e;
    kern<<<(unsigned)blocks, kTcThreads, ForwardPartsSmem::ALLOC, s>>>(maps[0], maps[1], maps[2], F);
    TPW_LAUNCH_OK("attention_forward_parts_kernel");
    return TPW_OK;
}
int attn_parts_backward(const AttnParams &P, void *scratch, cudaStream_t s) {
    CUtensorMap maps[4];
    if (const int e = make_parts(P, 4, scratch, maps, s)) return e;
    PartsParams F = parts_params(P);
    const long long keys = P.dk ? (P.Nk + TILE - 1) / TILE * P.B * P.Hk : 0, queries = P.dq ? F.tiles * P.B * P.Hq : 0;
    TPW_CHECK_ARG(keys + queries < (1LL << 31), "attention: more than 2^31 blocks of work");
    F.key_blocks = (unsigned)keys;
    constexpr auto *kern = &attention_backward_parts_kernel;
    if (const int e = allow_shared_memory<kern>((int)BackwardPartsSmem::ALLOC)) return e;
    kern<<<(unsigned)(keys + queries), kTcThreads, BackwardPartsSmem::ALLOC, s>>>(maps[0], maps[1], maps[2], maps[3], F);
    TPW_LAUNCH_OK("attention_backward_parts_kernel");
    return TPW_OK;
}

} // namespace tpw
