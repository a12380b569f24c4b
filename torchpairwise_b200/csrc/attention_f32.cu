// Attention and its gradients in float32 up to 128 features, rows on 16-byte boundaries: what attention_parts.cu does not take, more than 64 features, few tokens,
// and few rows against many keys.  (Above 64 features the three parts of a gradient walk's own two tiles alone are 192 KB and leave no room for walked ones.  The
// forward's would fit, with a tile of queries at 96 KB and one tile each of 64 keys and values at 48; there is no such kernel.)
//
// Every product runs on the tensor cores with tf32 operands at float32 accuracy: x = h + l, h the nearest number of 11 digits, l the rest,
// and x y = h h' + (h l' + l h') up to 2^-23.  The tensor cores add with truncation, so the large products are summed over at most 128
// features or 64 tokens before the sum moves to a register sum rounded to nearest, and the small ones have sums of their own.
//
// Why m16n8k8 in registers and not tcgen05: the probabilities come out of the first product in the very layout in which the second takes them
// (an accumulator's columns 2t, 2t+1 are the operand's elements t, t+4 when the tokens of a step are taken in that order), and are split
// there; and tiles of 64 rows and any number of features fit.  The instruction reaches 277 TFLOP/s of tf32 on one B200, so 92 after the
// split, where the CUDA cores have 71; these kernels 42 forward ([4, 1024, 8, 64] 200 us) and 47 backward (637 us).
//
// A CTA has 64 rows, four warps of 16, and walks over tiles of the other side, two CTAs to an SM.  Shared-memory rows are 4 floats apart modulo 32
// banks: operands along features read rows 4 g + t, along tokens 8 t + g, either without conflicts.  Fixed order everywhere, no atomics.
#include "attention.cuh"

namespace tpw {
namespace {

constexpr int ROWS = 64, THREADS = 128;

__device__ __forceinline__ void split(float x, uint32_t &h, uint32_t &l) {
    h = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    l = __float_as_uint(x - __uint_as_float(h));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// large and small parts of a step's products
__device__ __forceinline__ void mma3(float (&big)[4], float (&small)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
    uint32_t h0, l0, h1, l1;
    split(b0, h0, l0);
    split(b1, h1, l1);
    mma(small, al, h0, h1);
    mma(small, ah, l0, l1);
    mma(big, ah, h0, h1);
}

template <int DP> constexpr int kPitch = DP + 4;

// rows [row0, row0 + N) of a [tokens, D] slice to shared memory; zero from `rows` and D on
template <int N, int DP> __device__ __forceinline__ void fetch(float *dst, const float *src, long long stride, int row0, int rows, int D) {
    constexpr int PER = DP / 4;
#pragma unroll 4
    for (int c = threadIdx.x; c < N * PER; c += THREADS) {
        const int r = c / PER, d = (c % PER) * 4;
        float *to = dst + r * kPitch<DP> + d;
        if (row0 + r < rows && d < D)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(src + (long long)(row0 + r) * stride + d) : "memory");
        else
            *reinterpret_cast<float4 *>(to) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// s = X Y^T: 16 rows of X (the warp's, from x), N rows of Y, contracting 8 * steps features
template <int N, int DP> __device__ __forceinline__ void along_features(float (&s)[N / 8][4], const float *x, const float *y, int steps, int g, int t) {
    float small[N / 8][4];
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = small[n][e] = 0.f;
#pragma unroll 2
    for (int k = 0; k < steps; ++k) {
        uint32_t ah[4], al[4];
        const float *a = x + g * kPitch<DP> + 8 * k + t;
        split(a[0], ah[0], al[0]);
        split(a[8 * kPitch<DP>], ah[1], al[1]);
        split(a[4], ah[2], al[2]);
        split(a[8 * kPitch<DP> + 4], ah[3], al[3]);
#pragma unroll
        for (int n = 0; n < N / 8; ++n) {
            const float *b = y + (8 * n + g) * kPitch<DP> + 8 * k + t;
            mma3(s[n], small[n], ah, al, b[0], b[4]);
        }
    }
#pragma unroll
    for (int n = 0; n < N / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += small[n][e];
}

// sum = sum * by + P Y: P 16 x N in accumulator layout, Y N rows of D features; by[0] for rows g, by[1] for rows g + 8
template <int N, int DP> __device__ __forceinline__ void along_tokens(float (&sum)[DP / 8][4], const float (&by)[2], const float (&p)[N / 8][4], const float *y, int D, int g, int t) {
    constexpr int C = 4;   // feature groups of eight at a time
#pragma unroll
    for (int c = 0; c < DP / 8; c += C) {
        if (8 * c >= D) break;
        float big[C][4], small[C][4];
#pragma unroll
        for (int n = 0; n < C; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) big[n][e] = small[n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < N / 8; ++k) {
            uint32_t ah[4], al[4];
            split(p[k][0], ah[0], al[0]);
            split(p[k][2], ah[1], al[1]);
            split(p[k][1], ah[2], al[2]);
            split(p[k][3], ah[3], al[3]);
            const float *b = y + (8 * k + 2 * t) * kPitch<DP> + 8 * c + g;
#pragma unroll
            for (int n = 0; n < C; ++n) mma3(big[n], small[n], ah, al, b[8 * n], b[kPitch<DP> + 8 * n]);
        }
#pragma unroll
        for (int n = 0; n < C; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[c + n][e] = fmaf(sum[c + n][e], by[e >> 1], big[n][e] + small[n][e]);
    }
}

// 16 rows from `row` on to a dense [tokens, D] slice, times by; 0 is a row that sees nothing: zero, although its sums are 0 times what need not be finite
template <int DP> __device__ __forceinline__ void store(float *dst, long long stride, const float (&acc)[DP / 8][4], const float (&by)[2], int row, int rows, int D, int g, int t) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (row + g + 8 * r >= rows) continue;
        float *p = dst + (long long)(row + g + 8 * r) * stride + 2 * t;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            if (8 * n + 2 * t < D)
                *reinterpret_cast<float2 *>(p + 8 * n) = by[r] == 0.f ? make_float2(0.f, 0.f) : make_float2(acc[n][2 * r] * by[r], acc[n][2 * r + 1] * by[r]);
    }
}

constexpr float kLog2e = 1.4426950408889634f;

struct F32Params {
    AttnParams a;
    int tiles;                     // of 64 rows
    int splits, keys_per_split;    // ranges of keys (forward)
    float *part_out, *part_lse;
};

template <int DP, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS, 2) attention_forward_f32_kernel(const F32Params F) {
    const AttnParams &P = F.a;
    extern __shared__ __align__(16) float smem_f32[];
    float *Q = smem_f32, *ring = Q + ROWS * kPitch<DP>;
    constexpr int HALF = BN * kPitch<DP>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, D = (int)P.D, steps = (D + 7) / 8, nq = (int)P.Nq;
    const unsigned split_at = blockIdx.x % F.splits, item = blockIdx.x / F.splits, heads = (unsigned)(P.B * P.Hq);
    const int row0 = (F.tiles - 1 - (int)(item / heads)) * ROWS;   // a causal call's longest rows first
    const unsigned bh = item % heads;
    const long long h = bh % (unsigned)P.Hq, b = bh / (unsigned)P.Hq, hk = h / P.group;
    const Seen see(P, b);
    const float *k = static_cast<const float *>(P.k) + b * P.k_s[0] + hk * P.k_s[2], *v = static_cast<const float *>(P.v) + b * P.v_s[0] + hk * P.v_s[2];
    const int last = row0 + ROWS < nq ? row0 + ROWS - 1 : nq - 1;
    int first = see.lo(row0), end = see.hi(last);
    if (F.splits > 1) {
        const int from = (int)split_at * F.keys_per_split, to = from + F.keys_per_split;
        first = first > from ? first : from;
        end = end < to ? end : to;
    }
    const int begin = first / BN * BN, total = end > first ? (end - begin + BN - 1) / BN : 0;
    fetch<ROWS, DP>(Q, static_cast<const float *>(P.q) + b * P.q_s[0] + h * P.q_s[2], P.q_s[1], row0, nq, D);
    auto fetch_tile = [&](int u) {
        float *to = ring + (u % STAGES) * 2 * HALF;
        fetch<BN, DP>(to, k, P.k_s[1], begin + u * BN, see.length, D);
        fetch<BN, DP>(to + HALF, v, P.v_s[1], begin + u * BN, see.length, D);
    };
    if (total > 0) fetch_tile(0);
    fetch_commit();
    const float scale = (float)(P.scale * 1.4426950408889634074);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, O[DP / 8][4];
    int lo[2], hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = row0 + 16 * warp + g + 8 * r;
        lo[r] = see.lo(i) > first ? see.lo(i) : first;
        hi[r] = i < nq ? (see.hi(i) < end ? see.hi(i) : end) : 0;
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[n][e] = 0.f;
    for (int u = 0; u < total; ++u) {
        if (STAGES > 1 && u + 1 < total) fetch_tile(u + 1);
        fetch_commit();
        fetch_wait<STAGES - 1>();
        __syncthreads();
        const float *K = ring + (u % STAGES) * 2 * HALF, *V = K + HALF;
        const int j0 = begin + u * BN + 2 * t;
        float s[BN / 8][4], top[2] = {m[0], m[1]}, by[2];
        along_features<BN, DP>(s, Q + 16 * warp * kPitch<DP>, K, steps, g, t);
#pragma unroll
        for (int n = 0; n < BN / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = j0 + 8 * n + (e & 1), r = e >> 1;
                s[n][e] = j >= lo[r] && j < hi[r] ? s[n][e] * scale : -INFINITY;
                top[r] = fmaxf(top[r], s[n][e]);
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            const float base = top[r] == -INFINITY ? 0.f : top[r];   // nothing seen so far: every power below is 0
            by[r] = exp2f(m[r] - base);
            m[r] = top[r];
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < BN / 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][2 * r + e] = exp2f(s[n][2 * r + e] - base);
                    sum += s[n][2 * r + e];
                }
            l[r] = l[r] * by[r] + sum;
        }
        along_tokens<BN, DP>(O, by, s, V, D, g, t);
        __syncthreads();
        if (STAGES == 1 && u + 1 < total) fetch_tile(u + 1);
    }
    fetch_wait<0>();
    float inv[2];
    const long long all_rows = P.B * P.Hq * P.Nq;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        inv[r] = l[r] == 0.f ? 0.f : 1.f / l[r];
        const int i = row0 + 16 * warp + g + 8 * r;
        const float lse = l[r] == 0.f ? -INFINITY : m[r] / kLog2e + logf(l[r]);
        if (t == 0 && i < nq) {
            if (F.splits > 1) F.part_lse[split_at * all_rows + bh * P.Nq + i] = lse;
            else if (P.lse) static_cast<float *>(P.lse)[bh * P.Nq + i] = lse;
        }
    }
    if (F.splits > 1) {
        if (total > 0) store<DP>(F.part_out + (split_at * all_rows + bh * P.Nq) * P.D, P.D, O, inv, row0 + 16 * warp, nq, D, g, t);
    } else {
        store<DP>(static_cast<float *>(P.out) + (b * P.Nq * P.Hq + h) * P.D, P.Hq * P.D, O, inv, row0 + 16 * warp, nq, D, g, t);
    }
}

// One walk of the backward: KEYS holds 64 keys and walks over the queries of every head that shares them (dk, dv), otherwise 64 queries over
// the keys (dq).  Rows are the CTA's own side, columns the walked one.
template <int DP, int BN, int STAGES, bool KEYS>
__device__ __forceinline__ void walk(const F32Params &F, unsigned block) {
    const AttnParams &P = F.a;
    extern __shared__ __align__(16) float smem_f32[];
    constexpr int HALF = BN * kPitch<DP>;
    float *X = smem_f32, *W = X + ROWS * kPitch<DP>, *ring = W + ROWS * kPitch<DP>;   // own K, V or Q, dO; walked Q, dO or K, V
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, D = (int)P.D, steps = (D + 7) / 8, nq = (int)P.Nq;
    const unsigned per = (unsigned)(KEYS ? P.Hk : P.Hq), heads = (unsigned)P.B * per, bh = block % heads;
    const int tile = (int)(block / heads), row0 = (KEYS ? tile : F.tiles - 1 - tile) * ROWS;
    const long long h0 = bh % per, b = bh / per, hk = KEYS ? h0 : h0 / P.group;
    const Seen see(P, b);
    const int rows = KEYS ? see.length : nq, last = (row0 + ROWS < rows ? row0 + ROWS : rows) - 1;
    const float *q = static_cast<const float *>(P.q) + b * P.q_s[0], *go = static_cast<const float *>(P.dout) + b * P.do_s[0];
    const float *k = static_cast<const float *>(P.k) + b * P.k_s[0] + hk * P.k_s[2], *v = static_cast<const float *>(P.v) + b * P.v_s[0] + hk * P.v_s[2];
    const int first = last < row0 ? 0 : KEYS ? see.qlo(row0) : see.lo(row0), end = last < row0 ? 0 : KEYS ? see.qhi(last) : see.hi(last);
    const int begin = first / BN * BN, per_head = end > first ? (end - begin + BN - 1) / BN : 0, total = KEYS ? per_head * (int)P.group : per_head;
    if (KEYS) {
        fetch<ROWS, DP>(X, k, P.k_s[1], row0, see.length, D);
        fetch<ROWS, DP>(W, v, P.v_s[1], row0, see.length, D);
    } else {
        fetch<ROWS, DP>(X, q + h0 * P.q_s[2], P.q_s[1], row0, nq, D);
        fetch<ROWS, DP>(W, go + h0 * P.do_s[2], P.do_s[1], row0, nq, D);
    }
    auto fetch_tile = [&](int u) {
        float *to = ring + (u % STAGES) * 2 * HALF;
        if (KEYS) {
            const long long h = hk * P.group + u / per_head;
            const int i0 = begin + u % per_head * BN;
            fetch<BN, DP>(to, q + h * P.q_s[2], P.q_s[1], i0, nq, D);
            fetch<BN, DP>(to + HALF, go + h * P.do_s[2], P.do_s[1], i0, nq, D);
        } else {
            fetch<BN, DP>(to, k, P.k_s[1], begin + u * BN, see.length, D);
            fetch<BN, DP>(to + HALF, v, P.v_s[1], begin + u * BN, see.length, D);
        }
    };
    if (total > 0) fetch_tile(0);
    fetch_commit();
    const float scale = (float)(P.scale * 1.4426950408889634074);
    const float *all_lse = static_cast<const float *>(P.row_lse) + b * P.Hq * P.Nqp, *all_delta = static_cast<const float *>(P.row_delta) + b * P.Hq * P.Nqp;
    float one[2] = {1.f, 1.f}, dx[DP / 8][4], dw[KEYS ? DP / 8 : 1][4], own_lse[2], own_delta[2];
    int lo[2], hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int x = row0 + 16 * warp + g + 8 * r;
        lo[r] = KEYS ? see.qlo(x) : see.lo(x);
        hi[r] = KEYS ? see.qhi(x) : x < nq ? see.hi(x) : 0;
        own_lse[r] = !KEYS && x < nq ? all_lse[h0 * P.Nqp + x] : 0.f;
        own_delta[r] = !KEYS && x < nq ? all_delta[h0 * P.Nqp + x] : 0.f;
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            dx[n][e] = 0.f;
            if (KEYS) dw[KEYS ? n : 0][e] = 0.f;
        }
    for (int u = 0; u < total; ++u) {
        if (STAGES > 1 && u + 1 < total) fetch_tile(u + 1);
        fetch_commit();
        fetch_wait<STAGES - 1>();
        __syncthreads();
        const float *Y = ring + (u % STAGES) * 2 * HALF, *Z = Y + HALF;
        const int c0 = begin + (KEYS ? u % per_head : u) * BN + 2 * t;
        const long long terms = KEYS ? (hk * P.group + u / per_head) * P.Nqp + c0 : 0;
        float p[BN / 8][4], s[BN / 8][4];
        along_features<BN, DP>(p, X + 16 * warp * kPitch<DP>, Y, steps, g, t);
#pragma unroll
        for (int n = 0; n < BN / 8; ++n) {
            const float2 lse = KEYS ? *reinterpret_cast<const float2 *>(all_lse + terms + 8 * n) : make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = c0 + 8 * n + (e & 1), r = e >> 1;
                p[n][e] = c >= lo[r] && c < hi[r] ? exp2f(p[n][e] * scale - (KEYS ? (e & 1 ? lse.y : lse.x) : own_lse[r])) : 0.f;
            }
        }
        if (KEYS) along_tokens<BN, DP>(reinterpret_cast<float(&)[DP / 8][4]>(dw), one, p, Z, D, g, t);
        along_features<BN, DP>(s, W + 16 * warp * kPitch<DP>, Z, steps, g, t);
#pragma unroll
        for (int n = 0; n < BN / 8; ++n) {
            const float2 delta = KEYS ? *reinterpret_cast<const float2 *>(all_delta + terms + 8 * n) : make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {   // 0 times what need not be finite
                const int c = c0 + 8 * n + (e & 1), r = e >> 1;
                p[n][e] = c >= lo[r] && c < hi[r] ? p[n][e] * (s[n][e] - (KEYS ? (e & 1 ? delta.y : delta.x) : own_delta[r])) : 0.f;
            }
        }
        along_tokens<BN, DP>(dx, one, p, Y, D, g, t);
        __syncthreads();
        if (STAGES == 1 && u + 1 < total) fetch_tile(u + 1);
    }
    fetch_wait<0>();
    const bool some[2] = {lo[0] < hi[0], lo[1] < hi[1]};
    const float by[2] = {some[0] ? (float)P.scale : 0.f, some[1] ? (float)P.scale : 0.f}, as[2] = {some[0] ? 1.f : 0.f, some[1] ? 1.f : 0.f};
    if (KEYS) {
        const long long to = (b * P.Nk * P.Hk + hk) * P.D;
        store<DP>(static_cast<float *>(P.dk) + to, P.Hk * P.D, dx, by, row0 + 16 * warp, (int)P.Nk, D, g, t);
        store<DP>(static_cast<float *>(P.dv) + to, P.Hk * P.D, reinterpret_cast<const float(&)[DP / 8][4]>(dw), as, row0 + 16 * warp, (int)P.Nk, D, g, t);
    } else {
        store<DP>(static_cast<float *>(P.dq) + (b * P.Nq * P.Hq + h0) * P.D, P.Hq * P.D, dx, by, row0 + 16 * warp, nq, D, g, t);
    }
}

// both walks in one launch, the keys' blocks first
template <int DP, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS, 2) attention_backward_f32_kernel(const F32Params F, unsigned key_blocks) {
    if (blockIdx.x < key_blocks) walk<DP, BN, STAGES, true>(F, blockIdx.x);
    else walk<DP, BN, STAGES, false>(F, blockIdx.x - key_blocks);
}

template <int DP, int BN, int STAGES> int forward(const F32Params &F, cudaStream_t s) {
    constexpr size_t smem = 4 * (ROWS + STAGES * 2 * BN) * kPitch<DP>;
    const long long blocks = F.tiles * F.a.B * F.a.Hq * F.splits;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    constexpr auto *kern = &attention_forward_f32_kernel<DP, BN, STAGES>;
    if (const int e = allow_shared_memory<kern>((int)smem)) return e;
    kern<<<(unsigned)blocks, THREADS, smem, s>>>(F);
    TPW_LAUNCH_OK("attention_forward_f32_kernel");
    return TPW_OK;
}
template <int DP, int BN, int STAGES> int backward(const F32Params &F, cudaStream_t s) {
    constexpr size_t smem = 4 * (2 * ROWS + STAGES * 2 * BN) * kPitch<DP>;
    const AttnParams &P = F.a;
    const long long keys = P.dk ? (P.Nk + ROWS - 1) / ROWS * P.B * P.Hk : 0, queries = P.dq ? F.tiles * P.B * P.Hq : 0;
    TPW_CHECK_ARG(keys + queries < (1LL << 31), "attention: more than 2^31 blocks of work");
    constexpr auto *kern = &attention_backward_f32_kernel<DP, BN, STAGES>;
    if (const int e = allow_shared_memory<kern>((int)smem)) return e;
    kern<<<(unsigned)(keys + queries), THREADS, smem, s>>>(F, (unsigned)keys);
    TPW_LAUNCH_OK("attention_backward_f32_kernel");
    return TPW_OK;
}

bool fits_rows(const void *p, const long long (&st)[3]) {
    return aligned16(p) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

} // namespace

bool attn_f32_fits(int dtype, const AttnParams &P) {
    return dtype == TPW_F32 && P.D <= 128 && P.D % 4 == 0 && P.Nk > 0 && fits_rows(P.q, P.q_s) && fits_rows(P.k, P.k_s) && fits_rows(P.v, P.v_s) && aligned16(P.out);
}
bool attn_f32_backward_fits(int dtype, const AttnParams &P) {
    return attn_f32_fits(dtype, P) && fits_rows(P.dout, P.do_s) && aligned16(P.dq) && aligned16(P.dk) && aligned16(P.dv);
}

// Ranges of keys where the 64-row tiles are fewer than two CTAs per SM, at least 256 keys each.
AttnSplits attn_f32_splits(const AttnParams &P) {
    AttnSplits r;
    const long long blocks = (P.Nq + ROWS - 1) / ROWS * P.B * P.Hq, slots = 2LL * sm_count();
    if (blocks * 2 > slots || P.Nk < 512) return r;
    long long want = slots / blocks;
    if (want > P.Nk / 256) want = P.Nk / 256;
    r.keys = (int)(((P.Nk + want - 1) / want + 63) / 64 * 64);
    r.count = (int)((P.Nk + r.keys - 1) / r.keys);
    return r;
}

int attn_f32_forward(const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    F32Params F = {P, (int)((P.Nq + ROWS - 1) / ROWS), splits.count, splits.keys, splits.out, splits.lse};
    return P.D <= 64 ? forward<64, 64, 2>(F, s) : forward<128, 32, 2>(F, s);
}
int attn_f32_backward(const AttnParams &P, cudaStream_t s) {
    F32Params F = {P, (int)((P.Nq + ROWS - 1) / ROWS), 1, 0, nullptr, nullptr};
    return P.D <= 64 ? backward<64, 64, 2>(F, s) : backward<128, 32, 1>(F, s);
}

} // namespace tpw
