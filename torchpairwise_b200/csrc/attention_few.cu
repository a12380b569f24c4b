// Attention of few query rows (16-bit types, up to 128 features): one or a few new tokens against a long cache.
//
// Bound by HBM: every key and value is read once for all query heads that share it, up to 32 rows (heads of the group times
// queries) that make the M side of m16n8k16 products.  32 rows cannot fill a tcgen05 tile, and the tensor pipe is far from busy: 32 products
// per 16 keys and warp.  The keys are cut into ranges so that all SMs read; a range is one CTA: a warp issues TMA into a ring of 64-key stages,
// four warps take 16 keys of a stage each, with a running maximum, sum and output of their own that meet only at the end.  Ranges
// write outputs and log-sums that attention_join_kernel weighs together (skipped when there is one range).
// Measured bfloat16 [16, 1 x 16384, 32/8, 128], ragged lengths: 591 MB in 100 us, 5.9 TB/s, and 5 us for the join.
#include "attention_tc.cuh"

namespace tpw {
namespace {

constexpr int STEP = 64;   // keys per stage

struct FewParams {
    AttnParams a;
    float scale_log2;
    int rows;              // group * Nq
    int splits, keys_per_split;
    float *part_out, *part_lse;   // splits > 1
};

template <int BLOCKS> struct FewSmem {
    static constexpr int kStages = BLOCKS == 2 ? 3 : 6;
    static constexpr uint32_t HALF = BLOCKS * STEP * 128;   // bytes of the K or V part of a stage
    static constexpr uint32_t OFF_BAR = kStages * 2 * HALF;
    static constexpr uint32_t OFF_FLAG = OFF_BAR + 8 * 2 * kStages;
    static constexpr uint32_t ALLOC = OFF_FLAG + 16 + 1024;
};
constexpr int kFewThreads = 160;

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// MT: tiles of 16 rows
template <typename T, int BLOCKS, int MT>
__global__ void __launch_bounds__(kFewThreads, MT == 1 ? 2 : 1)
attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const FewParams F) {
    typedef FewSmem<BLOCKS> L;
    typedef Narrow<T> N;
    const AttnParams &P = F.a;
    constexpr int DP = 64 * BLOCKS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::OFF_BAR), *empty = full + L::kStages;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::OFF_FLAG);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int split = (int)(blockIdx.x % F.splits);
    const long long bh = blockIdx.x / F.splits;
    const int hk = (int)(bh % P.Hk), b = (int)(bh / P.Hk), nq = (int)P.Nq, group = (int)P.group, D = (int)P.D;
    const Seen see(P, b);
    // keys of this range that any row sees
    int first = see.lo(0), end = see.hi(nq - 1);
    if (first < split * F.keys_per_split) first = split * F.keys_per_split;
    if (end > (split + 1) * F.keys_per_split) end = (split + 1) * F.keys_per_split;
    const int begin = first / STEP * STEP, stages = end > first ? (end - begin + STEP - 1) / STEP : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 4); }
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_descriptor(&map_k);
        tma_prefetch_descriptor(&map_v);
    }
    __syncthreads();
    auto give_up = [&](int site) {
        *abort_flag = 1;
        if (P.status) atomicCAS(P.status, 0, (19 << 16) | site);
    };
    const uint32_t ring = smem_u32(smem);
    float m[MT][2], l[MT][2], o[MT][DP / 8][4];

    if (warp == 4) {
        if (lane == 0) {
            uint32_t issued = 0;
            for (int u = 0; u < stages; ++u) {
                const uint32_t st = u % L::kStages;
                if (u >= L::kStages && !wait_or_abort(&empty[st], parity_of_use(u, L::kStages) ^ 1, abort_flag)) {
                    give_up(1);
                    break;
                }
                mbar_expect_tx(&full[st], 2 * L::HALF);
                const uint32_t to = ring + st * 2 * L::HALF;
#pragma unroll
                for (int c = 0; c < BLOCKS; ++c) {
                    tma_load_4d(to + c * STEP * 128, &map_k, &full[st], 64 * c, begin + u * STEP, hk, b);
                    tma_load_4d(to + L::HALF + c * STEP * 128, &map_v, &full[st], 64 * c, begin + u * STEP, hk, b);
                }
                issued = u + 1;
            }
            if (*abort_flag)   // what was issued arrives before the CTA ends
                for (uint32_t u = first_of_last_uses(issued, L::kStages); u < issued; ++u) mbar_wait_bounded(&full[u % L::kStages], parity_of_use(u, L::kStages));
        }
    } else {
        // rows of this thread: 16 mt + g and 16 mt + g + 8; row r is query r % nq of head hk * group + r / nq
        uint32_t q[MT][DP / 16][4];
        int lo[MT][2], hi[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = 16 * mt + g + 8 * k;
                const bool valid = r < F.rows;
                const int i = valid ? r % nq : 0, h = hk * group + (valid ? r / nq : 0);
                lo[mt][k] = see.lo(i);
                hi[mt][k] = valid ? see.hi(i) : 0;
                const T *row = static_cast<const T *>(P.q) + b * P.q_s[0] + i * P.q_s[1] + h * P.q_s[2];
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int at = 16 * d + 8 * half + 2 * t4;
                        q[mt][d][k + 2 * half] = valid && at < D ? *reinterpret_cast<const uint32_t *>(row + at) : 0u;
                    }
                m[mt][k] = -INFINITY;
                l[mt][k] = 0.f;
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
        const int key = 16 * warp + (lane & 7);   // of the stage, plus 8 for some of the matrices that a lane addresses
        for (int u = 0; u < stages; ++u) {
            const uint32_t st = u % L::kStages;
            const bool ok = __all_sync(0xffffffffu, wait_or_abort(&full[st], parity_of_use(u, L::kStages), abort_flag));
            if (!ok) {
                give_up(2);
                break;
            }
            const int j0 = begin + u * STEP + 16 * warp;
            const uint32_t k_at = ring + st * 2 * L::HALF, v_at = k_at + L::HALF;
            if (j0 < end) {
                float s[MT][2][4] = {};
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    // keys 0-7 and 8-15 (lane bit 4), features 0-7 and 8-15 (lane bit 3)
                    uint32_t kb[4];
                    const int row = key + ((lane >> 4) & 1) * 8, chunk = 2 * (d & 3) + ((lane >> 3) & 1);
                    ldmatrix4(kb, k_at + (d >> 2) * STEP * 128 + swz128(row, chunk));
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        mma16<T>(s[mt][0], q[mt][d], kb[0], kb[1]);
                        mma16<T>(s[mt][1], q[mt][d], kb[2], kb[3]);
                    }
                }
                uint32_t p[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float top[2] = {m[mt][0], m[mt][1]};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = j0 + 8 * n + 2 * t4 + (e & 1);
                            if (j < lo[mt][e >> 1] || j >= hi[mt][e >> 1]) s[mt][n][e] = -INFINITY;
                            top[e >> 1] = fmaxf(top[e >> 1], s[mt][n][e]);
                        }
                    bool moved = false;
                    float shift[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
                        top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2));
                        moved = moved || top[k] > m[mt][k];
                        shift[k] = top[k] == -INFINITY ? 0.f : N::kLift - top[k] * F.scale_log2;
                    }
                    if (__any_sync(0xffffffffu, moved)) {
                        float by[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            by[k] = top[k] > m[mt][k] ? exp2_fast((m[mt][k] - top[k]) * F.scale_log2) : 1.f;
                            l[mt][k] *= by[k];
                            m[mt][k] = top[k];
                        }
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[mt][n][e] *= by[e >> 1];
                    }
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[mt][n][e] = exp2_fast(fmaf(s[mt][n][e], F.scale_log2, shift[e >> 1]));
                            l[mt][e >> 1] += s[mt][n][e];
                        }
                        p[mt][2 * n] = N::pack(s[mt][n][0], s[mt][n][1]);
                        p[mt][2 * n + 1] = N::pack(s[mt][n][2], s[mt][n][3]);
                    }
                }
                // values of keys that no row sees need not be finite: bits that are 0 for them
                uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
                if (j0 < first || j0 + 16 > end)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int j = j0 + 2 * t4 + 8 * k;
                        keep[k] = (j >= first && j < end ? 0xffffu : 0u) | (j + 1 >= first && j + 1 < end ? 0xffff0000u : 0u);
                    }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    // keys 0-7 and 8-15 (lane bit 3), features 0-7 and 8-15 (lane bit 4), transposed
                    uint32_t vb[4];
                    const int row = key + ((lane >> 3) & 1) * 8, chunk = 2 * (d & 3) + ((lane >> 4) & 1);
                    ldmatrix4t(vb, v_at + (d >> 2) * STEP * 128 + swz128(row, chunk));
#pragma unroll
                    for (int k = 0; k < 4; ++k) vb[k] &= keep[k & 1];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        mma16<T>(o[mt][2 * d], p[mt], vb[0], vb[1]);
                        mma16<T>(o[mt][2 * d + 1], p[mt], vb[2], vb[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
    }
    __syncthreads();
    if (*abort_flag) return;
    // the four warps' shares of each 16 rows meet in the ring: [warp][16][DP] outputs, then [warp][16] maxima and sums
    float *share = reinterpret_cast<float *>(smem), *stats = share + 4 * 16 * DP;
    static_assert(4 * 16 * DP * 4 + 4 * 32 * 4 <= (int)L::OFF_BAR, "the shares fit the ring");
    const long long all_rows = P.B * P.Hq * P.Nq;
    for (int mt = 0; mt < MT; ++mt) {
        if (mt > 0) __syncthreads();
        if (warp < 4) {
#pragma unroll
            for (int w = 0; w < MT; ++w) {
                if (w != mt) continue;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float sum = l[w][k];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    if (t4 == 0) {
                        stats[warp * 32 + g + 8 * k] = m[w][k];
                        stats[warp * 32 + 16 + g + 8 * k] = sum;
                    }
                }
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) share[(warp * 16 + g + 8 * (e >> 1)) * DP + 8 * n + 2 * t4 + (e & 1)] = o[w][n][e];
            }
        }
        __syncthreads();
        if (warp < 4) {
            for (int r = warp; r < 16 && 16 * mt + r < F.rows; r += 4) {
                const int row = 16 * mt + r, i = row % nq, h = hk * group + row / nq;
                float top = -INFINITY, sum = 0.f, by[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) top = fmaxf(top, stats[w * 32 + r]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float mw = stats[w * 32 + r];
                    by[w] = mw == -INFINITY ? (stats[w * 32 + 16 + r] == 0.f ? 0.f : 1.f) : exp2_fast((mw - top) * F.scale_log2);
                    sum += by[w] * stats[w * 32 + 16 + r];
                }
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const float lse = sum == 0.f ? -INFINITY : (top * F.scale_log2 - N::kLift + log2f(sum)) * 0.69314718055994531f;
                const long long flat = (P.Hq * (long long)b + h) * P.Nq + i;
                if (lane == 0) {
                    if (F.splits > 1) F.part_lse[split * all_rows + flat] = lse;
                    else if (P.lse) static_cast<float *>(P.lse)[flat] = lse;
                }
                for (int d = lane * 2; d < D; d += 64) {
                    float x = 0.f, y = 0.f;
                    if (sum != 0.f)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 z = *reinterpret_cast<const float2 *>(share + (w * 16 + r) * DP + d);
                            x += by[w] * z.x;
                            y += by[w] * z.y;
                        }
                    if (F.splits > 1) *reinterpret_cast<float2 *>(F.part_out + (split * all_rows + flat) * D + d) = make_float2(x * inv, y * inv);
                    else {
                        const long long to = ((b * P.Nq + i) * P.Hq + h) * P.D + d;
                        *reinterpret_cast<uint32_t *>(static_cast<T *>(P.out) + to) = N::pack(x * inv, y * inv);
                        if (P.rest) *reinterpret_cast<uint32_t *>(static_cast<T *>(P.rest) + to) = N::rest(x * inv, y * inv);
                    }
                }
            }
        }
    }
}

// out = sum_s w_s out_s, w_s = exp(lse_s - lse), lse = log sum_s exp(lse_s).  WARPS of a block's eight share a row: one, or all of them where the
// ranges are many.  A lane holds the weight of every 32nd range; the ranges' outputs are fetched four at a time, none waiting for
// another (one after the other they took 8 us for 10 ranges of 512 rows).  The order of the sums follows from the sizes alone.
template <typename T, int WARPS>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams P, const float *part_out, const float *part_lse, int splits) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % WARPS, D = (int)P.D;
    const long long rows = P.B * P.Hq * P.Nq, row = (long long)blockIdx.x * (8 / WARPS) + warp / WARPS;
    if (row >= rows) return;   // the whole block, or whole rows
    const float log2e = 1.4426950408889634f;
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) {
        const float x = part_lse[s * rows + row];
        top = x > top || x != x ? x : top;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, top, d);
        top = x > top || x != x ? x : top;
    }
    float sum = 0.f, x[2] = {}, y[2] = {};
    for (int s0 = 32 * share; s0 < splits; s0 += 32 * WARPS) {
        const float mine = s0 + lane < splits ? part_lse[(s0 + lane) * rows + row] : -INFINITY;
        const float w = mine == -INFINITY ? 0.f : exp2f((mine - top) * log2e);
        sum += w;
        const unsigned written = __ballot_sync(0xffffffffu, mine != -INFINITY);   // the others' outputs were not
        const int n = splits - s0 < 32 ? splits - s0 : 32;
        for (int s = 0; s < n; s += 4) {
            float2 z[4][2];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int d = lane * 2 + 64 * k;
                    z[u][k] = d < D && (written >> (s + u)) & 1 ? *reinterpret_cast<const float2 *>(part_out + ((s0 + s + u) * rows + row) * D + d) : make_float2(0.f, 0.f);
                }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float ws = __shfl_sync(0xffffffffu, w, s + u);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    x[k] += ws * z[u][k].x;
                    y[k] += ws * z[u][k].y;
                }
            }
        }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if constexpr (WARPS > 1) {
        __shared__ float parts[WARPS][5][32];
        const float mine[5] = {x[0], y[0], x[1], y[1], sum};
#pragma unroll
        for (int k = 0; k < 5; ++k) parts[share][k][lane] = mine[k];
        __syncthreads();
        if (share != 0) return;
        x[0] = x[1] = y[0] = y[1] = sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            x[0] += parts[w][0][lane];
            y[0] += parts[w][1][lane];
            x[1] += parts[w][2][lane];
            y[1] += parts[w][3][lane];
            sum += parts[w][4][lane];
        }
    }
    const long long bh = row / P.Nq, i = row % P.Nq, h = bh % P.Hq, b = bh / P.Hq;
    const long long to = ((b * P.Nq + i) * P.Hq + h) * P.D;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int d = lane * 2 + 64 * k;
        if (d >= D) continue;
        T *out = static_cast<T *>(P.out) + to + d;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float2 *>(out) = make_float2(x[k] * inv, y[k] * inv);
        } else {
            *reinterpret_cast<uint32_t *>(out) = Narrow<T>::pack(x[k] * inv, y[k] * inv);
            if (P.rest) *reinterpret_cast<uint32_t *>(static_cast<T *>(P.rest) + to + d) = Narrow<T>::rest(x[k] * inv, y[k] * inv);
        }
    }
    if (lane == 0 && P.lse) static_cast<float *>(P.lse)[row] = sum == 0.f ? -INFINITY : top + logf(sum);
}

template <typename T, int BLOCKS, int MT> int launch(const FewParams &F, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    typedef FewSmem<BLOCKS> L;
    const long long blocks = F.a.B * F.a.Hk * F.splits;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    constexpr auto *kern = &attention_few_kernel<T, BLOCKS, MT>;
    if (const int e = allow_shared_memory<kern>((int)L::ALLOC)) return e;
    kern<<<(unsigned)blocks, kFewThreads, L::ALLOC, s>>>(k, v, F);
    TPW_LAUNCH_OK("attention_few_kernel");
    return TPW_OK;
}
template <typename T> int launch_width(const FewParams &F, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    if (F.a.D <= 64) return F.rows <= 16 ? launch<T, 1, 1>(F, k, v, s) : launch<T, 1, 2>(F, k, v, s);
    return F.rows <= 16 ? launch<T, 2, 1>(F, k, v, s) : launch<T, 2, 2>(F, k, v, s);
}

// Keys of a range: so many that the ranges of full-length sequences make about four turns of two CTAs on every SM (ragged lengths and
// windows leave ranges empty, which then cost nothing), at least 512, whose 3 us are what the join and its launch cost, and no more ranges of a
// sequence than CTAs at a time.
int keys_per_split(const AttnParams &P) {
    const long long slots = 2LL * sm_count(), want = P.B * P.Hk * P.Nk / (4 * slots), least = (P.Nk + slots - 1) / slots;
    const long long keys = want > least ? want : least, whole = (P.Nk + STEP - 1) / STEP * STEP;
    const long long r = ((keys < 512 ? 512 : keys) + STEP - 1) / STEP * STEP;
    return (int)(r < whole ? r : whole);
}

} // namespace

bool attn_few_fits(int dtype, const AttnParams &P) { return attn_tc_fits(dtype, P) && P.group * P.Nq <= 32; }

AttnSplits attn_few_splits(const AttnParams &P) {
    AttnSplits r;
    r.keys = keys_per_split(P);
    r.count = (int)((P.Nk + r.keys - 1) / r.keys);
    return r;
}

int attn_few_forward(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    FewParams F = {};
    F.a = P;
    F.a.status = device_status_ptr();
    F.scale_log2 = (float)(P.scale * 1.4426950408889634074);
    F.rows = (int)(P.group * P.Nq);
    F.splits = splits.count;
    F.keys_per_split = splits.keys;
    F.part_out = splits.out;
    F.part_lse = splits.lse;
    CUtensorMap k, v;
    int e = make_tensor_map_heads(&k, P.k, P.D, P.Nk, P.Hk, P.B, 2 * P.k_s[1], 2 * P.k_s[2], 2 * P.k_s[0], STEP);
    if (e == TPW_OK) e = make_tensor_map_heads(&v, P.v, P.D, P.Nk, P.Hk, P.B, 2 * P.v_s[1], 2 * P.v_s[2], 2 * P.v_s[0], STEP);
    if (e != TPW_OK) return e;
    return dtype == TPW_F16 ? launch_width<__half>(F, k, v, s) : launch_width<__nv_bfloat16>(F, k, v, s);
}

template <typename T> static int join(const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    const long long rows = P.B * P.Hq * P.Nq, blocks = splits.count > 32 ? rows : (rows + 7) / 8;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    if (splits.count > 32) attention_join_kernel<T, 8><<<(unsigned)blocks, 256, 0, s>>>(P, splits.out, splits.lse, splits.count);
    else attention_join_kernel<T, 1><<<(unsigned)blocks, 256, 0, s>>>(P, splits.out, splits.lse, splits.count);
    TPW_LAUNCH_OK("attention_join_kernel");
    return TPW_OK;
}
int attn_join(int dtype, const AttnParams &P, const AttnSplits &splits, cudaStream_t s) {
    return dtype == TPW_F16 ? join<__half>(P, splits, s) : dtype == TPW_F32 ? join<float>(P, splits, s) : join<__nv_bfloat16>(P, splits, s);
}

} // namespace tpw
