// What both gradient walks need of each query row, formed once: delta_i = dO_i . out_i - dlse_i, and the forward's lse_i, +inf for a
// row that sees nothing (every probability is then exp(-inf) = 0), as powers of two for 32-bit walks.  The tensor-core walks add
// rather than subtract: they get -delta_i and lift - lse_i.  Rows are padded to whole tiles of 128 as rows that see nothing.
// Bound by HBM: reads dO and out once.  One warp per row.
//
// Half precision also needs three maxima: the tensor-core walks round exp(s - lse) and ds = p (dO . v - delta) to the inputs' type, whose numbers end
// at 65504 and lose digits below 2^-14.  |ds| <= p (|dO| (|v| + |out|) + |dlse|) <= p (2 max|dO| max|v| + max|dlse|), from which the walks take a power of two that
// brings ds to the top of the range.  A maximum does not depend on the order of its atomics.
#include "attention.cuh"

namespace tpw {
namespace {

template <typename T, int V> struct alignas(sizeof(T) * V) Piece { T v[V]; };
template <typename A> __device__ __forceinline__ A warp_sum(A x) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

template <typename T, int V>
__global__ void __launch_bounds__(256) attention_rows_kernel(const AttnParams P, double units, double lift, double sign, unsigned *row_max) {
    typedef typename AttnAcc<T>::type A;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= P.B * P.Hq * P.Nqp) return;
    const long long i = row % P.Nqp, bh = row / P.Nqp, h = bh % P.Hq, b = bh / P.Hq;
    A *lse = static_cast<A *>(P.row_lse), *delta = static_cast<A *>(P.row_delta);
    if (i >= P.Nq) {
        if (lane == 0) {
            lse[row] = (A)(sign * INFINITY);
            delta[row] = 0;
        }
        return;
    }
    const T *o = static_cast<const T *>(P.out) + ((b * P.Nq + i) * P.Hq + h) * P.D;
    const T *g = static_cast<const T *>(P.dout) + b * P.do_s[0] + i * P.do_s[1] + h * P.do_s[2];
    A dot = 0, sq = 0;
    for (int d = lane * V; d < P.D; d += 32 * V) {
        const Piece<T, V> x = *reinterpret_cast<const Piece<T, V> *>(o + d), y = *reinterpret_cast<const Piece<T, V> *>(g + d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            dot += (A)x.v[e] * (A)y.v[e];
            sq += (A)y.v[e] * (A)y.v[e];
        }
    }
    dot = warp_sum(dot);
    const A m = static_cast<const A *>(P.lse)[bh * P.Nq + i];
    const bool sees = m != -(A)INFINITY;
    const A more = P.dlse ? static_cast<const A *>(P.dlse)[bh * P.Nq + i] : (A)0;
    if (lane == 0) {
        lse[row] = sees ? m * (A)units + (A)lift : (A)(sign * INFINITY);
        delta[row] = sees ? (A)sign * (dot - more) : (A)0;
    }
    if (row_max) {
        sq = warp_sum(sq);
        if (lane == 0 && sees) {
            atomicMax(row_max, __float_as_uint(fabsf((float)sq)));
            if (P.dlse) atomicMax(row_max + 2, __float_as_uint(fabsf((float)more)));
        }
    }
}

template <int V>
__global__ void __launch_bounds__(256) attention_value_norm_kernel(const AttnParams P, unsigned *row_max) {
    const int lane = threadIdx.x & 31;
    float top = 0.f;
    for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < P.B * P.Nk * P.Hk; row += (long long)gridDim.x * 8) {
        const long long h = row % P.Hk, bj = row / P.Hk, j = bj % P.Nk, b = bj / P.Nk;
        if (P.key_lengths && j >= P.key_lengths[b]) continue;
        const __half *v = static_cast<const __half *>(P.v) + b * P.v_s[0] + j * P.v_s[1] + h * P.v_s[2];
        float sq = 0.f;
        for (int d = lane * V; d < P.D; d += 32 * V) {
            const Piece<__half, V> x = *reinterpret_cast<const Piece<__half, V> *>(v + d);
#pragma unroll
            for (int e = 0; e < V; ++e) sq += (float)x.v[e] * (float)x.v[e];
        }
        sq = warp_sum(sq);
        top = sq > top || sq != sq ? sq : top;
    }
    if (lane == 0) atomicMax(row_max, __float_as_uint(fabsf(top)));
}

template <typename T> int rows(AttnParams &P, double units, double lift, double sign, unsigned *row_max, cudaStream_t s) {
    constexpr int W = sizeof(T) == 8 ? 2 : 4;
    auto wide = [&](const void *p, const long long (&st)[3]) {
        return reinterpret_cast<uintptr_t>(p) % (W * sizeof(T)) == 0 && st[0] % W == 0 && st[1] % W == 0 && st[2] % W == 0;
    };
    const long long dense[3] = {P.D, P.D, P.D};
    const long long blocks = (P.B * P.Hq * P.Nqp + 7) / 8;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    if (P.D % W == 0 && wide(P.out, dense) && wide(P.dout, P.do_s)) attention_rows_kernel<T, W><<<(unsigned)blocks, 256, 0, s>>>(P, units, lift, sign, row_max);
    else attention_rows_kernel<T, 1><<<(unsigned)blocks, 256, 0, s>>>(P, units, lift, sign, row_max);
    TPW_LAUNCH_OK("attention_rows_kernel");
    if (row_max && P.Nk > 0) {
        const long long want = (P.B * P.Nk * P.Hk + 7) / 8, most = 16LL * sm_count();
        const unsigned grid = (unsigned)(want < most ? want : most);
        if (P.D % W == 0 && wide(P.v, P.v_s)) attention_value_norm_kernel<W><<<grid, 256, 0, s>>>(P, row_max + 1);
        else attention_value_norm_kernel<1><<<grid, 256, 0, s>>>(P, row_max + 1);
        TPW_LAUNCH_OK("attention_value_norm_kernel");
    }
    return TPW_OK;
}

} // namespace

long long attn_rows_bytes(int dtype, const AttnParams &P) {
    return 16 + 2 * P.B * P.Hq * P.Nqp * (dtype == TPW_F64 ? 8 : 4);
}

int attn_rows(int dtype, AttnParams &P, void *scratch, bool tensor, cudaStream_t s) {
    unsigned *row_max = static_cast<unsigned *>(scratch);
    P.row_lse = static_cast<unsigned char *>(scratch) + 16;
    P.row_delta = static_cast<unsigned char *>(P.row_lse) + P.B * P.Hq * P.Nqp * (dtype == TPW_F64 ? 8 : 4);
    const double log2e = 1.4426950408889634074;
    if (dtype == TPW_F64) return rows<double>(P, 1.0, 0.0, 1.0, nullptr, s);
    if (dtype == TPW_F32) return rows<float>(P, log2e, 0.0, 1.0, nullptr, s);
    if (dtype == TPW_BF16) return rows<__nv_bfloat16>(P, tensor ? -log2e : log2e, 0.0, tensor ? -1.0 : 1.0, nullptr, s);
    if (!tensor) return rows<__half>(P, log2e, 0.0, 1.0, nullptr, s);
    TPW_CUDA_OK(cudaMemsetAsync(row_max, 0, 16, s));
    P.row_max = row_max;
    return rows<__half>(P, -log2e, 12.0, -1.0, row_max, s);
}

} // namespace tpw
