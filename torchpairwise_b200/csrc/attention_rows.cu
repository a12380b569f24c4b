// What both gradient walks need of each query row, formed once: delta_i = dO_i . out_i - dlse_i (out with what rounding took from it), and the forward's lse_i, +inf for a
// row that sees nothing (every probability is then exp(-inf) = 0), as powers of two for 32-bit walks.  The tensor-core walks add
// rather than subtract: they get -delta_i and lift - lse_i.  Rows are padded to whole tiles of 128 as rows that see nothing.
// Reads dO and out (16-bit types: and what rounding took from it) once, which is what HBM would need 31 us for in bfloat16 [1, 8192, 32, 128], 201 MB; it takes
// 57, 3.5 TB/s, bound by latency: the loads of a row, its shuffles and its one store come one after the other.  Four rows a thread on their way instead of two (92 us) and tokens of all heads side by
// side (71 us) were slower.
//
// Half precision also needs three maxima: the tensor-core walks round exp(s - lse) and ds = p (dO . v - delta) to the inputs' type, whose numbers end
// at 65504 and lose digits below 2^-14.  |ds| <= p (|dO| (|v| + |out|) + |dlse|) <= p (2 max|dO| max|v| + max|dlse|), from which the walks take a power of two that
// brings ds to the top of the range.  The maxima are those of a query head (dO, dlse) and of a key head (v) of one sequence, so that no sequence's gradients
// depend on what else is in the batch.  A maximum does not depend on the order of its atomics.
#include "attention.cuh"

#include <type_traits>

namespace tpw {
namespace {

template <typename T, int V> struct alignas(sizeof(T) * V) Piece { T v[V]; };

constexpr int kTurns = 2;
// largest |v_j|^2 of the keys that are used
template <int V, int LANES> __device__ __forceinline__ void value_norms(const AttnParams &P, unsigned block) {
    constexpr int ROWS = 8 * (32 / LANES) * kTurns;
    const unsigned tiles = (unsigned)((P.Nk + ROWS - 1) / ROWS), bh = block / tiles;
    const int D = (int)P.D, h = (int)(bh % (unsigned)P.Hk), part = threadIdx.x % LANES;
    const long long b = bh / (unsigned)P.Hk, j0 = (long long)(block % tiles) * ROWS + threadIdx.x / LANES;
    const __half *v = static_cast<const __half *>(P.v) + b * P.v_s[0] + h * P.v_s[2];
    long long length = P.key_lengths ? P.key_lengths[b] : P.Nk;
    length = length < P.Nk ? length : P.Nk;
    float sq[kTurns] = {};
    for (int d = part * V; d < D; d += LANES * V) {
        Piece<__half, V> x[kTurns] = {};
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const long long j = j0 + t * (256 / LANES);
            if (j < length) x[t] = *reinterpret_cast<const Piece<__half, V> *>(v + j * P.v_s[1] + d);
        }
#pragma unroll
        for (int t = 0; t < kTurns; ++t)
#pragma unroll
            for (int e = 0; e < V; ++e) sq[t] += (float)x[t].v[e] * (float)x[t].v[e];
    }
    unsigned top = 0;
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) sq[t] += __shfl_xor_sync(0xffffffffu, sq[t], d);
        top = max(top, __float_as_uint(fabsf(sq[t])));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0 && top) atomicMax(P.row_max + 2 * P.B * P.Hq + bh, top);
}

// A block takes consecutive tokens of one head.  LANES threads read one row V elements at a time, a warp 32 / LANES rows side by side and
// kTurns times in a row, so that 2 * kTurns loads are in flight.
template <typename T, int V, int LANES>
__global__ void __launch_bounds__(256, 4) attention_rows_kernel(const AttnParams P, double units, double lift, double sign, unsigned row_blocks) {
    typedef typename AttnAcc<T>::type A;
    if constexpr (std::is_same_v<T, __half>)
        if (blockIdx.x >= row_blocks) {
            value_norms<V, LANES>(P, blockIdx.x - row_blocks);
            return;
        }
    constexpr int ROWS = 8 * (32 / LANES) * kTurns;   // of a block
    constexpr bool kHalf = std::is_same_v<T, __half>;
    const unsigned tiles = (unsigned)((P.Nqp + ROWS - 1) / ROWS), bh = blockIdx.x / tiles;
    const int D = (int)P.D, h = (int)(bh % (unsigned)P.Hq), part = threadIdx.x % LANES;
    const long long b = bh / (unsigned)P.Hq, i0 = (long long)(blockIdx.x % tiles) * ROWS + threadIdx.x / LANES;
    const T *out = static_cast<const T *>(P.out) + (b * P.Nq * P.Hq + h) * P.D, *dout = static_cast<const T *>(P.dout) + b * P.do_s[0] + h * P.do_s[2];
    const T *rest = P.rest ? static_cast<const T *>(P.rest) + (b * P.Nq * P.Hq + h) * P.D : nullptr;
    A *lse = static_cast<A *>(P.row_lse), *delta = static_cast<A *>(P.row_delta);
    A dot[kTurns] = {}, sq[kTurns] = {}, m[kTurns], more[kTurns];
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {   // on their way beside the rows
        const long long i = i0 + t * (256 / LANES);
        const bool own = part == 0 && i < P.Nq;
        m[t] = own ? static_cast<const A *>(P.lse)[bh * P.Nq + i] : -(A)INFINITY;
        more[t] = own && P.dlse ? static_cast<const A *>(P.dlse)[bh * P.Nq + i] : (A)0;
    }
#pragma unroll 1
    for (int d = part * V; d < D; d += LANES * V) {
        Piece<T, V> x[kTurns] = {}, y[kTurns] = {}, z[kTurns] = {};
#pragma unroll
        for (int t = 0; t < kTurns; ++t) {
            const long long i = i0 + t * (256 / LANES);
            if (i < P.Nq) {
                x[t] = *reinterpret_cast<const Piece<T, V> *>(out + i * P.Hq * P.D + d);
                y[t] = *reinterpret_cast<const Piece<T, V> *>(dout + i * P.do_s[1] + d);
                if (sizeof(T) == 2 && rest) z[t] = *reinterpret_cast<const Piece<T, V> *>(rest + i * P.Hq * P.D + d);
            }
        }
#pragma unroll
        for (int t = 0; t < kTurns; ++t)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                dot[t] += (sizeof(T) == 2 ? (A)x[t].v[e] + (A)z[t].v[e] : (A)x[t].v[e]) * (A)y[t].v[e];
                if (kHalf) sq[t] += (A)y[t].v[e] * (A)y[t].v[e];
            }
    }
    unsigned top = 0, top_more = 0;
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) {
            dot[t] += __shfl_xor_sync(0xffffffffu, dot[t], d);
            if (kHalf) sq[t] += __shfl_xor_sync(0xffffffffu, sq[t], d);
        }
        const long long i = i0 + t * (256 / LANES);
        if (part != 0 || i >= P.Nqp) continue;
        const bool sees = m[t] != -(A)INFINITY;
        lse[bh * P.Nqp + i] = sees ? m[t] * (A)units + (A)lift : (A)(sign * INFINITY);
        delta[bh * P.Nqp + i] = sees ? (A)sign * (dot[t] - more[t]) : (A)0;
        if (kHalf && P.row_max && sees) {
            top = max(top, __float_as_uint(fabsf((float)sq[t])));
            top_more = max(top_more, __float_as_uint(fabsf((float)more[t])));
        }
    }
    if (kHalf && P.row_max) {
        top = __reduce_max_sync(0xffffffffu, top);
        top_more = __reduce_max_sync(0xffffffffu, top_more);
        if ((threadIdx.x & 31) == 0) {
            if (top) atomicMax(P.row_max + 2 * bh, top);
            if (top_more) atomicMax(P.row_max + 2 * bh + 1, top_more);
        }
    }
}

template <typename T, int V, int LANES>
int launch(const AttnParams &P, double units, double lift, double sign, cudaStream_t s) {
    constexpr int ROWS = 8 * (32 / LANES) * kTurns;
    const long long blocks = (P.Nqp + ROWS - 1) / ROWS * P.Hq * P.B, values = P.row_max ? (P.Nk + ROWS - 1) / ROWS * P.Hk * P.B : 0;
    TPW_CHECK_ARG(blocks + values < (1LL << 31), "attention: more than 2^31 blocks of work");
    attention_rows_kernel<T, V, LANES><<<(unsigned)(blocks + values), 256, 0, s>>>(P, units, lift, sign, (unsigned)blocks);
    TPW_LAUNCH_OK("attention_rows_kernel");
    return TPW_OK;
}

template <typename T> int rows(const AttnParams &P, double units, double lift, double sign, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);   // elements of 16 bytes
    auto wide = [&](const void *p, const long long (&st)[3]) { return aligned16(p) && st[0] % W == 0 && st[1] % W == 0 && st[2] % W == 0; };
    const long long dense[3] = {P.D, P.D, P.D};
    if (P.D % W != 0 || !wide(P.out, dense) || !aligned16(P.rest) || !wide(P.dout, P.do_s) || (P.row_max && !wide(P.v, P.v_s))) return launch<T, 1, 32>(P, units, lift, sign, s);
    const long long pieces = P.D / W;
    if (pieces <= 8) return launch<T, W, 8>(P, units, lift, sign, s);
    if (pieces <= 16) return launch<T, W, 16>(P, units, lift, sign, s);
    return launch<T, W, 32>(P, units, lift, sign, s);
}

} // namespace

// [B, Hq] pairs of largest |dO_i|^2 and |dlse_i|, then [B, Hk] of largest |v_j|^2, as the bits of floats
static long long maxima_bytes(int dtype, const AttnParams &P) { return dtype == TPW_F16 ? (4 * P.B * (2 * P.Hq + P.Hk) + 15) / 16 * 16 : 0; }
long long attn_rows_bytes(int dtype, const AttnParams &P) {
    return maxima_bytes(dtype, P) + 2 * P.B * P.Hq * P.Nqp * (dtype == TPW_F64 ? 8 : 4);
}

int attn_rows(int dtype, AttnParams &P, void *scratch, bool tensor, cudaStream_t s) {
    P.row_lse = static_cast<unsigned char *>(scratch) + maxima_bytes(dtype, P);
    P.row_delta = static_cast<unsigned char *>(P.row_lse) + P.B * P.Hq * P.Nqp * (dtype == TPW_F64 ? 8 : 4);
    const double log2e = 1.4426950408889634074;
    if (dtype == TPW_F64) return rows<double>(P, 1.0, 0.0, 1.0, s);
    if (dtype == TPW_F32) return rows<float>(P, log2e, 0.0, 1.0, s);
    if (dtype == TPW_BF16) return rows<__nv_bfloat16>(P, tensor ? -log2e : log2e, 0.0, tensor ? -1.0 : 1.0, s);
    if (!tensor) return rows<__half>(P, log2e, 0.0, 1.0, s);
    P.row_max = static_cast<unsigned *>(scratch);
    TPW_CUDA_OK(cudaMemsetAsync(P.row_max, 0, maxima_bytes(dtype, P), s));
    return rows<__half>(P, -log2e, 12.0, -1.0, s);
}

} // namespace tpw
