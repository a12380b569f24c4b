// Attention and its gradients on the CUDA cores: every type, head width up to 256 and stride.  float64 always runs here; the other types where
// the tensor-core kernels' rules on layout and width are not met.
//
// Forward: one pass over the keys with a running maximum m and sum l of every row; a tile's probabilities exp(s - m) are
// multiplied into the output accumulators, which are scaled by exp(m_old - m_new) whenever the maximum moves.
// Backward: p_ij = exp(s_ij - lse_i) is formed anew, ds_ij = p_ij (dO_i . v_j - delta_i).  One walk over the queries per key
// tile (dk, dv; all heads that share the key head one after the other, so their sum has a fixed order) and one over the keys per
// query tile (dq); no atomics, the same bits each time.
//
// Bound by FP32 issue and by shared-memory reads: 2 D lane-operations per pair forward, 7 D backward; a 16-byte read takes four
// wavefronts, whether lanes share addresses or not, so an 8 x 8 block of a thread reads 64 wavefronts per 64 clocks of FMAs, and a
// 4 x 4 block twice as many.  16 x TX threads; up to 64 features TX = 8, whose blocks are 8 rows by 8 columns of what a product
// writes.  All operand tiles lie row-major with 4 elements of padding, so that products that contract the
// features read four features of a row at once (eight rows in eight bank groups) and products that contract tokens four features of
// one token.
#include "attention.cuh"

namespace tpw {
namespace {

constexpr int PAD = 4;

template <typename A> struct alignas(sizeof(A) * 4) Four { A v[4]; };

template <typename T> __device__ __forceinline__ typename AttnAcc<T>::type up(T v) { return (typename AttnAcc<T>::type)v; }

// exp(x scale - lse) in units where it costs least: float in powers of two (scale and lse carry the factor log2 e)
__device__ __forceinline__ float power(float x) { return exp2f(x); }
__device__ __forceinline__ double power(double x) { return exp(x); }
template <typename A> __device__ __forceinline__ A scale_of(const AttnParams &P);
template <> __device__ __forceinline__ float scale_of<float>(const AttnParams &P) { return (float)(P.scale * 1.4426950408889634074); }
template <> __device__ __forceinline__ double scale_of<double>(const AttnParams &P) { return P.scale; }
__device__ __forceinline__ float natural(float x) { return x * 0.69314718055994531f; }
__device__ __forceinline__ double natural(double x) { return x; }
__device__ __forceinline__ float log_of(float x) { return logf(x); }
__device__ __forceinline__ double log_of(double x) { return log(x); }
template <typename A> __device__ __forceinline__ A minus_infinity() { return -(A)INFINITY; }
template <typename A> __device__ __forceinline__ A max_of(A a, A b) { return a > b ? a : b; }

// Rows [row0, row0 + ROWS) of a [tokens, D] slice, widened, zero beyond `rows` and D.  `vec`: rows may be read four elements at a time.
template <typename T, typename A, int ROWS, int DP, int THREADS>
__device__ __forceinline__ void load_tile(A *dst, const T *src, long long stride, int row0, int rows, int D, bool vec) {
    constexpr int PER = DP / 4;
#pragma unroll 4
    for (int c = threadIdx.x; c < ROWS * PER; c += THREADS) {
        const int r = c / PER, d = (c % PER) * 4;
        Four<A> w = {};
        if (row0 + r < rows && d < D) {
            const T *p = src + (long long)(row0 + r) * stride + d;
            if (vec) {
                struct alignas(sizeof(T) * 4) Raw { T v[4]; };
                const Raw raw = *reinterpret_cast<const Raw *>(p);
#pragma unroll
                for (int e = 0; e < 4; ++e) w.v[e] = up(raw.v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < D) w.v[e] = up(p[e]);
            }
        }
        *reinterpret_cast<Four<A> *>(dst + r * (DP + PAD) + d) = w;
    }
}

// acc[m][n] = X[ty * RM + m] . Y[tx + TX n], contracting DP features
template <typename A, int RM, int RN, int DP, int TX>
__device__ __forceinline__ void product_nt(A (&acc)[RM][RN], const A *X, const A *Y, int ty, int tx) {
#pragma unroll
    for (int m = 0; m < RM; ++m)
#pragma unroll
        for (int n = 0; n < RN; ++n) acc[m][n] = 0;
#pragma unroll 2
    for (int d = 0; d < DP; d += 4) {
        Four<A> y[RN];
#pragma unroll
        for (int n = 0; n < RN; ++n) y[n] = *reinterpret_cast<const Four<A> *>(Y + (tx + TX * n) * (DP + PAD) + d);
#pragma unroll
        for (int m = 0; m < RM; ++m) {
            const Four<A> x = *reinterpret_cast<const Four<A> *>(X + (ty * RM + m) * (DP + PAD) + d);
#pragma unroll
            for (int n = 0; n < RN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][n] += x.v[e] * y[n].v[e];
        }
    }
}

// acc[m][4 c + e] += sum_j P[ty * RM + m][j] Y[j][4 TX c + 4 tx + e], contracting COLS tokens
template <typename A, int RM, int COLS, int DP, int TX>
__device__ __forceinline__ void product_nn(A (&acc)[RM][DP / TX], const A *P, const A *Y, int ty, int tx) {
#pragma unroll 1
    for (int j = 0; j < COLS; j += 4) {
        Four<A> p[RM];
#pragma unroll
        for (int m = 0; m < RM; ++m) p[m] = *reinterpret_cast<const Four<A> *>(P + (ty * RM + m) * (COLS + PAD) + j);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int c = 0; c < DP / (4 * TX); ++c) {
                const Four<A> y = *reinterpret_cast<const Four<A> *>(Y + (j + jj) * (DP + PAD) + 4 * TX * c + 4 * tx);
#pragma unroll
                for (int m = 0; m < RM; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][4 * c + e] += p[m].v[jj] * y.v[e];
            }
    }
}

// A factor of 0 is a row that sees nothing: zero, although its sums are 0 times what need not be finite.
template <typename T, typename A, int RM, int DP, int TX>
__device__ __forceinline__ void store_rows(T *dst, T *rest, long long row_stride, const A (&acc)[RM][DP / TX], const A (&factor)[RM], int row0, int rows, int D,
                                           int ty, int tx) {
#pragma unroll
    for (int m = 0; m < RM; ++m) {
        const int r = row0 + ty * RM + m;
        if (r >= rows) continue;
#pragma unroll
        for (int c = 0; c < DP / (4 * TX); ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * TX * c + 4 * tx + e;
                if (d >= D) continue;
                const A x = factor[m] == 0 ? (A)0 : acc[m][4 * c + e] * factor[m];
                dst[(long long)r * row_stride + d] = (T)x;
                if constexpr (sizeof(T) == 2)
                    if (rest) rest[(long long)r * row_stride + d] = rest_of<T>(x);
            }
    }
}

template <typename T> __device__ __forceinline__ bool in_fours(const void *p, const long long (&s)[3], long long D) {
    return (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T))) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0 && D % 4 == 0;
}

template <typename T, typename A, int DP, int BM, int BN, int TX>
__global__ void __launch_bounds__(16 * TX) attention_forward_simple_kernel(const AttnParams P, int tiles) {
    constexpr int RM = BM / 16, RN = BN / TX, THREADS = 16 * TX;
    extern __shared__ __align__(32) unsigned char smem[];
    A *Q = reinterpret_cast<A *>(smem), *K = Q + BM * (DP + PAD), *V = K + BN * (DP + PAD), *S = V + BN * (DP + PAD);
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    long long at = blockIdx.x;
    const int tile = (int)(P.causal ? tiles - 1 - at % tiles : at % tiles);   // the longest rows of a causal call first
    at /= tiles;
    const long long h = at % P.Hq, b = at / P.Hq, hk = h / P.group;
    const Seen see(P, b);
    const int row0 = tile * BM, nq = (int)P.Nq, D = (int)P.D;
    const T *q = static_cast<const T *>(P.q) + b * P.q_s[0] + h * P.q_s[2];
    const T *k = static_cast<const T *>(P.k) + b * P.k_s[0] + hk * P.k_s[2];
    const T *v = static_cast<const T *>(P.v) + b * P.v_s[0] + hk * P.v_s[2];
    const bool kvec = in_fours<T>(P.k, P.k_s, P.D), vvec = in_fours<T>(P.v, P.v_s, P.D);
    load_tile<T, A, BM, DP, THREADS>(Q, q, P.q_s[1], row0, nq, D, in_fours<T>(P.q, P.q_s, P.D));
    const A scale = scale_of<A>(P);
    const int last = row0 + BM < nq ? row0 + BM - 1 : nq - 1;
    const int j_lo = see.lo(row0) / BN * BN, j_hi = see.hi(last);
    A m[RM], l[RM], O[RM][DP / TX];
    int lo[RM], hi[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        m[r] = minus_infinity<A>();
        l[r] = 0;
        const int i = row0 + ty * RM + r;
        lo[r] = see.lo(i);
        hi[r] = i < nq ? see.hi(i) : 0;
#pragma unroll
        for (int c = 0; c < DP / TX; ++c) O[r][c] = 0;
    }
    for (int j0 = j_lo; j0 < j_hi; j0 += BN) {
        __syncthreads();
        load_tile<T, A, BN, DP, THREADS>(K, k, P.k_s[1], j0, see.length, D, kvec);
        load_tile<T, A, BN, DP, THREADS>(V, v, P.v_s[1], j0, see.length, D, vvec);
        __syncthreads();
        A s[RM][RN];
        product_nt<A, RM, RN, DP, TX>(s, Q, K, ty, tx);
#pragma unroll
        for (int r = 0; r < RM; ++r) {
            A top = minus_infinity<A>();
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const int j = j0 + tx + TX * n;
                s[r][n] = j >= lo[r] && j < hi[r] ? s[r][n] * scale : minus_infinity<A>();
                top = max_of(top, s[r][n]);
            }
#pragma unroll
            for (int d = TX / 2; d >= 1; d >>= 1) top = max_of(top, __shfl_xor_sync(0xffffffffu, top, d));
            const A m_new = max_of(m[r], top);
            const A base = m_new == minus_infinity<A>() ? (A)0 : m_new;   // nothing seen so far: every power below is 0
            const A rescale = power(m[r] - base);
            A sum = 0;
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const A p = power(s[r][n] - base);
                sum += p;
                S[(ty * RM + r) * (BN + PAD) + tx + TX * n] = p;
            }
            l[r] = l[r] * rescale + sum;
            m[r] = m_new;
#pragma unroll
            for (int c = 0; c < DP / TX; ++c) O[r][c] *= rescale;
        }
        __syncwarp();   // a row's probabilities are written and read by the same half warp
        product_nn<A, RM, BN, DP, TX>(O, S, V, ty, tx);
    }
    A inv[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
#pragma unroll
        for (int d = TX / 2; d >= 1; d >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
        inv[r] = l[r] == 0 ? (A)0 : 1 / l[r];
        const int i = row0 + ty * RM + r;
        if (P.lse && tx == 0 && i < nq)
            static_cast<A *>(P.lse)[(b * P.Hq + h) * P.Nq + i] = l[r] == 0 ? minus_infinity<A>() : natural(m[r]) + log_of(l[r]);
    }
    const long long to = (b * P.Nq * P.Hq + h) * P.D;
    store_rows<T, A, RM, DP, TX>(static_cast<T *>(P.out) + to, P.rest ? static_cast<T *>(P.rest) + to : nullptr, P.Hq * P.D, O, inv, row0, nq, D, ty, tx);
}

// dk, dv of BK keys: rows are keys, columns queries
template <typename T, typename A, int DP, int BK, int BQ, int TX>
__global__ void __launch_bounds__(16 * TX) attention_dkv_simple_kernel(const AttnParams P, int tiles) {
    constexpr int RM = BK / 16, RN = BQ / TX, THREADS = 16 * TX;
    extern __shared__ __align__(32) unsigned char smem[];
    A *K = reinterpret_cast<A *>(smem), *V = K + BK * (DP + PAD), *Q = V + BK * (DP + PAD), *G = Q + BQ * (DP + PAD),
      *S = G + BQ * (DP + PAD);
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    long long at = blockIdx.x;
    const int tile = (int)(at % tiles);
    at /= tiles;
    const long long hk = at % P.Hk, b = at / P.Hk;
    const Seen see(P, b);
    const int row0 = tile * BK, nk = (int)P.Nk, nq = (int)P.Nq, D = (int)P.D;
    const T *k = static_cast<const T *>(P.k) + b * P.k_s[0] + hk * P.k_s[2];
    const T *v = static_cast<const T *>(P.v) + b * P.v_s[0] + hk * P.v_s[2];
    load_tile<T, A, BK, DP, THREADS>(K, k, P.k_s[1], row0, see.length, D, in_fours<T>(P.k, P.k_s, P.D));
    load_tile<T, A, BK, DP, THREADS>(V, v, P.v_s[1], row0, see.length, D, in_fours<T>(P.v, P.v_s, P.D));
    const bool qvec = in_fours<T>(P.q, P.q_s, P.D), gvec = in_fours<T>(P.dout, P.do_s, P.D);
    const A scale = scale_of<A>(P);
    A dk[RM][DP / TX], dv[RM][DP / TX];
    int lo[RM], hi[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const int j = row0 + ty * RM + r;
        lo[r] = see.qlo(j);
        hi[r] = see.qhi(j);
#pragma unroll
        for (int c = 0; c < DP / TX; ++c) dk[r][c] = dv[r][c] = 0;
    }
    const int last = row0 + BK < see.length ? row0 + BK - 1 : see.length - 1;
    const int i_lo = see.qlo(row0) / BQ * BQ, i_hi = last < row0 ? 0 : see.qhi(last);
    for (long long h = hk * P.group; h < (hk + 1) * P.group; ++h) {
        const T *q = static_cast<const T *>(P.q) + b * P.q_s[0] + h * P.q_s[2];
        const T *g = static_cast<const T *>(P.dout) + b * P.do_s[0] + h * P.do_s[2];
        const A *lse = static_cast<const A *>(P.row_lse) + (b * P.Hq + h) * P.Nqp;
        const A *delta = static_cast<const A *>(P.row_delta) + (b * P.Hq + h) * P.Nqp;
        for (int i0 = i_lo; i0 < i_hi; i0 += BQ) {
            __syncthreads();
            load_tile<T, A, BQ, DP, THREADS>(Q, q, P.q_s[1], i0, nq, D, qvec);
            load_tile<T, A, BQ, DP, THREADS>(G, g, P.do_s[1], i0, nq, D, gvec);
            __syncthreads();
            A s[RM][RN];
            product_nt<A, RM, RN, DP, TX>(s, K, Q, ty, tx);
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const int i = i0 + tx + TX * n;
                const A row = i < nq ? lse[i] : (A)0;
#pragma unroll
                for (int r = 0; r < RM; ++r)
                    S[(ty * RM + r) * (BQ + PAD) + tx + TX * n] = i >= lo[r] && i < hi[r] ? power(s[r][n] * scale - row) : (A)0;
            }
            __syncwarp();   // a row's values are written and read by the same threads of one warp
            product_nn<A, RM, BQ, DP, TX>(dv, S, G, ty, tx);
            product_nt<A, RM, RN, DP, TX>(s, V, G, ty, tx);
            __syncwarp();
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const int i = i0 + tx + TX * n;
                const A mean = i < nq ? delta[i] : (A)0;
#pragma unroll
                for (int r = 0; r < RM; ++r) {   // ds in the place of p; 0 times what need not be finite
                    A *at = &S[(ty * RM + r) * (BQ + PAD) + tx + TX * n];
                    *at = i >= lo[r] && i < hi[r] ? *at * (s[r][n] - mean) : (A)0;
                }
            }
            __syncwarp();
            product_nn<A, RM, BQ, DP, TX>(dk, S, Q, ty, tx);
        }
    }
    A one[RM], by[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        one[r] = lo[r] < hi[r] ? (A)1 : (A)0;
        by[r] = lo[r] < hi[r] ? (A)P.scale : (A)0;
    }
    const long long to = (b * P.Nk * P.Hk + hk) * P.D;
    store_rows<T, A, RM, DP, TX>(static_cast<T *>(P.dk) + to, (T *)nullptr, P.Hk * P.D, dk, by, row0, nk, D, ty, tx);
    store_rows<T, A, RM, DP, TX>(static_cast<T *>(P.dv) + to, (T *)nullptr, P.Hk * P.D, dv, one, row0, nk, D, ty, tx);
}

// dq of BQ queries: rows are queries, columns keys
template <typename T, typename A, int DP, int BQ, int BK, int TX>
__global__ void __launch_bounds__(16 * TX) attention_dq_simple_kernel(const AttnParams P, int tiles) {
    constexpr int RM = BQ / 16, RN = BK / TX, THREADS = 16 * TX;
    extern __shared__ __align__(32) unsigned char smem[];
    A *Q = reinterpret_cast<A *>(smem), *G = Q + BQ * (DP + PAD), *K = G + BQ * (DP + PAD), *V = K + BK * (DP + PAD),
      *S = V + BK * (DP + PAD);
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    long long at = blockIdx.x;
    const int tile = (int)(P.causal ? tiles - 1 - at % tiles : at % tiles);
    at /= tiles;
    const long long h = at % P.Hq, b = at / P.Hq, hk = h / P.group;
    const Seen see(P, b);
    const int row0 = tile * BQ, nq = (int)P.Nq, D = (int)P.D;
    const T *q = static_cast<const T *>(P.q) + b * P.q_s[0] + h * P.q_s[2];
    const T *g = static_cast<const T *>(P.dout) + b * P.do_s[0] + h * P.do_s[2];
    const T *k = static_cast<const T *>(P.k) + b * P.k_s[0] + hk * P.k_s[2];
    const T *v = static_cast<const T *>(P.v) + b * P.v_s[0] + hk * P.v_s[2];
    const bool kvec = in_fours<T>(P.k, P.k_s, P.D), vvec = in_fours<T>(P.v, P.v_s, P.D);
    load_tile<T, A, BQ, DP, THREADS>(Q, q, P.q_s[1], row0, nq, D, in_fours<T>(P.q, P.q_s, P.D));
    load_tile<T, A, BQ, DP, THREADS>(G, g, P.do_s[1], row0, nq, D, in_fours<T>(P.dout, P.do_s, P.D));
    const A scale = scale_of<A>(P);
    A dq[RM][DP / TX], row[RM], mean[RM], by[RM];
    int lo[RM], hi[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const int i = row0 + ty * RM + r;
        lo[r] = see.lo(i);
        hi[r] = i < nq ? see.hi(i) : 0;
        const long long from = (b * P.Hq + h) * P.Nqp + i;
        row[r] = i < nq ? static_cast<const A *>(P.row_lse)[from] : (A)0;
        mean[r] = i < nq ? static_cast<const A *>(P.row_delta)[from] : (A)0;
        by[r] = lo[r] < hi[r] ? (A)P.scale : (A)0;
#pragma unroll
        for (int c = 0; c < DP / TX; ++c) dq[r][c] = 0;
    }
    const int last = row0 + BQ < nq ? row0 + BQ - 1 : nq - 1;
    const int j_lo = see.lo(row0) / BK * BK, j_hi = see.hi(last);
    for (int j0 = j_lo; j0 < j_hi; j0 += BK) {
        __syncthreads();
        load_tile<T, A, BK, DP, THREADS>(K, k, P.k_s[1], j0, see.length, D, kvec);
        load_tile<T, A, BK, DP, THREADS>(V, v, P.v_s[1], j0, see.length, D, vvec);
        __syncthreads();
        A s[RM][RN], p[RM][RN];
        product_nt<A, RM, RN, DP, TX>(s, Q, K, ty, tx);
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const int j = j0 + tx + TX * n;
                p[r][n] = j >= lo[r] && j < hi[r] ? power(s[r][n] * scale - row[r]) : (A)0;
            }
        product_nt<A, RM, RN, DP, TX>(s, G, V, ty, tx);
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
            for (int n = 0; n < RN; ++n) {
                const int j = j0 + tx + TX * n;
                S[(ty * RM + r) * (BK + PAD) + tx + TX * n] = j >= lo[r] && j < hi[r] ? p[r][n] * (s[r][n] - mean[r]) : (A)0;
            }
        __syncwarp();
        product_nn<A, RM, BK, DP, TX>(dq, S, K, ty, tx);
    }
    T *out = static_cast<T *>(P.dq) + (b * P.Nq * P.Hq + h) * P.D;
    store_rows<T, A, RM, DP, TX>(out, (T *)nullptr, P.Hq * P.D, dq, by, row0, nq, D, ty, tx);
}

template <auto *KERNEL>
int run(const char *name, const AttnParams &P, long long rows, int tile_rows, long long heads, int threads, size_t smem, cudaStream_t s) {
    const long long tiles = (rows + tile_rows - 1) / tile_rows, blocks = tiles * heads * P.B;
    TPW_CHECK_ARG(blocks < (1LL << 31), "attention: more than 2^31 blocks of work");
    if (blocks == 0) return TPW_OK;
    if (const int e = allow_shared_memory<KERNEL>((int)smem)) return e;
    KERNEL<<<(unsigned)blocks, threads, smem, s>>>(P, (int)tiles);
    TPW_LAUNCH_OK(name);
    return TPW_OK;
}

template <typename T, int DP, int BM, int BN, int TX> int forward(const AttnParams &P, cudaStream_t s) {
    typedef typename AttnAcc<T>::type A;
    constexpr size_t smem = sizeof(A) * ((BM + 2 * BN) * (DP + PAD) + BM * (BN + PAD));
    static_assert(smem <= 232448, "exceeds the dynamic shared memory of one CTA");
    return run<&attention_forward_simple_kernel<T, A, DP, BM, BN, TX>>("attention_forward_simple_kernel", P, P.Nq, BM, P.Hq, 16 * TX, smem, s);
}
// BR rows of the CTA's own, BC of the tiles it walks over
template <typename T, int DP, int BR, int BC, int TX> constexpr size_t backward_smem() {
    constexpr size_t smem = sizeof(typename AttnAcc<T>::type) * (2 * (BR + BC) * (DP + PAD) + BR * (BC + PAD));
    static_assert(smem <= 232448, "exceeds the dynamic shared memory of one CTA");
    return smem;
}
template <typename T, int DP, int BR, int BC, int TX> int dkv(const AttnParams &P, cudaStream_t s) {
    typedef typename AttnAcc<T>::type A;
    return run<&attention_dkv_simple_kernel<T, A, DP, BR, BC, TX>>("attention_dkv_simple_kernel", P, P.Nk, BR, P.Hk, 16 * TX, backward_smem<T, DP, BR, BC, TX>(), s);
}
template <typename T, int DP, int BR, int BC, int TX> int dq(const AttnParams &P, cudaStream_t s) {
    typedef typename AttnAcc<T>::type A;
    return run<&attention_dq_simple_kernel<T, A, DP, BR, BC, TX>>("attention_dq_simple_kernel", P, P.Nq, BR, P.Hq, 16 * TX, backward_smem<T, DP, BR, BC, TX>(), s);
}

template <typename T> int forward_width(const AttnParams &P, cudaStream_t s) {
    if constexpr (sizeof(T) == 8)
        return P.D <= 64 ? forward<T, 64, 32, 32, 16>(P, s) : P.D <= 128 ? forward<T, 128, 32, 32, 16>(P, s) : forward<T, 256, 32, 32, 16>(P, s);
    else
        return P.D <= 64 ? forward<T, 64, 128, 64, 8>(P, s) : P.D <= 128 ? forward<T, 128, 128, 64, 16>(P, s) : forward<T, 256, 64, 32, 16>(P, s);
}
template <typename T, int DP, int BR, int BC, int TX> int backward(const AttnParams &P, cudaStream_t s) {
    const int e = P.dk ? dkv<T, DP, BR, BC, TX>(P, s) : TPW_OK;
    return e != TPW_OK || !P.dq ? e : dq<T, DP, BR, BC, TX>(P, s);
}
template <typename T> int backward_width(const AttnParams &P, cudaStream_t s) {
    if constexpr (sizeof(T) == 8)
        return P.D <= 64 ? backward<T, 64, 32, 32, 16>(P, s) : P.D <= 128 ? backward<T, 128, 32, 32, 16>(P, s) : backward<T, 256, 16, 16, 16>(P, s);
    else
        return P.D <= 64 ? backward<T, 64, 128, 32, 8>(P, s) : P.D <= 128 ? backward<T, 128, 64, 64, 16>(P, s) : backward<T, 256, 32, 32, 16>(P, s);
}

} // namespace

int attn_simple_forward(int dtype, const AttnParams &P, cudaStream_t s) {
    switch (dtype) {
        case TPW_F64: return forward_width<double>(P, s);
        case TPW_F32: return forward_width<float>(P, s);
        case TPW_F16: return forward_width<__half>(P, s);
        default: return forward_width<__nv_bfloat16>(P, s);
    }
}
int attn_simple_backward(int dtype, const AttnParams &P, cudaStream_t s) {
    switch (dtype) {
        case TPW_F64: return backward_width<double>(P, s);
        case TPW_F32: return backward_width<float>(P, s);
        case TPW_F16: return backward_width<__half>(P, s);
        default: return backward_width<__nv_bfloat16>(P, s);
    }
}

} // namespace tpw
