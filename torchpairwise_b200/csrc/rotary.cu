// Rotary positions: each pair of features (a, b) of a row is turned by the angle of the row's position,
// (a cos - b sin, a sin + b cos); the gradient is the turn back.
//
// Bound by HBM: every element is read and written once, 3 flops per element; bfloat16 [4, 4096, 40, 128] 64 us, 5.3 TB/s.  A thread holds the cosines and sines of one
// 16-byte chunk of pairs in registers and walks over heads of its token with them, two at a time and the next two on their
// way, because loading them per head would move more bytes through L1 than the rows themselves.  Calls with too few rows to
// fill the GPU that way give each thread one head (latency instead of traffic is what counts there).
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tpw {
namespace {

struct RotaryParams {
    const void *x[2];
    void *out[2];
    long long stride[2][3];
    long long H[2];
    const float *cos, *sin;
    const long long *positions;
    long long pos_stride[2];
    long long N, D, half, length, tokens;
    int heads_per_thread, head_groups, chunks;   // chunks per row: turned ones first, then copied ones
    int small, keep;                             // fewer than 2^32 threads; results of at most 64 MB
    float sign;
};

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };

// W elements as they lie in memory, and two neighbours of them widened and narrowed at a time
template <typename T, int W> struct alignas(sizeof(T) * W) Chunk { T v[W]; };
// Every row is read and written once: past L1.  Results beyond what L2 holds are not kept there (bfloat16 [4, 4096, 40, 128] 67.4 -> 63.9 us);
// smaller ones are what the next kernel reads.
template <typename C> __device__ __forceinline__ C read_once(const void *p) {
    if constexpr (sizeof(C) == 16) {
        C c;
        *reinterpret_cast<uint4 *>(&c) = __ldcs(static_cast<const uint4 *>(p));
        return c;
    } else {
        return *static_cast<const C *>(p);
    }
}
template <typename C> __device__ __forceinline__ void write_once(void *p, const C &c, bool keep) {
    if constexpr (sizeof(C) == 16) {
        if (!keep) {
            __stcs(static_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&c));
            return;
        }
    }
    *static_cast<C *>(p) = c;
}
template <typename T> __device__ __forceinline__ void widen2(const T *p, typename Acc<T>::type &a, typename Acc<T>::type &b) {
    a = p[0];
    b = p[1];
}
template <> __device__ __forceinline__ void widen2<__nv_bfloat16>(const __nv_bfloat16 *p, float &a, float &b) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void widen2<__half>(const __half *p, float &a, float &b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(p));
    a = f.x;
    b = f.y;
}
template <typename T> __device__ __forceinline__ void narrow2(T *p, typename Acc<T>::type a, typename Acc<T>::type b) {
    p[0] = a;
    p[1] = b;
}
template <> __device__ __forceinline__ void narrow2<__nv_bfloat16>(__nv_bfloat16 *p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(a, b);
}
template <> __device__ __forceinline__ void narrow2<__half>(__half *p, float a, float b) { *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(a, b); }

// W elements per access (16 bytes, or one where a row or pointer is off that grid).  64 registers, so that 32 warps per SM keep
// eight 16-byte loads each in flight: with 128 registers and half of the warps DRAM was 37 % busy.  In the half layout that is too few for the angles of
// eight pairs beside four pieces on their way: 16-bit types store 88 bytes a thread to local memory and load 156 back (ptxas).
template <typename T, int W, bool INTER>
__global__ void __launch_bounds__(256, 4) rotary_kernel(const RotaryParams P) {
    typedef typename Acc<T>::type A;
    typedef Chunk<T, W> C;
    constexpr int PAIRS = INTER ? (W > 1 ? W / 2 : 1) : W;   // pairs per turned chunk
    unsigned chunk, group;
    long long token;
    if (P.small) {   // 32-bit divisions where they reach
        const unsigned at = blockIdx.x * 256u + threadIdx.x, rest = at / (unsigned)P.chunks;
        chunk = at - rest * P.chunks;
        token = rest / (unsigned)P.head_groups;
        group = rest - (unsigned)token * P.head_groups;
    } else {
        const long long at = (long long)blockIdx.x * 256 + threadIdx.x, rest = at / P.chunks;
        chunk = (unsigned)(at - rest * P.chunks);
        token = rest / P.head_groups;
        group = (unsigned)(rest - token * P.head_groups);
    }
    if (token >= P.tokens) return;
    const long long b = P.small ? (unsigned)token / (unsigned)P.N : token / P.N, n = token - b * P.N;
    const unsigned turned = (unsigned)(P.half / PAIRS);
    const bool turn = chunk < turned;
    // offsets of the one or two pieces of a row that this thread handles
    int o0, o1 = 0;
    bool two = false;
    if (turn) {
        if (INTER) {
            o0 = chunk * (2 * PAIRS);
            two = W == 1;
            o1 = o0 + 1;
        } else {
            o0 = chunk * W;
            o1 = (int)P.half + o0;
            two = true;
        }
    } else {
        o0 = 2 * (int)P.half + (chunk - turned) * W;
    }
    float c[PAIRS], s[PAIRS];
    if (turn) {
        const long long t = P.positions ? P.positions[b * P.pos_stride[0] + n * P.pos_stride[1]] : n;
        const bool inside = t >= 0 && t < P.length;
        const float *pc = P.cos + (inside ? t : 0) * P.half + chunk * PAIRS;
        const float *ps = P.sin + (inside ? t : 0) * P.half + chunk * PAIRS;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            c[i] = inside ? pc[i] : __int_as_float(0x7fffffff);
            s[i] = ps[i] * P.sign;
        }
    }
    const int h_first = (int)P.H[0], h_end = h_first + (int)P.H[1];
    int h = (int)(group * P.heads_per_thread);
    const int h_stop = h + P.heads_per_thread < h_end ? h + P.heads_per_thread : h_end;
    auto work = [&](const C &x0, const C &x1, C &y0, C &y1) {
        if constexpr (W == 1) {
            const A u = (A)x0.v[0], v = (A)x1.v[0];
            y0.v[0] = (T)(u * (A)c[0] - v * (A)s[0]);
            y1.v[0] = (T)(u * (A)s[0] + v * (A)c[0]);
        } else if constexpr (INTER) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                A u, v;
                widen2<T>(&x0.v[2 * i], u, v);
                narrow2<T>(&y0.v[2 * i], u * (A)c[i] - v * (A)s[i], u * (A)s[i] + v * (A)c[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PAIRS; i += 2) {
                A u0, u1, v0, v1;
                widen2<T>(&x0.v[i], u0, u1);
                widen2<T>(&x1.v[i], v0, v1);
                narrow2<T>(&y0.v[i], u0 * (A)c[i] - v0 * (A)s[i], u1 * (A)c[i + 1] - v1 * (A)s[i + 1]);
                narrow2<T>(&y1.v[i], u0 * (A)s[i] + v0 * (A)c[i], u1 * (A)s[i + 1] + v1 * (A)c[i + 1]);
            }
        }
    };
    const T *from[2];
    T *to[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {   // head 0 of either tensor, counted in the heads of both
        from[w] = static_cast<const T *>(P.x[w]) + b * P.stride[w][0] + n * P.stride[w][1] - (w ? h_first * P.stride[1][2] : 0);
        to[w] = static_cast<T *>(P.out[w]) + (token * P.H[w] - (w ? h_first : 0)) * P.D;
    }
    // two heads at a time, the next two on their way meanwhile
    constexpr int U = 2;
    auto fetch = [&](int h, C (&x0)[U], C (&x1)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h + u < h_stop) {
                const T *p = h + u < h_first ? from[0] + (h + u) * P.stride[0][2] : from[1] + (h + u) * P.stride[1][2];
                x0[u] = read_once<C>(p + o0);
                if (two) x1[u] = read_once<C>(p + o1);
            }
    };
    C x0[U], x1[U];
    fetch(h, x0, x1);
    for (; h < h_stop; h += U) {
        C z0[U], z1[U];
        fetch(h + U, z0, z1);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h + u < h_stop) {
                C y0 = x0[u], y1 = x1[u];
                if (turn) work(x0[u], x1[u], y0, y1);
                T *p = (h + u < h_first ? to[0] : to[1]) + (h + u) * P.D;
                write_once(p + o0, y0, P.keep);
                if (two) write_once(p + o1, y1, P.keep);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x0[u] = z0[u];
            x1[u] = z1[u];
        }
    }
}

// Angles in turns, reduced to [-1/2, 1/2] in 64 bits (position * frequency is exact to 2^-53 of itself, so a position of a
// million leaves the fraction good to 1e-9), then one float32 sine and cosine of a half-turn multiple.
__global__ void __launch_bounds__(256) rotary_table_kernel(const double *frequency, double magnitude, float *cos_, float *sin_,
                                                           long long length, long long half) {
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= length * half) return;
    const double turns = (double)(at / half) * (frequency[at % half] * 0.15915494309189533577);
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cos_[at] = (float)((double)c * magnitude);
    sin_[at] = (float)((double)s * magnitude);
}

template <typename T, bool INTER>
int launch(const tpw_rotary &a, RotaryParams &P, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    bool wide = a.D % W == 0 && (2 * a.half) % W == 0 && (INTER || a.half % W == 0);
    for (int w = 0; w < 2; ++w) {
        if (a.H[w] == 0) continue;
        wide = wide && aligned16(a.x[w]) && aligned16(a.out[w]);
        for (int i = 0; i < 3; ++i) wide = wide && a.stride[w][i] % W == 0;
    }
    const int width = wide ? W : 1;
    const long long pairs = INTER ? (width > 1 ? width / 2 : 1) : width;
    const long long chunks = a.half / pairs + (a.D - 2 * a.half) / width;
    const long long heads = a.H[0] + a.H[1];
    P.chunks = (int)chunks;
    // Heads per thread: as many as leave the GPU at least eight blocks per SM.  More threads read the table more often (float32 [3, 1777, 24,
    // 80], 32 turned, 8 heads 19.4 us, 2 heads 25.5); a new token of 8 sequences is 8 * 40 rows, one head per thread.
    long long per = 8;
    while (per > 1 && P.tokens * chunks * ((heads + per - 1) / per) < 8LL * 256 * sm_count()) per /= 2;
    P.heads_per_thread = (int)per;
    P.head_groups = (int)((heads + per - 1) / per);
    const long long threads = P.tokens * chunks * P.head_groups, blocks = (threads + 255) / 256;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_rotary_apply: more than 2^31 blocks of work");
    P.small = blocks < (1LL << 24);
    P.keep = P.tokens * heads * a.D * (long long)sizeof(T) <= (64LL << 20);
    if (wide) rotary_kernel<T, W, INTER><<<(unsigned)blocks, 256, 0, s>>>(P);
    else rotary_kernel<T, 1, INTER><<<(unsigned)blocks, 256, 0, s>>>(P);
    TPW_LAUNCH_OK("rotary_kernel");
    return TPW_OK;
}

} // namespace
} // namespace tpw

extern "C" {

int tpw_rotary_apply(const tpw_rotary *a, tpw_stream_t stream) {
    tpw::clear_error();
    TPW_CHECK_ARG(a != nullptr, "tpw_rotary_apply: NULL arguments");
    TPW_CHECK_ARG(a->dtype == TPW_F32 || a->dtype == TPW_F64 || a->dtype == TPW_F16 || a->dtype == TPW_BF16,
                  "tpw_rotary_apply: unsupported dtype %d", a->dtype);
    TPW_CHECK_ARG(a->B >= 0 && a->N >= 0 && a->D >= 0 && a->half >= 0 && a->H[0] >= 0 && a->H[1] >= 0 && a->length >= 0,
                  "tpw_rotary_apply: negative size");
    TPW_CHECK_ARG(2 * a->half <= a->D, "tpw_rotary_apply: %lld turned features of %lld", (long long)(2 * a->half), (long long)a->D);
    TPW_CHECK_ARG(a->D < (1LL << 30) && a->H[0] + a->H[1] < (1LL << 30), "tpw_rotary_apply: more than 2^30 features or heads");
    if (a->B == 0 || a->N == 0 || a->D == 0 || a->H[0] + a->H[1] == 0) return TPW_OK;
    TPW_CHECK_ARG(a->half == 0 || (a->cos && a->sin), "tpw_rotary_apply: NULL table");
    TPW_CHECK_ARG(a->half == 0 || a->length > 0, "tpw_rotary_apply: empty table");
    for (int w = 0; w < 2; ++w)
        TPW_CHECK_ARG(a->H[w] == 0 || (a->x[w] && a->out[w]), "tpw_rotary_apply: NULL tensor");
    tpw::RotaryParams P = {};
    for (int w = 0; w < 2; ++w) {
        P.x[w] = a->x[w];
        P.out[w] = a->out[w];
        P.H[w] = a->H[w];
        for (int i = 0; i < 3; ++i) P.stride[w][i] = a->stride[w][i];
    }
    P.cos = a->cos;
    P.sin = a->sin;
    P.positions = reinterpret_cast<const long long *>(a->positions);
    P.pos_stride[0] = a->position_stride[0];
    P.pos_stride[1] = a->position_stride[1];
    P.N = a->N;
    P.D = a->D;
    P.half = a->half;
    P.length = a->length;
    P.tokens = a->B * a->N;
    P.sign = a->inverse ? -1.f : 1.f;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case TPW_F32: return a->interleaved ? tpw::launch<float, true>(*a, P, s) : tpw::launch<float, false>(*a, P, s);
        case TPW_F64: return a->interleaved ? tpw::launch<double, true>(*a, P, s) : tpw::launch<double, false>(*a, P, s);
        case TPW_F16: return a->interleaved ? tpw::launch<__half, true>(*a, P, s) : tpw::launch<__half, false>(*a, P, s);
        default: return a->interleaved ? tpw::launch<__nv_bfloat16, true>(*a, P, s) : tpw::launch<__nv_bfloat16, false>(*a, P, s);
    }
}

int tpw_rotary_table(const double *frequency, double magnitude, float *cos, float *sin, int64_t length, int64_t half, tpw_stream_t stream) {
    tpw::clear_error();
    TPW_CHECK_ARG(length >= 0 && half >= 0, "tpw_rotary_table: negative size");
    if (length == 0 || half == 0) return TPW_OK;
    TPW_CHECK_ARG(frequency && cos && sin, "tpw_rotary_table: NULL pointer");
    TPW_CHECK_ARG(length < (1LL << 40) / half, "tpw_rotary_table: table of more than 2^40 values");
    const long long blocks = (length * half + 255) / 256;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_rotary_table: more than 2^31 blocks of work");
    tpw::rotary_table_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(frequency, magnitude, cos, sin, length, half);
    TPW_LAUNCH_OK("rotary_table_kernel");
    return TPW_OK;
}

} // extern "C"
