// Rotary positions: each pair of features (a, b) of a row is turned by the angle of the row's position,
// (a cos - b sin, a sin + b cos); the gradient is the turn back.
//
// Bound by HBM: every element is read and written once, 3 flops per element.  A thread holds the cosines and sines of one
// 16-byte chunk of pairs in registers and walks over heads of its token with them, 4 at a time so that enough loads are in
// flight, because loading them per head would move more bytes through L1 than the rows themselves.  Calls with too few rows to
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
    float sign;
};

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };

template <typename T> __device__ __forceinline__ typename Acc<T>::type widen(T v) { return (typename Acc<T>::type)v; }
template <typename T> __device__ __forceinline__ T narrow(typename Acc<T>::type v) { return (T)v; }

template <typename T, int W> struct alignas(sizeof(T) * W) Chunk { T v[W]; };

// W elements per access (16 bytes, or one where a row or pointer is off that grid)
template <typename T, int W, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams P) {
    typedef typename Acc<T>::type A;
    typedef Chunk<T, W> C;
    constexpr int PAIRS = INTER ? (W > 1 ? W / 2 : 1) : W;   // pairs per turned chunk
    long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int chunk = (int)(at % P.chunks);
    at /= P.chunks;
    const int group = (int)(at % P.head_groups);
    const long long token = at / P.head_groups;
    if (token >= P.tokens) return;
    const long long b = token / P.N, n = token % P.N;
    const int turned = (int)(P.half / PAIRS);
    const bool turn = chunk < turned;
    // offsets of the one or two pieces of a row that this thread handles
    long long o0, o1 = 0;
    bool two = false;
    if (turn) {
        if (INTER) {
            o0 = (long long)chunk * (2 * PAIRS);
            two = W == 1;
            o1 = o0 + 1;
        } else {
            o0 = (long long)chunk * W;
            o1 = P.half + o0;
            two = true;
        }
    } else {
        o0 = 2 * P.half + (long long)(chunk - turned) * W;
    }
    float c[PAIRS], s[PAIRS];
    if (turn) {
        const long long t = P.positions ? P.positions[b * P.pos_stride[0] + n * P.pos_stride[1]] : n;
        const bool inside = t >= 0 && t < P.length;
        const float *pc = P.cos + (inside ? t : 0) * P.half + (long long)chunk * PAIRS;
        const float *ps = P.sin + (inside ? t : 0) * P.half + (long long)chunk * PAIRS;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            c[i] = inside ? pc[i] : __int_as_float(0x7fffffff);
            s[i] = ps[i] * P.sign;
        }
    }
    const long long h_end = P.H[0] + P.H[1];
    long long h = (long long)group * P.heads_per_thread;
    const long long h_stop = h + P.heads_per_thread < h_end ? h + P.heads_per_thread : h_end;
    auto work = [&](const C &x0, const C &x1, C &y0, C &y1) {
        if (!turn) {
            y0 = x0;
        } else if (INTER && W > 1) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const A u = widen(x0.v[(2 * i) % W]), v = widen(x0.v[(2 * i + 1) % W]);
                y0.v[(2 * i) % W] = narrow<T>(u * (A)c[i] - v * (A)s[i]);
                y0.v[(2 * i + 1) % W] = narrow<T>(u * (A)s[i] + v * (A)c[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const A u = widen(x0.v[i]), v = widen(x1.v[i]);
                y0.v[i] = narrow<T>(u * (A)c[i] - v * (A)s[i]);
                y1.v[i] = narrow<T>(u * (A)s[i] + v * (A)c[i]);
            }
        }
    };
    auto from = [&](long long head) {
        const int w = head >= P.H[0];
        const long long hh = head - (w ? P.H[0] : 0);
        return static_cast<const T *>(P.x[w]) + b * P.stride[w][0] + n * P.stride[w][1] + hh * P.stride[w][2];
    };
    auto to = [&](long long head) {
        const int w = head >= P.H[0];
        const long long hh = head - (w ? P.H[0] : 0);
        return static_cast<T *>(P.out[w]) + (token * P.H[w] + hh) * P.D;
    };
    constexpr int U = 4;
    for (; h < h_stop; h += U) {
        C x0[U], x1[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h + u < h_stop) {
                const T *p = from(h + u);
                x0[u] = *reinterpret_cast<const C *>(p + o0);
                if (two) x1[u] = *reinterpret_cast<const C *>(p + o1);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h + u < h_stop) {
                C y0, y1;
                work(x0[u], x1[u], y0, y1);
                T *p = to(h + u);
                *reinterpret_cast<C *>(p + o0) = y0;
                if (two) *reinterpret_cast<C *>(p + o1) = y1;
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
    // Heads per thread: as many of 4, 8 as leave the GPU at least eight blocks per SM.  bfloat16 [4, 4096, 40, 128]:
    // DRAM-bound; a single new token of 8 sequences: 8 * 40 rows, one head per thread.
    long long per = 8;
    while (per > 1 && P.tokens * chunks * ((heads + per - 1) / per) < 8LL * 256 * sm_count()) per /= 2;
    P.heads_per_thread = (int)per;
    P.head_groups = (int)((heads + per - 1) / per);
    const long long threads = P.tokens * chunks * P.head_groups, blocks = (threads + 255) / 256;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_rotary_apply: more than 2^31 blocks of work");
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
