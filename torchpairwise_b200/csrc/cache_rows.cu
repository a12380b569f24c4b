// Tokens into a cache of quantised keys and values, and out of it.
//
// Bound by HBM on paper.  Storing waits for its loads first (5.5 warps of those that wait, 28 % of DRAM: a block asks for its sequence's length before its values, has one token a lane, and
// ends), and takes about 21 instructions a value, 64 % of the issue slots.  What keeps them few: a lane has a group's 32 values, quotients are refined on the FMA
// pipes (a test for middles on the logic pipe was 10 more), codes are added up above a constant instead of masked and shifted, and bytes become numbers by
// permutation.  Measured bfloat16, 4 bits: 2 x 8192 tokens of 8 heads of 128, 67 MB stored and read back in 43 us; 4 x 16384 ragged read in 53 us, 5.9 TB/s.
#include "attention_tc.cuh"
#include "cache.cuh"

namespace tpw {
namespace {

constexpr int kWriteTokens = 32, kReadTokens = 64;   // of a block

struct RowsParams {
    CacheParams c;
    void *x[2];
    long long stride[2][3];
    int N, tiles;              // tokens; blocks of tokens of a head
    Divider by_tiles, by_heads;
    int from_start, vector;    // vector: 16-byte pieces of a row
    int leave;                 // read: rows that are not stored are left as they were
    int last;                  // read: and those before the last so many and their block of 128; 0: none are
    const uint32_t *highest;   // read: what cache_ranges found, or NULL; values are then brought below 2^bring[0] (keys), 2^bring[1]
    int bring[2];
};

// NaN if an operand is
__device__ __forceinline__ float min_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// n of 8 features as they lie in memory, widened
template <typename T> __device__ __forceinline__ void load8(float (&x)[8], const T *p, int n, bool vector) {
    if (vector) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(p)), b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(p));
            const T *v = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (float)v[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = (float)p[k < n ? k : 0];
    }
}
// `keep`: what is read next
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8], int n, bool vector, bool keep) {
    if (vector) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = make_float4(x[0], x[1], x[2], x[3]), b = make_float4(x[4], x[5], x[6], x[7]);
            if (keep) {
                reinterpret_cast<float4 *>(p)[0] = a;
                reinterpret_cast<float4 *>(p)[1] = b;
            } else {
                __stcs(reinterpret_cast<float4 *>(p), a);
                __stcs(reinterpret_cast<float4 *>(p) + 1, b);
            }
        } else {
            const uint4 v = make_uint4(Narrow<T>::pack(x[0], x[1]), Narrow<T>::pack(x[2], x[3]), Narrow<T>::pack(x[4], x[5]), Narrow<T>::pack(x[6], x[7]));
            if (keep) *reinterpret_cast<uint4 *>(p) = v;
            else __stcs(reinterpret_cast<uint4 *>(p), v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) p[k] = (T)x[k];
    }
}

// Many bfloat16 queries go through half precision, which has the digits but not the exponents (cache_attention.cu): each head's keys and values
// are brought near a power of two.  `parts` has the highest magnitudes, as bits, of parts of a head; the factor is a power of two.
__device__ __forceinline__ int exponent_of(const uint32_t *parts) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kRangeParts; ++k) top = max(top, parts[k]);
    return top == 0 ? 0 : (int)(top >> 23) - 126;   // the magnitudes are below 2 to this
}
__device__ __forceinline__ float bring_by(const uint32_t *parts, int to) {
    const int e = to - exponent_of(parts) + 127;
    return __uint_as_float((uint32_t)(e < 1 ? 1 : e > 254 ? 254 : e) << 23);
}
// The first position of a sequence of `end` stored tokens that counts where only the last `last` (0: all) do: that of their first block of 128
__device__ __forceinline__ int first_of(int end, int last) { return last > 0 && end > last ? (end - last) & ~127 : 0; }
// the highest magnitude that the codes of a part of a head's keys (or values), those before first_of left out, can stand for; groups that are not numbers take no part
__global__ void __launch_bounds__(256) cache_ranges_kernel(const CacheParams P, int last, uint32_t *highest) {
    const long long bh = blockIdx.x;
    const int part = blockIdx.y, which = blockIdx.z, b = (int)(bh / P.H), cap = (int)P.capacity;
    int n = P.lengths[b];
    n = n < 0 ? 0 : n < cap ? n : cap;
    const int first = first_of(n, last);
    const unsigned count = (unsigned)(n - first) * P.groups, start = part * 256 + threadIdx.x;   // below 2^32: 2^30 - 64 places, 4 groups
    const uint32_t *scales = P.scales[which] + (bh * cap + first) * P.groups + start;
    const float most = P.bits == 4 ? 15.f : 255.f;
    uint32_t top = 0;
    for (unsigned left = start < count ? (count - start - 1) / (kRangeParts * 256) + 1 : 0; left > 0; --left, scales += kRangeParts * 256) {
        const float zero = zero_of(*scales), end = fmaf(step_of(*scales), most, zero), high = fmaxf(fabsf(zero), fabsf(end));
        if (fabsf(zero) <= high && high < 5.0706024009129176e30f) top = max(top, __float_as_uint(high));   // 2^102
    }
    __shared__ uint32_t tops[8];
    top = __reduce_max_sync(0xffffffffu, top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) top = max(top, tops[w]);
        highest[(which * P.B * P.H + bh) * kRangeParts + part] = top;
    }
}
// Rows of queries to half precision, times what their keys were divided by; rows of results back.  A thread has 8 features, a block 256 times that.
struct ConvertParams {
    const void *from;
    void *to;
    long long stride[3], pieces;   // of `from`; pieces of 8 features
    const uint32_t *highest;
    Divider by_d, by_heads, by_tokens, by_group;
    int H;                         // key heads
    int bring;
};
template <typename A, typename B> __global__ void __launch_bounds__(256) cache_convert_kernel(const ConvertParams C) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at >= C.pieces) return;
    const unsigned row = at / C.by_d, d = at - row * C.by_d.d, token = row / C.by_heads, h = row - token * C.by_heads.d, b = token / C.by_tokens, i = token - b * C.by_tokens.d;
    const uint32_t *parts = C.highest + (b * C.H + h / C.by_group) * kRangeParts;
    const int e = exponent_of(parts) - C.bring + 127;
    const float by = __uint_as_float((uint32_t)(e < 1 ? 1 : e > 254 ? 254 : e) << 23);
    const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const A *>(C.from) + b * C.stride[0] + i * C.stride[1] + h * C.stride[2] + 8 * d);
    const A *v = reinterpret_cast<const A *>(&w);
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (float)v[k] * by;
    reinterpret_cast<uint4 *>(C.to)[at] = make_uint4(Narrow<B>::pack(x[0], x[1]), Narrow<B>::pack(x[2], x[3]), Narrow<B>::pack(x[4], x[5]), Narrow<B>::pack(x[6], x[7]));
}

// What a block works on: TOKENS tokens of a head, this thread's first being i0; token i stands at position i + shift, and positions [0, end) have a place.
template <int TOKENS> struct Block {
    int b, h, i0, shift, end;
    long long row0;   // of the cache
    __device__ __forceinline__ Block(const RowsParams &R, int token) {
        const unsigned bh = blockIdx.x / R.by_tiles;
        b = (int)(bh / R.by_heads);
        h = (int)bh - b * (int)R.c.H;
        i0 = (int)(blockIdx.x - bh * R.tiles) * TOKENS + token;
        int n = R.c.lengths[b];
        n = n < 0 ? 0 : n;
        shift = R.from_start ? 0 : n - R.N;   // N < 2^30
        end = n < (int)R.c.capacity ? n : (int)R.c.capacity;
        row0 = (long long)bh * R.c.capacity;
    }
    __device__ __forceinline__ bool stored(int i) const { return i + shift >= 0 && i + shift < end; }
};

// where the 8 codes of lane l lie in a row: those of a key together, those of a value in two halves
template <int BITS, int W> __device__ __forceinline__ int key_place(int l) { return ((l & 3) * W + (l >> 2)) * BITS; }
template <int BITS, int W> __device__ __forceinline__ int value_place(int l, int half) { return ((2 * (l & 3) + half) * W + (l >> 2)) * (BITS / 2); }

// 8 codes into words, 4 bits in one, 8 bits in two; `y` holds them above 1.5 * 2^23, whose bits add up to a constant
template <int BITS> __device__ __forceinline__ void pack8(uint32_t (&w)[2], const float (&y)[8], int n) {
    constexpr int PER = 32 / BITS;
    constexpr uint32_t ONES = BITS == 4 ? 0x11111111u : 0x01010101u;
    w[1] = 0;
#pragma unroll
    for (int v = 0; v < 8 / PER; ++v) {
        uint32_t x = 0;
#pragma unroll
        for (int k = PER - 1; k >= 0; --k) x = (x << BITS) + __float_as_uint(y[v * PER + k]);
        x -= 0x4b400000u * ONES;
        const int there = n - v * PER;
        w[v] = there >= PER ? x : there <= 0 ? 0u : x & ((1u << (BITS * there)) - 1u);
    }
}

// Apart, so that 32 rare divisions do not lie between the others' instructions ([3, 1777, 12, 80] stored and read: 35 -> 33 us)
__device__ __noinline__ float code_in_64_bits(float x, float zero, float step) { return (float)rint(((double)x - (double)zero) / (double)step); }

// x - zero rounded to odd: where 32 bits do not hold it, that neighbour whose last bit is set, so that it lies on the true side of any number of 23 bits or fewer
__device__ __forceinline__ float distance(float x, float zero) {
    const uint32_t below = __float_as_uint(__fsub_rz(x, zero)), above = __float_as_uint(__fsub_ru(x, zero));   // x is not below the zero
    return __uint_as_float(below | ((below ^ above) & 1u));
}

// A lane has 32 features of a token, so that what a group's step costs is paid once; 2 or 4 lanes a token.
template <typename T, int BITS, int W>
__global__ void __launch_bounds__(kWriteTokens * (W == 2 ? 2 : 4)) cache_write_kernel(const RowsParams R) {
    constexpr int LANES = W == 2 ? 2 : 4;   // of a token; W of them have features
    constexpr float MOST = BITS == 4 ? 15.f : 255.f;
    const int which = blockIdx.y, w = threadIdx.x % LANES;
    const Block<kWriteTokens> B(R, threadIdx.x / LANES);
    const int n = R.c.D - 32 * w;   // features of this lane that there are
    const bool stored = B.i0 < R.N && B.stored(B.i0), live = stored && n > 0;
    const T *from = static_cast<const T *>(R.x[which]) + B.b * R.stride[which][0] + B.i0 * R.stride[which][1] + B.h * R.stride[which][2] + 32 * w;
    float x[4][8];
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (live && 8 * v < n) load8(x[v], from + 8 * v, n - 8 * v, R.vector);
    float lo = INFINITY, hi = -INFINITY;
    if (live)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (8 * v < n)
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    lo = min_nan(lo, x[v][k], x[v][k + 1]);
                    hi = max_nan(hi, x[v][k], x[v][k + 1]);
                }
    if (R.c.groups == 1)
#pragma unroll
        for (int d = 1; d < LANES; d <<= 1) {
            lo = min_nan(lo, lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = max_nan(hi, hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
    if (!stored || w >= W) return;
    // zero: down to bfloat16
    uint32_t zero_bits = __float_as_uint(lo);
    if ((int)zero_bits < 0) zero_bits += 0xffffu;
    zero_bits &= 0xffff0000u;
    const float zero = __uint_as_float(zero_bits);
    // step: the smallest bfloat16 number of which MOST (products of which are exact) reach the highest value.  The quotient's upper 16 bits are at
    // most one number off.
    const float range = __fsub_ru(hi, zero);
    uint32_t step_bits = (__float_as_uint(range * (1.f / MOST)) + 0xffffu) & 0xffff0000u;
    if (__uint_as_float(step_bits - 0x10000u) * MOST >= range) step_bits -= 0x10000u;
    if (__uint_as_float(step_bits) * MOST < range) step_bits += 0x10000u;
    const float least = 7.888609052210118e-31f;   // 2^-100
    const bool fine = lo > -1.2676506002282294e30f && hi < 1.2676506002282294e30f;   // 2^100; NaN is not
    const float step = fmaxf(__uint_as_float(step_bits), least);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
    const long long place = B.row0 + B.i0 + B.shift;
    unsigned char *to = R.c.codes[which] + place * (W * 4 * BITS);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        // The quotient, refined by what is left of it, exactly: it is off by half a unit and 2^-45 of itself at most, and a middle between two codes comes out as
        // that.  A sum with 1.5 * 2^23 ends in the nearest whole number, ties to even.  What 16-bit values lie on a middle but for lies too far down for 32 bits, but decides
        // (1 less -2^-40): their distances are rounded to odd.  A middle times the step has 17 bits at most, a distance of 24 bits beside it differs by one of its last places, which
        // is more than the quotient is off.  (A distance that is all ones lies beside a power of two; then the step is one too, and the quotient exact.)  2 x 8192 tokens: 41 -> 43 us.
        uint32_t code[2] = {0, 0};
        if (live && 8 * v < n) {   // pieces beyond the head have no values
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float d = sizeof(T) == 4 ? __fsub_rn(x[v][k], zero) : distance(x[v][k], zero), near = __fmul_rn(d, inv);
                const float quotient = fmaf(fmaf(-near, step, d), inv, near);
                y[k] = __fadd_rn(quotient, 12582912.f);
                // float32 values have digits that their distance from the zero has not: beside a middle 64 bits decide.  The distance and the quotient are
                // each off by 2^-24 and 2^-23 of at most MOST codes, 1.8e-7.
                if (sizeof(T) == 4 && fabsf(quotient - (y[k] - 12582912.f)) > 0.5f - MOST * 2.4e-7f)
                    y[k] = 12582912.f + code_in_64_bits(x[v][k], zero, step);
            }
            pack8<BITS>(code, y, fine ? n - 8 * v : 0);
        }
        const int l = 4 * w + v;
        if (which == 0) {
            if (BITS == 4) *reinterpret_cast<uint32_t *>(to + key_place<BITS, W>(l)) = code[0];
            else *reinterpret_cast<uint2 *>(to + key_place<BITS, W>(l)) = make_uint2(code[0], code[1]);
        } else if (BITS == 4) {
            *reinterpret_cast<uint16_t *>(to + value_place<BITS, W>(l, 0)) = (uint16_t)code[0];
            *reinterpret_cast<uint16_t *>(to + value_place<BITS, W>(l, 1)) = (uint16_t)(code[0] >> 16);
        } else {
            *reinterpret_cast<uint32_t *>(to + value_place<BITS, W>(l, 0)) = code[0];
            *reinterpret_cast<uint32_t *>(to + value_place<BITS, W>(l, 1)) = code[1];
        }
    }
    if (R.c.groups > 1 ? w < R.c.groups : w == 0) R.c.scales[which][place * R.c.groups + w] = fine ? __float_as_uint(step) >> 16 | zero_bits : 0x7fc07fc0u;
}

// A lane has what lies together in a row: features 8 l to 8 l + 7 of every group of 32, l < 4, which leave as pieces of 16 bytes, 64 side by side.
template <typename T, int BITS, int W>
__global__ void __launch_bounds__(4 * kReadTokens) cache_read_kernel(const RowsParams R) {
    constexpr int WORDS = W * BITS / 4;
    const int which = blockIdx.y, l = threadIdx.x & 3;
    const Block<kReadTokens> B(R, threadIdx.x >> 2);
    const int first = first_of(B.end, R.last);   // positions before it are left
    const bool there = B.i0 < R.N && B.stored(B.i0) && B.i0 + B.shift >= first;
    if (R.leave ? !there : B.i0 >= R.N) return;
    uint32_t w[WORDS] = {}, scales[W] = {};
    if (there) {
        const long long place = B.row0 + B.i0 + B.shift;
        const unsigned char *row = R.c.codes[which] + place * (W * 4 * BITS) + l * (W * BITS);
        if constexpr (WORDS % 4 == 0) {
#pragma unroll
            for (int k = 0; k < WORDS / 4; ++k) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(row) + k);
                w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
            }
        } else if constexpr (WORDS % 2 == 0) {
#pragma unroll
            for (int k = 0; k < WORDS / 2; ++k) {
                const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(row) + k);
                w[2 * k] = v.x; w[2 * k + 1] = v.y;
            }
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = __ldcs(reinterpret_cast<const uint32_t *>(row) + k);
        }
        const uint32_t *of = R.c.scales[which] + place * R.c.groups;
#pragma unroll
        for (int k = 0; k < W; ++k) scales[k] = R.c.groups == 1 ? of[0] : k < R.c.groups ? of[k] : 0u;
    }
    const float by = R.highest ? bring_by(R.highest + (which * R.c.B * R.c.H + B.b * R.c.H + B.h) * kRangeParts, R.bring[which]) : 1.f;
    T *to = static_cast<T *>(R.x[which]) + B.b * R.stride[which][0] + B.i0 * R.stride[which][1] + B.h * R.stride[which][2] + 8 * l;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const int n = R.c.D - 32 * k - 8 * l;
        if (n <= 0) break;
        // the 8 codes: a key's lie together, a value's in two runs of 4
        uint32_t c[2];
        if constexpr (BITS == 4) {
            const uint32_t word = which == 0 ? w[k] : __byte_perm(w[k / 2], w[(W + k) / 2], (k % 2 ? 0x32 : 0x10) | ((W + k) % 2 ? 0x7600 : 0x5400));
            c[0] = word & 0x0f0f0f0fu;
            c[1] = (word >> 4) & 0x0f0f0f0fu;
        } else {
            c[0] = which == 0 ? w[2 * k] : w[k];
            c[1] = which == 0 ? w[2 * k + 1] : w[W + k];
        }
        const float step = step_of(scales[k]) * by, zero = zero_of(scales[k]) * by;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // a byte to a code, then 2^23 + code less 2^23: the conversion instruction is a quarter as fast
            const uint32_t byte = BITS == 4 ? __byte_perm(c[e & 1], 0x4b000000u, 0x7440 + (e >> 1)) : __byte_perm(c[e >> 2], 0x4b000000u, 0x7440 + (e & 3));
            x[e] = fmaf(__uint_as_float(byte) - 8388608.f, step, zero);
        }
        store8(to + 32 * k, x, n, R.vector, R.leave);
    }
}

template <typename T, int BITS, int W> int launch(const RowsParams &R, bool write, cudaStream_t s) {
    const long long blocks = R.c.B * R.c.H * R.tiles;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_cache: more than 2^31 blocks of work");
    if (write) {
        cache_write_kernel<T, BITS, W><<<dim3((unsigned)blocks, 2), kWriteTokens * (W == 2 ? 2 : 4), 0, s>>>(R);
        TPW_LAUNCH_OK("cache_write_kernel");
    } else {
        cache_read_kernel<T, BITS, W><<<dim3((unsigned)blocks, 2), 4 * kReadTokens, 0, s>>>(R);
        TPW_LAUNCH_OK("cache_read_kernel");
    }
    return TPW_OK;
}
template <typename T> int launch_width(const RowsParams &R, bool write, cudaStream_t s) {
    if (R.c.bits == 4) return R.c.width == 2 ? launch<T, 4, 2>(R, write, s) : R.c.width == 3 ? launch<T, 4, 3>(R, write, s) : launch<T, 4, 4>(R, write, s);
    return R.c.width == 2 ? launch<T, 8, 2>(R, write, s) : R.c.width == 3 ? launch<T, 8, 3>(R, write, s) : launch<T, 8, 4>(R, write, s);
}
RowsParams params(const CacheParams &P, int dtype, long long N, int tokens, void *const (&x)[2], const int64_t (&stride)[2][3]) {
    RowsParams R = {};
    R.c = P;
    R.N = (int)N;
    R.tiles = (int)((N + tokens - 1) / tokens);
    R.by_tiles = divider(R.tiles);
    R.by_heads = divider(P.H);
    const long long piece = dtype == TPW_F32 ? 4 : 8;
    R.vector = P.D % 8 == 0;
    for (int w = 0; w < 2; ++w) {
        R.x[w] = x[w];
        R.vector = R.vector && aligned16(x[w]);
        for (int k = 0; k < 3; ++k) {
            R.stride[w][k] = stride[w][k];
            R.vector = R.vector && stride[w][k] % piece == 0;
        }
    }
    return R;
}
int run(int dtype, const RowsParams &R, bool write, cudaStream_t s) {
    return dtype == TPW_F32 ? launch_width<float>(R, write, s) : dtype == TPW_F16 ? launch_width<__half>(R, write, s) : launch_width<__nv_bfloat16>(R, write, s);
}

} // namespace

int cache_write(const CacheParams &P, const tpw_cache_rows &rows, cudaStream_t s) { return run(rows.dtype, params(P, rows.dtype, rows.N, kWriteTokens, rows.x, rows.stride), true, s); }

int cache_read(const CacheParams &P, const tpw_cache_rows &rows, cudaStream_t s) {
    const int64_t dense[3] = {rows.N * P.H * P.D, P.H * P.D, P.D}, stride[2][3] = {{dense[0], dense[1], dense[2]}, {dense[0], dense[1], dense[2]}};
    RowsParams R = params(P, rows.dtype, rows.N, kReadTokens, rows.x, stride);
    R.from_start = rows.from_start;
    return run(rows.dtype, R, false, s);
}

int cache_ranges(const CacheParams &P, long long last, uint32_t *highest, cudaStream_t s) {
    TPW_CHECK_ARG(P.B * P.H < (1LL << 31), "tpw_cache_attention: more than 2^31 heads of a slice");
    cache_ranges_kernel<<<dim3((unsigned)(P.B * P.H), kRangeParts, 2), 256, 0, s>>>(P, (int)(last < P.capacity ? last : 0), highest);
    TPW_LAUNCH_OK("cache_ranges_kernel");
    return TPW_OK;
}

int cache_expand(const CacheParams &P, int dtype, void *const (&x)[2], const int64_t (&stride)[3], long long last, const uint32_t *highest, const int (&bring)[2], cudaStream_t s) {
    const int64_t both[2][3] = {{stride[0], stride[1], stride[2]}, {stride[0], stride[1], stride[2]}};
    RowsParams R = params(P, dtype, P.capacity, kReadTokens, x, both);
    R.from_start = 1;
    R.leave = 1;
    R.last = (int)(last < P.capacity ? last : 0);
    R.highest = highest;
    for (int w = 0; w < 2; ++w) R.bring[w] = bring[w];
    return run(dtype, R, false, s);
}

int cache_convert(bool back, const void *from, void *to, const int64_t (&stride)[3], const uint32_t *highest, int bring, long long B, long long N, long long Hq, long long H, long long D,
                  cudaStream_t s) {
    ConvertParams C = {};
    C.from = from;
    C.to = to;
    for (int k = 0; k < 3; ++k) C.stride[k] = stride[k];
    C.pieces = B * N * Hq * (D / 8);
    C.highest = highest;
    C.by_d = divider(D / 8);
    C.by_heads = divider(Hq);
    C.by_tokens = divider(N);
    C.by_group = divider(Hq / H);
    C.H = (int)H;
    C.bring = bring;
    const long long blocks = (C.pieces + 255) / 256;
    TPW_CHECK_ARG(C.pieces < (1LL << 31), "tpw_cache_attention: more than 2^34 numbers of queries of a slice");
    if (back) cache_convert_kernel<__half, __nv_bfloat16><<<(unsigned)blocks, 256, 0, s>>>(C);
    else cache_convert_kernel<__nv_bfloat16, __half><<<(unsigned)blocks, 256, 0, s>>>(C);
    TPW_LAUNCH_OK("cache_convert_kernel");
    return TPW_OK;
}

} // namespace tpw
