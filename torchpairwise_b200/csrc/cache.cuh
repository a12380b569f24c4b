// What the kernels on a cache of quantised keys and values share: its layout (tpw_b200.h has the definition) and the arguments as a kernel
// gets them.
#pragma once
#include "attention.cuh"

namespace tpw {

struct CacheParams {
    unsigned char *codes[2];
    uint32_t *scales[2];      // a group's step (low half) and zero as bfloat16
    const int *lengths;
    long long B, H, capacity;
    int D, bits, groups, width, row_bytes;   // width: features of a row in storage / 32
};

inline int cache_width(long long D) { return D <= 64 ? 2 : (int)((D + 31) / 32); }
inline CacheParams cache_params(const tpw_cache &c) {
    CacheParams P = {};
    for (int w = 0; w < 2; ++w) {
        P.codes[w] = static_cast<unsigned char *>(c.codes[w]);
        P.scales[w] = static_cast<uint32_t *>(c.scales[w]);
    }
    P.lengths = c.lengths;
    P.B = c.B; P.H = c.H; P.capacity = c.capacity;
    P.D = (int)c.D; P.bits = c.bits; P.groups = c.groups;
    P.width = cache_width(c.D);
    P.row_bytes = P.width * 4 * c.bits;
    return P;
}

struct CacheAttnParams {
    CacheParams c;
    const void *q;
    long long q_s[3];         // batch, token, head
    void *out;
    float *lse;
    long long Nq, Hq, group, window;
    int causal, dtype;
    double scale;
    float scale_log2;
    int *status;
};

// cache_rows.cu
int cache_write(const CacheParams &P, const tpw_cache_rows &rows, cudaStream_t s);
int cache_read(const CacheParams &P, const tpw_cache_rows &rows, cudaStream_t s);
// what cache_attention.cu does beside, for tokens from the block of 128 on that the last `last` (0: all) of a sequence begin in:
// the highest magnitudes of kRangeParts parts of every head, [2, B, H, kRangeParts]
constexpr int kRangeParts = 16;
int cache_ranges(const CacheParams &P, long long last, uint32_t *highest, cudaStream_t s);
// every sequence's keys and values, those before the last `last` (0: none) and their block of 128 tokens left out, at [batch, token, head] strides of x;
// what is not stored or left out is not written.  With `highest` each head's are brought below 2^bring by a power of two.
int cache_expand(const CacheParams &P, int dtype, void *const (&x)[2], const int64_t (&stride)[3], long long last, const uint32_t *highest, const int (&bring)[2], cudaStream_t s);
// bfloat16 rows (strides of batch, token and head) to dense half precision ones and, `back`, the other way, times a head's highest power of two over 2^bring
int cache_convert(bool back, const void *from, void *to, const int64_t (&stride)[3], const uint32_t *highest, int bring, long long B, long long N, long long Hq, long long H, long long D,
                  cudaStream_t s);
// cache_attention.cu; -1: refused
long long cache_attention_bytes(const CacheAttnParams &P);
int cache_attention(const CacheAttnParams &P, void *scratch, long long bytes, cudaStream_t s);
// cache_few_4.cu, cache_few_8.cu; with `bytes` they only say how much scratch the call wants
int cache_few_4(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s);
int cache_few_8(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s);

#ifdef __CUDACC__
namespace {

__device__ __forceinline__ float step_of(uint32_t scales) { return __uint_as_float(scales << 16); }
__device__ __forceinline__ float zero_of(uint32_t scales) { return __uint_as_float(scales & 0xffff0000u); }

// The keys [lo, hi) that query i of sequence b sees.
struct CacheSeen {
    int length, off, window;   // keys that there are; position of query 0; window: 0 none
    bool causal;
    __device__ __forceinline__ CacheSeen(const CacheAttnParams &P, int b) {
        const int n = P.c.lengths[b], cap = (int)P.c.capacity;
        length = n < 0 ? 0 : n < cap ? n : cap;
        off = length - (int)P.Nq;
        causal = P.causal != 0;
        window = (int)(P.window < cap ? P.window : 0);   // a window over all keys is none
    }
    __device__ __forceinline__ int hi(int i) const {
        const int h = causal && i + off + 1 < length ? i + off + 1 : length;
        return h > 0 ? h : 0;
    }
    __device__ __forceinline__ int lo(int i) const {
        const int l = window ? i + off + 1 - window : 0;
        return l > 0 ? l : 0;
    }
};

} // namespace
#endif
} // namespace tpw
