// Attention over a cache of quantised keys and values: a warp to a query row, a lane to four neighbouring features, on the CUDA cores.
#include "cache.cuh"

namespace tpw {
namespace {

template <typename T> __global__ void __launch_bounds__(256) cache_attention_kernel(const CacheAttnParams P) {
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= P.c.B * P.Hq * P.Nq) return;
    const int i = (int)(r % P.Nq), h = (int)(r / P.Nq % P.Hq), b = (int)(r / P.Nq / P.Hq), hk = (int)(h / P.group), W = P.c.width, D = P.c.D;
    const CacheSeen see(P, b);
    const int w = lane >> 3, group = P.c.groups > 1 ? w : 0, n = D - 4 * lane;
    // the first of this lane's codes in a row of keys and of values
    const int key_at = ((lane >> 1 & 3) * W + w) * 8 + 4 * (lane & 1), value_at = ((lane & 7) * W + w) * 4;
    float q[4] = {}, o[4] = {};
    for (int k = 0; k < 4; ++k)
        if (k < n) q[k] = (float)(static_cast<const T *>(P.q)[b * P.q_s[0] + i * P.q_s[1] + h * P.q_s[2] + 4 * lane + k]);
    auto value = [&](int which, long long place, int at, int k) {
        const unsigned char *row = P.c.codes[which] + place * P.c.row_bytes;
        const int code = P.c.bits == 8 ? row[at + k] : row[(at + k) / 2] >> (4 * (k & 1)) & 15;
        const uint32_t scales = P.c.scales[which][place * P.c.groups + group];
        return fmaf((float)code, step_of(scales), zero_of(scales));
    };
    float m = -INFINITY, l = 0.f;
    const int lo = see.lo(i), hi = see.hi(i);
    for (int j = lo; j < hi; ++j) {
        const long long place = ((long long)b * P.c.H + hk) * P.c.capacity + j;
        float s = 0.f;
        for (int k = 0; k < 4; ++k)
            if (k < n) s = fmaf(q[k], value(0, place, key_at, k), s);
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= P.scale_log2;
        const float top = s > m || s != s ? s : m, by = exp2f(m - top), p = exp2f(s - top);
        l = l * by + p;
        for (int k = 0; k < 4; ++k)
            if (k < n) o[k] = fmaf(p, value(1, place, value_at, k), o[k] * by);
        m = top;
    }
    const bool none = hi <= lo;
    for (int k = 0; k < 4; ++k)
        if (k < n) static_cast<T *>(P.out)[((b * P.Nq + i) * P.Hq + h) * D + 4 * lane + k] = (T)(none ? 0.f : o[k] / l);
    if (lane == 0 && P.lse) P.lse[r] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

} // namespace

long long cache_attention_bytes(const CacheAttnParams &) { return 0; }

int cache_attention(const CacheAttnParams &P, void *, cudaStream_t s) {
    const long long blocks = (P.c.B * P.Hq * P.Nq + 7) / 8;
    TPW_CHECK_ARG(blocks < (1LL << 31), "tpw_cache_attention: more than 2^31 blocks of work");
    if (P.dtype == TPW_F32) cache_attention_kernel<float><<<(unsigned)blocks, 256, 0, s>>>(P);
    else if (P.dtype == TPW_F16) cache_attention_kernel<__half><<<(unsigned)blocks, 256, 0, s>>>(P);
    else cache_attention_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, s>>>(P);
    TPW_LAUNCH_OK("cache_attention_kernel");
    return TPW_OK;
}

} // namespace tpw
