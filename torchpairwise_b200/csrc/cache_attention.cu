// Attention over a cache of quantised keys and values: which kernel.
#include "cache.cuh"

namespace tpw {

static int few(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s) {
    TPW_CHECK_ARG(P.group * P.Nq < (1LL << 30), "tpw_cache_attention: more than 2^30 query rows to a key head");
    return P.c.bits == 4 ? cache_few_4(P, scratch, bytes, s) : cache_few_8(P, scratch, bytes, s);
}

long long cache_attention_bytes(const CacheAttnParams &P) {
    long long bytes = -1;
    few(P, nullptr, &bytes, nullptr);
    return bytes;
}

int cache_attention(const CacheAttnParams &P, void *scratch, cudaStream_t s) { return few(P, scratch, nullptr, s); }

} // namespace tpw
