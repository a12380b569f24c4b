// Attention over a cache of quantised keys and values: which kernel, and how many CTAs share a sequence.
#include "cache.cuh"

namespace tpw {

long long cache_attention_bytes(const CacheAttnParams &) { return 0; }

int cache_attention(const CacheAttnParams &P, void *, cudaStream_t s) {
    const long long rows = P.group * P.Nq;
    TPW_CHECK_ARG(rows < (1LL << 30), "tpw_cache_attention: more than 2^30 query rows to a key head");
    const int per = P.dtype == TPW_F32 || rows <= 8 ? 8 : 16, row_blocks = (int)((rows + per - 1) / per);
    // CTAs of a cluster: about four turns of two CTAs on every SM, at least 512 keys each
    const long long items = P.c.B * P.c.H * row_blocks, want = 8LL * sm_count();
    int splits = 1;
    while (splits < 8 && 2 * splits * items <= want && P.c.capacity >= 1024LL * splits) splits *= 2;
    return P.c.bits == 4 ? cache_few_4(P, (int)rows, row_blocks, splits, s) : cache_few_8(P, (int)rows, row_blocks, splits, s);
}

} // namespace tpw
