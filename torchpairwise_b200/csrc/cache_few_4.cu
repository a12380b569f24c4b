// Attention of few query rows over a cache in 4 bits: instances of cache_few.cuh, in a source of their own so that both compile at once.
#include "cache_few.cuh"

namespace tpw {
int cache_few_4(const CacheAttnParams &P, void *scratch, long long *bytes, cudaStream_t s) { return launch_width<4>(P, scratch, bytes, s); }
} // namespace tpw
