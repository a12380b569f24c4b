// Attention of few query rows over a cache in 8 bits: instances of cache_few.cuh, in a source of their own so that both compile at once.
#include "cache_few.cuh"

namespace tpw {
int cache_few_8(const CacheAttnParams &P, int rows, int row_blocks, int splits, cudaStream_t s) { return launch_width<8>({P, rows, row_blocks, splits}, s); }
} // namespace tpw
