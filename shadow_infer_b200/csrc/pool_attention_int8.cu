// The tensor-core attention over int8 pages (pool_attention_mma.cuh).
#include "pool_attention_mma.cuh"

namespace skv {
int attend_int8(const skv_pool_attention_args& a, cudaStream_t st) { return launch_mma_prec<2>(a, st); }
}  // namespace skv
