// The tensor-core attention over int4 pages (pool_attention_mma.cuh).
#include "pool_attention_mma.cuh"

namespace skv {
int attend_int4(const skv_pool_attention_args& a, cudaStream_t st) { return launch_mma_prec<3, false>(a, st); }
}  // namespace skv
