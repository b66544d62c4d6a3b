// The tensor-core attention over fp32 pages (pool_attention_mma.cuh).
#include "pool_attention_mma.cuh"

namespace skv {
int attend_fp32(const skv_pool_attention_args& a, cudaStream_t st) { return launch_mma_prec<0>(a, st); }
}  // namespace skv
