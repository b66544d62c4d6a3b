// The tensor-core attention over lists of fp16 pages (pool_attention_mma.cuh), a source of its own so that it compiles beside the others.
#include "pool_attention_mma.cuh"

namespace skv {
int attend_listed_fp16(const skv_pool_attention_args& a, cudaStream_t st) { return launch_mma_prec<1, true>(a, st); }
}  // namespace skv
