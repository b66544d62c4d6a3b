// The tensor-core attention over lists of int4 pages (pool_attention_mma.cuh), a source of its own so that it compiles beside the others.
#include "pool_attention_mma.cuh"

namespace skv {
int attend_listed_int4(const skv_pool_attention_args& a, cudaStream_t st) { return launch_mma_prec<3, true>(a, st); }
}  // namespace skv
