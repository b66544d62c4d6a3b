// The attention over fp16 and int8 pages for many query rows a key head (pool_attention_tc.cuh).
#include "pool_attention_tc.cuh"

namespace skv {
int attend_many(const skv_pool_attention_args& a, cudaStream_t st) {
    const bool narrow = a.pool.head_dim <= 64;
    if (a.pool.precision == 1) return narrow ? launch_tc<1, 64>(a, st) : launch_tc<1, 128>(a, st);
    return narrow ? launch_tc<2, 64>(a, st) : launch_tc<2, 128>(a, st);
}
}  // namespace skv
