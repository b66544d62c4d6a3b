// The attention over fp16, int8 and int4 pages for many query rows a key head (pool_attention_tc.cuh).
#include "pool_attention_tc.cuh"

namespace skv {
std::mutex& tc_launches() {
    static std::mutex m;
    return m;
}

int attend_many(const skv_pool_attention_args& a, cudaStream_t st) {
    const int D = a.pool.head_dim;
    if (a.pool.precision == 1) return D <= 64 ? launch_tc<1, 64>(a, st) : D <= 128 ? launch_tc<1, 128>(a, st) : launch_tc<1, 256>(a, st);
    if (a.pool.precision == 3) return D <= 64 ? launch_tc<3, 64>(a, st) : D <= 128 ? launch_tc<3, 128>(a, st) : launch_tc<3, 256>(a, st);
    return D <= 64 ? launch_tc<2, 64>(a, st) : D <= 128 ? launch_tc<2, 128>(a, st) : launch_tc<2, 256>(a, st);
}
}  // namespace skv
