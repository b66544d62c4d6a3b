// Which pages a query reads: bounds of every page's keys, and the choice of the pages that they rank highest.
//
// Bounds.  For the keys k_t of a page and head, lo_d = min_t k_td and hi_d = max_t k_td are kept in 8 bits, rounded
// outwards, in units of one power of two: dividing by it is exact, so equal pages have equal bounds however they are computed.
// Then  q k_t <= sum_d max(q_d lo_d, q_d hi_d) = sum_d (q_d > 0 ? q_d hi_d : q_d lo_d)  for every token of the page.
//
// Score.  With the query in 8 bits (n = rint(q / t), t a power of two as well) that sum is
//     max(n, 0) . highs + min(n, 0) . lows,
// a product of whole numbers with the 2 D bytes that a page's bounds are: at most 127 * 127 * D < 2^24, so that 32-bit floats
// hold every partial sum exactly.  The choice does not depend on any order of additions, and ties go to the lowest page.
#include "pool.cuh"

namespace skv {

// The least power of two of which 127 reach top, by its exponent + 127: 2^x m with m < 2 is at most 127 * 2^(x - 6) iff
// m <= 127/64.
__device__ __forceinline__ int step_exp(float top) {
    const uint32_t u = __float_as_uint(top);
    if (u == 0) return 127;
    return max(1, (int)(u >> 23) - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5));
}
__device__ __forceinline__ float exp_of(int e) { return __uint_as_float((uint32_t)e << 23); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float warp_max_nan(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// x / step rounded down (the product with a power of two is exact unless it falls below the smallest float).
__device__ __forceinline__ int down(float x, float inverse) {
    const float v = __fmul_rn(x, inverse);
    return v == 0.0f && x < 0.0f ? -1 : (int)floorf(v);
}
__device__ __forceinline__ int up(float x, float inverse) { return -down(-x, inverse); }

// ---------------------------------------------------------------------------------------- bounds
constexpr int kBoundsThreads = 256;

// The pages of all sequences that are to be looked at, numbered through; every thread of the block calls prepare.
struct TouchedPages {
    int64_t before[kBoundsThreads + 1];   // pages of the sequences before thread t's
    int64_t part[kBoundsThreads / 32];

    static __device__ __forceinline__ int tokens(const skv_pool_bounds_args& a, int b) {
        const int64_t n = __ldg(a.lengths + b), cap = (int64_t)a.pool.table_width * a.pool.page_size;
        if ((n < 0 || n > cap) && a.error_flag) atomicExch(a.error_flag, 1);
        return (int)max((int64_t)0, min(n, min(cap, (int64_t)0x7fffff00)));
    }
    static __device__ __forceinline__ int first(const skv_pool_bounds_args& a, int b) {
        return a.start ? max(0, __ldg(a.start + b)) / a.pool.page_size : 0;
    }
    static __device__ __forceinline__ int count(const skv_pool_bounds_args& a, int b) {
        const int start = a.start ? __ldg(a.start + b) : 0, n = tokens(a, b);
        return start >= n ? 0 : (n - 1) / a.pool.page_size + 1 - max(0, start) / a.pool.page_size;
    }
    __device__ __forceinline__ void prepare(const skv_pool_bounds_args& a) {
        const int tid = threadIdx.x, lane = tid & 31, B = a.pool.batch, per = (B + kBoundsThreads - 1) / kBoundsThreads;
        int64_t mine = 0;
        for (int b = tid * per; b < min(B, (tid + 1) * per); ++b) mine += count(a, b);
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) part[tid >> 5] = incl;
        __syncthreads();
        for (int w = 0; w < (tid >> 5); ++w) incl += part[w];
        if (tid == 0) before[0] = 0;
        before[tid + 1] = incl;
        __syncthreads();
    }
    __device__ __forceinline__ int64_t total() const { return before[kBoundsThreads]; }
    // Page `at` of all: its sequence and its number there.
    __device__ __forceinline__ void find(const skv_pool_bounds_args& a, int64_t at, int& b, int& j) const {
        int lo = 0, hi = kBoundsThreads - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= at) lo = mid; else hi = mid - 1;
        }
        const int per = (a.pool.batch + kBoundsThreads - 1) / kBoundsThreads;
        int64_t rest = at - before[lo];
        for (b = lo * per;; ++b) {
            const int n = count(a, b);
            if (rest < n) break;
            rest -= n;
        }
        j = first(a, b) + (int)rest;
    }
};

// The least and the largest of 8 columns over the rows that a lane has seen.  fp16 rows are compared two values at a time as they are.
template <int PREC> struct Extremes {
    float lo[8], hi[8];
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int i = 0; i < 8; ++i) { lo[i] = INFINITY; hi[i] = -INFINITY; }
    }
    __device__ __forceinline__ void add(const PoolRaw<PREC, 8>& x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x.get(i);
            lo[i] = min_nan(lo[i], y);
            hi[i] = max_nan(hi[i], y);
        }
    }
    __device__ __forceinline__ void join(int from) {   // with lane `from`'s
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = min_nan(lo[i], __shfl_sync(0xffffffffu, lo[i], from));
            hi[i] = max_nan(hi[i], __shfl_sync(0xffffffffu, hi[i], from));
        }
    }
    __device__ __forceinline__ float low(int i) const { return lo[i]; }
    __device__ __forceinline__ float high(int i) const { return hi[i]; }
};
template <> struct Extremes<1> {
    __half2 lo[4], hi[4];
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int i = 0; i < 4; ++i) { lo[i] = __float2half2_rn(INFINITY); hi[i] = __float2half2_rn(-INFINITY); }
    }
    __device__ __forceinline__ void add(const PoolRaw<1, 8>& x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 y = *reinterpret_cast<const __half2*>(&x.w[i]);
            lo[i] = __hmin2_nan(lo[i], y);
            hi[i] = __hmax2_nan(hi[i], y);
        }
    }
    __device__ __forceinline__ void join(int from) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = __hmin2_nan(lo[i], __shfl_sync(0xffffffffu, lo[i], from));
            hi[i] = __hmax2_nan(hi[i], __shfl_sync(0xffffffffu, hi[i], from));
        }
    }
    __device__ __forceinline__ float low(int i) const { return i & 1 ? __high2float(lo[i / 2]) : __low2float(lo[i / 2]); }
    __device__ __forceinline__ float high(int i) const { return i & 1 ? __high2float(hi[i / 2]) : __low2float(hi[i / 2]); }
};

// A warp a run of (page, head) items: an item's rows are one block of memory, 8 values a lane.  VEC: D a multiple of 8, at most
// 256, int4 groups of whole lanes, payload on 16-byte boundaries; else value by value, the rows read twice.
template <int PREC, bool VEC>
__global__ void __launch_bounds__(kBoundsThreads) pool_bounds_kernel(const __grid_constant__ skv_pool_bounds_args a) {
    __shared__ TouchedPages s;
    const int lane = threadIdx.x & 31, D = a.pool.head_dim, P = a.pool.page_size, H = a.pool.heads;
    // up to 32 sequences a warp numbers by itself, a lane a sequence
    const bool few = a.pool.batch <= 32;
    int64_t mine = 0, before = 0, all;
    if (few) {
        before = mine = lane < a.pool.batch ? TouchedPages::count(a, lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        all = __shfl_sync(0xffffffffu, before, 31);
        before -= mine;
    } else {
        s.prepare(a);
        all = s.total();
    }
    const int64_t items = all * H, warp = (int64_t)blockIdx.x * (kBoundsThreads / 32) + (threadIdx.x >> 5);
    const int64_t warps = (int64_t)gridDim.x * (kBoundsThreads / 32);
    const int64_t each = items < warps ? 0 : items >> 32 ? items / warps : (uint32_t)items / (uint32_t)warps, more = items - each * warps;
    const int64_t i0 = each * warp + min(warp, more), i1 = i0 + each + (warp < more);
    if (i0 >= i1) return;
    const int64_t page0 = i0 >> 32 ? i0 / H : (uint32_t)i0 / (uint32_t)H;
    int b = 0, j = 0, h = (int)(i0 - page0 * H), left = 0, rows = 0;   // left: pages of the sequence from this one on
    int64_t page = -1;
    auto take_page = [&]() {
        const int64_t first_row = pool_row(a.pool, b, (int64_t)j * P);
        if (first_row < 0 && a.error_flag) atomicExch(a.error_flag, 1);
        page = first_row < 0 ? -1 : first_row >> 32 ? first_row / P : (uint32_t)first_row / (uint32_t)P;   // counted in (page, head) blocks
        rows = min(P, TouchedPages::tokens(a, b) - j * P);
    };
    if (few) {
        b = 31 - __clz(__ballot_sync(0xffffffffu, mine > 0 && before <= page0));   // (the last sequence with pages that starts there or before)
        j = TouchedPages::first(a, b) + (int)(page0 - __shfl_sync(0xffffffffu, before, b));
    } else {
        s.find(a, page0, b, j);
    }
    left = TouchedPages::first(a, b) + TouchedPages::count(a, b) - j;
    take_page();
    for (int64_t item = i0;;) {
        if (page >= 0) {
            const int64_t page_head = page + h, row = page_head * P;
            int8_t* out = a.bounds + page_head * 2 * D;
            if constexpr (VEC) {
                const int lanes = D / 8, at_once = 32 / lanes, r0 = lane / lanes, col = lane % lanes * 8;
                constexpr int FLY = PREC == 0 ? 4 : 8;
                Extremes<PREC> x;
                x.start();
                // (a row that is not there is read as the page's first again: its values change nothing)
                for (int r = 0; r < rows; r += FLY * at_once) {
                    PoolRaw<PREC, 8> y[FLY];
#pragma unroll
                    for (int f = 0; f < FLY; ++f) {
                        const int mine = r + f * at_once + r0;
                        y[f].load(a.pool, false, row + (r0 < at_once && mine < rows ? mine : 0), col);
                    }
#pragma unroll
                    for (int f = 0; f < FLY; ++f) x.add(y[f]);
                }
                for (int g = 1; g < at_once; ++g) x.join((lane + g * lanes) % (at_once * lanes));   // (lanes behind the groups: unused)
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max_nan(top, max_nan(fabsf(x.low(i)), fabsf(x.high(i))));
                top = warp_max_nan(top);
                const bool finite = top < INFINITY;
                const int e = finite ? step_exp(top) : 127;
                const float inverse = exp_of(254 - e);
                // the first group of lanes writes the lows, the second the highs; one group writes both
                for (int side = r0 >= at_once ? 2 : at_once > 1 ? r0 : 0; side < 2; side += at_once > 1 ? 2 : 1) {
                    uint32_t w[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int n = down(side ? -x.high(i) : x.low(i), inverse);
                        w[i / 4] |= (uint32_t)((side ? -n : n) & 255) << (8 * (i % 4));
                    }
                    *reinterpret_cast<uint2*>(out + side * D + col) = finite ? make_uint2(w[0], w[1]) : make_uint2(0, 0);
                }
                if (lane == 0) a.steps[page_head] = finite ? exp_of(e) : INFINITY;
            } else {
                float top = 0.0f;
                for (int r = 0; r < rows; ++r)
                    for (int d = lane; d < D; d += 32)
                        top = max_nan(top, fabsf(pool_value<PREC>(a.pool, false, row + r, d, PREC == 3 ? d / a.pool.int4_group : 0)));
                top = warp_max_nan(top);
                const bool finite = top < INFINITY;
                const int e = finite ? step_exp(top) : 127;
                const float inverse = exp_of(254 - e);
                for (int d = lane; d < D; d += 32) {
                    float lo = INFINITY, hi = -INFINITY;
                    for (int r = 0; r < rows; ++r) {
                        const float y = pool_value<PREC>(a.pool, false, row + r, d, PREC == 3 ? d / a.pool.int4_group : 0);
                        lo = fminf(lo, y);
                        hi = fmaxf(hi, y);
                    }
                    out[d] = (int8_t)(finite ? down(lo, inverse) : 0);
                    out[D + d] = (int8_t)(finite ? up(hi, inverse) : 0);
                }
                if (lane == 0) a.steps[page_head] = finite ? exp_of(e) : INFINITY;
            }
        }
        if (++item >= i1) break;
        if (++h < H) continue;
        h = 0;
        if (--left > 0) {
            ++j;
        } else {
            do ++b; while ((left = TouchedPages::count(a, b)) == 0);
            j = TouchedPages::first(a, b);
        }
        take_page();
    }
}

template <int PREC>
int launch_bounds(const skv_pool_bounds_args& a, cudaStream_t st) {
    const int D = a.pool.head_dim;
    const bool vec = D % 8 == 0 && D <= 256 && (reinterpret_cast<uintptr_t>(a.pool.k) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(a.bounds) & 7) == 0 && (PREC != 3 || a.pool.int4_group % 8 == 0);
    const int64_t most = (int64_t)a.pool.batch * a.pool.table_width * a.pool.heads;   // (page, head) items at most
    const int64_t ctas = (most + kBoundsThreads / 32 - 1) / (kBoundsThreads / 32), resident = (int64_t)sm_count() * 4;
    const unsigned grid = (unsigned)(ctas < resident ? ctas : resident);
    if (vec) pool_bounds_kernel<PREC, true><<<grid, kBoundsThreads, 0, st>>>(a);
    else pool_bounds_kernel<PREC, false><<<grid, kBoundsThreads, 0, st>>>(a);
    return check_launch("pool_bounds");
}

// ---------------------------------------------------------------------------------------- scores
// What query i of sequence b sees (as in pool_attention.cuh).
__device__ __forceinline__ int select_tokens(const skv_pool_select_args& a, int b) {
    const int64_t n = __ldg(a.lengths + b), cap = (int64_t)a.table_width * a.page_size;
    return (int)max((int64_t)0, min(n, min(cap, (int64_t)0x7fffff00)));
}
__device__ __forceinline__ int select_pages(const skv_pool_select_args& a, int b, int i) {
    const int tokens = select_tokens(a, b), fresh = a.new_lengths ? __ldg(a.new_lengths + b) : a.S_q;
    const int seen = i >= fresh ? 0 : a.causal ? max(0, tokens - fresh + 1 + i) : tokens;
    return seen > 0 ? (seen - 1) / a.page_size + 1 : 0;
}

// Order-preserving image of a score; a page whose step is not finite is above all, one without a number below.
__device__ __forceinline__ uint32_t score_key(float dot, float t, float step) {
    return score_bits(step < INFINITY ? __fmul_rn(__fmul_rn(dot, t), step) : INFINITY);
}

// Query rows n = rint(q / t) as [min(n, 0) (D), max(n, 0) (D)], put(place, n) for each place, and t; a warp a row.
// Returns the sum of all n.
template <class T, class Put>
__device__ __forceinline__ int whole_query(const T* q, int D, Put put, float* t_out) {
    const int lane = threadIdx.x & 31;
    float top = 0.0f;
    for (int d = lane; d < D; d += 32) top = max_nan(top, fabsf(to_float(q[d])));
    top = warp_max_nan(top);
    const bool finite = top < INFINITY;
    const int e = finite ? step_exp(top) : 127;
    const float inverse = exp_of(254 - e);
    int sum = 0;
    for (int d = lane; d < D; d += 32) {
        const int n = finite ? (int)rintf(__fmul_rn(to_float(q[d]), inverse)) : 0;
        sum += n;
        put(d, min(n, 0));
        put(D + d, max(n, 0));
    }
    if (lane == 0) *t_out = exp_of(e);
    return __reduce_add_sync(0xffffffffu, sum);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kScoreWarps = 8, kScoreTiles = 4;   // column tiles of 8 that a block takes

// Scores of 16 pages a warp for the columns of a block.  Columns are (new token, query head): the rep heads of a token fill
// `span` (a power of two up to 8) of them, the head repeated in those that are over, so that the largest of a token
// is found with its neighbours; more than 8 heads take several tiles.  Lane g = lane / 4, c = lane % 4 holds 16 bytes c of every 64
// of pages g and g + 8.  A byte x becomes an fp16 operand by its place alone: the bits of x + 128 are those of the subnormal
// (x + 128) 2^-24, so an MMA over a word of 4 bytes a lane gives 2^-24 (n . x + 128 sum n), exactly (at most 255 * 127 * 256 < 2^23 of
// these units); the accumulators start at what is too much.  (Integer MMAs are not native here.)
template <class T, int SEGS>
__global__ void __launch_bounds__(32 * kScoreWarps) page_scores_kernel(const __grid_constant__ skv_pool_select_args a, int span) {
    extern __shared__ __align__(16) __half s_raw[];
    __half* s_q = s_raw;                                          // [columns][64 * SEGS + 8], the bytes 0, 2, 1, 3 of each word
    __shared__ float s_t[8 * kScoreTiles], s_start[8 * kScoreTiles];
    constexpr int BYTES = 64 * SEGS, PITCH = BYTES + 8;
    const int D = a.head_dim, H = a.heads, rep = a.q.heads / H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.z / H, h = blockIdx.z % H;
    const int pages = (select_tokens(a, b) + a.page_size - 1) / a.page_size;
    if (pages <= a.keep || blockIdx.x * kScoreWarps * 16 >= pages) return;   // (all are kept, or none here)
    const int head_tiles = (rep + span - 1) / span;               // tiles of a token (1 unless rep > 8)
    const int block_tokens = head_tiles > 1 ? 1 : 8 * kScoreTiles / span;
    const int i0 = blockIdx.y * block_tokens;
    for (int first = 0; first < head_tiles; first += kScoreTiles) {
        // (further rounds are for more than 8 * kScoreTiles heads only: their largest joins what is written already)
        const int tiles = head_tiles > 1 ? min(kScoreTiles, head_tiles - first)
                                         : (min(block_tokens, a.S_q - i0) * span + 7) / 8;
        __syncthreads();
        for (int col = warp; col < 8 * tiles; col += kScoreWarps) {
            const int i = head_tiles > 1 ? i0 : min(a.S_q - 1, i0 + col / span);
            int head = head_tiles > 1 ? 8 * first + col : col % span;
            if (head >= rep) head = rep - 1;
            __half* to = s_q + col * PITCH;
            for (int p = 2 * D + lane; p < BYTES; p += 32) to[p] = __float2half_rn(0.0f);   // (whole words: D is a multiple of 8)
            const int sum = whole_query(
                static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + (int64_t)(h * rep + head) * a.q.stride_h + i * a.q.stride_s, D,
                [&](int p, int n) { to[(p & ~3) + (p & 1) * 2 + (p >> 1 & 1)] = __int2half_rn(n); }, s_t + col);
            if (lane == 0) s_start[col] = -128.0f * (float)sum * 0x1p-24f;
        }
        __syncthreads();
        const int g = lane >> 2, c = lane & 3;
        for (int p0 = (blockIdx.x * kScoreWarps + warp) * 16; p0 < pages; p0 += gridDim.x * kScoreWarps * 16) {
            uint4 x[2][SEGS];
            float step[2];
            bool named[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int j = p0 + g + 8 * r;
                const int page = j < pages ? __ldg(a.block_table + b * a.table_stride + j) : -1;
                named[r] = page >= 0 && page < a.num_pages;
                if (j < pages && !named[r] && a.error_flag) atomicExch(a.error_flag, 1);
                const int64_t at = named[r] ? (int64_t)page * H + h : 0;
                step[r] = named[r] ? __ldg(a.steps + at) : 1.0f;
                const uint4* row = reinterpret_cast<const uint4*>(a.bounds + at * 2 * D);
#pragma unroll
                for (int s = 0; s < SEGS; ++s)
                    x[r][s] = named[r] && 64 * s + 16 * c < 2 * D ? __ldg(row + 4 * s + c) : make_uint4(0, 0, 0, 0);
            }
            float best[2] = {-INFINITY, -INFINITY};               // more than 8 heads
            for (int t = 0; t < tiles; ++t) {
                const float at0 = s_start[8 * t + 2 * c], at1 = s_start[8 * t + 2 * c + 1];
                float acc[4] = {at0, at1, at0, at1};
                const __half* column = s_q + (8 * t + g) * PITCH + 16 * c;
#pragma unroll
                for (int s = 0; s < SEGS; ++s) {
                    const uint4 y0 = *reinterpret_cast<const uint4*>(column + 64 * s), y1 = *reinterpret_cast<const uint4*>(column + 64 * s + 8);
                    const uint32_t u[4] = {x[0][s].x, x[0][s].y, x[0][s].z, x[0][s].w}, v[4] = {x[1][s].x, x[1][s].y, x[1][s].z, x[1][s].w};
                    const uint32_t y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        mma_f16(acc, (u[w] & 0x00FF00FFu) ^ 0x00800080u, (v[w] & 0x00FF00FFu) ^ 0x00800080u,
                                ((u[w] >> 8) & 0x00FF00FFu) ^ 0x00800080u, ((v[w] >> 8) & 0x00FF00FFu) ^ 0x00800080u, y[2 * w], y[2 * w + 1]);
                }
                // columns 2 c and 2 c + 1 of pages g (acc 0, 1) and g + 8
                const float t0 = s_t[8 * t + 2 * c], t1 = s_t[8 * t + 2 * c + 1];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float u = __fmul_rn(acc[2 * r] * 0x1p24f, t0), v = __fmul_rn(acc[2 * r + 1] * 0x1p24f, t1);
                    if (span > 1) u = v = fmaxf(u, v);
                    if (span > 2) u = v = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 1));
                    if (span > 4) u = v = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 2));
                    const int j = p0 + g + 8 * r;
                    if (head_tiles > 1) {
                        best[r] = fmaxf(best[r], u);
                        if (t + 1 < tiles) continue;
                        u = v = best[r];
                    }
                    if (j >= pages) continue;
                    const int i_u = head_tiles > 1 ? i0 : i0 + (8 * t + 2 * c) / span, i_v = i0 + (8 * t + 2 * c + 1) / span;
                    uint32_t* keys = static_cast<uint32_t*>(a.scratch) + ((int64_t)blockIdx.z * a.S_q) * a.table_width + j;
                    if ((head_tiles > 1 ? c == 0 : 2 * c % span == 0) && i_u < a.S_q) {
                        uint32_t key = named[r] ? score_key(u, 1.0f, step[r]) : 0;
                        if (first > 0) key = max(key, keys[(int64_t)i_u * a.table_width]);
                        keys[(int64_t)i_u * a.table_width] = key;
                    }
                    if (span == 1 && i_v < a.S_q) keys[(int64_t)i_v * a.table_width] = named[r] ? score_key(v, 1.0f, step[r]) : 0;
                }
            }
        }
    }
}

// Heads that are not whole 16-byte rows of bounds, or above 256 values: a warp a page and column.
template <class T>
__global__ void __launch_bounds__(32 * kScoreWarps) page_scores_any_kernel(const __grid_constant__ skv_pool_select_args a) {
    extern __shared__ __align__(16) __half s_raw[];
    int8_t* s_q = reinterpret_cast<int8_t*>(s_raw);               // [2 D]
    __shared__ float s_t;
    const int D = a.head_dim, H = a.heads, rep = a.q.heads / H, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.z / H, h = blockIdx.z % H, i = blockIdx.y;
    const int pages = (select_tokens(a, b) + a.page_size - 1) / a.page_size;
    if (pages <= a.keep) return;
    uint32_t* keys = static_cast<uint32_t*>(a.scratch) + ((int64_t)blockIdx.z * a.S_q + i) * a.table_width;
    for (int head = 0; head < rep; ++head) {
        __syncthreads();
        if (warp == 0)
            whole_query(static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + (int64_t)(h * rep + head) * a.q.stride_h + i * a.q.stride_s, D,
                        [&](int p, int n) { s_q[p] = (int8_t)n; }, &s_t);
        __syncthreads();
        for (int j = blockIdx.x * kScoreWarps + warp; j < pages; j += gridDim.x * kScoreWarps) {
            const int page = __ldg(a.block_table + b * a.table_stride + j);
            const bool named = page >= 0 && page < a.num_pages;
            if (!named && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
            const int64_t at = named ? (int64_t)page * H + h : 0;
            int sum = 0;
            if (named)
                for (int d = lane; d < 2 * D; d += 32) sum += (int)s_q[d] * (int)__ldg(a.bounds + at * 2 * D + d);
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) {
                const uint32_t key = named ? score_key((float)sum, s_t, __ldg(a.steps + at)) : 0;
                keys[j] = head == 0 ? key : max(keys[j], key);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------- the choice
constexpr int kSelectThreads = 256, kSelectHeld = 8;   // keys that a thread keeps in registers

// A block a (sequence, key head, new token).  The want-th largest key is found bit by bit (how many keys are at least a
// candidate), then the pages above it, and the first of those equal to it, are listed in order.
__global__ void __launch_bounds__(kSelectThreads) page_select_kernel(const __grid_constant__ skv_pool_select_args a) {
    __shared__ int s_count[3], s_part[2][kSelectThreads / 32];
    __shared__ uint32_t s_min[kSelectThreads / 32], s_max[kSelectThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t unit = blockIdx.x;
    const int i = (int)(unit % a.S_q), b = (int)(unit / a.S_q / a.heads);
    const int pages = select_pages(a, b, i);
    int32_t* out = a.pages + unit * a.keep;
    if (tid == 0 && a.error_flag && __ldg(a.lengths + b) != select_tokens(a, b)) atomicExch(a.error_flag, 1);
    if (pages <= a.keep) {
        for (int k = tid; k < a.keep; k += kSelectThreads) out[k] = k < pages ? k : -1;
        return;
    }
    const int lo = a.first, hi = pages - a.recent, want = a.keep - a.first - a.recent;   // of the pages [lo, hi), more than want
    const uint32_t* keys = static_cast<const uint32_t*>(a.scratch) + unit * a.table_width;
    for (int k = tid; k < a.first; k += kSelectThreads) out[k] = k;
    for (int k = tid; k < a.recent; k += kSelectThreads) out[a.keep - a.recent + k] = hi + k;
    if (want == 0) return;
    uint32_t held[kSelectHeld], least = 0xffffffffu, most = 0;
    const bool all = hi - lo <= kSelectThreads * kSelectHeld;
    if (all) {
#pragma unroll
        for (int k = 0; k < kSelectHeld; ++k) {
            const int j = lo + tid + k * kSelectThreads;
            held[k] = j < hi ? keys[j] : 0;
            if (j < hi) { least = min(least, held[k]); most = max(most, held[k]); }
        }
    } else {
        for (int j = lo + tid; j < hi; j += kSelectThreads) { least = min(least, keys[j]); most = max(most, keys[j]); }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) { s_min[warp] = least; s_max[warp] = most; }
    if (tid < 3) s_count[tid] = 0;
    __syncthreads();
    for (int w = 0; w < kSelectThreads / 32; ++w) { least = min(least, s_min[w]); most = max(most, s_max[w]); }
    int round = 0;
    auto count_from = [&](uint32_t x) {   // keys >= x; x > 0
        int n = 0;
        if (all) {
#pragma unroll
            for (int k = 0; k < kSelectHeld; ++k) n += held[k] >= x;
        } else {
            for (int j = lo + tid; j < hi; j += kSelectThreads) n += keys[j] >= x;
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0 && n) atomicAdd(&s_count[round % 3], n);
        if (tid == 0) s_count[(round + 1) % 3] = 0;
        __syncthreads();
        return s_count[round++ % 3];
    };
    const int differ = 32 - __clz(least ^ most);                 // bits below those that all keys share
    uint32_t at = differ == 32 ? 0 : most >> differ << differ;
    bool exact = false;                                          // as many keys are at least `at` as are wanted
    for (int bit = differ - 1; bit >= 0 && !exact; --bit) {
        const uint32_t x = at | 1u << bit;
        const int n = count_from(x);
        if (n >= want) at = x;
        exact = n == want;
    }
    const int above = exact ? want : at == 0xffffffffu ? 0 : count_from(at + 1), ties = want - above;
    int before = 0, equal_before = 0;                            // of the keys below those looked at
    for (int j0 = lo, k = 0; j0 < hi; j0 += kSelectThreads, ++k) {
        const int j = j0 + tid;
        const uint32_t key = j < hi ? keys[j] : 0;
        const bool over = j < hi && (exact ? key >= at : key > at), equal = j < hi && !exact && key == at;
        const unsigned o = __ballot_sync(0xffffffffu, over), e = __ballot_sync(0xffffffffu, equal), mask = (1u << lane) - 1;
        if (lane == 0) s_part[k & 1][warp] = __popc(o) | __popc(e) << 16;
        __syncthreads();
        int packed = 0, total = 0;
        for (int w = 0; w < kSelectThreads / 32; ++w) {
            if (w < warp) packed += s_part[k & 1][w];
            total += s_part[k & 1][w];
        }
        const int o_before = before + (packed & 0xffff) + __popc(o & mask), e_before = equal_before + (packed >> 16) + __popc(e & mask);
        if (over || (equal && e_before < ties)) out[a.first + o_before + min(e_before, ties)] = j;
        before += total & 0xffff;
        equal_before += total >> 16;
    }
}

template <class T>
int launch_select(const skv_pool_select_args& a, cudaStream_t st) {
    const int D = a.head_dim, H = a.heads, rep = a.q.heads / H;
    const int64_t groups = (int64_t)a.batch * H;
    const bool vec = D % 8 == 0 && D <= 256 && (reinterpret_cast<uintptr_t>(a.bounds) & 15) == 0;
    if (a.table_width > a.keep && a.keep > a.first + a.recent) {
        if (vec) {
            int span = 1;
            while (span < rep && span < 8) span *= 2;
            const int block_tokens = rep > 8 ? 1 : 8 * kScoreTiles / span;
            const int chunks = (a.table_width + 16 * kScoreWarps - 1) / (16 * kScoreWarps);
            const dim3 grid(chunks, (a.S_q + block_tokens - 1) / block_tokens, (unsigned)groups);
            const int segs = D <= 64 ? 2 : D <= 128 ? 4 : 8;
            const size_t smem = (size_t)8 * kScoreTiles * (64 * segs + 8) * sizeof(__half);
            if (segs == 2) page_scores_kernel<T, 2><<<grid, 32 * kScoreWarps, smem, st>>>(a, span);
            else if (segs == 4) page_scores_kernel<T, 4><<<grid, 32 * kScoreWarps, smem, st>>>(a, span);
            else page_scores_kernel<T, 8><<<grid, 32 * kScoreWarps, smem, st>>>(a, span);
        } else {
            const dim3 grid((a.table_width + 8 * kScoreWarps - 1) / (8 * kScoreWarps), a.S_q, (unsigned)groups);
            page_scores_any_kernel<T><<<grid, 32 * kScoreWarps, 2 * (size_t)D, st>>>(a);
        }
        if (const int rc = check_launch("pool_select")) return rc;
    }
    page_select_kernel<<<(unsigned)(groups * a.S_q), kSelectThreads, 0, st>>>(a);
    return check_launch("pool_select");
}

}  // namespace skv

using namespace skv;

extern "C" {

int skv_pool_bounds(const skv_pool_bounds_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_bounds: null pointer");
    skv_pool_bounds_args a = *args;
    if (!a.pool.v) a.pool.v = a.pool.k;
    if (!a.pool.scale_v) a.pool.scale_v = a.pool.scale_k;
    if (const int rc = check_pool(a.pool, "pool_bounds")) return rc;
    if (a.pool.batch == 0 || a.pool.table_width == 0 || a.pool.num_pages == 0) return SKV_OK;
    if (!a.lengths || !a.bounds || !a.steps) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_bounds: null pointer");
    cudaStream_t st = as_stream(stream);
    switch (a.pool.precision) {
        case 0: return launch_bounds<0>(a, st);
        case 1: return launch_bounds<1>(a, st);
        case 2: return launch_bounds<2>(a, st);
        default: return launch_bounds<3>(a, st);
    }
}

size_t skv_pool_select_scratch_bytes(int batch, int heads, int S_q, int table_width) {
    return batch < 0 || heads < 0 || S_q < 0 || table_width < 0 ? 0 : (size_t)batch * heads * S_q * table_width * 4;
}

int skv_pool_select(const skv_pool_select_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_select: null pointer");
    const skv_pool_select_args& a = *args;
    if (a.batch < 0 || a.num_pages < 0 || a.page_size <= 0 || a.heads <= 0 || a.head_dim <= 0 || a.table_width < 0 || a.S_q < 0)
        return fail(SKV_ERR_INVALID_ARGUMENT, "pool_select: bad size");
    if (a.keep < 1 || a.first < 0 || a.recent < 1 || (int64_t)a.first + a.recent > a.keep)
        return fail(SKV_ERR_INVALID_ARGUMENT, "pool_select: %d first and %d recent of %d pages", a.first, a.recent, a.keep);
    if (const int rc = check_rows(a.q, a.batch > 0 && a.S_q > 0, "pool_select", "q")) return rc;
    if (a.q.heads <= 0 || a.q.heads % a.heads)
        return fail(SKV_ERR_SHAPE, "pool_select: %d query heads, %d key heads", a.q.heads, a.heads);
    if (a.batch == 0 || a.S_q == 0) return SKV_OK;
    if (!a.lengths || !a.pages || (a.table_width > 0 && (!a.block_table || !a.scratch)) || (a.num_pages > 0 && (!a.bounds || !a.steps)))
        return fail(SKV_ERR_INVALID_ARGUMENT, "pool_select: null pointer");
    if (a.head_dim > 1024) return fail(SKV_ERR_UNSUPPORTED, "pool_select: head_dim %d above 1024", a.head_dim);
    if ((int64_t)a.batch * a.heads > 65535 || a.S_q > 65535 || (int64_t)a.batch * a.heads * a.S_q > 0x7fffffff)
        return fail(SKV_ERR_TOO_LARGE, "pool_select: %d sequences of %d heads and %d queries", a.batch, a.heads, a.S_q);
    if (a.scratch_bytes < (int64_t)skv_pool_select_scratch_bytes(a.batch, a.heads, a.S_q, a.table_width))
        return fail(SKV_ERR_SCRATCH, "pool_select: scratch of %lld bytes", (long long)a.scratch_bytes);
    cudaStream_t st = as_stream(stream);
    if (a.q.dtype == kF32) return launch_select<float>(a, st);
    if (a.q.dtype == kF16) return launch_select<__half>(a, st);
    return launch_select<__nv_bfloat16>(a, st);
}

}  // extern "C"
