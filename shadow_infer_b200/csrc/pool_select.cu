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
//
// What bounds it.  Bounds of a prompt: HBM, 32768 fp16 tokens of 32 heads of 128 values in 48.4 us, 5.7 TB/s (87 % of the copy
// rate; values compared one by one in 32 bits took 76), of int8 and int4 tokens instructions, 73.9 and 91.3 (each value by itself); of 8 sequences' newest pages: 6.9 us of latency.  A choice: latency, one step after
// the other in one kernel (lengths, table, bounds, queries, products, a cluster's barrier, keys, bins, the list): 1024 pages of 32 heads
// 11.4 us, 2049 pages of 8 heads for 4 query heads each 11.7, 64 sequences of 2 to 256 pages with 8 key heads 16.4, 64 queries of 128 pages
// with 8 key heads 13.7.  Two launches, with the want-th key found bit by bit, took 14 to 27; loads a round ahead of their use
// 0.8 to 2.6 more.
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
// What the kernel is told besides the call's arguments: query heads a key head, tokens a block takes, blocks that share them, and a
// division by the page size as a product (mul = ceil(2^shift / page_size), shift = 31 + ceil(log2 page_size), exact below 2^31).
struct SelectShape {
    int rep, log_span, block_tokens, blocks;
    uint32_t mul;
    int shift;
    __device__ __forceinline__ int pages_of(int tokens) const {   // that tokens > 0 reach
        return tokens > 0 ? (int)(((uint64_t)(uint32_t)(tokens - 1) * mul) >> shift) + 1 : 0;
    }
};

// What query i of sequence b sees (as in pool_attention.cuh).  (The kernel waits for those before it by itself: no read-only loads here and below.)
__device__ __forceinline__ int select_tokens(const skv_pool_select_args& a, int b) {
    const int64_t n = a.lengths[b], cap = (int64_t)a.table_width * a.page_size;
    return (int)max((int64_t)0, min(n, min(cap, (int64_t)0x7fffff00)));
}
__device__ __forceinline__ int select_pages(const skv_pool_select_args& a, const SelectShape& shape, int b, int i, int tokens) {
    const int fresh = a.new_lengths ? a.new_lengths[b] : a.S_q;
    return shape.pages_of(i >= fresh ? 0 : a.causal ? max(0, tokens - fresh + 1 + i) : tokens);
}

// Order-preserving image of a score; a page whose step is not finite is above all (+inf, where a product is too large, among them), one
// without a number below.
__device__ __forceinline__ uint32_t score_key(float dot, float t, float step) {
    return step < INFINITY ? score_bits(__fmul_rn(__fmul_rn(dot, t), step)) : 0xffffffffu;
}

// A query row n = rint(q / t) as [min(n, 0) (D), max(n, 0) (D)], put(place, n) for each place, and t; a warp a row, N values a lane
// that are loaded first.  Returns the sum of all n.
template <int N, class T>
__device__ __forceinline__ void load_query(const T* q, int D, float (&x)[N]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = 32 * k + lane < D ? to_float(q[32 * k + lane]) : 0.0f;
}
template <int N, class Put>
__device__ __forceinline__ int whole_query(const float (&x)[N], int D, float top, Put put, float* t_out) {
    const int lane = threadIdx.x & 31;
    const bool finite = top < INFINITY;
    const int e = finite ? step_exp(top) : 127;
    const float inverse = exp_of(254 - e);
    int sum = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int d = 32 * k + lane;
        if (d >= D) continue;
        const int n = finite ? (int)rintf(__fmul_rn(x[k], inverse)) : 0;
        sum += n;
        put(d, min(n, 0));
        put(D + d, max(n, 0));
    }
    if (lane == 0) *t_out = exp_of(e);
    return sum;
}
template <int N>
__device__ __forceinline__ float largest_of(const float (&x)[N]) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) top = max_nan(top, fabsf(x[k]));
    return warp_max_nan(top);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kSelectWarps = 8, kSelectThreads = 32 * kSelectWarps, kScoreTiles = 4;   // column tiles of 8 that a block takes
constexpr int kSelectCluster = 8;       // most blocks that share a (sequence, key head)
constexpr int kSelectKeys = 4096;        // keys that a block keeps in shared memory


// Scores of 16 pages a warp for the columns of a block.  Columns are (new token, query head): the rep heads of a token fill
// `span` (a power of two up to 8) of them, the head repeated in those that are over, so that the largest of a token
// is found with its neighbours; more than 8 heads take several tiles.  Lane g = lane / 4, c = lane % 4 holds 16 bytes c of every 64
// of pages g and g + 8.  A byte x becomes an fp16 operand by its place alone: the bits of x + 128 are those of the subnormal
// (x + 128) 2^-24, so an MMA over a word of 4 bytes a lane gives 2^-24 (n . x + 128 sum n), exactly (at most 255 * 127 * 256 < 2^23 of
// these units); the accumulators start at what is too much.  (Integer MMAs are not native here.)
// The first pages' loads are on their way while the queries are laid out.
template <class T, int SEGS>
__device__ __forceinline__ void score_pages(const skv_pool_select_args& a, const SelectShape& shape, int rank, int b, int h, int pages, int i0,
                                            __half* s_q, float* s_t, float* s_start, uint32_t* keys, int pitch) {
    constexpr int BYTES = 64 * SEGS, PITCH = BYTES + 8;
    const int D = a.head_dim, H = a.heads, rep = shape.rep, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int log_span = shape.log_span, span = 1 << log_span;
    const int head_tiles = (rep + span - 1) >> log_span;          // tiles of a token (1 unless rep > 8)
    const int g = lane >> 2, c = lane & 3;
    const int32_t* table = a.block_table + b * a.table_stride;
    const int p_first = (rank * kSelectWarps + warp) * 16, p_step = shape.blocks * kSelectWarps * 16;
    for (int first = 0; first < head_tiles; first += kScoreTiles) {
        // (further rounds are for more than 8 * kScoreTiles heads only: their largest joins what is written already)
        const int tiles = head_tiles > 1 ? min(kScoreTiles, head_tiles - first)
                                         : ((min(shape.block_tokens, a.S_q - i0) << log_span) + 7) / 8;
        int ahead[2];                                             // numbers of the pages that are loaded next
#pragma unroll
        for (int r = 0; r < 2; ++r) ahead[r] = p_first + g + 8 * r < pages ? table[p_first + g + 8 * r] : -1;
        if (first > 0) __syncthreads();
        bool laid_out = false;
#pragma unroll 1
        for (int p0 = p_first; p0 < pages || !laid_out; p0 += p_step) {
            uint4 y[2][SEGS];
            float step[2];
            bool named[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int j = p0 + g + 8 * r, page = ahead[r];
                named[r] = j < pages && page >= 0 && page < a.num_pages;
                if (j < pages && !named[r] && a.error_flag) atomicExch(a.error_flag, 1);
                ahead[r] = j + p_step < pages ? table[j + p_step] : -1;
                // (page 0 in place of none, the row's first bytes in place of those behind it: loads without a branch that waits for
                // them; their scores are not used, the queries are zero there)
                const int64_t at = named[r] ? (int64_t)page * H + h : 0;
                const int8_t* row = a.bounds + at * (2 * D);
                step[r] = a.steps[at];
#pragma unroll
                for (int s = 0; s < SEGS; ++s)
                    y[r][s] = *reinterpret_cast<const uint4*>(row + (64 * s + 16 * c < 2 * D ? 64 * s + 16 * c : 0));
            }
            if (!laid_out) {
                laid_out = true;
#pragma unroll 1
                for (int col = warp; col < 8 * tiles; col += kSelectWarps) {
                    const int i = head_tiles > 1 ? i0 : min(a.S_q - 1, i0 + (col >> log_span));
                    const int head = min(rep - 1, head_tiles > 1 ? 8 * first + col : col & (span - 1));
                    float x[SEGS];
                    load_query(static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + (int64_t)(h * rep + head) * a.q.stride_h + i * a.q.stride_s, D, x);
                    __half* to = s_q + col * PITCH;
#pragma unroll 1
                    for (int p = 2 * D + lane; p < BYTES; p += 32) to[p] = __float2half_rn(0.0f);   // (whole words: D is a multiple of 8)
                    const int sum = __reduce_add_sync(0xffffffffu, whole_query(x, D, largest_of(x),
                        [&](int p, int n) { to[(p & ~3) + (p & 1) * 2 + (p >> 1 & 1)] = __int2half_rn(n); }, s_t + col));
                    if (lane == 0) s_start[col] = -128.0f * (float)sum * 0x1p-24f;
                }
                __syncthreads();
            }
            float best[2] = {-INFINITY, -INFINITY};               // more than 8 heads
#pragma unroll 1
            for (int t = 0; t < tiles; ++t) {
                const float at0 = s_start[8 * t + 2 * c], at1 = s_start[8 * t + 2 * c + 1];
                float acc[2][4] = {{at0, at1, at0, at1}, {}};     // (chains of their own: whole numbers add up in any order)
                const __half* column = s_q + (8 * t + g) * PITCH + 16 * c;
#pragma unroll
                for (int s = 0; s < SEGS; ++s) {
                    const uint4 z0 = *reinterpret_cast<const uint4*>(column + 64 * s), z1 = *reinterpret_cast<const uint4*>(column + 64 * s + 8);
                    const uint32_t z[8] = {z0.x, z0.y, z0.z, z0.w, z1.x, z1.y, z1.z, z1.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t u = (&y[0][s].x)[w], v = (&y[1][s].x)[w];
                        mma_f16(acc[w & 1], (u & 0x00FF00FFu) ^ 0x00800080u, (v & 0x00FF00FFu) ^ 0x00800080u,
                                ((u >> 8) & 0x00FF00FFu) ^ 0x00800080u, ((v >> 8) & 0x00FF00FFu) ^ 0x00800080u, z[2 * w], z[2 * w + 1]);
                    }
                }
                // columns 2 c and 2 c + 1 of pages g (acc 0, 1) and g + 8
                const float t0 = s_t[8 * t + 2 * c], t1 = s_t[8 * t + 2 * c + 1];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float u = __fmul_rn(__fmul_rn(acc[0][2 * r] + acc[1][2 * r], 0x1p24f), t0);   // (not 2^24 t: it may pass the largest float)
                    float v = __fmul_rn(__fmul_rn(acc[0][2 * r + 1] + acc[1][2 * r + 1], 0x1p24f), t1);
                    if (span > 1) u = fmaxf(u, v);
                    if (span > 2) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 1));
                    if (span > 4) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 2));
                    const int j = p0 + g + 8 * r;
                    if (head_tiles > 1) {
                        best[r] = fmaxf(best[r], u);
                        if (t + 1 < tiles) continue;
                        u = best[r];
                    }
                    // each lane that has a token's largest writes it, two where a token is a column
                    const int writers = head_tiles > 1 ? 3 : span > 1 ? (span >> 1) - 1 : 0;
                    if (j >= pages || (c & writers)) continue;
                    const int i = head_tiles > 1 ? i0 : i0 + ((8 * t + 2 * c) >> log_span);
                    uint32_t* to = keys + (int64_t)i * pitch + j;
                    if (i < a.S_q) {
                        const uint32_t key = named[r] ? score_key(u, 1.0f, step[r]) : 1;
                        to[0] = first > 0 ? max(key, to[0]) : key;
                    }
                    if (span == 1 && i + 1 < a.S_q) to[pitch] = named[r] ? score_key(v, 1.0f, step[r]) : 1;
                }
            }
        }
    }
}

// Heads that are not whole 16-byte rows of bounds, or above 256 values: a warp a page, a column at a time.
template <class T>
__device__ __forceinline__ void score_pages_any(const skv_pool_select_args& a, const SelectShape& shape, int rank, int b, int h, int pages, int i,
                                                int8_t* s_q, float* s_t,
                                                uint32_t* keys, int pitch) {
    const int D = a.head_dim, H = a.heads, rep = shape.rep, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int head = 0; head < rep; ++head) {
        __syncthreads();
        if (warp == 0) {
            float x[32];                                          // (of up to 1024 values)
            load_query<32>(static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + (int64_t)(h * rep + head) * a.q.stride_h + i * a.q.stride_s, D, x);
            whole_query(x, D, largest_of(x), [&](int p, int n) { s_q[p] = (int8_t)n; }, s_t);
        }
        __syncthreads();
        for (int j = rank * kSelectWarps + warp; j < pages; j += shape.blocks * kSelectWarps) {
            const int page = a.block_table[b * a.table_stride + j];
            const bool named = page >= 0 && page < a.num_pages;
            if (!named && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
            const int64_t at = named ? (int64_t)page * H + h : 0;
            int sum = 0;
            if (named)
                for (int d = lane; d < 2 * D; d += 32) sum += (int)s_q[d] * (int)a.bounds[at * 2 * D + d];
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) {
                const uint32_t key = named ? score_key((float)sum, *s_t, a.steps[at]) : 1;
                keys[(int64_t)i * pitch + j] = head == 0 ? key : max(key, keys[(int64_t)i * pitch + j]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------- the choice
constexpr int kSelectBins = 2048, kSelectList = 256;

struct SelectShared {                       // of a block, or a part of each array for each warp
    int bins[kSelectBins];
    uint32_t keys[kSelectKeys];
    uint32_t list[kSelectList];             // keys of one bin and their pages
    int page[kSelectList];
    uint32_t bits[kSelectKeys / 32];        // pages that are taken, and how many before each word
    int before[kSelectKeys / 32];
    int part[2][kSelectWarps];
    uint32_t least[kSelectWarps], most[kSelectWarps];
    int bin[kSelectWarps], above[kSelectWarps], inside[kSelectWarps], listed[kSelectWarps];
    uint32_t cut_key[kSelectWarps];
    int cut_page[kSelectWarps];
};

// Of the keys of pages [lo, hi), more than `want` > 0, the `want` largest, equal ones from the lowest page on, listed in order.
// WARPS warps together: all of the block, or each warp by itself.  The range of the keys is cut into bins; the bin in which the
// want-th largest lies holds a few keys, which are ranked one by one.  Where it holds many (equal scores), the want-th
// largest key, and the page up to which equal ones are taken, are found by halving their ranges instead.
template <int WARPS>
__device__ __forceinline__ void choose_pages(SelectShared& s, const uint32_t* global, int lo, int hi, int want, int32_t* out, int tid) {
    constexpr int THREADS = 32 * WARPS, SHARE = kSelectWarps / WARPS;   // of the arrays
    constexpr int BINS = kSelectBins / SHARE, LIST = kSelectList / SHARE, KEYS = kSelectKeys / SHARE, EACH = BINS / THREADS;
    const int lane = tid & 31, warp = tid >> 5, w0 = WARPS > 1 ? 0 : threadIdx.x >> 5;   // w0: the warp's own part
    int* bins = s.bins + w0 * BINS;
    uint32_t* list = s.list + w0 * LIST;
    int* listed_page = s.page + w0 * LIST;
    auto sync = [] {
        if constexpr (WARPS > 1) __syncthreads();
        else __syncwarp();
    };
    const bool kept = hi - lo <= KEYS;
    const uint32_t* keys = kept ? s.keys + w0 * KEYS - lo : global;
    uint32_t least = 0xffffffffu, most = 0;
#pragma unroll 4
    for (int j = lo + tid; j < hi; j += THREADS) {
        const uint32_t x = global[j];
        if (kept) s.keys[w0 * KEYS + j - lo] = x;
        least = min(least, x);
        most = max(most, x);
    }
#pragma unroll
    for (int i = 0; i < EACH; i += 4) *reinterpret_cast<int4*>(bins + EACH * tid + i) = make_int4(0, 0, 0, 0);
    if (tid == 0) s.listed[w0] = 0;
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (WARPS > 1)
        if (lane == 0) { s.least[warp] = least; s.most[warp] = most; }
    sync();
    if constexpr (WARPS > 1) {
        least = __reduce_min_sync(0xffffffffu, s.least[lane % WARPS]);
        most = __reduce_max_sync(0xffffffffu, s.most[lane % WARPS]);
    }
    const int shift = max(0, 32 - __clz(most - least) - (31 - __clz(BINS)));
#pragma unroll 1
    for (int j = lo + tid; j < hi; j += THREADS) atomicAdd(bins + ((keys[j] - least) >> shift), 1);
    sync();
    // the bin from which on there are `want`: sums from the last bin down
    int sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; i += 4) {
        const int4 u = *reinterpret_cast<const int4*>(bins + EACH * tid + i);
        sum += u.x + u.y + u.z + u.w;
    }
    int from = sum;                                                   // keys in this thread's bins and those above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_down_sync(0xffffffffu, from, o);
        if (lane + o < 32) from += x;
    }
    if constexpr (WARPS > 1) {
        if (lane == 0) s.part[0][warp] = from;
        sync();
        from += __reduce_add_sync(0xffffffffu, lane > warp && lane < WARPS ? s.part[0][lane] : 0);
    }
    if (from >= want && from - sum < want) {                          // one thread
        int above = from - sum, i = EACH * tid + EACH - 1;
        while (above + bins[i] < want) above += bins[i--];
        s.bin[w0] = i;
        s.above[w0] = above;
        s.inside[w0] = bins[i];
    }
    sync();
    const int bin = s.bin[w0], need = want - s.above[w0], inside = s.inside[w0];
    uint32_t cut_key = least + ((uint32_t)bin << shift);              // taken: larger keys, and equal ones up to cut_page
    int cut_page = 0x7fffffff;
    if (inside > need && inside <= LIST) {
#pragma unroll 1
        for (int j = lo + tid; j < hi; j += THREADS) {
            const uint32_t x = keys[j];
            if ((int)((x - least) >> shift) != bin) continue;
            const int to = atomicAdd(&s.listed[w0], 1);
            list[to] = x;
            listed_page[to] = j;
        }
        sync();
#pragma unroll 1
        for (int i = tid; i < inside; i += THREADS) {
            const uint32_t x = list[i];
            const int j = listed_page[i];
            int rank = 0;
#pragma unroll 1
            for (int o = 0; o < inside; ++o) rank += list[o] > x || (list[o] == x && listed_page[o] < j);
            if (rank == need - 1) { s.cut_key[w0] = x; s.cut_page[w0] = j; }
        }
        sync();
        cut_key = s.cut_key[w0];
        cut_page = s.cut_page[w0];
    } else if (inside > need) {
        int round = 0;
        auto taken_with = [&](uint32_t x, int page) {                 // keys above x, and equal ones up to the page
            int n = 0;
#pragma unroll 1
            for (int j = lo + tid; j < hi; j += THREADS) n += keys[j] > x || (keys[j] == x && j <= page);
            n = __reduce_add_sync(0xffffffffu, n);
            if constexpr (WARPS > 1) {
                if (lane == 0) s.part[round & 1][warp] = n;
                sync();
                n = __reduce_add_sync(0xffffffffu, lane < WARPS ? s.part[round & 1][lane] : 0);
                ++round;
            }
            return n;
        };
        sync();
        uint32_t below = cut_key, over = most - cut_key >> shift ? cut_key + ((1u << shift) - 1) : most;   // the want-th largest is in [below, over]
#pragma unroll 1
        while (below < over) {
            const uint32_t x = below + (over - below + 1) / 2;
            if (taken_with(x, 0x7fffffff) >= want) below = x; else over = x - 1;
        }
        cut_key = below;
        int first = lo, last = hi - 1;                                // the least page up to which, with the larger keys, there are `want`
#pragma unroll 1
        while (first < last) {
            const int x = first + (last - first) / 2;
            if (taken_with(cut_key, x) >= want) last = x; else first = x + 1;
        }
        cut_page = first;
    }
    // listed in order, KEYS pages at a time
    uint32_t* bits = s.bits + w0 * (KEYS / 32);
    int* before = s.before + w0 * (KEYS / 32);
#pragma unroll 1
    for (int base = lo; base < hi; base += KEYS) {
        const int n = min(KEYS, hi - base);
        auto takes = [&](int i) {
            const uint32_t x = i < n ? keys[base + i] : 0;
            return x > cut_key || (x == cut_key && i < n && base + i <= cut_page);
        };
#pragma unroll 1
        for (int i = tid; i < (n + 31 & ~31); i += THREADS) {
            const unsigned these = __ballot_sync(0xffffffffu, takes(i));
            if (lane == 0) bits[i / 32] = these;
        }
        sync();
        int at = 0;                                                   // taken in the words before this thread's (every warp adds up all)
#pragma unroll 1
        for (int w = 0; w < (n + 31) / 32; w += 32) {
            const int mine = w + lane < (n + 31) / 32 ? __popc(bits[w + lane]) : 0;
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (warp == 0 && w + lane < (n + 31) / 32) before[w + lane] = at + incl - mine;
            at += __shfl_sync(0xffffffffu, incl, 31);
        }
        sync();
#pragma unroll 1
        for (int i = tid; i < n; i += THREADS) {
            const uint32_t word = bits[i / 32];
            if (word >> (i & 31) & 1) out[before[i / 32] + __popc(word & ((1u << (i & 31)) - 1))] = base + i;
        }
        out += at;
        sync();                                                       // (the memory is used again)
    }
}

// A block scores a share of a (sequence, key head)'s pages for up to 32 columns of queries.  The blocks that share them are a cluster:
// once all of its scores are there, each chooses for some of the queries.
template <class T, int SEGS>
__global__ void __launch_bounds__(kSelectThreads, SEGS == 8 ? 1 : 2) page_select_kernel(const __grid_constant__ skv_pool_select_args a, const __grid_constant__ SelectShape shape) {
    extern __shared__ __align__(16) __half s_raw[];               // SEGS: [columns][64 SEGS + 8], the bytes 0, 2, 1, 3 of each word; else [2 D] bytes
    __shared__ float s_t[8 * kScoreTiles], s_start[8 * kScoreTiles];
    SelectShared& s_choice = *reinterpret_cast<SelectShared*>(s_raw);   // (the queries are not needed any more then)
    start_dependents();
    wait_for_dependency();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.z, h = blockIdx.y;
    int rank = 0, group = blockIdx.x;                             // of the cluster, of the new tokens
    if (shape.blocks > 1) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(group));
    }
    const int i0 = group * shape.block_tokens, i1 = min(a.S_q, i0 + shape.block_tokens);
    const int tokens = select_tokens(a, b), pages = shape.pages_of(tokens), want = a.keep - a.first - a.recent, pitch = a.table_width;
    const int64_t unit0 = ((int64_t)b * a.heads + h) * a.S_q;
    uint32_t* keys = static_cast<uint32_t*>(a.scratch) + unit0 * pitch;
    if (pages > a.keep && want > 0) {
        if (a.num_pages == 0) {                                   // no table can name a page
            for (int i = i0; i < i1; ++i)
                for (int j = rank * kSelectThreads + tid; j < pages; j += shape.blocks * kSelectThreads) keys[(int64_t)i * pitch + j] = 1;
            if (a.error_flag) atomicExch(a.error_flag, 1);
        } else if constexpr (SEGS > 0) score_pages<T, SEGS>(a, shape, rank, b, h, pages, i0, s_raw, s_t, s_start, keys, pitch);
        else score_pages_any<T>(a, shape, rank, b, h, pages, i0, reinterpret_cast<int8_t*>(s_raw), s_t, keys, pitch);
        if (shape.blocks > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            __syncthreads();
        }
    }
    if (tid == 0 && a.error_flag && a.lengths[b] != tokens) atomicExch(a.error_flag, 1);
    const bool by_warp = i1 - i0 > 2 * shape.blocks && pages <= kSelectKeys / kSelectWarps;
    const int one_of = by_warp ? shape.blocks * kSelectWarps : shape.blocks, first_of = by_warp ? rank * kSelectWarps + warp : rank;
    for (int i = i0 + first_of; i < i1; i += one_of) {
        const int n = select_pages(a, shape, b, i, tokens), step = by_warp ? 32 : kSelectThreads, me = by_warp ? lane : tid;
        int32_t* out = a.pages + (unit0 + i) * a.keep;
        if (n <= a.keep) {
            for (int k = me; k < a.keep; k += step) out[k] = k < n ? k : -1;
            continue;
        }
        for (int k = me; k < a.first + a.recent; k += step) out[k < a.first ? k : want + k] = k < a.first ? k : n - a.recent - a.first + k;
        if (want == 0) continue;
        if (by_warp) choose_pages<1>(s_choice, keys + (int64_t)i * pitch, a.first, n - a.recent, want, out + a.first, lane);
        else choose_pages<kSelectWarps>(s_choice, keys + (int64_t)i * pitch, a.first, n - a.recent, want, out + a.first, tid);
    }
}

template <class T, int SEGS>
int launch_select_kernel(const skv_pool_select_args& a, SelectShape shape, size_t smem, cudaStream_t st) {
    shape.shift = 31;
    while ((1ll << (shape.shift - 31)) < a.page_size) ++shape.shift;
    shape.mul = (uint32_t)(((1ull << shape.shift) + a.page_size - 1) / a.page_size);
    // as many blocks as fill the GPU, no more than there are shares and a cluster has (heads above 128 values: one block an SM, by its registers; 32
    // sequences of 256 pages with 8 such heads 32.2 us with shares for two, 20.9 with one, other batches the same)
    const int share = SEGS > 0 ? 16 * kSelectWarps : 8 * kSelectWarps, groups = (a.S_q + shape.block_tokens - 1) / shape.block_tokens;
    const int64_t all = (int64_t)a.batch * a.heads * groups, fill = ((SEGS == 8 ? 1ll : 2ll) * sm_count() + all - 1) / all;
    if (smem < sizeof(SelectShared)) smem = sizeof(SelectShared);
    int x = (a.table_width + share - 1) / share;
    if (x > fill) x = (int)fill;
    if (x > kSelectCluster) x = kSelectCluster;
    if (x < 1) x = 1;
    shape.blocks = x;
    launch_cluster_after(page_select_kernel<T, SEGS>, dim3((unsigned)groups * x, a.heads, a.batch), dim3(x), kSelectThreads, smem, st, a, shape);
    return check_launch("pool_select");
}

template <class T>
int launch_select(const skv_pool_select_args& a, cudaStream_t st) {
    const int D = a.head_dim;
    SelectShape shape = {};
    shape.rep = a.q.heads / a.heads;
    shape.block_tokens = 1;
    if (D % 8 || D > 256 || (reinterpret_cast<uintptr_t>(a.bounds) & 15)) return launch_select_kernel<T, 0>(a, shape, 2 * (size_t)D, st);
    while (1 << shape.log_span < shape.rep && shape.log_span < 3) ++shape.log_span;
    if (shape.rep <= 8) shape.block_tokens = 8 * kScoreTiles >> shape.log_span;
    const auto smem = [](int segs) { return (size_t)8 * kScoreTiles * (64 * segs + 8) * sizeof(__half); };
    if (D <= 64) return launch_select_kernel<T, 2>(a, shape, smem(2), st);
    if (D <= 128) return launch_select_kernel<T, 4>(a, shape, smem(4), st);
    return launch_select_kernel<T, 8>(a, shape, smem(8), st);
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
    if (reinterpret_cast<uintptr_t>(a.scratch) & 15) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_select: scratch is not on a 16-byte boundary");
    if (a.head_dim > 1024) return fail(SKV_ERR_UNSUPPORTED, "pool_select: head_dim %d above 1024", a.head_dim);
    if (a.table_width > 1 << 30) return fail(SKV_ERR_TOO_LARGE, "pool_select: tables of %d pages", a.table_width);
    if (a.batch > 65535 || a.heads > 65535 || a.S_q > 0x7fffffff / kSelectCluster || (int64_t)a.batch * a.heads * a.S_q > 0x7fffffff)
        return fail(SKV_ERR_TOO_LARGE, "pool_select: %d sequences of %d heads and %d queries", a.batch, a.heads, a.S_q);
    if (a.scratch_bytes < (int64_t)skv_pool_select_scratch_bytes(a.batch, a.heads, a.S_q, a.table_width))
        return fail(SKV_ERR_SCRATCH, "pool_select: scratch of %lld bytes", (long long)a.scratch_bytes);
    cudaStream_t st = as_stream(stream);
    if (a.q.dtype == kF32) return launch_select<float>(a, st);
    if (a.q.dtype == kF16) return launch_select<__half>(a, st);
    return launch_select<__nv_bfloat16>(a, st);
}

}  // extern "C"
