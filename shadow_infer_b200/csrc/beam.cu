// Beam search over the page pool: the best continuations of a search's beams, and the block tables and pages that
// follow them.
//
// Selection.  A continuation's score is  s_r + x_rv - m_r - ln sum_v e^(x_rv - m_r),  m_r the row's largest logit.  Within a row
// scores are ordered as logits are, so the logits are read once (and a few pieces of them again).  A warp takes a part of a row, as
// many parts as there are warps on the GPU at a time, and leaves the part's maximum, its sum and its `keep` best logits.  A second
// launch, a block a search, joins the sums, turns the lists' logits into scores in 64 bits and merges the lists; it is set
// up while the first still runs.
//
// Few searches, or small ones, are one launch of clusters, whose first block merges what the others found.
//
// What bounds it.  256 rows of 131072 16-bit logits (205 of them not finished, 54 MB): 26.4 us, of which the lists take about 20 (2.7 TB/s:
// a warp has one block of 4 KB ahead of the one at work, and 16 warps fit an SM's registers, of which about 11 are at work: a warp's part is of one
// beam, finished or not, and 256 blocks are two on some SMs; 24 without the block ahead were no faster, nor
// were more parts than warps) and the merge 6, one step's latency after the other (in two launches 27.4).  4 rows of 32000 fp32 logits: 8.5 us,
// the same steps; from Python such a call costs 14.
//
// Reordering moves what a step has to copy, about a third of the beams' last pages: 256 beams with 63 int8 tokens of 10 heads of 128 values
// in theirs, 28 MB read and written in 11.3 us (2.6 TB/s; blocks that copy 16 KB each wait for parents, lengths, tables and rows in turn);
// a step of 8 searches of 4 beams takes 3.8 us.
#include <float.h>

#include <mutex>
#include <type_traits>

#include "pool.cuh"

namespace skv {

constexpr int kBeamKeep = 128, kBeamMost = 4096;      // most continuations; most beams of a search
constexpr int kMergeEntries = 8192, kMergeFew = 2048;  // entries of lists that a merge holds, and is given if it can
constexpr int kBeamWarps = 4, kBeamHeld = 256;        // warps of a block, candidates that a warp holds
constexpr int kManyLoads = 8, kFewLoads = 4;          // 16-byte loads a lane, of a block
constexpr int kBeamBatch = 16;                        // blocks between two looks for candidates
constexpr int kBeamPieces = 128;                      // (lane, block) pieces that are looked through then

// What a warp leaves for the merge; its list follows the headers.
struct BeamPart {
    double sum;     // of e^(x - top), or how many are +inf where top is
    float top;
    int count;      // entries of the list: logits above -inf, best first
};

// Blocks of a row that are taken at once, and warps that share a row.
struct BeamShape {
    int loads, parts;
    int64_t block, blocks;
};
inline BeamShape beam_shape(int B, int beams, int V, int keep, int bytes, bool aligned) {
    BeamShape s;
    const int64_t rows = (int64_t)B * beams;
    auto cut = [&](int loads) {
        s.loads = loads;
        s.block = 32ll * loads * (16 / bytes);
        s.blocks = (V + (aligned ? 0 : 16 / bytes) + s.block - 1) / s.block;   // (else the first piece is empty: see realign)
    };
    cut(kManyLoads);
    if (rows * s.blocks < sm_count() * 8) cut(kFewLoads);          // too few warps to fill the GPU: more and smaller blocks
    // 16 warps an SM at a time; but a merge's time grows with its entries: 2048, or 4096 where that leaves few warps (a search of 8 beams of
    // 131072 fp32 logits, 16 kept: 8192 entries 21.2 us, 4096 15.7, 2048 15.6, 1024 19.3; of 32 beams of 32000, 32 kept: 27, 26, 34, 51)
    int64_t most = kMergeFew / keep / beams, resident = sm_count() * 16 / rows;
    if (rows * most < 128) most = 2 * kMergeFew / keep / beams;
    if (most > resident) most = resident;
    if (most < 1) most = 1;
    s.parts = (int)(s.blocks < most ? s.blocks : most);
    return s;
}

// The same for searches that a cluster of blocks takes in one launch; parts 0 where it does not: the clusters would not be resident together, or would
// leave SMs idle while a warp has more than 8 blocks, or the merge would hold more than its share.  (One launch against two, device time: a
// search of 4 beams of 32000 fp32 logits 8.1 against 8.9 us, 8 searches 9.4 and 11.4, 32 searches 10.4 and 11.5, 64 searches 20.9 and 15.7;
// 16 blocks a warp: one search 13.9 and 11.0.  8 beams of 131072 bf16 logits: 16 searches 24.3 and 22.0, 20 25.5 and 24.9, 22 26.2 and 25.3, 24 25.9 and 25.5, 26 26.7 and 27.3,
// 28 25.7 and 26.9, 32 27.0 and 28.2, 37 37.6 and 27.9; of 65536 fp32 logits 16 19.3 and 20.0, 24 21.9 and 22.8, 32 24.4 and 25.2; 4 beams of 131072 fp32
// logits 16 15.0 and 13.3, 20 15.7 and 15.2, 24 16.3 and 16.8, 32 18.1 and 19.2.  From Python a call costs 3 us less.)
constexpr int kCluster = 8, kClusterWarps = 8;        // blocks of a search, warps of a block
inline BeamShape small_shape(int B, int beams, int V, int keep, int bytes, bool aligned) {
    BeamShape s;
    const int most = kCluster * kClusterWarps / beams;
    auto cut = [&](int loads) {
        s.loads = loads;
        s.block = 32ll * loads * (16 / bytes);
        s.blocks = (V + (aligned ? 0 : 16 / bytes) + s.block - 1) / s.block;
        s.parts = (int)(s.blocks < most ? s.blocks : most);
    };
    cut(kFewLoads);
    const bool short_rows = s.blocks <= 8 * s.parts, fill = 4ll * B * kCluster >= 5 * sm_count();
    const bool resident = 4ll * B * kCluster <= 7 * sm_count();   // (not all SMs of a GPC make up clusters)
    if (!short_rows && s.parts > 0) cut(kManyLoads);
    if (!(short_rows || fill) || !resident || (int64_t)s.parts * beams * keep > kMergeFew) s.parts = 0;
    return s;
}

// Whether beam r of search b has continuations of its own, and whether it has but one.  (The kernels of the selection wait for those before them by
// themselves: no read-only loads in them, which could be moved before that.)
__device__ __forceinline__ bool beam_dead(const skv_beam_args& a, int64_t row) { return !(fabsf(a.scores[row]) < INFINITY); }
__device__ __forceinline__ bool beam_done(const skv_beam_args& a, int64_t row) { return a.finished && a.finished[row]; }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// 32 bits of logits: one or two.
template <class T> struct Word {
    static constexpr int N = 2;
    using Pair = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    static __device__ __forceinline__ Pair pair(uint32_t w) { return *reinterpret_cast<const Pair*>(&w); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {   // of a number and a NaN: the number
        const Pair m = __hmax2(pair(a), pair(b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    static __device__ __forceinline__ uint32_t larger_nan(uint32_t a, uint32_t b) {   // the NaN
        const Pair m = __hmax2_nan(pair(a), pair(b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    static __device__ __forceinline__ uint32_t bits(__half x) { return __half_as_ushort(x); }
    static __device__ __forceinline__ uint32_t bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
    static __device__ __forceinline__ uint32_t from(T x, T y) { return bits(x) | bits(y) << 16; }
    static __device__ __forceinline__ uint32_t both(float x) { return from(from_float<T>(x), from_float<T>(x)); }
    static __device__ __forceinline__ float at(uint32_t w, int i) {
        if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffff)));
        else return __uint_as_float(i ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ float largest(uint32_t w) { return max_nan(at(w, 0), at(w, 1)); }
    static constexpr float kLowest = std::is_same_v<T, __half> ? -65504.0f : -3.3895313892515355e38f;
};
template <> struct Word<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ uint32_t larger_nan(uint32_t a, uint32_t b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ uint32_t both(float x) { return __float_as_uint(x); }
    static __device__ __forceinline__ float at(uint32_t w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ float largest(uint32_t w) { return __uint_as_float(w); }
    static constexpr float kLowest = -FLT_MAX;
};

__device__ __forceinline__ uint64_t pack2(float x, float y) { return (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float low_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }

// The number that score_bits gives an image of.
__device__ __forceinline__ float of_score_bits(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// Whether (x, i) comes before (y, j).
__device__ __forceinline__ bool ahead(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

// The value of rank `rank` (0: the largest) among the lanes' values, none a NaN: sorted by compare and exchange.
template <class V>
__device__ __forceinline__ V warp_ranked(V x, int rank) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const V y = __shfl_xor_sync(0xffffffffu, x, o);
            x = ((lane & o) == 0) == ((lane & size) == 0) ? max(x, y) : min(x, y);
        }
    return __shfl_sync(0xffffffffu, x, rank);
}

// Logits [first, first + count) of a row have more candidates, from `from` to `most`, than were collected (many are equal, or many are
// to be kept): halves the range of their images until a list with `held` entries has room for what is left, at the end with the
// place up to which equal ones are taken.  Returns the entries of the list then.  A warp calls this, seldom: the logits are read again.
template <class T>
__device__ __noinline__ int beam_many(const T* x0, int first, int count, int V, float from, float most, int keep, int held, float2* list,
                                      int* s_count) {
    const int lane = threadIdx.x & 31, begin = max(first, 0), end = min((int64_t)V, (int64_t)first + count), room = kBeamHeld - held;
    auto logit = [&](int i) { return fmaxf(to_float(x0[i]), -INFINITY); };
    auto count_from = [&](uint32_t image) {
        int m = 0;
        for (int i = begin + lane; i < end; i += 32) m += score_bits(logit(i)) >= image;
        return __reduce_add_sync(0xffffffffu, m);
    };
    uint32_t lo = score_bits(from), hi = score_bits(most);   // if more than `room` are from lo on, the keep-th largest is in [lo, hi]
    int from_lo = count_from(lo);
    while (lo < hi && from_lo > room) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        const int m = count_from(mid);
        if (m >= keep) { lo = mid; from_lo = m; } else hi = mid - 1;
    }
    const float cut = of_score_bits(lo);
    int last = end - 1;                                       // equal ones up to here are taken
    if (from_lo > room) {                                     // (then fewer than `keep` are larger)
        int lower = begin - 1;                                // there is room for those up to here
        last = end - 1;
        while (lower < last) {
            const int mid = lower + (last - lower + 1) / 2;
            int m = 0;
            for (int i = begin + lane; i < end; i += 32) { const float x = logit(i); m += x > cut || (x == cut && i <= mid); }
            m = __reduce_add_sync(0xffffffffu, m);
            if (m <= room) lower = mid; else last = mid - 1;
        }
    }
    if (lane == 0) *s_count = held;
    __syncwarp();
    for (int i = begin + lane; i < end; i += 32) {
        const float x = logit(i);
        if (x > cut || (x == cut && i <= last)) list[atomicAdd(s_count, 1)] = make_float2(x, __int_as_float(i));
    }
    __syncwarp();
    return *s_count;
}

// Rows that do not all begin on 16 bytes are read in pieces on such boundaries all the same, and then moved: a row's pieces are its logits
// 0 to 7, 8 to 15 (or 0 to 3, 4 to 7) and so on wherever it begins, so that equal rows add up to equal sums, bit by bit, and
// their continuations tie.  A piece as it was read, which begins Q words and `bits` bits before the row's own, gives way to what it
// completes: the row's piece that begins in the one before it, which is the lane's below or, for lane 0, lane 31's of the load
// before (`carry`: of the block before).  (8 searches of 4 beams of 50257 bf16 logits take 12.8 us, with sums by the places of pieces in memory
// 11.5; 32 searches of 8 beams of 131071 36.5 and 33.2; rows on 16 bytes do without.)
template <class T, int LOADS, int Q>
__device__ __forceinline__ void realign(uint32_t (&w)[4 * LOADS], const uint32_t (&carry)[4], int bits) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int l = LOADS - 1; l >= 0; --l) {
        uint32_t z[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= Q) z[k] = __shfl_sync(0xffffffffu, lane < 31 ? w[4 * l + k] : l > 0 ? w[4 * (l > 0 ? l - 1 : 0) + k] : carry[k], (lane + 31) & 31);
            z[4 + k] = w[4 * l + k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * l + k] = sizeof(T) == 4 ? z[Q + k] : __funnelshift_r(z[Q + k], z[Q + k + 1], bits);
    }
}

// A row's part in batches of up to kBeamBatch blocks.  The first look at a batch adds up its exponentials and keeps the largest logit of
// every lane and block; the keep-th largest of the lanes' largest is a bound that few (lane, block) pieces reach, about `keep` and a
// half, and only these are read again (they are in L2 still) for their candidates.  (Candidates looked for block by block, as they
// come, took as many instructions again as all else: 34 us for 33.5 M 16-bit logits, 20 without them.)
struct ListShared {                                       // of a warp
    float2 list[kBeamHeld], ranked[kBeamKeep];
    float best[kBeamBatch][32];
    int piece[kBeamPieces], held;
};
template <class T, int LOADS, bool ALIGNED>
__device__ __forceinline__ void beam_list(const skv_beam_args& a, int parts, int64_t blocks, int64_t job, ListShared& s) {
    using W = Word<T>;
    constexpr int PER = 16 / (int)sizeof(T), WORDS = 4 * LOADS, BLOCK = 32 * LOADS * PER;
    const int lane = threadIdx.x & 31, keep = a.keep;
    const int64_t row = job / parts;
    if (row >= (int64_t)a.B * a.beams) return;
    const int part = (int)(job - row * parts);
    if (beam_dead(a, row) || beam_done(a, row)) return;   // the merge does not look at their lists
    const T* x0 = static_cast<const T*>(a.logits) + row / a.beams * a.stride_b + row % a.beams * a.stride_r;
    // piece i holds logits i * PER - LEAD and on, as it is read (on 16 bytes) i * PER - shift and on
    constexpr int LEAD = ALIGNED ? 0 : PER;
    const int shift = ALIGNED ? 0 : (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    float2* list = s.list;
    const int b0 = (int)(blocks * part / parts), b1 = (int)(blocks * (part + 1) / parts);
    float top = -INFINITY;                                // of the lane
    double sum = 0.0;
    int held = 0;
    float low = -INFINITY;                                // the keep-th best so far
    // The list's n entries ranked (each counts those ahead of it), the best `keep` of them in order at its front.
    auto rank = [&](int n) {
        for (int i = lane; i < n; i += 32) {
            const float2 e = list[i];
            int before = 0;
            for (int j = 0; j < n; ++j) {
                const float2 f = list[j];
                before += ahead(f.x, __float_as_int(f.y), e.x, __float_as_int(e.y));
            }
            if (before < keep) s.ranked[before] = e;
        }
        __syncwarp();
        held = min(n, keep);
        for (int i = lane; i < held; i += 32) list[i] = s.ranked[i];
        __syncwarp();
        if (held == keep) low = list[keep - 1].x;
    };
    auto word = [&](int i) {                              // logit i, and the next one, one by one
        const T none = from_float<T>(-INFINITY), x = i >= 0 && i < a.V ? x0[i] : none;
        if constexpr (W::N == 2) return W::from(x, i + 1 >= 0 && i + 1 < a.V ? x0[i + 1] : none);
        else return __float_as_uint(x);
    };
    uint32_t next[WORDS];                                 // the block after the one at work, on its way
    auto load = [&](int block) {
        const int first0 = (block * 32 * LOADS + lane) * PER - shift;
        if (block * BLOCK >= shift && (block + 1) * BLOCK - shift <= a.V) {
            const uint4* y = reinterpret_cast<const uint4*>(x0 + first0);
#pragma unroll
            for (int l = 0; l < LOADS; ++l) {
                const uint4 u = y[32 * l];
                next[4 * l] = u.x; next[4 * l + 1] = u.y; next[4 * l + 2] = u.z; next[4 * l + 3] = u.w;
            }
            return;
        }
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
#pragma unroll
            for (int k = 0; k < 4; ++k) next[4 * l + k] = word(first0 + 32 * PER * l + k * W::N);
    };
    uint32_t carry[4];
    if constexpr (!ALIGNED) {
#pragma unroll
        for (int k = 0; k < 4; ++k) carry[k] = word((b0 * 32 * LOADS - 1) * PER - shift + k * W::N);
    }
    load(b0);
    for (int batch = b0; batch < b1; batch += kBeamBatch) {
        const int count = min(kBeamBatch, b1 - batch);
        for (int i = 0; i < count; ++i) {
            const int block = batch + i;
            uint32_t w[WORDS];
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = next[k];
            if (block + 1 < b1) load(block + 1);
            if constexpr (!ALIGNED) {
                const uint32_t last[4] = {w[WORDS - 4], w[WORDS - 3], w[WORDS - 2], w[WORDS - 1]};
                const int bytes = shift * (int)sizeof(T), bits = 8 * (bytes & 3);
                switch (bytes >> 2) {
                    case 0: realign<T, LOADS, 0>(w, carry, bits); break;
                    case 1: realign<T, LOADS, 1>(w, carry, bits); break;
                    case 2: realign<T, LOADS, 2>(w, carry, bits); break;
                    default: realign<T, LOADS, 3>(w, carry, bits);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) carry[k] = last[k];
            }
            auto find_best = [&]() {
                uint32_t best[4];
#pragma unroll
                for (int k = 0; k < WORDS; ++k) best[k % 4] = k < 4 ? w[k] : W::larger_nan(best[k % 4], w[k]);
                return W::largest(W::larger_nan(W::larger_nan(best[0], best[1]), W::larger_nan(best[2], best[3])));
            };
            float best = find_best();
            if (__any_sync(0xffffffffu, best != best)) {  // a NaN becomes -inf
                const uint32_t none = W::both(-INFINITY);
#pragma unroll
                for (int k = 0; k < WORDS; ++k) w[k] = W::larger(w[k], none);
                best = find_best();
            }
            s.best[i][lane] = best;
            // ---- the lane's sum, relative to its own largest logit so far
            if (best == -INFINITY) continue;
            float more;
            if (best == INFINITY) {
                more = 0.0f;                              // (seldom)
#pragma unroll
                for (int k = 0; k < WORDS; ++k)
#pragma unroll
                    for (int j = 0; j < W::N; ++j) more += W::at(w[k], j) == INFINITY ? 1.0f : 0.0f;
            } else {
                const uint64_t less = pack2(-best, -best), by = pack2(kLog2e, kLog2e);
                uint64_t total[2] = {0, 0};
#pragma unroll
                for (int k = 0; k < WORDS; k += W::N == 2 ? 1 : 2) {
                    const float x = W::at(w[k], 0), y = W::N == 2 ? W::at(w[k], 1) : W::at(w[k + 1], 0);
                    const uint64_t d = mul2(add2(pack2(x, y), less), by);
                    total[k / 2 % 2] = add2(total[k / 2 % 2], pack2(exp2_fast(low_of(d)), exp2_fast(high_of(d))));
                }
                total[0] = add2(total[0], total[1]);
                more = low_of(total[0]) + high_of(total[0]);
            }
            if (best > top) {
                sum = sum * exp2_fast((top - best) * kLog2e) + more;     // (of -inf: 0)
                top = best;
            } else if (top < INFINITY || best == INFINITY) {
                sum += best == top ? more : more * exp2_fast((best - top) * kLog2e);
            }
        }
        // ---- candidates: larger than the keep-th best so far (equal ones come behind it), not below the bound
        float mine[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // the lane's largest of every fourth block
#pragma unroll
        for (int i = 0; i < kBeamBatch; ++i)
            if (i < count) mine[i & 3] = fmaxf(mine[i & 3], s.best[i][lane]);
        const uint32_t largest = score_bits(fmaxf(fmaxf(mine[0], mine[1]), fmaxf(mine[2], mine[3])));
        const float most = of_score_bits(__reduce_max_sync(0xffffffffu, largest));
        if (most <= low || most == -INFINITY) continue;
        float from = W::kLowest;
        if (low > -INFINITY) {                            // the next number of the type
            uint32_t u = W::both(low == 0.0f ? 0.0f : low);
            if constexpr (W::N == 2) u &= 0xffffu;
            u = u & (W::N == 2 ? 0x8000u : 0x80000000u) ? u - 1 : u + 1;
            from = W::at(u, 0);
        }
        // Where `keep` is near 32 the least of the lanes' largest would let many through: the keep-th largest of up to 128, which a range of
        // images that holds it is halved to, until not many more are above its lower end.
        if (keep <= 16) {
            from = fmaxf(from, of_score_bits(warp_ranked(largest, keep - 1)));
        } else if (keep <= 32 || 32 * min(count, 4) >= keep) {
            uint32_t lo = score_bits(from), hi = score_bits(most);
            if (keep <= 32) lo = max(lo, __reduce_min_sync(0xffffffffu, largest));
            int above = 2 * kBeamKeep;
            while (lo < hi && above > keep + 4) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                int m = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) m += score_bits(mine[j]) >= mid;
                m = __reduce_add_sync(0xffffffffu, m);
                if (m >= keep) { lo = mid; above = m; } else hi = mid - 1;
            }
            from = fmaxf(from, of_score_bits(lo));
        } else if (count * 32 >= keep) {                  // of all that was kept
            uint32_t lo = score_bits(from), hi = score_bits(most);
            int above = 2 * kBeamKeep;
            while (lo < hi && above > keep + 4) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                int m = 0;
                for (int i = 0; i < count; ++i) m += score_bits(s.best[i][lane]) >= mid;
                m = __reduce_add_sync(0xffffffffu, m);
                if (m >= keep) { lo = mid; above = m; } else hi = mid - 1;
            }
            from = fmaxf(from, of_score_bits(lo));
        }
        int n = held, pieces = 0;
        for (int i = 0; i < count; ++i) {
            const unsigned these = __ballot_sync(0xffffffffu, s.best[i][lane] >= from);
            const int to = pieces + __popc(these & ((1u << lane) - 1));
            if (these >> lane & 1 && to < kBeamPieces) s.piece[to] = ((batch + i) * 32 * LOADS + lane) * PER - LEAD;
            pieces += __popc(these);
        }
        __syncwarp();
        const bool many = pieces > kBeamPieces;           // (many equal logits)
        // a load of one piece a lane, two at a time
        constexpr int AT_ONCE = 32 / LOADS;
        for (int i = lane / LOADS; i - lane / LOADS < pieces && !many; i += 2 * AT_ONCE) {
            uint32_t y[2][4];
            int first[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool is = i + h * AT_ONCE < pieces;
                first[h] = (is ? s.piece[i + h * AT_ONCE] : 0) + lane % LOADS * 32 * PER;
                if (ALIGNED && is && first[h] >= 0 && first[h] + PER <= a.V) {
                    const uint4 u = *reinterpret_cast<const uint4*>(x0 + first[h]);
                    y[h][0] = u.x; y[h][1] = u.y; y[h][2] = u.z; y[h][3] = u.w;
                } else if (!ALIGNED && is && first[h] > 0 && first[h] + PER + 2 <= a.V) {   // (the words may hold a neighbour)
                    const uintptr_t at = reinterpret_cast<uintptr_t>(x0 + first[h]);
                    const uint32_t* z = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
                    uint32_t u[5];
#pragma unroll
                    for (int k = 0; k < 3 + W::N; ++k) u[k] = z[k];
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[h][k] = W::N == 1 ? u[k] : __funnelshift_r(u[k], u[k + 1], 8 * (int)(at & 3));
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[h][k] = is ? word(first[h] + k * W::N) : W::both(-INFINITY);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const float x = W::at(y[h][k / W::N], k % W::N);
                    const unsigned is = __ballot_sync(0xffffffffu, x >= from);
                    const int to = n + __popc(is & ((1u << lane) - 1));
                    if (x >= from && to < kBeamHeld) list[to] = make_float2(x, __int_as_float(first[h] + k));
                    n += __popc(is);
                }
        }
        __syncwarp();
        if (many || n > kBeamHeld) n = beam_many(x0, batch * BLOCK - LEAD, count * BLOCK, a.V, from, most, keep, held, list, &s.held);
        rank(n);
    }
    const float most = warp_max(top);
    if (top < most) sum = most < INFINITY ? sum * exp2_fast((top - most) * kLog2e) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) static_cast<BeamPart*>(a.scratch)[job] = BeamPart{sum, most, held};
    float2* out = reinterpret_cast<float2*>(static_cast<BeamPart*>(a.scratch) + (int64_t)a.B * a.beams * parts) + job * keep;
    for (int i = lane; i < held; i += 32) out[i] = list[i];
}
template <class T, int LOADS, bool ALIGNED>
__global__ void __launch_bounds__(32 * kBeamWarps, LOADS == kManyLoads ? 4 : 6) beam_lists_kernel(const __grid_constant__ skv_beam_args a, int parts, int64_t blocks) {
    __shared__ ListShared s[kBeamWarps];
    start_dependents();
    const int warp = threadIdx.x >> 5;
    beam_list<T, LOADS, ALIGNED>(a, parts, blocks, (int64_t)blockIdx.x * kBeamWarps + warp, s[warp]);
}

// ------------------------------------------------------------------------------------------ the merge
constexpr int kMergeThreads = 256, kMergeHeld = 512;

// A continuation as it is compared: the order-preserving image of its score in 64 bits (0: none), then its beam; within a beam its logit, which
// tells apart what 64 bits do not (and orders the lists, whose ends are cut by it), then its token.
struct BeamBest {
    uint64_t score, place;   // place: beam * 2^32 + token
    float logit;
    __device__ __forceinline__ bool before(const BeamBest& o) const {
        if (score != o.score) return score > o.score;
        if ((place ^ o.place) >> 32 || logit == o.logit) return place < o.place;
        return logit > o.logit;
    }
};
__device__ __forceinline__ uint64_t score_image(double x) {
    if (x == 0.0) x = 0.0;   // (-0 ties with 0)
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double score_of_image(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u ^ 1ull << 63 : ~u)); }

// ln x for a normal x > 0: x = 2^e m with m in [sqrt(1/2), sqrt(2)), ln m = 2 atanh(s) with s = (m - 1) / (m + 1), |s| < 0.172, by its series
// up to s^17 (what is left out is below 2e-15).
__device__ __forceinline__ double logarithm(double x) {
    const int high = __double2hiint(x), e = ((high >> 20) - 1022) - ((high & 0xfffff) < 0x6a09e);
    const double m = x * __hiloint2double((1023 - e) << 20, 0), d = m + 1.0;
    double r = (double)(1.0f / (float)d);   // two steps of Newton's method: 24, 48, 53 bits
    r = r * (2.0 - d * r);
    r = r * (2.0 - d * r);
    const double s = (m - 1.0) * r, q = s * s;
    double sum = 1.0 / 17;
#pragma unroll
    for (int k = 15; k > 0; k -= 2) sum = fma(sum, q, 1.0 / k);
    return fma((double)e, 0.69314718055994531, 2.0 * s * sum);
}

// by_parts, by_keep: 1 / parts, 1 / keep (numbers below 2^20 are divided by a product: half of a unit is more than its error).
// A block a search.  It runs once, so its time is the latency of one step after another, instructions fetched included: loops are not
// unrolled where that gains no overlap.
struct MergeShared {
    BeamBest held[kMergeHeld], best[2][kMergeThreads / 32];
    uint32_t front[kMergeThreads / 32], top[kMergeThreads / 32];
    int part[2][kMergeThreads / 32], n, owner[2][kMergeThreads / 32];
};
template <class T>
__device__ __forceinline__ void beam_merge(const skv_beam_args& a, int parts, bool staged, float by_parts, float by_keep, int search,
                                           MergeShared& s, unsigned char* s_raw) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, keep = a.keep, beams = a.beams, lists = beams * parts, all = lists * keep;
    const int64_t row0 = (int64_t)search * beams;
    double* s_from = reinterpret_cast<double*>(s_raw);              // [beams] what a logit less the largest is added to
    float2* s_entry = reinterpret_cast<float2*>(s_from + beams);    // staged: [lists][keep]
    uint64_t* s_score = reinterpret_cast<uint64_t*>(s_entry + (staged ? all : 0));   // staged: [lists][keep] images
    float* s_most = reinterpret_cast<float*>(s_score + (staged ? all : 0));          // [beams] the largest logit
    int* s_count = reinterpret_cast<int*>(s_most + beams);          // [lists] entries; -1: a finished beam's one continuation
    int* s_at = s_count + lists;                                    // [lists] places of the fronts
    uint32_t* s_upper = reinterpret_cast<uint32_t*>(s_at + lists);  // staged: [lists][keep] the images' upper halves
    const BeamPart* part = static_cast<const BeamPart*>(a.scratch) + row0 * parts;
    const float2* entries = reinterpret_cast<const float2*>(static_cast<const BeamPart*>(a.scratch) + (int64_t)a.B * lists) +
                            row0 * parts * keep;
    if (tid == 0) s.n = 0;
    if (staged)
#pragma unroll 4
        for (int i = tid; i < all; i += kMergeThreads) s_entry[i] = entries[i];
#pragma unroll 1
    for (int r = warp; r < beams; r += kMergeThreads / 32) {        // a warp a beam
        const float cum = a.scores[row0 + r];
        const bool done = beam_done(a, row0 + r), dead = !(fabsf(cum) < INFINITY);
        float most = -INFINITY;
        double sum = 0.0;
#pragma unroll 1
        for (int p0 = 0; p0 < parts; p0 += 32) {
            BeamPart y{0.0, -INFINITY, 0};
            if (p0 + lane < parts && !done && !dead) y = part[r * parts + p0 + lane];
            if (p0 + lane < parts) s_count[r * parts + p0 + lane] = y.count;
            const float now = fmaxf(most, warp_max(y.top));
            double x = y.top == -INFINITY ? 0.0 : y.sum;
            if (y.top < now) x = now < INFINITY ? x * exp2_fast((y.top - now) * kLog2e) : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            if (most < now) sum = most == -INFINITY || now == INFINITY ? 0.0 : sum * exp2_fast((most - now) * kLog2e);
            sum += x;
            most = now;
        }
        if (lane == 0) {
            s_from[r] = done || dead ? (double)cum : cum - logarithm(sum);   // (without a logit above -inf: not used)
            s_most[r] = done || dead ? -INFINITY : most;
            if (done && !dead) s_count[r * parts] = -1;
        }
    }
    __syncthreads();
    // entry `at` of list l; its score's image is 0 where there is none, or it scores -inf
    auto entry = [&](int l, int at) {
        const int r = (int)(((float)l + 0.5f) * by_parts), count = s_count[l];
        if (at >= count)
            return BeamBest{count < 0 && at == 0 ? score_image(s_from[r]) : 0, (uint64_t)r << 32 | (uint32_t)a.pad_token, 0.0f};
        const float2 x = staged ? s_entry[l * keep + at] : entries[(int64_t)l * keep + at];
        const float most = s_most[r];
        const double score = x.x == most ? s_from[r] : s_from[r] + ((double)x.x - (double)most);
        return BeamBest{x.x == most || most < INFINITY ? score_image(score) : 0, (uint64_t)r << 32 | (uint32_t)__float_as_int(x.y), x.x};
    };
    // ---- candidates: by the images' upper halves.  The keep-th best of 32 lists' fronts is no better than the keep-th best of all; from there
    // on the range is halved until not many more than keep are left.
    int n = kMergeHeld + 1, found = 0, round = 0;
    if (staged) {
        uint32_t best = 0, front = 0;                               // of a thread's entries, of its lists' fronts
        // (entry() without its branches)
#pragma unroll 1
        for (int i = tid; i < all; i += kMergeThreads) {
            const int l = (int)(((float)i + 0.5f) * by_keep), r = (int)(((float)l + 0.5f) * by_parts), at = i - l * keep;
            const int count = s_count[l];
            const float logit = s_entry[i].x, most = s_most[r];
            const double from = s_from[r], score = logit == most || count < 0 ? from : from + ((double)logit - (double)most);
            const bool is = count < 0 ? at == 0 : at < count && (logit == most || most < INFINITY);
            const uint64_t x = is ? score_image(score) : 0;
            s_score[i] = x;
            s_upper[i] = (uint32_t)(x >> 32);
            best = max(best, (uint32_t)(x >> 32));
        }
        __syncthreads();
#pragma unroll 1
        for (int l = tid; l < lists; l += kMergeThreads) front = max(front, s_upper[l * keep]);
        front = keep <= 32 && lists >= keep ? warp_ranked(front, keep - 1) : 0;
        best = __reduce_max_sync(0xffffffffu, best);
        if (lane == 0) { s.front[warp] = front; s.top[warp] = best; }
        __syncthreads();
        uint32_t lo = max(__reduce_max_sync(0xffffffffu, s.front[lane % (kMergeThreads / 32)]), 1u);
        uint32_t hi = __reduce_max_sync(0xffffffffu, s.top[lane % (kMergeThreads / 32)]), x = lo;
#pragma unroll 1
        for (bool first = true; first || (lo < hi && n > keep + 32); first = false) {
            int m = 0;
#pragma unroll 2
            for (int i = tid; i < all; i += kMergeThreads) m += s_upper[i] >= x;
            m = __reduce_add_sync(0xffffffffu, m);
            if (lane == 0) s.part[round & 1][warp] = m;
            __syncthreads();
            m = __reduce_add_sync(0xffffffffu, lane < kMergeThreads / 32 ? s.part[round & 1][lane] : 0);
            ++round;
            if (first || m >= keep) { lo = x; n = m; } else hi = x - 1;
            x = lo + (hi - lo + 1) / 2;
        }
        if (n <= kMergeHeld) {
#pragma unroll 2
            for (int i = tid; i < all; i += kMergeThreads) {
                if (s_upper[i] < lo) continue;
                const int l = (int)(((float)i + 0.5f) * by_keep), r = (int)(((float)l + 0.5f) * by_parts);
                const int token = s_count[l] < 0 ? a.pad_token : __float_as_int(s_entry[i].y);
                s.held[atomicAdd(&s.n, 1)] = BeamBest{s_score[i], (uint64_t)r << 32 | (uint32_t)token, s_entry[i].x};
            }
            __syncthreads();
        }
    }
    auto put = [&](int rank, const BeamBest& x) {
        const int64_t to = (int64_t)search * keep + rank;
        a.values[to] = (float)score_of_image(x.score);
        a.parents[to] = (int64_t)(x.place >> 32);
        a.tokens[to] = (int64_t)(x.place & 0xffffffffu);
    };
    if (n <= kMergeHeld) {
        // a warp an entry: how many are before it
#pragma unroll 1
        for (int i = warp; i < n; i += kMergeThreads / 32) {
            const BeamBest x = s.held[i];
            int rank = 0;
#pragma unroll 1
            for (int j = lane; j < n; j += 32) rank += s.held[j].before(x);
            rank = __reduce_add_sync(0xffffffffu, rank);
            if (lane == 0 && rank < keep) put(rank, x);
        }
        found = min(n, keep);
    } else {
        // more candidates than are held (many equal ones): the best of the lists' fronts, `keep` times
        __syncthreads();
        for (int l = tid; l < lists; l += kMergeThreads) s_at[l] = 0;
#pragma unroll 1
        for (; found < keep; ++found) {
            BeamBest best{0, ~0ull, 0.0f};
            int owner = -1;
#pragma unroll 1
            for (int l = tid; l < lists; l += kMergeThreads) {      // (each thread reads and advances its own lists only)
                const BeamBest e = entry(l, s_at[l]);
                if (e.score && e.before(best)) { best = e; owner = l; }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const BeamBest y{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.place, o),
                                 __shfl_xor_sync(0xffffffffu, best.logit, o)};
                const int y_owner = __shfl_xor_sync(0xffffffffu, owner, o);
                if (y.before(best)) { best = y; owner = y_owner; }
            }
            if (lane == 0) { s.best[found & 1][warp] = best; s.owner[found & 1][warp] = owner; }
            __syncthreads();
            best = s.best[found & 1][0];
            owner = s.owner[found & 1][0];
#pragma unroll 1
            for (int w = 1; w < kMergeThreads / 32; ++w)
                if (s.best[found & 1][w].before(best)) { best = s.best[found & 1][w]; owner = s.owner[found & 1][w]; }
            if (owner < 0) break;
            if (tid == 0) put(found, best);
            if (owner % kMergeThreads == tid) ++s_at[owner];
        }
    }
    // ---- too few: continuations of -inf, from the first on
#pragma unroll 1
    for (int64_t i0 = 0; found < keep && i0 < (int64_t)beams * a.V; i0 += kMergeThreads, ++round) {
        const int64_t i = i0 + tid;
        bool none = false;
        int64_t r = 0, t = 0;
        if (i < (int64_t)beams * a.V) {
            r = i / a.V;
            t = i - r * a.V;
            if (beam_dead(a, row0 + r)) none = true;
            else if (beam_done(a, row0 + r)) none = t != a.pad_token;
            else {
                const float x = to_float(static_cast<const T*>(a.logits)[search * a.stride_b + r * a.stride_r + t]);
                none = !(x > -INFINITY) || (s_most[r] == INFINITY && x < INFINITY);
            }
        }
        const unsigned these = __ballot_sync(0xffffffffu, none);
        if (lane == 0) s.part[round & 1][warp] = __popc(these);
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll 1
        for (int w = 0; w < kMergeThreads / 32; ++w) {
            if (w < warp) before += s.part[round & 1][w];
            total += s.part[round & 1][w];
        }
        const int to = found + before + __popc(these & ((1u << lane) - 1));
        if (none && to < keep) {
            a.values[(int64_t)search * keep + to] = -INFINITY;
            a.parents[(int64_t)search * keep + to] = r;
            a.tokens[(int64_t)search * keep + to] = t;
        }
        found += total;
    }
}

template <class T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ skv_beam_args a, int parts, bool staged, float by_parts, float by_keep) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    __shared__ MergeShared s;
    wait_for_dependency();
    beam_merge<T>(a, parts, staged, by_parts, by_keep, blockIdx.x, s, s_raw);
}

// The same in one launch: a cluster of blocks makes a search's lists, and its first block merges them.
static_assert(kMergeThreads == 32 * kClusterWarps);   // (a warp a part of a beam: at most kCluster * kClusterWarps beams and lists)
template <class T, int LOADS, bool ALIGNED>
__global__ void __launch_bounds__(kMergeThreads, 2) beam_small_kernel(const __grid_constant__ skv_beam_args a, int parts, int64_t blocks, float by_parts, float by_keep) {
    extern __shared__ __align__(16) unsigned char s_raw[];       // the warps' lists, then the merge's
    int rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int warp = threadIdx.x >> 5, search = blockIdx.x / kCluster, job = rank + kCluster * warp, lists = a.beams * parts;
    wait_for_dependency();
    if (job < lists) beam_list<T, LOADS, ALIGNED>(a, parts, blocks, (int64_t)search * lists + job, reinterpret_cast<ListShared*>(s_raw)[warp]);
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (rank == 0) beam_merge<T>(a, parts, true, by_parts, by_keep, search, *reinterpret_cast<MergeShared*>(s_raw), s_raw + sizeof(MergeShared));
}

template <class T, bool ALIGNED>
int launch_beam(const skv_beam_args& a, cudaStream_t st) {
    const BeamShape small = small_shape(a.B, a.beams, a.V, a.keep, sizeof(T), ALIGNED);
    if (small.parts > 0) {
        const size_t entries = (size_t)a.beams * small.parts * a.keep, merge = sizeof(MergeShared) + a.beams * 12 + a.beams * small.parts * 8 + entries * 20;
        constexpr size_t some = kClusterWarps * sizeof(ListShared), most = sizeof(MergeShared) + kCluster * kClusterWarps * 20 + kMergeFew * 20;   // 45, 55 KB
        const size_t smem = merge > some ? merge : some;
        const auto kernel = small.loads == kManyLoads ? beam_small_kernel<T, kManyLoads, ALIGNED> : beam_small_kernel<T, kFewLoads, ALIGNED>;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(most > some ? most : some));
        if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "beam_select: %s", cudaGetErrorString(e));
        launch_cluster_after(kernel, dim3((unsigned)a.B * kCluster), dim3(kCluster), kMergeThreads, smem, st, a, small.parts, small.blocks,
                             1.0f / (float)small.parts, 1.0f / (float)a.keep);
        return check_launch("beam_select");
    }
    const BeamShape s = beam_shape(a.B, a.beams, a.V, a.keep, sizeof(T), ALIGNED);
    const int64_t jobs = (int64_t)a.B * a.beams * s.parts;
    const unsigned grid = (unsigned)((jobs + kBeamWarps - 1) / kBeamWarps);
    prefer_shared<beam_lists_kernel<T, kManyLoads, ALIGNED>>(50);   // (32 searches of 8 beams 32.5 -> 27.7 us)
    prefer_shared<beam_lists_kernel<T, kFewLoads, ALIGNED>>(50);
    prefer_shared<beam_merge_kernel<T>>(50);
    if (s.loads == kManyLoads) beam_lists_kernel<T, kManyLoads, ALIGNED><<<grid, 32 * kBeamWarps, 0, st>>>(a, s.parts, s.blocks);
    else beam_lists_kernel<T, kFewLoads, ALIGNED><<<grid, 32 * kBeamWarps, 0, st>>>(a, s.parts, s.blocks);
    if (const int rc = check_launch("beam_select")) return rc;
    const int64_t lists = (int64_t)a.beams * s.parts, entries = lists * a.keep;
    const size_t fixed = (size_t)a.beams * 12 + lists * 8;   // at most 80 KB
    const bool staged = entries <= kMergeEntries && fixed + entries * 20 <= 200 * 1024;
    const size_t smem = fixed + (staged ? entries * 20 : 0);
    if (smem > 24 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(beam_merge_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024);
        if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "beam_select: %s", cudaGetErrorString(e));
    }
    launch_after(beam_merge_kernel<T>, dim3(a.B), kMergeThreads, smem, st, a, s.parts, staged, 1.0f / (float)s.parts, 1.0f / (float)a.keep);
    return check_launch("beam_select");
}

template <class T>
int launch_beam(const skv_beam_args& a, cudaStream_t st) {
    constexpr int PER = 16 / (int)sizeof(T);
    const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.stride_b % PER == 0 && a.stride_r % PER == 0;
    return aligned ? launch_beam<T, true>(a, st) : launch_beam<T, false>(a, st);
}

// ------------------------------------------------------------------------------------------ reordering
constexpr int kReorderThreads = 256, kReorderBeams = 1024;
constexpr int kReorderBytes = 16 * 1024;   // that a block copies at least, where there are as many

// Copies `bytes` bytes with a block, four 16-byte loads a thread on the way where both ends are on 16-byte boundaries.
__device__ __noinline__ void move_block(char* to, const char* from, int bytes) {
    constexpr int FLY = 4;
    const int n = ((reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(from)) & 15) == 0 ? bytes / 16 : 0;
    uint4* d = reinterpret_cast<uint4*>(to);
    const uint4* s = reinterpret_cast<const uint4*>(from);
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += FLY * kReorderThreads) {
        uint4 x[FLY];
#pragma unroll
        for (int f = 0; f < FLY; ++f) x[f] = s[min(i + f * kReorderThreads, n - 1)];
#pragma unroll
        for (int f = 0; f < FLY; ++f)
            if (i + f * kReorderThreads < n) d[i + f * kReorderThreads] = x[f];
    }
#pragma unroll 1
    for (int i = 16 * n + threadIdx.x; i < bytes; i += kReorderThreads) to[i] = from[i];
}

// A block a beam and a share of its last page's (key head, K or V) blocks.  Every block finds out by itself where its beam comes from: a
// beam is the keeper of its parent's last page if it is the parent, or the first child of a parent that does not go on from itself; the
// n-th beam that is no keeper takes the last page of the n-th beam without children.  Pages are copied from keepers' parents, which have
// children, to pages of beams that have none, so no block reads what another writes; the old table is only read.  A full page may be
// shared, so one is neither taken from a beam without children nor left behind the tokens of a beam that was longer (beams of a group
// that are not equally long).
__global__ void __launch_bounds__(kReorderThreads, 5) pool_reorder_kernel(const __grid_constant__ skv_pool_reorder_args a) {
    __shared__ int s_parent[kReorderBeams];
    __shared__ bool s_extra[kReorderBeams], s_childless[kReorderBeams];
    __shared__ int s_donor;
    const int tid = threadIdx.x, lane = tid & 31, R = a.beams, P = a.pool.page_size, width = a.pool.table_width;
    const int64_t row = blockIdx.x, row0 = row / R * R;
    const int c = (int)(row - row0);
    auto parent = [&](int r) {
        const int64_t p = a.parents_bytes == 8 ? __ldg(static_cast<const long long*>(a.parents) + row0 + r)
                                               : (long long)__ldg(static_cast<const int32_t*>(a.parents) + row0 + r);
        return p >= 0 && p < R ? (int)p : -1;
    };
    int p, donor = -1;                                           // donor: -1 where the beam keeps its parent's last page
    bool extra;
    if (R <= 32) {                                               // a warp by itself, a lane a beam
        const int mine = lane < R ? parent(lane) : -1;
        const unsigned some = __reduce_or_sync(0xffffffffu, mine >= 0 ? 1u << mine : 0u), alike = __match_any_sync(0xffffffffu, mine);
        const unsigned self = __ballot_sync(0xffffffffu, mine == lane);
        const bool keeps = mine == lane || (mine >= 0 && !(self >> mine & 1) && __ffs(alike) - 1 == lane);
        const unsigned extras = __ballot_sync(0xffffffffu, mine >= 0 && !keeps);
        p = __shfl_sync(0xffffffffu, mine, c);
        extra = extras >> c & 1;
        if (!extra && blockIdx.y) return;
        unsigned childless = ~some & (R == 32 ? 0xffffffffu : (1u << R) - 1);
        if (extra) {
            for (int n = __popc(extras & ((1u << c) - 1)); n > 0; --n) childless &= childless - 1;
            donor = __ffs(childless) - 1;
        }
    } else {
        for (int r = tid; r < R; r += kReorderThreads) s_parent[r] = parent(r);
        if (tid == 0) s_donor = -1;
        __syncthreads();
        p = s_parent[c];
        for (int r = tid; r < R; r += kReorderThreads) {
            bool childless = true, first = true;
            const int q = s_parent[r];
            for (int o = 0; o < R; ++o) {
                childless &= s_parent[o] != r;
                if (o < r) first &= s_parent[o] != q;
            }
            s_childless[r] = childless;
            s_extra[r] = q >= 0 && q != r && !(first && s_parent[q] != q);
        }
        __syncthreads();
        extra = s_extra[c];
        if (!extra && blockIdx.y) return;
        if (extra && tid < 32) {
            int rank = 0, seen = 0;
            for (int r0 = 0; r0 < c; r0 += 32) rank += __popc(__ballot_sync(0xffffffffu, r0 + lane < c && s_extra[r0 + lane]));
            for (int r0 = 0; r0 < R; r0 += 32) {
                const bool mine = r0 + lane < R && s_childless[r0 + lane];
                const unsigned these = __ballot_sync(0xffffffffu, mine);
                if (mine && seen + __popc(these & ((1u << lane) - 1)) == rank) s_donor = r0 + lane;
                seen += __popc(these);
            }
        }
        __syncthreads();
        donor = s_donor;
    }
    const int length = p < 0 ? 0 : __ldg(a.lengths + row0 + p), tokens = max(0, length), j = tokens / P;
    const int rows = j < width ? tokens - j * P : 0;             // of the last page, if it is partly filled
    const int32_t* old = a.pool.block_table + (row0 + max(p, 0)) * a.pool.table_stride;
    const bool copy = extra && rows > 0;
    int target = -1;
    if (copy) {
        const int source = __ldg(old + j);
        if (donor >= 0 && max(0, __ldg(a.lengths + row0 + donor)) / P <= j)   // (else its page there is full)
            target = __ldg(a.pool.block_table + (row0 + donor) * a.pool.table_stride + j);
        if (target < 0 || target >= a.pool.num_pages || source < 0 || source >= a.pool.num_pages || source == target) {
            target = -1;
            if (a.error_flag && tid == 0) atomicExch(a.error_flag, 1);
        } else {
            const int64_t bytes = pool_row_bytes(a.pool.precision, a.pool.head_dim);
            const int64_t scales = a.pool.precision < 2 ? 0 : a.pool.precision == 2 ? 4 : 4ll * (a.pool.head_dim / a.pool.int4_group);
            for (int part = blockIdx.y; part < 2 * a.pool.heads; part += gridDim.y) {
                const int head = part >> 1;
                const bool is_v = part & 1;
                const int64_t s = (int64_t)source * a.pool.heads + head, d = (int64_t)target * a.pool.heads + head;
                char* values = static_cast<char*>(is_v ? a.pool.v : a.pool.k);
                move_block(values + d * P * bytes, values + s * P * bytes, (int)(rows * bytes));
                if (scales) {
                    char* base = reinterpret_cast<char*>(is_v ? a.pool.scale_v : a.pool.scale_k);
                    move_block(base + d * P * scales, base + s * P * scales, (int)(rows * scales));
                }
                if (a.bounds && !is_v) {
                    const int64_t n = 2ll * a.pool.head_dim;
                    move_block(reinterpret_cast<char*>(a.bounds) + d * n, reinterpret_cast<const char*>(a.bounds) + s * n, (int)n);
                    if (tid == 0) a.steps[d] = a.steps[s];
                }
            }
        }
    }
    if (blockIdx.y) return;
    int32_t* table = a.new_table + row * width;
    const int32_t* own = a.pool.block_table + row * a.pool.table_stride;
    const int behind = j + (rows > 0), had = max(0, __ldg(a.lengths + row)), held = had > 0 ? (had - 1) / P + 1 : 0;   // pages; of its own
    for (int i = tid; i < width; i += kReorderThreads)
        table[i] = p < 0 || (i >= behind && i < held) ? -1 : copy && i == j ? target : __ldg((i < behind ? old : own) + i);
    if (tid == 0) {
        a.new_lengths[row] = length;
        if (a.error_flag && (p < 0 || length < 0 || tokens > (int64_t)width * P || held > behind)) atomicExch(a.error_flag, 1);
    }
}

}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_beam_scratch_bytes(int B, int beams, int V, int keep) {
    if (B <= 0 || beams <= 0 || beams > kBeamMost || V <= 0 || keep <= 0) return 0;
    int parts = 1;   // of whichever type and alignment has most
    for (int i = 0; i < 4; ++i) {
        const int some = beam_shape(B, beams, V, keep, i & 1 ? 2 : 4, i & 2).parts;
        const int few = small_shape(B, beams, V, keep, i & 1 ? 2 : 4, i & 2).parts;
        if (some > parts) parts = some;
        if (few > parts) parts = few;
    }
    return (size_t)B * beams * parts * (sizeof(BeamPart) + (size_t)keep * 8);
}

int skv_beam_select(const skv_beam_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: null pointer");
    const skv_beam_args& a = *args;
    if (a.B < 0 || a.beams < 1 || a.V < 1 || a.keep < 1) return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: bad size");
    if (a.dtype < 0 || a.dtype > 2) return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: dtype %d", a.dtype);
    if (a.keep > (int64_t)a.beams * a.V)
        return fail(SKV_ERR_SHAPE, "beam_select: %d continuations of %d beams and %d tokens", a.keep, a.beams, a.V);
    if (a.finished && (a.pad_token < 0 || a.pad_token >= a.V))
        return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: pad token %d", a.pad_token);
    if (a.keep > kBeamKeep || a.beams > kBeamMost || a.V > 0x7fff0000)
        return fail(SKV_ERR_TOO_LARGE, "beam_select: keep %d (at most %d), %d beams (at most %d), %d tokens", a.keep, kBeamKeep, a.beams,
                    kBeamMost, a.V);
    if (a.B == 0) return SKV_OK;
    if (!a.logits || !a.scores || !a.values || !a.parents || !a.tokens || !a.scratch)
        return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: null pointer");
    if (reinterpret_cast<uintptr_t>(a.scratch) & 15 || reinterpret_cast<uintptr_t>(a.logits) % dtype_bytes(a.dtype))
        return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: scratch or logits are not aligned");
    if ((int64_t)a.B * a.beams > 0x7fffffff / kBeamMost) return fail(SKV_ERR_TOO_LARGE, "beam_select: too many rows");
    if (a.scratch_bytes < (int64_t)skv_beam_scratch_bytes(a.B, a.beams, a.V, a.keep))
        return fail(SKV_ERR_SCRATCH, "beam_select: scratch of %lld bytes", (long long)a.scratch_bytes);
    cudaStream_t st = as_stream(stream);
    static std::mutex launches;   // a call's two launches stay together: host threads may share a stream and its scratch
    const std::lock_guard<std::mutex> both(launches);
    if (a.dtype == kF32) return launch_beam<float>(a, st);
    if (a.dtype == kF16) return launch_beam<__half>(a, st);
    return launch_beam<__nv_bfloat16>(a, st);
}

int skv_pool_reorder(const skv_pool_reorder_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_reorder: null pointer");
    const skv_pool_reorder_args& a = *args;
    if (const int rc = check_pool(a.pool, "pool_reorder")) return rc;
    if (a.beams < 1 || a.pool.batch % a.beams) return fail(SKV_ERR_SHAPE, "pool_reorder: %d rows in groups of %d", a.pool.batch, a.beams);
    if (a.parents_bytes != 4 && a.parents_bytes != 8) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_reorder: parents of %d bytes", a.parents_bytes);
    if (a.pool.batch == 0) return SKV_OK;
    if (!a.lengths || !a.parents || !a.new_lengths || (a.pool.table_width > 0 && !a.new_table) || (!a.bounds != !a.steps))
        return fail(SKV_ERR_INVALID_ARGUMENT, "pool_reorder: null pointer");
    if (a.beams > kReorderBeams || a.pool.heads > 32767)
        return fail(SKV_ERR_TOO_LARGE, "pool_reorder: %d beams (at most %d), %d heads", a.beams, kReorderBeams, a.pool.heads);
    const int64_t scales = a.pool.precision < 2 ? 0 : a.pool.precision == 2 ? 4 : 4ll * (a.pool.head_dim / a.pool.int4_group);
    const int64_t part = a.pool.page_size * (pool_row_bytes(a.pool.precision, a.pool.head_dim) + scales), most = 2ll * a.pool.heads * part;
    if (part > 0x7fffffff || a.pool.head_dim > 1 << 28)
        return fail(SKV_ERR_TOO_LARGE, "pool_reorder: pages of %d rows of %d values", a.pool.page_size, a.pool.head_dim);
    int64_t blocks = (most + kReorderBytes - 1) / kReorderBytes;
    if (blocks > 2 * a.pool.heads) blocks = 2 * a.pool.heads;
    pool_reorder_kernel<<<dim3((unsigned)a.pool.batch, (unsigned)blocks), kReorderThreads, 0, as_stream(stream)>>>(a);
    return check_launch("pool_reorder");
}

}  // extern "C"
