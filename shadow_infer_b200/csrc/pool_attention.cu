// Attention of new tokens over the page pool: out = softmax(scale q k^T) v, one pass over the pages.
//
// Work.  The rows that share a key head (H_q / heads query heads times S_q new tokens) are cut
// into row tiles, a sequence's tokens into tiles; a unit is (sequence, key head, row tile).
// Lengths are device memory, so the host cannot split the work: the grid is as many CTAs as stay
// resident, every CTA counts the tiles of all sequences and takes an even share of their
// concatenation.  A share may cut a unit; a CTA that holds a part of one publishes (O, max, sum) of
// its part, and the last CTA of the unit to arrive joins the parts in token order,
//     O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i,    m = max_i m_i,
// so the result does not depend on the order of arrival.  Nothing waits for another CTA.
//
// Numbers.  Scores, the running maximum and sum and the accumulators are fp32; the scale and
// log2(e) are folded into q.
#include "pool.cuh"

namespace skv {

constexpr int kMaxCtas = 4096;   // arrival counters in the scratch

// ------------------------------------------------------------------------------ shares of the work
struct Share {
    long long lo, hi, total;   // this CTA's tiles [lo, hi) of all
    long long base;            // tiles of the sequences before b
    int b;                     // the sequence that holds tile lo
    int ctas;                  // CTAs that share the work
};

__device__ __forceinline__ int64_t seq_tokens(const skv_pool_attention_args& a, int b) {
    const int64_t n = a.lengths[b], cap = (int64_t)a.pool.table_width * a.pool.page_size;
    return n < 0 ? 0 : n > cap ? cap : n;
}
// Tiles of a sequence for one row tile of one head; an empty sequence keeps one, to write its zeros.
__device__ __forceinline__ int64_t seq_tiles(int64_t tokens, int tile) {
    return tokens == 0 ? 1 : (tokens + tile - 1) / tile;
}

// Every thread of the block calls this; *s is valid for all after it.  At least min_tiles a CTA.
template <int THREADS>
__device__ __forceinline__ void take_share(const skv_pool_attention_args& a, int tile, int units, int min_tiles,
                                           Share* s) {
    __shared__ long long s_part[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, B = a.pool.batch;
    const int per = (B + THREADS - 1) / THREADS, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += seq_tiles(seq_tokens(a, b), tile) * units;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_part[tid >> 5] = incl;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < (tid >> 5)) before += s_part[w];
        total += s_part[w];
    }
    before += incl - mine;
    const long long want = (total + min_tiles - 1) / min_tiles;
    const int ctas = (int)min((long long)gridDim.x, max(want, 1ll)), c = blockIdx.x;
    const long long lo = c < ctas ? c * total / ctas : total, hi = c < ctas ? (c + 1) * total / ctas : total;
    if (tid == 0) {
        s->lo = lo;
        s->hi = hi;
        s->total = total;
        s->ctas = ctas;
    }
    if (lo >= before && lo < before + mine) {
        long long base = before;
        int b = b0;
        for (;; ++b) {
            const long long n = seq_tiles(seq_tokens(a, b), tile) * units;
            if (lo < base + n) break;
            base += n;
        }
        s->b = b;
        s->base = base;
    }
    __syncthreads();
}

// The CTA whose share holds tile i.
__device__ __forceinline__ int owner_of(const Share& s, long long i) {
    return (int)(((i + 1) * s.ctas - 1) / s.total);
}

// Tokens [0, n) of its sequence that query i of sequence b sees.
__device__ __forceinline__ int64_t seen_by(const skv_pool_attention_args& a, int b, int64_t tokens, int i) {
    const int n_new = a.new_lengths ? a.new_lengths[b] : a.S_q;
    return i >= n_new ? 0 : a.causal ? tokens - n_new + 1 + i : tokens;
}

struct Segment {
    int b, hk, rt;             // unit
    int64_t tokens;            // of the sequence
    long long t0, t1;          // its tiles [t0, t1) are this CTA's
    long long first, last;     // global numbers of the unit's first and last tile
    bool whole;
    int slot;                  // partial slot of this CTA (0 or 1) if not whole
};

// The segment that starts at tile `at` of the share.
__device__ __forceinline__ Segment segment_at(const skv_pool_attention_args& a, const Share& s, long long at, int tile,
                                              int row_tiles, int& b, long long& base) {
    Segment g;
    const int units = a.pool.heads * row_tiles;
    for (;;) {
        g.tokens = seq_tokens(a, b);
        const long long nt = seq_tiles(g.tokens, tile);
        if (at < base + nt * units) {
            const long long u = (at - base) / nt;
            g.b = b;
            g.hk = (int)(u / row_tiles);
            g.rt = (int)(u % row_tiles);
            g.first = base + u * nt;
            g.last = g.first + nt - 1;
            g.t0 = at - g.first;
            g.t1 = min(nt, g.t0 + (s.hi - at));
            g.whole = g.t0 == 0 && g.t1 == nt;
            g.slot = at == s.lo ? 0 : 1;
            if (a.error_flag && a.lengths[b] > g.tokens && threadIdx.x == 0) atomicExch(a.error_flag, 1);
            return g;
        }
        base += nt * units;
        ++b;
    }
}

// ------------------------------------------------------------------------------------- publishing
// Scratch: kMaxCtas arrival counters (zeroed before the launch), then two slots a CTA of
// rows * (D + 2) floats: O [rows][D], max [rows], sum [rows].
__device__ __forceinline__ float* slot_of(const skv_pool_attention_args& a, int cta, int slot, int rows) {
    return reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kMaxCtas * 4) +
           ((int64_t)2 * cta + slot) * rows * (a.pool.head_dim + 2);
}

// Called by all threads once the CTA's part is in its slot; true for the CTA that joins.
__device__ __forceinline__ bool arrive(const skv_pool_attention_args& a, const Share& s, const Segment& g) {
    __shared__ int s_last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const int c0 = owner_of(s, g.first), c1 = owner_of(s, g.last);
        s_last = atomicAdd(reinterpret_cast<int*>(a.scratch) + c0, 1) == c1 - c0;
    }
    __syncthreads();
    const bool last = s_last;
    if (last) __threadfence();
    return last;
}

// Where query row r of a unit lives (r counts head-major: H_q / heads heads of S_q tokens).
template <class T>
__device__ __forceinline__ T* row_ptr(const skv_rows& x, int S_q, int rep, int b, int hk, int r) {
    return static_cast<T*>(x.ptr) + b * x.stride_b + (int64_t)(hk * rep + r / S_q) * x.stride_h + (r % S_q) * x.stride_s;
}

// Joins the parts of a unit in token order, a thread for each value of each row.
template <class T, int ROWS>
__device__ __forceinline__ void join(const skv_pool_attention_args& a, const Share& s, const Segment& g, int R) {
    const int D = a.pool.head_dim, rep = a.q.heads / a.pool.heads;
    const int c0 = owner_of(s, g.first), c1 = owner_of(s, g.last);
    const bool c0_starts = g.first == c0 * s.total / s.ctas;   // the unit starts at c0's first tile
    for (int i = threadIdx.x; i < ROWS * D; i += blockDim.x) {
        const int j = i / D, d = i - j * D, r = g.rt * ROWS + j;
        if (r >= R) break;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int c = c0; c <= c1; ++c) {
            const float* p = slot_of(a, c, c == c0 && !c0_starts ? 1 : 0, ROWS);
            const float mi = __ldcg(p + ROWS * D + j), li = __ldcg(p + ROWS * D + ROWS + j), oi = __ldcg(p + j * D + d);
            const float mn = fmaxf(m, mi), ref = mn == -INFINITY ? 0.0f : mn;
            const float wa = exp2f(m - ref), wb = exp2f(mi - ref);
            l = l * wa + li * wb;
            o = o * wa + oi * wb;
            m = mn;
        }
        row_ptr<T>(a.out, a.S_q, rep, g.b, g.hk, r)[d] = from_float<T>(l == 0.0f ? 0.0f : o / l);
    }
}

// --------------------------------------------------------------------------- any size and alignment
// Products on the FMA pipe from fp32 tiles in shared memory: 8 rows, 32 tokens at a time.  Thread =
// (token, rows w and w + 4) for the scores, value d for the sums.
constexpr int kAnyRows = 8, kAnyTile = 32, kAnyThreads = 128, kAnyMaxD = 512;

__host__ __device__ inline size_t any_smem(int D) {
    return ((size_t)kAnyRows * D + (size_t)kAnyTile * (D + 1) + (size_t)kAnyTile * D + kAnyRows * kAnyTile + kAnyRows) * 4;
}

template <class T>
__global__ void __launch_bounds__(kAnyThreads) pool_attention_any_kernel(const __grid_constant__ skv_pool_attention_args a,
                                                                         int row_tiles) {
    extern __shared__ float any_sm[];
    __shared__ Share s;
    const int D = a.pool.head_dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* sq = any_sm;
    float* sk = sq + kAnyRows * D;
    float* sv = sk + kAnyTile * (D + 1);
    float* sp = sv + kAnyTile * D;
    float* sc = sp + kAnyRows * kAnyTile;
    const int rep = a.q.heads / a.pool.heads, R = rep * a.S_q;
    take_share<kAnyThreads>(a, kAnyTile, a.pool.heads * row_tiles, 2, &s);
    int b = s.b;
    long long base = s.base;
    for (long long at = s.lo; at < s.hi;) {
        const Segment g = segment_at(a, s, at, kAnyTile, row_tiles, b, base);
        at += g.t1 - g.t0;
        const int r0 = g.rt * kAnyRows;
        __syncthreads();
        for (int i = tid; i < kAnyRows * D; i += kAnyThreads) {
            const int r = r0 + i / D;
            sq[i] = r < R ? to_float(row_ptr<const T>(a.q, a.S_q, rep, g.b, g.hk, r)[i % D]) * (a.scale * 1.4426950408889634f)
                          : 0.0f;
        }
        int64_t see[2];   // tokens that each of this warp's two rows sees
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[kAnyRows][kAnyMaxD / kAnyThreads];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            see[i] = seen_by(a, g.b, g.tokens, (r0 + warp + 4 * i) % a.S_q);
#pragma unroll
        for (int j = 0; j < kAnyRows; ++j)
#pragma unroll
            for (int i = 0; i < kAnyMaxD / kAnyThreads; ++i) o[j][i] = 0.0f;
        for (long long t = g.t0; t < g.t1; ++t) {
            const int64_t tok0 = t * kAnyTile;
            __syncthreads();
            for (int j = warp; j < kAnyTile; j += kAnyThreads / 32) {
                int64_t row = tok0 + j < g.tokens ? pool_row(a.pool, g.b, tok0 + j) : -1;
                if (row < 0 && tok0 + j < g.tokens && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
                if (row >= 0) row += (int64_t)g.hk * a.pool.page_size;
                for (int d = lane; d < D; d += 32) {
                    sk[j * (D + 1) + d] = row >= 0 ? pool_value(a.pool, false, row, d) : 0.0f;
                    sv[j * D + d] = row >= 0 ? pool_value(a.pool, true, row, d) : 0.0f;
                }
                if (lane == 0) sp[j] = row >= 0 ? 1.0f : 0.0f;   // whether there is such a token
            }
            __syncthreads();
            const bool held = sp[lane] != 0.0f;
            float x[2] = {0.0f, 0.0f};
#pragma unroll 4
            for (int d = 0; d < D; ++d) {
                const float kd = sk[lane * (D + 1) + d];
                x[0] = fmaf(kd, sq[warp * D + d], x[0]);
                x[1] = fmaf(kd, sq[(warp + 4) * D + d], x[1]);
            }
            __syncthreads();   // sp is about to hold the weights
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!held || tok0 + lane >= see[i]) x[i] = -INFINITY;
                const float mn = fmaxf(m[i], warp_max(x[i])), ref = mn == -INFINITY ? 0.0f : mn;
                const float p = exp2f(x[i] - ref), c = exp2f(m[i] - ref);
                float sum = p;
#pragma unroll
                for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                l[i] = l[i] * c + sum;
                m[i] = mn;
                sp[(warp + 4 * i) * kAnyTile + lane] = p;
                if (lane == 0) sc[warp + 4 * i] = c;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kAnyMaxD / kAnyThreads; ++i) {
                const int d = tid + i * kAnyThreads;
                if (d >= D) break;
#pragma unroll
                for (int j = 0; j < kAnyRows; ++j) o[j][i] *= sc[j];
#pragma unroll 4
                for (int k = 0; k < kAnyTile; ++k) {
                    const float v = sv[k * D + d];
#pragma unroll
                    for (int j = 0; j < kAnyRows; ++j) o[j][i] = fmaf(sp[j * kAnyTile + k], v, o[j][i]);
                }
            }
        }
        __syncthreads();
        if (lane == 0) {   // sums and maxima to where every thread reads them
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sp[warp + 4 * i] = l[i];
                sp[kAnyRows + warp + 4 * i] = m[i];
            }
        }
        __syncthreads();
        if (g.whole) {
#pragma unroll
            for (int i = 0; i < kAnyMaxD / kAnyThreads; ++i) {
                const int d = tid + i * kAnyThreads;
                if (d >= D) break;
#pragma unroll
                for (int j = 0; j < kAnyRows; ++j)
                    if (r0 + j < R)
                        row_ptr<T>(a.out, a.S_q, rep, g.b, g.hk, r0 + j)[d] =
                            from_float<T>(sp[j] == 0.0f ? 0.0f : o[j][i] / sp[j]);
            }
            continue;
        }
        float* part = slot_of(a, blockIdx.x, g.slot, kAnyRows);
#pragma unroll
        for (int i = 0; i < kAnyMaxD / kAnyThreads; ++i) {
            const int d = tid + i * kAnyThreads;
            if (d >= D) break;
#pragma unroll
            for (int j = 0; j < kAnyRows; ++j) part[j * D + d] = o[j][i];
        }
        if (tid < kAnyRows) {
            part[kAnyRows * D + tid] = sp[kAnyRows + tid];
            part[kAnyRows * D + kAnyRows + tid] = sp[tid];
        }
        if (arrive(a, s, g)) join<T, kAnyRows>(a, s, g, R);
    }
}

template <class T>
int launch_any(const skv_pool_attention_args& a, cudaStream_t st) {
    const int R = a.q.heads / a.pool.heads * a.S_q, row_tiles = (R + kAnyRows - 1) / kAnyRows;
    const size_t smem = any_smem(a.pool.head_dim);
    cudaError_t e = cudaFuncSetAttribute(pool_attention_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    int per_sm = 1;
    if (e == cudaSuccess)
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, pool_attention_any_kernel<T>, kAnyThreads, smem);
    if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
    int grid = sm_count() * (per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm);
    if (grid > kMaxCtas) grid = kMaxCtas;
    pool_attention_any_kernel<T><<<grid, kAnyThreads, smem, st>>>(a, row_tiles);
    return check_launch("pool_attention");
}

}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_pool_attention_scratch_bytes(int D) {
    return D <= 0 ? 0 : (size_t)kMaxCtas * 4 + (size_t)sm_count() * 8 * 2 * kAnyRows * (D + 2) * 4;
}

int skv_pool_attention(const skv_pool_attention_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: null pointer");
    const skv_pool_attention_args& a = *args;
    int rc;
    if ((rc = check_pool(a.pool, "pool_attention")) || (rc = check_rows(a.q, a.pool.batch > 0 && a.S_q > 0, "pool_attention", "q")) ||
        (rc = check_rows(a.out, a.pool.batch > 0 && a.S_q > 0, "pool_attention", "out")))
        return rc;
    if (a.S_q < 0) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: bad size");
    if (a.q.heads != a.out.heads || a.q.heads % a.pool.heads || a.q.dtype != a.out.dtype)
        return fail(SKV_ERR_SHAPE, "pool_attention: %d query heads, %d outputs, %d key heads", a.q.heads, a.out.heads,
                    a.pool.heads);
    if (a.pool.batch == 0 || a.S_q == 0 || a.q.heads == 0) return SKV_OK;
    if (!a.lengths || !a.scratch) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: null pointer");
    if (a.pool.head_dim > kAnyMaxD)
        return fail(SKV_ERR_UNSUPPORTED, "pool_attention: head_dim %d above %d", a.pool.head_dim, kAnyMaxD);
    if ((int64_t)a.q.heads * a.S_q > (1 << 28) || a.pool.batch > (1 << 24))
        return fail(SKV_ERR_TOO_LARGE, "pool_attention: too many rows");
    if (a.scratch_bytes < (int64_t)skv_pool_attention_scratch_bytes(a.pool.head_dim))
        return fail(SKV_ERR_SCRATCH, "pool_attention: scratch of %lld bytes", (long long)a.scratch_bytes);
    cudaStream_t st = as_stream(stream);
    const cudaError_t e = cudaMemsetAsync(a.scratch, 0, kMaxCtas * 4, st);
    if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
    if (a.q.dtype == kF32) return launch_any<float>(a, st);
    if (a.q.dtype == kF16) return launch_any<__half>(a, st);
    return launch_any<__nv_bfloat16>(a, st);
}

}  // extern "C"
