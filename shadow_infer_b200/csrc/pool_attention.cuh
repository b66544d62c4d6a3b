// What the attention kernels over the page pool share: their CTAs' shares of the work, and the
// publishing and joining of parts (the split is described in pool_attention.cu).
#pragma once

#include "pool.cuh"

namespace skv {

constexpr int kMaxCtas = 4096;      // arrival counters in the scratch
constexpr int kRowsPerSm = 128;     // rows of partial results in the scratch for each SM: CTAs x 2 slots x rows

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

// Value d of output row r of a unit, rounded to the output's type.
__device__ __forceinline__ void store_out(const skv_pool_attention_args& a, int b, int hk, int r, int d, float x) {
    const int rep = a.q.heads / a.pool.heads;
    if (a.out.dtype == kF32) row_ptr<float>(a.out, a.S_q, rep, b, hk, r)[d] = x;
    else if (a.out.dtype == kF16) row_ptr<__half>(a.out, a.S_q, rep, b, hk, r)[d] = __float2half_rn(x);
    else row_ptr<__nv_bfloat16>(a.out, a.S_q, rep, b, hk, r)[d] = __float2bfloat16_rn(x);
}

// Joins the parts of a unit in token order, a thread for each value of each row.
template <int ROWS>
__device__ __forceinline__ void join(const skv_pool_attention_args& a, const Share& s, const Segment& g, int R) {
    const int D = a.pool.head_dim;
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
        store_out(a, g.b, g.hk, r, d, l == 0.0f ? 0.0f : o / l);
    }
}

}  // namespace skv
