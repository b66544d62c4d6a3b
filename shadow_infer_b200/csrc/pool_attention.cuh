// What the attention kernels over the page pool share: their CTAs' shares of the work, and the
// publishing and joining of parts (the split is described in pool_attention.cu).
#pragma once

#include "pool.cuh"

namespace skv {

constexpr int kMaxCtas = 4096;      // arrival counters in the scratch
// Rows of partial results in the scratch for each SM, CTAs x 2 slots x rows; the tcgen05 kernel takes heads of up to kManyD values.
constexpr int kRowsPerSm = 128, kManyD = 256;
__host__ __device__ constexpr int rows_per_sm(int D) { return D <= 128 ? 512 : D <= kManyD ? 256 : kRowsPerSm; }

// ------------------------------------------------------------------------------ shares of the work
// Tile numbers fit 31 bits: a launch takes no more sequences than the most that their tables allow (by_sequences).
struct Share {
    int lo, hi, total;         // this CTA's tiles [lo, hi) of all
    int base;                  // tiles of the sequences before b
    int b;                     // the sequence that holds tile lo
    int pad;                   // tiles that a unit costs on top of its own
    int each, more;            // a share is `each` tiles, one more for the first `more` CTAs
    // `total` tiles over at most `grid` CTAs, at least min_tiles each; returns how many CTAs have a share.
    __device__ __forceinline__ int cut(int all, int grid, int min_tiles, int on_top) {
        const int ctas = min(grid, max(1, (all + min_tiles - 1) / min_tiles));
        each = all / ctas;
        more = all - each * ctas;
        total = all;
        pad = on_top;
        return ctas;
    }
    __device__ __forceinline__ int first_of(int cta) const { return cta * each + min(cta, more); }
    __device__ __forceinline__ int owner_of(int tile) const {
        const int head = more * (each + 1);
        return tile < head ? tile / (each + 1) : more + (tile - head) / each;
    }
};

// The most tokens of a sequence: what its table names, and what leaves room to round up to a tile in 31 bits.
__host__ __device__ inline int64_t token_cap(const skv_pool_attention_args& a) {
    const int64_t cap = (int64_t)a.pool.table_width * a.pool.page_size;
    return cap < 0x7fffff00 ? cap : 0x7fffff00;
}
template <bool FRESH = false>
__device__ __forceinline__ int seq_tokens(const skv_pool_attention_args& a, int b) {
    const int64_t n = number_at<FRESH>(a.lengths + b), cap = token_cap(a);
    return (int)(n < 0 ? 0 : n > cap ? cap : n);
}
// Tiles of a sequence for one row tile of one head; an empty sequence keeps one, to write its zeros.
__device__ __forceinline__ int seq_tiles(int tokens, int tile) { return max(1, (tokens + tile - 1) / tile); }
// A unit costs its tiles and what it takes to lay out its queries and to join its warps' sums, about as long as `pad` tiles
// more: the shares count them as tiles behind the unit's own, in which nothing is done.  (Without them a CTA that got only
// short sequences was the last by far: 32 int8 sequences of 1 to 4096 tokens took 68 us, with three tiles a unit 45.)

// Every thread of the block calls this; *s is valid for all after it.  At least min_tiles a CTA.
// cost(b): the tiles of sequence b's units, with what each counts on top.
// few: units that are not to be cut, as no sequence has more than min_tiles tiles (0: cut anywhere).
template <int THREADS, class Cost>
__device__ __forceinline__ void take_share(const skv_pool_attention_args& a, Cost cost, int pad, int min_tiles, Share* s, int few = 0) {
    __shared__ int s_part[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, B = a.pool.batch;
    const int per = (B + THREADS - 1) / THREADS, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += cost(b);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_part[tid >> 5] = incl;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < (tid >> 5)) before += s_part[w];
        total += s_part[w];
    }
    before += incl - mine;
    Share t;
    const int ctas = t.cut(total, few > 0 && few <= (int)gridDim.x ? few : gridDim.x, min_tiles, pad);
    const int c = blockIdx.x;
    t.lo = c < ctas ? t.first_of(c) : total;
    t.hi = c < ctas ? t.first_of(c + 1) : total;
    t.b = 0;
    t.base = 0;
    if (t.lo >= before && t.lo < before + mine) {   // one thread
        t.base = before;
        for (t.b = b0;; ++t.b) {
            const int n = cost(t.b);
            if (t.lo < t.base + n) break;
            t.base += n;
        }
        *s = t;
    } else if (t.lo == total && tid == 0) {         // nothing for this CTA
        *s = t;
    }
    __syncthreads();
}

// The same for units that all see their whole sequence.
template <int THREADS, bool FRESH = false>
__device__ __forceinline__ void take_share(const skv_pool_attention_args& a, int tile, int units, int pad, int min_tiles,
                                           Share* s) {
    // a single short sequence: a CTA a unit and nothing to join (128 tokens of 32 fp16 heads 11.3 -> 7.8 us)
    const bool whole = a.pool.batch == 1 && seq_tiles(seq_tokens<FRESH>(a, 0), tile) <= min_tiles;
    take_share<THREADS>(a, [&](int b) { return (seq_tiles(seq_tokens<FRESH>(a, b), tile) + pad) * units; }, pad, min_tiles, s, whole ? units : 0);
}

// ------------------------------------------------------------------------------- listed pages only
// A query's own choice of pages makes a (sequence, new token, key head) a sequence of its own: its table holds the listed pages,
// its length their tokens, and its one head is that head's block of a page (a pool of num_pages * heads pages of one head is the
// same memory).  The last page that the query sees, the only one that may be partly seen, comes last in an ascending list, so
// the tokens seen are a prefix as they are of any other sequence, and the kernels need no other case.  The tables are made by a
// launch of their own, or where units are split by their number by every CTA for its own unit.
struct AttentionCall : skv_pool_attention_args {
    const skv_pool_sparse_args* lists;   // where reserved < 0 (in a kernel's arguments it is the CTAs of a unit, or 0)
};
__host__ __device__ inline int64_t list_stride(int keep) { return ((int64_t)keep + 31) & ~31ll; }   // tables on 128-byte lines

// A warp makes unit u's table and length.  (Its kernel may have started before the choice of pages had ended: nothing here, nor behind it, is
// read by a read-only load.)
__device__ __forceinline__ void list_table(const skv_pool_sparse_args& s, int u, int units) {
    const skv_pool_attention_args& a = s.attention;
    const int lane = threadIdx.x & 31, P = a.pool.page_size;
    const int h = u % a.pool.heads, bi = u / a.pool.heads, i = bi % a.S_q, b = bi / a.S_q;
    const int32_t* list = s.pages + b * s.pages_stride_b + h * s.pages_stride_h + i * s.pages_stride_s;
    int e = lane < s.keep ? list[lane] : -1;
    const int tokens = seq_tokens<true>(a, b), n_new = a.new_lengths ? a.new_lengths[b] : a.S_q;
    const int seen = i >= n_new ? 0 : a.causal ? max(0, tokens - n_new + 1 + i) : tokens, pages = seen > 0 ? (seen - 1) / P + 1 : 0;
    int32_t* table = static_cast<int32_t*>(s.tables) + u * list_stride(s.keep);
    int top = -1, count = 0, last = -1;   // the largest entry so far, those that count and the last of them
    bool bad = a.lengths[b] != tokens;
#pragma unroll 1
    for (int k0 = 0; k0 < s.keep; k0 += 32) {
        if (k0 > 0) e = k0 + lane < s.keep ? list[k0 + lane] : -1;
        int upto = e;   // the largest of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto = max(upto, x);
        }
        upto = max(top, upto);
        int before = __shfl_up_sync(0xffffffffu, upto, 1);
        if (lane == 0) before = top;
        const bool counts = e > before && e < pages;
        bad |= e < -1 || e >= a.pool.table_width || (e >= 0 && e <= before);
        const unsigned these = __ballot_sync(0xffffffffu, counts);
        if (counts) {
            const int page = a.pool.block_table[b * a.pool.table_stride + e];
            table[count + __popc(these & ((1u << lane) - 1))] = page >= 0 && page < a.pool.num_pages ? page * a.pool.heads + h : -1;
        }
        if (these) last = __shfl_sync(0xffffffffu, e, 31 - __clz(these));
        count += __popc(these);
        top = __shfl_sync(0xffffffffu, upto, 31);
    }
    if (bad && a.error_flag) atomicExch(a.error_flag, 1);
    if (lane == 0)
        static_cast<int32_t*>(s.tables)[units * list_stride(s.keep) + u] =
            count == 0 ? 0 : last == pages - 1 ? (count - 1) * P + (seen - last * P) : count * P;
}
int launch_tables(const skv_pool_sparse_args& s, cudaStream_t st);   // of all units

// Instead of an even share of everything (the sequences have one head, and their tables and lengths are made here, too):
// the tiles of one unit (sequence and row tile) over `splits` CTAs, tiles numbered as if every CTA of a unit had `each`, so that a
// tile's CTA is found as in a share;  or, where there are fewer CTAs than sequences, a run of whole sequences a CTA.
template <int THREADS>
__device__ __forceinline__ void take_listed(const skv_pool_attention_args& a, const skv_pool_sparse_args& lists, int tile, int row_tiles, Share* s) {
    const int splits = a.reserved, warp = threadIdx.x >> 5, B = a.pool.batch;
    const bool run = gridDim.x < (unsigned)B;
    int unit = 0, b0, b1;
    if (run) {
        const int each = (unsigned)B / gridDim.x, more = B - each * gridDim.x, c = blockIdx.x;
        b0 = c * each + min(c, more);
        b1 = b0 + each + (c < more);
    } else {
        unit = splits > 1 ? blockIdx.x / splits : blockIdx.x;
        b0 = row_tiles > 1 ? unit / row_tiles : unit;
        b1 = b0 + 1;
    }
#pragma unroll 1
    for (int b = b0 + warp; b < b1; b += THREADS / 32) list_table(lists, b, B);
    __syncthreads();
    if (threadIdx.x == 0) {
        Share t;
        t.more = t.pad = 0;
        t.total = 0x7fffffff;
        t.b = b0;
        if (run) {
            t.each = 0x7fffffff;
            t.lo = t.hi = t.base = 0;
            for (int b = b0; b < b1; ++b) t.hi += seq_tiles(seq_tokens<true>(a, b), tile) * row_tiles;
        } else {
            const int rt = unit - b0 * row_tiles, tiles = seq_tiles(seq_tokens<true>(a, b0), tile);
            t.each = (tiles + splits - 1) / splits;
            const int first = unit * splits * t.each;
            t.lo = (int)blockIdx.x * t.each;
            t.hi = min(t.lo + t.each, first + tiles);
            t.base = first - rt * tiles;
        }
        *s = t;
    }
    __syncthreads();
}

// Tokens [0, n) of its sequence that query i of sequence b sees.
__device__ __forceinline__ int seen_by(const skv_pool_attention_args& a, int b, int tokens, int i) {
    const int n_new = a.new_lengths ? __ldg(a.new_lengths + b) : a.S_q;
    return i >= n_new ? 0 : a.causal ? max(0, tokens - n_new + 1 + i) : tokens;
}

struct Segment {
    int b, hk, rt;             // unit
    int tokens;                // of the sequence
    int t0, t1;                // its tiles [t0, t1) are this CTA's (none: the share starts behind the unit's last)
    int next;                  // the tile of the share behind them
    int first, last;           // global numbers of the unit's first and last tile
    bool whole;
    int slot;                  // partial slot of this CTA (0 or 1) if not whole
};

// The segment that starts at tile `at` of the share.
template <bool FRESH = false>
__device__ __forceinline__ Segment segment_at(const skv_pool_attention_args& a, const Share& s, int at, int tile,
                                              int row_tiles, int& b, int& base) {
    Segment g;
    const int units = a.pool.heads * row_tiles;
    for (;;) {
        g.tokens = seq_tokens<FRESH>(a, b);
        const int nt = seq_tiles(g.tokens, tile), all = nt + s.pad;
        if (at < base + all * units) {
            const int u = (at - base) / all;
            g.b = b;
            g.hk = u / row_tiles;
            g.rt = u - g.hk * row_tiles;
            g.first = base + u * all;
            g.last = g.first + nt - 1;
            g.t0 = at - g.first;
            g.next = min(g.first + all, s.hi);
            g.t1 = min(nt, g.next - g.first);
            g.whole = g.t0 == 0 && g.t1 == nt;
            g.slot = at == s.lo ? 0 : 1;
            if (a.error_flag && a.lengths[b] != g.tokens && threadIdx.x == 0) atomicExch(a.error_flag, 1);
            return g;
        }
        base += all * units;
        ++b;
    }
}

// ------------------------------------------------------------------------------------- publishing
// Scratch: kMaxCtas arrival counters (zero between launches: the last to arrive resets its counter), then two slots a CTA of
// rows * (D + 2) floats: O [rows][D], max [rows], sum [rows].
__device__ __forceinline__ float* slot_of(const skv_pool_attention_args& a, int cta, int slot, int rows) {
    return reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kMaxCtas * 4) +
           ((int64_t)2 * cta + slot) * rows * (a.pool.head_dim + 2);
}

// Called by all threads once the CTA's part is in its slot; true for the CTA that joins.  The barrier puts
// every thread's stores before thread 0's fence, which puts them before its arrival.
__device__ __forceinline__ bool arrive(const skv_pool_attention_args& a, const Share& s, const Segment& g) {
    __shared__ int s_last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const int c0 = s.owner_of(g.first), c1 = s.owner_of(g.last);
        int* count = reinterpret_cast<int*>(a.scratch) + c0;
        s_last = atomicAdd(count, 1) == c1 - c0;
        if (s_last) *count = 0;
        __threadfence();
    }
    __syncthreads();
    return s_last;
}

// Where query row r of a unit lives (r counts head-major: H_q / heads heads of S_q tokens).
template <class T>
__device__ __forceinline__ T* row_ptr(const skv_rows& x, int S_q, int rep, int b, int hk, int r) {
    return static_cast<T*>(x.ptr) + b * x.stride_b + (int64_t)(hk * rep + r / S_q) * x.stride_h + (r % S_q) * x.stride_s;
}

// Values d .. d + VEC - 1 of output row r of a unit, rounded to the output's type (VEC 4: aligned rows).
template <int VEC>
__device__ __forceinline__ void store_out(const skv_pool_attention_args& a, int b, int hk, int r, int d, const float (&x)[VEC]) {
    const int rep = a.q.heads / a.pool.heads;
    if (a.out.dtype == kF32) {
        float* p = row_ptr<float>(a.out, a.S_q, rep, b, hk, r) + d;
        if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else p[0] = x[0];
    } else if (a.out.dtype == kF16) {
        __half* p = row_ptr<__half>(a.out, a.S_q, rep, b, hk, r) + d;
        if constexpr (VEC == 4) {
            const __half2 u = __floats2half2_rn(x[0], x[1]), v = __floats2half2_rn(x[2], x[3]);
            *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
        } else {
            p[0] = __float2half_rn(x[0]);
        }
    } else {
        __nv_bfloat16* p = row_ptr<__nv_bfloat16>(a.out, a.S_q, rep, b, hk, r) + d;
        if constexpr (VEC == 4) {
            const __nv_bfloat162 u = __floats2bfloat162_rn(x[0], x[1]), v = __floats2bfloat162_rn(x[2], x[3]);
            *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
        } else {
            p[0] = __float2bfloat16_rn(x[0]);
        }
    }
}

__device__ __forceinline__ void store_row(const skv_pool_attention_args& a, const Segment& g, int r, int d, bool vec, const float (&y)[4]) {
    if (vec) {
        store_out<4>(a, g.b, g.hk, r, d, y);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float one[1] = {y[k]};
            store_out<1>(a, g.b, g.hk, r, d + k, one);
        }
    }
}

template <int VEC>
__device__ __forceinline__ void load_part(const float* p, float (&x)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        x[0] = __ldcg(p);
    }
}

// Joins the parts of a unit in token order.  A joining CTA's time is latency, one L2 round trip after the
// other, so loads are issued in batches of 16 a thread: first the maxima and sums of all parts (THREADS / ROWS
// threads a row), which leave the parts' factors in shared memory, then the values, VEC to a load.  Where
// the rows have fewer loads than the block has threads, `ways` threads take every ways-th part of a value, and
// their sums are added in order.  r0, rows: the unit's query rows.  buf: join_floats of shared memory.
constexpr int kJoinWays = 8;
template <int ROWS, int THREADS, int PARTS>
__host__ __device__ constexpr int join_floats() { return (PARTS * ROWS > THREADS * 4 ? PARTS * ROWS : THREADS * 4) + 2 * ROWS; }

template <int ROWS, int THREADS, int VEC, int PARTS>
__device__ __forceinline__ void join(const skv_pool_attention_args& a, const Share& s, const Segment& g, int r0, int rows, float* buf, bool out_vec = false) {
    const int D = a.pool.head_dim, tid = threadIdx.x, items = rows * D / VEC;
    const int c0 = s.owner_of(g.first), parts = s.owner_of(g.last) - c0 + 1;
    // part i lies at base + i * stride, the first one in its CTA's second slot unless it starts that CTA's share
    const int64_t stride = (int64_t)2 * ROWS * (D + 2);
    const float* base = slot_of(a, c0, 0, ROWS);
    const float* part0 = slot_of(a, c0, g.first == s.first_of(c0) ? 0 : 1, ROWS);
    auto part = [&](int i) { return i == 0 ? part0 : base + i * stride; };
    float* s_m = buf;                  // [ROWS] max over all parts (0 if there is none)
    float* s_l = s_m + ROWS;           // [ROWS] sum over all parts
    float* s_f = s_l + ROWS;           // [PARTS][ROWS] 2^(m_i - m) of a block of parts
    float* s_add = s_f;                // [THREADS][VEC] once the factors are used
    __syncthreads();
    {
        constexpr int TPR = THREADS / ROWS;   // a power of two, at most 32
        const int j = tid / TPR, sub = tid % TPR;
        float m = -INFINITY, l = 0.0f;
        for (int i0 = sub; i0 < parts; i0 += 8 * TPR) {
            float mi[8], li[8], top = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = i0 + k * TPR;
                const float* p = part(min(i, parts - 1)) + ROWS * D + min(j, rows - 1);
                mi[k] = i < parts ? __ldcg(p) : -INFINITY;
                li[k] = i < parts ? __ldcg(p + ROWS) : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                top = fmaxf(top, mi[k]);
                if (i0 + k * TPR < min(parts, PARTS)) s_f[(i0 + k * TPR) * ROWS + j] = mi[k];
            }
            const float r = top == -INFINITY ? 0.0f : top;
            l *= exp2f(m - r);
#pragma unroll
            for (int k = 0; k < 8; ++k) l += li[k] * exp2f(mi[k] - r);
            m = top;
        }
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
            const float top = fmaxf(m, m2), r = top == -INFINITY ? 0.0f : top;
            l = l * exp2f(m - r) + l2 * exp2f(m2 - r);
            m = top;
        }
        const float r = m == -INFINITY ? 0.0f : m;
        for (int i = sub; i < min(parts, PARTS); i += TPR) s_f[i * ROWS + j] = exp2f(s_f[i * ROWS + j] - r);
        if (sub == 0) {
            s_m[j] = r;
            s_l[j] = l;
        }
    }
    __syncthreads();
    const int ways = items >= THREADS ? 1 : min(THREADS / items, kJoinWays), wide = THREADS / ways;
    const int way = tid / wide;
    constexpr int I = ROWS >= 16 ? 4 : 2;   // values of a thread at a time
    for (int v0 = 0; v0 < items; v0 += I * wide) {
        float y[I][VEC];
        int v[I], row[I];
#pragma unroll
        for (int n = 0; n < I; ++n) {
            v[n] = v0 + n * wide + tid - way * wide;
            row[n] = v[n] < items ? v[n] * VEC / D : 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[n][e] = 0.0f;
        }
        for (int i0 = 0; i0 < parts; i0 += PARTS) {
            const int count = min(PARTS, parts - i0);
            if (parts > PARTS) {   // more parts than factors fit: block by block
                __syncthreads();
                for (int i = tid; i < count * rows; i += THREADS) {
                    const int k = i / rows, r = i - k * rows;
                    s_f[k * ROWS + r] = exp2f(__ldcg(part(i0 + k) + ROWS * D + r) - s_m[r]);
                }
                __syncthreads();
            }
            if (way >= ways) continue;
            for (int k0 = way; k0 < count; k0 += 16 / I * ways) {
                float x[16 / I][I][VEC];
#pragma unroll
                for (int u = 0; u < 16 / I; ++u)
#pragma unroll
                    for (int n = 0; n < I; ++n) {
                        const int k = k0 + u * ways;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) x[u][n][e] = 0.0f;
                        if (k < count && v[n] < items) load_part<VEC>(part(i0 + k) + v[n] * VEC, x[u][n]);
                    }
#pragma unroll
                for (int u = 0; u < 16 / I; ++u)
#pragma unroll
                    for (int n = 0; n < I; ++n) {
                        const int k = k0 + u * ways;
                        const float f = k < count ? s_f[k * ROWS + row[n]] : 0.0f;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) y[n][e] = fmaf(x[u][n][e], f, y[n][e]);
                    }
            }
        }
        if (ways > 1) {   // items < THREADS: one value a thread, n = 0
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) s_add[tid * VEC + e] = y[0][e];
            __syncthreads();
            if (way == 0)
                for (int w = 1; w < ways; ++w)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[0][e] += s_add[(w * wide + tid) * VEC + e];
        }
        if (way == 0) {
#pragma unroll
            for (int n = 0; n < I; ++n)
                if (v[n] < items && (ways == 1 || n == 0)) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[n][e] = s_l[row[n]] == 0.0f ? 0.0f : y[n][e] / s_l[row[n]];
                    if constexpr (VEC == 4) store_row(a, g, r0 + row[n], v[n] * VEC - row[n] * D, out_vec, y[n]);
                    else store_out<1>(a, g.b, g.hk, r0 + row[n], v[n] - row[n] * D, y[n]);
                }
        }
    }
    __syncthreads();
}

// ------------------------------------------------------------------------ values that are not finite
// A weight of zero does not hide an infinite or NaN value: 0 x inf is NaN.  Under a causal limit a tile has tokens that only
// some of a unit's rows see, so from the first such tile on (not_all_from: a multiple of the tile) the kernels put zeros for
// values that are not finite, remember that they did, and add them at the unit's end to the rows that see them.  A weight is
// positive, so what a value that is not finite contributes is that value.
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ int not_all_from(int see_least, int tokens, int tile) { return see_least < tokens ? see_least / tile * tile : 0x7fffffff; }
// Bits that are set if one of two fp16 values is not finite (its exponent's bits are all ones: one more carries out of them).
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t odd_halves(uint4 w) { return odd_halves(w.x) | odd_halves(w.y) | odd_halves(w.z) | odd_halves(w.w); }
// The two values, zero for those.
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
    const uint32_t odd = odd_halves(w);
    return w & ~((odd & 0x8000u ? 0xffffu : 0u) | (odd >> 16 ? 0xffff0000u : 0u));
}
__device__ __forceinline__ uint4 finite_halves(uint4 w) {
    return make_uint4(finite_halves(w.x), finite_halves(w.y), finite_halves(w.z), finite_halves(w.w));
}

// Adds what is not finite among the values of tokens [from, to) to rows r0 .. r0 + rows - 1 of a unit, in its part or, where that is
// null, in the output.  Rare, so it reads the pages again; thread tid of `threads`, which has every threads-th value of a row,
// between barriers of them.
template <int PREC, bool FRESH = false>
__device__ __noinline__ void add_not_finite(const skv_pool_attention_args& a, int b, int hk, int tokens, int r0, int rows, int from, int to,
                                            float* part, int tid, int threads) {
    const int D = a.pool.head_dim, rep = a.q.heads / a.pool.heads;
    for (int d = tid; d < D; d += threads) {
        const int block = PREC == 3 ? d / a.pool.int4_group : 0;
#pragma unroll 4
        for (int t = from; t < to; ++t) {
            const int64_t row = pool_row<FRESH>(a.pool, b, t);
            const float v = row < 0 ? 0.0f : pool_value<PREC, FRESH>(a.pool, true, row + (int64_t)hk * a.pool.page_size, d, block);
            if (finite(v)) continue;
            for (int j = 0; j < rows; ++j) {
                const int r = r0 + j;
                if (t >= seen_by(a, b, tokens, r % a.S_q)) continue;
                if (part) {
                    part[j * D + d] += v;
                } else {
                    const float x = a.out.dtype == kF32   ? row_ptr<float>(a.out, a.S_q, rep, b, hk, r)[d]
                                    : a.out.dtype == kF16 ? to_float(row_ptr<__half>(a.out, a.S_q, rep, b, hk, r)[d])
                                                          : to_float(row_ptr<__nv_bfloat16>(a.out, a.S_q, rep, b, hk, r)[d]);
                    const float one[1] = {x + v};
                    store_out<1>(a, b, hk, r, d, one);
                }
            }
        }
    }
}

// How many sequences a launch takes at most, so that tile numbers hold their tiles (the lengths are on the device, so the tables'
// width counts): row_tiles a key head, `tile` tokens each, `pad` on top of a unit.  0, with the failure recorded: not even one.
inline int64_t sequences_a_launch(const skv_pool_attention_args& a, int64_t row_tiles, int tile, int pad) {
    constexpr int64_t most = 1 << 30;   // half of 31 bits: sums on the way stay below them too
    const int64_t tiles = (token_cap(a) + tile - 1) / tile, units = row_tiles * a.pool.heads, each = (tiles > 1 ? tiles : 1) + pad;
    if (units <= most / each) return most / (units * each);
    fail(SKV_ERR_TOO_LARGE, "pool_attention: %lld units of up to %lld tiles of %d tokens in one sequence", (long long)units, (long long)each, tile);
    return 0;
}

// Launches the call, `step` sequences at a time.
template <class Launch>
int by_sequences(const skv_pool_attention_args& a, int64_t step, Launch launch) {
    for (int64_t b = 0; b < a.pool.batch; b += step) {
        skv_pool_attention_args part = a;
        part.pool.batch = (int32_t)(a.pool.batch - b < step ? a.pool.batch - b : step);
        part.pool.block_table += b * a.pool.table_stride;
        part.q.ptr = static_cast<char*>(a.q.ptr) + b * a.q.stride_b * dtype_bytes(a.q.dtype);
        part.out.ptr = static_cast<char*>(a.out.ptr) + b * a.out.stride_b * dtype_bytes(a.out.dtype);
        part.lengths += b;
        if (part.new_lengths) part.new_lengths += b;
        const int rc = launch(part);
        if (rc != SKV_OK) return rc;
    }
    return SKV_OK;
}

}  // namespace skv
