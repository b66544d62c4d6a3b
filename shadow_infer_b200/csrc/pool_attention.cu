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
//
// Three kernels: tensor cores for a few query rows a key head (pool_attention_mma.cuh), tcgen05 for many
// (pool_attention_tc.cuh), and the one below for what neither takes: heads above 256 values or of odd sizes, pages that
// are not on 16-byte boundaries.
#include <mutex>

#include "pool_attention.cuh"

namespace skv {

// --------------------------------------------------------------------------- any size and alignment
// Products on the FMA pipe from fp32 tiles in shared memory: 8 rows, 32 tokens at a time (16384 tokens of 8 fp32 key heads of 128
// values in 102 us, bound by the tiles' latency at 1.3 TB/s).  Thread = (token, rows w and
// w + 4) for the scores, value d for the sums.  A warp widens 8 tokens a tile, a lane a value of each, so that 16 loads are on
// their way; the lanes look up the tokens' rows one tile ahead.
constexpr int kAnyRows = 8, kAnyTile = 32, kAnyThreads = 128, kAnyMaxD = 512, kAnyParts = 64, kAnyPad = 1;

__host__ __device__ inline size_t any_smem(int D) {
    return ((size_t)kAnyRows * D + (size_t)kAnyTile * (D + 1) + (size_t)kAnyTile * D + kAnyRows * kAnyTile + kAnyRows +
            join_floats<kAnyRows, kAnyThreads, kAnyParts>()) * 4;
}

template <class T, int PREC>
__global__ void __launch_bounds__(kAnyThreads) pool_attention_any_kernel(const __grid_constant__ skv_pool_attention_args a,
                                                                         int row_tiles) {
    extern __shared__ float any_sm[];
    __shared__ Share s;
    __shared__ int s_see[kAnyRows];   // tokens that each row sees
    const int D = a.pool.head_dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* sq = any_sm;
    float* sk = sq + kAnyRows * D;
    float* sv = sk + kAnyTile * (D + 1);
    float* sp = sv + kAnyTile * D;
    float* sc = sp + kAnyRows * kAnyTile;
    float* sj = sc + kAnyRows;
    const int rep = a.q.heads / a.pool.heads, R = rep * a.S_q;
    take_share<kAnyThreads>(a, kAnyTile, a.pool.heads * row_tiles, kAnyPad, 2, &s);
    int b = s.b, base = s.base;
    for (int at = s.lo; at < s.hi;) {
        const Segment g = segment_at(a, s, at, kAnyTile, row_tiles, b, base);
        at = g.next;
        if (g.t0 >= g.t1) continue;
        const int r0 = g.rt * kAnyRows;
        __syncthreads();
        for (int i = tid; i < kAnyRows * D; i += kAnyThreads) {
            const int r = r0 + i / D;
            sq[i] = r < R ? to_float(row_ptr<const T>(a.q, a.S_q, rep, g.b, g.hk, r)[i % D]) * (a.scale * 1.4426950408889634f)
                          : 0.0f;
        }
        int see[2];   // tokens that each of this warp's two rows sees
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[kAnyRows][kAnyMaxD / kAnyThreads];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            see[i] = seen_by(a, g.b, g.tokens, (r0 + warp + 4 * i) % a.S_q);
        if (lane < 2) s_see[warp + 4 * lane] = lane ? see[1] : see[0];
#pragma unroll
        for (int j = 0; j < kAnyRows; ++j)
#pragma unroll
            for (int i = 0; i < kAnyMaxD / kAnyThreads; ++i) o[j][i] = 0.0f;
        // the pool row of token lane % 8 of this warp's eight, -1 where there is none
        auto row_of = [&](int first) -> int64_t {
            const int t = first + warp * 8 + (lane & 7);
            if (t >= g.tokens) return -1;
            const int64_t r = pool_row(a.pool, g.b, t);
            if (r < 0 && a.error_flag) atomicExch(a.error_flag, 1);
            return r < 0 ? -1 : r + (int64_t)g.hk * a.pool.page_size;
        };
        int64_t next_row = row_of(g.t0 * kAnyTile);
        for (int t = g.t0; t < g.t1; ++t) {
            const int tok0 = t * kAnyTile;
            __syncthreads();
            const int64_t row = next_row;
            if (t + 1 < g.t1) next_row = row_of(tok0 + kAnyTile);
            if (lane < 8) sp[warp * 8 + lane] = row >= 0 ? 1.0f : 0.0f;   // whether there is such a token
            int64_t rows[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) rows[j] = __shfl_sync(0xffffffffu, row, j);
            for (int d = lane; d < D; d += 32) {
                const int block = PREC == 3 ? d / a.pool.int4_group : 0;
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int64_t r = rows[j];
                    x[j] = r >= 0 ? pool_value<PREC>(a.pool, false, r, d, block) : 0.0f;
                    y[j] = r >= 0 ? pool_value<PREC>(a.pool, true, r, d, block) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sk[(warp * 8 + j) * (D + 1) + d] = x[j];
                    sv[(warp * 8 + j) * D + d] = y[j];
                }
            }
            __syncthreads();
            const bool held = sp[lane] != 0.0f;
            int see_least = g.tokens;
            for (int j = 0; j < kAnyRows; ++j)
                if (s_see[j] > 0) see_least = min(see_least, s_see[j]);
            const bool not_all = tok0 >= not_all_from(see_least, g.tokens, kAnyTile);
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
                    if (not_all && !finite(v)) {   // (pool_attention.cuh)
#pragma unroll
                        for (int j = 0; j < kAnyRows; ++j)
                            if (tok0 + k < s_see[j]) o[j][i] += v;
                        continue;
                    }
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
        if (arrive(a, s, g)) join<kAnyRows, kAnyThreads, 1, kAnyParts>(a, s, g, r0, min(kAnyRows, R - r0), sj);
    }
}

template <class T, int PREC>
int launch_any_prec(const skv_pool_attention_args& a, cudaStream_t st) {
    const int R = a.q.heads / a.pool.heads * a.S_q, row_tiles = (R + kAnyRows - 1) / kAnyRows;
    const int64_t step = sequences_a_launch(a, row_tiles, kAnyTile, kAnyPad);
    if (step == 0) return SKV_ERR_TOO_LARGE;
    const size_t smem = any_smem(a.pool.head_dim);
    cudaError_t e = cudaFuncSetAttribute(pool_attention_any_kernel<T, PREC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    int per_sm = 1;
    if (e == cudaSuccess)
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, pool_attention_any_kernel<T, PREC>, kAnyThreads, smem);
    if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
    int grid = sm_count() * (per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm);
    if (grid > kMaxCtas) grid = kMaxCtas;
    return by_sequences(a, step, [&](const skv_pool_attention_args& part) {
        pool_attention_any_kernel<T, PREC><<<grid, kAnyThreads, smem, st>>>(part, row_tiles);
        return check_launch("pool_attention");
    });
}

template <class T>
int launch_any(const skv_pool_attention_args& a, cudaStream_t st) {
    switch (a.pool.precision) {
        case 0: return launch_any_prec<T, 0>(a, st);
        case 1: return launch_any_prec<T, 1>(a, st);
        case 2: return launch_any_prec<T, 2>(a, st);
        default: return launch_any_prec<T, 3>(a, st);
    }
}

// The tensor-core kernels (pool_attention_mma.cuh), one translation unit a precision, of whole sequences and of lists of pages.
int attend_fp32(const skv_pool_attention_args& a, cudaStream_t st);
int attend_fp16(const skv_pool_attention_args& a, cudaStream_t st);
int attend_int8(const skv_pool_attention_args& a, cudaStream_t st);
int attend_int4(const skv_pool_attention_args& a, cudaStream_t st);
int attend_listed_fp32(const skv_pool_attention_args& a, cudaStream_t st);
int attend_listed_fp16(const skv_pool_attention_args& a, cudaStream_t st);
int attend_listed_int8(const skv_pool_attention_args& a, cudaStream_t st);
int attend_listed_int4(const skv_pool_attention_args& a, cudaStream_t st);

// The tcgen05 kernel (pool_attention_tc.cuh), and the query rows a key head from which it is taken.  The lengths are on the device,
// so the rule cannot look at them; it is set by long sequences, and short ones lose a few us by it.  8 key heads of 128
// values, causal, us there / on the small kernel, for fp16, int8 and int4 pages:
//     32 rows over 4 x 4096 tokens   36.3 / 37.6   41.0 / 36.5   46.2 / 40.5      (fp16 queries 38.1 / 38.3   43.5 / 37.5   48.2 / 41.6)
//     48 rows                        37.1 / 41.6   41.6 / 44.6   47.3 / 50.6                   (39.6 / 45.0   44.3 / 46.4   49.4 / 53.4)
//     64 rows                        38.5 / 49.7   42.7 / 52.4   49.6 / 63.0                   (38.4 / 53.3   45.4 / 55.4   50.8 / 66.9)
//     48 rows over 512 tokens        18.0 / 16.8   21.0 / 17.4   20.0 / 18.8                   (19.0 / 17.3   21.9 / 18.2   20.3 / 19.2)
//     128 rows over 512 tokens       21.1 / 18.0   23.2 / 20.4   22.1 / 21.5                   (21.6 / 18.5   24.1 / 20.8   22.6 / 22.0)
// Heads of 256 values (2 query heads), which leave an SM one CTA:
//     48 rows over 4 x 4096 tokens   70.1 / 83.1   84.2 / 64.6   110 / 89                      (74.1 / 91.0   84.4 / 71.4   111 / 96)
//     64 rows                        73.4 / 99.5   86.0 / 78.8   111 / 112                     (77.1 / 109    87.0 / 88.1   110 / 122)
//     128 rows                       88.8 / 174    98.2 / 133    124 / 198                     (92.4 / 197    100 / 149     125 / 216)
constexpr int many_rows(int D) { return D <= 128 ? 48 : 64; }
int attend_many(const skv_pool_attention_args& a, cudaStream_t st);

// They need heads of up to 256 values in rows of whole 16-byte (fp16) or 8-byte chunks, int4 groups of whole 16-value blocks,
// payloads on 16-byte boundaries, a row 0, and row numbers of 31 bits.
bool fits_mma(const skv_pool& p) {
    const int D = p.head_dim;
    const int64_t rows = (int64_t)p.num_pages * p.heads * p.page_size;
    if (rows == 0 || rows > 0x7fffffff || D > 256) return false;
    if (D % (p.precision == 3 ? 16 : 8) || (p.precision == 3 && p.int4_group % 16)) return false;
    return ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0;
}

// The tcgen05 kernel takes 16-bit queries (32-bit ones want sums that the tensor cores do not cut off) over fp16, int8 and int4
// pages, heads of up to 256 values in whole swizzled chunks of 16, int4 rows in whole 16-byte chunks.
bool fits_tc(const skv_pool_attention_args& a) {
    const int D = a.pool.head_dim;
    return a.q.heads / a.pool.heads * (int64_t)a.S_q >= many_rows(D) && a.q.dtype != kF32 && a.pool.precision != 0 && D <= kManyD &&
           D % (a.pool.precision == 3 ? 32 : 16) == 0 && rows_aligned(a.q);
}

}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_pool_attention_scratch_bytes(int D) {
    return D <= 0 ? 0 : (size_t)kMaxCtas * 4 + (size_t)sm_count() * rows_per_sm(D) * (D + 2) * 4;
}

size_t skv_pool_attention_scratch_zeros(void) { return (size_t)kMaxCtas * 4; }

}  // extern "C"

namespace skv {

// What skv_pool_attention refuses, and whether there is nothing to do.
int check_attention(const skv_pool_attention_args& a, bool& nothing) {
    int rc;
    nothing = false;
    if ((rc = check_pool(a.pool, "pool_attention")) || (rc = check_rows(a.q, a.pool.batch > 0 && a.S_q > 0, "pool_attention", "q")) ||
        (rc = check_rows(a.out, a.pool.batch > 0 && a.S_q > 0, "pool_attention", "out")))
        return rc;
    if (a.S_q < 0) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: bad size");
    if (a.q.heads != a.out.heads || a.q.heads % a.pool.heads || a.q.dtype != a.out.dtype)
        return fail(SKV_ERR_SHAPE, "pool_attention: %d query heads, %d outputs, %d key heads", a.q.heads, a.out.heads,
                    a.pool.heads);
    nothing = a.pool.batch == 0 || a.S_q == 0 || a.q.heads == 0;
    if (nothing) return SKV_OK;
    if (!a.lengths || !a.scratch) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: null pointer");
    if (reinterpret_cast<uintptr_t>(a.scratch) & 15) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: scratch is not on a 16-byte boundary");
    if (a.pool.head_dim > kAnyMaxD)
        return fail(SKV_ERR_UNSUPPORTED, "pool_attention: head_dim %d above %d", a.pool.head_dim, kAnyMaxD);
    if ((int64_t)a.q.heads * a.S_q > (1 << 28) || a.pool.batch > (1 << 24))
        return fail(SKV_ERR_TOO_LARGE, "pool_attention: too many rows");
    if (a.scratch_bytes < (int64_t)skv_pool_attention_scratch_bytes(a.pool.head_dim))
        return fail(SKV_ERR_SCRATCH, "pool_attention: scratch of %lld bytes", (long long)a.scratch_bytes);
    return SKV_OK;
}

int attend(const skv_pool_attention_args& a, cudaStream_t st) {
    const bool mma = fits_mma(a.pool), many = mma && fits_tc(a);
    if (a.reserved < 0 && (!mma || many))
        if (const int rc = launch_tables(*static_cast<const AttentionCall&>(a).lists, st)) return rc;
    if (many) return attend_many(a, st);
    if (mma) {
        const bool listed = a.reserved < 0;
        switch (a.pool.precision) {
            case 0: return listed ? attend_listed_fp32(a, st) : attend_fp32(a, st);
            case 1: return listed ? attend_listed_fp16(a, st) : attend_fp16(a, st);
            case 2: return listed ? attend_listed_int8(a, st) : attend_int8(a, st);
            default: return listed ? attend_listed_int4(a, st) : attend_int4(a, st);
        }
    }
    if (a.q.dtype == kF32) return launch_any<float>(a, st);
    if (a.q.dtype == kF16) return launch_any<__half>(a, st);
    return launch_any<__nv_bfloat16>(a, st);
}

// ------------------------------------------------------------------------------- listed pages only
constexpr int kTableWarps = 8;

// A warp a unit.
__global__ void __launch_bounds__(32 * kTableWarps) sparse_tables_kernel(const __grid_constant__ skv_pool_sparse_args s, int units) {
    start_dependents();
    wait_for_dependency();
    const int u = blockIdx.x * kTableWarps + (threadIdx.x >> 5);
    if (u < units) list_table(s, u, units);
}

int launch_tables(const skv_pool_sparse_args& s, cudaStream_t st) {
    const int units = s.attention.pool.batch * s.attention.S_q * s.attention.pool.heads;
    launch_after(sparse_tables_kernel, dim3((unsigned)((units + kTableWarps - 1) / kTableWarps)), 32 * kTableWarps, 0, st, s, units);
    return check_launch("pool_sparse_attention");
}

// Values from one unit's rows to the next one's, units counted (sequence, new token, key head); false where they are not evenly spaced.
bool unit_stride(const skv_rows& r, int B, int S_q, int heads, int64_t& stride) {
    const int rep = r.heads / heads;
    int64_t steps[3] = {r.stride_b, r.stride_s, rep * r.stride_h};
    const int sizes[3] = {B, S_q, heads};
    int64_t inner = 1;
    stride = 0;
    for (int i = 2; i >= 0; --i) {
        if (sizes[i] == 1) continue;
        if (inner == 1) stride = steps[i];
        else if (steps[i] != inner * stride) return false;
        inner *= sizes[i];
    }
    return true;
}

}  // namespace skv

extern "C" {

int skv_pool_attention(const skv_pool_attention_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_attention: null pointer");
    bool nothing;
    skv_pool_attention_args a = *args;
    a.reserved = 0;
    const int rc = check_attention(a, nothing);
    return rc || nothing ? rc : attend(a, as_stream(stream));
}

int skv_pool_sparse_attention(const skv_pool_sparse_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_sparse_attention: null pointer");
    const skv_pool_sparse_args& s = *args;
    AttentionCall a;
    static_cast<skv_pool_attention_args&>(a) = s.attention;
    a.lists = &s;
    bool nothing;
    const int rc = check_attention(a, nothing);
    if (rc || nothing) return rc;
    if (reinterpret_cast<uintptr_t>(s.tables) & 127) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_sparse_attention: tables are not on a 128-byte boundary");
    if (s.keep < 1) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_sparse_attention: %d pages a query", s.keep);
    if (!s.pages || !s.tables) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_sparse_attention: null pointer");
    const int64_t units = (int64_t)a.pool.batch * a.S_q * a.pool.heads;
    if (units > (1 << 24) || (int64_t)a.pool.num_pages * a.pool.heads > 0x7fffffff)
        return fail(SKV_ERR_TOO_LARGE, "pool_sparse_attention: %lld units over %d pages", (long long)units, a.pool.num_pages);
    if (s.tables_bytes < units * (list_stride(s.keep) + 1) * 4)
        return fail(SKV_ERR_SCRATCH, "pool_sparse_attention: tables of %lld bytes", (long long)s.tables_bytes);
    if (!unit_stride(a.q, a.pool.batch, a.S_q, a.pool.heads, a.q.stride_b) ||
        !unit_stride(a.out, a.pool.batch, a.S_q, a.pool.heads, a.out.stride_b))
        return fail(SKV_ERR_UNSUPPORTED, "pool_sparse_attention: rows are not evenly spaced");
    cudaStream_t st = as_stream(stream);
    static std::mutex launches;   // the tables stay with the attention that reads them: host threads may share a stream and its scratch
    const std::lock_guard<std::mutex> together(launches);
    a.q.heads = a.out.heads = a.q.heads / a.pool.heads;
    a.pool.num_pages *= a.pool.heads;
    a.pool.heads = a.S_q = 1;
    a.pool.batch = (int)units;
    a.pool.block_table = static_cast<const int32_t*>(s.tables);
    a.pool.table_stride = list_stride(s.keep);
    a.pool.table_width = s.keep;
    a.lengths = a.pool.block_table + units * list_stride(s.keep);
    a.new_lengths = nullptr;
    a.causal = 0;
    a.reserved = -1;
    return attend(a, st);
}

}  // extern "C"
