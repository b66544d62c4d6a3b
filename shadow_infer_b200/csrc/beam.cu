// Beam search over the page pool: the best continuations of a search's beams, and the block tables and pages that
// follow them.
//
// Selection.  A continuation's score is  s_r + x_rv - m_r - ln sum_v e^(x_rv - m_r),  m_r the row's largest logit.  Within a row
// scores are ordered as logits are, so one pass over the logits is enough: a block takes a part of a row, 4096 logits at a time,
// adds up its maximum and sum, and keeps the part's `keep` best logits; a second launch, a block a search, joins the
// sums, turns the lists' logits into scores in 64 bits and merges the lists.  Bound by reading the logits.
#include <float.h>

#include "pool.cuh"

namespace skv {

constexpr int kBeamThreads = 256, kBeamValues = 16, kBeamChunk = kBeamThreads * kBeamValues;   // logits a thread, a block at a time
constexpr int kBeamKeep = 128, kBeamMost = 4096;      // most continuations; most beams, and most lists of a search
constexpr int kBeamHeld = 1024;                       // candidates that a block holds before it ranks them

// What a part of a row leaves for the merge; its list follows the headers.
struct BeamPart {
    double sum;     // of e^(x - top), or how many are +inf where top is
    float top;
    int count;      // entries of the list: logits above -inf, best first
};

__host__ __device__ inline int64_t beam_chunks(int V) { return ((int64_t)V + kBeamChunk - 1) / kBeamChunk; }

// Parts of a row: enough blocks to fill the GPU, no less than a chunk each, and no more lists than a merge takes.
inline int beam_parts(int B, int beams, int V) {
    const int64_t rows = (int64_t)B * beams;
    int64_t parts = ((int64_t)sm_count() * 6 + rows - 1) / rows;
    if (parts > beam_chunks(V)) parts = beam_chunks(V);
    if (parts > kBeamMost / beams) parts = kBeamMost / beams;
    return parts < 1 ? 1 : (int)parts;
}

// Whether beam r of search b has continuations of its own, and whether it has but one.
__device__ __forceinline__ bool beam_dead(const skv_beam_args& a, int64_t row) { return !(fabsf(__ldg(a.scores + row)) < INFINITY); }
__device__ __forceinline__ bool beam_done(const skv_beam_args& a, int64_t row) { return a.finished && __ldg(a.finished + row); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// Whether (x, i) comes before (y, j).
__device__ __forceinline__ bool ahead(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

// Entries of the list [0, n) ranked, the best `keep` of them in order at its front; returns how many are left.  Every
// entry counts the entries ahead of it.  All threads call this; barriers before and after.
__device__ __forceinline__ int rank_list(float* value, int* index, int n, int keep, float* value2, int* index2) {
    for (int i = threadIdx.x; i < n; i += kBeamThreads) {
        const float x = value[i];
        const int at = index[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += ahead(value[j], index[j], x, at);
        if (rank < keep) { value2[rank] = x; index2[rank] = at; }
    }
    __syncthreads();
    n = min(n, keep);
    for (int i = threadIdx.x; i < n; i += kBeamThreads) { value[i] = value2[i]; index[i] = index2[i]; }
    __syncthreads();
    return n;
}

template <class T>
__global__ void __launch_bounds__(kBeamThreads) beam_parts_kernel(const __grid_constant__ skv_beam_args a, int parts) {
    constexpr int PER = 16 / (int)sizeof(T), LOADS = kBeamValues / PER;
    __shared__ float s_value[kBeamHeld], s_value2[kBeamKeep];
    __shared__ int s_index[kBeamHeld], s_index2[kBeamKeep];
    __shared__ float s_low[kBeamThreads / 32], s_top[kBeamThreads / 32];
    __shared__ double s_sum[kBeamThreads / 32];
    __shared__ int s_count[3], s_held;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, keep = a.keep;
    const int64_t row = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    if (beam_dead(a, row) || beam_done(a, row)) return;   // the merge does not look at their lists
    const T* x0 = static_cast<const T*>(a.logits) + row / a.beams * a.stride_b + row % a.beams * a.stride_r;
    // 16-byte pieces on their boundaries: piece i holds logits i * PER - shift and on, the first and the last piece not all of theirs
    const int shift = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const int64_t pieces = ((int64_t)a.V + shift + PER - 1) / PER, chunk_pieces = kBeamThreads * LOADS;
    const int64_t chunks = (pieces + chunk_pieces - 1) / chunk_pieces;
    const int64_t c0 = chunks * part / parts, c1 = chunks * (part + 1) / parts;
    int groups = kBeamThreads / 32;                       // threads in groups, at least `keep` of them
    while (groups < keep) groups *= 2;
    const int members = kBeamThreads / groups;
    float top = -INFINITY, sum = 0.0f, low = -INFINITY;   // low: candidates are at least this
    int held = 0, rounds = 0;
    bool full = false;                                    // the list has `keep` entries
    if (tid < 3) s_count[tid] = 0;
    if (tid == 0) s_held = 0;
    __syncthreads();
    // How many of the block's predicates hold, summed over the threads.
    auto total_of = [&](int n) {
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0 && n) atomicAdd(&s_count[rounds % 3], n);
        if (tid == 0) s_count[(rounds + 1) % 3] = 0;
        __syncthreads();
        return s_count[rounds++ % 3];
    };
    for (int64_t chunk = c0; chunk < c1; ++chunk) {
        float x[kBeamValues];
        const int64_t piece0 = chunk * chunk_pieces + tid;
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const int64_t first = (piece0 + (int64_t)l * kBeamThreads) * PER - shift;
            if (first >= 0 && first + PER <= a.V) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x0 + first));
                const T* y = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int i = 0; i < PER; ++i) x[l * PER + i] = fmaxf(to_float(y[i]), -INFINITY);   // (a NaN becomes -inf)
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    x[l * PER + i] = first + i >= 0 && first + i < a.V ? fmaxf(to_float(x0[first + i]), -INFINITY) : -INFINITY;
            }
        }
        float most = x[0];
#pragma unroll
        for (int i = 1; i < kBeamValues; ++i) most = fmaxf(most, x[i]);
        if (most > top) {
            sum *= exp2_fast((top - most) * kLog2e);      // (of -inf: 0)
            top = most;
        }
        if (top == INFINITY) {
            if (most == INFINITY)
#pragma unroll
                for (int i = 0; i < kBeamValues; ++i) sum += x[i] == INFINITY ? 1.0f : 0.0f;
        } else {
            const float from = top == -INFINITY ? 0.0f : top;
            float more = 0.0f;
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i) more += exp2_fast((x[i] - from) * kLog2e);
            sum += more;
        }
        if (!full) {
            // the best of each group of threads are `keep` different logits: what is below all of them is not among the best
            float best = most;
            for (int o = 1; o < members; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
            if (lane == 0) s_low[warp] = best;
            __syncthreads();
            best = s_low[0];
            for (int w = 1; w < kBeamThreads / 32; ++w) best = fminf(best, s_low[w]);
            low = fmaxf(best, -FLT_MAX);                  // -inf is no candidate
        }
        int n = 0;
#pragma unroll
        for (int i = 0; i < kBeamValues; ++i) n += x[i] >= low;
        const int total = total_of(n);
        float cut = low;                                  // candidates are above `cut`, or equal to it with a piece up to last
        int64_t last = INT64_MAX;
        if (held + total > kBeamHeld) {
            // more than the list holds (many equal logits): the keep-th largest by halving the range of their images, then the
            // place up to which those equal to it are taken
            uint32_t at = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t y = at | 1u << bit;
                int m = 0;
#pragma unroll
                for (int i = 0; i < kBeamValues; ++i) m += x[i] >= low && score_bits(x[i]) >= y;
                if (total_of(m) >= keep) at = y;
            }
            cut = __uint_as_float(at & 0x80000000u ? at ^ 0x80000000u : ~at);
            int m = 0;
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i) m += x[i] > cut;
            const int ties = keep - total_of(m);
            // places in the chunk run over 4096 numbers
            int end = 0;                                  // the largest number below which there are at most `ties`
            for (int bit = 12; bit >= 0; --bit) {
                const int y = end | 1 << bit;
                m = 0;
#pragma unroll
                for (int i = 0; i < kBeamValues; ++i) m += x[i] == cut && (tid + i / PER * kBeamThreads) * PER + i % PER < y;
                if (total_of(m) <= ties) end = y;
            }
            last = end;
            n = 0;
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i)
                n += x[i] > cut || (x[i] == cut && (tid + i / PER * kBeamThreads) * PER + i % PER < last);
        }
        if (__any_sync(0xffffffffu, n)) {
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            int at = lane == 31 ? atomicAdd(&s_held, incl) : 0;
            at = __shfl_sync(0xffffffffu, at, 31) + incl - n;
#pragma unroll
            for (int i = 0; i < kBeamValues; ++i)
                if (x[i] > cut || (x[i] == cut && (tid + i / PER * kBeamThreads) * PER + i % PER < last)) {
                    s_value[at] = x[i];
                    s_index[at++] = (int)((piece0 + i / PER * kBeamThreads) * PER + i % PER - shift);
                }
        }
        __syncthreads();
        held = s_held;
        if (held > 2 * keep + 64 || (!full && held >= keep) || (chunk + 1 == c1 && held > 0)) {
            held = rank_list(s_value, s_index, held, keep, s_value2, s_index2);
            full = held == keep;
            if (full) {
                // a later logit has to be larger than the last of the list
                const float v = s_value[keep - 1];
                low = v == INFINITY ? NAN : v == 0.0f ? FLT_TRUE_MIN : __int_as_float(__float_as_int(v) + (v > 0.0f ? 1 : -1));
            }
            if (tid == 0) s_held = held;
            __syncthreads();
        }
    }
    // the part's sum, relative to its largest logit
    float most = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) s_top[warp] = most;
    __syncthreads();
    for (int w = 0; w < kBeamThreads / 32; ++w) most = fmaxf(most, s_top[w]);
    double whole = top == most ? (double)sum : most == INFINITY || top == -INFINITY ? 0.0 : (double)sum * exp2((double)(top - most) * 1.4426950408889634);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, o);
    if (lane == 0) s_sum[warp] = whole;
    __syncthreads();
    const int64_t list = blockIdx.x, lists = (int64_t)a.B * a.beams * parts;
    if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < kBeamThreads / 32; ++w) s += s_sum[w];
        static_cast<BeamPart*>(a.scratch)[list] = BeamPart{s, most, held};
    }
    float2* out = reinterpret_cast<float2*>(static_cast<BeamPart*>(a.scratch) + lists) + list * keep;
    for (int i = tid; i < held; i += kBeamThreads) out[i] = make_float2(s_value[i], __int_as_float(s_index[i]));
}

// ------------------------------------------------------------------------------------------ the merge
struct BeamBest {
    double score;
    uint64_t place;    // beam * 2^32 + token; the largest number for none
    int list;
    __device__ __forceinline__ bool before(const BeamBest& o) const { return score > o.score || (score == o.score && place < o.place); }
};

// A block a search.  Each list's front is in shared memory; `keep` times the best of the fronts is taken.
template <class T>
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const __grid_constant__ skv_beam_args a, int parts, bool staged) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    __shared__ BeamBest s_best[2][kBeamThreads / 32];
    __shared__ int s_part[2][kBeamThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, keep = a.keep, beams = a.beams, lists = beams * parts;
    const int64_t row0 = (int64_t)blockIdx.x * beams;
    double* s_front = reinterpret_cast<double*>(s_raw);             // [lists] score of each list's front
    double* s_from = s_front + lists;                               // [beams] what a logit less the largest is added to
    int* s_token = reinterpret_cast<int*>(s_from + beams);          // [lists] token of the front
    float* s_most = reinterpret_cast<float*>(s_token + lists);      // [beams] the largest logit
    int* s_at = reinterpret_cast<int*>(s_most + beams);             // [lists] places of the fronts
    int* s_count = s_at + lists;                                    // [lists]
    float2* s_list = reinterpret_cast<float2*>(reinterpret_cast<uintptr_t>(s_count + lists + 1) & ~(uintptr_t)7);   // staged: [lists][keep]
    const BeamPart* part = static_cast<const BeamPart*>(a.scratch) + row0 * parts;
    const float2* entries = reinterpret_cast<const float2*>(static_cast<const BeamPart*>(a.scratch) + (int64_t)a.B * lists) +
                            row0 * parts * keep;
    if (staged)
        for (int i = tid; i < lists * keep; i += kBeamThreads) s_list[i] = entries[i];
    for (int r = tid; r < beams; r += kBeamThreads) {
        const double cum = __ldg(a.scores + row0 + r);
        if (beam_dead(a, row0 + r) || beam_done(a, row0 + r)) {
            s_from[r] = cum;
            s_most[r] = -INFINITY;
            continue;
        }
        float most = -INFINITY;
        for (int p = 0; p < parts; ++p) most = fmaxf(most, part[r * parts + p].top);
        double sum = 0.0;
        for (int p = 0; p < parts; ++p) {
            const BeamPart& y = part[r * parts + p];
            if (y.top == most) sum += y.sum;
            else if (most < INFINITY && y.top > -INFINITY) sum += y.sum * exp((double)y.top - (double)most);
        }
        s_from[r] = cum - log(sum);                                 // (without a logit above -inf: not used)
        s_most[r] = most;
    }
    __syncthreads();
    auto score_of = [&](int r, float x) {
        return x == s_most[r] ? s_from[r] : s_most[r] == INFINITY ? -(double)INFINITY : s_from[r] + ((double)x - (double)s_most[r]);
    };
    auto place_front = [&](int l) {
        const int at = s_at[l];
        if (at >= s_count[l]) { s_front[l] = -(double)INFINITY; return; }
        const float2 e = staged ? s_list[(int64_t)l * keep + at] : entries[(int64_t)l * keep + at];
        s_front[l] = score_of(l / parts, e.x);
        s_token[l] = __float_as_int(e.y);
    };
    for (int l = tid; l < lists; l += kBeamThreads) {
        const int r = l / parts;
        s_at[l] = 0;
        if (beam_dead(a, row0 + r)) {
            s_count[l] = 0;
            s_front[l] = -(double)INFINITY;
        } else if (beam_done(a, row0 + r)) {                        // the one continuation, no list behind it
            s_count[l] = 0;
            s_front[l] = l % parts == 0 ? s_from[r] : -(double)INFINITY;
            s_token[l] = a.pad_token;
        } else {
            s_count[l] = part[l].count;
            place_front(l);
        }
    }
    int found = 0;
    for (; found < keep; ++found) {
        BeamBest best{-(double)INFINITY, ~0ull, -1};
        for (int l = tid; l < lists; l += kBeamThreads) {           // (each thread reads and advances its own lists only)
            const BeamBest y{s_front[l], (uint64_t)(l / parts) << 32 | (uint32_t)s_token[l], l};
            if (y.score > -(double)INFINITY && y.before(best)) best = y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const BeamBest y{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.place, o),
                             __shfl_xor_sync(0xffffffffu, best.list, o)};
            if (y.before(best)) best = y;
        }
        if (lane == 0) s_best[found & 1][warp] = best;
        __syncthreads();
        best = s_best[found & 1][0];
        for (int w = 1; w < kBeamThreads / 32; ++w)
            if (s_best[found & 1][w].before(best)) best = s_best[found & 1][w];
        if (best.list < 0) break;
        if (tid == 0) {
            const int64_t to = (int64_t)blockIdx.x * keep + found;
            a.values[to] = (float)best.score;
            a.parents[to] = (int64_t)(best.place >> 32);
            a.tokens[to] = (int64_t)(best.place & 0xffffffffu);
        }
        if (best.list % kBeamThreads == tid) {
            ++s_at[best.list];
            place_front(best.list);
        }
    }
    // too few: continuations of -inf, from the first on
    for (int64_t i0 = 0, round = 0; found < keep; i0 += kBeamThreads, ++round) {
        const int64_t i = i0 + tid;
        bool none = false;
        int64_t r = 0, t = 0;
        if (i < (int64_t)beams * a.V) {
            r = i / a.V;
            t = i - r * a.V;
            if (beam_dead(a, row0 + r)) none = true;
            else if (beam_done(a, row0 + r)) none = t != a.pad_token;
            else {
                const float x = to_float(static_cast<const T*>(a.logits)[blockIdx.x * a.stride_b + r * a.stride_r + t]);
                none = !(x > -INFINITY) || (s_most[r] == INFINITY && x < INFINITY);
            }
        }
        const unsigned these = __ballot_sync(0xffffffffu, none);
        if (lane == 0) s_part[round & 1][warp] = __popc(these);
        __syncthreads();
        int before = 0, total = 0;
        for (int w = 0; w < kBeamThreads / 32; ++w) {
            if (w < warp) before += s_part[round & 1][w];
            total += s_part[round & 1][w];
        }
        const int to = found + before + __popc(these & ((1u << lane) - 1));
        if (none && to < keep) {
            a.values[(int64_t)blockIdx.x * keep + to] = -INFINITY;
            a.parents[(int64_t)blockIdx.x * keep + to] = r;
            a.tokens[(int64_t)blockIdx.x * keep + to] = t;
        }
        found += total;
        if (i0 >= (int64_t)beams * a.V) break;
    }
}

template <class T>
int launch_beam(const skv_beam_args& a, cudaStream_t st) {
    const int parts = beam_parts(a.B, a.beams, a.V), lists = a.beams * parts;
    beam_parts_kernel<T><<<(unsigned)((int64_t)a.B * lists), kBeamThreads, 0, st>>>(a, parts);
    if (const int rc = check_launch("beam_select")) return rc;
    size_t smem = (size_t)lists * 20 + (size_t)a.beams * 12 + 16;
    const size_t with = smem + (size_t)lists * a.keep * 8;
    const bool staged = with <= 96 * 1024;
    if (staged) smem = with;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(beam_merge_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 140 * 1024);
        if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "beam_select: %s", cudaGetErrorString(e));
    }
    beam_merge_kernel<T><<<a.B, kBeamThreads, smem, st>>>(a, parts, staged);
    return check_launch("beam_select");
}

// ------------------------------------------------------------------------------------------ reordering
constexpr int kReorderThreads = 256, kReorderBeams = 1024;

// A block a (beam, key head, K or V).  Every block finds out by itself where its beam comes from: a beam is the keeper of its
// parent's last page if it is the parent, or the first child of a parent that does not go on from itself; the n-th beam that
// is no keeper takes the last page of the n-th beam without children.  Pages are copied from keepers' parents, which have
// children, to pages of beams that have none, so no block reads what another writes; the old table is only read.
__global__ void __launch_bounds__(kReorderThreads) pool_reorder_kernel(const __grid_constant__ skv_pool_reorder_args a) {
    __shared__ int s_parent[kReorderBeams];
    __shared__ bool s_extra[kReorderBeams], s_childless[kReorderBeams];
    __shared__ int s_donor;
    const int tid = threadIdx.x, lane = tid & 31, R = a.beams, P = a.pool.page_size, width = a.pool.table_width;
    const int64_t row = blockIdx.x, row0 = row / R * R;
    const int c = (int)(row - row0);
    for (int r = tid; r < R; r += kReorderThreads) {
        const int64_t p = a.parents_bytes == 8 ? __ldg(static_cast<const long long*>(a.parents) + row0 + r)
                                               : (long long)__ldg(static_cast<const int32_t*>(a.parents) + row0 + r);
        s_parent[r] = p >= 0 && p < R ? (int)p : -1;
    }
    __syncthreads();
    const int p = s_parent[c];
    const int64_t tokens = p < 0 ? 0 : max(0, __ldg(a.lengths + row0 + p)), j = tokens / P;
    const int rows = j < width ? (int)(tokens - j * P) : 0;      // of the last page, if it is partly filled
    const int32_t* old = a.pool.block_table + (row0 + max(p, 0)) * a.pool.table_stride;
    bool copy = rows > 0 && p != c;
    if (copy) {                                                  // an own page is needed, unless this is the first child of a parent that ends
        if (s_parent[p] != p) {
            int before = 0;
            for (int r = tid; r < c; r += kReorderThreads) before |= s_parent[r] == p;
            copy = __syncthreads_or(before);
        }
    }
    int target = -1;
    if (copy) {                                                  // (the same for the whole block)
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
        if (tid == 0) s_donor = -1;
        __syncthreads();
        if (tid < 32) {
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
        const int source = __ldg(old + j);
        if (s_donor >= 0) target = __ldg(a.pool.block_table + (row0 + s_donor) * a.pool.table_stride + j);
        if (target < 0 || target >= a.pool.num_pages || source < 0 || source >= a.pool.num_pages || source == target) {
            target = -1;
            if (a.error_flag && tid == 0) atomicExch(a.error_flag, 1);
        } else {
            const int head = blockIdx.y >> 1;
            const bool is_v = blockIdx.y & 1;
            const int64_t from = ((int64_t)source * a.pool.heads + head) * P, to = ((int64_t)target * a.pool.heads + head) * P;
            const int64_t bytes = pool_row_bytes(a.pool.precision, a.pool.head_dim);
            auto move = [&](char* base, int64_t row_bytes, int n) {   // n rows of row_bytes
                char* d = base + to * row_bytes;
                const char* s = base + from * row_bytes;
                const int64_t all = n * row_bytes;
                const uintptr_t odd = reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(s) | (uintptr_t)all;
                if ((odd & 15) == 0) {
                    for (int64_t i = tid; i < all / 16; i += kReorderThreads)
                        reinterpret_cast<uint4*>(d)[i] = reinterpret_cast<const uint4*>(s)[i];
                } else if ((odd & 3) == 0) {
                    for (int64_t i = tid; i < all / 4; i += kReorderThreads)
                        reinterpret_cast<uint32_t*>(d)[i] = reinterpret_cast<const uint32_t*>(s)[i];
                } else {
                    for (int64_t i = tid; i < all; i += kReorderThreads) d[i] = s[i];
                }
            };
            move(static_cast<char*>(is_v ? a.pool.v : a.pool.k), bytes, rows);
            if (a.pool.precision >= 2)
                move(reinterpret_cast<char*>(is_v ? a.pool.scale_v : a.pool.scale_k),
                     a.pool.precision == 2 ? 4 : 4ll * (a.pool.head_dim / a.pool.int4_group), rows);
            if (a.bounds && !is_v) {
                const int64_t d = (int64_t)target * a.pool.heads + head, s = (int64_t)source * a.pool.heads + head;
                const int64_t n = 2ll * a.pool.head_dim;
                for (int64_t i = tid; i < n; i += kReorderThreads) a.bounds[d * n + i] = a.bounds[s * n + i];
                if (tid == 0) a.steps[d] = a.steps[s];
            }
        }
    }
    if (blockIdx.y) return;
    int32_t* table = a.new_table + row * width;
    const int32_t* own = a.pool.block_table + row * a.pool.table_stride;
    for (int i = tid; i < width; i += kReorderThreads)
        table[i] = p < 0 ? -1 : copy && i == j ? target : __ldg((i < j + (rows > 0) ? old : own) + i);
    if (tid == 0) {
        a.new_lengths[row] = p < 0 ? 0 : __ldg(a.lengths + row0 + p);
        if (a.error_flag && (p < 0 || __ldg(a.lengths + row0 + p) < 0 || tokens > (int64_t)width * P)) atomicExch(a.error_flag, 1);
    }
}

}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_beam_scratch_bytes(int B, int beams, int V, int keep) {
    if (B <= 0 || beams <= 0 || beams > kBeamMost || V <= 0 || keep <= 0) return 0;
    return (size_t)B * beams * beam_parts(B, beams, V) * (sizeof(BeamPart) + (size_t)keep * 8);
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
    if (a.keep > kBeamKeep || a.beams > kBeamMost || a.V > 0x7fffffff - kBeamChunk)
        return fail(SKV_ERR_TOO_LARGE, "beam_select: keep %d (at most %d), %d beams (at most %d), %d tokens", a.keep, kBeamKeep, a.beams,
                    kBeamMost, a.V);
    if (a.B == 0) return SKV_OK;
    if (!a.logits || !a.scores || !a.values || !a.parents || !a.tokens || !a.scratch)
        return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: null pointer");
    if (reinterpret_cast<uintptr_t>(a.scratch) & 15 || reinterpret_cast<uintptr_t>(a.logits) % dtype_bytes(a.dtype))
        return fail(SKV_ERR_INVALID_ARGUMENT, "beam_select: scratch or logits are not aligned");
    const int64_t blocks = (int64_t)a.B * a.beams * beam_parts(a.B, a.beams, a.V);
    if (blocks > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "beam_select: too many rows");
    if (a.scratch_bytes < (int64_t)skv_beam_scratch_bytes(a.B, a.beams, a.V, a.keep))
        return fail(SKV_ERR_SCRATCH, "beam_select: scratch of %lld bytes", (long long)a.scratch_bytes);
    cudaStream_t st = as_stream(stream);
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
    const dim3 grid((unsigned)a.pool.batch, 2 * a.pool.heads);
    pool_reorder_kernel<<<grid, kReorderThreads, 0, as_stream(stream)>>>(a);
    return check_launch("pool_reorder");
}

}  // extern "C"
