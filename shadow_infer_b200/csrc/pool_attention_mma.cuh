// Attention over the page pool on the tensor cores.
//
// A decoding step is bound by the pages' bytes, but at 4 or 8 bits a value the FMA pipe cannot keep up with
// HBM, nor can it where several query rows share a key head.  So both products run as mma.m16n8k16 (fp16 operands, fp32
// sums), transposed so that the few query rows are the narrow side:
//     S^T [16 tokens x 8 rows] = K [16 x D] Q^T,     O^T [16 values x 8 rows] += V^T [16 x 16 tokens] P^T.
// (tcgen05 wants 128 rows of A and brings its sums back through TMEM; below 48 query rows it is the slower one.)
//
// Feeding.  A warp owns every W-th tile of 16 tokens of its CTA's share and a ring of slots in shared memory; it
// copies its next tiles' rows and scales with cp.async while it multiplies this one's, across segments, and waits for no
// other warp.  Slots are swizzled in 16-byte chunks, so the fragments are read without bank conflicts: fp16 by ldmatrix
// (transposed for V), int8 and int4 as words whose integers become fp16 in registers.  The contraction order of an MMA is
// free as long as both operands agree: the queries are laid out, once a segment, in the order the words come in.  P^T's
// operand is S^T's result transposed by movmatrix.  fp32 pages run as m16n8k8 of tf32 terms instead.
//
// What bounds it (8 key heads of 4 query heads, 128 values).  fp16: the pages' bytes, 64 sequences of up to 8192 tokens in 163 us
// = the copy rate.  int8 and int4: the instructions that make operands of the bytes, about 540 and 725 a warp for a tile of 16
// tokens: 131071 int8 tokens with fp32 queries in 76 us (57 % of the copy rate), 32768 int4 tokens of 32 heads in 82 us (38 %).
// fp32: 16 KB a tile leave room for 4 warps an SM, 16384 tokens in 36 us (57 %).  Small calls: 4 to 5 us until the first rows
// are there, 1.7 us a unit and 3 to 6 us for a join; 512 tokens of 32 heads in 12 us, 8 int8 sequences of up to 2048 tokens in 18.
// Lists of pages: a unit's table is made first, 2 to 4 us; 32 units of 2048 int4 tokens in 19 us, 8 of 4096 int8 tokens in 16, of 512 in 11, 512 of 512 int8
// tokens in 26 (from L2; instructions fill 47 % of the issue slots, their waits and the units' barriers the rest), 512 of up to 1024 fp16 tokens in 52 with its tables' launch (256 MB, 5 TB/s).
//
// Exactness.  Page values enter the MMAs exactly: fp16 as it is, int8 and int4 as small integers, fp32 as two terms of 11 bits
// (of the products of small parts only that of both is left out, 2^-24 of a value).  For the scores they stay
// biased, as fp16 subnormals (their bits are the operand), and the sums start at minus the bias times the query's sum;
// the values' sums would cancel too much that way, so V's integers are made signed.  An int8 row's scale multiplies its
// score (K) or its weight (V) in fp32.  An int4 group's scale multiplies the group's own MMA result (K), or is split into
// parts of 7 bits, an MMA each, that times a 4-bit integer are exact in fp16 (V), after a power of two a token is taken out
// into its weight.  Queries are scaled by a power of two a row; 16-bit ones fit one fp16 operand, fp32 ones take two
// (22 bits).  Weights are 2^(z - ref) <= 2^15 with z the score plus the exponent of V's scale; one operand for bf16
// outputs, whose own rounding is 8 times coarser (two cost calls of one token up to 5 %, prompts 4 to 15), else two.  Against 64 bits fp32 outputs are 2e-7 to 5e-7 off.
//
// ref follows the running maximum lazily (sums are rescaled only when a weight would pass 2^15), so most tiles need one
// vote and no shuffles; row sums stay in the lanes until the segment ends.
#pragma once

#include <atomic>

#include "pool_attention.cuh"

namespace skv {

constexpr int kMmaPad = 3, kMinTiles = 2;   // what a unit costs on top of its tiles, and the least that a CTA takes
constexpr int kMmaParts = 64;       // parts whose factors a joining CTA holds at a time
constexpr float kRefDrop = 11.0f;   // a fresh maximum's weight is 2^11: fp16's last step, 2^-25, is then 2^-36 of it
constexpr float kRefRoom = 14.0f;   // weights may grow to 2^14 (times a mantissa < 2) before ref moves

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
// The same with new sums: c = a b + (c0, c1 for every row of A).
__device__ __forceinline__ void mma16816_from(float (&c)[4], const uint32_t (&a)[4], uint2 b, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(c0), "f"(c1));
}
// c += a b of tf32 operands (fp32 bits whose lower 13 do not count), 16 x 8 by 8 x 8.
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
// The first 11 significant bits of x, cut off or rounded.  (Rounding hides a NaN of all ones, which what is left then shows.)
__device__ __forceinline__ uint32_t tf32_cut(float x) { return __float_as_uint(x) & 0xFFFFE000u; }
__device__ __forceinline__ uint32_t tf32_round(float x) { return (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u; }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two columns of an 8 x 8 matrix of 32-bit words, 16 bits at a time: of the result's row, columns 2c and 2c + 1.
__device__ __forceinline__ uint2 transpose8x8(uint32_t x, uint32_t y) {
    const uint32_t lo = transpose8x8(__byte_perm(x, y, 0x5410)), hi = transpose8x8(__byte_perm(x, y, 0x7632));
    return make_uint2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
__device__ __forceinline__ void load_matrix(uint32_t (&f)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrix_trans(uint32_t (&f)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_pack(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Bytes n + 128 as fp16: 1024 + b has b in its low bits; less 1152 it is n.
__device__ __forceinline__ uint32_t i8_pair(uint32_t biased, uint32_t sel) {
    return h2_sub(__byte_perm(biased, 0x64646464u, sel), 0x64806480u);
}
// Nibbles n + 8 in bits 4-7 of each half as 64 + (n + 8).
__device__ __forceinline__ uint32_t i4_pair(uint32_t w) { return (w & 0x00F000F0u) | 0x54005400u; }
// The first 7 significant bits of x, rounded; x becomes what is left.
__device__ __forceinline__ float take7(float& x) {
    const float r = __uint_as_float((__float_as_uint(x) + 0x10000u) & 0xFFFE0000u);
    x -= r;
    return r;
}
// The exponent field of a float, kept where the powers of two below stay normal.
__device__ __forceinline__ int clamp_exp(uint32_t bits) { return min(max((int)(bits >> 23), 35), 219); }
// 2^(127 + to - e) scales a float of exponent field e to [2^to, 2^(to + 1)).
__device__ __forceinline__ float exp_down(int e, int to) { return __uint_as_float((uint32_t)(254 + to - e) << 23); }
__device__ __forceinline__ float exp_up(int e, int to) { return __uint_as_float((uint32_t)(e - to) << 23); }
constexpr int kQueryExp = 10, kValueExp = 8;   // where a query row's and a token's int4 scales' maxima are put

// t / page_size for t < 2^31 as a product: mul = ceil(2^shift / page_size), shift = 31 + ceil(log2 page_size).
struct PageDivide {
    uint32_t mul;
    int shift;
};

// The page rows of a sequence's tokens for one key head.  A warp keeps the next 64 entries of the
// block table in its lanes and asks them by shuffle: tiles need no dependent load.
template <bool FRESH>
struct PageRows {
    const int32_t* table;
    int width, base, cur, next, lane;
    __device__ __forceinline__ int entry(int i) const { return i < width ? number_at<FRESH>(table + i) : -1; }
    __device__ __forceinline__ void start(const skv_pool& p, int b, int first) {
        table = p.block_table + b * p.table_stride;
        width = p.table_width;
        lane = threadIdx.x & 31;
        base = first;
        cur = entry(base + lane);
        next = entry(base + 32 + lane);
    }
    __device__ __forceinline__ int page(int j) {   // j does not decrease
        while (j >= base + 32) {
            base += 32;
            cur = next;
            next = entry(base + 32 + lane);
        }
        return __shfl_sync(0xffffffffu, cur, j - base);
    }
};

// E values of a row of which `left` exist, with one load where rows are aligned to them (their count is a
// multiple of E then, as head sizes here are multiples of 8).
template <int E, class T>
__device__ __forceinline__ void load_row(const T* p, int left, bool vec, float (&x)[E]) {
    if (vec) {
        constexpr int WORDS = E * (int)sizeof(T) / 4;
        uint32_t w[WORDS];
        if constexpr (WORDS >= 4) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (WORDS == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_float(reinterpret_cast<const T*>(w)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < left) x[i] = to_float(p[i]);
    }
}

// Where value d of a query row sits in the B operands (MMA, lane column c, register and half), and what it is
// multiplied by there: the high nibbles of int4 bytes are read as 16 (n + 8) (32-bit queries: both as 64 (n + 8)).
template <int PREC, int DP, int NQ>
__device__ __forceinline__ float query_place(int d, int& mma, int& c, int& reg, int& half) {
    if (PREC == 0) {   // lane column c reads every second chunk of 4 values
        const int chunk = d / 4;
        mma = 2 * (2 * (chunk / 8) + chunk % 2) + d % 4 / 2; c = chunk % 8 / 2; reg = d % 2; half = 0;
        return 1.0f;
    }
    if (PREC == 1) {   // ldmatrix order
        mma = d / 16; c = (d % 8) / 2; reg = (d % 16) / 8; half = d % 2;
        return 1.0f;
    }
    const int r = d % 4;   // of a word's or a byte pair's values: 0 and 2 in one register, 1 and 3 in the other
    reg = r % 2; half = r / 2;
    if (PREC == 2) {       // lane column c reads DP / 64 neighbouring chunks
        const int chunk = d / 16, per = DP / 64;
        mma = 4 * (chunk % per) + (d % 16) / 4; c = chunk / per;
        return 1.0f;
    }
    mma = d / 16; c = (d % 16) / 4;
    return NQ == 2 || r % 2 ? 1.0f : 0.0625f;
}
// An fp16 whose bits are m < 1024 has the value m 2^-24.  The tensor cores align a product by its factors' exponent fields, so
// a small m loses as many of the sum's last bits as it has leading zeros: for 32-bit queries int4 values are moved up to m's top
// (without that the output was 1.2e-6 off, with it 3e-7; an int8 value has 8 of the 10 bits).
template <int PREC, int NQ>
__host__ __device__ constexpr float subnormal_unit() { return PREC == 3 && NQ == 2 ? 3.814697265625e-06f : 5.9604644775390625e-08f; }
template <int PREC, int DP>
__host__ __device__ constexpr int bias_blocks() { return PREC == 3 ? DP / 16 : 1; }

// A slot: 16 rows of K and of V, their scales (int4: one for each 16 values), and the tokens' pool rows.
template <int PREC, int DP>
struct Slot {
    static constexpr int ROW = PREC == 0 ? 4 * DP : PREC == 1 ? 2 * DP : PREC == 2 ? DP : DP / 2, CHUNKS = ROW / 16, BLOCKS = DP / 16;
    static constexpr int SCALES = PREC <= 1 ? 0 : PREC == 2 ? 1 : BLOCKS;   // a token
    static constexpr int K = 0, V = 16 * ROW, SK = 2 * V, SV = SK + 64 * SCALES, ID = SV + 64 * SCALES, USED = ID + 64;
    static constexpr int MERGE = 8 * (DP + 4) * 4;   // the warp's sums of 8 rows pass through a free slot
    static constexpr int BYTES = ((USED > MERGE ? USED : MERGE) + 127) & ~127;   // lines stay on 128-byte boundaries
    // The same for row my_row + i STEP, from the address of row my_row (STEP rows: what a warp copies at a time).
    __device__ static __forceinline__ uint32_t step(uint32_t to, int i, int rows) {
        return (CHUNKS >= 8 ? to ^ (((i * rows) & 7) << 4) : to) + i * rows * ROW;
    }
    // Byte of chunk ch of a row: chunks are exchanged within lines of 128 bytes so that the same chunk of 8 rows, and
    // neighbouring chunks of the rows a fragment takes, fall into different banks.
    __device__ static __forceinline__ int at(int row, int ch) {
        if (CHUNKS >= 8) return row * ROW + ((ch & ~7) | ((ch ^ row) & 7)) * 16;
        constexpr int PER = 8 / (CHUNKS < 8 ? CHUNKS : 8);   // rows in a line
        const int line = row / PER;
        return line * 128 + ((row % PER) * CHUNKS + (ch ^ (line % CHUNKS))) * 16;
    }
};

template <int PREC, int DP, int NT>
struct MmaShape {
    // Warps a CTA, CTAs an SM, slots a warp: what 64 K registers and 227 KB of shared memory hold, with at least 60 KB of
    // rows on their way (HBM's latency times its rate is about 43 KB an SM).
    static constexpr int W = PREC == 0 ? 512 / DP : PREC >= 2 && (NT == 1 || DP == 256) ? 8 : 4;
    static constexpr int CTAS = PREC == 0 || DP == 256 ? 1 : NT == 2 ? (PREC == 1 ? 2 : 3) : PREC == 1 ? 3 : 2;
    static constexpr int SLOTS = PREC == 1 && DP < 256 ? 2 : 3;
    static constexpr int MQ = PREC == 0 ? DP / 8 : DP / 16;   // MMAs that a tile's scores take a term
};

// Zeros for what is not finite in a warp's fp16 or fp32 values; whether this lane found any.
template <int PREC, int PIECES>
__device__ __noinline__ bool leave_out(uint4* values) {
    bool any = false;
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < PIECES; i += 32) {
        const uint4 u = values[i];
        if constexpr (PREC == 1) {
            if (odd_halves(u) == 0) continue;
            values[i] = finite_halves(u);
        } else {
            const bool x = finite(__uint_as_float(u.x)), y = finite(__uint_as_float(u.y)), z = finite(__uint_as_float(u.z)), w = finite(__uint_as_float(u.w));
            if (x && y && z && w) continue;
            values[i] = make_uint4(x ? u.x : 0u, y ? u.y : 0u, z ? u.z : 0u, w ? u.w : 0u);
        }
        any = true;
    }
    return any;
}

template <int PREC, int DP, int NT, int NQ>
__host__ __device__ constexpr size_t mma_smem() {
    constexpr int W = MmaShape<PREC, DP, NT>::W, ROWS = 8 * NT;
    return (size_t)W * MmaShape<PREC, DP, NT>::SLOTS * Slot<PREC, DP>::BYTES + (size_t)MmaShape<PREC, DP, NT>::MQ * NT * NQ * 32 * 8 +
           (join_floats<ROWS, 32 * W, kMmaParts>() + (3 * W + 2 + bias_blocks<PREC, DP>()) * ROWS) * 4;
}

// exact: the head has DP values (and, for int4, groups of 16): rows and scales are copied whole, in steps known here.
// LIMIT: rows may see different tokens (several new ones under a causal limit).  Without it the look at fp16 and fp32 values is
// left out, which costs a call of one token 3 %.
// LISTED: lists of pages, whose tables and lengths the CTAs make (a.reserved > 0) or a launch before this one.  A kernel of its own, as their
// plain loads and the second way to a share cost calls of whole sequences 2 to 5 % (one of 32768 int4 tokens 82.6 -> 84.6 us, 128 fp16 tokens 12.7 -> 13.1).
template <int PREC, int DP, int NT, int NQ, int NP, bool LIMIT, bool LISTED>
__global__ void __launch_bounds__(32 * MmaShape<PREC, DP, NT>::W, MmaShape<PREC, DP, NT>::CTAS)
pool_attention_mma_kernel(const __grid_constant__ skv_pool_attention_args a, const __grid_constant__ skv_pool_sparse_args lists,
                          int row_tiles, PageDivide magic, bool exact, bool q_vec, bool out_vec) {
    using L = Slot<PREC, DP>;
    constexpr int M = DP / 16, MQ = MmaShape<PREC, DP, NT>::MQ, ROWS = 8 * NT, W = MmaShape<PREC, DP, NT>::W, S = MmaShape<PREC, DP, NT>::SLOTS;
    constexpr int THREADS = 32 * W, TILE = 16 * W;
    extern __shared__ __align__(128) char mma_sm[];
    __shared__ Share s;
    __shared__ int s_free[W];
    __shared__ int s_odd;   // whether values of the segment that are not finite were left out
    char* s_ring = mma_sm;                                                       // [W][S] slots
    uint2* s_q = reinterpret_cast<uint2*>(s_ring + W * S * L::BYTES);            // [MQ][NT][NQ][32]
    float* s_join = reinterpret_cast<float*>(s_q + MQ * NT * NQ * 32);
    float* s_ref = s_join + join_floats<ROWS, THREADS, kMmaParts>();             // [W][ROWS]
    float* s_sum = s_ref + W * ROWS;                                             // [W][ROWS]
    float* s_w = s_sum + W * ROWS;                                               // [W][ROWS]
    float* s_c = s_w + W * ROWS;                                                 // [ROWS] factor of a row's scores; later its max
    float* s_l = s_c + ROWS;                                                     // [ROWS]
    float* s_bias = s_l + ROWS;                                                  // [blocks][ROWS] where the score sums start
    const int D = a.pool.head_dim, P = a.pool.page_size;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lg = lane >> 2, lc = lane & 3;
    const int rep = a.q.heads / a.pool.heads, R = rep * a.S_q;
    const bool p16 = P % 16 == 0;   // a tile lies in one page
    auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * magic.mul) >> magic.shift); };
    if constexpr (LISTED) wait_for_dependency();
    if (LISTED && a.reserved > 0) take_listed<THREADS>(a, lists, TILE, row_tiles, &s);
    else take_share<THREADS, LISTED>(a, TILE, a.pool.heads * row_tiles, kMmaPad, kMinTiles, &s);
    if (s.lo >= s.hi) return;
    char* ring = s_ring + warp * S * L::BYTES;
    if (!exact) {   // chunks that the head does not have are never copied: they count as zero
        for (int i = lane; i < S * L::BYTES / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }

    // ---- copying ahead: this warp's tiles in order, over all segments of the share
    struct {
        int at, b, base;             // the next segment to open
        int hk, tokens, st, end;     // the open one: tiles [st, end), every W-th is this warp's
    } f;
    f.at = s.lo;
    f.b = s.b;
    f.base = s.base;
    f.st = f.end = f.hk = f.tokens = 0;
    PageRows<LISTED> pages;
    const int row_bytes = PREC == 0 ? 4 * D : PREC == 1 ? 2 * D : PREC == 2 ? D : D / 2;
    constexpr int WIDE = L::CHUNKS > 32 ? L::CHUNKS / 32 : 1;   // copies a row takes
    constexpr int STEP = 32 * WIDE / L::CHUNKS, COPIES = 16 / STEP;   // rows a warp's copy takes, copies a tile takes
    const int my_row = lane / L::CHUNKS, my_chunk = lane % L::CHUNKS;
    const char* k_lane = static_cast<const char*>(a.pool.k) + my_chunk * 16;
    const char* v_lane = static_cast<const char*>(a.pool.v) + my_chunk * 16;
    const int to_lane = L::at(my_row, my_chunk);
    auto copy_next = [&](char* slot) {
        while (f.st >= f.end) {
            if (f.at >= s.hi) {
                copy_commit();   // an empty group keeps the count
                return;
            }
            const Segment g = segment_at<LISTED>(a, s, f.at, TILE, row_tiles, f.b, f.base);
            f.at = g.next;
            f.hk = g.hk;
            f.tokens = g.tokens;
            f.end = min(g.t1 * W, (g.tokens + 15) / 16);
            f.st = g.t0 * W + warp;
            pages.start(a.pool, g.b, p16 ? page_of(f.st * 16) : 0);
        }
        // the pool row of token lane % 16 of the tile, -1 where there is none; absent rows copy row 0, unused
        const int t0 = f.st * 16, t = t0 + (lane & 15);
        int row = -1, first = 0;
        if (p16) {
            const int j = page_of(t0), page = pages.page(j);
            if (page >= 0 && page < a.pool.num_pages) {
                first = (page * a.pool.heads + f.hk) * P + (t0 - j * P);
                row = t < f.tokens ? first + (lane & 15) : -1;
            } else if (a.error_flag) {
                atomicExch(a.error_flag, 1);
            }
        } else if (t < f.tokens) {
            const int j = page_of(t), page = number_at<LISTED>(pages.table + j);   // t is below the table's width
            if (page >= 0 && page < a.pool.num_pages) row = (page * a.pool.heads + f.hk) * P + (t - j * P);
            else if (a.error_flag) atomicExch(a.error_flag, 1);
        }
        const uint32_t to = shared_address(slot), to_rows = to + L::K + to_lane;
        if (lane < 16) *reinterpret_cast<int*>(slot + L::ID + 4 * lane) = row;
        if (p16 && exact) {
            const char* k = k_lane + (int64_t)(first + my_row) * L::ROW;
            const char* v = v_lane + (int64_t)(first + my_row) * L::ROW;
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const uint32_t y = L::step(to_rows, i, STEP);
#pragma unroll
                for (int h = 0; h < WIDE; ++h) {   // 512 bytes on, a chunk has the same place in its line
                    copy_async<16>(y + 512 * h, k + i * STEP * L::ROW + 512 * h);
                    copy_async<16>(y + 512 * h + L::V, v + i * STEP * L::ROW + 512 * h);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const int r = p16 ? first + my_row + i * STEP : max(__shfl_sync(0xffffffffu, row, my_row + i * STEP), 0);
                const uint32_t y = L::step(to_rows, i, STEP);
                if (PREC <= 1 || row_bytes % 16 == 0) {
#pragma unroll
                    for (int h = 0; h < WIDE; ++h)
                        if (my_chunk * 16 + 512 * h < row_bytes) {
                            copy_async<16>(y + 512 * h, k_lane + (int64_t)r * row_bytes + 512 * h);
                            copy_async<16>(y + 512 * h + L::V, v_lane + (int64_t)r * row_bytes + 512 * h);
                        }
                } else {   // rows end in half a chunk, and every second one starts in the middle of 16 bytes
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (my_chunk * 16 + 8 * h < row_bytes) {
                            copy_async<8>(y + 8 * h, k_lane + (int64_t)r * row_bytes + 8 * h);
                            copy_async<8>(y + L::V + 8 * h, v_lane + (int64_t)r * row_bytes + 8 * h);
                        }
                }
            }
        }
        if constexpr (PREC == 2) {
            copy_async<4>(to + (lane < 16 ? L::SK : L::SV) + 4 * (lane & 15),
                          (lane < 16 ? a.pool.scale_k : a.pool.scale_v) + (p16 ? first + (lane & 15) : max(row, 0)));
        } else if constexpr (PREC == 3) {
            constexpr int PARTS = L::BLOCKS / 4;   // 16-byte pieces of a token's scales
            if (exact) {
#pragma unroll
                for (int i = 0; i < (PARTS + 1) / 2; ++i) {
                    const int tok = (lane + 32 * i) / PARTS & 15, piece = (lane + 32 * i) % PARTS;
                    const int r = p16 ? first + tok : max(__shfl_sync(0xffffffffu, row, tok), 0);
                    const int64_t x = (int64_t)r * L::BLOCKS + 4 * piece;
                    const uint32_t y = to + L::SK + tok * L::BLOCKS * 4 + piece * 16;
                    if (PARTS > 1 || lane < 16) copy_async<16>(y, a.pool.scale_k + x);
                    if (PARTS > 1 || lane >= 16) copy_async<16>(y + (L::SV - L::SK), a.pool.scale_v + x);
                }
            } else {
                const int groups = D / a.pool.int4_group;
#pragma unroll
                for (int i = 0; i < L::BLOCKS / 2; ++i) {
                    const int tok = (lane + 32 * i) / L::BLOCKS, block = (lane + 32 * i) % L::BLOCKS;
                    const int r = p16 ? first + tok : max(__shfl_sync(0xffffffffu, row, tok), 0);
                    if (block * 16 < D) {
                        const int64_t x = (int64_t)r * groups + block * 16 / a.pool.int4_group;
                        copy_async<4>(to + L::SK + (lane + 32 * i) * 4, a.pool.scale_k + x);
                        copy_async<4>(to + L::SV + (lane + 32 * i) * 4, a.pool.scale_v + x);
                    }
                }
            }
        }
        copy_commit();
        f.st += W;
    };
    int head = 0;   // slot of the tile to multiply; the one before it is free
    int merged = -1;   // the slot that held sums when the segment before ended
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy_next(ring + i * L::BYTES);

    int at = s.lo, b = s.b, base = s.base;
    while (at < s.hi) {
        const Segment g = segment_at<LISTED>(a, s, at, TILE, row_tiles, b, base);
        at = g.next;
        if (g.t0 >= g.t1) continue;
        const int n = g.tokens, r0 = g.rt * ROWS;
        // ---- queries: a power of two taken out of each row, laid out as B operands
        __syncthreads();
        if (tid == 0) s_odd = 0;
        if (!exact && merged >= 0) {   // chunks that are never copied count as zero again
            for (int i = lane; i < L::BYTES / 16; i += 32) reinterpret_cast<uint4*>(s_ring + merged)[i] = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        {
            constexpr int RW = ROWS / W, E = DP / 32;   // a warp's rows, a lane's values of each
            float x[RW][E];
#pragma unroll
            for (int i = 0; i < RW; ++i) {   // every load before the first use
                const int r = r0 + warp * RW + i, d = lane * E;
#pragma unroll
                for (int k = 0; k < E; ++k) x[i][k] = 0.0f;
                if (r < R && d < D) {
                    if (a.q.dtype == kF32) load_row<E>(row_ptr<const float>(a.q, a.S_q, rep, g.b, g.hk, r) + d, D - d, q_vec, x[i]);
                    else if (a.q.dtype == kF16) load_row<E>(row_ptr<const __half>(a.q, a.S_q, rep, g.b, g.hk, r) + d, D - d, q_vec, x[i]);
                    else load_row<E>(row_ptr<const __nv_bfloat16>(a.q, a.S_q, rep, g.b, g.hk, r) + d, D - d, q_vec, x[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const int j = warp * RW + i;
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < E; ++k) top = fmaxf(top, fabsf(x[i][k]));
                const int e = clamp_exp(__float_as_uint(warp_max(top)));
                const float down = exp_down(e, kQueryExp);
                if (lane == 0) s_c[j] = a.scale * 1.4426950408889634f * exp_up(e, kQueryExp) * (PREC <= 1 ? 1.0f : 1.0f / subnormal_unit<PREC, NQ>());
                float total = 0.0f;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    int mma, c, reg, half;
                    const float part = query_place<PREC, DP, NQ>(lane * E + k, mma, c, reg, half);
                    const float y = x[i][k] * down * part;
                    if constexpr (PREC == 0) {
                        uint32_t* q = reinterpret_cast<uint32_t*>(s_q + ((mma * NT + j / 8) * NQ) * 32 + (j % 8) * 4 + c) + reg;
                        q[0] = NQ == 1 ? tf32_cut(y) : tf32_round(y);   // all of it where the query has 16 bits
                        if (NQ == 2) q[32 * 2] = __float_as_uint(y - __uint_as_float(tf32_round(y)));
                        continue;
                    }
                    const __half hi = __float2half_rn(y);
                    __half* q = reinterpret_cast<__half*>(s_q + ((mma * NT + j / 8) * NQ) * 32 + (j % 8) * 4 + c) + 2 * reg + half;
                    q[0] = hi;
                    float used = __half2float(hi);
                    if (NQ == 2) {
                        const __half lo = __float2half_rn(y - used);
                        q[32 * 4] = lo;
                        used += __half2float(lo);
                    }
                    total += used / part;
                }
                if constexpr (PREC >= 2) {
                    constexpr int LANES = PREC == 2 ? 32 : 16 / E;   // that share a bias
#pragma unroll
                    for (int w = 1; w < LANES; w <<= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
                    if (lane % LANES == 0) s_bias[lane / LANES * ROWS + j] = total * ((PREC == 2 ? -128.0f : -8.0f) * subnormal_unit<PREC, NQ>());
                }
            }
        }
        __syncthreads();
        float start_at[NT][2];   // of the score sums
        float cf[NT][2], ref[NT][2], base_of[NT][2], sum[NT][2], o[NT][M][4];   // base_of: ref, or 0 before there is one
        int see[NT][2], see_all = n, see_least = n;   // tokens that a row sees, that all do, that all do which see any
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = 8 * t + 2 * lc + i;
                cf[t][i] = s_c[j];
                start_at[t][i] = PREC == 2 ? s_bias[j] : 0.0f;
                ref[t][i] = -INFINITY;
                base_of[t][i] = 0.0f;
                sum[t][i] = 0.0f;
                see[t][i] = r0 + j < R ? seen_by(a, g.b, n, (r0 + j) % a.S_q) : n;
                see_all = min(see_all, see[t][i]);
                if (see[t][i] > 0) see_least = min(see_least, see[t][i]);
            }
        see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 1));
        see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 2));
        see_least = min(see_least, __shfl_xor_sync(0xffffffffu, see_least, 1));
        see_least = min(see_least, __shfl_xor_sync(0xffffffffu, see_least, 2));
        const int not_all = not_all_from(see_least, n, 16);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][m][i] = 0.0f;

        const int end = min(g.t1 * W, (n + 15) / 16);
        for (int st = g.t0 * W + warp; st < end; st += W) {
            copy_wait<S - 2>();
            __syncwarp();
            copy_next(ring + (head == 0 ? S - 1 : head - 1) * L::BYTES);
            char* slot = ring + head * L::BYTES;
            head = head + 1 == S ? 0 : head + 1;
            // ---- tokens that are there
            const int t0 = st * 16;
            const bool held = *reinterpret_cast<const int*>(slot + L::ID + 4 * (lane & 15)) >= 0;   // token lane % 16
            const bool all = __all_sync(0xffffffffu, held) && t0 + 16 <= see_all;
            bool here[2] = {true, true};
            if (!all) {
#pragma unroll
                for (int i = 0; i < 2; ++i) here[i] = __shfl_sync(0xffffffffu, (int)held, lg + 8 * i);
                // a weight of zero would not hide a NaN in what an absent token's row or scale happens to hold
                if (!held && lane < 16) {
                    if constexpr (PREC <= 1)
                        for (int i = 0; i < L::CHUNKS; ++i) *reinterpret_cast<uint4*>(slot + L::V + lane * L::ROW + i * 16) = make_uint4(0, 0, 0, 0);
                    else
                        for (int i = 0; i < L::SCALES; ++i) reinterpret_cast<float*>(slot + L::SV)[lane * L::SCALES + i] = 1.0f;
                }
                __syncwarp();
            }
            if constexpr (PREC <= 1 && LIMIT) {
                if (t0 >= not_all) {   // values that are not finite wait until the rows that see them are known apart
                    const bool odd = leave_out<PREC, 16 * L::CHUNKS>(reinterpret_cast<uint4*>(slot + L::V));
                    if (odd) s_odd = 1;
                    __syncwarp();
                }
            }
            // ---- scores
            float x[NT][4], k_factor[2] = {1.0f, 1.0f};
            if constexpr (PREC < 3) {
                // CH chains of dependent MMAs at a time: one would be as long as their latencies added up
                constexpr int CH = NT == 1 ? 4 : NT == 2 ? 2 : 1;
                float acc[CH][NT][4];
                auto qk = [&](const uint32_t (&f)[4], int m) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            const int h = (m * NQ + q) % CH;
                            const uint2 bq = s_q[((m * NT + t) * NQ + q) * 32 + lane];
                            if (m * NQ + q == 0) mma16816_from(acc[h][t], f, bq, start_at[t][0], start_at[t][1]);
                            else if (m * NQ + q < CH) mma16816_from(acc[h][t], f, bq, 0.0f, 0.0f);
                            else mma16816(acc[h][t], f, bq);
                        }
                };
                if constexpr (PREC == 0) {
                    // high part times the query's first term; the terms 2^-12 of that (low times first, high times second)
                    // have a chain of their own, where an MMA cuts off less
                    float small[NT][4];
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            small[t][i] = 0.0f;
#pragma unroll
                            for (int h = 0; h < CH; ++h) acc[h][t][i] = 0.0f;
                        }
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j) {
                        const int ch = 8 * (j / 2) + 2 * lc + j % 2;
                        const float4 u = *reinterpret_cast<const float4*>(slot + L::K + L::at(lg, ch));
                        const float4 v = *reinterpret_cast<const float4*>(slot + L::K + L::at(lg + 8, ch));
                        const float y[2][4] = {{u.x, v.x, u.y, v.y}, {u.z, v.z, u.w, v.w}};
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int m = 2 * j + w;
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                hi[i] = tf32_round(y[w][i]);
                                lo[i] = __float_as_uint(y[w][i] - __uint_as_float(hi[i]));
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                const uint2 bq = s_q[(m * NT + t) * NQ * 32 + lane];
                                mma1688(acc[m % CH][t], hi, bq);
                                mma1688(small[t], lo, bq);
                                if constexpr (NQ == 2) mma1688(small[t], hi, s_q[((m * NT + t) * NQ + 1) * 32 + lane]);
                            }
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[0][t][i] += small[t][i];
                } else if constexpr (PREC == 1) {
                    const uint32_t k = shared_address(slot + L::K);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        uint32_t f[4];
                        load_matrix(f, k + L::at(lane & 15, 2 * m + (lane >> 4)));
                        qk(f, m);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) {
                        const int ch = DP / 64 * lc + j;
                        const uint4 u4 = *reinterpret_cast<const uint4*>(slot + L::K + L::at(lg, ch));
                        const uint4 v4 = *reinterpret_cast<const uint4*>(slot + L::K + L::at(lg + 8, ch));
                        const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t f[4] = {(u[w] & 0x00FF00FFu) ^ 0x00800080u, (v[w] & 0x00FF00FFu) ^ 0x00800080u,
                                                   ((u[w] >> 8) & 0x00FF00FFu) ^ 0x00800080u, ((v[w] >> 8) & 0x00FF00FFu) ^ 0x00800080u};
                            qk(f, 4 * j + w);
                        }
                    }
                    k_factor[0] = reinterpret_cast<const float*>(slot + L::SK)[lg];
                    k_factor[1] = reinterpret_cast<const float*>(slot + L::SK)[lg + 8];
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[t][i] = acc[0][t][i];
#pragma unroll
                        for (int h = 1; h < CH; ++h) x[t][i] += acc[h][t][i];
                    }
            } else {
                // A group of 16 values is one MMA, so that its scale can multiply the result: lane column c takes bytes
                // 2c, 2c + 1 of each group, of two groups at a time (blocks k and k + M / 2) in one register.
                const uint32_t pick = lc & 1 ? 0x7362 : 0x5140;
                float sc[2][M];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int k = 0; k < M / 4; ++k) {
                        const float4 y = *reinterpret_cast<const float4*>(slot + L::SK + ((lg + 8 * t) * M + 4 * k) * 4);
                        sc[t][4 * k] = y.x; sc[t][4 * k + 1] = y.y; sc[t][4 * k + 2] = y.z; sc[t][4 * k + 3] = y.w;
                    }
                auto word = [&](int row, int block) {
                    return *reinterpret_cast<const uint32_t*>(slot + L::K + L::at(row, block / 2) + 8 * (block % 2) + 4 * (lc >> 1));
                };
#pragma unroll
                for (int k = 0; k < M / 2; ++k) {
                    const uint32_t u = __byte_perm(word(lg, k), word(lg, k + M / 2), pick);
                    const uint32_t v = __byte_perm(word(lg + 8, k), word(lg + 8, k + M / 2), pick);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int m = k + M / 2 * h;
                        constexpr uint32_t mask = 0x03C003C0u;
                        const uint32_t uh = u >> (8 * h), vh = v >> (8 * h);
                        const uint32_t f[4] = {NQ == 2 ? (h ? u >> 6 : u << 2) & mask : uh & 0x00F000F0u,
                                               NQ == 2 ? (h ? v >> 6 : v << 2) & mask : vh & 0x00F000F0u,
                                               NQ == 2 ? (h ? u >> 2 : u << 6) & mask : uh & 0x000F000Fu,
                                               NQ == 2 ? (h ? v >> 2 : v << 6) & mask : vh & 0x000F000Fu};
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float acc[4];
                            const float2 start = *reinterpret_cast<const float2*>(s_bias + m * ROWS + 8 * t + 2 * lc);
#pragma unroll
                            for (int q = 0; q < NQ; ++q) {
                                const uint2 bq = s_q[((m * NT + t) * NQ + q) * 32 + lane];
                                if (q == 0) mma16816_from(acc, f, bq, start.x, start.y);
                                else mma16816(acc, f, bq);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                x[t][i] = k + h == 0 ? acc[i] * sc[i >> 1][m] : fmaf(acc[i], sc[i >> 1][m], x[t][i]);
                        }
                    }
                }
            }
            // ---- weights
            float v_add[2] = {0.0f, 0.0f}, v_mul[2] = {1.0f, 1.0f}, v_sum[2] = {1.0f, 1.0f};
            int token_exp = 0;   // int4: of token lane % 16
            if constexpr (PREC == 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float sv = reinterpret_cast<const float*>(slot + L::SV)[lg + 8 * i];
                    const int e = clamp_exp(__float_as_uint(sv) & 0x7fffffffu);
                    v_add[i] = (float)(e - 127);
                    v_sum[i] = __uint_as_float((uint32_t)(254 - e) << 23);   // 2^-(e - 127)
                    v_mul[i] = sv * v_sum[i];
                }
            } else if constexpr (PREC == 3) {
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < M / 4; ++k) {
                    const uint4 y = *reinterpret_cast<const uint4*>(slot + L::SV + ((lane & 15) * M + 4 * k) * 4);
                    top = max(max(top, y.x & 0x7fffffffu), max(y.y & 0x7fffffffu, max(y.z & 0x7fffffffu, y.w & 0x7fffffffu)));
                }
                if (__any_sync(0xffffffffu, top >= 0x7f800000u)) {   // a group that is not finite says nothing of the others' size
                    __syncwarp();
                    top = 0;
#pragma unroll 1
                    for (int k = 0; k < M; ++k) {
                        uint32_t* at = reinterpret_cast<uint32_t*>(slot + L::SV) + (lane & 15) * M + k;
                        const uint32_t y = *at & 0x7fffffffu;
                        if (y < 0x7f800000u) top = max(top, y);
                        else if (lane < 16) *at = 0;
                    }
                    s_odd = 1;
                    __syncwarp();
                }
                token_exp = clamp_exp(top);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = __shfl_sync(0xffffffffu, token_exp, lg + 8 * i);
                    v_add[i] = (float)(e - 127 - kValueExp);
                    v_sum[i] = exp_down(e, kValueExp);                      // 2^-(e - 127 - kValueExp)
                }
            }
            bool grow = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = i >> 1, col = i & 1;
                    float z = x[t][i] * (cf[t][col] * k_factor[tok]);
                    if (PREC >= 2) z += v_add[tok];
                    if (!all && (!here[tok] || t0 + lg + 8 * tok >= see[t][col])) z = -INFINITY;
                    x[t][i] = z;
                    grow |= z > ref[t][col] + kRefRoom;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(x[t][i], x[t][i + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float now = fmaxf(ref[t][i], top - kRefDrop);
                        const float f = now == -INFINITY ? 1.0f : fast_exp2(ref[t][i] - now);
                        ref[t][i] = now;
                        base_of[t][i] = now == -INFINITY ? 0.0f : now;
                        sum[t][i] *= f;
#pragma unroll
                        for (int m = 0; m < M; ++m) {
                            o[t][m][i] *= f;
                            o[t][m][i + 2] *= f;
                        }
                    }
            }
            uint2 p[NT][NP];   // (PREC 0: of tokens 0 to 7, and in p8 of 8 to 15)
            uint2 p8[NT][NP];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = i >> 1, col = i & 1;
                    const float y = fast_exp2(x[t][i] - base_of[t][col]);
                    sum[t][col] = PREC >= 2 ? fmaf(y, v_sum[tok], sum[t][col]) : sum[t][col] + y;
                    w[i] = PREC == 2 ? y * v_mul[tok] : y;
                    if (PREC == 2 && !all && x[t][i] == -INFINITY) w[i] = 0.0f;   // (a scale may be infinite)
                }
                if constexpr (PREC == 0) {   // (a NaN that rounding would hide is in the sum)
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        uint32_t r[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            r[i] = tf32_round(w[i]);
                            w[i] -= __uint_as_float(r[i]);
                        }
                        p[t][k] = transpose8x8(r[0], r[1]);
                        p8[t][k] = transpose8x8(r[2], r[3]);
                    }
                    continue;
                }
                const uint32_t lo = h2_pack(w[0], w[1]), hi = h2_pack(w[2], w[3]);
                p[t][0] = make_uint2(transpose8x8(lo), transpose8x8(hi));
                if constexpr (NP == 2) {
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                    const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    p[t][1] = make_uint2(transpose8x8(h2_pack(w[0] - f0.x, w[1] - f0.y)),
                                         transpose8x8(h2_pack(w[2] - f1.x, w[3] - f1.y)));
                }
            }
            // ---- values
            // An MMA cuts its sum off where an addition would round: a relative 2^-24 of the sums is lost with each on average,
            // all in one direction.  32-bit outputs add a tile's own sums to those before instead (256 tiles a warp cost
            // 3e-5 of the result; 16-bit outputs, whose rounding is 100 times that, let the MMAs add).
            constexpr bool kFresh = NQ == 2;
            float fresh[NT][4];
            auto pv = [&](const uint32_t (&f)[4], int m, int terms, bool first, bool last) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const int q = kFresh ? NP - 1 - i : i;   // the small term first
                        if (q >= terms) continue;
                        if (!kFresh) mma16816(o[t][m], f, p[t][q]);
                        else if (first && q == terms - 1) mma16816_from(fresh[t], f, p[t][q], 0.0f, 0.0f);
                        else mma16816(fresh[t], f, p[t][q]);
                    }
                    if (kFresh && last)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[t][m][i] += fresh[t][i];
                }
            };
            if constexpr (PREC == 0) {
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    float4 y[2][2];   // tokens 8 h + 2 c and the next, values 4 (8 j + g) ..
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            y[h][i] = *reinterpret_cast<const float4*>(slot + L::V + L::at(8 * h + 2 * lc + i, 8 * j + lg));
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        float acc[NT][4];
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[t][i] = kFresh ? 0.0f : o[t][2 * j + w][i];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float z[4] = {w ? y[h][0].z : y[h][0].x, w ? y[h][0].w : y[h][0].y,
                                                w ? y[h][1].z : y[h][1].x, w ? y[h][1].w : y[h][1].y};
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                hi[i] = tf32_round(z[i]);
                                lo[i] = __float_as_uint(z[i] - __uint_as_float(hi[i]));
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                mma1688(acc[t], lo, h ? p8[t][0] : p[t][0]);
                                if constexpr (NP == 2) mma1688(acc[t], hi, h ? p8[t][1] : p[t][1]);
                                mma1688(acc[t], hi, h ? p8[t][0] : p[t][0]);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[t][2 * j + w][i] = kFresh ? o[t][2 * j + w][i] + acc[t][i] : acc[t][i];
                    }
                }
            } else if constexpr (PREC == 1) {
                const uint32_t v = shared_address(slot + L::V);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    uint32_t f[4];
                    load_matrix_trans(f, v + L::at((lane & 7) + (lane >> 4) * 8, 2 * m + ((lane >> 3) & 1)));
                    pv(f, m, NP, true, true);
                }
            } else if constexpr (PREC == 2) {
                uint32_t vx[4][DP / 32];   // values DP/8 g .. of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = 2 * lc + (i & 1) + 8 * (i >> 1);
                    if constexpr (DP >= 128) {
#pragma unroll
                        for (int j = 0; j < DP / 128; ++j) {
                            const uint4 y = *reinterpret_cast<const uint4*>(slot + L::V + L::at(tok, DP / 128 * lg + j));
                            vx[i][4 * j] = y.x; vx[i][4 * j + 1] = y.y; vx[i][4 * j + 2] = y.z; vx[i][4 * j + 3] = y.w;
                        }
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2*>(slot + L::V + L::at(tok, lg / 2) + 8 * (lg & 1));
                        vx[i][0] = y.x; vx[i][1] = y.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < DP / 32; ++w) {
                    uint32_t y[2][2];   // [tokens low / high][values 0,1 / 2,3]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = vx[2 * h][w] ^ 0x80808080u, v = vx[2 * h + 1][w] ^ 0x80808080u;
                        y[h][0] = __byte_perm(u, v, 0x5140);
                        y[h][1] = __byte_perm(u, v, 0x7362);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t f[4] = {i8_pair(y[0][i], 0x4140), i8_pair(y[0][i], 0x4342),
                                               i8_pair(y[1][i], 0x4140), i8_pair(y[1][i], 0x4342)};
                        pv(f, 2 * w + i, NP, true, true);
                    }
                }
            } else {
                // A group's scale in parts of 7 bits (two, or three for 32-bit outputs): x = 64 + (n + 8) times a part
                // less 72 times it is exact in one fp16 fma.
                constexpr int PARTS = NQ == 2 ? 3 : 2, BLOCKS = DP >= 128 ? DP / 128 : 1, WORDS = DP / 64 / BLOCKS;   // a lane's
                uint32_t vx[4][DP / 64];
                float down[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = 2 * lc + (i & 1) + 8 * (i >> 1);
                    if constexpr (DP == 256) {
                        const uint4 z = *reinterpret_cast<const uint4*>(slot + L::V + L::at(tok, lg));
                        vx[i][0] = z.x; vx[i][1] = z.y; vx[i][2] = z.z; vx[i][3] = z.w;
                    } else if constexpr (DP == 128) {
                        const uint2 z = *reinterpret_cast<const uint2*>(slot + L::V + L::at(tok, lg / 2) + 8 * (lg & 1));
                        vx[i][0] = z.x; vx[i][1] = z.y;
                    } else {
                        vx[i][0] = *reinterpret_cast<const uint32_t*>(slot + L::V + L::at(tok, lg / 4) + 4 * (lg & 3));
                    }
                    down[i] = exp_down(__shfl_sync(0xffffffffu, token_exp, tok), kValueExp);
                }
#pragma unroll
                for (int w = 0; w < DP / 64; ++w) {
                    uint32_t r[PARTS][2], r72[PARTS][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float y[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            y[i] = reinterpret_cast<const float*>(slot + L::SV)[(2 * lc + i + 8 * h) * M + lg * M / 8 + w / WORDS] * down[2 * h + i];
#pragma unroll
                        for (int k = 0; k < PARTS; ++k) {
                            const float y0 = take7(y[0]), y1 = take7(y[1]);
                            r[k][h] = h2_pack(y0, y1);
                            r72[k][h] = h2_pack(-72.0f * y0, -72.0f * y1);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t u = __byte_perm(vx[0][w], vx[1][w], i ? 0x7632 : 0x5410);
                        const uint32_t v = __byte_perm(vx[2][w], vx[3][w], i ? 0x7632 : 0x5410);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {   // values 0, 1 and 2, 3 of the two bytes
                            const uint32_t f[4] = {i4_pair(h ? u >> 8 : u), i4_pair(h ? u >> 4 : u << 4),
                                                   i4_pair(h ? v >> 8 : v), i4_pair(h ? v >> 4 : v << 4)};
#pragma unroll
                            for (int n = 0; n < PARTS; ++n) {
                                const int k = kFresh ? PARTS - 1 - n : n;
                                const uint32_t y[4] = {h2_fma(f[0], r[k][0], r72[k][0]), h2_fma(f[1], r[k][0], r72[k][0]),
                                                       h2_fma(f[2], r[k][1], r72[k][1]), h2_fma(f[3], r[k][1], r72[k][1])};
                                pv(y, 4 * w + 2 * i + h, k == 0 || k < PARTS - 1 ? NP : 1, k == PARTS - 1, k == 0);
                            }
                        }
                    }
                }
            }
        }

        // ---- the warps' parts joined, 8 rows at a time through their free slots
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float l = sum[t][i];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (lg == 0) {
                    s_ref[warp * ROWS + 8 * t + 2 * lc + i] = ref[t][i];
                    s_sum[warp * ROWS + 8 * t + 2 * lc + i] = l;
                }
            }
        const int free_at = (warp * S + (head == 0 ? S - 1 : head - 1)) * L::BYTES;
        merged = free_at;
        if (lane == 0) s_free[warp] = free_at;
        float* part = slot_of(a, blockIdx.x, g.slot, ROWS);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float* mine = reinterpret_cast<float*>(s_ring + free_at);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float* row = mine + (2 * lc + i) * (DP + 4);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    if constexpr (PREC == 0) {
                        *reinterpret_cast<float2*>(row + 32 * (m / 2) + 4 * lg + 2 * (m % 2)) = make_float2(o[t][m][i], o[t][m][i + 2]);
                    } else if constexpr (PREC == 1) {
                        row[16 * m + lg] = o[t][m][i];
                        row[16 * m + 8 + lg] = o[t][m][i + 2];
                    } else {
                        *reinterpret_cast<float2*>(row + lg * (DP / 8) + 2 * m) = make_float2(o[t][m][i], o[t][m][i + 2]);
                    }
                }
            }
            __syncthreads();
            if (t == 0) {
                if (tid < ROWS) {
                    float m = -INFINITY, l = 0.0f;
                    for (int w = 0; w < W; ++w) m = fmaxf(m, s_ref[w * ROWS + tid]);
                    const float r = m == -INFINITY ? 0.0f : m;
                    for (int w = 0; w < W; ++w) {
                        const float y = exp2f(s_ref[w * ROWS + tid] - r);
                        s_w[w * ROWS + tid] = y;
                        l += s_sum[w * ROWS + tid] * y;
                    }
                    s_c[tid] = m;
                    s_l[tid] = l;
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = tid; i < 8 * DP / 4; i += THREADS) {
                const int j = 8 * t + i / (DP / 4), d = i % (DP / 4) * 4;
                if (r0 + j >= R || d >= D) continue;
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(s_ring + s_free[w] + ((j - 8 * t) * (DP + 4) + d) * 4);
                    const float z = s_w[w * ROWS + j];
                    y[0] = fmaf(v.x, z, y[0]); y[1] = fmaf(v.y, z, y[1]); y[2] = fmaf(v.z, z, y[2]); y[3] = fmaf(v.w, z, y[3]);
                }
                if (!g.whole) {
                    *reinterpret_cast<float4*>(part + j * D + d) = make_float4(y[0], y[1], y[2], y[3]);
                    continue;
                }
                const float l = s_l[j];
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = l == 0.0f ? 0.0f : y[k] / l;
                store_row(a, g, r0 + j, d, out_vec, y);
            }
            if (t + 1 < NT) __syncthreads();
        }
        if ((PREC == 3 || (PREC <= 1 && LIMIT)) && s_odd) {   // (set before the barriers above)
            const int first = g.t0 * TILE;
            __syncthreads();
            add_not_finite<PREC, LISTED>(a, g.b, g.hk, n, r0, min(ROWS, R - r0), PREC == 3 ? first : max(first, not_all), min(n, g.t1 * TILE),
                                 g.whole ? nullptr : part, tid, THREADS);
        }
        if (!g.whole) {
            if (tid < ROWS) {
                part[ROWS * D + tid] = s_c[tid];
                part[ROWS * D + ROWS + tid] = s_l[tid];
            }
            if (arrive(a, s, g)) join<ROWS, THREADS, 4, kMmaParts>(a, s, g, r0, min(ROWS, R - r0), s_join, out_vec);
        }
    }
}

// Raises the kernel's limit on shared memory, once a device.
template <auto KERNEL>
int allow_shared(size_t bytes) {
    static std::atomic<uint64_t> allowed{0};   // devices where that was done
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(allowed.load(std::memory_order_relaxed) >> dev & 1))) {
        e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return e == cudaSuccess ? SKV_OK : fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
}

template <int PREC, int DP, int NT, int NQ, int NP, bool LIMIT, bool LISTED>
int launch_mma(const skv_pool_attention_args& a, cudaStream_t st) {
    using Shape = MmaShape<PREC, DP, NT>;
    static_assert(Shape::CTAS * 2 * 8 * NT <= kRowsPerSm, "the scratch holds every CTA's slots");
    constexpr size_t smem = mma_smem<PREC, DP, NT, NQ>();
    static_assert(Shape::CTAS * (smem + 2048) <= 228 * 1024, "an SM holds the CTAs");
    const int R = a.q.heads / a.pool.heads * a.S_q, row_tiles = (R + 8 * NT - 1) / (8 * NT);
    const int64_t step = sequences_a_launch(a, row_tiles, 16 * Shape::W, kMmaPad);
    if (step == 0) return SKV_ERR_TOO_LARGE;
    PageDivide magic;
    magic.shift = 31;
    while ((1ll << (magic.shift - 31)) < a.pool.page_size) ++magic.shift;
    magic.mul = (uint32_t)(((1ull << magic.shift) + a.pool.page_size - 1) / a.pool.page_size);
    const bool exact = a.pool.head_dim == DP &&
                       (PREC != 3 || (a.pool.int4_group == 16 && ((reinterpret_cast<uintptr_t>(a.pool.scale_k) |
                                                                   reinterpret_cast<uintptr_t>(a.pool.scale_v)) & 15) == 0));
    const bool q_vec = rows_aligned(a.q), out_vec = rows_aligned(a.out);
    const unsigned all = sm_count() * Shape::CTAS, threads = 32 * Shape::W;
    const skv_pool_sparse_args none = {};
    constexpr auto kernel = pool_attention_mma_kernel<PREC, DP, NT, NQ, NP, LIMIT, LISTED>;
    if (const int rc = allow_shared<kernel>(smem)) return rc;
    if constexpr (LISTED) {
        const skv_pool_sparse_args& lists = *static_cast<const AttentionCall&>(a).lists;
        // Sequences of one head and of known length at most (lists of pages).  Where there are fewer units than CTAs, a unit's tiles are split
        // over those that would be idle; else units stay whole, unless too many CTAs would idle in the last round, where even shares of
        // all tiles are the better cut (512 units of 1024 fp16 tokens on 444 CTAs 57 against 52 us, of 512 int8 tokens on 296 26 against 37).
        const int64_t units = (int64_t)a.pool.batch * row_tiles, resident = (int64_t)sm_count() * Shape::CTAS;
        const int64_t most = (token_cap(a) + 16 * Shape::W - 1) / (16 * Shape::W), rounds = (units + resident - 1) / resident;
        int64_t splits = resident / units < most ? resident / units : most;
        // Units of 4 tiles stay whole, of 8 where two CTAs would be the cut: there is nothing to join then.  Else one CTA an SM where it has 256 tokens
        // at most: two on an SM would have fewer, slower ones, and a longer join.  (With the choice of pages before it: 8 units of 512 int8 tokens
        // 21.3 -> 17.9 us, 128 of 512 28.0 -> 23.3, 64 of 512 fp16 tokens 22.6 -> 20.2; 8 of 4096 int8 tokens 26.1 -> 24.7, 16 of 2048 fp16 tokens
        // 24.7 -> 23.3.  With twice the tokens 32 of 2048 fp16 or int8 tokens 24.2 -> 26.0, 24.0 -> 25.3.  int4, whose tiles are
        // more instructions: 32 of 1024 tokens 23.3 -> 24.3, 64 whole ones 26.3 -> 27.1.)
        const int64_t single = sm_count() / units;
        if (most <= 4 || (most <= 8 && (single == 1 || (single == 2 && PREC != 3)))) splits = 1;
        else if (PREC != 3 && single > 0 && single < splits && (most + single - 1) / single * 16 * Shape::W <= 256) splits = single;
        if (splits < 1) splits = 1;
        if (units * (most > splits ? most : splits) < (1ll << 30) && (rounds == 1 || 4 * units >= 3 * rounds * resident)) {
            skv_pool_attention_args part = a;
            part.reserved = (int32_t)splits;
            const int64_t ctas = rounds > 1 && a.pool.batch > resident ? resident : units * splits;   // (runs of whole sequences)
            launch_after(kernel, dim3((unsigned)ctas), threads, smem, st, part, lists, row_tiles, magic, exact, q_vec, out_vec);
            return check_launch("pool_attention");
        }
        if (const int rc = launch_tables(lists, st)) return rc;
        return by_sequences(a, step, [&](skv_pool_attention_args part) {
            part.reserved = 0;
            launch_after(kernel, dim3(all), threads, smem, st, part, none, row_tiles, magic, exact, q_vec, out_vec);
            return check_launch("pool_attention");
        });
    } else {
        return by_sequences(a, step, [&](const skv_pool_attention_args& part) {
            kernel<<<all, threads, smem, st>>>(part, none, row_tiles, magic, exact, q_vec, out_vec);
            return check_launch("pool_attention");
        });
    }
}

template <int PREC, int DP, int NT, int NQ, int NP, bool LISTED>
int launch_mma_limit(const skv_pool_attention_args& a, cudaStream_t st) {
    if constexpr (PREC <= 1 && !LISTED)   // (a unit of lists is one token)
        if (a.causal && a.S_q > 1) return launch_mma<PREC, DP, NT, NQ, NP, true, false>(a, st);
    return launch_mma<PREC, DP, NT, NQ, NP, false, LISTED>(a, st);
}

template <int PREC, int DP, int NT, bool LISTED>
int launch_mma_type(const skv_pool_attention_args& a, cudaStream_t st) {
    if (a.q.dtype == kF32) return launch_mma_limit<PREC, DP, NT, 2, 2, LISTED>(a, st);
    if (a.q.dtype == kF16) return launch_mma_limit<PREC, DP, NT, 1, 2, LISTED>(a, st);
    return launch_mma_limit<PREC, DP, NT, 1, 1, LISTED>(a, st);
}

// Row tiles of 8 or 16 rows.  (32 rows a tile were 10 to 20 % faster where hundreds of rows meet 8 K tokens or more,
// 212 against 255 us for 1024 rows of 8 key heads, and 1.5 times slower below: 50 against 33 us for 32 rows.)
template <int PREC, bool LISTED>
int launch_mma_prec(const skv_pool_attention_args& a, cudaStream_t st) {
    const int R = a.q.heads / a.pool.heads * a.S_q, D = a.pool.head_dim;
    if (D <= 64) return R <= 8 ? launch_mma_type<PREC, 64, 1, LISTED>(a, st) : launch_mma_type<PREC, 64, 2, LISTED>(a, st);
    if (D <= 128) return R <= 8 ? launch_mma_type<PREC, 128, 1, LISTED>(a, st) : launch_mma_type<PREC, 128, 2, LISTED>(a, st);
    if constexpr (PREC == 0) return launch_mma_type<0, 256, 1, LISTED>(a, st);   // slots of 32 KB leave no room for more rows
    else return R <= 8 ? launch_mma_type<PREC, 256, 1, LISTED>(a, st) : launch_mma_type<PREC, 256, 2, LISTED>(a, st);
}

}  // namespace skv
