// Attention over the page pool on the tensor cores, pages read straight into MMA fragments.
//
// A decoding step is bound by the pages' bytes, but at 4 bits a value the FMA pipe cannot keep up with
// HBM, and neither can one operand row a value where several query rows share a key head.  So
// both products run as mma.m16n8k16 (fp16 operands, fp32 sums), transposed so that the few query rows
// are the narrow side:
//     S^T [16 tokens x 8 rows] = K [16 x D] Q^T,     O^T [16 values x 8 rows] += V^T [16 x 16 tokens] P^T.
// (tcgen05 wants 128 rows of A in shared memory and its sums back through TMEM; with 8..32 query
// rows the pages would pass through shared memory only to be read once.)
//
// The contraction order of an MMA is free as long as both operands agree, so a lane's 16-byte load of
// a page row IS its share of the A operand: lane (g, c) = (lane / 4, lane % 4) takes chunks c, c+4, ...
// of the rows of tokens g and g+8 (K), and the g-th chunks of tokens 2c, 2c+1, 2c+8, 2c+9 (V), whose
// token pairs are interleaved with byte permutes.  No shared memory, no transposes of pages; the
// queries are laid out once per segment to match.  P^T's operand is S^T's result transposed by
// movmatrix.
//
// Exactness.  Page values enter the MMAs exactly: fp16 as it is, int8 and int4 as small integers.  An
// int8 row's scale multiplies its score (K) or its weight (V) in fp32.  An int4 group's scale is split into an
// 8-bit part r1 (times a 4-bit integer exact in fp16) and an 11-bit remainder r2, two MMAs, after a
// power of two is taken out (per tile for K, per token for V), so range is no concern.  Queries are
// scaled by a power of two a row; 16-bit ones fit one fp16 operand, fp32 ones take two (22 bits).  Weights are
// 2^(z - ref) <= 2^15 with z the score plus the exponent of V's scale; one operand for bf16 outputs, whose
// own rounding is 8 times coarser, else two.
//
// ref follows the running maximum lazily (only when a weight would pass 2^15 are sums rescaled), so
// most tiles need one vote and no shuffles; row sums stay in the lanes until the segment ends.
#pragma once

#include "pool_attention.cuh"

namespace skv {

constexpr int kMmaParts = 128;      // parts whose factors a joining CTA holds at a time
constexpr float kRefDrop = 5.0f;    // a fresh maximum's weight is 2^5: small weights keep their bits in fp16
constexpr float kRefRoom = 14.0f;   // weights may grow to 2^14 (times a mantissa < 2) before ref moves

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Page loads that keep the register's value where `on` is 0 (predicated: no branch in the loop).
__device__ __forceinline__ void load_page(uint4& v, const void* p, int on) {
    asm volatile("{ .reg .pred t; setp.ne.s32 t, %5, 0; @t ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4]; }"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w) : "l"(p), "r"(on));
}
__device__ __forceinline__ void load_page(uint2& v, const void* p, int on) {
    asm volatile("{ .reg .pred t; setp.ne.s32 t, %3, 0; @t ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2]; }"
                 : "+r"(v.x), "+r"(v.y) : "l"(p), "r"(on));
}
__device__ __forceinline__ void load_page(uint32_t& v, const void* p, int on) {
    asm volatile("{ .reg .pred t; setp.ne.s32 t, %2, 0; @t ld.global.nc.L1::no_allocate.u32 %0, [%1]; }"
                 : "+r"(v) : "l"(p), "r"(on));
}
__device__ __forceinline__ void load_scale(float& v, const float* p, int on) {
    asm volatile("{ .reg .pred t; setp.ne.s32 t, %2, 0; @t ld.global.nc.f32 %0, [%1]; }" : "+f"(v) : "l"(p), "r"(on));
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
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
// Small integers as fp16: 1024 + n has n in its low bits.
__device__ __forceinline__ uint32_t i8_pair(uint32_t biased, uint32_t sel) {        // bytes n + 128
    return h2_sub(__byte_perm(biased, 0x64646464u, sel), 0x64806480u);              // - 1152
}
__device__ __forceinline__ uint32_t i4_low(uint32_t w) {                            // nibbles n + 8 in bits 0-3
    return h2_sub((w & 0x000F000Fu) | 0x64006400u, 0x64086408u);                    // - 1032
}
__device__ __forceinline__ uint32_t i4_high(uint32_t w) {                           // in bits 4-7: 1024 + 16 (n + 8)
    return h2_fma((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);       // / 16 - 72
}
// x as an 8-bit value and an 11-bit remainder, each twice in a register.
__device__ __forceinline__ void split_scale(float x, float& r1, float& r2) {
    r1 = __uint_as_float((__float_as_uint(x) + 0x8000u) & 0xFFFF0000u);
    r2 = x - r1;
}
// 2^(127 + 10 - e) scales a float of exponent field e to [2^10, 2^11).
__device__ __forceinline__ int clamp_exp(uint32_t bits) { return min(max((int)(bits >> 23), 11), 253); }
__device__ __forceinline__ float exp_down(int e) { return __uint_as_float((uint32_t)(264 - e) << 23); }
__device__ __forceinline__ float exp_up(int e) { return __uint_as_float((uint32_t)(e - 10) << 23); }

// t / page_size for t < 2^31 as a product: mul = ceil(2^shift / page_size), shift = 31 + ceil(log2 page_size).
struct PageDivide {
    uint32_t mul;
    int shift;
};

// The page rows of a sequence's tokens for one key head.  A warp keeps the next 64 entries of the
// block table in its lanes and asks them by shuffle: tiles need no dependent load.
struct PageRows {
    const int32_t* table;
    int width, base, cur, next, lane;
    __device__ __forceinline__ int entry(int i) const { return i < width ? __ldg(table + i) : -1; }
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

// A lane's place in the pages: addresses of its chunk in row 0, and which of its chunks the head has.
template <int PREC, int DP>
struct LanePlace {
    static constexpr int KC = PREC == 1 ? DP / 32 : DP / 64;   // chunks of a K row
    static constexpr int VC = PREC == 1 ? DP / 64 : 1;         // of a V row
    const char *k, *v;
    const float *sk[PREC == 3 ? KC : 1], *sv, *sv_own[PREC == 3 ? KC : 1];
    int row_bytes, groups;
    int k_on[KC], v_on[VC];
    __device__ __forceinline__ void set(const skv_pool& p, int g, int c) {
        const int D = p.head_dim;
        row_bytes = PREC == 1 ? 2 * D : PREC == 2 ? D : D / 2;
        groups = PREC == 3 ? D / p.int4_group : 1;
        const int kb = PREC == 3 ? 8 : 16, vb = PREC == 1 ? 16 : PREC == 2 ? DP / 8 : DP / 16;
        k = static_cast<const char*>(p.k) + c * kb;
        v = static_cast<const char*>(p.v) + g * vb;
#pragma unroll
        for (int j = 0; j < KC; ++j) k_on[j] = (c + 4 * j) * kb < row_bytes;
#pragma unroll
        for (int j = 0; j < VC; ++j) v_on[j] = (g + 8 * j) * vb < row_bytes;
        sk[0] = p.scale_k;
        sv = p.scale_v;
        sv_own[0] = p.scale_v;
        if constexpr (PREC == 3) {
            sv += g * (DP / 8) / p.int4_group;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                sk[j] = p.scale_k + (c + 4 * j) * 16 / p.int4_group;
                sv_own[j] = p.scale_v + (c + 4 * j) * 16 / p.int4_group;
            }
        }
    }
};

// One warp's tile of 16 tokens, as loaded.  Chunks that the head does not have stay zero from clear().
template <int PREC, int DP>
struct KTile;
template <int PREC, int DP>
struct VTile;

template <int BYTES> struct PageChunk;
template <> struct PageChunk<16> { using type = uint4; };
template <> struct PageChunk<8> { using type = uint2; };
template <> struct PageChunk<4> { using type = uint32_t; };
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word_of(const uint2& v, int i) { return i == 0 ? v.x : v.y; }
__device__ __forceinline__ uint32_t word_of(uint32_t v, int) { return v; }

template <int DP>
struct KTile<1, DP> {
    uint4 x[2][DP / 32];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 32; ++j) x[t][j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const LanePlace<1, DP>& at, const int (&row)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char* q = at.k + (int64_t)row[t] * at.row_bytes;
#pragma unroll
            for (int j = 0; j < DP / 32; ++j)
                load_page(x[t][j], q + 64 * j, at.k_on[j]);
        }
    }
    __device__ __forceinline__ void only(const bool (&)[2]) {}   // scores of absent tokens are overwritten
};
template <int DP>
struct KTile<2, DP> {
    uint4 x[2][DP / 64];
    float s[2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) x[t][j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const LanePlace<2, DP>& at, const int (&row)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char* q = at.k + (int64_t)row[t] * at.row_bytes;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                load_page(x[t][j], q + 64 * j, at.k_on[j]);
            s[t] = __ldg(at.sk[0] + row[t]);
        }
    }
    __device__ __forceinline__ void only(const bool (&)[2]) {}
};
template <int DP>
struct KTile<3, DP> {
    uint2 x[2][DP / 64];
    float s[2][DP / 64];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {
                x[t][j] = make_uint2(0, 0);
                s[t][j] = 0.0f;
            }
    }
    __device__ __forceinline__ void load(const LanePlace<3, DP>& at, const int (&row)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char* q = at.k + (int64_t)row[t] * at.row_bytes;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {
                load_page(x[t][j], q + 32 * j, at.k_on[j]);
                load_scale(s[t][j], at.sk[j] + (int64_t)row[t] * at.groups, at.k_on[j]);
            }
        }
    }
    __device__ __forceinline__ void only(const bool (&own)[2]) {   // the tile's exponent is that of its tokens
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) s[t][j] = own[t] ? s[t][j] : 0.0f;
    }
};

template <int DP>
struct VTile<1, DP> {
    uint4 x[4][DP / 64];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) x[t][j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const LanePlace<1, DP>& at, const int (&row)[4], const int (&)[2]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const char* q = at.v + (int64_t)row[t] * at.row_bytes;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                load_page(x[t][j], q + 128 * j, at.v_on[j]);
        }
    }
    // a weight of zero does not hide a NaN or an infinity in a row that holds no token
    __device__ __forceinline__ void only(const bool (&four)[4], const bool (&)[2]) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (!four[t])
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) x[t][j] = make_uint4(0, 0, 0, 0);
    }
};
template <int DP>
struct VTile<2, DP> {
    using Chunk = typename PageChunk<DP / 8>::type;
    Chunk x[4];
    float s[2];   // of tokens g and g + 8
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = Chunk{};
    }
    __device__ __forceinline__ void load(const LanePlace<2, DP>& at, const int (&row)[4], const int (&own)[2]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) load_page(x[t], at.v + (int64_t)row[t] * at.row_bytes, at.v_on[0]);
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = __ldg(at.sv + own[t]);
    }
    __device__ __forceinline__ void only(const bool (&)[4], const bool (&own)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = own[t] ? s[t] : 1.0f;
    }
};
template <int DP>
struct VTile<3, DP> {
    using Chunk = typename PageChunk<DP / 16>::type;
    Chunk x[4];
    float s[4];              // of this lane's values, tokens 2c, 2c + 1, 2c + 8, 2c + 9
    float own[2][DP / 64];   // this lane's quarter of the scales of tokens g and g + 8
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = 0.0f;
            x[t] = Chunk{};
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) own[t][j] = 0.0f;
    }
    __device__ __forceinline__ void load(const LanePlace<3, DP>& at, const int (&row)[4], const int (&mine)[2]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            load_page(x[t], at.v + (int64_t)row[t] * at.row_bytes, at.v_on[0]);
            load_scale(s[t], at.sv + (int64_t)row[t] * at.groups, at.v_on[0]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) load_scale(own[t][j], at.sv_own[j] + (int64_t)mine[t] * at.groups, at.k_on[j]);
    }
    __device__ __forceinline__ void only(const bool (&four)[4], const bool (&mine)[2]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t] = four[t] ? s[t] : 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) own[t][j] = mine[t] ? own[t][j] : 0.0f;
    }
};

// E values of a row of which `left` exist, with one load where rows are aligned to them (their count is a
// multiple of E then, as head sizes here are multiples of 8).
template <int E, class T>
__device__ __forceinline__ void load_row(const T* p, int left, bool vec, float (&x)[E]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            if constexpr (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(p);
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(p);
                x[0] = v.x; x[1] = v.y;
            }
        } else {
            uint32_t w[E / 2];
            if constexpr (E == 4) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[0] = v.x; w[1] = v.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            }
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                const T* h = reinterpret_cast<const T*>(&w[i]);
                x[2 * i] = to_float(h[0]);
                x[2 * i + 1] = to_float(h[1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < left) x[i] = to_float(p[i]);
    }
}

// Where value d of a query row sits in the B operands: MMA, lane column c, register and half.
template <int PREC>
__device__ __forceinline__ void query_place(int d, int& mma, int& c, int& reg, int& half) {
    if (PREC == 1) {
        const int chunk = d / 8, h = d % 8;
        mma = 2 * (chunk / 4) + h / 4; c = chunk % 4; reg = (h % 4) / 2; half = h % 2;
    } else if (PREC == 2) {
        const int chunk = d / 16, h = d % 16;
        mma = 4 * (chunk / 4) + h / 4; c = chunk % 4; reg = (h % 4) / 2; half = h % 2;
    } else {
        const int chunk = d / 16, h = d % 8;
        mma = 2 * (2 * (chunk / 4) + (d % 16) / 8) + (h % 4) / 2; c = chunk % 4; reg = h % 2; half = h / 4;
    }
}

template <int DP, int NT, int NQ, int W>
__host__ __device__ constexpr size_t mma_smem() {
    static_assert(join_floats<8 * NT, 32 * W, kMmaParts>() <= W * 8 * NT * (DP + 4), "the join works in the warps' sums");
    return (size_t)(DP / 16) * NT * NQ * 32 * 8 + (size_t)W * 8 * NT * (DP + 4) * 4 + (3 * W + 2) * 8 * NT * 4;
}

template <int PREC, int DP, int NT, int NQ, int NP, int W, int CTAS>
__global__ void __launch_bounds__(32 * W, CTAS)
pool_attention_mma_kernel(const __grid_constant__ skv_pool_attention_args a, int row_tiles, PageDivide magic, bool q_vec, bool out_vec) {
    constexpr int M = DP / 16, ROWS = 8 * NT, THREADS = 32 * W, TILE = 16 * W;
    extern __shared__ __align__(16) char mma_sm[];
    __shared__ Share s;
    uint2* s_q = reinterpret_cast<uint2*>(mma_sm);                       // [M][NT][NQ][32]
    float* s_o = reinterpret_cast<float*>(s_q + M * NT * NQ * 32);       // [warps][ROWS][DP + 4]
    float* s_ref = s_o + W * ROWS * (DP + 4);                    // [warps][ROWS]
    float* s_sum = s_ref + W * ROWS;                             // [warps][ROWS]
    float* s_w = s_sum + W * ROWS;                               // [warps][ROWS]
    float* s_c = s_w + W * ROWS;                                 // [ROWS] factor of a row's scores; later its max
    float* s_l = s_c + ROWS;                                             // [ROWS]
    const int D = a.pool.head_dim, P = a.pool.page_size;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lg = lane >> 2, lc = lane & 3;
    const int rep = a.q.heads / a.pool.heads, R = rep * a.S_q;
    const bool p16 = P % 16 == 0;   // a tile lies in one page
    auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * magic.mul) >> magic.shift); };
    take_share<THREADS>(a, TILE, a.pool.heads * row_tiles, 2, &s);
    if (s.lo >= s.hi) return;
    int b = s.b, base = s.base, at = s.lo;
    PageRows pages;
    // Where a tile's tokens are: the pool row of its first token where a tile lies in one page, else the row of
    // token lane % 16; -1 where there is none (past the end, or no page).
    auto row_of = [&](const Segment& g, int tile) {
        const int t0 = tile * 16;
        int row = -1;
        bool lost = false;
        if (p16) {
            const int j = page_of(t0), page = pages.page(j);
            if (page >= 0 && page < a.pool.num_pages) row = (page * a.pool.heads + g.hk) * P + (t0 - j * P);
            else lost = true;
        } else if (t0 + (lane & 15) < g.tokens) {
            const int t = t0 + (lane & 15), j = page_of(t), page = __ldg(pages.table + j);   // t is below the table's width
            if (page >= 0 && page < a.pool.num_pages) row = (page * a.pool.heads + g.hk) * P + (t - j * P);
            else lost = true;
        }
        if (lost && a.error_flag) atomicExch(a.error_flag, 1);
        return row;
    };
    // The rows of the tokens whose K (g, g + 8) and V (2c, 2c + 1, 2c + 8, 2c + 9) this lane loads.  What has no row
    // reads row 0, and what it reads is not used.
    auto k_rows = [&](int row, int (&own)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) own[i] = max(p16 ? row : __shfl_sync(0xffffffffu, row, lg + 8 * i), 0) + (p16 ? lg + 8 * i : 0);
    };
    auto v_rows = [&](int row, int (&four)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = 2 * lc + (i & 1) + 8 * (i >> 1);
            four[i] = max(p16 ? row : __shfl_sync(0xffffffffu, row, k), 0) + (p16 ? k : 0);
        }
    };
    LanePlace<PREC, DP> place;
    place.set(a.pool, lg, lc);
    KTile<PREC, DP> kt;
    VTile<PREC, DP> vt;
    kt.clear();
    vt.clear();
    int st = 0, end = 0, row = -1;   // this warp's tile, the end of its tiles, the rows of the tile's tokens
    // The next segment, its first tile on the way.
    auto open = [&]() {
        const Segment g = segment_at(a, s, at, TILE, row_tiles, b, base);
        at += g.t1 - g.t0;
        end = min(g.t1 * W, (g.tokens + 15) / 16);
        st = g.t0 * W + warp;
        pages.start(a.pool, g.b, p16 ? page_of(st * 16) : 0);
        row = -1;
        if (st < end) {
            int own[2], four[4];
            row = row_of(g, st);
            k_rows(row, own);
            v_rows(row, four);
            kt.load(place, own);
            vt.load(place, four, own);
        }
        return g;
    };
    Segment g = open();
    for (;;) {
        const int n = g.tokens, r0 = g.rt * ROWS;
        // ---- queries: a power of two taken out of each row, laid out as B operands
        __syncthreads();
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
                const float down = exp_down(e);
                if (lane == 0) s_c[j] = a.scale * 1.4426950408889634f * exp_up(e);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    int mma, c, reg, half;
                    query_place<PREC>(lane * E + k, mma, c, reg, half);
                    const float y = x[i][k] * down;
                    const __half hi = __float2half_rn(y);
                    __half* q = reinterpret_cast<__half*>(s_q + ((mma * NT + j / 8) * NQ) * 32 + (j % 8) * 4 + c) + 2 * reg + half;
                    q[0] = hi;
                    if (NQ == 2) q[32 * 4] = __float2half_rn(y - __half2float(hi));
                }
            }
        }
        __syncthreads();
        float cf[NT][2], ref[NT][2], base_of[NT][2], sum[NT][2], o[NT][M][4];   // base_of: ref, or 0 before there is one
        int see[NT][2], see_all = n;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = 8 * t + 2 * lc + i;
                cf[t][i] = s_c[j];
                ref[t][i] = -INFINITY;
                base_of[t][i] = 0.0f;
                sum[t][i] = 0.0f;
                see[t][i] = r0 + j < R ? seen_by(a, g.b, n, (r0 + j) % a.S_q) : n;
                see_all = min(see_all, see[t][i]);
            }
        see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 1));
        see_all = min(see_all, __shfl_xor_sync(0xffffffffu, see_all, 2));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][m][i] = 0.0f;

        for (; st < end; st += W) {
            const bool more = st + W < end;
            const int next = more ? row_of(g, st + W) : -1;
            // ---- tokens that are there
            const int t0 = st * 16;
            const bool all = t0 + 16 <= see_all && (p16 ? row >= 0 : __all_sync(0xffffffffu, row >= 0));
            bool here[2] = {true, true};
            if (!all) {
                bool four[4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    here[i] = (p16 ? row : __shfl_sync(0xffffffffu, row, lg + 8 * i)) >= 0 && t0 + lg + 8 * i < n;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = 2 * lc + (i & 1) + 8 * (i >> 1);
                    four[i] = (p16 ? row : __shfl_sync(0xffffffffu, row, k)) >= 0 && t0 + k < n;
                }
                kt.only(here);
                vt.only(four, here);
            }
            // ---- scores
            // CH chains of dependent MMAs at a time: one would be as long as their latencies added up
            constexpr int CH = NT == 1 ? 4 : NT == 2 ? 2 : 1;
            float x[NT][4], acc[CH][NT][4];
#pragma unroll
            for (int h = 0; h < CH; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[h][t][i] = 0.0f;
            float k_factor[2] = {1.0f, 1.0f};
            auto qk = [&](const uint32_t (&f)[4], int m, int terms) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        if (q < terms) mma16816(acc[(m * NQ + q) % CH][t], f, s_q[((m * NT + t) * NQ + q) * 32 + lane]);
            };
            if constexpr (PREC == 1) {
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    const uint4 u = kt.x[0][j], v = kt.x[1][j];
                    const uint32_t f0[4] = {u.x, v.x, u.y, v.y}, f1[4] = {u.z, v.z, u.w, v.w};
                    qk(f0, 2 * j, NQ);
                    qk(f1, 2 * j + 1, NQ);
                }
            } else if constexpr (PREC == 2) {
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    const uint32_t u[4] = {kt.x[0][j].x, kt.x[0][j].y, kt.x[0][j].z, kt.x[0][j].w};
                    const uint32_t v[4] = {kt.x[1][j].x, kt.x[1][j].y, kt.x[1][j].z, kt.x[1][j].w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t p = u[w] ^ 0x80808080u, q = v[w] ^ 0x80808080u;
                        const uint32_t f[4] = {i8_pair(p, 0x4140), i8_pair(q, 0x4140), i8_pair(p, 0x4342), i8_pair(q, 0x4342)};
                        qk(f, 4 * j + w, NQ);
                    }
                }
                k_factor[0] = kt.s[0];
                k_factor[1] = kt.s[1];
            } else {
                uint32_t top = 0;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) top = max(top, __float_as_uint(kt.s[t][j]) & 0x7fffffffu);
                const int e = clamp_exp(__reduce_max_sync(0xffffffffu, top));
                const float down = exp_down(e);
                k_factor[0] = k_factor[1] = exp_up(e);
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    uint32_t r1[2], r2[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float y1, y2;
                        split_scale(kt.s[t][j] * down, y1, y2);
                        r1[t] = h2_pack(y1, y1);
                        r2[t] = h2_pack(y2, y2);
                    }
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        uint32_t p = w ? kt.x[0][j].y : kt.x[0][j].x, q = w ? kt.x[1][j].y : kt.x[1][j].x;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t f[4] = {i4_high(p), i4_high(q), i4_low(p), i4_low(q)};
                            const uint32_t f1[4] = {h2_mul(f[0], r1[0]), h2_mul(f[1], r1[1]), h2_mul(f[2], r1[0]), h2_mul(f[3], r1[1])};
                            const uint32_t f2[4] = {h2_mul(f[0], r2[0]), h2_mul(f[1], r2[1]), h2_mul(f[2], r2[0]), h2_mul(f[3], r2[1])};
                            qk(f1, 2 * (2 * j + w) + h, NQ);
                            qk(f2, 2 * (2 * j + w) + h, 1);
                            p >>= 8;
                            q >>= 8;
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[t][i] = acc[0][t][i];
#pragma unroll
                    for (int h = 1; h < CH; ++h) x[t][i] += acc[h][t][i];
                }
            int own[2];
            if (more) {
                k_rows(next, own);
                kt.load(place, own);
            }
            // ---- weights
            float v_add[2] = {0.0f, 0.0f}, v_mul[2] = {1.0f, 1.0f}, v_sum[2] = {1.0f, 1.0f};
            int ve[2] = {0, 0};
            if constexpr (PREC == 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ve[i] = clamp_exp(__float_as_uint(vt.s[i]) & 0x7fffffffu);
                    v_add[i] = (float)(ve[i] - 127);
                    v_sum[i] = __uint_as_float((uint32_t)(254 - ve[i]) << 23);   // 2^-(ve - 127)
                    v_mul[i] = vt.s[i] * v_sum[i];
                }
            } else if constexpr (PREC == 3) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t top = 0;
#pragma unroll
                    for (int j = 0; j < DP / 64; ++j) top = max(top, __float_as_uint(vt.own[i][j]) & 0x7fffffffu);
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    ve[i] = clamp_exp(top);
                    v_add[i] = (float)(ve[i] - 137);
                    v_sum[i] = exp_down(ve[i]);                                 // 2^-(ve - 137)
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
            uint2 p[NT][NP];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = i >> 1, col = i & 1;
                    const float y = fast_exp2(x[t][i] - base_of[t][col]);
                    sum[t][col] = PREC >= 2 ? fmaf(y, v_sum[tok], sum[t][col]) : sum[t][col] + y;
                    w[i] = PREC == 2 ? y * v_mul[tok] : y;
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
            auto pv = [&](const uint32_t (&f)[4], int m, int terms) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        if (q < terms) mma16816(o[t][m], f, p[t][q]);
            };
            if constexpr (PREC == 1) {
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    const uint32_t u[4][4] = {{vt.x[0][j].x, vt.x[0][j].y, vt.x[0][j].z, vt.x[0][j].w},
                                              {vt.x[1][j].x, vt.x[1][j].y, vt.x[1][j].z, vt.x[1][j].w},
                                              {vt.x[2][j].x, vt.x[2][j].y, vt.x[2][j].z, vt.x[2][j].w},
                                              {vt.x[3][j].x, vt.x[3][j].y, vt.x[3][j].z, vt.x[3][j].w}};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t f[4] = {__byte_perm(u[0][w], u[1][w], 0x5410), __byte_perm(u[0][w], u[1][w], 0x7632),
                                               __byte_perm(u[2][w], u[3][w], 0x5410), __byte_perm(u[2][w], u[3][w], 0x7632)};
                        pv(f, 4 * j + w, NP);
                    }
                }
            } else if constexpr (PREC == 2) {
#pragma unroll
                for (int w = 0; w < DP / 32; ++w) {
                    uint32_t y[2][2];   // [tokens low / high][values 0,1 / 2,3]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = word_of(vt.x[2 * h], w) ^ 0x80808080u, v = word_of(vt.x[2 * h + 1], w) ^ 0x80808080u;
                        y[h][0] = __byte_perm(u, v, 0x5140);
                        y[h][1] = __byte_perm(u, v, 0x7362);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t f[4] = {i8_pair(y[0][i], 0x4140), i8_pair(y[0][i], 0x4342),
                                               i8_pair(y[1][i], 0x4140), i8_pair(y[1][i], 0x4342)};
                        pv(f, 2 * w + i, NP);
                    }
                }
            } else {
                // the exponents of tokens 2c, 2c + 1 (+ 8) sit in lanes 4 (2c), 4 (2c + 1)
                uint32_t r1[2], r2[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float y1[2], y2[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int e = __shfl_sync(0xffffffffu, ve[h], 4 * (2 * lc + i));
                        split_scale(vt.s[2 * h + i] * exp_down(e), y1[i], y2[i]);
                    }
                    r1[h] = h2_pack(y1[0], y1[1]);
                    r2[h] = h2_pack(y2[0], y2[1]);
                }
#pragma unroll
                for (int w = 0; w < DP / 64; ++w)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t u = __byte_perm(word_of(vt.x[0], w), word_of(vt.x[1], w), i ? 0x7632 : 0x5410);
                        uint32_t v = __byte_perm(word_of(vt.x[2], w), word_of(vt.x[3], w), i ? 0x7632 : 0x5410);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t f[4] = {i4_high(u), i4_low(u), i4_high(v), i4_low(v)};
                            const uint32_t f1[4] = {h2_mul(f[0], r1[0]), h2_mul(f[1], r1[0]), h2_mul(f[2], r1[1]), h2_mul(f[3], r1[1])};
                            const uint32_t f2[4] = {h2_mul(f[0], r2[0]), h2_mul(f[1], r2[0]), h2_mul(f[2], r2[1]), h2_mul(f[3], r2[1])};
                            pv(f1, 4 * w + 2 * i + h, NP);
                            pv(f2, 4 * w + 2 * i + h, 1);
                            u >>= 8;
                            v >>= 8;
                        }
                    }
            }
            if (more) {
                int four[4];
                v_rows(next, four);
                vt.load(place, four, own);
            }
            row = next;
        }

        // ---- the warps' parts joined, while the next segment's first tiles load
        const bool another = at < s.hi;
        Segment following;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float l = sum[t][i];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                const int j = 8 * t + 2 * lc + i;
                if (lg == 0) {
                    s_ref[warp * ROWS + j] = ref[t][i];
                    s_sum[warp * ROWS + j] = l;
                }
                float* row = s_o + (warp * ROWS + j) * (DP + 4);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const int d = PREC == 1 ? 64 * (m / 4) + 8 * lg + 2 * (m % 4) : lg * (DP / 8) + 2 * m;
                    *reinterpret_cast<float2*>(row + d) = make_float2(o[t][m][i], o[t][m][i + 2]);
                }
            }
        if (another) following = open();
        __syncthreads();
        if (tid < ROWS) {
            float m = -INFINITY, l = 0.0f;
            for (int w = 0; w < W; ++w) m = fmaxf(m, s_ref[w * ROWS + tid]);
            const float r = m == -INFINITY ? 0.0f : m;
            for (int w = 0; w < W; ++w) {
                const float f = exp2f(s_ref[w * ROWS + tid] - r);
                s_w[w * ROWS + tid] = f;
                l += s_sum[w * ROWS + tid] * f;
            }
            s_c[tid] = m;
            s_l[tid] = l;
        }
        __syncthreads();
        float* part = slot_of(a, blockIdx.x, g.slot, ROWS);
#pragma unroll
        for (int i = tid; i < ROWS * DP / 4; i += THREADS) {
            const int j = i / (DP / 4), d = i % (DP / 4) * 4;
            if (r0 + j >= R || d >= D) continue;
            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(s_o + (w * ROWS + j) * (DP + 4) + d);
                const float f = s_w[w * ROWS + j];
                y[0] = fmaf(v.x, f, y[0]); y[1] = fmaf(v.y, f, y[1]); y[2] = fmaf(v.z, f, y[2]); y[3] = fmaf(v.w, f, y[3]);
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
        if (!g.whole) {
            if (tid < ROWS) {
                part[ROWS * D + tid] = s_c[tid];
                part[ROWS * D + ROWS + tid] = s_l[tid];
            }
            if (arrive(a, s, g)) join<ROWS, THREADS, 4, kMmaParts>(a, s, g, R, s_o, out_vec);
        }
        if (!another) break;
        g = following;
    }
}

// CTAs an SM: what their registers allow.
template <int PREC, int DP, int NT, int NQ, int NP>
int launch_mma(const skv_pool_attention_args& a, cudaStream_t st) {
    constexpr int W = NT == 1 && PREC >= 2 ? 8 : 4;
    constexpr int CTAS = NT >= 4 ? 2 : NT == 2 ? 3 : PREC == 1 ? 3 : 2;
    static_assert(CTAS * 2 * 8 * NT <= kRowsPerSm, "the scratch holds every CTA's slots");
    constexpr size_t smem = mma_smem<DP, NT, NQ, W>();
    const auto kernel = pool_attention_mma_kernel<PREC, DP, NT, NQ, NP, W, CTAS>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
    }
    const int R = a.q.heads / a.pool.heads * a.S_q;
    PageDivide magic;
    magic.shift = 31;
    while ((1ll << (magic.shift - 31)) < a.pool.page_size) ++magic.shift;
    magic.mul = (uint32_t)(((1ull << magic.shift) + a.pool.page_size - 1) / a.pool.page_size);
    kernel<<<sm_count() * CTAS, 32 * W, smem, st>>>(a, (R + 8 * NT - 1) / (8 * NT), magic, rows_aligned(a.q), rows_aligned(a.out));
    return check_launch("pool_attention");
}

template <int PREC, int DP, int NT>
int launch_mma_type(const skv_pool_attention_args& a, cudaStream_t st) {
    if (a.q.dtype == kF32) return launch_mma<PREC, DP, NT, 2, 2>(a, st);
    if (a.q.dtype == kF16) return launch_mma<PREC, DP, NT, 1, 2>(a, st);
    return launch_mma<PREC, DP, NT, 1, 1>(a, st);
}

// Row tiles of 8, 16 or 32 rows: the pages are read once for up to 32 rows of a key head.
template <int PREC>
int launch_mma_prec(const skv_pool_attention_args& a, cudaStream_t st) {
    const int R = a.q.heads / a.pool.heads * a.S_q;
    if (a.pool.head_dim <= 64) {
        if (R <= 8) return launch_mma_type<PREC, 64, 1>(a, st);
        return R <= 16 ? launch_mma_type<PREC, 64, 2>(a, st) : launch_mma_type<PREC, 64, 4>(a, st);
    }
    if (R <= 8) return launch_mma_type<PREC, 128, 1>(a, st);
    return R <= 16 ? launch_mma_type<PREC, 128, 2>(a, st) : launch_mma_type<PREC, 128, 4>(a, st);
}

}  // namespace skv
