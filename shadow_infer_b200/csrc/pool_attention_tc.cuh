// Attention over the page pool for many query rows a key head: blocks of new tokens and whole prompts.
//
// A few query rows leave tcgen05 idle (pool_attention_mma.cuh), 128 fill it: a unit is (sequence, key head, 128 query rows), and
//     S [128 rows x 128 tokens] = Q K^T,     O [128 rows x D] += P V     (int4 pages: 64 tokens)
// run as tcgen05.mma with the sums in TMEM.  Where a head has 128 new tokens or more a unit's rows are neighbours of one head, and
// with a causal limit the unit ends at the last token that its rows see: the shares count each unit's own tiles, by a closed
// form, so a prompt costs its triangle.
//
// A CTA is a pipeline of two roles:
//     warps 0-3   softmax, a query row a thread (TMEM lane): S from TMEM, the running maximum (moved lazily), weights P as fp16
//                 back into TMEM over S's first columns; O read, divided and stored, or published for the join, at a unit's end.
//                 They also lay out Q once a unit (a power of two taken out of each row).  Thread 0 issues the MMAs in between (they are on this role's path in any case, so a warp for them would
//                 only take registers: 256 threads leave two CTAs 128 each, with 96 the softmax spilled);
//     warps 4-7   each tile's page rows: fp16 copied, int8 made fp16 integers (exact), int4 fp16 values in two parts (so its
//                 tiles have 64 tokens, in the same memory), in the swizzled layout that the tensor cores read, and what a token's scales do to scores and weights; they run ahead across units.
// Two CTAs share an SM (TMEM: 128 columns of S and P, 128 of O each), so that one's MMAs run during the other's softmax.  Heads
// of more than 128 values leave room for one.
//
// What bounds it: instructions and the chain S -> softmax -> P V of two CTAs; a tile of int8 pages takes 10 thousand warp
// instructions (41 % of the issue slots; tensor pipe 20 %, exponentials 21 % busy).  8 key heads of 4 query heads of 128 values: a prompt of 4096 fp16 tokens in 303 us (453 TFLOP/s of the
// causal half's operations, 0.27 of cuBLAS's burst), int8 383 us, int4 541 us; 128 new tokens behind 16384 in 84, 101 and 135 us
// (bf16; fp16 queries 5 to 11 % more).
// Measured and dropped: a warp of its own for the MMAs (96 registers a thread: spills, twice the time), weights of all
// 128 columns in registers until the maximum is known (spills), the next 32 scores fetched ahead (spills, 15 % slower).
//
// Numbers: as in pool_attention_mma.cuh.  Page values and queries are exact in fp16, an int8 row's scale multiplies its scores (K)
// and weights (V) in fp32, int4 values are two operands (18 bits).  A weight of at most 2^15 is one fp16 operand for bf16 outputs,
// whose own rounding is 8 times coarser, else two (with one, fp16 outputs were up to twice as far off as rounding alone).
//
// Every wait is bounded: after a second without progress the roles leave, TMEM is freed and the outputs are NaN.
#pragma once

#include <atomic>
#include <mutex>

#include "pool_attention.cuh"
#include "sm100_ptx.cuh"

namespace skv {

constexpr int kTcRows = 128, kTcThreads = 256, kTcPad = 1, kTcOddWords = 8;
// A fresh maximum's weight is 2^10 to 2^11 and may grow to 2^15: with one fp16 operand a weight, its subnormals' 2^-25 is then
// 2^-35 of the largest weight.
constexpr float kTcDrop = 11.0f, kTcRoom = 14.0f;

// Tokens a tile: an int4 value takes two operands, so its tiles are half as long.
__host__ __device__ constexpr int tc_tile(int precision) { return precision == 3 ? 64 : 128; }

// The units of a sequence and key head, and what each costs.
template <int TILE>
struct TcUnits {
    static constexpr int STEP = kTcRows / TILE;   // tiles that a block sees more than the one before
    int S_q, rep, blocks, row_tiles;   // blocks: of 128 new tokens of a head (0: a unit's rows are any heads' and tokens')
    bool causal;
    __device__ __forceinline__ TcUnits(const skv_pool_attention_args& a)
        : S_q(a.S_q), rep(a.q.heads / a.pool.heads), blocks(a.S_q >= kTcRows ? (a.S_q + kTcRows - 1) / kTcRows : 0),
          row_tiles(blocks ? rep * blocks : (rep * a.S_q + kTcRows - 1) / kTcRows), causal(a.causal && blocks) {}
    // With n tiles and `past` tiles before the new tokens, block i sees past + (i + 1) STEP tiles, at least one and no more than n.
    __device__ __forceinline__ int tiles(int i, int n, int past) const { return causal ? min(max(past + (i + 1) * STEP, 1), n) : n; }
    // What blocks [0, k) cost.
    __device__ __forceinline__ int before(int k, int n, int past, int pad) const {
        if (!causal) return k * (n + pad);
        const int lo = min(max(-past, 0) / STEP, k), hi = min(max((n - past) / STEP, lo), k);   // blocks below lo see one tile, from hi on n
        return lo + (hi - lo) * past + STEP * (hi * (hi + 1) - lo * (lo + 1)) / 2 + (k - hi) * n + k * pad;
    }
    __device__ __forceinline__ void sequence(const skv_pool_attention_args& a, int b, int& tokens, int& n, int& past) const {
        tokens = seq_tokens(a, b);
        n = seq_tiles(tokens, TILE);
        const int old = tokens - (a.new_lengths ? __ldg(a.new_lengths + b) : S_q);
        past = old >= 0 ? (old + TILE - 1) / TILE : -((-old) / TILE);
    }
    __device__ __forceinline__ int a_head(int n, int past, int pad) const {   // a key head's units
        return blocks ? rep * before(blocks, n, past, pad) : row_tiles * (n + pad);
    }
};

struct TcSegment : Segment {
    int r0, rows;   // the unit's query rows
};

template <int TILE>
__device__ __forceinline__ TcSegment tc_segment_at(const skv_pool_attention_args& a, const TcUnits<TILE>& u, const Share& s, int at, int& b,
                                                   int& base) {
    TcSegment g;
    for (;;) {
        int n, past;
        u.sequence(a, b, g.tokens, n, past);
        const int each = u.a_head(n, past, s.pad);
        if (at >= base + each * a.pool.heads) {
            base += each * a.pool.heads;
            ++b;
            continue;
        }
        g.b = b;
        g.hk = (at - base) / each;
        g.first = base + g.hk * each;
        int nt = n;
        if (u.blocks) {
            const int head = each / u.rep, h = (at - g.first) / head;
            g.first += h * head;
            int i = 0, end = u.blocks;   // the block that holds `at`
            while (end - i > 1) {
                const int m = (i + end) / 2;
                if (g.first + u.before(m, n, past, s.pad) <= at) i = m;
                else end = m;
            }
            nt = u.tiles(i, n, past);
            g.first += u.before(i, n, past, s.pad);
            g.rt = h * u.blocks + i;
            g.r0 = h * u.S_q + i * kTcRows;
            g.rows = min(kTcRows, u.S_q - i * kTcRows);
        } else {
            g.rt = (at - g.first) / (n + s.pad);
            g.first += g.rt * (n + s.pad);
            g.r0 = g.rt * kTcRows;
            g.rows = min(kTcRows, u.rep * u.S_q - g.r0);
        }
        g.last = g.first + nt - 1;
        g.t0 = at - g.first;
        g.next = min(g.first + nt + s.pad, s.hi);
        g.t1 = min(nt, g.next - g.first);
        g.whole = g.t0 == 0 && g.t1 == nt;
        g.slot = at == s.lo ? 0 : 1;
        if (a.error_flag && a.lengths[b] != g.tokens && threadIdx.x == 0) atomicExch(a.error_flag, 1);
        return g;
    }
}

// Shared memory of a CTA.
template <int DP>
struct TcLayout {
    static constexpr int TILE = DP / 64 * 128 * 128;   // atoms of 128 rows of 64 values
    static constexpr int PART = TILE / 2;              // of a tile of 64 tokens whose values have two parts
    static constexpr int Q = 0, K = TILE, V = 2 * TILE;
    static constexpr int TOKENS = 3 * TILE;            // [2][4][128] of a tile's tokens: score factor, score term, weight factor, 1 / sum factor
    static constexpr int CTAS = DP > 128 ? 1 : 2, COLUMNS = DP > 128 ? 512 : 256;   // on an SM; of TMEM (128 for S, DP for O)
    static constexpr int BARS = TOKENS + 2 * 4 * 128 * 4;
    static constexpr int BYTES = BARS + 80, ALLOC = BYTES + 1024;   // tiles start on 1024-byte boundaries
};

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }   // warps 0 to 3
__device__ __forceinline__ float tc_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 32 lanes x 16 consecutive 32-bit columns: thread t of the warp gets lane (base_lane + t).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ uint32_t tc_pack(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Bytes n + 128 as fp16 n: 1024 + b has b in its low bits.
__device__ __forceinline__ uint32_t tc_i8_pair(uint32_t biased, uint32_t sel) {
    const uint32_t x = __byte_perm(biased, 0x64646464u, sel), c = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// NP: fp16 operands of a weight.
template <int PREC, int DP, int NP>
__global__ void __launch_bounds__(kTcThreads, TcLayout<DP>::CTAS) pool_attention_tc_kernel(const __grid_constant__ skv_pool_attention_args a, bool out_vec) {
    using namespace sm100;
    using L = TcLayout<DP>;
    extern __shared__ uint8_t tc_raw[];
    __shared__ Share s;
    __shared__ uint32_t s_tmem;
    __shared__ int s_error, s_late;
    __shared__ uint32_t s_odd[kTcOddWords];   // a bit a unit (of its number's last ones): values of it that are not finite were left out
    __shared__ __align__(16) int s_gap[2][4];   // whether the tile misses a token of the sequence, by the warp that looked it up
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    float* s_tokens = reinterpret_cast<float*>(sm + L::TOKENS);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BARS);
    uint64_t *k_full = bars, *k_free = bars + 2, *v_full = bars + 3, *v_free = bars + 4, *s_full = bars + 5, *o_full = bars + 6,
             *drained = bars + 7;   // k_full: of even and of odd tiles (the softmax may look when the next is full)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = a.pool.head_dim, P = a.pool.page_size, rep = a.q.heads / a.pool.heads;
    constexpr int TILE = tc_tile(PREC), PARTS = 128 / TILE;   // operands a value
    constexpr int COLUMNS = 16 * NP;                           // of P for 32 of S
    const TcUnits<TILE> u(a);
    if (tid == 0) {
        mbar_init(k_full, 4);
        mbar_init(k_full + 1, 4);
        mbar_init(k_free, 1);
        mbar_init(v_full, 4);
        mbar_init(v_free, 1);
        mbar_init(s_full, 1);
        mbar_init(o_full, 1);
        mbar_init(drained, 1);
        fence_mbarrier_init();
        s_error = s_late = 0;
        for (int i = 0; i < kTcOddWords; ++i) s_odd[i] = 0;
    }
    take_share<kTcThreads>(a, [&](int b) {
        int tokens, n, past;
        u.sequence(a, b, tokens, n, past);
        return u.a_head(n, past, kTcPad) * a.pool.heads;
    }, kTcPad, 1, &s);
    if (s.lo >= s.hi) return;
    if (warp == 0) {
        tmem_alloc(&s_tmem, L::COLUMNS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    int at = s.lo, b = s.b, base = s.base;
    int g = 0;      // tiles so far: the barriers complete once a tile (k_full: every second, o_full: once a unit)
    int units = 0;  // units so far
    bool ok = true;
    // the first token of the tiles that not all rows of a unit see (or an earlier one where the rows are of several heads)
    auto odd_from = [&](const TcSegment& sg) {
        const int new_before = u.blocks ? sg.rt % u.blocks * kTcRows : 0;
        const int old = sg.tokens - (a.new_lengths ? __ldg(a.new_lengths + sg.b) : a.S_q);
        return not_all_from(a.causal ? max(1, old + 1 + new_before) : sg.tokens, sg.tokens, TILE);
    };

    if (warp < 4) {
        // ------------------------------------------------------------------- softmax, and the MMAs
        const uint32_t t_s = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_s + 128;
        const uint32_t k_tile = smem_u32(sm + L::K), v_tile = smem_u32(sm + L::V), q_tile = smem_u32(sm + L::Q);
        bool issued = false;
        for (; at < s.hi;) {
            const TcSegment sg = tc_segment_at(a, u, s, at, b, base);
            at = sg.next;
            if (sg.t0 >= sg.t1) continue;
            const int r = sg.r0 + tid;
            const int see = tid < sg.rows ? seen_by(a, sg.b, sg.tokens, r % a.S_q) : 0;
            const int see_min = __reduce_min_sync(0xffffffffu, tid < sg.rows ? see : 0x7fffffff);
            float ref = -INFINITY, base_of = 0.0f, l = 0.0f, c_row = 0.0f;
            {   // a power of two taken out of the row (the MMAs of the unit before, which read Q, are done: O was)
                const bool have = tid < sg.rows;
                const uint16_t* from = have ? row_ptr<const uint16_t>(a.q, a.S_q, rep, sg.b, sg.hk, r) : nullptr;
                uint4 q[DP / 8];
#pragma unroll
                for (int i = 0; i < DP / 8; ++i)
                    q[i] = have && i * 8 < D ? __ldg(reinterpret_cast<const uint4*>(from) + i) : make_uint4(0, 0, 0, 0);
                // the largest magnitude by its bits (a NaN is left to the score); it goes to [2^10, 2^11)
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = max(max(top, w[e] & 0x7fffu), w[e] >> 16 & 0x7fffu);
                }
                const bool half = a.q.dtype == kF16;
                const float most = half ? __half2float(__ushort_as_half((unsigned short)top)) : __uint_as_float(top << 16);
                const int e2 = min(max((int)(__float_as_uint(most) >> 23), 35), 219);
                const float down = __uint_as_float((uint32_t)(264 - e2) << 23);
                c_row = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(e2 - 10) << 23);
                uint8_t* to = sm + L::Q;
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
                    if (half) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                            w[e] = tc_pack(f.x * down, f.y * down);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = tc_pack(__uint_as_float(w[e] << 16) * down, __uint_as_float(w[e] & 0xffff0000u) * down);
                    }
                    *reinterpret_cast<uint4*>(to + i / 8 * 128 * 128 + sw128_offset(tid, i % 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            fence_proxy_async_smem();
            softmax_sync();
            for (int t = sg.t0; t < sg.t1; ++t, ++g) {
                if (tid == 0 && ok && mbar_wait_spin(k_full + (g & 1), g >> 1 & 1, &s_error, 1)) {
                    tc_fence_after();
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i) {
                            const uint32_t in = (i & 3) * 32, atom = i >> 2;
                            umma_f16(tmem, smem_desc_sw128(q_tile + atom * (128 * 128) + in, 16, 1024),
                                     smem_desc_sw128(k_tile + part * L::PART + atom * (TILE * 128) + in, 16, 1024),
                                     idesc_f16_f32(128, TILE, false, false), part + i > 0);
                        }
                    umma_commit(s_full);
                    umma_commit(k_free);
                    issued = true;
                }
                __syncwarp();
                // (k_full has completed before s_full: this makes the producers' plain stores visible here)
                ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(s_full, g & 1, &s_error, 2) &&
                                                       mbar_wait_spin(k_full + (g & 1), g >> 1 & 1, &s_error, 3));
                tc_fence_after();
                const float* tk = s_tokens + (g & 1) * 4 * 128;
                const int left = see - t * TILE;   // columns that this row sees
                const int4 gaps = *reinterpret_cast<const int4*>(s_gap[g & 1]);
                const bool masked = see_min - t * TILE < TILE, gap = gaps.x | gaps.y | gaps.z | gaps.w;
                // 32 columns at a time.  The reference is an integer that moves only where a weight would grow too large; what the
                // old one scaled (O, the sum, the columns before) is a power of two off, which is exact.  (O holds the tiles
                // before: s_full says that their MMAs are done.  P's columns replace S's that have been read.)
#pragma unroll 1
                for (int c = 0; c < TILE / 32 && ok; ++c) {
                    float y[32];
                    {
                        uint32_t x[32];
                        tmem_ld32(t_s + c * 32, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            if constexpr (PREC >= 2) {
                                const float4 k = *reinterpret_cast<const float4*>(tk + c * 32 + i);
                                const float4 add = *reinterpret_cast<const float4*>(tk + 128 + c * 32 + i);
                                y[i] = fmaf(__uint_as_float(x[i]), k.x * c_row, add.x);
                                y[i + 1] = fmaf(__uint_as_float(x[i + 1]), k.y * c_row, add.y);
                                y[i + 2] = fmaf(__uint_as_float(x[i + 2]), k.z * c_row, add.z);
                                y[i + 3] = fmaf(__uint_as_float(x[i + 3]), k.w * c_row, add.w);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e) y[i + e] = __uint_as_float(x[i + e]) * c_row;
                            }
                        }
                    }
                    if (masked) {
                        const int there = left - c * 32;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i >= there) y[i] = -INFINITY;
                    }
                    if (gap) {
#pragma unroll 1
                        for (int i = 0; i < 32; i += 8)
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e / 8 * 8 == i && tk[128 + c * 32 + e] == -INFINITY) y[e] = -INFINITY;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], y[i]);
                    const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    if (__any_sync(0xffffffffu, high > ref + kTcRoom)) {
                        const float now = fmaxf(ref, ceilf(high - kTcDrop)), f = now == -INFINITY ? 1.0f : tc_exp2(ref - now);
                        ref = now;
                        base_of = now == -INFINITY ? 0.0f : now;
                        l *= f;
                        if (t > sg.t0) {
#pragma unroll 1
                            for (int d = 0; d < DP / 32; ++d) {
                                uint32_t o[32];
                                tmem_ld32(t_o + d * 32, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tmem_st32(t_o + d * 32, o);
                            }
                        }
#pragma unroll 1
                        for (int d = 0; d < c * NP; ++d) {
                            uint32_t w[16];
                            tmem_wait_st();
                            tmem_ld16(t_s + d * 16, w);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));   // (f may be below fp16's range)
                                w[i] = tc_pack(z.x * f, z.y * f);
                            }
                            tmem_st16(t_s + d * 16, w);
                        }
                    }
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint32_t p[16], rest[NP == 2 ? 16 : 1];
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[i + e] = tc_exp2(y[i + e] - base_of);
                        if constexpr (PREC >= 2) {
                            const float4 w = *reinterpret_cast<const float4*>(tk + 384 + c * 32 + i);
                            sum[0] = fmaf(y[i], w.x, sum[0]);
                            sum[1] = fmaf(y[i + 1], w.y, sum[1]);
                            sum[2] = fmaf(y[i + 2], w.z, sum[2]);
                            sum[3] = fmaf(y[i + 3], w.w, sum[3]);
                            if constexpr (PREC == 2) {
                                const float4 v = *reinterpret_cast<const float4*>(tk + 256 + c * 32 + i);
                                y[i] *= v.x; y[i + 1] *= v.y; y[i + 2] *= v.z; y[i + 3] *= v.w;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[e] += y[i + e];
                        }
                        p[i / 2] = tc_pack(y[i], y[i + 1]);
                        p[i / 2 + 1] = tc_pack(y[i + 2], y[i + 3]);
                        if constexpr (NP == 2) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[i / 2 + e]));
                                rest[i / 2 + e] = tc_pack(y[i + 2 * e] - f.x, y[i + 2 * e + 1] - f.y);
                            }
                        }
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st16(t_s + c * COLUMNS, p);
                    if constexpr (NP == 2) tmem_st16(t_s + c * COLUMNS + 16, rest);
                }
                tmem_wait_st();
                tc_fence_before();
                softmax_sync();
                if (tid == 0 && ok && mbar_wait_spin(v_full, g & 1, &s_error, 4)) {
                    tc_fence_after();
#pragma unroll
                    for (int w = 0; w < NP; ++w)
#pragma unroll
                        for (int part = 0; part < PARTS; ++part) {
                            if (w + part > 1) continue;   // the small part of a value and the rest of a weight
#pragma unroll
                            for (int i = 0; i < TILE / 16; ++i)
                                umma_f16_ts(tmem + 128, tmem + i / 2 * COLUMNS + i % 2 * 8 + w * 16,
                                            smem_desc_sw128(v_tile + part * L::PART + i * 16 * 128, TILE * 128, 1024),
                                            idesc_f16_f32(128, DP, false, true), t > sg.t0 || w + part + i > 0);
                        }
                    umma_commit(v_free);
                    if (t + 1 == sg.t1) umma_commit(o_full);
                }
                __syncwarp();
            }
            // ------------------------------------------------------------------------ the unit's end
            ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(o_full, units & 1, &s_error, 5));
            ++units;
            tc_fence_after();
            float* part = slot_of(a, blockIdx.x, sg.slot, kTcRows);
            const float nan = __int_as_float(0x7fc00000);
            const float mul = !ok ? nan : !sg.whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + c * 32, o);
                tmem_wait_ld();
                float y[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = l == 0.0f && ok ? 0.0f : __uint_as_float(o[i]) * mul;
                if (tid < sg.rows) {
                    if (!sg.whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (c * 32 + i < D) *reinterpret_cast<float4*>(part + tid * D + c * 32 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                    } else if (out_vec) {   // 16 bytes a store
                        uint4* to = reinterpret_cast<uint4*>(row_ptr<uint16_t>(a.out, a.S_q, rep, sg.b, sg.hk, r) + c * 32);
                        uint32_t w[16];
                        if (a.out.dtype == kF16) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) w[i] = tc_pack(y[2 * i], y[2 * i + 1]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const __nv_bfloat162 z = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                                w[i] = *reinterpret_cast<const uint32_t*>(&z);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (c * 32 + i * 8 < D) to[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (c * 32 + i < D) {
                                const float one[1] = {y[i]};
                                store_out<1>(a, sg.b, sg.hk, r, c * 32 + i, one);
                            }
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
            if (!sg.whole && tid < sg.rows) {
                part[kTcRows * D + tid] = ref;
                part[kTcRows * D + kTcRows + tid] = ok ? l : nan;
            }
        }
        if (tid == 0 && issued) {   // every MMA has completed before TMEM is freed
            umma_commit(drained);
            mbar_wait_spin(drained, 0, &s_late, 6);   // (also after an error elsewhere, so not with s_error)
        }
        __syncwarp();
        // What was left out, unit by unit.  (Thread 0 has waited for all values, so what the other warps noted of them is here, and so
        // are the outputs, behind this barrier.  In the loop above the call would cost it 2 %, for the registers it takes.)
        softmax_sync();
        uint32_t any = 0;
        for (int i = 0; i < kTcOddWords; ++i) any |= s_odd[i];
        if (any) {
            at = s.lo;
            b = s.b;
            base = s.base;
            units = 0;
            while (at < s.hi) {
                const TcSegment sg = tc_segment_at(a, u, s, at, b, base);
                at = sg.next;
                if (sg.t0 >= sg.t1) continue;
                if (s_odd[units / 32 % kTcOddWords] >> (units % 32) & 1) {
                    const int first = sg.t0 * TILE;
                    add_not_finite<PREC>(a, sg.b, sg.hk, sg.tokens, sg.r0, sg.rows, PREC == 3 ? first : max(first, odd_from(sg)),
                                         min(sg.tokens, sg.t1 * TILE), sg.whole ? nullptr : slot_of(a, blockIdx.x, sg.slot, kTcRows), tid, 128);
                }
                ++units;
            }
        }
    } else {
        // ------------------------------------------------------------------------- pages and queries
        const int pw = warp - 4;
        constexpr int VALUES = PREC == 1 ? 8 : PREC == 2 ? 16 : 32;   // of a 16-byte chunk
        constexpr int CHUNKS = DP / VALUES, ROWS = TILE / 4;          // chunks of a row, rows that a warp has of a tile
        constexpr int STEP = 32 / CHUNKS, N = ROWS / STEP;            // rows that it takes at a time
        const int my_chunk = lane % CHUNKS, my_row = lane / CHUNKS;
        const bool have_chunk = my_chunk * VALUES < D;
        const int row_bytes = D / VALUES * 16;
        const int groups = PREC == 3 ? D / a.pool.int4_group : 1;
        const int block0 = PREC == 3 ? my_chunk * 32 / a.pool.int4_group : 0, block1 = PREC == 3 ? (my_chunk * 32 + 16) / a.pool.int4_group : 0;
        // int8, int4: the next tile's chunks, and int4's scales of their halves, on their way
        struct Ahead {
            uint4 raw[PREC >= 2 ? N : 1];
            float scale[PREC == 3 ? N : 1][2];
            // the exponent field of the largest of row i's scales
            __device__ __forceinline__ int exponent(int i) const {
                uint32_t top = max(__float_as_uint(scale[i][0]) & 0x7fffffffu, __float_as_uint(scale[i][1]) & 0x7fffffffu);
#pragma unroll
                for (int w = 1; w < CHUNKS; w <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
                return min(max((int)(top >> 23), 35), 219);
            }
        } k_next, v_next;
        auto load = [&](Ahead& next, const void* pages, const float* scales, int row) {
            if constexpr (PREC >= 2) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int x = __shfl_sync(0xffffffffu, row, i * STEP + my_row);
                    const bool there = x >= 0 && have_chunk;
                    next.raw[i] = make_uint4(0, 0, 0, 0);
                    if (there)
                        next.raw[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(pages) + (int64_t)x * row_bytes + my_chunk * 16));
                    if constexpr (PREC == 3) {
                        next.scale[i][0] = there ? __ldg(scales + (int64_t)x * groups + block0) : 0.0f;
                        next.scale[i][1] = there ? __ldg(scales + (int64_t)x * groups + block1) : 0.0f;
                    }
                }
            }
        };
        auto write = [&](const Ahead& next, uint8_t* tile) {
            if constexpr (PREC == 3) {
                // A value is its integer times its scale (a power of two a token taken out), in two parts: times the scale's first 7
                // bits, which is exact, and times the rest, rounded at 2^-18 of the value.  A byte becomes
                // 1024 + 16 (n + 8) of its high nibble and 1024 + (n + 8) of its low one, and one exact fma both n.  Four chunks
                // of an atom, the order exchanged for every second one (banks).
                const int atom = my_chunk / 2, swap = atom & 1, c = my_chunk % 2 * 4;
                const __half2 by = __floats2half2_rn(0.0625f, 1.0f), add = __floats2half2_rn(-72.0f, -1032.0f);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int x = pw * ROWS + i * STEP + my_row;
                    const float down = __uint_as_float((uint32_t)(262 - next.exponent(i)) << 23);   // the largest scale to [2^8, 2^9)
                    const uint32_t w[4] = {next.raw[i].x, next.raw[i].y, next.raw[i].z, next.raw[i].w};
                    __half2 y[4][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t z = (__byte_perm(w[j], 0, 0x4040 + 0x0101 * e) & 0x000F00F0u) | 0x64006400u;
                            y[j][e] = __hfma2(*reinterpret_cast<const __half2*>(&z), by, add);
                        }
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        __half2 f[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float scale = next.scale[i][h] * down;
                            const float first = __uint_as_float((__float_as_uint(scale) + 0x10000u) & 0xFFFE0000u);
                            f[h] = __float2half2_rn(part == 0 ? first : scale - first);
                        }
                        uint8_t* line = tile + part * L::PART + atom * TILE * 128;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t r[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const __half2 one = __hmul2(y[j][e], f[j / 2]), other = __hmul2(y[j ^ 2][e], f[1 - j / 2]);
                                r[e] = swap ? *reinterpret_cast<const uint32_t*>(&other) : *reinterpret_cast<const uint32_t*>(&one);
                            }
                            *reinterpret_cast<uint4*>(line + sw128_offset(x, c + (swap ? j ^ 2 : j))) = make_uint4(r[0], r[1], r[2], r[3]);
                        }
                    }
                }
            }
            if constexpr (PREC == 2) {   // 16 values: two chunks of an atom, exchanged for every second atom (banks)
                const int atom = my_chunk / 4, swap = atom & 1, c = my_chunk % 4 * 2;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int x = pw * ROWS + i * STEP + my_row;
                    const uint4 raw = next.raw[i];
                    const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
                    const uint4 lo = make_uint4(tc_i8_pair(w[0], 0x4140), tc_i8_pair(w[0], 0x4342), tc_i8_pair(w[1], 0x4140), tc_i8_pair(w[1], 0x4342));
                    const uint4 hi = make_uint4(tc_i8_pair(w[2], 0x4140), tc_i8_pair(w[2], 0x4342), tc_i8_pair(w[3], 0x4140), tc_i8_pair(w[3], 0x4342));
                    uint8_t* line = tile + atom * 128 * 128;
                    *reinterpret_cast<uint4*>(line + sw128_offset(x, c + swap)) = swap ? hi : lo;
                    *reinterpret_cast<uint4*>(line + sw128_offset(x, c + 1 - swap)) = swap ? lo : hi;
                }
            }
        };
        auto copy = [&](uint8_t* tile, const void* pages, int row) {
            if constexpr (PREC == 1) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int x = __shfl_sync(0xffffffffu, row, i * STEP + my_row);
                    const uint32_t to = smem_u32(tile + my_chunk / 8 * 128 * 128 + sw128_offset(pw * ROWS + i * STEP + my_row, my_chunk % 8));
                    const bool there = x >= 0 && have_chunk;
                    const char* from = static_cast<const char*>(pages) + (there ? (int64_t)x * row_bytes + my_chunk * 16 : 0);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
                }
            }
        };
        auto note = [&]() { atomicOr(&s_odd[units / 32 % kTcOddWords], 1u << (units % 32)); };
        // Whether one of a tile's fp16 values is not finite: looked at while the tile before is still multiplied.  (A prompt of 4096 tokens
        // 296 -> 302 us; on their way to the tile, or in shared memory behind it, 302 to 305.)
        auto any_odd = [&](const void* pages, int row) -> bool {
            uint32_t out = 0;
            if constexpr (PREC == 1) {
#pragma unroll 8
                for (int i = 0; i < N; ++i) {
                    const int x = __shfl_sync(0xffffffffu, row, i * STEP + my_row);
                    if (x >= 0 && have_chunk) out |= odd_halves(__ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(pages) + (int64_t)x * row_bytes + my_chunk * 16)));
                }
            }
            return __any_sync(0xffffffffu, out != 0);
        };
        // Zeros for them, in the chunks that this lane copied.
        auto clean = [&](uint8_t* tile) {
#pragma unroll 1
            for (int i = 0; i < N; ++i) {
                uint4* x = reinterpret_cast<uint4*>(tile + my_chunk / 8 * 128 * 128 + sw128_offset(pw * ROWS + i * STEP + my_row, my_chunk % 8));
                *x = finite_halves(*x);
            }
            note();
        };
        auto publish = [&](uint64_t* full) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
        };
        for (; ok && at < s.hi;) {
            const TcSegment sg = tc_segment_at(a, u, s, at, b, base);
            at = sg.next;
            if (sg.t0 >= sg.t1) continue;
            // the pool row of token lane % ROWS of this warp's ROWS of a tile, -1 where there is none
            bool gap;
            auto row_of = [&](int t) -> int {
                const int tok = t * TILE + pw * ROWS + lane % ROWS;
                gap = false;
                if (t >= sg.t1 || tok >= sg.tokens) return -1;
                const int64_t row = pool_row(a.pool, sg.b, tok);
                if (row < 0 && a.error_flag) atomicExch(a.error_flag, 1);
                gap = row < 0;
                return row < 0 ? -1 : (int)row + sg.hk * P;
            };
            const int odd = odd_from(sg);
            int row = row_of(sg.t0);
            load(k_next, a.pool.k, a.pool.scale_k, row);
            load(v_next, a.pool.v, a.pool.scale_v, row);
            for (int t = sg.t0; t < sg.t1; ++t, ++g) {
                float* tk = s_tokens + (g & 1) * 4 * 128 + pw * ROWS + lane % ROWS;
                float sk = 0.0f, sv = 1.0f;
                if (PREC == 2 && row >= 0) {
                    sk = __ldg(a.pool.scale_k + row);
                    sv = __ldg(a.pool.scale_v + row);
                }
                const bool any_gap = __any_sync(0xffffffffu, gap);
                const int next = row_of(t + 1);
                // the scores of the tile before are done: K is free, and what the softmax of the tile before that read
                if (g > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(k_free, (g - 1) & 1, &s_error, 7));
                if (!ok) break;
                write(k_next, sm + L::K);
                copy(sm + L::K, a.pool.k, row);
                if constexpr (PREC == 2) {   // V's scale as a power of two in the exponent and a factor in [1, 2)
                    const bool out = t * TILE >= odd && !finite(sv);
                    if (out) {
                        sv = 1.0f;
                        note();
                    }
                    const int e = min(max((int)((__float_as_uint(sv) & 0x7fffffffu) >> 23), 35), 219);
                    const float down = __uint_as_float((uint32_t)(254 - e) << 23);
                    tk[0] = sk;
                    tk[128] = row >= 0 ? (float)(e - 127) : -INFINITY;
                    tk[256] = out ? 0.0f : sv * down;
                    tk[384] = down;
                } else if constexpr (PREC == 3) {   // of the rows that this lane took, by the first lane of each
                    bool out = false;
#pragma unroll
                    for (int i = 0; i < 2 * N; ++i) out |= !finite(v_next.scale[i / 2][i % 2]);
                    if (out) {   // a group that is not finite says nothing of the others' size
#pragma unroll
                        for (int i = 0; i < 2 * N; ++i)
                            if (!finite(v_next.scale[i / 2][i % 2])) v_next.scale[i / 2][i % 2] = 0.0f;
                        note();
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int ek = k_next.exponent(i), ev = v_next.exponent(i), x = i * STEP + my_row;
                        const bool there = __shfl_sync(0xffffffffu, row, x) >= 0;
                        float* of = s_tokens + (g & 1) * 4 * 128 + pw * ROWS + x;
                        if (my_chunk == 0) {
                            of[0] = __uint_as_float((uint32_t)(ek - 8) << 23);
                            of[128] = there ? (float)(ev - 135) : -INFINITY;
                            of[384] = __uint_as_float((uint32_t)(262 - ev) << 23);
                        }
                    }
                } else {
                    tk[128] = row >= 0 ? 0.0f : -INFINITY;
                }
                if (lane == 0) s_gap[g & 1][pw] = any_gap;
                if constexpr (PREC == 1) asm volatile("cp.async.wait_all;" ::: "memory");
                publish(k_full + (g & 1));
                load(k_next, a.pool.k, a.pool.scale_k, next);
                const bool dirty = PREC == 1 && t * TILE >= odd && any_odd(a.pool.v, row);
                if (g > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait_spin(v_free, (g - 1) & 1, &s_error, 8));
                if (!ok) break;
                write(v_next, sm + L::V);
                copy(sm + L::V, a.pool.v, row);
                if constexpr (PREC == 1) {
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    if (dirty) clean(sm + L::V);
                }
                publish(v_full);
                load(v_next, a.pool.v, a.pool.scale_v, next);
                row = next;
            }
            ++units;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, L::COLUMNS);
    }
    if (tid == 0 && s_error && a.error_flag) atomicExch(a.error_flag, 1);
}

// Joins the parts of the units that the shares of `ctas` CTAs cut, in token order.  A launch of its own: a part is 64 KB, and one
// CTA would fetch no more than 30 GB/s of them (with the last CTA to arrive joining, 128 rows of 8 key heads over 16384 tokens
// took 228 us, so 56).  Few units have many parts each: a block takes 16 rows of unit blockIdx.x.  Many have few: with `by_cta` it
// takes all rows of the unit that CTA blockIdx.x began and did not finish.
constexpr int kTcMaxParts = 512, kTcJoinRows = 16;
template <int DP, int TILE>
__global__ void __launch_bounds__(256) pool_attention_tc_join_kernel(const __grid_constant__ skv_pool_attention_args a, int ctas, bool by_cta,
                                                                     bool out_vec) {
    __shared__ Share s;
    __shared__ int s_sum[2];
    __shared__ float s_f[kTcMaxParts][kTcJoinRows];   // 2^(m_i - m) of a part
    __shared__ float s_l[kTcJoinRows];
    const int tid = threadIdx.x, D = a.pool.head_dim;
    const TcUnits<TILE> u(a);
    int b, base, at;
    const auto cost = [&](int i) {
        int tokens, n, past;
        u.sequence(a, i, tokens, n, past);
        return u.a_head(n, past, kTcPad) * a.pool.heads;
    };
    Share sh;
    if (by_cta) {
        take_share<256>(a, cost, kTcPad, 1, &s);
        sh = s;
        if (sh.lo >= sh.hi) return;
        b = sh.b;
        base = sh.base;
        at = sh.hi - 1;
    } else {
        const int per = u.row_tiles * a.pool.heads;
        b = blockIdx.x / per;
        int before = 0, all = 0;
        for (int i = tid; i < a.pool.batch; i += 256) {
            const int c = cost(i);
            all += c;
            before += i < b ? c : 0;
        }
        if (tid < 2) s_sum[tid] = 0;
        __syncthreads();
        before = __reduce_add_sync(0xffffffffu, before);
        all = __reduce_add_sync(0xffffffffu, all);
        if (tid % 32 == 0) {
            atomicAdd(&s_sum[0], before);
            atomicAdd(&s_sum[1], all);
        }
        __syncthreads();
        base = s_sum[0];
        sh.cut(s_sum[1], ctas, 1, kTcPad);
        sh.lo = 0;
        sh.hi = sh.total;
        int tokens, n, past;
        u.sequence(a, b, tokens, n, past);
        const int unit = blockIdx.x - b * per, hk = unit / u.row_tiles, rt = unit - hk * u.row_tiles, each = u.a_head(n, past, kTcPad);
        at = base + hk * each + (u.blocks ? rt / u.blocks * (each / u.rep) + u.before(rt % u.blocks, n, past, kTcPad) : rt * (n + kTcPad));
    }
    const TcSegment g = tc_segment_at(a, u, sh, at, b, base);
    const int c0 = sh.owner_of(g.first), parts = sh.owner_of(g.last) - c0 + 1;
    if (parts == 1 || (by_cta && c0 != (int)blockIdx.x)) return;
    const int64_t stride = (int64_t)2 * kTcRows * (D + 2);
    const float* next = slot_of(a, c0, 0, kTcRows);
    const float* part0 = slot_of(a, c0, g.first == sh.first_of(c0) ? 0 : 1, kTcRows);
    auto part = [&](int i) { return i == 0 ? part0 : next + i * stride; };
    for (int r_block = blockIdx.y * kTcJoinRows; r_block < g.rows; r_block += gridDim.y * kTcJoinRows) {
        __syncthreads();
        {
            const int j = tid / 16, sub = tid % 16, row = min(r_block + j, g.rows - 1);
            float m = -INFINITY, l = 0.0f;
            for (int i = sub; i < parts; i += 16) {
                const float mi = __ldcg(part(i) + kTcRows * D + row);
                s_f[i][j] = mi;
                m = fmaxf(m, mi);
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
            const float r = m == -INFINITY ? 0.0f : m;
            for (int i = sub; i < parts; i += 16) {
                const float f = exp2f(s_f[i][j] - r);
                s_f[i][j] = f;
                l += __ldcg(part(i) + kTcRows * D + kTcRows + row) * f;
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
            if (sub == 0) s_l[j] = l;
        }
        __syncthreads();
        constexpr int PER = kTcJoinRows * DP / 4 / 256;   // values (4 at a time) of a thread
        float y[PER][4];
        int row[PER], d[PER];
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            row[n] = (tid + 256 * n) / (DP / 4);
            d[n] = (tid + 256 * n) % (DP / 4) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[n][e] = 0.0f;
        }
        for (int i0 = 0; i0 < parts; i0 += 8) {
            float x[8][PER][4];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int n = 0; n < PER; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i][n][e] = 0.0f;
                    if (i0 + i < parts && r_block + row[n] < g.rows && d[n] < D)
                        load_part<4>(part(i0 + i) + (r_block + row[n]) * D + d[n], x[i][n]);
                }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int n = 0; n < PER; ++n) {
                    const float f = i0 + i < parts ? s_f[i0 + i][row[n]] : 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[n][e] = fmaf(x[i][n][e], f, y[n][e]);
                }
        }
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            if (r_block + row[n] >= g.rows || d[n] >= D) continue;
            const float l = s_l[row[n]];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[n][e] = l == 0.0f ? 0.0f : y[n][e] / l;
            store_row(a, g, g.r0 + r_block + row[n], d[n], out_vec, y[n]);
        }
    }
}

// Held while the two launches of a call are put on their stream: the second reads what the first left in the scratch, and another
// host thread's call on the same stream (and so with the same scratch) must not come between them.
std::mutex& tc_launches();

template <int PREC, int DP, int NP>
int launch_tc_weights(const skv_pool_attention_args& a, cudaStream_t st) {
    using L = TcLayout<DP>;
    static_assert(L::CTAS * 2 * kTcRows <= rows_per_sm(DP), "the scratch holds every CTA's slots");
    static_assert(L::CTAS * (L::ALLOC + 2048) <= 228 * 1024, "an SM holds the CTAs");
    const int rep = a.q.heads / a.pool.heads;
    const int64_t row_tiles = a.S_q >= kTcRows ? (int64_t)rep * ((a.S_q + kTcRows - 1) / kTcRows) : ((int64_t)rep * a.S_q + kTcRows - 1) / kTcRows;
    const int64_t step = sequences_a_launch(a, row_tiles, tc_tile(PREC), kTcPad);
    if (step == 0) return SKV_ERR_TOO_LARGE;
    const auto kernel = pool_attention_tc_kernel<PREC, DP, NP>;
    static std::atomic<uint64_t> allowed{0};   // devices whose limit on the kernel's shared memory was raised
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(allowed.load(std::memory_order_relaxed) >> dev & 1))) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC);
        if (e == cudaSuccess && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return fail(SKV_ERR_CUDA, "pool_attention: %s", cudaGetErrorString(e));
    const int ctas = min(sm_count() * L::CTAS, kTcMaxParts);
    const bool out_vec = rows_aligned(a.out);
    return by_sequences(a, step, [&](const skv_pool_attention_args& part) {
        const std::lock_guard<std::mutex> both(tc_launches());
        kernel<<<ctas, kTcThreads, L::ALLOC, st>>>(part, out_vec);
        const int64_t units = part.pool.batch * part.pool.heads * row_tiles;
        const bool by_cta = units > ctas;
        const dim3 grid(by_cta ? ctas : (int)units, by_cta ? 1 : kTcRows / kTcJoinRows);
        pool_attention_tc_join_kernel<DP, tc_tile(PREC)><<<grid, 256, 0, st>>>(part, ctas, by_cta, out_vec);
        return check_launch("pool_attention");
    });
}

template <int PREC, int DP>
int launch_tc(const skv_pool_attention_args& a, cudaStream_t st) {
    return a.q.dtype == kF16 ? launch_tc_weights<PREC, DP, 2>(a, st) : launch_tc_weights<PREC, DP, 1>(a, st);
}

}  // namespace skv
