// The page pool's data plane: the append that rotates and quantises as it writes, and the read back.
//
// Appending token t = lengths[b] + s: the key is turned to its position (rotary.cu), then key and
// value are stored in the pool's precision, bit-identical to the paged store's rows (paged.cu):
//     int8: scale = amax / 127 over the row, int4: amax / 7 over a group; 1 where the amax is 0;
//     n = rint(x / scale), clamped; int4 keeps n + 8, the even value in the high nibble.
// A NaN makes its scale NaN, so that its row or group is read as NaN (paged.cu's leaves it out of the scale).
// A token without a page, or whose position the rotary tables do not hold, leaves its rows as they were.
// Everything is read once and written once.  A token a sequence is bound by its latency: 8 sequences, 32 + 8 + 8 heads of 128
// values, 3.0 us.  A prompt is bound by what it computes: 8 x 2048 fp16 tokens of 32 + 32 heads into int8 take 107 us, about 320
// instructions for 4 rows of a warp (77 M in all, three quarters of the issue slots) at 3.4 TB/s.  The rows of padding are read
// too (13398 of the 16384 are tokens).  Reading them back as fp32 writes 4 bytes for one read: 105 us, 6.2 TB/s.
#include "pool.cuh"

namespace skv {

int check_pool(const skv_pool& p, const char* what) {
    if (p.batch < 0 || p.num_pages < 0 || p.page_size <= 0 || p.heads <= 0 || p.head_dim <= 0 || p.table_width < 0)
        return fail(SKV_ERR_INVALID_ARGUMENT, "%s: bad pool size", what);
    if (p.precision < 0 || p.precision > 3) return fail(SKV_ERR_INVALID_ARGUMENT, "%s: precision %d", what, p.precision);
    if (p.batch > 0 && p.table_width > 0 && !p.block_table)
        return fail(SKV_ERR_INVALID_ARGUMENT, "%s: the block table is null", what);
    if (p.num_pages > 0 && (!p.k || !p.v || (p.precision >= 2 && (!p.scale_k || !p.scale_v))))
        return fail(SKV_ERR_INVALID_ARGUMENT, "%s: the pool has a null payload", what);
    if (p.precision == 3 && (p.int4_group <= 0 || p.head_dim % p.int4_group))
        return fail(SKV_ERR_GROUP_SIZE, "%s: int4 group %d does not divide %d", what, p.int4_group, p.head_dim);
    return SKV_OK;
}

constexpr int kPoolWarps = 4;

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Over aligned groups of `width` lanes (a power of two <= 32).
__device__ __forceinline__ float group_max_nan(float x, int width) {
    for (int o = width >> 1; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// A warp's view of one source row: value d, turned where the row is a query or a key.
template <class T>
struct TurnedRow {
    const T* x;
    const float* cs;
    const float* sn;
    int rot, half;
    bool interleaved, known;
    float sign;
    __device__ __forceinline__ float operator()(int d) const {
        const float y = to_float(x[d]);
        if (d >= rot) return y;
        const int j = interleaved ? d / 2 : d % half;
        const bool second = interleaved ? d & 1 : d >= half;
        const float o = to_float(x[interleaved ? d ^ 1 : (second ? d - half : d + half)]);
        const float c = known ? cs[j] : __int_as_float(0x7fffffff);
        const float s = known ? sign * sn[j] : c;
        return second ? rope_second(o, y, c, s) : rope_first(y, o, c, s);
    }
};

// Any D, group, strides and alignment: a warp per (token, head) row of q, k or v.
template <class T>
__global__ void __launch_bounds__(32 * kPoolWarps) pool_append_any_kernel(const __grid_constant__ skv_pool_append_args a) {
    const int lane = threadIdx.x & 31;
    const int H = a.q.heads + 2 * a.pool.heads;
    const int64_t item = (int64_t)blockIdx.x * kPoolWarps + (threadIdx.x >> 5);
    if (item >= (int64_t)a.pool.batch * a.S * H) return;
    int h = (int)(item % H);
    const int64_t bs = item / H;
    const int b = (int)(bs / a.S), s = (int)(bs % a.S);
    const int kind = h < a.q.heads ? 0 : h < a.q.heads + a.pool.heads ? 1 : 2;   // q, k, v
    h -= kind == 0 ? 0 : kind == 1 ? a.q.heads : a.q.heads + a.pool.heads;
    const skv_rows& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t t = (int64_t)a.lengths[b] + s;
    const int64_t pos = rope_position(a.rope, b, s, t);
    TurnedRow<T> x;
    x.x = static_cast<const T*>(in.ptr) + b * in.stride_b + h * in.stride_h + s * in.stride_s;
    x.rot = kind == 2 ? 0 : a.rope.rot;
    x.half = a.rope.rot / 2;
    x.interleaved = a.rope.interleaved;
    x.sign = a.rope.inverse ? -1.0f : 1.0f;
    x.known = a.rope.rot == 0 || (pos >= 0 && pos < a.rope.max_positions);   // a value goes with its key
    x.cs = a.rope.cos + pos * x.half;
    x.sn = a.rope.sin + pos * x.half;
    const int D = a.pool.head_dim;
    if (kind == 0) {
        T* out = static_cast<T*>(a.q_out.ptr) + b * a.q_out.stride_b + h * a.q_out.stride_h + s * a.q_out.stride_s;
        for (int d = lane; d < D; d += kWarp) out[d] = from_float<T>(x(d));
        return;
    }
    if (a.new_lengths != nullptr && s >= a.new_lengths[b]) return;
    int64_t row = pool_row(a.pool, b, t);
    if (row < 0 || !x.known) {
        if (lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
        return;
    }
    row += (int64_t)h * a.pool.page_size;
    uint8_t* base = static_cast<uint8_t*>(kind == 2 ? a.pool.v : a.pool.k);
    float* sc = kind == 2 ? a.pool.scale_v : a.pool.scale_k;
    if (a.pool.precision == 0) {
        for (int d = lane; d < D; d += kWarp) reinterpret_cast<float*>(base)[row * D + d] = x(d);
    } else if (a.pool.precision == 1) {
        for (int d = lane; d < D; d += kWarp) reinterpret_cast<__half*>(base)[row * D + d] = __float2half_rn(x(d));
    } else if (a.pool.precision == 2) {
        float m = 0.0f;
        for (int d = lane; d < D; d += kWarp) m = max_nan(m, fabsf(x(d)));
        const float scale = quant_scale(group_max_nan(m, kWarp), 127.0f), rcp = __frcp_rn(scale);
        for (int d = lane; d < D; d += kWarp) base[row * D + d] = (uint8_t)quant_value_fast(x(d), scale, rcp, -128, 127);
        if (lane == 0) sc[row] = scale;
    } else {
        const int G = a.pool.int4_group, ng = D / G;
        for (int g = lane; g < ng; g += kWarp) {
            float m = 0.0f;
            for (int d = g * G; d < (g + 1) * G; ++d) m = max_nan(m, fabsf(x(d)));
            sc[row * ng + g] = quant_scale(m, 7.0f);
        }
        __syncwarp();
        const int rb = (D + 1) / 2;
        for (int j = lane; j < rb; j += kWarp) {
            unsigned byte = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 2 * j + i;
                if (d < D) {
                    const float scale = *reinterpret_cast<volatile float*>(sc + row * ng + d / G);
                    byte |= ((unsigned)(quant_value_fast(x(d), scale, __frcp_rn(scale), -8, 7) + 8) & 15u) << (i ? 0 : 4);
                }
            }
            base[row * rb + j] = (uint8_t)byte;
        }
    }
}

constexpr float kRoundMagic = 12582912.0f;   // 1.5 2^23: x + this has rint(x) in its low bits for |x| < 2^22

// t[e] = 1.5 2^23 + add + rint(fl(x[e] / s)), whose low byte is the integer (+ add) that is stored.  r is the correctly
// rounded 1 / s; then q + r (x - q s), the residual by one fma, is the correctly rounded quotient (Markstein's correction,
// IBM J. Res. Dev. 34, 1990), so the integers are those of a division at a third of its instructions.  `odd`: the
// row's scale leaves that theorem's range (NaN, infinite, near the ends of fp32); then the division is made.
__device__ __forceinline__ void quotients(const float (&x)[8], float s, float r, bool odd, int lo, int hi, float add, float (&t)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = __fmul_rn(x[e], r);
        t[e] = __fadd_rn(__fmaf_rn(__fmaf_rn(-q, s, x[e]), r, q), kRoundMagic + add);
    }
    if (__builtin_expect(odd, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (kRoundMagic + add) + (float)quant_value(x[e], s, lo, hi);
    }
}
// The low bytes of four of them.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040),
                       0x5410);
}

// Division of a non-negative m by 7 or 127 (r: its correctly rounded reciprocal), as quant_scale.
__device__ __forceinline__ float scale_of(float m, float top, float r) {
    const float q = __fmul_rn(m, r), s = __fmaf_rn(__fmaf_rn(-q, top, m), r, q);
    return m > 1e-30f && m < 1e30f ? s : quant_scale(m, top);
}

// 16 values a lane, two chunks of 8: where halves are paired (SPLIT) chunk i of each half of the turned part, then of the rest;
// else 16 neighbours.  blockDim = (lanes a row: a power of two >= D / 16, rows at a time, tokens at a time); a block takes
// FLY * rows heads of q, of k or of v (blockIdx.y: first the slices of q, then of k, then of v), every row asked for before the
// token's position and page are known.  Every thread stays to the end: rows and int4 groups reduce over aligned lane blocks.
// (The prompt above with a warp a row: 845 us for append and read; blocks of one kind of rows and quotients without
// divisions: append 163 -> 130; three blocks an SM, which hide what four rows on the way a thread do not: 112; NaN kept in the maxima, so
// no second pass: 107.)
template <class T, bool SPLIT>
__global__ void __launch_bounds__(256, 3) pool_append_kernel(const __grid_constant__ skv_pool_append_args a, int q_slices, int kv_slices) {
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    const int D = a.pool.head_dim, half = a.rope.rot / 2, i0 = threadIdx.x;
    const int slice = blockIdx.y, kind = slice < q_slices ? 0 : slice < q_slices + kv_slices ? 1 : 2;   // q, k, v
    const int rot = kind == 2 ? 0 : a.rope.rot, H = kind == 0 ? a.q.heads : a.pool.heads;
    const int h0 = (kind == 0 ? slice : kind == 1 ? slice - q_slices : slice - q_slices - kv_slices) * FLY * blockDim.y + threadIdx.y;
    const int tokens = a.pool.batch * a.S, token = blockIdx.x * blockDim.z + threadIdx.z;
    const bool there = token < tokens && 16 * i0 < D;
    const int b = there ? token / a.S : 0, s = there ? token - b * a.S : 0;
    const bool paired = SPLIT && 16 * i0 < a.rope.rot;
    const int d0 = SPLIT ? (paired ? 8 * i0 : half + 8 * i0) : 16 * i0;   // copied chunks start at rot: lane rot / 16 is the first
    const int d1 = SPLIT ? d0 + (paired ? half : (D - a.rope.rot) / 2) : d0 + 8;
    const skv_rows& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const T* from = static_cast<const T*>(in.ptr) + b * in.stride_b + s * in.stride_s;
    const int64_t stride_h = in.stride_h;
    Raw8<T> u[FLY], v[FLY];
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
        const int h = h0 + i * blockDim.y;
        if (there && h < H) {
            u[i].load(from + h * stride_h + d0);
            v[i].load(from + h * stride_h + d1);
        }
    }
    const int64_t t = there ? (int64_t)a.lengths[b] + s : 0;
    // cos and sin of 8 pairs: of both chunks (SPLIT), or 4 of each
    float c[8], w[8];
    bool known = true;
    const bool turn0 = there && d0 < rot, turn1 = there && d1 < rot;
    if (turn0) {
        const int64_t pos = rope_position(a.rope, b, s, t);
        known = pos >= 0 && pos < a.rope.max_positions;
        if (known && (SPLIT || turn1)) {
            load8(a.rope.cos + pos * half + (SPLIT ? d0 : d0 / 2), c);
            load8(a.rope.sin + pos * half + (SPLIT ? d0 : d0 / 2), w);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool have = known && i < 4;
                c[i] = have ? a.rope.cos[pos * half + d0 / 2 + i] : __int_as_float(0x7fffffff);
                w[i] = have ? a.rope.sin[pos * half + d0 / 2 + i] : __int_as_float(0x7fffffff);
            }
        }
        if (a.rope.inverse)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = -w[i];
    } else if (kind == 2 && there && a.rope.rot > 0) {   // a value goes with its key
        const int64_t pos = rope_position(a.rope, b, s, t);
        known = pos >= 0 && pos < a.rope.max_positions;
    }
    const bool stored = kind != 0 && there && (a.new_lengths == nullptr || s < a.new_lengths[b]);
    const int64_t row0 = stored ? pool_row(a.pool, b, t) : -1;
    if (stored && (row0 < 0 || !known) && a.error_flag) atomicExch(a.error_flag, 1);
    // a key whose position is not known is not stored, and neither is its value: the row's first lane speaks for the row
    if (kind != 0 && !__any_sync(0xffffffffu, row0 >= 0)) return;   // padding of a ragged prompt
    const bool ok = __shfl_sync(0xffffffffu, (int)known, (threadIdx.y * blockDim.x + threadIdx.z * blockDim.x * blockDim.y) & 31);
    const int p = kind == 0 ? 0 : a.pool.precision, G = p == 3 ? a.pool.int4_group : 16;
    const int row_bytes = (int)pool_row_bytes(p, D), groups = D / G;
    uint8_t* to = static_cast<uint8_t*>(kind == 1 ? a.pool.k : a.pool.v) + row0 * row_bytes;
    float* sc = (kind == 1 ? a.pool.scale_k : a.pool.scale_v) + row0 * (p == 3 ? groups : 1);
    T* q_to = static_cast<T*>(a.q_out.ptr) + b * a.q_out.stride_b + s * a.q_out.stride_s;
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
        const int h = h0 + i * blockDim.y;
        const bool here = there && h < H;
        float x[8], y[8];   // the chunks
        if (here) {
            u[i].get(x);
            v[i].get(y);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
        }
        if constexpr (SPLIT) {
            if (turn0)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = rope_first(x[e], y[e], c[e], w[e]);
                    y[e] = rope_second(x[e], y[e], c[e], w[e]);
                    x[e] = z;
                }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (turn0) {
                    const float z = rope_first(x[2 * e], x[2 * e + 1], c[e], w[e]);
                    x[2 * e + 1] = rope_second(x[2 * e], x[2 * e + 1], c[e], w[e]);
                    x[2 * e] = z;
                }
                if (turn1) {
                    const float z = rope_first(y[2 * e], y[2 * e + 1], c[4 + e], w[4 + e]);
                    y[2 * e + 1] = rope_second(y[2 * e], y[2 * e + 1], c[4 + e], w[4 + e]);
                    y[2 * e] = z;
                }
            }
        }
        if (kind == 0) {
            if (here) {
                store8(q_to + h * a.q_out.stride_h + d0, x);
                store8(q_to + h * a.q_out.stride_h + d1, y);
            }
            continue;
        }
        const int64_t off = (int64_t)h * a.pool.page_size;
        const bool write = here && row0 >= 0 && ok;
        if (p < 2) {
            if (!write) continue;
            if (p == 0) {
                store8(reinterpret_cast<float*>(to + off * row_bytes) + d0, x);
                store8(reinterpret_cast<float*>(to + off * row_bytes) + d1, y);
            } else {
                store8(reinterpret_cast<__half*>(to + off * row_bytes) + d0, x);
                store8(reinterpret_cast<__half*>(to + off * row_bytes) + d1, y);
            }
            continue;
        }
        float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m0 = max_nan(m0, fabsf(x[e]));
            m1 = max_nan(m1, fabsf(y[e]));
        }
        float f[8], g[8];
        if (p == 2) {
            const float m = group_max_nan(max_nan(m0, m1), blockDim.x);
            if (!write) continue;
            const float scale = scale_of(m, 127.0f, 1.0f / 127.0f), rcp = __frcp_rn(scale);
            const bool odd = !(scale > 1e-30f && scale < 1e30f);
            quotients(x, scale, rcp, odd, -128, 127, 0.0f, f);
            quotients(y, scale, rcp, odd, -128, 127, 0.0f, g);
            uint8_t* dst = to + off * row_bytes;
            *reinterpret_cast<uint2*>(dst + d0) = make_uint2(low_bytes(f[0], f[1], f[2], f[3]), low_bytes(f[4], f[5], f[6], f[7]));
            *reinterpret_cast<uint2*>(dst + d1) = make_uint2(low_bytes(g[0], g[1], g[2], g[3]), low_bytes(g[4], g[5], g[6], g[7]));
            if (i0 == 0) sc[off] = scale;
        } else {
            if (SPLIT) {           // a group is the same chunk of G / 8 lanes
                m0 = group_max_nan(m0, G / 8);
                m1 = group_max_nan(m1, G / 8);
            } else if (G > 8) {    // both chunks of G / 16 lanes
                m0 = m1 = group_max_nan(max_nan(m0, m1), G / 16);
            }
            if (!write) continue;
            const float s0 = scale_of(m0, 7.0f, 1.0f / 7.0f), s1 = scale_of(m1, 7.0f, 1.0f / 7.0f);
            const bool odd = !(s0 > 1e-30f && s1 > 1e-30f && s0 < 1e30f && s1 < 1e30f);
            quotients(x, s0, __frcp_rn(s0), odd, -8, 7, 8.0f, f);
            quotients(y, s1, __frcp_rn(s1), odd, -8, 7, 8.0f, g);
            uint8_t* dst = to + off * row_bytes;
            *reinterpret_cast<uint32_t*>(dst + d0 / 2) = low_bytes(f[0], f[2], f[4], f[6]) << 4 | low_bytes(f[1], f[3], f[5], f[7]);
            *reinterpret_cast<uint32_t*>(dst + d1 / 2) = low_bytes(g[0], g[2], g[4], g[6]) << 4 | low_bytes(g[1], g[3], g[5], g[7]);
            if (d0 % G == 0) sc[off * groups + d0 / G] = s0;
            if (d1 % G == 0) sc[off * groups + d1 / G] = s1;
        }
    }
}

// A warp per (token, head) row of K and of V; any D, group, strides and alignment.
template <class T, int PREC>
__global__ void __launch_bounds__(32 * kPoolWarps) pool_read_any_kernel(const __grid_constant__ skv_pool_read_args a) {
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * kPoolWarps + (threadIdx.x >> 5);
    const int H = a.pool.heads, D = a.pool.head_dim;
    if (item >= (int64_t)a.pool.batch * H * a.S) return;
    const int s = (int)(item % a.S);
    const int64_t bh = item / a.S;
    const int b = (int)(bh / H), h = (int)(bh % H);
    const int64_t t = (a.start ? (int64_t)a.start[b] : 0) + s;
    const bool held = t >= 0 && t < a.lengths[b];
    if (a.lengths[b] < 0 && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
    int64_t row = held ? pool_row(a.pool, b, t) : -1;
    if (held && row < 0 && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
    if (row >= 0) row += (int64_t)h * a.pool.page_size;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const skv_rows& o = v ? a.v_out : a.k_out;
        T* out = static_cast<T*>(o.ptr) + b * o.stride_b + h * o.stride_h + s * o.stride_s;
        for (int d = lane; d < D; d += kWarp)
            out[d] = from_float<T>(row < 0 ? 0.0f : pool_value<PREC>(a.pool, v, row, d, PREC == 3 ? d / a.pool.int4_group : 0));
    }
}

// 16 bytes of output a lane (V values), of K and V, FLY tokens on the way: blockDim = (D / V, tokens), grid (token blocks,
// B * heads).
template <class T, int PREC>
__global__ void __launch_bounds__(256) pool_read_kernel(const __grid_constant__ skv_pool_read_args a) {
    constexpr int V = 16 / sizeof(T), FLY = 4;
    const int b = blockIdx.y / a.pool.heads, h = blockIdx.y - b * a.pool.heads, d = V * threadIdx.x;
    const int64_t first = a.start ? (int64_t)a.start[b] : 0, length = a.lengths[b];
    const int s0 = blockIdx.x * blockDim.y * FLY + threadIdx.y;
    if (length < 0 && threadIdx.x == 0 && a.error_flag) atomicExch(a.error_flag, 1);
    PoolRaw<PREC, V> k[FLY], v[FLY];
    int64_t row[FLY];
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
        const int s = s0 + i * blockDim.y;
        const int64_t t = first + s;
        const bool held = s < a.S && t >= 0 && t < length;
        row[i] = held ? pool_row(a.pool, b, t) : -1;
        if (held && row[i] < 0 && a.error_flag) atomicExch(a.error_flag, 1);
    }
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
        if (row[i] >= 0) {
            k[i].load(a.pool, false, row[i] + (int64_t)h * a.pool.page_size, d);
            v[i].load(a.pool, true, row[i] + (int64_t)h * a.pool.page_size, d);
        } else {
            k[i].zero();
            v[i].zero();
        }
    }
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
        const int s = s0 + i * blockDim.y;
        if (s >= a.S) break;
        float x[V], y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[e] = k[i].get(e);
            y[e] = v[i].get(e);
        }
        T* to = static_cast<T*>(a.k_out.ptr) + b * a.k_out.stride_b + h * a.k_out.stride_h + s * a.k_out.stride_s + d;
        T* vo = static_cast<T*>(a.v_out.ptr) + b * a.v_out.stride_b + h * a.v_out.stride_h + s * a.v_out.stride_s + d;
        if constexpr (V == 4) {
            *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(vo) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            store8(to, x);
            store8(vo, y);
        }
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <class T>
int launch_append(const skv_pool_append_args& a, cudaStream_t st) {
    const int D = a.pool.head_dim, H = a.q.heads + 2 * a.pool.heads;
    const int64_t tokens = (int64_t)a.pool.batch * a.S;
    // halves are paired only where something turns that way; int4 groups must be whole lane blocks of a chunk then
    const int rot = a.rope.rot, G = a.pool.precision == 3 ? a.pool.int4_group : 16;
    const bool split = rot > 0 && !a.rope.interleaved;
    const auto power = [](int n) { return n > 0 && (n & (n - 1)) == 0; };
    bool vec = D % 16 == 0 && D <= 512 && rows_aligned(a.q) && rows_aligned(a.k) && rows_aligned(a.v) && rows_aligned(a.q_out) &&
               aligned16(a.pool.k) && aligned16(a.pool.v) && aligned16(a.rope.cos) && aligned16(a.rope.sin);
    if (split) vec = vec && rot % 16 == 0 && (a.pool.precision != 3 || (G % 8 == 0 && power(G / 8) && rot / 2 % G == 0 && (D - rot) / 2 % G == 0));
    else vec = vec && rot % 8 == 0 && (a.pool.precision != 3 || G == 8 || (G % 16 == 0 && power(G / 16)));
    vec = vec && H <= 65535 && tokens <= 0x7fffffff - 64;   // grid.y; tokens are numbered in 31 bits there
    if (!vec) {
        const int64_t blocks = (tokens * H + kPoolWarps - 1) / kPoolWarps;
        pool_append_any_kernel<T><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a);
        return check_launch("pool_append");
    }
    // a block takes FLY rows a thread of a token's heads of one kind, or one row a thread while there are too few tokens to
    // fill the GPU; the rest of 256 threads takes other tokens
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    int lanes = 1, rows = 1, z = 1;
    while (lanes * 16 < D) lanes *= 2;
    const int want = tokens * (a.q.heads + 2 * a.pool.heads) * lanes < 256ll * 2 * sm_count() ? a.pool.heads : (a.pool.heads + FLY - 1) / FLY;
    while (rows < want && lanes * rows < 256) rows *= 2;
    while (lanes * rows * z < 32 || (z < 64 && lanes * rows * z * 2 <= 256 && tokens >= 8ll * sm_count() * z)) z *= 2;   // blockDim.z <= 64
    const int q_slices = (a.q.heads + rows * FLY - 1) / (rows * FLY), kv_slices = (a.pool.heads + rows * FLY - 1) / (rows * FLY);
    const dim3 block(lanes, rows, z), grid((unsigned)((tokens + z - 1) / z), q_slices + 2 * kv_slices);
    if (split) pool_append_kernel<T, true><<<grid, block, 0, st>>>(a, q_slices, kv_slices);
    else pool_append_kernel<T, false><<<grid, block, 0, st>>>(a, q_slices, kv_slices);
    return check_launch("pool_append");
}

template <class T>
int launch_read(const skv_pool_read_args& a, cudaStream_t st) {
    const int D = a.pool.head_dim;
    const int64_t rows = (int64_t)a.pool.batch * a.pool.heads;
    const bool vec = D % 8 == 0 && D <= 1024 && rows <= 65535 && rows_aligned(a.k_out) && rows_aligned(a.v_out) && aligned16(a.pool.k) &&
                     aligned16(a.pool.v) && (a.pool.precision != 3 || a.pool.int4_group % 8 == 0);
    if (!vec) {
        const int64_t blocks = (rows * a.S + kPoolWarps - 1) / kPoolWarps;
        switch (a.pool.precision) {
            case 0: pool_read_any_kernel<T, 0><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a); break;
            case 1: pool_read_any_kernel<T, 1><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a); break;
            case 2: pool_read_any_kernel<T, 2><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a); break;
            default: pool_read_any_kernel<T, 3><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a);
        }
        return check_launch("pool_read");
    }
    const int lanes = D / (16 / (int)sizeof(T));
    int tokens = 256 / lanes;
    tokens = tokens < 1 ? 1 : tokens > a.S ? a.S : tokens;
    const dim3 block(lanes, tokens), grid((a.S + tokens * 4 - 1) / (tokens * 4), (unsigned)rows);
    switch (a.pool.precision) {
        case 0: pool_read_kernel<T, 0><<<grid, block, 0, st>>>(a); break;
        case 1: pool_read_kernel<T, 1><<<grid, block, 0, st>>>(a); break;
        case 2: pool_read_kernel<T, 2><<<grid, block, 0, st>>>(a); break;
        default: pool_read_kernel<T, 3><<<grid, block, 0, st>>>(a);
    }
    return check_launch("pool_read");
}

}  // namespace skv

using namespace skv;

extern "C" {

int skv_pool_append(const skv_pool_append_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_append: null pointer");
    const skv_pool_append_args& a = *args;
    int rc;
    if ((rc = check_pool(a.pool, "pool_append")) || (rc = check_rows(a.k, a.pool.batch > 0 && a.S > 0, "pool_append", "k")) ||
        (rc = check_rows(a.v, a.pool.batch > 0 && a.S > 0, "pool_append", "v")) || (rc = check_rows(a.q, a.pool.batch > 0 && a.S > 0, "pool_append", "q")) ||
        (rc = check_rows(a.q_out, a.pool.batch > 0 && a.S > 0, "pool_append", "q_out")) || (rc = check_rope(a.rope, a.pool.head_dim, "pool_append")))
        return rc;
    if (a.S < 0) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_append: bad size");
    if (a.k.heads != a.pool.heads || a.v.heads != a.pool.heads || a.q.heads != a.q_out.heads ||
        a.k.dtype != a.v.dtype || (a.q.heads && (a.q.dtype != a.k.dtype || a.q_out.dtype != a.k.dtype)))
        return fail(SKV_ERR_SHAPE, "pool_append: rows disagree in heads or dtype");
    if (a.q.heads && a.rope.rot == 0) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_append: q without rotary tables");
    if (a.pool.batch == 0 || a.S == 0) return SKV_OK;
    if (!a.lengths) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_append: lengths is null");
    const int64_t blocks = ((int64_t)a.pool.batch * a.S * (a.q.heads + 2 * a.pool.heads) + kPoolWarps - 1) / kPoolWarps;
    if (blocks > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "pool_append: too many rows");
    cudaStream_t st = as_stream(stream);
    if (a.k.dtype == kF32) return launch_append<float>(a, st);
    if (a.k.dtype == kF16) return launch_append<__half>(a, st);
    return launch_append<__nv_bfloat16>(a, st);
}

int skv_pool_read(const skv_pool_read_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_read: null pointer");
    const skv_pool_read_args& a = *args;
    int rc;
    if ((rc = check_pool(a.pool, "pool_read")) || (rc = check_rows(a.k_out, a.pool.batch > 0 && a.S > 0, "pool_read", "k_out")) ||
        (rc = check_rows(a.v_out, a.pool.batch > 0 && a.S > 0, "pool_read", "v_out")))
        return rc;
    if (a.S < 0) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_read: bad size");
    if (a.k_out.heads != a.pool.heads || a.v_out.heads != a.pool.heads || a.k_out.dtype != a.v_out.dtype)
        return fail(SKV_ERR_SHAPE, "pool_read: outputs disagree in heads or dtype");
    if (a.pool.batch == 0 || a.S == 0) return SKV_OK;
    if (!a.lengths) return fail(SKV_ERR_INVALID_ARGUMENT, "pool_read: lengths is null");
    if (a.S > 0x7fffffff - 4096) return fail(SKV_ERR_TOO_LARGE, "pool_read: too many tokens");   // a block's last is numbered in 31 bits
    const int64_t blocks = ((int64_t)a.pool.batch * a.S * a.pool.heads + kPoolWarps - 1) / kPoolWarps;
    if (blocks > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "pool_read: too many rows");
    cudaStream_t st = as_stream(stream);
    if (a.k_out.dtype == kF32) return launch_read<float>(a, st);
    if (a.k_out.dtype == kF16) return launch_read<__half>(a, st);
    return launch_read<__nv_bfloat16>(a, st);
}

}  // extern "C"
