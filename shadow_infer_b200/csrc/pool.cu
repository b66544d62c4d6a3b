// The page pool's data plane: the append that rotates and quantises as it writes, and the read back.
//
// Appending token t = lengths[b] + s: the key is turned to its position (rotary.cu), then key and
// value are stored in the pool's precision, bit-identical to the paged store's rows (paged.cu):
//     int8: scale = amax / 127 over the row, int4: amax / 7 over a group; 1 where the amax is 0;
//     n = rint(x / scale), clamped; int4 keeps n + 8, the even value in the high nibble.
// Everything is read once and written once: memory-bound, or latency-bound for a token a sequence.
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
    x.known = x.rot == 0 || (pos >= 0 && pos < a.rope.max_positions);
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
        for (int d = lane; d < D; d += kWarp) m = fmaxf(m, fabsf(x(d)));
        const float scale = quant_scale(warp_max(m), 127.0f), rcp = __frcp_rn(scale);
        for (int d = lane; d < D; d += kWarp) base[row * D + d] = (uint8_t)quant_value_fast(x(d), scale, rcp, -128, 127);
        if (lane == 0) sc[row] = scale;
    } else {
        const int G = a.pool.int4_group, ng = D / G;
        for (int g = lane; g < ng; g += kWarp) {
            float m = 0.0f;
            for (int d = g * G; d < (g + 1) * G; ++d) m = fmaxf(m, fabsf(x(d)));
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

// 16 values a lane, two chunks of 8: where halves are paired (SPLIT) chunk i of each half of the turned part, then of the rest;
// else 16 neighbours.  blockDim = (lanes a row: a power of two >= D / 16, rows at a time, tokens at a time).  A thread keeps its
// chunks of one token, reads their cos and sin and finds the token's page once, and walks the q, k and v heads with FLY rows on
// the way, the first ones asked for before anything else.  Every thread stays to the end: rows and int4 groups reduce
// over aligned lane blocks.
template <class T, bool SPLIT>
__global__ void __launch_bounds__(256) pool_append_kernel(const __grid_constant__ skv_pool_append_args a) {
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    const int D = a.pool.head_dim, Hk = a.pool.heads, Hq = a.q.heads, H = Hq + 2 * Hk, rot = a.rope.rot, half = rot / 2;
    const int tokens = a.pool.batch * a.S, token = blockIdx.x * blockDim.z + threadIdx.z;
    const int i0 = threadIdx.x;
    const bool there = token < tokens && 16 * i0 < D, paired = SPLIT && 16 * i0 < rot;
    const int d0 = SPLIT ? (paired ? 8 * i0 : half + 8 * i0) : 16 * i0;   // copied chunks start at rot: lane rot / 16 is the first
    const int d1 = SPLIT ? d0 + (paired ? half : (D - rot) / 2) : d0 + 8;
    const int b = there ? token / a.S : 0, s = there ? token - b * a.S : 0;
    const int step = blockDim.y * gridDim.y;
    Raw8<T> u[FLY], v[FLY];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int i = 0; i < FLY; ++i) {
            const int h = h0 + threadIdx.y + i * step;
            if (there && h < H) {
                const skv_rows& in = h < Hq ? a.q : h < Hq + Hk ? a.k : a.v;
                const T* x = static_cast<const T*>(in.ptr) + b * in.stride_b +
                             (h < Hq ? h : h < Hq + Hk ? h - Hq : h - Hq - Hk) * in.stride_h + s * in.stride_s;
                u[i].load(x + d0);
                v[i].load(x + d1);
            }
        }
    };
    fetch(blockIdx.y * blockDim.y);
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
    }
    const bool stored = there && (a.new_lengths == nullptr || s < a.new_lengths[b]);
    const int64_t row0 = stored ? pool_row(a.pool, b, t) : -1;
    if (stored && (row0 < 0 || !known) && a.error_flag) atomicExch(a.error_flag, 1);
    // a key whose position is not known is not stored: the row's first lane speaks for the row
    const bool key_known = __shfl_sync(0xffffffffu, (int)known, (threadIdx.y * blockDim.x + threadIdx.z * blockDim.x * blockDim.y) & 31);
    const int p = a.pool.precision, G = p == 3 ? a.pool.int4_group : 16;
    const int64_t row_bytes = pool_row_bytes(p, D);
    for (int h0 = blockIdx.y * blockDim.y; h0 < H;) {   // alike for all threads of the block
#pragma unroll
        for (int i = 0; i < FLY; ++i) {
            const int h = h0 + threadIdx.y + i * step;
            const bool is_q = h < Hq, is_k = !is_q && h < Hq + Hk, here = there && h < H;
            float x[8], y[8];   // the chunks
            if (here) {
                u[i].get(x);
                v[i].get(y);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.0f;
            }
            if (is_q || is_k) {
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
            }
            float m0 = 0.0f, m1 = 0.0f;
            if (p >= 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    m0 = fmaxf(m0, fabsf(x[e]));
                    m1 = fmaxf(m1, fabsf(y[e]));
                }
                if (p == 2) {
                    m0 = m1 = group_max(fmaxf(m0, m1), blockDim.x);
                } else if (SPLIT) {           // a group is the same chunk of G / 8 lanes
                    m0 = group_max(m0, G / 8);
                    m1 = group_max(m1, G / 8);
                } else if (G > 8) {           // both chunks of G / 16 lanes
                    m0 = m1 = group_max(fmaxf(m0, m1), G / 16);
                }
            }
            if (!here) continue;
            if (is_q) {
                T* to = static_cast<T*>(a.q_out.ptr) + b * a.q_out.stride_b + h * a.q_out.stride_h + s * a.q_out.stride_s;
                store8(to + d0, x);
                store8(to + d1, y);
                continue;
            }
            if (row0 < 0 || (is_k && !key_known)) continue;
            const int64_t row = row0 + (int64_t)(is_k ? h - Hq : h - Hq - Hk) * a.pool.page_size;
            uint8_t* to = static_cast<uint8_t*>(is_k ? a.pool.k : a.pool.v) + row * row_bytes;
            float* sc = is_k ? a.pool.scale_k : a.pool.scale_v;
            if (p == 0) {
                store8(reinterpret_cast<float*>(to) + d0, x);
                store8(reinterpret_cast<float*>(to) + d1, y);
            } else if (p == 1) {
                store8(reinterpret_cast<__half*>(to) + d0, x);
                store8(reinterpret_cast<__half*>(to) + d1, y);
            } else {
                int q[8];
                float f[8];
                const float s0 = quant_scale(m0, p == 2 ? 127.0f : 7.0f), s1 = m1 == m0 ? s0 : quant_scale(m1, p == 2 ? 127.0f : 7.0f);
                const float r0 = __frcp_rn(s0), r1 = __frcp_rn(s1);
                if (p == 2) {
                    quant_values<0>(x, s0, r0, -128, 127, q, f);
                    *reinterpret_cast<uint2*>(to + d0) = make_uint2(pack_s8(q[1], q[0], pack_s8(q[3], q[2], 0u)),
                                                                    pack_s8(q[5], q[4], pack_s8(q[7], q[6], 0u)));
                    quant_values<0>(y, s0, r0, -128, 127, q, f);
                    *reinterpret_cast<uint2*>(to + d1) = make_uint2(pack_s8(q[1], q[0], pack_s8(q[3], q[2], 0u)),
                                                                    pack_s8(q[5], q[4], pack_s8(q[7], q[6], 0u)));
                    if (i0 == 0) sc[row] = s0;
                } else {
                    quant_values<8>(x, s0, r0, -8, 7, q, f);
                    *reinterpret_cast<uint32_t*>(to + d0 / 2) =
                        pack_u4(q[0], q[1], pack_u4(q[2], q[3], pack_u4(q[4], q[5], pack_u4(q[6], q[7], 0u))));
                    quant_values<8>(y, s1, r1, -8, 7, q, f);
                    *reinterpret_cast<uint32_t*>(to + d1 / 2) =
                        pack_u4(q[0], q[1], pack_u4(q[2], q[3], pack_u4(q[4], q[5], pack_u4(q[6], q[7], 0u))));
                    float* g = sc + row * (D / G);
                    if (d0 % G == 0) g[d0 / G] = s0;
                    if (d1 % G == 0) g[d1 / G] = s1;
                }
            }
        }
        h0 += FLY * step;
        if (h0 < H) fetch(h0);
    }
}

// A warp per (token, head) row of K and of V; any D, group, strides and alignment.
template <class T>
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
    int64_t row = held ? pool_row(a.pool, b, t) : -1;
    if (held && row < 0 && lane == 0 && a.error_flag) atomicExch(a.error_flag, 1);
    if (row >= 0) row += (int64_t)h * a.pool.page_size;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const skv_rows& o = v ? a.v_out : a.k_out;
        T* out = static_cast<T*>(o.ptr) + b * o.stride_b + h * o.stride_h + s * o.stride_s;
        for (int d = lane; d < D; d += kWarp)
            out[d] = from_float<T>(row < 0 ? 0.0f : pool_value(a.pool, v, row, d));
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
    if (!vec) {
        const int64_t blocks = (tokens * H + kPoolWarps - 1) / kPoolWarps;
        pool_append_any_kernel<T><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a);
        return check_launch("pool_append");
    }
    int lanes = 1;
    while (lanes * 16 < D) lanes *= 2;
    // a token's rows in one pass of FLY rows a thread where up to 256 threads hold them; rows over more blocks while there are
    // too few tokens to fill the GPU; whole warps
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    const int fit = 256 / lanes, whole = 32 / lanes > 1 ? 32 / lanes : 1;
    int rows = (H + FLY - 1) / FLY < fit ? (H + FLY - 1) / FLY : fit, slices = 1, z = 1;
    while (rows > whole && tokens * slices < 2 * sm_count()) {
        slices *= 2;
        rows = (rows + 1) / 2;
    }
    rows = (rows + whole - 1) / whole * whole;
    while (z * 2 * rows <= fit && tokens * slices >= 8ll * sm_count() * z) z *= 2;
    const dim3 block(lanes, rows, z), grid((unsigned)((tokens + z - 1) / z), slices);
    if (split) pool_append_kernel<T, true><<<grid, block, 0, st>>>(a);
    else pool_append_kernel<T, false><<<grid, block, 0, st>>>(a);
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
        pool_read_any_kernel<T><<<(unsigned)blocks, 32 * kPoolWarps, 0, st>>>(a);
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
    const int64_t blocks = ((int64_t)a.pool.batch * a.S * a.pool.heads + kPoolWarps - 1) / kPoolWarps;
    if (blocks > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "pool_read: too many rows");
    cudaStream_t st = as_stream(stream);
    if (a.k_out.dtype == kF32) return launch_read<float>(a, st);
    if (a.k_out.dtype == kF16) return launch_read<__half>(a, st);
    return launch_read<__nv_bfloat16>(a, st);
}

}  // extern "C"
