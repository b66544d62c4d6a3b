// Rotary positions: rows [B, H, S, D] turned pair by pair, queries and keys in one launch.
//
// A pair (a, b) of the first `rot` values of a row at position p becomes
//     (a c - b s, b c + a s),   c = cos[p][i], s = sin[p][i]   (s negated to turn back),
// with (a, b) = (x[i], x[i + rot/2]) or, interleaved, (x[2i], x[2i+1]); the other values are
// copied.  Two products and a sum a value against 2 x 2..4 bytes moved: memory-bound.  A prompt of 8192 tokens of 40 bf16
// heads of 128 values (172 MB with its tables) takes 35 us, 4.9 TB/s; 3 x 517 tokens of 9 fp32 heads 3.3 us, the launch's latency.
#include "pool.cuh"

namespace skv {

int check_rows(const skv_rows& r, bool some, const char* what, const char* name) {
    if (r.heads < 0 || (some && r.heads > 0 && !r.ptr)) return fail(SKV_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
    if (r.dtype < 0 || r.dtype > 2) return fail(SKV_ERR_INVALID_ARGUMENT, "%s: %s has dtype %d", what, name, r.dtype);
    return SKV_OK;
}

int check_rope(const skv_rope& r, int D, const char* what) {
    if (r.rot < 0 || r.rot > D || r.rot % 2) return fail(SKV_ERR_SHAPE, "%s: %d rotated values of %d", what, r.rot, D);
    if (r.rot == 0) return SKV_OK;
    if (!r.cos || !r.sin || r.max_positions <= 0)
        return fail(SKV_ERR_INVALID_ARGUMENT, "%s: rotary tables are missing", what);
    if (r.positions && r.pos_bytes != 4 && r.pos_bytes != 8)
        return fail(SKV_ERR_INVALID_ARGUMENT, "%s: positions of %d bytes", what, r.pos_bytes);
    return SKV_OK;
}

// Any D, strides and alignment: grid (B * S, head slices), a thread per value.
template <class T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const __grid_constant__ skv_rotary_args a) {
    const int bs = blockIdx.x, b = bs / a.S, s = bs % a.S;
    const int64_t pos = rope_position(a.rope, b, s, s);
    const bool known = pos >= 0 && pos < a.rope.max_positions;
    const int half = a.rope.rot / 2, H = a.q.heads + a.k.heads;
    const float* cs = a.rope.cos + pos * half;
    const float* sn = a.rope.sin + pos * half;
    for (int64_t i = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; i < (int64_t)H * a.D;
         i += (int64_t)gridDim.y * blockDim.x) {
        const int hh = (int)(i / a.D), d = (int)(i % a.D);
        const bool is_k = hh >= a.q.heads;
        const skv_rows& in = is_k ? a.k : a.q;
        const skv_rows& out = is_k ? a.k_out : a.q_out;
        const int h = is_k ? hh - a.q.heads : hh;
        const T* x = static_cast<const T*>(in.ptr) + b * in.stride_b + h * in.stride_h + s * in.stride_s;
        float y = to_float(x[d]);
        if (d < a.rope.rot) {
            const int j = a.rope.interleaved ? d / 2 : d % half;
            const bool second = a.rope.interleaved ? d & 1 : d >= half;
            const float o = to_float(x[a.rope.interleaved ? d ^ 1 : (second ? d - half : d + half)]);
            const float c = known ? cs[j] : __int_as_float(0x7fffffff);
            const float w = known ? (a.rope.inverse ? -sn[j] : sn[j]) : c;
            y = second ? rope_second(o, y, c, w) : rope_first(y, o, c, w);
        }
        static_cast<T*>(out.ptr)[b * out.stride_b + h * out.stride_h + s * out.stride_s + d] = from_float<T>(y);
    }
}

// 8 values a load.  A row is cut into items: 16 half-split values (8 of each half) or 8 interleaved ones that turn, or 8 that
// are copied.  blockDim = (items, heads at a time, tokens at a time): a thread keeps its item of one token, so it reads cos and
// sin once, and walks the heads with FLY rows on the way; the first rows are asked for before the position is known.
template <class T, bool SPLIT>
__global__ void __launch_bounds__(256, 3) rotary_kernel(const __grid_constant__ skv_rotary_args a, int turned, int tokens) {
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    const int token = blockIdx.x * blockDim.z + threadIdx.z;
    if (token >= tokens) return;
    const int b = token / a.S, s = token - b * a.S, item = threadIdx.x, half = a.rope.rot / 2;
    const bool turns = item < turned;
    const int d = SPLIT ? (turns ? 8 * item : a.rope.rot + 8 * (item - turned)) : 8 * item;
    const T* q = static_cast<const T*>(a.q.ptr) + b * a.q.stride_b + s * a.q.stride_s + d;
    const T* k = static_cast<const T*>(a.k.ptr) + b * a.k.stride_b + s * a.k.stride_s + d;
    T* qo = static_cast<T*>(a.q_out.ptr) + b * a.q_out.stride_b + s * a.q_out.stride_s + d;
    T* ko = static_cast<T*>(a.k_out.ptr) + b * a.k_out.stride_b + s * a.k_out.stride_s + d;
    const int H = a.q.heads + a.k.heads, step = blockDim.y * gridDim.y;
    Raw8<T> u[FLY], v[FLY];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int i = 0; i < FLY; ++i) {
            const int h = h0 + i * step;
            if (h < H) {
                const T* p = h < a.q.heads ? q + h * a.q.stride_h : k + (h - a.q.heads) * a.k.stride_h;
                u[i].load(p);
                if (SPLIT && turns) v[i].load(p + half);
            }
        }
    };
    int h0 = blockIdx.y * blockDim.y + threadIdx.y;
    fetch(h0);
    float c[8], w[8];
    if (turns) {
        const int64_t pos = rope_position(a.rope, b, s, s);
        if (pos >= 0 && pos < a.rope.max_positions) {
            const float* cs = a.rope.cos + pos * half + (SPLIT ? d : d / 2);
            const float* sn = a.rope.sin + pos * half + (SPLIT ? d : d / 2);
            if constexpr (SPLIT) {
                load8(cs, c);
                load8(sn, w);
            } else {
                const float4 x = *reinterpret_cast<const float4*>(cs), y = *reinterpret_cast<const float4*>(sn);
                c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
                w[0] = y.x; w[1] = y.y; w[2] = y.z; w[3] = y.w;
            }
            if (a.rope.inverse)
#pragma unroll
                for (int i = 0; i < (SPLIT ? 8 : 4); ++i) w[i] = -w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = w[i] = __int_as_float(0x7fffffff);
        }
    }
    for (;;) {
#pragma unroll
        for (int i = 0; i < FLY; ++i) {
            const int h = h0 + i * step;
            if (h >= H) break;
            T* p = h < a.q.heads ? qo + h * a.q_out.stride_h : ko + (h - a.q.heads) * a.k_out.stride_h;
            float x[8];
            u[i].get(x);
            if (turns) {
                if constexpr (SPLIT) {
                    float y[8], z[8];
                    v[i].get(y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        z[e] = rope_first(x[e], y[e], c[e], w[e]);
                        y[e] = rope_second(x[e], y[e], c[e], w[e]);
                    }
                    store8(p, z);
                    store8(p + half, y);
                    continue;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float z = rope_first(x[2 * e], x[2 * e + 1], c[e], w[e]);
                        x[2 * e + 1] = rope_second(x[2 * e], x[2 * e + 1], c[e], w[e]);
                        x[2 * e] = z;
                    }
                }
            }
            store8(p, x);
        }
        h0 += FLY * step;
        if (h0 >= H) break;
        fetch(h0);
    }
}

template <class T>
int launch_rotary(const skv_rotary_args& a, cudaStream_t st) {
    const int tokens = a.B * a.S, H = a.q.heads + a.k.heads;
    const bool split = !a.rope.interleaved;
    // 8-value items: rows on 16-byte boundaries, turned parts of whole items, tables on 16 bytes too
    const bool vec = a.D % 8 == 0 && a.rope.rot % (split ? 16 : 8) == 0 && a.D <= 1024 && rows_aligned(a.q) && rows_aligned(a.k) &&
                     rows_aligned(a.q_out) && rows_aligned(a.k_out) &&
                     ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 15) == 0;
    if (!vec) {
        const int64_t slices = ((int64_t)H * a.D + 1023) / 1024;
        rotary_any_kernel<T><<<dim3((unsigned)tokens, (unsigned)(slices < 65535 ? slices : 65535)), 256, 0, st>>>(a);
        return check_launch("rotary");
    }
    const int turned = split ? a.rope.rot / 16 : a.rope.rot / 8;
    const int items = turned + (a.D - a.rope.rot) / 8;
    // a block of up to 256 threads: a token's heads in as many steps as a thread has rows on the way (more where they do not
    // fit), then more tokens; heads over more blocks while there are too few tokens to fill the GPU
    constexpr int FLY = sizeof(T) == 2 ? 4 : 2;
    int steps = H < FLY ? H : FLY;
    while ((H + steps - 1) / steps * items > 256) ++steps;
    int heads = (H + steps - 1) / steps;
    int slices = 1;
    while (heads > 1 && (int64_t)tokens * slices < sm_count() && slices * 2 <= H) {
        slices *= 2;
        heads = (H + slices * steps - 1) / (slices * steps);
    }
    const int together = 256 / (items * heads) > 1 ? 256 / (items * heads) : 1;
    const int z = (int64_t)tokens * slices >= (int64_t)together * 4 * sm_count() ? (together < 64 ? together : 64) : 1;
    const dim3 block(items, heads, z), grid((tokens + z - 1) / z, slices);
    if (split) rotary_kernel<T, true><<<grid, block, 0, st>>>(a, turned, tokens);
    else rotary_kernel<T, false><<<grid, block, 0, st>>>(a, turned, tokens);
    return check_launch("rotary");
}

}  // namespace skv

using namespace skv;

extern "C" int skv_rotary(const skv_rotary_args* args, void* stream) {
    if (!args) return fail(SKV_ERR_INVALID_ARGUMENT, "rotary: null pointer");
    const skv_rotary_args& a = *args;
    if (a.B < 0 || a.S < 0 || a.D <= 0) return fail(SKV_ERR_INVALID_ARGUMENT, "rotary: bad size");
    const bool some = a.B > 0 && a.S > 0;
    int rc;
    if ((rc = check_rows(a.q, some, "rotary", "q")) || (rc = check_rows(a.k, some, "rotary", "k")) ||
        (rc = check_rows(a.q_out, some, "rotary", "q_out")) || (rc = check_rows(a.k_out, some, "rotary", "k_out")) ||
        (rc = check_rope(a.rope, a.D, "rotary")))
        return rc;
    if (a.q.heads != a.q_out.heads || a.k.heads != a.k_out.heads || a.q.dtype != a.q_out.dtype ||
        (a.k.heads && (a.k.dtype != a.q.dtype || a.k_out.dtype != a.q.dtype)))
        return fail(SKV_ERR_SHAPE, "rotary: q, k and their outputs disagree in heads or dtype");
    const int64_t tokens = (int64_t)a.B * a.S, H = (int64_t)a.q.heads + a.k.heads;
    if (tokens == 0 || H == 0) return SKV_OK;
    if (tokens > 0x7fffffff - 64 || H * a.D > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "rotary: too many rows");
    cudaStream_t st = as_stream(stream);
    if (a.q.dtype == kF32) return launch_rotary<float>(a, st);
    if (a.q.dtype == kF16) return launch_rotary<__half>(a, st);
    return launch_rotary<__nv_bfloat16>(a, st);
}
