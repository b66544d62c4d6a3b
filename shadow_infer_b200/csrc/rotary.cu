// Rotary positions: rows [B, H, S, D] turned pair by pair, queries and keys in one launch.
//
// A pair (a, b) of the first `rot` values of a row at position p becomes
//     (a c - b s, b c + a s),   c = cos[p][i], s = sin[p][i]   (s negated to turn back),
// with (a, b) = (x[i], x[i + rot/2]) or, interleaved, (x[2i], x[2i+1]); the other values are
// copied.  Two products and a sum a value against 2 x 2..4 bytes moved: memory-bound.
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
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ skv_rotary_args a) {
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
    if (tokens > 0x7fffffff || H * a.D > 0x7fffffff) return fail(SKV_ERR_TOO_LARGE, "rotary: too many rows");
    cudaStream_t st = as_stream(stream);
    const int64_t slices = (H * a.D + 1023) / 1024;
    const dim3 grid((unsigned)tokens, (unsigned)(slices < 65535 ? slices : 65535));
    if (a.q.dtype == kF32) rotary_kernel<float><<<grid, 256, 0, st>>>(a);
    else if (a.q.dtype == kF16) rotary_kernel<__half><<<grid, 256, 0, st>>>(a);
    else rotary_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
    return check_launch("rotary");
}
