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
__global__ void __launch_bounds__(32 * kPoolWarps) pool_append_kernel(const __grid_constant__ skv_pool_append_args a) {
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

// A warp per (token, head) row of K and of V.
template <class T>
__global__ void __launch_bounds__(32 * kPoolWarps) pool_read_kernel(const __grid_constant__ skv_pool_read_args a) {
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
    const int threads = 32 * kPoolWarps;
    if (a.k.dtype == kF32) pool_append_kernel<float><<<(unsigned)blocks, threads, 0, st>>>(a);
    else if (a.k.dtype == kF16) pool_append_kernel<__half><<<(unsigned)blocks, threads, 0, st>>>(a);
    else pool_append_kernel<__nv_bfloat16><<<(unsigned)blocks, threads, 0, st>>>(a);
    return check_launch("pool_append");
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
    const int threads = 32 * kPoolWarps;
    if (a.k_out.dtype == kF32) pool_read_kernel<float><<<(unsigned)blocks, threads, 0, st>>>(a);
    else if (a.k_out.dtype == kF16) pool_read_kernel<__half><<<(unsigned)blocks, threads, 0, st>>>(a);
    else pool_read_kernel<__nv_bfloat16><<<(unsigned)blocks, threads, 0, st>>>(a);
    return check_launch("pool_read");
}

}  // extern "C"
