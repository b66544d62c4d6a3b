// What the page pool's kernels share: typed row access, page lookup and the decode of a page row.
#pragma once

#include <cuda_bf16.h>

#include "skv_common.cuh"

namespace skv {

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };   // skv_rows.dtype

__host__ __device__ inline int dtype_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 8 consecutive values as loaded, so that several loads are on the way before the first is widened.
template <class T> struct Raw8 {   // 16-bit types
    uint4 v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T* h = reinterpret_cast<const T*>(&w[i]);
            x[2 * i] = to_float(h[0]);
            x[2 * i + 1] = to_float(h[1]);
        }
    }
};
template <> struct Raw8<float> {
    float4 u, v;
    __device__ __forceinline__ void load(const float* p) {
        u = reinterpret_cast<const float4*>(p)[0];
        v = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    }
};

// 8 consecutive values (16-byte aligned rows).
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A number that the kernel only reads.  FRESH: one that it may have written itself, or has waited for after it had started
// (wait_for_dependency): a read-only load could be moved before that.
template <bool FRESH, class T>
__device__ __forceinline__ T number_at(const T* p) {
    if constexpr (FRESH) return *p;
    else return __ldg(p);
}

// The pool row (all heads of a page counted, head 0's block) that holds token t of sequence b, or
// -1 where the table names no page for it.  + head * page_size gives the head's row.
template <bool FRESH = false>
__device__ __forceinline__ int64_t pool_row(const skv_pool& p, int b, int64_t t) {
    if (t < 0 || t >= (int64_t)p.table_width * p.page_size) return -1;
    const int64_t j = t <= 0xffffffffll ? (int64_t)((uint32_t)t / (uint32_t)p.page_size) : t / p.page_size;
    const int page = number_at<FRESH>(p.block_table + b * p.table_stride + j);
    if (page < 0 || page >= p.num_pages) return -1;
    return (int64_t)page * p.heads * p.page_size + (t - j * p.page_size);
}

__host__ __device__ inline int64_t pool_row_bytes(int precision, int D) {
    return precision == 0 ? (int64_t)D * 4 : precision == 1 ? (int64_t)D * 2 : precision == 2 ? D : ((int64_t)D + 1) / 2;
}

// Value col of pool rows, any D and group; block: col / int4_group.
template <int PREC, bool FRESH = false>
__device__ __forceinline__ float pool_value(const skv_pool& p, bool is_v, int64_t row, int col, int block) {
    const uint8_t* base = static_cast<const uint8_t*>(is_v ? p.v : p.k);
    const float* sc = is_v ? p.scale_v : p.scale_k;
    const int D = p.head_dim;
    if constexpr (PREC == 0) return number_at<FRESH>(reinterpret_cast<const float*>(base) + row * D + col);
    else if constexpr (PREC == 1) return __half2float(number_at<FRESH>(reinterpret_cast<const __half*>(base) + row * D + col));
    else if constexpr (PREC == 2) return __fmul_rn((float)number_at<FRESH>(reinterpret_cast<const signed char*>(base) + row * D + col), number_at<FRESH>(sc + row));
    else {
        const uint8_t byte = number_at<FRESH>(base + row * ((D + 1) / 2) + col / 2);
        const int q = (col & 1) ? (byte & 15) : (byte >> 4);
        return __fmul_rn((float)(q - 8), number_at<FRESH>(sc + row * (D / p.int4_group) + block));
    }
}

// V consecutive values (4 or 8) of a pool row as loaded, with their scale; D and the int4 group multiples of 8, aligned payload.
template <int PREC, int V> struct PoolRaw {
    static constexpr int BYTES = V * (PREC == 0 ? 4 : PREC == 1 ? 2 : 1) / (PREC == 3 ? 2 : 1), WORDS = (BYTES + 3) / 4;
    uint32_t w[WORDS];
    float s;
    __device__ __forceinline__ void load(const skv_pool& p, bool is_v, int64_t row, int col) {
        const char* base = static_cast<const char*>(is_v ? p.v : p.k) + (PREC == 3 ? (row * p.head_dim + col) / 2
                                                                                   : (row * p.head_dim + col) * (PREC == 0 ? 4 : PREC == 1 ? 2 : 1));
        if constexpr (BYTES == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(base);
        } else if constexpr (BYTES == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(base);
        } else if constexpr (BYTES == 8) {
            const uint2 u = *reinterpret_cast<const uint2*>(base);
            w[0] = u.x; w[1] = u.y;
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const uint4 u = reinterpret_cast<const uint4*>(base)[i];
                w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
            }
        }
        const float* sc = is_v ? p.scale_v : p.scale_k;
        s = PREC == 2 ? sc[row] : PREC == 3 ? sc[row * (p.head_dim / p.int4_group) + col / p.int4_group] : 1.0f;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = PREC == 3 ? 0x88888888u : 0u;
        s = 0.0f;
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (PREC == 0) return __uint_as_float(w[i]);
        else if constexpr (PREC == 1) return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1)))));
        else if constexpr (PREC == 2) return __fmul_rn((float)(int8_t)(w[i / 4] >> (8 * (i & 3))), s);
        else return __fmul_rn((float)((int)((w[i / 8] >> (8 * ((i % 8) / 2) + (i & 1 ? 0 : 4))) & 15u) - 8), s);
    }
};

// The position of token s of sequence b: rope.positions, or `own`.
__device__ __forceinline__ int64_t rope_position(const skv_rope& r, int b, int s, int64_t own) {
    if (r.positions == nullptr) return own;
    const int64_t i = b * r.pos_stride_b + s * r.pos_stride_s;
    return r.pos_bytes == 8 ? static_cast<const int64_t*>(r.positions)[i]
                            : (int64_t) static_cast<const int32_t*>(r.positions)[i];
}

// The two outputs of a pair; every product and sum rounded by itself (no contraction), so that the
// keys a cache quantises do not depend on how a kernel was compiled.
__device__ __forceinline__ float rope_first(float a, float b, float c, float s) {
    return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float rope_second(float a, float b, float c, float s) {
    return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

// Host checks shared by the entry points; SKV_OK or the recorded failure.
int check_pool(const skv_pool& p, const char* what);
int check_rows(const skv_rows& r, bool some, const char* what, const char* name);   // some: there are tokens
int check_rope(const skv_rope& r, int D, const char* what);

// Whether rows can be read 8 values at a time: address and strides on 16-byte boundaries.
inline bool rows_aligned(const skv_rows& r) {
    const int per = 16 / dtype_bytes(r.dtype);
    return r.heads == 0 || ((reinterpret_cast<uintptr_t>(r.ptr) & 15) == 0 && r.stride_b % per == 0 &&
                            r.stride_h % per == 0 && r.stride_s % per == 0);
}

}  // namespace skv
