// What the kernels of neighbour attention share: rows in pieces of 16 bytes a lane, and how a warp's lanes divide heads and edges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dynb {

// A warp works on `heads` heads of one row at a time: G lanes a head hold the head's elements in pieces of 16 bytes (NV pieces a
// lane, piece p of lane l at element (p * G + l) * VEC), and where G * heads < 32 the rest of the warp takes further edges ("slots").
constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ void unpack(const uint4 u, float (&f)[4])
    {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4])
    {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void unpack(const uint4 u, float (&f)[8])
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Piece<__half> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ void unpack(const uint4 u, float (&f)[8])
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __half2 b = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

// Elements [at, at + VEC) of a head of `dim` elements; zeros behind its end.  `wide`: every piece starts on 16 bytes and dim is a
// multiple of VEC (the same for all lanes of a launch).
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* head, int at, int dim, bool wide)
{
    if (wide) return at < dim ? __ldg(reinterpret_cast<const uint4*>(head + at)) : make_uint4(0, 0, 0, 0);
    float f[Piece<T>::VEC];
#pragma unroll
    for (int i = 0; i < Piece<T>::VEC; i++) f[i] = at + i < dim ? Piece<T>::one(head[at + i]) : 0.0f;
    return Piece<T>::pack(f);   // exact: the values are of the type
}
template <typename T>
__device__ __forceinline__ void store_piece(T* head, int at, int dim, bool wide, const float (&f)[Piece<T>::VEC])
{
    if (wide) {
        if (at < dim) *reinterpret_cast<uint4*>(head + at) = Piece<T>::pack(f);
        return;
    }
#pragma unroll
    for (int i = 0; i < Piece<T>::VEC; i++)
        if (at + i < dim) head[at + i] = Piece<T>::round(f[i]);
}

template <int G>
__device__ __forceinline__ float head_sum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct AttnRows { const void* at; int64_t row, head; };   // strides in elements, the elements of a head are consecutive

struct AttnArgs {
    AttnRows q, k, v, d_out;
    const float* bias;          // [E, heads] or null
    const float* out32;         // [targets, heads, dim]: the result, unrounded
    const float* stats;         // [targets, 2, heads]: largest logit and 1 / sum of exponentials (a logarithm of the sum beside a
                                // largest logit of -3e38, as masks of the type's lowest value give, would be lost)
    float* delta;               // [targets, heads]: d_out . out
    void *out, *dq, *dk, *dv;   // contiguous
    float *out32_w, *stats_w, *d_bias;
    const int32_t *rows, *row_start, *src, *cols, *col_start, *in_edge, *in_dst;
    int64_t n_targets, n_sources, n_edges;
    int heads, kv_heads, shared, dim, warp_heads, wide;
    float scale;
};

cudaError_t attn_forward(const AttnArgs& a, int dtype, cudaStream_t s);
cudaError_t attn_backward_rows(const AttnArgs& a, int dtype, cudaStream_t s);
cudaError_t attn_backward_cols(const AttnArgs& a, int dtype, cudaStream_t s);

// Lanes a head and pieces a lane for a head of `dim` elements of type T.
static inline int attn_lanes(int dim, int vec)
{
    int g = 1;
    while (g < 32 && g * vec < dim) g *= 2;
    return g;
}

template <typename T, template <typename, int, int> class Launch>
static inline cudaError_t attn_by_dim(const AttnArgs& a, cudaStream_t s)
{
    switch (attn_lanes(a.dim, Piece<T>::VEC)) {
    case 1: return Launch<T, 1, 1>::go(a, s);
    case 2: return Launch<T, 2, 1>::go(a, s);
    case 4: return Launch<T, 4, 1>::go(a, s);
    case 8: return Launch<T, 8, 1>::go(a, s);
    case 16: return Launch<T, 16, 1>::go(a, s);
    default: return a.dim <= 32 * Piece<T>::VEC ? Launch<T, 32, 1>::go(a, s) : Launch<T, 32, 2>::go(a, s);
    }
}
template <template <typename, int, int> class Launch>
static inline cudaError_t attn_by_type(const AttnArgs& a, int dtype, cudaStream_t s)
{
    if (dtype == DYNB_F32) return attn_by_dim<float, Launch>(a, s);
    if (dtype == DYNB_F16) return attn_by_dim<__half, Launch>(a, s);
    return attn_by_dim<__nv_bfloat16, Launch>(a, s);
}

// Heads of a warp: as many as its lanes hold, no more than the next power of two above `heads`.
static inline int attn_warp_heads(int heads, int g)
{
    int h = 1;
    while (h < heads && h * g < 32) h *= 2;
    return h;
}

}  // namespace dynb
