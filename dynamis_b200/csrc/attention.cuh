// What the kernels of neighbour attention share: rows in pieces of 16 bytes a lane, and how a warp's lanes divide heads and edges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dynb {

// A warp works on `warp_heads` heads of one row at a time.  G lanes a head hold eight of its elements each, and where G * warp_heads < 32 the
// rest of the warp takes further edges ("slots"): eight elements a lane leave few instructions for addresses, sums over lanes and exponentials
// per edge, which is what bounds these kernels (113 warp instructions an edge and 1.48 ms with four elements a lane, 64-bit indices and checks at
// every load, forward, 10.5 M edges of 8 x 16 fp32).
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float2 fma2(const float2 a, const float2 b, const float2 c)
{
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)),
          "l"(*reinterpret_cast<const unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(const float2 a, const float2 b)
{
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
// 2^x to 2 ulp; results below the smallest normal number are zero.
__device__ __forceinline__ float pow2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Eight elements of a head as they are loaded.
template <typename T> struct Raw { uint4 v[sizeof(T) / 2]; };

template <typename T> __device__ __forceinline__ float attn_get(T v);
template <> __device__ __forceinline__ float attn_get<float>(float v) { return v; }
template <> __device__ __forceinline__ float attn_get<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float attn_get<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T attn_put(float v);
template <> __device__ __forceinline__ float attn_put<float>(float v) { return v; }
template <> __device__ __forceinline__ __half attn_put<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 attn_put<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void attn_pairs(const Raw<float>& r, float2 (&f)[4])
{
#pragma unroll
    for (int p = 0; p < 2; p++) {
        f[2 * p] = make_float2(__uint_as_float(r.v[p].x), __uint_as_float(r.v[p].y));
        f[2 * p + 1] = make_float2(__uint_as_float(r.v[p].z), __uint_as_float(r.v[p].w));
    }
}
__device__ __forceinline__ void attn_pairs(const Raw<__nv_bfloat16>& r, float2 (&f)[4])
{
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void attn_pairs(const Raw<__half>& r, float2 (&f)[4])
{
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}

// Where a lane's elements stand in their head.  Two pieces of 16 bytes in fp32, of which every second run of lanes takes the second one first:
// eight lanes then meet eight different pieces of 128 bytes, whatever G is.  One piece in 16 bits.
template <typename T, int G>
struct Place {
    static constexpr int PIECES = (int)sizeof(T) / 2, VEC = 16 / (int)sizeof(T);
    int at[PIECES];
    __device__ __forceinline__ Place(int part, int head)
    {
#pragma unroll
        for (int p = 0; p < PIECES; p++) at[p] = PIECES == 1 ? part * VEC : ((p ^ ((head * G >> 2) & 1)) * G + part) * VEC;
    }
};

// FULL: heads of 8 G elements whose pieces start on 16 bytes.  Otherwise `wide` says whether pieces do (and end with the head).
template <typename T, int G, bool FULL>
__device__ __forceinline__ Raw<T> attn_load(const T* head, const Place<T, G>& place, int dim, bool wide)
{
    Raw<T> r;
    constexpr int VEC = Place<T, G>::VEC;
#pragma unroll
    for (int p = 0; p < Place<T, G>::PIECES; p++) {
        const int at = place.at[p];
        if (FULL) {
            r.v[p] = __ldg(reinterpret_cast<const uint4*>(head + at));
        } else if (wide) {
            r.v[p] = at < dim ? __ldg(reinterpret_cast<const uint4*>(head + at)) : make_uint4(0, 0, 0, 0);
        } else {
            __align__(16) T e[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) e[i] = at + i < dim ? head[at + i] : attn_put<T>(0.0f);
            r.v[p] = *reinterpret_cast<const uint4*>(e);
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ Raw<T> attn_nothing()
{
    Raw<T> r;
#pragma unroll
    for (int p = 0; p < (int)(sizeof(T) / 2); p++) r.v[p] = make_uint4(0, 0, 0, 0);
    return r;
}
// f holds the pieces in the lane's order: pairs 0, 1 of piece 0, then of piece 1 (fp32), or the four pairs of the one piece.
template <typename T, int G, bool FULL>
__device__ __forceinline__ void attn_store(T* head, const Place<T, G>& place, int dim, bool wide, const float2 (&f)[4])
{
    constexpr int VEC = Place<T, G>::VEC;
#pragma unroll
    for (int p = 0; p < Place<T, G>::PIECES; p++) {
        const int at = place.at[p];
        __align__(16) T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            e[i] = attn_put<T>(f[(p * VEC + i) / 2].x);
            e[i + 1] = attn_put<T>(f[(p * VEC + i) / 2].y);
        }
        if (FULL || wide) {
            if (FULL || at < dim) *reinterpret_cast<uint4*>(head + at) = *reinterpret_cast<const uint4*>(e);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (at + i < dim) head[at + i] = e[i];
        }
    }
}

template <int G>
__device__ __forceinline__ float head_sum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float dot8(const float2 (&a)[4], const float2 (&b)[4])
{
    float2 s = mul2(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < 4; i++) s = fma2(a[i], b[i], s);
    return s.x + s.y;
}

// Sources and biases of the edges [e, e + BATCH) of a slot, asked for a batch before the rows they name.
template <int BATCH>
struct AttnEdges {
    int32_t s[BATCH];
    float z[BATCH];
    __device__ __forceinline__ void fetch(const int32_t* src, const float* bias, int e, int n, int heads)
    {
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            s[u] = e + u < n ? __ldg(src + e + u) : -1;
            z[u] = 0.0f;
            if (bias != nullptr && e + u < n) z[u] = __ldg(bias + (int64_t)(e + u) * heads);
        }
    }
    __device__ __forceinline__ bool live(int u, uint32_t sources) const { return (uint32_t)s[u] < sources && z[u] != -INFINITY; }
};

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

// Lanes a head.
static inline int attn_lanes(int dim)
{
    int g = 1;
    while (g * 8 < dim) g *= 2;
    return g;
}

template <typename T, template <typename, int, bool> class Launch, int G>
static inline cudaError_t attn_by_full(const AttnArgs& a, cudaStream_t s)
{
    return a.wide && a.dim == 8 * G ? Launch<T, G, true>::go(a, s) : Launch<T, G, false>::go(a, s);
}
template <typename T, template <typename, int, bool> class Launch>
static inline cudaError_t attn_by_dim(const AttnArgs& a, cudaStream_t s)
{
    switch (attn_lanes(a.dim)) {
    case 1: return attn_by_full<T, Launch, 1>(a, s);
    case 2: return attn_by_full<T, Launch, 2>(a, s);
    case 4: return attn_by_full<T, Launch, 4>(a, s);
    case 8: return attn_by_full<T, Launch, 8>(a, s);
    case 16: return attn_by_full<T, Launch, 16>(a, s);
    default: return attn_by_full<T, Launch, 32>(a, s);
    }
}
template <template <typename, int, bool> class Launch>
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

// Whether four warps share a row: where there are too few rows for the SMs (148 x 16 warps), or the lists are long.
static inline bool attn_split(int64_t warps, int64_t edges) { return warps < 148 * 16 || edges > warps * 512; }

}  // namespace dynb
