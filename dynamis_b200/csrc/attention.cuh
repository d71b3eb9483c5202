// What the kernels of neighbour attention share: rows as 32 bytes a lane, and how a warp's lanes divide heads and edges.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dynb {

// A warp works on `warp_heads` heads of one row at a time.  G lanes a head hold 32 bytes of it each, and where G * warp_heads < 32 the rest of the
// warp takes further edges ("slots"): 32 bytes a lane leave few instructions an edge for addresses, sums over lanes and exponentials
// (forward, 8 x 16 fp32: 34 warp instructions an edge; with 16 bytes a lane, 64-bit indices and checks at every load 113, and 1.48 ms in place of 0.70 for
// 10.5 M edges).
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

struct AttnRows { const void* at; int64_t row, head; };   // strides in elements, the elements of a head are consecutive

// EL elements of a head (8 or 16) as they are loaded: pieces of 16 bytes.
template <typename T, int EL> struct Raw { uint4 v[EL * (int)sizeof(T) / 16]; };

template <typename T> __device__ __forceinline__ T attn_put(float v);
template <> __device__ __forceinline__ float attn_put<float>(float v) { return v; }
template <> __device__ __forceinline__ __half attn_put<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 attn_put<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float2 attn_pair(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 attn_pair(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T, int EL>
__device__ __forceinline__ void attn_pairs(const Raw<T, EL>& r, float2 (&f)[EL / 2])
{
#pragma unroll
    for (int p = 0; p < EL * (int)sizeof(T) / 16; p++) {
        const uint32_t w[4] = {r.v[p].x, r.v[p].y, r.v[p].z, r.v[p].w};
        if constexpr (sizeof(T) == 4) {
            f[2 * p] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
            f[2 * p + 1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) f[4 * p + i] = attn_pair(w[i], T());
        }
    }
}

// Where a lane's pieces stand in their head: 32 bytes in a row.
template <typename T, int G, int EL>
struct Place {
    static constexpr int PIECES = EL * (int)sizeof(T) / 16, VEC = 16 / (int)sizeof(T);
    int at[PIECES];
    __device__ __forceinline__ explicit Place(int part)
    {
#pragma unroll
        for (int p = 0; p < PIECES; p++) at[p] = (part * PIECES + p) * VEC;
    }
};

// FULL: heads of EL G elements that start on 32 bytes.  Otherwise `wide` says on how many bytes (16, 8 or fewer) heads start and end.
template <typename T, int G, int EL, bool FULL>
__device__ __forceinline__ Raw<T, EL> attn_load(const T* head, const Place<T, G, EL>& place, int dim, int wide)
{
    Raw<T, EL> r;
    constexpr int VEC = Place<T, G, EL>::VEC;
#pragma unroll
    for (int p = 0; p < Place<T, G, EL>::PIECES; p++) {
        const int at = place.at[p];
        if (FULL) {
            r.v[p] = __ldg(reinterpret_cast<const uint4*>(head + at));
        } else if (wide >= 16) {
            r.v[p] = at < dim ? __ldg(reinterpret_cast<const uint4*>(head + at)) : make_uint4(0, 0, 0, 0);
        } else if (wide == 8) {
            const uint2 lo = at < dim ? __ldg(reinterpret_cast<const uint2*>(head + at)) : make_uint2(0, 0);
            const uint2 hi = at + VEC / 2 < dim ? __ldg(reinterpret_cast<const uint2*>(head + at + VEC / 2)) : make_uint2(0, 0);
            r.v[p] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            __align__(16) T e[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) e[i] = at + i < dim ? head[at + i] : attn_put<T>(0.0f);
            r.v[p] = *reinterpret_cast<const uint4*>(e);
        }
    }
    return r;
}
// Rows of full heads: a lane's 32 bytes by one load, in units of 32 bytes from the tensor's start, in 32 bits (128 GB): a pointer and two loads of 16 bytes
// took five more instructions an edge.
template <typename T, int G, int EL>
struct Lane {
    const char* base;
    uint32_t step, at;
    __device__ __forceinline__ Lane(const AttnRows& rows, int head, const Place<T, G, EL>& place)
    {
        base = static_cast<const char*>(rows.at);
        step = (uint32_t)(rows.row * (int)sizeof(T) / 32);
        at = (uint32_t)((rows.head * head + place.at[0]) * (int)sizeof(T) / 32);
    }
    __device__ __forceinline__ Raw<T, EL> load(uint32_t row) const
    {
        Raw<T, EL> r;
        static_assert(sizeof(r) == 32, "a lane holds 32 bytes");
        asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(r.v[0].x), "=r"(r.v[0].y), "=r"(r.v[0].z), "=r"(r.v[0].w), "=r"(r.v[1].x), "=r"(r.v[1].y), "=r"(r.v[1].z), "=r"(r.v[1].w)
            : "l"(base + (uint64_t)(row * step + at) * 32));
        return r;
    }
};
template <typename T, int EL>
__device__ __forceinline__ void attn_clear(Raw<T, EL>& r, bool keep)
{
#pragma unroll
    for (int p = 0; p < EL * (int)sizeof(T) / 16; p++) {
        r.v[p].x = keep ? r.v[p].x : 0u;
        r.v[p].y = keep ? r.v[p].y : 0u;
        r.v[p].z = keep ? r.v[p].z : 0u;
        r.v[p].w = keep ? r.v[p].w : 0u;
    }
}
// A batch of edges on its way: what they read from two tensors, their biases, and whether they take part.  (The loads of those that do not go to
// row 0, which is there: an edge has both ends.)
template <typename T, int EL, int BATCH>
struct AttnStep {
    Raw<T, EL> x[BATCH], y[BATCH];
    float z[BATCH];
    bool ok[BATCH];

    template <int G, bool FULL>
    __device__ __forceinline__ void load(const Lane<T, G, EL>& a, const Lane<T, G, EL>& b, const Place<T, G, EL>& place, const AttnRows& ar, const AttnRows& br,
                                         int head_a, int head_b, const uint32_t (&row)[BATCH], int dim, int wide)
    {
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            if constexpr (FULL) {
                x[u] = a.load(row[u]);
                y[u] = b.load(row[u]);
            } else if (ok[u]) {
                x[u] = attn_load<T, G, EL, false>(static_cast<const T*>(ar.at) + (row[u] * ar.row + head_a * ar.head), place, dim, wide);
                y[u] = attn_load<T, G, EL, false>(static_cast<const T*>(br.at) + (row[u] * br.row + head_b * br.head), place, dim, wide);
            }
        }
    }
    // Zeros in place of what masked edges read: not even a product is formed with it.  All lanes of a warp call it.
    __device__ __forceinline__ void clear()
    {
        bool all = true;
#pragma unroll
        for (int u = 0; u < BATCH; u++) all = all && ok[u];
        if (__all_sync(0xffffffffu, all)) return;
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            attn_clear(x[u], ok[u]);
            attn_clear(y[u], ok[u]);
        }
    }
};
// f holds the elements in the lane's order of pieces.
template <typename T, int G, int EL, bool FULL>
__device__ __forceinline__ void attn_store(T* head, const Place<T, G, EL>& place, int dim, int wide, const float2 (&f)[EL / 2])
{
    constexpr int VEC = Place<T, G, EL>::VEC;
#pragma unroll
    for (int p = 0; p < Place<T, G, EL>::PIECES; p++) {
        const int at = place.at[p];
        __align__(16) T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            e[i] = attn_put<T>(f[(p * VEC + i) / 2].x);
            e[i + 1] = attn_put<T>(f[(p * VEC + i) / 2].y);
        }
        if (FULL || wide >= 16) {
            if (FULL || at < dim) *reinterpret_cast<uint4*>(head + at) = *reinterpret_cast<const uint4*>(e);
        } else if (wide == 8) {
            if (at < dim) *reinterpret_cast<uint2*>(head + at) = *reinterpret_cast<const uint2*>(e);
            if (at + VEC / 2 < dim) *reinterpret_cast<uint2*>(head + at + VEC / 2) = *reinterpret_cast<const uint2*>(e + VEC / 2);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (at + i < dim) head[at + i] = e[i];
        }
    }
}
// What stands for the operands of a row that is not there (a block's last rows, numbers out of range), read 16 bytes at a time.
static __device__ __align__(16) unsigned char attn_zeros[DYNB_ATTENTION_MAX_DIM * 4];

template <int G>
__device__ __forceinline__ float head_sum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int N>
__device__ __forceinline__ float inner(const float2 (&a)[N], const float2 (&b)[N])
{
    float2 s = mul2(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < N; i++) s = fma2(a[i], b[i], s);
    return s.x + s.y;
}

// Sources and biases of the edges [e, e + BATCH) of a slot, asked for a batch before the rows they name.
template <int BATCH>
struct AttnEdges {
    int32_t s[BATCH];
    float z[BATCH];
    __device__ __forceinline__ void fetch(const int32_t* src, const float* bias, int e, int n, int heads)
    {
        src += e;
        bias += (int64_t)e * heads;
        if (e + BATCH <= n) {
#pragma unroll
            for (int u = 0; u < BATCH; u++) s[u] = __ldg(src + u);
#pragma unroll
            for (int u = 0; u < BATCH; u++, bias += heads) z[u] = heads > 0 ? __ldg(bias) : 0.0f;
        } else {
#pragma unroll
            for (int u = 0; u < BATCH; u++, bias += heads) {
                s[u] = e + u < n ? __ldg(src + u) : -1;
                z[u] = heads > 0 && e + u < n ? __ldg(bias) : 0.0f;
            }
        }
    }
    // Rows to read and whether the edges take part.
    __device__ __forceinline__ void rows(uint32_t sources, uint32_t (&row)[BATCH], bool (&ok)[BATCH]) const
    {
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const bool in = (uint32_t)s[u] < sources;
            row[u] = in ? (uint32_t)s[u] : 0u;
            ok[u] = in && z[u] != -INFINITY;
        }
    }
};

struct AttnArgs {
    AttnRows q, k, v, d_out;
    const float* bias;          // [E, heads] or null
    const float* out32;         // [targets, heads, dim]: the result, unrounded
    const float* stats;         // [targets, 2, heads]: largest logit and 1 / sum of exponentials (a logarithm of the sum beside a
                                // largest logit of -3e38, as masks of the type's lowest value give, would be lost)
    float4* delta;              // [targets, heads]: largest logit, 1 / sum, d_out . out, 0 (one load an edge for the pass by source)
    void *out, *dq, *dk, *dv;   // contiguous
    float *out32_w, *stats_w, *d_bias;
    const int32_t *rows, *row_start, *src, *cols, *col_start, *in_edge, *in_dst;
    int64_t n_targets, n_sources, n_edges;
    int heads, kv_heads, shared, dim, warp_heads;
    int wide;                   // bytes on which all heads start and end: 32, 16, 8 or fewer
    int narrow;                 // offsets in units of 32 bytes fit 32 bits
    int block_rows;             // rows of a block, a multiple of those that it takes at once
    float scale;
};

cudaError_t attn_forward(const AttnArgs& a, int dtype, cudaStream_t s);
cudaError_t attn_backward_rows(const AttnArgs& a, int dtype, cudaStream_t s);
cudaError_t attn_backward_cols(const AttnArgs& a, int dtype, cudaStream_t s);

// Elements a lane: 32 bytes.
template <typename T> struct LaneElements { static constexpr int N = 32 / (int)sizeof(T); };

template <typename T, template <typename, int, bool> class Launch, int G>
static inline cudaError_t attn_by_full(const AttnArgs& a, cudaStream_t s)
{
    return a.wide == 32 && a.narrow && a.dim == LaneElements<T>::N * G ? Launch<T, G, true>::go(a, s) : Launch<T, G, false>::go(a, s);
}
template <typename T, template <typename, int, bool> class Launch>
static inline cudaError_t attn_by_dim(const AttnArgs& a, cudaStream_t s)
{
    const int lanes = (a.dim + LaneElements<T>::N - 1) / LaneElements<T>::N;
    if (lanes <= 1) return attn_by_full<T, Launch, 1>(a, s);
    if (lanes <= 2) return attn_by_full<T, Launch, 2>(a, s);
    if (lanes <= 4) return attn_by_full<T, Launch, 4>(a, s);
    if (lanes <= 8) return attn_by_full<T, Launch, 8>(a, s);
    if constexpr (sizeof(T) == 4) {
        if (lanes > 16) return attn_by_full<T, Launch, 32>(a, s);
    }
    return attn_by_full<T, Launch, 16>(a, s);
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

// Rows of a block that takes `at_once` at once: neighbouring rows read the same rows of the other side, so a block goes on with the next ones
// while L1 holds these, as long as there are eight blocks for every place on the SMs (200 k targets, 8 x 16 fp32, forward and gradients: a turn 2793 us, two
// 2664, four 2632, eight 2647).
constexpr int ATTN_TURNS = 4;
static inline int attn_block_rows(int64_t rows, int at_once)
{
    int turns = ATTN_TURNS;
    while (turns > 1 && rows < (int64_t)at_once * turns * 148 * 4 * 8) turns /= 2;
    return at_once * turns;
}
// Whether four warps share a row: where there are too few rows for the SMs (148 x 16 warps), or the lists are long.
static inline bool attn_split(int64_t warps, int64_t edges) { return warps < 148 * 16 || edges > warps * 512; }

}  // namespace dynb
