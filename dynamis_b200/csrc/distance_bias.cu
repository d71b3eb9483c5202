// A learned bias of attention logits from distances (no counterpart in the reference): `buckets` values a head over the distances
// [0, cutoff], joined by cubic B-splines so that forces are continuous, and a switch function at the cutoff.  With u = r / cutoff,
// x = u (buckets - 3), i = floor(x), t = x - i:
//     bias[e, h] = sum_j w_j(t) table[i + j, h] + log f(u),   f(u) = (1 - u)^3 (1 + 3 u + 6 u^2)   (the last term if `smooth`),
// and -inf from the cutoff on: these pairs take no part in the attention.  f has two continuous derivatives of zero at the cutoff,
// so an attention weight, which is proportional to it, comes and goes smoothly.
// Gradients: d_dist = sum_h g_h (sum_j w'_j table[i + j, h] (buckets - 3) - 30 u^2 / ((1 - u)(1 + 3 u + 6 u^2))) / cutoff and
// d_table[i + j, h] += w_j g_h.  1 - u is taken as (cutoff - r) / cutoff, which is exact next to the cutoff.

#include <algorithm>

#include "common.cuh"

namespace dynb {

constexpr int DB_THREADS = 256;

struct DbArgs {
    const float *dist, *table, *d_bias;
    float *bias, *d_dist, *partial, *d_table;
    int64_t n;
    int heads, buckets, smooth;
    float cutoff;
};

struct DbPlace {
    int at;
    float t, u, rest;
    bool inside;
};

__device__ __forceinline__ DbPlace db_place(float r, const DbArgs& a)
{
    DbPlace p;
    const float pos = r < 0.0f ? 0.0f : r;   // NaN stays
    p.inside = !(pos >= a.cutoff);
    p.u = pos / a.cutoff;
    p.rest = (a.cutoff - pos) / a.cutoff;
    const float x = p.u * (float)(a.buckets - 3);
    p.at = min(max((int)x, 0), a.buckets - 4);
    p.t = x - (float)p.at;
    return p;
}

__device__ __forceinline__ void db_weights(float t, float (&w)[4])
{
    const float m = 1.0f - t;
    w[0] = m * m * m * (1.0f / 6.0f);
    w[1] = fmaf(t * t, fmaf(t, 0.5f, -1.0f), 2.0f / 3.0f);
    w[2] = fmaf(m * m, fmaf(m, 0.5f, -1.0f), 2.0f / 3.0f);
    w[3] = t * t * t * (1.0f / 6.0f);
}
__device__ __forceinline__ void db_slopes(float t, float (&w)[4])
{
    const float m = 1.0f - t;
    w[0] = -0.5f * m * m;
    w[1] = t * fmaf(t, 1.5f, -2.0f);
    w[2] = -m * fmaf(m, 1.5f, -2.0f);
    w[3] = 0.5f * t * t;
}

__global__ void __launch_bounds__(DB_THREADS)
db_forward_kernel(const DbArgs a)
{
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < a.n; e += (int64_t)gridDim.x * blockDim.x) {
        const DbPlace p = db_place(a.dist[e], a);
        float w[4];
        db_weights(p.t, w);
        float add = 0.0f;
        if (a.smooth) add = 3.0f * logf(p.rest) + logf(fmaf(p.u, fmaf(p.u, 6.0f, 3.0f), 1.0f));
        for (int h = 0; h < a.heads; h++) {
            float v = add;
#pragma unroll
            for (int j = 0; j < 4; j++) v = fmaf(w[j], a.table[(p.at + j) * a.heads + h], v);
            a.bias[e * a.heads + h] = p.inside ? v : -INFINITY;
        }
    }
}

__global__ void __launch_bounds__(DB_THREADS)
db_dist_kernel(const DbArgs a)
{
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < a.n; e += (int64_t)gridDim.x * blockDim.x) {
        const float r = a.dist[e];
        const DbPlace p = db_place(r, a);
        float w[4];
        db_slopes(p.t, w);
        const float pull = a.smooth ? -30.0f * p.u * p.u / (p.rest * fmaf(p.u, fmaf(p.u, 6.0f, 3.0f), 1.0f)) : 0.0f;
        float sum = 0.0f;
        if (p.inside)
            for (int h = 0; h < a.heads; h++) {
                float v = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) v = fmaf(w[j], a.table[(p.at + j) * a.heads + h], v);
                sum = fmaf(a.d_bias[e * a.heads + h], fmaf(v, (float)(a.buckets - 3), pull), sum);
            }
        a.d_dist[e] = r < 0.0f ? 0.0f : sum / a.cutoff;
    }
}

// Gradient of the table.  A warp's lanes are `slots` edges times `wide` heads; every slot has a copy of the table in shared memory that
// no other slot touches, so the sums need no atomics and their order is that of the edges.  Blocks take fixed stretches of the
// edges and write their sums; db_table_join_kernel adds these in 64 bits.
__global__ void
db_table_kernel(const DbArgs a, int wide)
{
    extern __shared__ float copies[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, slots = 32 / wide;
    const int h = blockIdx.y * wide + lane % wide, slot = lane / wide;
    const bool live = h < a.heads;
    const int words = a.buckets * 32;
    for (int i = threadIdx.x; i < warps * words; i += blockDim.x) copies[i] = 0.0f;
    __syncthreads();
    float* const mine = copies + warp * words + slot * a.buckets * wide + lane % wide;
    const int64_t per = (a.n + gridDim.x - 1) / gridDim.x;
    const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, a.n);
    for (int64_t e = begin + warp * slots + slot; e < end; e += (int64_t)warps * slots) {
        const DbPlace p = db_place(a.dist[e], a);
        if (!p.inside || !live) continue;
        const float g = a.d_bias[e * a.heads + h];
        float w[4];
        db_weights(p.t, w);
#pragma unroll
        for (int j = 0; j < 4; j++) mine[(p.at + j) * wide] = fmaf(w[j], g, mine[(p.at + j) * wide]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.buckets * wide; i += blockDim.x) {
        const int hh = blockIdx.y * wide + i % wide;
        if (hh >= a.heads) continue;
        float sum = 0.0f;
        for (int c = 0; c < warps; c++)
            for (int s = 0; s < slots; s++) sum += copies[c * words + s * a.buckets * wide + i];
        a.partial[((int64_t)blockIdx.x * a.buckets + i / wide) * a.heads + hh] = sum;
    }
}

__global__ void __launch_bounds__(DB_THREADS)
db_table_join_kernel(const DbArgs a, int blocks)
{
    const int64_t cells = (int64_t)a.buckets * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < cells; i += (int64_t)gridDim.x * blockDim.x) {
        double sum = 0.0;
        for (int b = 0; b < blocks; b++) sum += (double)a.partial[b * cells + i];
        a.d_table[i] = (float)sum;
    }
}

static int db_table_blocks(int64_t n)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>((n + 1023) / 1024, 148));
}

static int db_check(int64_t n, int heads, int buckets, double cutoff)
{
    if (n < 0) return fail_arg("distance_bias: sizes must be non-negative");
    if (heads < 1 || heads > DYNB_DISTANCE_BIAS_MAX_HEADS) return fail_arg("distance_bias: heads must lie in [1, 1024]");
    if (buckets < 4 || buckets > DYNB_DISTANCE_BIAS_MAX_BUCKETS) return fail_arg("distance_bias: buckets must lie in [4, 1024]");
    if (!(cutoff > 0.0) || !(cutoff < 3.0e38)) return fail_arg("distance_bias: cutoff must be positive and finite");
    return DYNB_OK;
}

static unsigned db_blocks(int64_t n)
{
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + DB_THREADS - 1) / DB_THREADS, (int64_t)sm_count_cached() * 8));
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_distance_bias(const float* dist_dev, int64_t n, const float* table_dev, int buckets, int heads, double cutoff, int smooth,
                                  float* bias_dev, void* stream)
{
    const int rc = db_check(n, heads, buckets, cutoff);
    if (rc != DYNB_OK) return rc;
    if (n == 0) return DYNB_OK;
    if (!dist_dev || !table_dev || !bias_dev) return fail_arg("null pointer");
    DbArgs a = {};
    a.dist = dist_dev; a.table = table_dev; a.bias = bias_dev;
    a.n = n; a.heads = heads; a.buckets = buckets; a.smooth = smooth; a.cutoff = (float)cutoff;
    db_forward_kernel<<<db_blocks(n), DB_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(a);
    DYNB_CUDA_OK(cudaGetLastError());
    return DYNB_OK;
}

extern "C" int dynb_distance_bias_workspace_bytes(int64_t n, int buckets, int heads, int64_t* bytes)
{
    if (bytes == nullptr) return fail_arg("null pointer");
    const int rc = db_check(n, heads, buckets, 1.0);
    if (rc != DYNB_OK) return rc;
    *bytes = (int64_t)db_table_blocks(n) * buckets * heads * 4;
    return DYNB_OK;
}

extern "C" int dynb_distance_bias_backward(const float* dist_dev, int64_t n, const float* table_dev, int buckets, int heads, double cutoff,
                                           int smooth, const float* d_bias_dev, float* d_dist_dev, float* d_table_dev, void* workspace_dev,
                                           int64_t workspace_bytes, void* stream)
{
    const int rc = db_check(n, heads, buckets, cutoff);
    if (rc != DYNB_OK) return rc;
    if (n > 0 && (!dist_dev || !table_dev || !d_bias_dev)) return fail_arg("null pointer");
    DbArgs a = {};
    a.dist = dist_dev; a.table = table_dev; a.d_bias = d_bias_dev; a.d_dist = d_dist_dev; a.d_table = d_table_dev;
    a.n = n; a.heads = heads; a.buckets = buckets; a.smooth = smooth; a.cutoff = (float)cutoff;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d_dist_dev != nullptr && n > 0) {
        db_dist_kernel<<<db_blocks(n), DB_THREADS, 0, s>>>(a);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    if (d_table_dev != nullptr) {
        const int blocks = db_table_blocks(n);
        if (workspace_dev == nullptr || workspace_bytes < (int64_t)blocks * buckets * heads * 4) return fail_arg("workspace too small");
        a.partial = static_cast<float*>(workspace_dev);
        int wide = 1;
        while (wide < heads && wide < 32) wide *= 2;
        // as many warps as have their copies in 128 KB, and no more than 16
        const int warps = std::max(1, std::min(16, (128 << 10) / (buckets * 128)));
        const int smem = warps * buckets * 128;
        DYNB_CUDA_OK(cudaFuncSetAttribute(db_table_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        db_table_kernel<<<dim3(blocks, (heads + wide - 1) / wide), warps * 32, smem, s>>>(a, wide);
        DYNB_CUDA_OK(cudaGetLastError());
        const unsigned join = (unsigned)std::min<int64_t>(((int64_t)buckets * heads + DB_THREADS - 1) / DB_THREADS, 1024);
        db_table_join_kernel<<<join, DB_THREADS, 0, s>>>(a, blocks);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    return DYNB_OK;
}
