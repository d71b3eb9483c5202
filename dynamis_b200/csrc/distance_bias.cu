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
constexpr int DB_COPIES_BYTES = 40 << 10;  // eight copies of a table
constexpr int DB_TABLE_BYTES = 24 << 10;   // tables that blocks copy to shared memory: eight blocks an SM hold one each

struct DbArgs {
    const float *dist, *table, *d_bias;
    float *bias, *d_dist, *partial, *d_table;
    int64_t n;
    int heads, buckets, smooth;
    float cutoff, per;   // per: (buckets - 3) / cutoff
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
    // What rounding took from the quotient and from the product comes back behind the subtraction, which is exact: t is off by 2^-24 whatever the number
    // of buckets is (without it by 2^-24 of x; both products that it takes are exact).  A t that falls beside [0, 1] by it stays with its bucket: the neighbour's
    // cubic differs by the third power of that.
    const float pieces = (float)(a.buckets - 3), x = p.u * pieces;
    p.at = min(max((int)x, 0), a.buckets - 4);
    p.t = (x - (float)p.at) + fmaf(fmaf(-p.u, a.cutoff, pos), a.per, fmaf(p.u, pieces, -x));
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

// log f(u): one logarithm of the product, which is at least 2^-72.
__device__ __forceinline__ float db_switch(const DbPlace& p)
{
    return logf(p.rest * p.rest * p.rest * fmaf(p.u, fmaf(p.u, 6.0f, 3.0f), 1.0f));
}

// A thread takes VEC heads of an edge.  Eight of them where the table fits into shared memory eight times: four heads of a bucket are 16 bytes, which stand
// there in eight copies beside one another, one for each of the eight lanes that are served at once, so that no two of them meet in a bank
// whatever their distances are.  Otherwise the table is in shared memory once (IN_SMEM) or stays where it is.  10.5 M edges, 64 x 8: four heads a
// thread and one copy 112 us, eight heads and one copy 156.
template <int VEC, bool IN_SMEM>
__global__ void __launch_bounds__(DB_THREADS)
db_forward_kernel(const DbArgs a)
{
    extern __shared__ __align__(16) float copies[];
    const float* const table = IN_SMEM ? copies + (VEC == 8 ? threadIdx.x % 8 * 4 : 0) : a.table;
    if (IN_SMEM) {
        if (VEC == 8) {
            for (int i = threadIdx.x; i < a.buckets * a.heads * 8; i += DB_THREADS) {
                const int line = i >> 5, four = line / a.buckets;   // lines of 32 floats: buckets of heads 0 to 3, of heads 4 to 7, ...
                copies[i] = a.table[(line - four * a.buckets) * a.heads + 4 * four + (i & 3)];
            }
        } else {
            for (int i = threadIdx.x; i < a.buckets * a.heads; i += DB_THREADS) copies[i] = a.table[i];
        }
        __syncthreads();
    }
    const uint32_t per = (uint32_t)(a.heads / VEC);
    const int64_t total = a.n * per;
    for (int64_t i = (int64_t)blockIdx.x * DB_THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * DB_THREADS) {
        const int64_t e = per == 2 ? i >> 1 : per == 1 ? i : i / per;
        const int h = (int)(i - e * per) * VEC;
        const DbPlace p = db_place(__ldg(a.dist + e), a);
        float w[4], v[VEC];
        db_weights(p.t, w);
        const float add = a.smooth ? db_switch(p) : 0.0f;
#pragma unroll
        for (int k = 0; k < VEC; k++) v[k] = add;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float* const row = VEC == 8 ? table + (h / 4 * a.buckets + p.at + j) * 32 : table + (p.at + j) * a.heads + h;
            if constexpr (VEC == 1) {
                v[0] = fmaf(w[j], row[0], v[0]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; k += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(row + (k == 0 ? 0 : a.buckets * 32));
                    v[k] = fmaf(w[j], t.x, v[k]);
                    v[k + 1] = fmaf(w[j], t.y, v[k + 1]);
                    v[k + 2] = fmaf(w[j], t.z, v[k + 2]);
                    v[k + 3] = fmaf(w[j], t.w, v[k + 3]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < VEC; k++) v[k] = p.inside ? v[k] : -INFINITY;
        float* const out = a.bias + e * a.heads + h;
        if constexpr (VEC == 1) {
            out[0] = v[0];
        } else if constexpr (VEC == 4) {
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                         "f"(v[6]), "f"(v[7])
                         : "memory");
        }
    }
}

// Both gradients from one reading of the bias's gradient, for up to 32 heads.  A warp takes 32 edges at a time: every lane works out the
// place, the weights and the slopes of one of them, then WIDE rounds follow in which the lanes are 32 / WIDE edges times WIDE heads.  A lane has
// a column of its own in the warp's copy of the table's gradient, [buckets][32]: no atomics, no two lanes in one bank, and the order of
// its sums is that of the edges.  Sums of a column and of a block are in 32 bits: short ones (10.5 M edges, 64 x 8: a column of fifty terms, 88
// columns a block) whose roundings are independent; db_table_join_kernel adds those of the blocks in 64.
// What bounds it are the 16 reads and writes of shared memory a round, at 77 % of the pipe's peak, and the chain of read, sum and write of a column (10.5 M edges,
// 64 x 8: 0.30 ms, 1.3 TB/s; 16 warps 0.33).  The two gradients in kernels of their own, without rounds: 0.30 and 1.10 ms.  The table's sums are made
// also when nobody wants them (d_dist alone: 0.29 ms).  A warp's copy takes 128 bytes a bucket, so the warps go down with the buckets: 0.30 ms up to 64, 0.46 with
// 128, 0.93 with 256, 2.2 with 512, 4.5 with 700.
constexpr int DB_SCRATCH = 32 * 12;   // floats of a warp: weights, slopes, {place, pull} of 32 edges, 16 + 16 + 16 bytes each
template <int WIDE>
__global__ void __launch_bounds__(704, 1)
db_backward_kernel(const DbArgs a)
{
    extern __shared__ __align__(16) float copies[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr int SLOTS = 32 / WIDE;
    const int h = lane % WIDE, slot = lane / WIDE, words = a.buckets * 32;
    float* const table = copies;                                   // [buckets][32], the columns of a slot each
    float* const mine = copies + words + warp * (words + DB_SCRATCH);
    float4* const weights = reinterpret_cast<float4*>(mine + words);
    float4* const slopes = weights + 32;
    float2* const places = reinterpret_cast<float2*>(slopes + 32);
    for (int i = threadIdx.x; i < words; i += blockDim.x) {
        const int hh = i % WIDE;
        table[i] = a.d_dist != nullptr && hh < a.heads ? a.table[i / 32 * a.heads + hh] : 0.0f;
    }
    for (int i = lane; i < words; i += 32) mine[i] = 0.0f;
    __syncthreads();
    const bool live = h < a.heads;
    const float pieces = (float)(a.buckets - 3);
    const int64_t step = (int64_t)gridDim.x * warps * 32;
    int64_t base = ((int64_t)blockIdx.x * warps + warp) * 32;
    auto distance = [&](int64_t at) { return at + lane < a.n ? __ldg(a.dist + at + lane) : INFINITY; };
    float r = distance(base);
    for (; base < a.n; base += step) {
        float g[WIDE];
#pragma unroll
        for (int k = 0; k < WIDE; k++) {
            const int64_t e = base + k * SLOTS + slot;
            g[k] = live && e < a.n ? __ldg(a.d_bias + e * a.heads + h) : 0.0f;
        }
        const float r_next = distance(base + step);
        const DbPlace p = db_place(r, a);
        float w[4], s[4];
        db_weights(p.t, w);
        db_slopes(p.t, s);
        // 1 / cutoff is taken at the end; pull: slope of the switch times the cutoff
        const float pull = a.smooth && p.inside ? -30.0f * p.u * p.u / (p.rest * fmaf(p.u, fmaf(p.u, 6.0f, 3.0f), 1.0f)) : 0.0f;
        __syncwarp();
        const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        weights[lane] = p.inside ? make_float4(w[0], w[1], w[2], w[3]) : none;
        slopes[lane] = p.inside ? make_float4(s[0] * pieces, s[1] * pieces, s[2] * pieces, s[3] * pieces) : none;
        places[lane] = make_float2(__int_as_float(p.inside ? p.at : -1), pull);
        __syncwarp();
        float total = 0.0f;   // of edge base + lane, once its round has come
#pragma unroll
        for (int k = 0; k < WIDE; k++) {
            const int at_edge = k * SLOTS + slot;
            const float2 where = places[at_edge];
            const int at = max(__float_as_int(where.x), 0);
            const float gk = __float_as_int(where.x) < 0 ? 0.0f : g[k];   // beyond the cutoff: whatever the gradient holds
            const float4 wk = weights[at_edge];
            float* const column = mine + at * 32 + lane;
            column[0] = fmaf(wk.x, gk, column[0]);
            column[32] = fmaf(wk.y, gk, column[32]);
            column[64] = fmaf(wk.z, gk, column[64]);
            column[96] = fmaf(wk.w, gk, column[96]);
            if (a.d_dist != nullptr) {
                const float4 sk = slopes[at_edge];
                const float* const t = table + at * 32 + lane;
                float v = fmaf(sk.x, t[0], fmaf(sk.y, t[32], fmaf(sk.z, t[64], fmaf(sk.w, t[96], where.y)))) * gk;
#pragma unroll
                for (int o = WIDE / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                // the sum of edge k SLOTS + s is with the lanes of slot s
                const float mine_now = __shfl_sync(0xffffffffu, v, (lane % SLOTS) * WIDE);
                if (lane / SLOTS == k) total = mine_now;
            }
        }
        if (a.d_dist != nullptr && base + lane < a.n) a.d_dist[base + lane] = r < 0.0f ? 0.0f : total / a.cutoff;
        r = r_next;
    }
    if (a.partial == nullptr) return;
    __syncthreads();
    for (int i = threadIdx.x; i < a.buckets * WIDE; i += blockDim.x) {
        const int hh = i % WIDE, k = i / WIDE;
        if (hh >= a.heads) continue;
        float sum = 0.0f;
        for (int c = 0; c < warps; c++)
            for (int s = 0; s < SLOTS; s++) sum += copies[words + c * (words + DB_SCRATCH) + k * 32 + s * WIDE + hh];
        a.partial[((int64_t)blockIdx.x * a.buckets + k) * a.heads + hh] = sum;
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

// Gradient of the table for more heads or buckets than the kernel above has room for (33 heads, 891 buckets).  10.5 M edges, 1024 x 8: 11.5 ms, with one warp
// an SM; 2 M edges, 64 x 64: 1.0 ms.  A warp's lanes are `slots` edges times `wide` heads; every slot has a copy of the table in shared memory that
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

// 32 cells a block, eight runs of blocks each.
__global__ void __launch_bounds__(DB_THREADS)
db_table_join_kernel(const DbArgs a, int blocks)
{
    __shared__ double part[8][32];
    const int64_t cells = (int64_t)a.buckets * a.heads, i = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
    const int run = threadIdx.x / 32;
    double sum = 0.0;
    if (i < cells)
        for (int b = run; b < blocks; b += 8) sum += (double)a.partial[b * cells + i];
    part[run][threadIdx.x % 32] = sum;
    __syncthreads();
    if (run != 0 || i >= cells) return;
#pragma unroll
    for (int k = 1; k < 8; k++) sum += part[k][threadIdx.x];
    a.d_table[i] = (float)sum;
}

static int db_table_blocks(int64_t n)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>((n + 1023) / 1024, 148));
}

// The kernel for both gradients: warps of a block, 0 where the heads or the buckets are too many for it.
static int db_backward_warps(int buckets, int heads)
{
    if (heads > 32) return 0;
    const int words = buckets * 32, room = (224 << 10) / 4 - words;
    return std::min(22, room / (words + DB_SCRATCH));
}

template <int WIDE>
static cudaError_t db_backward(const DbArgs& a, int blocks, int warps, cudaStream_t s)
{
    const int words = a.buckets * 32, smem = 4 * (words + warps * (words + DB_SCRATCH));
    const cudaError_t rc = cudaFuncSetAttribute(db_backward_kernel<WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    db_backward_kernel<WIDE><<<blocks, warps * 32, smem, s>>>(a);
    return cudaGetLastError();
}

static int db_check(int64_t n, int heads, int buckets, double cutoff)
{
    if (n < 0) return fail_arg("distance_bias: sizes must be non-negative");
    if (heads < 1 || heads > DYNB_DISTANCE_BIAS_MAX_HEADS) return fail_arg("distance_bias: heads must lie in [1, 1024]");
    if (buckets < 4 || buckets > DYNB_DISTANCE_BIAS_MAX_BUCKETS) return fail_arg("distance_bias: buckets must lie in [4, 1024]");
    if (!(cutoff > 0.0) || !(cutoff < 3.0e38)) return fail_arg("distance_bias: cutoff must be positive and finite");
    return DYNB_OK;
}

// Of cutoffs so small that the remainder of a quotient by them has no room, 0.
static float db_per(int buckets, float cutoff) { return cutoff > 1e-30f ? (float)(buckets - 3) / cutoff : 0.0f; }

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
    a.n = n; a.heads = heads; a.buckets = buckets; a.smooth = smooth; a.cutoff = (float)cutoff; a.per = db_per(buckets, a.cutoff);
    const bool aligned = reinterpret_cast<uintptr_t>(bias_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(table_dev) % 16 == 0;
    const bool eight = aligned && heads % 8 == 0 && reinterpret_cast<uintptr_t>(bias_dev) % 32 == 0 && buckets * heads * 32 <= DB_COPIES_BYTES;
    const int vec = eight ? 8 : aligned && heads % 4 == 0 ? 4 : 1;
    const bool held = buckets * heads * 4 <= DB_TABLE_BYTES;
    const unsigned blocks = db_blocks(n * (heads / vec));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (eight) db_forward_kernel<8, true><<<blocks, DB_THREADS, buckets * heads * 32, s>>>(a);
    else if (vec == 4 && held) db_forward_kernel<4, true><<<blocks, DB_THREADS, buckets * heads * 4, s>>>(a);
    else if (vec == 4) db_forward_kernel<4, false><<<blocks, DB_THREADS, 0, s>>>(a);
    else if (held) db_forward_kernel<1, true><<<blocks, DB_THREADS, buckets * heads * 4, s>>>(a);
    else db_forward_kernel<1, false><<<blocks, DB_THREADS, 0, s>>>(a);
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
    a.n = n; a.heads = heads; a.buckets = buckets; a.smooth = smooth; a.cutoff = (float)cutoff; a.per = db_per(buckets, a.cutoff);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int blocks = db_table_blocks(n);
    if (d_table_dev != nullptr) {
        if (workspace_dev == nullptr || workspace_bytes < (int64_t)blocks * buckets * heads * 4) return fail_arg("workspace too small");
        a.partial = static_cast<float*>(workspace_dev);
    }
    const int warps = db_backward_warps(buckets, heads);
    if (warps > 0) {
        if (d_table_dev != nullptr || (d_dist_dev != nullptr && n > 0)) {
            const cudaError_t e = heads <= 1 ? db_backward<1>(a, blocks, warps, s) : heads <= 2 ? db_backward<2>(a, blocks, warps, s)
                                : heads <= 4 ? db_backward<4>(a, blocks, warps, s) : heads <= 8 ? db_backward<8>(a, blocks, warps, s)
                                : heads <= 16 ? db_backward<16>(a, blocks, warps, s) : db_backward<32>(a, blocks, warps, s);
            DYNB_CUDA_OK(e);
        }
    } else {
        if (d_dist_dev != nullptr && n > 0) {
            db_dist_kernel<<<db_blocks(n), DB_THREADS, 0, s>>>(a);
            DYNB_CUDA_OK(cudaGetLastError());
        }
        if (d_table_dev != nullptr) {
            int wide = 1;
            while (wide < heads && wide < 32) wide *= 2;
            // as many warps as have their copies in 128 KB, and no more than 16
            const int table_warps = std::max(1, std::min(16, (128 << 10) / (buckets * 128)));
            const int smem = table_warps * buckets * 128;
            DYNB_CUDA_OK(cudaFuncSetAttribute(db_table_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            db_table_kernel<<<dim3(blocks, (heads + wide - 1) / wide), table_warps * 32, smem, s>>>(a, wide);
            DYNB_CUDA_OK(cudaGetLastError());
        }
    }
    if (d_table_dev != nullptr) {
        db_table_join_kernel<<<(unsigned)(((int64_t)buckets * heads + 31) / 32), DB_THREADS, 0, s>>>(a, blocks);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    return DYNB_OK;
}
