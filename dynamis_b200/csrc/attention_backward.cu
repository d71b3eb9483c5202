// Gradients of neighbour attention.  The probabilities are computed again from the largest logit and the sum that the forward pass
// kept.  With dp_e = d_out_t . v_s, delta_t = d_out_t . out_t and ds_e = p_e (dp_e - delta_t):
//     d_bias_e = ds_e,  dq_t = scale sum_e ds_e k_s  (by target),  dk_s = scale sum_e ds_e q_t,  dv_s = sum_e p_e d_out_t  (by source).
// Two passes, one over the lists by target and one over the lists by source, each of which adds up a row in registers in the order of
// its list: no atomics, results do not change from run to run, and nothing of the size of the edges is kept but the bias's gradient.
//
// Latency and issue bound both, as forward.  200 k targets, 10.5 M edges, 8 x 16 fp32: by target 851 us, by source 1049 us (there an edge also gathers its
// target's statistics and its own bias); 42 k targets of 60 k rows, bf16, 4 x 64, a quarter of the edges masked: 336 and 473 us.  Not all of it fits the
// registers: by source full rows of 16 bits spill 72 bytes a thread (92 where a lane has a whole head), heads that do not fill their lanes 92 to 200, by target, too,
// in every type (92 to 176).

#include <algorithm>

#include "attention.cuh"

namespace dynb {

constexpr int AB_WARPS = 4;
// Edges of a slot in a batch, by target and by source, and blocks an SM by target.  200 k targets, 8 x 16 fp32: by target two edges and 20 warps 894 us, four
// edges and 16 warps 1010; by source three edges 1043, two 1192.  bf16, 4 x 64, by source: two edges 464, three 591 (its rows are unpacked).
constexpr int AB_BATCH = 2;
template <typename T> constexpr int AC_BATCH = sizeof(T) == 4 ? 3 : 2;
template <typename T> constexpr int AB_BLOCKS = sizeof(T) == 4 ? 5 : 4;

// Sums of the warps of a row, in their order, with the first of them (turn 0).  All warps of the block call it.
template <int N, int WPR>
__device__ __forceinline__ void attn_join(float2 (&acc)[N], int warp, int lane)
{
    __shared__ float2 joint[AB_WARPS][N][32];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) joint[warp][i][lane] = acc[i];
    __syncthreads();
    if (warp % WPR != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; w++)
#pragma unroll
        for (int i = 0; i < N; i++) {
            acc[i].x += joint[warp + w][i][lane].x;
            acc[i].y += joint[warp + w][i][lane].y;
        }
}

template <typename T, int G, bool FULL, int WPR>
__global__ void __launch_bounds__(AB_WARPS * 32, AB_BLOCKS<T>)
attn_backward_rows_kernel(const AttnArgs a)
{
    constexpr int EL = LaneElements<T>::N, BATCH = AB_BATCH;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool mine = head < a.heads;
    const int wide = a.wide;
    const int h = mine ? head : 0, kv = h / a.shared;
    const Place<T, G, EL> place(part);
    const uint32_t sources = (uint32_t)a.n_sources;
    const Lane<T, G, EL> k_lane(a.k, kv, place), v_lane(a.v, kv, place);
    constexpr int ROWS = AB_WARPS / WPR;
    const int turn = warp % WPR, step = BATCH * slots, bias_step = a.bias != nullptr ? a.heads : 0;
    const char* const zeros = reinterpret_cast<const char*>(attn_zeros);

    const int64_t last = min(((int64_t)blockIdx.x + 1) * a.block_rows, a.n_targets);
    for (int64_t r0 = (int64_t)blockIdx.x * a.block_rows; r0 < last; r0 += ROWS) {
        const int64_t r = r0 + warp / WPR;
        int32_t t = r < last ? a.rows[r] : -1;
        if ((uint32_t)t >= (uint32_t)a.n_targets) t = -1;
        if (WPR == 1 && t < 0) continue;
        int64_t begin = 0, end = 0;
        if (t >= 0) {
            begin = max(a.row_start[r], 0);
            end = min((int64_t)a.row_start[r + 1], a.n_edges);
        }
        const int n = (int)max(end - begin, (int64_t)0);
        const int32_t* const src = a.src + begin;
        const float* const bias = a.bias + (begin * bias_step + h);   // not read where there is none
        float* const d_bias = a.d_bias != nullptr && mine && part == 0 ? a.d_bias + begin * a.heads + h : nullptr;
        const int64_t own = ((int64_t)max(t, 0) * a.heads + h) * a.dim;

        float2 q[EL / 2], g[EL / 2], acc[EL / 2];
        float delta = 0.0f, top = 0.0f, inv = 0.0f;
        const T* const nothing = reinterpret_cast<const T*>(zeros);
        attn_pairs(attn_load<T, G, EL, FULL>(t >= 0 ? static_cast<const T*>(a.q.at) + t * a.q.row + h * a.q.head : nothing, place, a.dim, wide), q);
        attn_pairs(attn_load<T, G, EL, FULL>(t >= 0 ? static_cast<const T*>(a.d_out.at) + t * a.d_out.row + h * a.d_out.head : nothing, place, a.dim, wide), g);
        if (t >= 0) {
            top = a.stats[(int64_t)t * 2 * a.heads + h];
            inv = a.stats[(int64_t)t * 2 * a.heads + a.heads + h];
        }
        constexpr int VEC = Place<T, G, EL>::VEC;
#pragma unroll
        for (int i = 0; i < EL / 2; i++) {
            q[i] = mul2(q[i], make_float2(a.scale, a.scale));
            acc[i] = make_float2(0.0f, 0.0f);
            const int d = place.at[2 * i / VEC] + 2 * i % VEC;
            if (t >= 0 && d < a.dim) delta = fmaf(g[i].x, a.out32[own + d], delta);
            if (t >= 0 && d + 1 < a.dim) delta = fmaf(g[i].y, a.out32[own + d + 1], delta);
        }
        delta = head_sum<G>(delta);
        if (mine && part == 0 && slot == 0 && turn == 0 && t >= 0) a.delta[(int64_t)t * a.heads + h] = make_float4(top, inv, delta, 0.0f);

        int e = turn * step + slot * BATCH, at = e;
        AttnEdges<BATCH> ahead;
        ahead.fetch(src, bias, e, n, bias_step);
        auto load = [&](AttnStep<T, EL, BATCH>& s) {
            uint32_t row[BATCH];
            ahead.rows(sources, row, s.ok);
            s.template load<G, FULL>(k_lane, v_lane, place, a.k, a.v, kv, kv, row, a.dim, wide);
#pragma unroll
            for (int u = 0; u < BATCH; u++) s.z[u] = ahead.z[u];
            e += WPR * step;
            ahead.fetch(src, bias, e, n, bias_step);
        };
        auto work = [&](AttnStep<T, EL, BATCH>& s) {
            s.clear();
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                float2 k[EL / 2], v[EL / 2];
                attn_pairs(s.x[u], k);
                attn_pairs(s.y[u], v);
                const float dot = head_sum<G>(inner(q, k)), dp = head_sum<G>(inner(g, v));
                const float ds = s.ok[u] ? pow2((s.z[u] + dot - top) * LOG2E) * inv * (dp - delta) : 0.0f;
#pragma unroll
                for (int i = 0; i < EL / 2; i++) acc[i] = fma2(make_float2(ds, ds), k[i], acc[i]);
                if (d_bias != nullptr && at + u < n) d_bias[(int64_t)(at + u) * a.heads] = ds;
            }
            at += WPR * step;
        };
        for (int base = turn * step; base < n; base += WPR * step) {   // the same for all lanes
            AttnStep<T, EL, BATCH> s;
            load(s);
            work(s);
        }
        for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < EL / 2; i++) {
                acc[i].x += __shfl_xor_sync(0xffffffffu, acc[i].x, o);
                acc[i].y += __shfl_xor_sync(0xffffffffu, acc[i].y, o);
            }
        if (WPR > 1) attn_join<EL / 2, WPR>(acc, warp, lane);
        if (turn != 0 || !mine || slot != 0 || a.dq == nullptr || t < 0) continue;
#pragma unroll
        for (int i = 0; i < EL / 2; i++) acc[i] = mul2(acc[i], make_float2(a.scale, a.scale));
        attn_store<T, G, EL, FULL>(static_cast<T*>(a.dq) + own, place, a.dim, wide, acc);
    }
}

// Lanes divide the heads of keys and values; the heads of queries that share one are taken one after the other, into the same sums.
template <typename T, int G, bool FULL, int WPR>
__global__ void __launch_bounds__(AB_WARPS * 32, 4)
attn_backward_cols_kernel(const AttnArgs a)
{
    constexpr int EL = LaneElements<T>::N, BATCH = AC_BATCH<T>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool mine = head < a.kv_heads;
    const int wide = a.wide;
    const int kv = mine ? head : 0;
    const Place<T, G, EL> place(part);
    const uint32_t targets = (uint32_t)a.n_targets, edges = (uint32_t)a.n_edges, bias_bytes = 4u * a.heads;
    constexpr int ROWS = AB_WARPS / WPR;
    const int turn = warp % WPR, step = BATCH * slots;
    const char* const zeros = reinterpret_cast<const char*>(attn_zeros);

    const int64_t last = min(((int64_t)blockIdx.x + 1) * a.block_rows, a.n_sources);
    for (int64_t c0 = (int64_t)blockIdx.x * a.block_rows; c0 < last; c0 += ROWS) {
        const int64_t c = c0 + warp / WPR;
        int32_t s = c < last ? a.cols[c] : -1;
        if ((uint32_t)s >= (uint32_t)a.n_sources) s = -1;
        if (WPR == 1 && s < 0) continue;
        int64_t begin = 0, end = 0;
        if (s >= 0) {
            begin = max(a.col_start[c], 0);
            end = min((int64_t)a.col_start[c + 1], a.n_edges);
        }
        const int n = (int)max(end - begin, (int64_t)0);
        const int32_t *const in_dst = a.in_dst + begin, *const in_edge = a.in_edge + begin;

        float2 k[EL / 2], v[EL / 2], acc[EL];
        const T* const nothing = reinterpret_cast<const T*>(zeros);
        attn_pairs(attn_load<T, G, EL, FULL>(s >= 0 ? static_cast<const T*>(a.k.at) + s * a.k.row + kv * a.k.head : nothing, place, a.dim, wide), k);
        attn_pairs(attn_load<T, G, EL, FULL>(s >= 0 ? static_cast<const T*>(a.v.at) + s * a.v.row + kv * a.v.head : nothing, place, a.dim, wide), v);
#pragma unroll
        for (int i = 0; i < EL / 2; i++) {
            k[i] = mul2(k[i], make_float2(a.scale, a.scale));
            acc[i] = acc[EL / 2 + i] = make_float2(0.0f, 0.0f);
        }
        // A step is a batch of edges and one of the heads that share keys and values.
        int32_t t_ahead[BATCH], e_ahead[BATCH];
        auto fetch = [&](int i) {
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                t_ahead[u] = i + u < n ? __ldg(in_dst + i + u) : -1;
                e_ahead[u] = i + u < n && a.bias != nullptr ? __ldg(in_edge + i + u) : 0;
            }
        };
        struct ColStep : AttnStep<T, EL, BATCH> { float4 stats[BATCH]; };
        int i = turn * step + slot * BATCH, shared_head = 0;
        fetch(i);
        auto load = [&](ColStep& s) {
            const int h = kv * a.shared + shared_head;
            const Lane<T, G, EL> q_lane(a.q, h, place), g_lane(a.d_out, h, place);
            uint32_t t[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                const bool in = (uint32_t)t_ahead[u] < targets && (uint32_t)e_ahead[u] < edges;
                t[u] = in ? (uint32_t)t_ahead[u] : 0u;
                const uint32_t e = in ? (uint32_t)e_ahead[u] : 0u;
                s.z[u] = a.bias != nullptr ? __ldg(reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.bias + h) + (uint64_t)e * bias_bytes)) : 0.0f;
                s.stats[u] = a.delta[(int64_t)t[u] * a.heads + h];
                s.ok[u] = in;
            }
            s.template load<G, FULL>(q_lane, g_lane, place, a.q, a.d_out, h, h, t, a.dim, wide);
            if (++shared_head == a.shared) {
                shared_head = 0;
                i += WPR * step;
                fetch(i);
            }
        };
        auto work = [&](ColStep& s) {
#pragma unroll
            for (int u = 0; u < BATCH; u++) s.ok[u] = s.ok[u] && s.z[u] != -INFINITY;
            s.clear();
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                float2 q[EL / 2], g[EL / 2];
                attn_pairs(s.x[u], q);
                attn_pairs(s.y[u], g);
                const float dot = head_sum<G>(inner(k, q)), dp = head_sum<G>(inner(v, g));
                const float w = s.ok[u] ? pow2((s.z[u] + dot - s.stats[u].x) * LOG2E) * s.stats[u].y : 0.0f, ds = s.ok[u] ? w * (dp - s.stats[u].z) : 0.0f;
#pragma unroll
                for (int j = 0; j < EL / 2; j++) {
                    acc[j] = fma2(make_float2(ds, ds), q[j], acc[j]);
                    acc[EL / 2 + j] = fma2(make_float2(w, w), g[j], acc[EL / 2 + j]);
                }
            }
        };
        const int first = turn * step, stride = WPR * step;
        int steps = n > first ? (n - first + stride - 1) / stride * a.shared : 0;
        for (; steps > 0; steps--) {   // the same for all lanes
            ColStep s;
            load(s);
            work(s);
        }
        for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
            for (int j = 0; j < EL; j++) {
                acc[j].x += __shfl_xor_sync(0xffffffffu, acc[j].x, o);
                acc[j].y += __shfl_xor_sync(0xffffffffu, acc[j].y, o);
            }
        if (WPR > 1) attn_join<EL, WPR>(acc, warp, lane);
        if (turn != 0 || !mine || slot != 0 || s < 0) continue;
        const int64_t own = ((int64_t)s * a.kv_heads + kv) * a.dim;
        float2 dk[EL / 2], dv[EL / 2];
#pragma unroll
        for (int j = 0; j < EL / 2; j++) {
            dk[j] = mul2(acc[j], make_float2(a.scale, a.scale));
            dv[j] = acc[EL / 2 + j];
        }
        if (a.dk != nullptr) attn_store<T, G, EL, FULL>(static_cast<T*>(a.dk) + own, place, a.dim, wide, dk);
        if (a.dv != nullptr) attn_store<T, G, EL, FULL>(static_cast<T*>(a.dv) + own, place, a.dim, wide, dv);
    }
}

template <typename T, int G, bool FULL>
struct AttnBackwardRows {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.heads, G);
        const int blocks = (a.heads + a.warp_heads - 1) / a.warp_heads;
        const bool split = attn_split(a.n_targets * blocks, a.n_edges * blocks);
        const int rows = split ? AB_WARPS / 4 : AB_WARPS;
        a.block_rows = attn_block_rows(a.n_targets * blocks, rows);
        const dim3 grid((unsigned)((a.n_targets + a.block_rows - 1) / a.block_rows), blocks);
        if (split) attn_backward_rows_kernel<T, G, FULL, 4><<<grid, AB_WARPS * 32, 0, s>>>(a);
        else attn_backward_rows_kernel<T, G, FULL, 1><<<grid, AB_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

template <typename T, int G, bool FULL>
struct AttnBackwardCols {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.kv_heads, G);
        const int blocks = (a.kv_heads + a.warp_heads - 1) / a.warp_heads;
        const bool split = attn_split(a.n_sources * blocks, a.n_edges * blocks);
        const int rows = split ? AB_WARPS / 4 : AB_WARPS;
        a.block_rows = attn_block_rows(a.n_sources * blocks, rows);
        const dim3 grid((unsigned)((a.n_sources + a.block_rows - 1) / a.block_rows), blocks);
        if (split) attn_backward_cols_kernel<T, G, FULL, 4><<<grid, AB_WARPS * 32, 0, s>>>(a);
        else attn_backward_cols_kernel<T, G, FULL, 1><<<grid, AB_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

cudaError_t attn_backward_rows(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardRows>(a, dtype, s); }
cudaError_t attn_backward_cols(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardCols>(a, dtype, s); }

}  // namespace dynb
