// Gradients of neighbour attention.  The probabilities are computed again from the largest logit and the sum that the forward pass
// kept.  With dp_e = d_out_t . v_s, delta_t = d_out_t . out_t and ds_e = p_e (dp_e - delta_t):
//     d_bias_e = ds_e,  dq_t = scale sum_e ds_e k_s  (by target),  dk_s = scale sum_e ds_e q_t,  dv_s = sum_e p_e d_out_t  (by source).
// Two passes, one over the lists by target and one over the lists by source, each of which adds up a row in registers in the order of
// its list: no atomics, results do not change from run to run, and nothing of the size of the edges is kept but the bias's gradient.

#include <algorithm>

#include "attention.cuh"

namespace dynb {

constexpr int AB_WARPS = 8;
constexpr int AB_BATCH = 4;    // edges of a slot in flight, by target
constexpr int AC_BATCH = 2;    // by source

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
__global__ void __launch_bounds__(AB_WARPS * 32)
attn_backward_rows_kernel(const AttnArgs a)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool mine = head < a.heads, wide = a.wide != 0;
    const int h = mine ? head : 0, kv = h / a.shared;
    const Place<T, G> place(part, h);
    const uint32_t sources = (uint32_t)a.n_sources;
    const uint32_t k_step = (uint32_t)(a.k.row * (int)sizeof(T)), v_step = (uint32_t)(a.v.row * (int)sizeof(T));
    const char* const kb = reinterpret_cast<const char*>(static_cast<const T*>(a.k.at) + kv * a.k.head);
    const char* const vb = reinterpret_cast<const char*>(static_cast<const T*>(a.v.at) + kv * a.v.head);
    constexpr int ROWS = AB_WARPS / WPR;
    const int turn = warp % WPR, step = AB_BATCH * slots;

    const int64_t r = (int64_t)blockIdx.x * ROWS + warp / WPR;
    int32_t t = r < a.n_targets ? a.rows[r] : -1;
    if ((uint32_t)t >= (uint32_t)a.n_targets) t = -1;
    if (WPR == 1 && t < 0) return;
    int64_t begin = 0, end = 0;
    if (t >= 0) {
        begin = max(a.row_start[r], 0);
        end = min((int64_t)a.row_start[r + 1], a.n_edges);
    }
    const int n = (int)max(end - begin, (int64_t)0);
    const int32_t* const src = a.src + begin;
    const float* const bias = a.bias != nullptr ? a.bias + begin * a.heads + h : nullptr;
    float* const d_bias = a.d_bias != nullptr && mine && part == 0 ? a.d_bias + begin * a.heads + h : nullptr;
    const int64_t own = ((int64_t)max(t, 0) * a.heads + h) * a.dim;

    float2 q[4], g[4], acc[4];
    float delta = 0.0f, top = 0.0f, inv = 0.0f;
    Raw<T> qu = attn_nothing<T>(), gu = attn_nothing<T>();
    if (t >= 0) {
        qu = attn_load<T, G, FULL>(static_cast<const T*>(a.q.at) + t * a.q.row + h * a.q.head, place, a.dim, wide);
        gu = attn_load<T, G, FULL>(static_cast<const T*>(a.d_out.at) + t * a.d_out.row + h * a.d_out.head, place, a.dim, wide);
        top = a.stats[(int64_t)t * 2 * a.heads + h];
        inv = a.stats[(int64_t)t * 2 * a.heads + a.heads + h];
    }
    attn_pairs(qu, q);
    attn_pairs(gu, g);
    constexpr int VEC = Place<T, G>::VEC;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        q[i] = mul2(q[i], make_float2(a.scale, a.scale));
        acc[i] = make_float2(0.0f, 0.0f);
        const int d = place.at[2 * i / VEC] + 2 * i % VEC;
        if (t >= 0 && d < a.dim) delta = fmaf(g[i].x, a.out32[own + d], delta);
        if (t >= 0 && d + 1 < a.dim) delta = fmaf(g[i].y, a.out32[own + d + 1], delta);
    }
    delta = head_sum<G>(delta);
    if (mine && part == 0 && slot == 0 && turn == 0 && t >= 0) a.delta[(int64_t)t * a.heads + h] = delta;

    int e = turn * step + slot * AB_BATCH;
    AttnEdges<AB_BATCH> now;
    now.fetch(src, bias, e, n, a.heads);
    for (int base = turn * step; base < n; base += WPR * step) {
        Raw<T> ku[AB_BATCH], vu[AB_BATCH];
        float z[AB_BATCH];
        bool ok[AB_BATCH];
#pragma unroll
        for (int u = 0; u < AB_BATCH; u++) {
            ok[u] = now.live(u, sources);
            ku[u] = attn_nothing<T>();
            vu[u] = attn_nothing<T>();   // masked: not even a product with what its rows hold
            if (ok[u]) {
                ku[u] = attn_load<T, G, FULL>(reinterpret_cast<const T*>(kb + (uint64_t)(uint32_t)now.s[u] * k_step), place, a.dim, wide);
                vu[u] = attn_load<T, G, FULL>(reinterpret_cast<const T*>(vb + (uint64_t)(uint32_t)now.s[u] * v_step), place, a.dim, wide);
            }
            z[u] = now.z[u];
        }
        const int at = e;
        e += WPR * step;
        now.fetch(src, bias, e, n, a.heads);
#pragma unroll
        for (int u = 0; u < AB_BATCH; u++) {
            float2 k[4], v[4];
            attn_pairs(ku[u], k);
            attn_pairs(vu[u], v);
            const float dot = head_sum<G>(dot8(q, k)), dp = head_sum<G>(dot8(g, v));
            const float ds = ok[u] ? pow2((z[u] + dot - top) * LOG2E) * inv * (dp - delta) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fma2(make_float2(ds, ds), k[i], acc[i]);
            if (d_bias != nullptr && at + u < n) d_bias[(int64_t)(at + u) * a.heads] = ds;
        }
    }
    for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            acc[i].x += __shfl_xor_sync(0xffffffffu, acc[i].x, o);
            acc[i].y += __shfl_xor_sync(0xffffffffu, acc[i].y, o);
        }
    if (WPR > 1) attn_join<4, WPR>(acc, warp, lane);
    if (turn != 0 || !mine || slot != 0 || a.dq == nullptr || t < 0) return;
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = mul2(acc[i], make_float2(a.scale, a.scale));
    attn_store<T, G, FULL>(static_cast<T*>(a.dq) + own, place, a.dim, wide, acc);
}

// Lanes divide the heads of keys and values; the heads of queries that share one are taken one after the other, into the same sums.
template <typename T, int G, bool FULL, int WPR>
__global__ void __launch_bounds__(AB_WARPS * 32)
attn_backward_cols_kernel(const AttnArgs a)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool mine = head < a.kv_heads, wide = a.wide != 0;
    const int kv = mine ? head : 0;
    const Place<T, G> place(part, kv);
    const uint32_t targets = (uint32_t)a.n_targets, edges = (uint32_t)a.n_edges;
    const uint32_t q_step = (uint32_t)(a.q.row * (int)sizeof(T)), g_step = (uint32_t)(a.d_out.row * (int)sizeof(T));
    constexpr int ROWS = AB_WARPS / WPR;
    const int turn = warp % WPR, step = AC_BATCH * slots;

    const int64_t c = (int64_t)blockIdx.x * ROWS + warp / WPR;
    int32_t s = c < a.n_sources ? a.cols[c] : -1;
    if ((uint32_t)s >= (uint32_t)a.n_sources) s = -1;
    if (WPR == 1 && s < 0) return;
    int64_t begin = 0, end = 0;
    if (s >= 0) {
        begin = max(a.col_start[c], 0);
        end = min((int64_t)a.col_start[c + 1], a.n_edges);
    }
    const int n = (int)max(end - begin, (int64_t)0);
    const int32_t *const in_dst = a.in_dst + begin, *const in_edge = a.in_edge + begin;

    float2 k[4], v[4], acc[8];
    Raw<T> ku = attn_nothing<T>(), vu = attn_nothing<T>();
    if (s >= 0) {
        ku = attn_load<T, G, FULL>(static_cast<const T*>(a.k.at) + s * a.k.row + kv * a.k.head, place, a.dim, wide);
        vu = attn_load<T, G, FULL>(static_cast<const T*>(a.v.at) + s * a.v.row + kv * a.v.head, place, a.dim, wide);
    }
    attn_pairs(ku, k);
    attn_pairs(vu, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        k[i] = mul2(k[i], make_float2(a.scale, a.scale));
        acc[i] = acc[4 + i] = make_float2(0.0f, 0.0f);
    }
    int32_t t_next[AC_BATCH], e_next[AC_BATCH];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < AC_BATCH; u++) {
            t_next[u] = i + u < n ? __ldg(in_dst + i + u) : -1;
            e_next[u] = i + u < n && a.bias != nullptr ? __ldg(in_edge + i + u) : 0;
        }
    };
    int i = turn * step + slot * AC_BATCH;
    fetch(i);
    for (int base = turn * step; base < n; base += WPR * step) {
        int32_t t[AC_BATCH], e[AC_BATCH];
        bool in[AC_BATCH];
#pragma unroll
        for (int u = 0; u < AC_BATCH; u++) {
            in[u] = (uint32_t)t_next[u] < targets && (uint32_t)e_next[u] < edges;
            t[u] = in[u] ? t_next[u] : 0;
            e[u] = in[u] ? e_next[u] : 0;
        }
        i += WPR * step;
        fetch(i);
        for (int i0 = 0; i0 < a.shared; i0++) {
            const int h = kv * a.shared + i0;
            const char* const qb = reinterpret_cast<const char*>(static_cast<const T*>(a.q.at) + h * a.q.head);
            const char* const gb = reinterpret_cast<const char*>(static_cast<const T*>(a.d_out.at) + h * a.d_out.head);
            Raw<T> qu[AC_BATCH], gu[AC_BATCH];
            float z[AC_BATCH], top[AC_BATCH], inv[AC_BATCH], delta[AC_BATCH];
            bool ok[AC_BATCH];
#pragma unroll
            for (int u = 0; u < AC_BATCH; u++) {
                const float b = a.bias != nullptr ? __ldg(a.bias + (int64_t)e[u] * a.heads + h) : 0.0f;
                ok[u] = in[u] && b != -INFINITY;
                z[u] = b;
                top[u] = a.stats[(int64_t)t[u] * 2 * a.heads + h];
                inv[u] = a.stats[(int64_t)t[u] * 2 * a.heads + a.heads + h];
                delta[u] = a.delta[(int64_t)t[u] * a.heads + h];
                qu[u] = gu[u] = attn_nothing<T>();
                if (in[u]) {
                    qu[u] = attn_load<T, G, FULL>(reinterpret_cast<const T*>(qb + (uint64_t)(uint32_t)t[u] * q_step), place, a.dim, wide);
                    gu[u] = attn_load<T, G, FULL>(reinterpret_cast<const T*>(gb + (uint64_t)(uint32_t)t[u] * g_step), place, a.dim, wide);
                }
            }
#pragma unroll
            for (int u = 0; u < AC_BATCH; u++) {
                float2 q[4], g[4];
                attn_pairs(qu[u], q);
                attn_pairs(gu[u], g);
                const float dot = head_sum<G>(dot8(k, q)), dp = head_sum<G>(dot8(v, g));
                const float w = pow2((z[u] + dot - top[u]) * LOG2E) * inv[u], ds = w * (dp - delta[u]);
                if (ok[u]) {   // masked: not even a product with what the target's rows hold
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        acc[j] = fma2(make_float2(ds, ds), q[j], acc[j]);
                        acc[4 + j] = fma2(make_float2(w, w), g[j], acc[4 + j]);
                    }
                }
            }
        }
    }
    for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            acc[j].x += __shfl_xor_sync(0xffffffffu, acc[j].x, o);
            acc[j].y += __shfl_xor_sync(0xffffffffu, acc[j].y, o);
        }
    if (WPR > 1) attn_join<8, WPR>(acc, warp, lane);
    if (turn != 0 || !mine || slot != 0 || s < 0) return;
    const int64_t own = ((int64_t)s * a.kv_heads + kv) * a.dim;
    float2 dk[4], dv[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        dk[j] = mul2(acc[j], make_float2(a.scale, a.scale));
        dv[j] = acc[4 + j];
    }
    if (a.dk != nullptr) attn_store<T, G, FULL>(static_cast<T*>(a.dk) + own, place, a.dim, wide, dk);
    if (a.dv != nullptr) attn_store<T, G, FULL>(static_cast<T*>(a.dv) + own, place, a.dim, wide, dv);
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
        const dim3 grid((unsigned)((a.n_targets + rows - 1) / rows), blocks);
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
        const dim3 grid((unsigned)((a.n_sources + rows - 1) / rows), blocks);
        if (split) attn_backward_cols_kernel<T, G, FULL, 4><<<grid, AB_WARPS * 32, 0, s>>>(a);
        else attn_backward_cols_kernel<T, G, FULL, 1><<<grid, AB_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

cudaError_t attn_backward_rows(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardRows>(a, dtype, s); }
cudaError_t attn_backward_cols(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardCols>(a, dtype, s); }

}  // namespace dynb
