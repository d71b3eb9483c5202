// Gradients of neighbour attention.  The probabilities are computed again from the largest logit and the sum that the forward pass
// kept.  With dp_e = d_out_t . v_s, delta_t = d_out_t . out_t and ds_e = p_e (dp_e - delta_t):
//     d_bias_e = ds_e,  dq_t = scale sum_e ds_e k_s  (by target),  dk_s = scale sum_e ds_e q_t,  dv_s = sum_e p_e d_out_t  (by source).
// Two passes, one over the lists by target and one over the lists by source, each of which adds up a row in registers in the order of
// its list: no atomics, results do not change from run to run, and nothing of the size of the edges is kept but the bias's gradient.

#include "attention.cuh"

namespace dynb {

constexpr int AB_WARPS = 4;
constexpr int AB_BATCH = 4;

template <typename T, int G, int NV>
__global__ void __launch_bounds__(AB_WARPS * 32)
attn_backward_rows_kernel(const AttnArgs a)
{
    constexpr int VEC = Piece<T>::VEC;
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * AB_WARPS + (threadIdx.x >> 5);
    if (r >= a.n_targets) return;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool live = head < a.heads;
    const int h = live ? head : 0, kv = h / a.shared;
    const int32_t t = a.rows[r];
    if ((uint32_t)t >= (uint64_t)a.n_targets) return;
    const int64_t begin = max(a.row_start[r], 0), end = min((int64_t)a.row_start[r + 1], a.n_edges);
    const bool wide = a.wide != 0;
    const int64_t own = ((int64_t)t * a.heads + h) * a.dim;

    float q[NV][VEC], g[NV][VEC], acc[NV][VEC];
    float delta = 0.0f;
#pragma unroll
    for (int p = 0; p < NV; p++) {
        const int d = (p * G + part) * VEC;
        Piece<T>::unpack(load_piece(static_cast<const T*>(a.q.at) + t * a.q.row + h * a.q.head, d, a.dim, wide), q[p]);
        Piece<T>::unpack(load_piece(static_cast<const T*>(a.d_out.at) + t * a.d_out.row + h * a.d_out.head, d, a.dim, wide), g[p]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            q[p][i] *= a.scale;
            acc[p][i] = 0.0f;
            if (d + i < a.dim) delta = fmaf(g[p][i], a.out32[own + d + i], delta);
        }
    }
    delta = head_sum<G>(delta);
    const float top = a.stats[(int64_t)t * 2 * a.heads + h], inv = a.stats[(int64_t)t * 2 * a.heads + a.heads + h];
    if (live && part == 0 && slot == 0) a.delta[(int64_t)t * a.heads + h] = delta;
    const T* const kb = static_cast<const T*>(a.k.at) + kv * a.k.head;
    const T* const vb = static_cast<const T*>(a.v.at) + kv * a.v.head;
    for (int64_t base = begin; base < end; base += AB_BATCH * slots) {
        uint4 ku[AB_BATCH][NV], vu[AB_BATCH][NV];
        float z[AB_BATCH];
#pragma unroll
        for (int u = 0; u < AB_BATCH; u++) {
            const int64_t e = base + u * slots + slot;
            const int32_t s = e < end ? a.src[e] : -1;
            const bool ok = (uint32_t)s < (uint64_t)a.n_sources;
            z[u] = !ok ? -INFINITY : a.bias != nullptr ? a.bias[e * a.heads + h] : 0.0f;
            const int64_t at = ok ? s : 0;
#pragma unroll
            for (int p = 0; p < NV; p++) {
                ku[u][p] = ok ? load_piece(kb + at * a.k.row, (p * G + part) * VEC, a.dim, wide) : make_uint4(0, 0, 0, 0);
                vu[u][p] = ok ? load_piece(vb + at * a.v.row, (p * G + part) * VEC, a.dim, wide) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < AB_BATCH; u++) {
            const int64_t e = base + u * slots + slot;
            float kf[NV][VEC], dot = 0.0f, dp = 0.0f;
#pragma unroll
            for (int p = 0; p < NV; p++) {
                float f[VEC];
                Piece<T>::unpack(ku[u][p], kf[p]);
                Piece<T>::unpack(vu[u][p], f);
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    dot = fmaf(q[p][i], kf[p][i], dot);
                    dp = fmaf(g[p][i], f[i], dp);
                }
            }
            dot = head_sum<G>(dot);
            dp = head_sum<G>(dp);
            if (z[u] != -INFINITY) z[u] += dot;
            float ds = 0.0f;
            if (z[u] != -INFINITY) {   // masked edges: no product with what their rows hold
                ds = exp2f((z[u] - top) * LOG2E) * inv * (dp - delta);
#pragma unroll
                for (int p = 0; p < NV; p++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) acc[p][i] = fmaf(ds, kf[p][i], acc[p][i]);
            }
            if (a.d_bias != nullptr && live && part == 0 && e < end) a.d_bias[e * a.heads + h] = ds;
        }
    }
    for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
        for (int p = 0; p < NV; p++)
#pragma unroll
            for (int i = 0; i < VEC; i++) acc[p][i] += __shfl_xor_sync(0xffffffffu, acc[p][i], o);
    if (!live || slot != 0 || a.dq == nullptr) return;
#pragma unroll
    for (int p = 0; p < NV; p++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) acc[p][i] *= a.scale;
        store_piece(static_cast<T*>(a.dq) + own, (p * G + part) * VEC, a.dim, wide, acc[p]);
    }
}

// Lanes divide the heads of keys and values; the heads of queries that share one are taken one after the other, into the same sums.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(AB_WARPS * 32)
attn_backward_cols_kernel(const AttnArgs a)
{
    constexpr int VEC = Piece<T>::VEC;
    const int lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * AB_WARPS + (threadIdx.x >> 5);
    if (c >= a.n_sources) return;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool live = head < a.kv_heads;
    const int kv = live ? head : 0;
    const int32_t s = a.cols[c];
    if ((uint32_t)s >= (uint64_t)a.n_sources) return;
    const int64_t begin = max(a.col_start[c], 0), end = min((int64_t)a.col_start[c + 1], a.n_edges);
    const bool wide = a.wide != 0;

    float k[NV][VEC], v[NV][VEC], dk[NV][VEC], dv[NV][VEC];
#pragma unroll
    for (int p = 0; p < NV; p++) {
        const int d = (p * G + part) * VEC;
        Piece<T>::unpack(load_piece(static_cast<const T*>(a.k.at) + s * a.k.row + kv * a.k.head, d, a.dim, wide), k[p]);
        Piece<T>::unpack(load_piece(static_cast<const T*>(a.v.at) + s * a.v.row + kv * a.v.head, d, a.dim, wide), v[p]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            k[p][i] *= a.scale;
            dk[p][i] = dv[p][i] = 0.0f;
        }
    }
    for (int64_t base = begin; base < end; base += AB_BATCH * slots)
        for (int i0 = 0; i0 < a.shared; i0++) {
            const int h = kv * a.shared + i0;
            const T* const qb = static_cast<const T*>(a.q.at) + h * a.q.head;
            const T* const gb = static_cast<const T*>(a.d_out.at) + h * a.d_out.head;
            uint4 qu[AB_BATCH][NV], gu[AB_BATCH][NV];
            float z[AB_BATCH], top[AB_BATCH], inv[AB_BATCH], delta[AB_BATCH];
#pragma unroll
            for (int u = 0; u < AB_BATCH; u++) {
                const int64_t i = base + u * slots + slot;
                const int32_t t = i < end ? a.in_dst[i] : -1;
                const int32_t e = i < end && a.bias != nullptr ? a.in_edge[i] : 0;
                const bool ok = (uint32_t)t < (uint64_t)a.n_targets && (uint32_t)e < (uint64_t)a.n_edges;
                z[u] = !ok ? -INFINITY : a.bias != nullptr ? a.bias[(int64_t)e * a.heads + h] : 0.0f;
                const int64_t at = ok ? t : 0;
                top[u] = a.stats[at * 2 * a.heads + h];
                inv[u] = a.stats[at * 2 * a.heads + a.heads + h];
                delta[u] = a.delta[at * a.heads + h];
#pragma unroll
                for (int p = 0; p < NV; p++) {
                    qu[u][p] = ok ? load_piece(qb + at * a.q.row, (p * G + part) * VEC, a.dim, wide) : make_uint4(0, 0, 0, 0);
                    gu[u][p] = ok ? load_piece(gb + at * a.d_out.row, (p * G + part) * VEC, a.dim, wide) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int u = 0; u < AB_BATCH; u++) {
                float qf[NV][VEC], gf[NV][VEC], dot = 0.0f, dp = 0.0f;
#pragma unroll
                for (int p = 0; p < NV; p++) {
                    Piece<T>::unpack(qu[u][p], qf[p]);
                    Piece<T>::unpack(gu[u][p], gf[p]);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        dot = fmaf(k[p][i], qf[p][i], dot);
                        dp = fmaf(v[p][i], gf[p][i], dp);
                    }
                }
                dot = head_sum<G>(dot);
                dp = head_sum<G>(dp);
                if (z[u] != -INFINITY) z[u] += dot;
                if (z[u] == -INFINITY) continue;
                const float w = exp2f((z[u] - top[u]) * LOG2E) * inv[u];
                const float ds = w * (dp - delta[u]);
#pragma unroll
                for (int p = 0; p < NV; p++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        dk[p][i] = fmaf(ds, qf[p][i], dk[p][i]);
                        dv[p][i] = fmaf(w, gf[p][i], dv[p][i]);
                    }
            }
        }
    for (int o = G * a.warp_heads; o < 32; o <<= 1)
#pragma unroll
        for (int p = 0; p < NV; p++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                dk[p][i] += __shfl_xor_sync(0xffffffffu, dk[p][i], o);
                dv[p][i] += __shfl_xor_sync(0xffffffffu, dv[p][i], o);
            }
    if (!live || slot != 0) return;
    const int64_t own = ((int64_t)s * a.kv_heads + kv) * a.dim;
#pragma unroll
    for (int p = 0; p < NV; p++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) dk[p][i] *= a.scale;
        const int d = (p * G + part) * VEC;
        if (a.dk != nullptr) store_piece(static_cast<T*>(a.dk) + own, d, a.dim, wide, dk[p]);
        if (a.dv != nullptr) store_piece(static_cast<T*>(a.dv) + own, d, a.dim, wide, dv[p]);
    }
}

template <typename T, int G, int NV>
struct AttnBackwardRows {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.heads, G);
        const dim3 grid((unsigned)((a.n_targets + AB_WARPS - 1) / AB_WARPS), (a.heads + a.warp_heads - 1) / a.warp_heads);
        attn_backward_rows_kernel<T, G, NV><<<grid, AB_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

template <typename T, int G, int NV>
struct AttnBackwardCols {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.kv_heads, G);
        const dim3 grid((unsigned)((a.n_sources + AB_WARPS - 1) / AB_WARPS), (a.kv_heads + a.warp_heads - 1) / a.warp_heads);
        attn_backward_cols_kernel<T, G, NV><<<grid, AB_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

cudaError_t attn_backward_rows(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardRows>(a, dtype, s); }
cudaError_t attn_backward_cols(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnBackwardCols>(a, dtype, s); }

}  // namespace dynb
