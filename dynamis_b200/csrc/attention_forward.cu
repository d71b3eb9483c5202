// Attention of every target to its neighbours (no counterpart in the reference): for the edges e = (s -> t) of a target, per head,
//     z_e = scale q_t . k_s + bias_e,   p = softmax of z over the edges of t,   out_t = sum_e p_e v_s.
// Edges whose bias is -inf take no part, whatever their rows hold; a target without edges (or with none that takes part) gives zeros.
// One pass over the edges with the running maximum and sum of the softmax.  Sums, maxima and probabilities are in 32 bits; the
// result is rounded once.

#include "attention.cuh"

namespace dynb {

constexpr int AF_WARPS = 4;
constexpr int AF_BATCH = 4;   // edges of a slot in flight

template <typename T, int G, int NV>
__global__ void __launch_bounds__(AF_WARPS * 32)
attn_forward_kernel(const AttnArgs a)
{
    constexpr int VEC = Piece<T>::VEC;
    const int lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * AF_WARPS + (threadIdx.x >> 5);
    if (r >= a.n_targets) return;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool live = head < a.heads;
    const int h = live ? head : 0, kv = h / a.shared;
    const int32_t t = a.rows[r];
    if ((uint32_t)t >= (uint64_t)a.n_targets) return;
    const int64_t begin = max(a.row_start[r], 0), end = min((int64_t)a.row_start[r + 1], a.n_edges);
    const bool wide = a.wide != 0;

    float q[NV][VEC], acc[NV][VEC];
#pragma unroll
    for (int p = 0; p < NV; p++) {
        Piece<T>::unpack(load_piece(static_cast<const T*>(a.q.at) + t * a.q.row + h * a.q.head, (p * G + part) * VEC, a.dim, wide), q[p]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            q[p][i] *= a.scale;
            acc[p][i] = 0.0f;
        }
    }
    float top = -INFINITY, sum = 0.0f;
    const T* const kb = static_cast<const T*>(a.k.at) + kv * a.k.head;
    const T* const vb = static_cast<const T*>(a.v.at) + kv * a.v.head;
    for (int64_t base = begin; base < end; base += AF_BATCH * slots) {
        uint4 ku[AF_BATCH][NV], vu[AF_BATCH][NV];
        float z[AF_BATCH];
#pragma unroll
        for (int u = 0; u < AF_BATCH; u++) {
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
        float most = top;
#pragma unroll
        for (int u = 0; u < AF_BATCH; u++) {
            float dot = 0.0f;
#pragma unroll
            for (int p = 0; p < NV; p++) {
                float f[VEC];
                Piece<T>::unpack(ku[u][p], f);
#pragma unroll
                for (int i = 0; i < VEC; i++) dot = fmaf(q[p][i], f[i], dot);
            }
            dot = head_sum<G>(dot);
            if (z[u] != -INFINITY) z[u] += dot;
            most = fmaxf(most, z[u]);
        }
        // NaN logits must not vanish in the maximum: they reach the sums through their own exponentials
        if (most != -INFINITY) {
            const float turn = exp2f((top - most) * LOG2E);
            top = most;
            sum *= turn;
#pragma unroll
            for (int p = 0; p < NV; p++)
#pragma unroll
                for (int i = 0; i < VEC; i++) acc[p][i] *= turn;
        }
#pragma unroll
        for (int u = 0; u < AF_BATCH; u++) {
            if (z[u] == -INFINITY) continue;   // masked: not even a product with what its rows hold
            const float w = exp2f((z[u] - top) * LOG2E);
            sum += w;
#pragma unroll
            for (int p = 0; p < NV; p++) {
                float f[VEC];
                Piece<T>::unpack(vu[u][p], f);
#pragma unroll
                for (int i = 0; i < VEC; i++) acc[p][i] = fmaf(w, f[i], acc[p][i]);
            }
        }
    }
    // the slots of the warp join
    for (int o = G * a.warp_heads; o < 32; o <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        const float most = fmaxf(top, other);
        const float turn = most == -INFINITY ? 1.0f : exp2f((top - most) * LOG2E);
        top = most;
        sum *= turn;
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int p = 0; p < NV; p++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                acc[p][i] *= turn;
                acc[p][i] += __shfl_xor_sync(0xffffffffu, acc[p][i], o);
            }
    }
    if (!live || slot != 0) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t at = ((int64_t)t * a.heads + head) * a.dim;
#pragma unroll
    for (int p = 0; p < NV; p++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) acc[p][i] *= inv;
        const int d = (p * G + part) * VEC;
        store_piece(static_cast<T*>(a.out) + at, d, a.dim, wide, acc[p]);
        if (a.out32_w != nullptr) {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (d + i < a.dim) a.out32_w[at + d + i] = acc[p][i];
        }
    }
    if (a.stats_w != nullptr && part == 0) {
        a.stats_w[(int64_t)t * 2 * a.heads + head] = top;
        a.stats_w[(int64_t)t * 2 * a.heads + a.heads + head] = inv;
    }
}

template <typename T, int G, int NV>
struct AttnForward {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.heads, G);
        const dim3 grid((unsigned)((a.n_targets + AF_WARPS - 1) / AF_WARPS), (a.heads + a.warp_heads - 1) / a.warp_heads);
        attn_forward_kernel<T, G, NV><<<grid, AF_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

cudaError_t attn_forward(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnForward>(a, dtype, s); }

}  // namespace dynb
