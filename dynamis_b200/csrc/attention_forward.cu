// Attention of every target to its neighbours (no counterpart in the reference): for the edges e = (s -> t) of a target, per head,
//     z_e = scale q_t . k_s + bias_e,   p = softmax of z over the edges of t,   out_t = sum_e p_e v_s.
// Edges whose bias is -inf take no part, whatever their rows hold; a target without edges (or with none that takes part) gives zeros.
// One pass over the edges with the running maximum and sum of the softmax.  Sums, maxima and probabilities are in 32 bits; the
// result is rounded once.
//
// A warp takes a row and keeps its queries and sums in registers; what it reads an edge is a row of keys and one of values, gathered, mostly from L2
// and L1.  What bounds it is latency and issue with 16 warps an SM (with neighbouring rows in all of them half the bytes come from L2, and it is no
// faster).  200 k targets, 10.5 M edges, 8 x 16 fp32: 699 us (the bytes that have to be read once take 0.12 ms of memory's time); 150 k targets, bf16, 8 heads
// on 2 of 32: 686 us.

#include <algorithm>

#include "attention.cuh"

namespace dynb {

constexpr int AF_WARPS = 4;
// Edges of a slot in a batch: what 128 registers hold (4 bytes at most spill).  Rows of 16 bits are unpacked; heads of odd sizes need registers for their loads.
template <typename T, bool FULL> constexpr int AF_BATCH = !FULL ? 2 : sizeof(T) == 4 ? 4 : 3;

// WPR warps take turns at the batches of a row and join through shared memory.
template <typename T, int G, bool FULL, int WPR>
__global__ void __launch_bounds__(AF_WARPS * 32, 4)
attn_forward_kernel(const AttnArgs a)
{
    constexpr int EL = LaneElements<T>::N, BATCH = AF_BATCH<T, FULL>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane % G, slots = 32 / (G * a.warp_heads), slot = lane / (G * a.warp_heads);
    const int head = blockIdx.y * a.warp_heads + (lane / G) % a.warp_heads;
    const bool mine = head < a.heads;
    const int wide = a.wide;
    const int h = mine ? head : 0, kv = h / a.shared;
    const Place<T, G, EL> place(part);
    const uint32_t sources = (uint32_t)a.n_sources;
    const Lane<T, G, EL> k_lane(a.k, kv, place), v_lane(a.v, kv, place);
    constexpr int ROWS = AF_WARPS / WPR;
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

        float2 q[EL / 2], acc[EL / 2];
        attn_pairs(attn_load<T, G, EL, FULL>(t >= 0 ? static_cast<const T*>(a.q.at) + t * a.q.row + h * a.q.head : reinterpret_cast<const T*>(zeros), place, a.dim, wide), q);
#pragma unroll
        for (int i = 0; i < EL / 2; i++) {
            q[i] = mul2(q[i], make_float2(a.scale, a.scale));
            acc[i] = make_float2(0.0f, 0.0f);
        }
        float top = -INFINITY, sum = 0.0f;
        int e = turn * step + slot * BATCH;
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
            float most = top;
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                float2 f[EL / 2];
                attn_pairs(s.x[u], f);
                const float product = head_sum<G>(inner(q, f));
                s.z[u] = s.ok[u] ? s.z[u] + product : -INFINITY;
                most = fmaxf(most, s.z[u]);
            }
            // NaN logits are not in the maximum: they reach the sums through their own exponentials
            const float from = most == -INFINITY ? 0.0f : most, back = pow2((top - from) * LOG2E);
            top = most;
            sum *= back;
#pragma unroll
            for (int i = 0; i < EL / 2; i++) acc[i] = mul2(acc[i], make_float2(back, back));
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                const float w = pow2((s.z[u] - from) * LOG2E);
                sum += w;
                float2 f[EL / 2];
                attn_pairs(s.y[u], f);
#pragma unroll
                for (int i = 0; i < EL / 2; i++) acc[i] = fma2(make_float2(w, w), f[i], acc[i]);
            }
        };
        for (int base = turn * step; base < n; base += WPR * step) {   // the same for all lanes
            AttnStep<T, EL, BATCH> s;
            load(s);
            work(s);
        }
        // the slots of the warp join
        for (int o = G * a.warp_heads; o < 32; o <<= 1) {
            const float most = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float back = most == -INFINITY ? 1.0f : pow2((top - most) * LOG2E);
            top = most;
            sum *= back;
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
            for (int i = 0; i < EL / 2; i++) {
                acc[i].x *= back;
                acc[i].y *= back;
                acc[i].x += __shfl_xor_sync(0xffffffffu, acc[i].x, o);
                acc[i].y += __shfl_xor_sync(0xffffffffu, acc[i].y, o);
            }
        }
        if (WPR > 1) {   // the warps of the row join in their order
            __shared__ float joint[AF_WARPS][EL + 2][32];
            __syncthreads();
            joint[warp][EL][lane] = top;
            joint[warp][EL + 1][lane] = sum;
#pragma unroll
            for (int i = 0; i < EL / 2; i++) {
                joint[warp][2 * i][lane] = acc[i].x;
                joint[warp][2 * i + 1][lane] = acc[i].y;
            }
            __syncthreads();
            if (turn != 0) continue;
            float most = top;
#pragma unroll
            for (int w = 1; w < WPR; w++) most = fmaxf(most, joint[warp + w][EL][lane]);
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < EL / 2; i++) acc[i] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WPR; w++) {
                const float back = most == -INFINITY ? 1.0f : pow2((joint[warp + w][EL][lane] - most) * LOG2E);
                sum = fmaf(joint[warp + w][EL + 1][lane], back, sum);
#pragma unroll
                for (int i = 0; i < EL / 2; i++) {
                    acc[i].x = fmaf(joint[warp + w][2 * i][lane], back, acc[i].x);
                    acc[i].y = fmaf(joint[warp + w][2 * i + 1][lane], back, acc[i].y);
                }
            }
            top = most;
        }
        if (!mine || slot != 0 || t < 0) continue;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t at = ((int64_t)t * a.heads + head) * a.dim;
#pragma unroll
        for (int i = 0; i < EL / 2; i++) acc[i] = mul2(acc[i], make_float2(inv, inv));
        attn_store<T, G, EL, FULL>(static_cast<T*>(a.out) + at, place, a.dim, wide, acc);
        if (sizeof(T) != 4 && a.out32_w != nullptr) {
            constexpr int VEC = Place<T, G, EL>::VEC;
#pragma unroll
            for (int i = 0; i < EL / 2; i++) {
                const int d = place.at[2 * i / VEC] + 2 * i % VEC;
                if (FULL) {
                    *reinterpret_cast<float2*>(a.out32_w + at + d) = acc[i];
                } else {
                    if (d < a.dim) a.out32_w[at + d] = acc[i].x;
                    if (d + 1 < a.dim) a.out32_w[at + d + 1] = acc[i].y;
                }
            }
        }
        if (a.stats_w != nullptr && part == 0) {
            a.stats_w[(int64_t)t * 2 * a.heads + head] = top;
            a.stats_w[(int64_t)t * 2 * a.heads + a.heads + head] = inv;
        }
    }
}

template <typename T, int G, bool FULL>
struct AttnForward {
    static cudaError_t go(const AttnArgs& args, cudaStream_t s)
    {
        AttnArgs a = args;
        a.warp_heads = attn_warp_heads(a.heads, G);
        const int blocks = (a.heads + a.warp_heads - 1) / a.warp_heads;
        const bool split = attn_split(a.n_targets * blocks, a.n_edges * blocks);
        const int rows = split ? AF_WARPS / 4 : AF_WARPS;
        a.block_rows = attn_block_rows(a.n_targets * blocks, rows);
        const dim3 grid((unsigned)((a.n_targets + a.block_rows - 1) / a.block_rows), blocks);
        if (split) attn_forward_kernel<T, G, FULL, 4><<<grid, AF_WARPS * 32, 0, s>>>(a);
        else attn_forward_kernel<T, G, FULL, 1><<<grid, AF_WARPS * 32, 0, s>>>(a);
        return cudaGetLastError();
    }
};

cudaError_t attn_forward(const AttnArgs& a, int dtype, cudaStream_t s) { return attn_by_type<AttnForward>(a, dtype, s); }

}  // namespace dynb
