// Queries and keys of every row normalised per head and turned by the row's position (no counterpart in the reference, whose models leave
// it to their libraries):  r = 1 / sqrt(mean x^2 + eps),  n = x r g,  the pair (a, b) number p of n becomes (a c - b s, a s + b c) with c, s = cos, sin
// of 2 pi wave_p . pos_i.  Pairs are (p, p + dim / 2), or (2 p, 2 p + 1).
//     back:  dn = the gradient turned back;  dg = sum dn x r;  dx = r (g dn - x r^2 mean(g dn x));  dpos_i = 2 pi sum over pairs of wave_p
//     times the sum over the heads of q and k of (dn_b n_a - dn_a n_b).
// A head's pairs lie over 1 to 32 lanes, and these lanes take the heads of a row one after the other: what the heads share (cosines, sines and the gradient of the
// position) stays in their registers, every cosine is formed once, and the norms' sums are a few exchanges.  Where there are few rows, the heads of one are
// shared out among several such groups.  Turns are in 64 bits, whole ones are dropped, and what is left goes to 32 bits.
//
// 1 M rows of 8 + 8 heads of 16 in fp32: 328 us (6.2 TB/s), gradients 605 us (5.1 TB/s); bound by memory and the warps that registers leave.  90 k rows, 63 k of them with 8 heads of
// 64 queries, all with 2 of keys, bf16: 49 and 125 us, bound by instructions and latency.  With a warp a row and its heads side by side 394, 984, 103 and 368 us.

#include <algorithm>

#include "type_linear.cuh"

namespace dynb {

constexpr int RH_WARPS = 8, RH_MAX_HALF = 128, RH_MAX_AXES = 3;

struct RhSide {
    const void *x, *dy;          // [n, heads, dim]; the gradient of the result
    void* out;                   // result, or gradient of x
    const float* weight;
    int64_t n, row, head, dy_row, dy_head;
    int heads;
};
struct RhArgs {
    RhSide side[2];              // queries, keys
    const void* pos;
    const float* wave;
    void* d_pos;
    float* partial;              // [blocks][2][dim]: sums for the weights
    int64_t rows;
    int half, axes, pos64, norm, per_head, shares;   // per_head: lanes of a head; shares: groups of them that share the heads of a row
    float eps;
};

template <typename T, int N> struct __align__(sizeof(T) * N) RhPack { T v[N]; };

// VP pairs from pair p0 on of the head at `at`, as they stand in memory.
template <typename T, int VP, bool MIXED> struct RhRaw {
    static constexpr int N = !MIXED ? VP : VP == 1 ? 1 : 2 * VP * sizeof(T) > 16 ? VP : 2 * VP;   // of one load; one pair may stand on any element
    RhPack<T, N> v[2 * VP / N];

    __device__ __forceinline__ void load(const T* at, int p0, int half)
    {
        if constexpr (MIXED) {
#pragma unroll
            for (int i = 0; i < 2 * VP / N; i++) v[i] = *reinterpret_cast<const RhPack<T, N>*>(at + 2 * p0 + i * N);
        } else {
            v[0] = *reinterpret_cast<const RhPack<T, N>*>(at + p0);
            v[1] = *reinterpret_cast<const RhPack<T, N>*>(at + half + p0);
        }
    }
    __device__ __forceinline__ void get(float (&a)[VP], float (&b)[VP]) const
    {
#pragma unroll
        for (int i = 0; i < VP; i++) {
            a[i] = MIXED ? tl_get(&v[2 * i / N].v[2 * i % N]) : tl_get(&v[0].v[i]);
            b[i] = MIXED ? tl_get(&v[(2 * i + 1) / N].v[(2 * i + 1) % N]) : tl_get(&v[1].v[i]);
        }
    }
};
template <typename T, int VP, bool MIXED>
__device__ __forceinline__ void rh_store(T* at, int p0, int half, const float (&a)[VP], const float (&b)[VP])
{
    if constexpr (MIXED) {
        constexpr int N = VP == 1 ? 1 : 2 * VP * sizeof(T) > 16 ? VP : 2 * VP;   // one pair may stand on any element
        RhPack<T, N> v[2 * VP / N];
#pragma unroll
        for (int i = 0; i < VP; i++) {
            tl_put(&v[2 * i / N].v[2 * i % N], a[i]);
            tl_put(&v[(2 * i + 1) / N].v[(2 * i + 1) % N], b[i]);
        }
#pragma unroll
        for (int i = 0; i < 2 * VP / N; i++) *reinterpret_cast<RhPack<T, N>*>(at + 2 * p0 + i * N) = v[i];
    } else {
        RhPack<T, VP> u, w;
#pragma unroll
        for (int i = 0; i < VP; i++) {
            tl_put(&u.v[i], a[i]);
            tl_put(&w.v[i], b[i]);
        }
        *reinterpret_cast<RhPack<T, VP>*>(at + p0) = u;
        *reinterpret_cast<RhPack<T, VP>*>(at + half + p0) = w;
    }
}

// Sum over neighbouring lanes, a power of two of them, all of which call it.
__device__ __forceinline__ float rh_sum(float v, int lanes, uint32_t mask)
{
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}
__device__ __forceinline__ uint32_t rh_mask(int lanes) { return lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << ((threadIdx.x & 31) & ~(lanes - 1)); }

// Cosine and sine of a pair with the waves `wave` of a row at `at`.
template <int AXES>
__device__ __forceinline__ float2 rh_turn(const double (&at)[RH_MAX_AXES], const double* wave)
{
    double turns = 0.0;
#pragma unroll
    for (int x = 0; x < AXES; x++) turns = fma(at[x], wave[x], turns);
    const float rest = (float)(turns - rint(turns));
    float2 cs;
    sincospif(2.0f * rest, &cs.y, &cs.x);
    return cs;
}

template <typename T, int VP, int PIECES, bool MIXED, bool BACK>
__global__ void __launch_bounds__(RH_WARPS * 32, BACK ? 2 : 4)
rh_kernel(const RhArgs a)
{
    __shared__ __align__(16) float weight[2][2][RH_MAX_HALF];   // of the first and of the second elements of the pairs
    __shared__ double wave[RH_MAX_HALF * RH_MAX_AXES];           // in 64 bits once for all rows: conversions cost a row more than the sums
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, half = a.half, dim = 2 * half;
    for (int i = threadIdx.x; i < 2 * dim; i += RH_WARPS * 32) {
        const int s = i / dim, at = i % dim;
        const float v = a.side[s].weight != nullptr ? a.side[s].weight[at] : 1.0f;
        weight[s][MIXED ? at % 2 : at / half][MIXED ? at / 2 : at % half] = v;
    }
    for (int i = threadIdx.x; i < half * a.axes; i += RH_WARPS * 32) wave[i] = (double)a.wave[i];
    __syncthreads();
    const int per_row = a.per_head * a.shares, in_head = lane & (a.per_head - 1), share = (lane & (per_row - 1)) / a.per_head, rows_here = 32 / per_row;
    const uint32_t head_mask = rh_mask(a.per_head), row_mask = rh_mask(per_row);
    const float over_dim = 1.0f / (float)dim;
    float sa[2][PIECES][VP], sb[2][PIECES][VP];                  // sums for the weights' gradients
    if constexpr (BACK) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < PIECES; c++)
#pragma unroll
                for (int i = 0; i < VP; i++) sa[s][c][i] = sb[s][c][i] = 0.0f;
    }
    for (int64_t row = ((int64_t)blockIdx.x * RH_WARPS + warp) * rows_here + lane / per_row; row < a.rows; row += (int64_t)gridDim.x * RH_WARPS * rows_here) {
        float2 cs[PIECES][VP];
        float dtheta[PIECES][VP];
        double at[RH_MAX_AXES];
#pragma unroll
        for (int x = 0; x < RH_MAX_AXES; x++)
            if (x < a.axes) at[x] = a.pos64 ? static_cast<const double*>(a.pos)[row * a.axes + x] : (double)static_cast<const float*>(a.pos)[row * a.axes + x];
#pragma unroll
        for (int c = 0; c < PIECES; c++)
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const int p = (c * a.per_head + in_head) * VP + i;
                if (p >= half) cs[c][i] = make_float2(1.0f, 0.0f);
                else if (a.axes == 3) cs[c][i] = rh_turn<3>(at, wave + 3 * p);
                else if (a.axes == 2) cs[c][i] = rh_turn<2>(at, wave + 2 * p);
                else cs[c][i] = rh_turn<1>(at, wave + p);
                dtheta[c][i] = 0.0f;
            }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const RhSide& side = a.side[s];
            if (row >= side.n) continue;
            const T* const x = static_cast<const T*>(side.x) + row * side.row;
            const T* const dy = static_cast<const T*>(side.dy) + row * side.dy_row;
            T* const out = static_cast<T*>(side.out) + row * side.heads * dim;
            // In fp32 the next head's elements are on their way while one is worked on (1 M rows of 8 + 8 heads of 16, gradients: 600 against 645 us).  In 16 bits a lane
            // has eight pairs, and with four of them, which leave room for that, it takes longer (90 k rows of 8 + 2 heads of 64: 164 against 123 us).
            constexpr bool AHEAD = sizeof(T) == 4;
            RhRaw<T, VP, MIXED> x_raw[PIECES], y_raw[PIECES];
            auto fetch = [&](int h) {
#pragma unroll
                for (int c = 0; c < PIECES; c++) {
                    const int p = (c * a.per_head + in_head) * VP;
                    if (p >= half || h >= side.heads) continue;
                    x_raw[c].load(x + h * side.head, p, half);
                    if constexpr (BACK) y_raw[c].load(dy + h * side.dy_head, p, half);
                }
            };
            if constexpr (AHEAD) fetch(share);
#pragma unroll 1
            for (int h = share; h < side.heads; h += a.shares) {
                float xa[PIECES][VP], xb[PIECES][VP], ya[PIECES][VP], yb[PIECES][VP];
                float squares = 0.0f, dot = 0.0f;
#pragma unroll
                for (int c = 0; c < PIECES; c++) {
                    if ((c * a.per_head + in_head) * VP < half) {
                        if constexpr (AHEAD) {
                            x_raw[c].get(xa[c], xb[c]);
                            if constexpr (BACK) y_raw[c].get(ya[c], yb[c]);
                        } else {
                            const int p = (c * a.per_head + in_head) * VP;
                            RhRaw<T, VP, MIXED> raw;
                            raw.load(x + h * side.head, p, half);
                            raw.get(xa[c], xb[c]);
                            if constexpr (BACK) {
                                raw.load(dy + h * side.dy_head, p, half);
                                raw.get(ya[c], yb[c]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < VP; i++) xa[c][i] = xb[c][i] = ya[c][i] = yb[c][i] = 0.0f;
                    }
                }
                if constexpr (AHEAD) fetch(h + a.shares);
#pragma unroll
                for (int c = 0; c < PIECES; c++) {
                    const int p = min((c * a.per_head + in_head) * VP, half - VP);
#pragma unroll
                    for (int i = 0; i < VP; i++) {
                        squares = fmaf(xa[c][i], xa[c][i], fmaf(xb[c][i], xb[c][i], squares));
                        if constexpr (BACK) {
                            const float da = ya[c][i] * cs[c][i].x + yb[c][i] * cs[c][i].y, db = yb[c][i] * cs[c][i].x - ya[c][i] * cs[c][i].y;
                            ya[c][i] = da;
                            yb[c][i] = db;
                            dot = fmaf(weight[s][0][p + i] * da, xa[c][i], fmaf(weight[s][1][p + i] * db, xb[c][i], dot));
                        }
                    }
                }
                float r = 1.0f, back = 0.0f;
                if (a.norm) {
                    r = 1.0f / sqrtf(rh_sum(squares, a.per_head, head_mask) * over_dim + a.eps);
                    if constexpr (BACK) back = r * r * (rh_sum(dot, a.per_head, head_mask) * over_dim);
                }
#pragma unroll
                for (int c = 0; c < PIECES; c++) {
                    const int p = (c * a.per_head + in_head) * VP;
                    if (p >= half) continue;
                    float oa[VP], ob[VP];
#pragma unroll
                    for (int i = 0; i < VP; i++) {
                        const float wa = weight[s][0][p + i], wb = weight[s][1][p + i];
                        const float ua = xa[c][i] * r, ub = xb[c][i] * r;
                        if constexpr (BACK) {
                            dtheta[c][i] += yb[c][i] * (ua * wa) - ya[c][i] * (ub * wb);
                            sa[s][c][i] = fmaf(ya[c][i], ua, sa[s][c][i]);
                            sb[s][c][i] = fmaf(yb[c][i], ub, sb[s][c][i]);
                            oa[i] = r * (wa * ya[c][i] - xa[c][i] * back);
                            ob[i] = r * (wb * yb[c][i] - xb[c][i] * back);
                        } else {
                            const float na = ua * wa, nb = ub * wb;
                            oa[i] = na * cs[c][i].x - nb * cs[c][i].y;
                            ob[i] = na * cs[c][i].y + nb * cs[c][i].x;
                        }
                    }
                    if (side.out != nullptr) rh_store<T, VP, MIXED>(out + h * dim, p, half, oa, ob);
                }
            }
        }
        if constexpr (BACK) {
            if (a.d_pos != nullptr) {
                for (int x = 0; x < a.axes; x++) {
                    float d = 0.0f;
#pragma unroll
                    for (int c = 0; c < PIECES; c++)
#pragma unroll
                        for (int i = 0; i < VP; i++) {
                            const int p = (c * a.per_head + in_head) * VP + i;
                            if (p < half) d = fmaf(dtheta[c][i], (float)wave[p * a.axes + x], d);
                        }
                    __syncwarp(row_mask);
                    d = 6.2831853071795865f * rh_sum(d, per_row, row_mask);
                    if ((lane & (per_row - 1)) == 0) {
                        if (a.pos64) static_cast<double*>(a.d_pos)[row * a.axes + x] = d;
                        else static_cast<float*>(a.d_pos)[row * a.axes + x] = d;
                    }
                }
            }
        }
    }
    if constexpr (BACK) {
        if (a.partial == nullptr) return;
        // the groups of a warp, then the warps of the block, in their order
        __shared__ float sums[RH_WARPS][2][2 * RH_MAX_HALF];
        __syncwarp();
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < PIECES; c++)
#pragma unroll
                for (int i = 0; i < VP; i++) {
                    float va = sa[s][c][i], vb = sb[s][c][i];
                    for (int o = a.per_head; o < 32; o <<= 1) {
                        va += __shfl_xor_sync(0xffffffffu, va, o);
                        vb += __shfl_xor_sync(0xffffffffu, vb, o);
                    }
                    const int p = (c * a.per_head + in_head) * VP + i;
                    if (lane < a.per_head && p < half) {
                        sums[warp][s][MIXED ? 2 * p : p] = va;
                        sums[warp][s][MIXED ? 2 * p + 1 : half + p] = vb;
                    }
                }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * dim; i += RH_WARPS * 32) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < RH_WARPS; w++) v += sums[w][i / dim][i % dim];
            a.partial[(int64_t)blockIdx.x * 2 * dim + i] = v;
        }
    }
}

// The blocks' sums for the weights joined, in 64 bits: blockIdx.x is an element of [2][dim].
__global__ void __launch_bounds__(128)
rh_join_kernel(const float* partial, int blocks, int dim, float* d_q_weight, float* d_k_weight)
{
    __shared__ double sums[4];
    const int at = blockIdx.x;
    double v = 0.0;
    for (int b = threadIdx.x; b < blocks; b += 128) v += (double)partial[(int64_t)b * 2 * dim + at];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x != 0) return;
    float* const to = at < dim ? d_q_weight : d_k_weight;
    if (to != nullptr) to[at % dim] = (float)(sums[0] + sums[1] + sums[2] + sums[3]);
}

// Blocks for rows of `lanes` lanes each: no more than eight an SM, as they leave a sum each.  Four stay there together forward, two backward, and the next follow (90 k rows bf16
// with gradients: eight 48 + 124 us, four 48 + 117, two 70 + 113; 1 M rows fp32: 328 + 598, 327 + 598, 415 + 594).
static int rh_blocks(int64_t rows, int lanes)
{
    const int64_t need = (rows * lanes + 32 * RH_WARPS - 1) / (32 * RH_WARPS);
    return (int)std::max<int64_t>(1, std::min<int64_t>(need, (int64_t)sm_count_cached() * 8));
}

static int rh_args(const dynb_rotary* in, RhArgs* a)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("rotary_heads: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->pos_dtype != DYNB_F32 && in->pos_dtype != DYNB_F64) return fail_arg("rotary_heads: pos_dtype must be DYNB_F32 or DYNB_F64");
    if (in->n_q < 0 || in->n_k < 0 || in->n_q >= INT32_MAX || in->n_k >= INT32_MAX) return fail_arg("rotary_heads: rows must lie in [0, 2^31 - 1)");
    if (in->heads < 1 || in->kv_heads < 1 || in->heads > 65535 || in->kv_heads > 65535) return fail_arg("rotary_heads: heads must lie in [1, 65535]");
    if (in->dim < 2 || in->dim > DYNB_ROTARY_MAX_DIM || in->dim % 2 != 0) return fail_arg("rotary_heads: dim must be even and lie in [2, 256]");
    if (in->axes < 1 || in->axes > DYNB_ROTARY_MAX_AXES) return fail_arg("rotary_heads: axes must lie in [1, 3]");
    if (in->norm && !(in->eps >= 0.0f && in->eps <= 3.0e38f)) return fail_arg("rotary_heads: eps must be finite and not negative");
    const int64_t rows = std::max(in->n_q, in->n_k);
    if (rows > 0 && (!in->pos_dev || !in->wave_dev)) return fail_arg("null pointer");
    if ((in->n_q > 0 && !in->q_dev) || (in->n_k > 0 && !in->k_dev)) return fail_arg("null pointer");
    *a = RhArgs{};
    a->side[0].x = in->q_dev; a->side[0].row = in->q_row; a->side[0].head = in->q_head; a->side[0].n = in->n_q; a->side[0].heads = in->heads;
    a->side[1].x = in->k_dev; a->side[1].row = in->k_row; a->side[1].head = in->k_head; a->side[1].n = in->n_k; a->side[1].heads = in->kv_heads;
    a->side[0].weight = in->norm ? in->q_weight_dev : nullptr;
    a->side[1].weight = in->norm ? in->k_weight_dev : nullptr;
    a->pos = in->pos_dev; a->wave = in->wave_dev;
    a->rows = rows;
    a->half = in->dim / 2; a->axes = in->axes; a->pos64 = in->pos_dtype == DYNB_F64; a->norm = in->norm != 0; a->eps = in->eps;
    return DYNB_OK;
}

template <typename T, int VP, int PIECES, bool BACK>
static int rh_start(RhArgs& a, bool mixed, cudaStream_t s)
{
    const int lanes = (a.half + VP - 1) / VP, heads = std::max(a.side[0].heads, a.side[1].heads);
    a.per_head = 1;
    while (a.per_head < lanes && a.per_head < 32) a.per_head *= 2;
    a.shares = 1;
    while (a.per_head * a.shares < 32 && a.shares < heads && a.rows * a.per_head * a.shares < (int64_t)sm_count_cached() * 1024) a.shares *= 2;
    const int blocks = rh_blocks(a.rows, a.per_head * a.shares);
    if (mixed) rh_kernel<T, VP, PIECES, true, BACK><<<blocks, RH_WARPS * 32, 0, s>>>(a);
    else rh_kernel<T, VP, PIECES, false, BACK><<<blocks, RH_WARPS * 32, 0, s>>>(a);
    return blocks;
}

template <typename T, bool BACK>
static int rh_launch(RhArgs& a, bool mixed, cudaStream_t s)   // the number of blocks
{
    // the widest pieces that all addresses allow: a piece is VP elements of one half of a head, or 2 VP of pairs side by side
    constexpr int MOST = 16 / (int)sizeof(T);
    int vp = MOST;
    for (; vp > 1; vp /= 2) {
        const int64_t bytes = std::min(16, (int)sizeof(T) * vp * (mixed ? 2 : 1));
        bool ok = a.half % vp == 0;
        for (const RhSide& d : a.side) {
            if (d.n == 0) continue;
            const uint64_t all = reinterpret_cast<uint64_t>(d.x) | reinterpret_cast<uint64_t>(d.dy) | reinterpret_cast<uint64_t>(d.out) |
                                 (uint64_t)(sizeof(T) * d.row) | (uint64_t)(sizeof(T) * d.head) | (uint64_t)(sizeof(T) * d.dy_row) | (uint64_t)(sizeof(T) * d.dy_head);
            ok = ok && all % bytes == 0;
        }
        if (ok) break;
    }
    if constexpr (MOST == 8) {
        if (vp == 8) return rh_start<T, 8, 1, BACK>(a, mixed, s);
    }
    if (vp == 4) return rh_start<T, 4, 1, BACK>(a, mixed, s);
    // pieces of a lane: as few as 32 lanes need (100 k rows of 8 + 8 heads of 10 in fp16 with four, three of them empty: 102 and 257 us)
    if (vp == 2) return a.half <= 64 ? rh_start<T, 2, 1, BACK>(a, mixed, s) : rh_start<T, 2, 2, BACK>(a, mixed, s);
    return a.half <= 32 ? rh_start<T, 1, 1, BACK>(a, mixed, s) : a.half <= 64 ? rh_start<T, 1, 2, BACK>(a, mixed, s) : rh_start<T, 1, 4, BACK>(a, mixed, s);
}

template <bool BACK>
static int rh_run(RhArgs& a, int dtype, bool mixed, cudaStream_t s)
{
    if (dtype == DYNB_F32) return rh_launch<float, BACK>(a, mixed, s);
    if (dtype == DYNB_F16) return rh_launch<__half, BACK>(a, mixed, s);
    return rh_launch<__nv_bfloat16, BACK>(a, mixed, s);
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_rotary_heads(const dynb_rotary* args, void* q_out_dev, void* k_out_dev, void* stream)
{
    RhArgs a;
    const int rc = rh_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (a.rows == 0) return DYNB_OK;
    if ((args->n_q > 0 && !q_out_dev) || (args->n_k > 0 && !k_out_dev)) return fail_arg("null pointer");
    a.side[0].out = q_out_dev;
    a.side[1].out = k_out_dev;
    (void)rh_run<false>(a, args->dtype, args->interleaved != 0, static_cast<cudaStream_t>(stream));
    DYNB_CUDA_OK(cudaGetLastError());
    return DYNB_OK;
}

extern "C" int dynb_rotary_heads_workspace_bytes(const dynb_rotary* args, int64_t* bytes)
{
    RhArgs a;
    const int rc = rh_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (bytes == nullptr) return fail_arg("null pointer");
    *bytes = (int64_t)rh_blocks(a.rows, 32) * 4 * a.half * 4;
    return DYNB_OK;
}

extern "C" int dynb_rotary_heads_backward(const dynb_rotary* args, const void* d_q_out_dev, int64_t d_q_row, int64_t d_q_head, const void* d_k_out_dev,
                                          int64_t d_k_row, int64_t d_k_head, void* d_q_dev, void* d_k_dev, void* d_pos_dev, float* d_q_weight_dev,
                                          float* d_k_weight_dev, void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    RhArgs a;
    const int rc = rh_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if ((args->n_q > 0 && !d_q_out_dev) || (args->n_k > 0 && !d_k_out_dev)) return fail_arg("null pointer");
    const bool weights = d_q_weight_dev != nullptr || d_k_weight_dev != nullptr;
    if (weights && (workspace_dev == nullptr || !starts_on(workspace_dev, 4) || workspace_bytes < (int64_t)rh_blocks(a.rows, 32) * 4 * a.half * 4))
        return fail_arg("workspace too small");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    a.side[0].dy = d_q_out_dev; a.side[0].dy_row = d_q_row; a.side[0].dy_head = d_q_head; a.side[0].out = d_q_dev;
    a.side[1].dy = d_k_out_dev; a.side[1].dy_row = d_k_row; a.side[1].dy_head = d_k_head; a.side[1].out = d_k_dev;
    a.d_pos = d_pos_dev;
    a.partial = weights ? static_cast<float*>(workspace_dev) : nullptr;
    if (a.rows == 0 && !weights) return DYNB_OK;
    const int blocks = rh_run<true>(a, args->dtype, args->interleaved != 0, s);
    DYNB_CUDA_OK(cudaGetLastError());
    if (weights) {
        rh_join_kernel<<<4 * a.half, 128, 0, s>>>(a.partial, blocks, 2 * a.half, d_q_weight_dev, d_k_weight_dev);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    return DYNB_OK;
}
