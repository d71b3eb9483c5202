// Experts for rows (no counterpart in the reference, whose models leave it to their libraries).  From a row's logits l:
//     s = softmax(l), or sigmoid(l);   key = s + bias;   a group's key is the sum of its two largest keys; the largest `kept` groups stay, and of their
//     experts the `choices` largest keys are chosen, in falling order, the lowest number first among equal ones;   w = scale s, or scale s / (sum of the chosen s).
// Logits or biases of -inf close an expert.  A place that no expert is left for gets number -1 and weight 0.
// Keys are compared in 64 bits, and where nothing but the logits decides, by the logits themselves: which expert is chosen does not depend on how a
// 32-bit exponential rounds.
//
// The (row, choice) pairs by expert, ascending inside one: every block counts its rows' choices, the counts are summed over the blocks, and every block
// puts its pairs where its counts say.  No atomics on memory, no wait of the host: the same order each time, and the calls can be captured.
//
// 200 k rows of 64 experts, six choices of four of eight groups, bias: 102 us (choice 81) and 35 for the gradient; 1 M rows of 32 experts in bf16, two choices: 89 and 59 us.  Bound by the
// instructions of a row (keys, lists), not by its bytes.

#include <algorithm>

#include "type_linear.cuh"

namespace dynb {

constexpr int RE_WARPS = 8;

struct ReArgs {
    const void* logits;
    const float* bias;
    int32_t *experts, *order, *start, *counts, *sums;   // counts [experts + 1][blocks], sums [experts + 1]
    float* weights;
    int64_t n, row;          // row: stride of the logits
    int64_t chunk;           // rows of a block
    int count, choices, groups, kept, sigmoid, renormalize;
    float scale;
};

__device__ __forceinline__ uint64_t re_max(uint64_t v)   // of a warp
{
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}
// A key as a whole number in the same order: 0 for what is closed, NaN above all.
__device__ __forceinline__ uint64_t re_order(double key)
{
    if (isnan(key)) return ~0ull;
    return key == -INFINITY ? 0ull : ordered_u64(key + 0.0);   // -0 and 0 are equal
}

// A row by a warp.  V: experts of a lane; scratch: room for the experts and the groups.
template <typename T, int V>
__device__ __forceinline__ void re_row(const ReArgs& a, int64_t row, double* scratch, int32_t* counts)
{
    const int lane = threadIdx.x & 31, per = a.count / a.groups;
    const bool plain = a.bias == nullptr && a.groups == 1;   // the logits decide
    const T* const l = static_cast<const T*>(a.logits) + row * a.row;
    float logit[V];
    uint64_t key[V];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane + 32 * i;
        logit[i] = e < a.count ? tl_get(l + e) : -INFINITY;
        top = fmaxf(top, logit[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (plain) {
#pragma unroll
        for (int i = 0; i < V; i++) key[i] = re_order((double)logit[i]);
    } else {
        double s[V], sum = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (a.sigmoid) {
                s[i] = 1.0 / (1.0 + exp(-(double)logit[i]));
            } else {
                s[i] = logit[i] == -INFINITY ? 0.0 : exp((double)logit[i] - (double)top);
                sum += s[i];
            }
        }
        if (!a.sigmoid) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = lane + 32 * i;
            const double v = (a.sigmoid ? s[i] : s[i] / sum) + (a.bias != nullptr && e < a.count ? (double)a.bias[e] : 0.0);
            key[i] = logit[i] == -INFINITY ? 0ull : re_order(v);
        }
        if (a.groups > 1) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < V; i++)
                if (lane + 32 * i < a.count) scratch[lane + 32 * i] = __longlong_as_double((long long)key[i]);
            __syncwarp();
            uint64_t* const of_group = reinterpret_cast<uint64_t*>(scratch + a.count);
            for (int g = lane; g < a.groups; g += 32) {
                uint64_t one = 0, two = 0;
                for (int j = 0; j < per; j++) {
                    const uint64_t k = (uint64_t)__double_as_longlong(scratch[g * per + j]);
                    two = max(two, min(one, k));
                    one = max(one, k);
                }
                uint64_t both = one;
                if (one == ~0ull || two == ~0ull) both = ~0ull;
                else if (two != 0) both = re_order(unordered_f64(one) + unordered_f64(two));
                if (one != 0 && both == 0) both = 1;   // open, however low
                of_group[g] = both;
            }
            __syncwarp();
            // a group stays when fewer than `kept` come before it
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int e = lane + 32 * i;
                if (e >= a.count) continue;
                const int g = e / per;
                const uint64_t mine = of_group[g];
                int before = 0;
                for (int h = 0; h < a.groups; h++) before += of_group[h] > mine || (of_group[h] == mine && h < g);
                if (before >= a.kept) key[i] = 0;
            }
        }
    }
    // the choices, one after the other; lane j keeps choice j
    int32_t mine = -1;
    float mine_logit = -INFINITY;
    for (int j = 0; j < a.choices; j++) {
        uint64_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; i++) best = max(best, key[i]);
        best = re_max(best);
        if (best == 0) break;
        uint32_t at = 0xffffffffu;
        float with = 0.0f;
#pragma unroll
        for (int i = V - 1; i >= 0; i--)
            if (key[i] == best) { at = lane + 32 * i; with = logit[i]; }
        const uint32_t chosen = __reduce_min_sync(0xffffffffu, at);
        with = __shfl_sync(0xffffffffu, with, chosen & 31);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (chosen == lane + 32 * i) key[i] = 0;
        if (lane == j) { mine = (int32_t)chosen; mine_logit = with; }
    }
    float w = 0.0f;
    if (a.sigmoid && !a.renormalize) {
        w = 1.0f / (1.0f + expf(-mine_logit));
    } else {
        // log s up to what all share; sums of exponentials below the largest
        const float z = a.sigmoid ? fminf(mine_logit, 0.0f) - log1pf(expf(-fabsf(mine_logit))) : mine_logit;
        const float zz = mine < 0 ? -INFINITY : isnan(mine_logit) ? mine_logit : z;
        float most = zz;
        if (a.renormalize) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        } else {
            most = top;
        }
        w = mine < 0 ? 0.0f : expf(zz - most);
        float sum = 0.0f;
        if (a.renormalize) {
            sum = w;
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) sum += logit[i] == -INFINITY ? 0.0f : expf(logit[i] - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (mine >= 0) w /= sum;
        if (!a.sigmoid) {   // a NaN or +inf anywhere leaves no score of the row a number
            bool odd = top == INFINITY;
#pragma unroll
            for (int i = 0; i < V; i++) odd = odd || isnan(logit[i]);
            if (__any_sync(0xffffffffu, odd)) w = NAN;
        }
    }
    if (lane < a.choices) {
        a.experts[row * a.choices + lane] = mine;
        a.weights[row * a.choices + lane] = mine < 0 ? 0.0f : a.scale * w;
        atomicAdd(counts + (mine < 0 ? a.count : mine), 1);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(RE_WARPS * 32)
re_choose_kernel(const ReArgs a)
{
    extern __shared__ unsigned char raw_smem[];
    int32_t* const counts = reinterpret_cast<int32_t*>(raw_smem);                              // [experts + 1]
    double* const scratch = reinterpret_cast<double*>(raw_smem + ((a.count + 1) * 4 + 15) / 16 * 16) + (threadIdx.x / 32) * (a.count + a.groups);
    for (int i = threadIdx.x; i <= a.count; i += RE_WARPS * 32) counts[i] = 0;
    __syncthreads();
    const int64_t first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.n);
    for (int64_t row = first + threadIdx.x / 32; row < last; row += RE_WARPS) re_row<T, V>(a, row, scratch, counts);
    __syncthreads();
    for (int i = threadIdx.x; i <= a.count; i += RE_WARPS * 32) a.counts[(int64_t)i * gridDim.x + blockIdx.x] = counts[i];
}

// ------------------------------------------------------------------------------------------------ a thread a row
// Up to 128 experts, 8 choices and 16 groups: a warp brings 32 rows to shared memory and every lane goes along one.  (A warp a row spends its time on exchanges between
// lanes: 1 M rows of 32 bf16 logits, two choices, 350 us and now 65; gradient 292 and 59.)  Where more than the logits decide, keys are formed in 32 bits first; rows in which two that
// matter lie nearer to one another than these may be off are looked at again in 64 bits.
constexpr int RT_WARPS = 4, RT_MAX_EXPERTS = 128, RT_MAX_CHOICES = 8, RT_MAX_GROUPS = 16;

// As re_order: 0 for -infinity, NaN above all (arithmetic gives the one NaN whose bits below the sign are all set); adding zero makes zeros of both signs equal.
__device__ __forceinline__ uint32_t rt_order(float key)
{
    const uint32_t bits = __float_as_uint(key + 0.0f);
    return (bits ^ (uint32_t)((int32_t)bits >> 31 | (int32_t)0x80000000)) - 0x007fffffu;
}
__device__ __forceinline__ float rt_value(uint32_t order)
{
    const uint32_t bits = order + 0x007fffffu;
    return __uint_as_float(bits ^ (uint32_t)(~((int32_t)bits >> 31) | (int32_t)0x80000000));
}
__device__ __forceinline__ bool rt_nan(uint32_t order) { return order == 0xff800000u; }
// 32 rows from `row0` on to `tile` (`pitch` floats a row).  Rows behind the last are not written, and nobody reads them.
template <typename T>
__device__ __forceinline__ void rt_bring(const ReArgs& a, int64_t row0, float* tile, int pitch, int wide)
{
    const int lane = threadIdx.x & 31;
    const T* const l = static_cast<const T*>(a.logits);
    constexpr int N = 16 / (int)sizeof(T);
    if (wide) {
        const int per = a.count / N;
        int r = lane / per, c = lane % per;
        const int rows = 32 / per, rest = 32 % per;      // 32 pieces on
#pragma unroll 4
        for (int u = lane; u < 32 * per; u += 32) {
            if (row0 + r < a.n) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(l + (row0 + r) * a.row + c * N));
                const T* const e = reinterpret_cast<const T*>(&v);
#pragma unroll
                for (int i = 0; i < N; i++) tile[r * pitch + c * N + i] = tl_get(e + i);
            }
            r += rows;
            c += rest;
            if (c >= per) { c -= per; r++; }
        }
    } else {
        for (int u = lane; u < 32 * a.count; u += 32) {
            const int r = u / a.count, c = u % a.count;
            if (row0 + r >= a.n) break;
            tile[r * pitch + c] = tl_get(l + (row0 + r) * a.row + c);
        }
    }
}

// Puts key k of expert e where it belongs among the largest: behind those that are equal.
template <int MOST>
__device__ __forceinline__ void rt_insert(uint32_t k, int e, int (&chosen)[MOST], uint32_t (&order)[MOST])
{
    if (k <= order[MOST - 1]) return;
#pragma unroll
    for (int j = MOST - 1; j >= 0; j--) {
        if (k <= order[j]) continue;
        if (j + 1 < MOST) {
            order[j + 1] = order[j];
            chosen[j + 1] = chosen[j];
        }
        order[j] = k;
        chosen[j] = e;
    }
}

// The experts of a lane's row.  key_of(e): keys in their order, as often as asked; MOST: choices and two or more, the first that are left out.
// False: keys that are off by up to `near` may have decided.  same(p, q): two experts have the same logit and bias, and so the same key, whatever its type.
template <int MOST, int GROUPS, typename Key, typename Same>
__device__ __forceinline__ bool rt_choose(const ReArgs& a, float near, int (&chosen)[MOST], Key&& key_of, Same&& same)
{
    bool sure = true;
    uint32_t kept = 0;
    const int per = a.count / a.groups;
    if constexpr (GROUPS > 1) {
        uint32_t of_group[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            of_group[g] = 0;
            if (g >= a.groups) continue;
            uint32_t one = 0, two = 0;
#pragma unroll 4
            for (int i = 0; i < per; i++) {
                const uint32_t k = key_of(g * per + i);
                two = max(two, min(one, k));
                one = max(one, k);
            }
            uint32_t both = one;
            if (two != 0) both = rt_nan(one) ? one : rt_order(rt_value(one) + rt_value(two));
            if (one != 0 && both == 0) both = 1;   // open, however low
            of_group[g] = both;
        }
        uint32_t lowest = ~0u, highest = 0;   // of those that stay, and of the others
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            if (g >= a.groups) continue;
            int before = 0;
#pragma unroll
            for (int h = 0; h < GROUPS; h++) before += h < a.groups && (of_group[h] > of_group[g] || (of_group[h] == of_group[g] && h < g));
            if (before < a.kept) {
                kept |= 1u << g;
                lowest = min(lowest, of_group[g]);
            } else {
                highest = max(highest, of_group[g]);
            }
        }
        if (highest != 0) sure = rt_value(lowest) - rt_value(highest) > 6.0f * near;
    }
    uint32_t order[MOST];
#pragma unroll
    for (int j = 0; j < MOST; j++) {
        order[j] = 0;
        chosen[j] = -1;
    }
    if constexpr (GROUPS > 1) {
        // the groups that stay, ascending: each lane its own, so that none waits for those of the others
        for (int i0 = 0; i0 < a.kept; i0++, kept &= kept - 1) {
            const int first = (__ffs(kept) - 1) * per;
#pragma unroll 4
            for (int i = 0; i < per; i++) rt_insert(key_of(first + i), first + i, chosen, order);
        }
    } else {
#pragma unroll 4
        for (int e = 0; e < a.count; e++) rt_insert(key_of(e), e, chosen, order);
    }
    bool tie = false;   // the last choice and the first that is left out have the same key
#pragma unroll
    for (int j = 0; j + 1 < MOST; j++) {
        if (order[j + 1] == 0 || j > a.choices || (j == a.choices && !tie)) continue;
        if (rt_value(order[j]) - rt_value(order[j + 1]) > 2.0f * near) continue;
        tie = j == a.choices - 1;
        if (j == a.choices || !same(chosen[j], chosen[j + 1])) sure = false;
    }
    return sure;
}

// The weights of a row's choices and its entries in the counts.  sum: of the row's exponentials below `top`, for softmax without renormalising; odd: a logit is NaN.
template <typename T, int MOST>
__device__ __forceinline__ void rt_weigh(const ReArgs& a, int64_t row, const int (&chosen)[MOST], float top, float sum, bool odd, int32_t* counts)
{
    const T* const from = static_cast<const T*>(a.logits) + row * a.row;
    odd = odd || top == INFINITY;
    float w[MOST], most = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < MOST; j++) {
        const bool have = j < a.choices && chosen[j] >= 0;
        const float v = have ? tl_get(from + chosen[j]) : 0.0f;
        // log s up to what all share; sums of exponentials below the largest
        w[j] = !a.sigmoid || !a.renormalize ? v : isnan(v) ? v : fminf(v, 0.0f) - log1pf(expf(-fabsf(v)));
        if (have) most = fmaxf(most, w[j]);
    }
#pragma unroll
    for (int j = 0; j < MOST; j++) {
        if (j >= a.choices || chosen[j] < 0) continue;
        if (a.renormalize) {
            w[j] = expf(w[j] - most);
            total += w[j];
        } else {
            w[j] = a.sigmoid ? 1.0f / (1.0f + expf(-w[j])) : expf(w[j] - top) / sum;
        }
    }
#pragma unroll
    for (int j = 0; j < MOST; j++) {
        if (j >= a.choices) continue;
        float v = chosen[j] < 0 ? 0.0f : a.renormalize ? w[j] / total : w[j];
        if (!a.sigmoid && odd && chosen[j] >= 0) v = NAN;   // a NaN or +inf anywhere leaves no score of the row a number
        a.experts[row * a.choices + j] = chosen[j];
        a.weights[row * a.choices + j] = chosen[j] < 0 ? 0.0f : a.scale * v;
        atomicAdd(counts + (chosen[j] < 0 ? a.count : chosen[j]), 1);
    }
}

// A row from the start in 64 bits, by the whole warp (by the lane alone, for which the others wait, 200 k rows of 64 experts in groups take 131 in place of 91 us).
template <typename T>
__device__ __noinline__ void rt_again(const ReArgs& a, int64_t row, double* scratch, int32_t* counts) { re_row<T, RT_MAX_EXPERTS / 32>(a, row, scratch, counts); }

// GROUPS: 0 where the logits decide, 1 without groups, else their largest number.
template <typename T, int MOST, int GROUPS>
__global__ void __launch_bounds__(RT_WARPS * 32, GROUPS == 0 ? 12 : 8)
rt_choose_kernel(const ReArgs a, int pitch, int wide)
{
    constexpr bool PLAIN = GROUPS == 0;
    extern __shared__ unsigned char raw_smem[];
    int32_t* const counts = reinterpret_cast<int32_t*>(raw_smem);   // [experts + 1], then the biases [experts], then the rows of every warp
    float* const bias = reinterpret_cast<float*>(counts + a.count + 1);
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    float* const tile = bias + a.count + warp * 32 * pitch;
    float* const l = tile + lane * pitch;
    float far = 0.0f;
    for (int i = threadIdx.x; i <= a.count; i += RT_WARPS * 32) counts[i] = 0;
    for (int i = threadIdx.x; i < a.count; i += RT_WARPS * 32) bias[i] = a.bias != nullptr ? a.bias[i] : 0.0f;
    __syncthreads();
    if constexpr (!PLAIN)
        for (int i = lane; i < a.count; i += 32) far = fmaxf(far, isinf(bias[i]) ? 0.0f : fabsf(bias[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) far = fmaxf(far, __shfl_xor_sync(0xffffffffu, far, o));
    // how far a key in 32 bits may be off: a score by (experts + 16) 2^-24 (sigmoids 8: exponential and division (3 + |v|) s (1 - s) and 2), the sum with the bias by half a step.
    // One bound for all keys: where those that decide are all small (a peaked softmax, sigmoids far below zero, no bias), many rows are looked at again.  200 k rows of 64
    // experts in groups, logits of spread 1.5, 4 and 8: softmax 91, 116 and 308 us, sigmoids 69, 92 and 570; with a bias 67 to 86 at any spread.
    const float near = ((a.sigmoid ? 8.0f : a.count + 16.0f) + 2.0f * far) * 0x1p-24f;
    const int64_t first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.n);
    for (int64_t row0 = first + warp * 32; row0 < last; row0 += RT_WARPS * 32) {
        const int64_t row = row0 + lane;
        __syncwarp();
        rt_bring<T>(a, row0, tile, pitch, wide);
        __syncwarp();
        bool again = false;
        if (row < last) {
        int chosen[MOST];
        float top = -INFINITY, sum = 0.0f;
        bool odd = false;
        if constexpr (PLAIN) {
            uint32_t order[MOST];
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                order[j] = 0;
                chosen[j] = -1;
            }
#pragma unroll 8
            for (int e = 0; e < a.count; e++) {
                const float v = l[e];
                top = fmaxf(top, v);
                odd = odd || isnan(v);
                rt_insert(rt_order(v), e, chosen, order);
            }
            if (!a.sigmoid && !a.renormalize) {
#pragma unroll 8
                for (int e = 0; e < a.count; e++) sum += l[e] == -INFINITY ? 0.0f : __expf(l[e] - top);   // off by 2 + |l - top| units in the last place, of what is small where that is large
            }
        } else {
            // logits give way to their keys
            if (!a.sigmoid) {
#pragma unroll 4
                for (int e = 0; e < a.count; e++) {
                    top = fmaxf(top, l[e]);
                    odd = odd || isnan(l[e]);
                }
#pragma unroll 4
                for (int e = 0; e < a.count; e++) {
                    const float v = l[e] == -INFINITY ? -1.0f : __expf(l[e] - top);
                    sum += fmaxf(v, 0.0f) + (v - v);   // a NaN stays one
                    l[e] = v;
                }
            }
            const float over = 1.0f / sum;
#pragma unroll 4
            for (int e = 0; e < a.count; e++) {
                const float v = l[e];
                const float key = a.sigmoid ? __fdividef(1.0f, 1.0f + __expf(-v)) : v * over;
                const bool closed = v < (a.sigmoid ? -3.402823466e38f : 0.0f);   // -infinity, or its mark
                l[e] = __uint_as_float(closed ? 0u : rt_order(key + bias[e]));
            }
            const T* const from = static_cast<const T*>(a.logits) + row * a.row;
            // what is to be done once more waits until nothing else is in registers
            again = !rt_choose<MOST, GROUPS>(
                a, near, chosen, [&](int e) { return __float_as_uint(l[e]); },
                [&](int p, int q) { return tl_get(from + p) == tl_get(from + q) && bias[p] == bias[q]; });
        }
        if (!again) rt_weigh<T, MOST>(a, row, chosen, top, sum, odd, counts);
        }
        if constexpr (!PLAIN) {   // the rows' places serve as scratch meanwhile
            double* const scratch = reinterpret_cast<double*>(tile + (reinterpret_cast<uintptr_t>(tile) % 8 != 0));
            for (uint32_t todo = __ballot_sync(0xffffffffu, again); todo != 0; todo &= todo - 1) rt_again<T>(a, row0 + __ffs(todo) - 1, scratch, counts);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= a.count; i += RT_WARPS * 32) a.counts[(int64_t)i * gridDim.x + blockIdx.x] = counts[i];
}

// Counts of an expert (blockIdx.x) over the blocks become the pairs of it before each block; their sum.
__global__ void __launch_bounds__(256)
re_sums_kernel(int32_t* counts, int32_t* sums, int blocks)
{
    __shared__ int warp_sums[8];
    chain_begin();
    int32_t* const mine = counts + (int64_t)blockIdx.x * blocks;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int before = 0;
    for (int b0 = 0; b0 < blocks; b0 += 256) {
        const int b = b0 + threadIdx.x, v = b < blocks ? mine[b] : 0;
        int total;
        int at = warp_excl_scan(v, lane, &total);
        if (lane == 0) warp_sums[warp] = total;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) {
            if (w < warp) at += warp_sums[w];
            all += warp_sums[w];
        }
        if (b < blocks) mine[b] = before + at;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) sums[blockIdx.x] = before;
}

// Pairs of a block's rows to their places: a warp takes a run of them, 32 at a time.
__global__ void __launch_bounds__(RE_WARPS * 32)
re_place_kernel(const ReArgs a)
{
    extern __shared__ unsigned char raw_smem[];
    int32_t* const start = reinterpret_cast<int32_t*>(raw_smem);          // [experts + 1]; then [warps][experts + 1]
    int32_t* const next = start + a.count + 1;
    __shared__ int warp_sums[RE_WARPS];
    chain_begin();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, all = a.count + 1;
    for (int i = threadIdx.x; i < RE_WARPS * all; i += RE_WARPS * 32) next[i] = 0;
    int before = 0;
    for (int e0 = 0; e0 < all; e0 += RE_WARPS * 32) {
        const int e = e0 + threadIdx.x, v = e < all ? a.sums[e] : 0;
        int total;
        int at = warp_excl_scan(v, lane, &total);
        if (lane == 0) warp_sums[warp] = total;
        __syncthreads();
        int sum = 0;
#pragma unroll
        for (int w = 0; w < RE_WARPS; w++) {
            if (w < warp) at += warp_sums[w];
            sum += warp_sums[w];
        }
        if (e < all) {
            start[e] = before + at;
            if (blockIdx.x == 0) a.start[e] = before + at;
        }
        before += sum;
        __syncthreads();
    }
    const int64_t first = blockIdx.x * a.chunk * a.choices, last = min(blockIdx.x * a.chunk + a.chunk, a.n) * a.choices;
    const int64_t run = ((last - first + RE_WARPS - 1) / RE_WARPS + 31) / 32 * 32, from = min(first + warp * run, last), to = min(from + run, last);
    for (int64_t p = from + lane; p < to; p += 32) {
        const int e = a.experts[p];
        atomicAdd(next + warp * all + (e < 0 ? a.count : e), 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < all; e += RE_WARPS * 32) {
        int at = start[e] + a.counts[(int64_t)e * gridDim.x + blockIdx.x];
        for (int w = 0; w < RE_WARPS; w++) {
            const int v = next[w * all + e];
            next[w * all + e] = at;
            at += v;
        }
    }
    __syncthreads();
    for (int64_t p0 = from; p0 < to; p0 += 32) {
        const int64_t p = p0 + lane;
        const bool live = p < to;
        const int e = live ? a.experts[p] : -2, slot = e < 0 ? a.count : e;
        const uint32_t same = __match_any_sync(0xffffffffu, live ? slot : -2);
        const int at = live ? next[warp * all + slot] : 0, rank = __popc(same & lanemask_lt());
        __syncwarp();
        if (live) {
            a.order[at + rank] = (int32_t)p;
            if (rank == 0) next[warp * all + slot] = at + __popc(same);
        }
        __syncwarp();
    }
}

__device__ __forceinline__ float re_sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

// The gradient of the logits.  p: the weights without the scale, g: their gradient times the scale.
//     renormalised: d = p (g - sum p g), for sigmoids times 1 - s;   sigmoid: g s (1 - s);   softmax: s_e (g_e - sum s g) for every expert e.
// 1 - s is formed as the sigmoid of -l: the difference has lost its digits for a gate that is open (half a per cent off at l = 12, zero from 17 on).
template <typename T, int V>
__global__ void __launch_bounds__(RE_WARPS * 32)
re_backward_kernel(const ReArgs a, const float* d_weights, T* d_logits)
{
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int64_t row = (int64_t)blockIdx.x * RE_WARPS + warp; row < a.n; row += (int64_t)gridDim.x * RE_WARPS) {
        const T* const l = static_cast<const T*>(a.logits) + row * a.row;
        int32_t e = -1;
        float w = 0.0f, g = 0.0f;
        if (lane < a.choices) {
            e = a.experts[row * a.choices + lane];
            if ((uint32_t)e >= (uint32_t)a.count) e = -1;
            w = a.weights[row * a.choices + lane] / a.scale;
            g = d_weights[row * a.choices + lane] * a.scale;
        }
        const bool live = e >= 0;
        const float v = live ? tl_get(l + e) : 0.0f;
        float dot = live ? w * g : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        float d = 0.0f;
        if (live) {
            if (a.renormalize) d = w * (g - dot) * (a.sigmoid ? re_sigmoid(-v) : 1.0f);
            else d = a.sigmoid ? g * re_sigmoid(v) * re_sigmoid(-v) : g;
        }
        float out[V];
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = 0.0f;
        for (int j = 0; j < a.choices; j++) {
            const int at = __shfl_sync(0xffffffffu, e, j);
            const float v = __shfl_sync(0xffffffffu, d, j);
#pragma unroll
            for (int i = 0; i < V; i++)
                if (at == lane + 32 * i) out[i] = v;
        }
        if (!a.sigmoid && !a.renormalize) {
            float logit[V], top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) {
                logit[i] = lane + 32 * i < a.count ? tl_get(l + lane + 32 * i) : -INFINITY;
                top = fmaxf(top, logit[i]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
            for (int i = 0; i < V; i++) {
                logit[i] = logit[i] == -INFINITY ? 0.0f : expf(logit[i] - top);
                sum += logit[i];
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
            for (int i = 0; i < V; i++) out[i] = sum == 0.0f ? 0.0f : logit[i] / sum * (out[i] - dot);
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane + 32 * i < a.count) tl_put(d_logits + row * a.count + lane + 32 * i, out[i]);
    }
}

// The same, a thread a row (see rt_choose_kernel): the gradients of 32 rows are put together in shared memory.
template <typename T>
__global__ void __launch_bounds__(RT_WARPS * 32, 10)
rt_backward_kernel(const ReArgs a, const float* d_weights, T* d_logits, int pitch, int wide, int wide_out)
{
    extern __shared__ unsigned char raw_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    float* const tile = reinterpret_cast<float*>(raw_smem) + warp * 32 * pitch;
    float* const l = tile + lane * pitch;
    const bool dense = !a.sigmoid && !a.renormalize;   // every logit has a gradient
    for (int64_t row0 = ((int64_t)blockIdx.x * RT_WARPS + warp) * 32; row0 < a.n; row0 += (int64_t)gridDim.x * RT_WARPS * 32) {
        const int64_t row = row0 + lane;
        __syncwarp();
        if (dense) rt_bring<T>(a, row0, tile, pitch, wide);
        else
            for (int i = lane; i < 32 * pitch; i += 32) tile[i] = 0.0f;
        __syncwarp();
        if (row < a.n) {
            // all of a row's choices at once: their loads do not wait for one another
            int e[RT_MAX_CHOICES];
            float w[RT_MAX_CHOICES], g[RT_MAX_CHOICES], dot = 0.0f;
#pragma unroll
            for (int j = 0; j < RT_MAX_CHOICES; j++) {
                e[j] = j < a.choices ? a.experts[row * a.choices + j] : -1;
                w[j] = j < a.choices ? a.weights[row * a.choices + j] / a.scale : 0.0f;
                g[j] = j < a.choices ? d_weights[row * a.choices + j] * a.scale : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < RT_MAX_CHOICES; j++) {
                if ((uint32_t)e[j] >= (uint32_t)a.count) e[j] = -1;
                if (e[j] >= 0) dot = fmaf(w[j], g[j], dot);
            }
            if (dense) {
                float top = -INFINITY, sum = 0.0f;
#pragma unroll 8
                for (int i = 0; i < a.count; i++) top = fmaxf(top, l[i]);
#pragma unroll 8
                for (int i = 0; i < a.count; i++) {
                    l[i] = l[i] == -INFINITY ? 0.0f : __expf(l[i] - top);   // as in the choice
                    sum += l[i];
                }
                const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
                float add[RT_MAX_CHOICES];
#pragma unroll
                for (int j = 0; j < RT_MAX_CHOICES; j++) add[j] = e[j] >= 0 ? l[e[j]] * over * (g[j] - dot) : 0.0f;
#pragma unroll 8
                for (int i = 0; i < a.count; i++) l[i] = l[i] * over * -dot;
#pragma unroll
                for (int j = 0; j < RT_MAX_CHOICES; j++)
                    if (e[j] >= 0) l[e[j]] = add[j];
            } else {
                float s[RT_MAX_CHOICES];
#pragma unroll
                for (int j = 0; j < RT_MAX_CHOICES; j++) s[j] = a.sigmoid && e[j] >= 0 ? tl_get(static_cast<const T*>(a.logits) + row * a.row + e[j]) : 0.0f;
#pragma unroll
                for (int j = 0; j < RT_MAX_CHOICES; j++) {
                    if (e[j] < 0) continue;
                    l[e[j]] = a.renormalize ? w[j] * (g[j] - dot) * (a.sigmoid ? re_sigmoid(-s[j]) : 1.0f) : g[j] * re_sigmoid(s[j]) * re_sigmoid(-s[j]);
                }
            }
        }
        __syncwarp();
        constexpr int N = 16 / (int)sizeof(T);
        if (wide_out) {
            const int per = a.count / N, rows = 32 / per, rest = 32 % per;   // 32 pieces on
            int r = lane / per, c = lane % per;
#pragma unroll 4
            for (int u = lane; u < 32 * per; u += 32) {
                if (row0 + r < a.n) {
                    uint4 v;
                    T* const out = reinterpret_cast<T*>(&v);
#pragma unroll
                    for (int i = 0; i < N; i++) tl_put(out + i, tile[r * pitch + c * N + i]);
                    *reinterpret_cast<uint4*>(d_logits + (row0 + r) * a.count + c * N) = v;
                }
                r += rows;
                c += rest;
                if (c >= per) { c -= per; r++; }
            }
        } else {
            for (int u = lane; u < 32 * a.count; u += 32) {
                const int r = u / a.count, c = u % a.count;
                if (row0 + r >= a.n) break;
                tl_put(d_logits + (row0 + r) * a.count + c, tile[r * pitch + c]);
            }
        }
    }
}

struct ReLayout { int64_t chunk, blocks, counts, sums, total; };
// Whether a thread takes a row.
static bool rt_takes(const ReArgs& a) { return a.count <= RT_MAX_EXPERTS && a.choices <= RT_MAX_CHOICES && a.groups <= RT_MAX_GROUPS; }
static ReLayout re_layout(const ReArgs& a)
{
    ReLayout l;
    const int64_t n = a.n;
    const int count = a.count;
    const int64_t most = (int64_t)sm_count_cached() * (rt_takes(a) ? 16 : 4), least = rt_takes(a) ? RT_WARPS * 32 : RE_WARPS;   // blocks
    l.chunk = std::max<int64_t>(least, ((n + most - 1) / most + least - 1) / least * least);
    l.blocks = std::max<int64_t>(1, (n + l.chunk - 1) / l.chunk);
    l.counts = 0;
    l.sums = align_up(4 * l.blocks * (count + 1), 256);
    l.total = l.sums + align_up(4 * (count + 1), 256);
    return l;
}

static int re_args(const dynb_routing* in, ReArgs* a)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("route_experts: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->experts < 1 || in->experts > DYNB_ROUTING_MAX_EXPERTS) return fail_arg("route_experts: experts must lie in [1, 1024]");
    if (in->choices < 1 || in->choices > DYNB_ROUTING_MAX_CHOICES || in->choices > in->experts)
        return fail_arg("route_experts: choices must lie in [1, 32] and be no more than the experts");
    if (in->n_rows < 0 || in->n_rows >= INT32_MAX || in->n_rows * in->choices >= INT32_MAX) return fail_arg("route_experts: rows times choices must lie in [0, 2^31 - 1)");
    if (in->groups < 1 || in->experts % in->groups != 0 || in->kept_groups < 1 || in->kept_groups > in->groups)
        return fail_arg("route_experts: groups must divide the experts, and kept_groups lie in [1, groups]");
    if (in->score != DYNB_SCORE_SOFTMAX && in->score != DYNB_SCORE_SIGMOID) return fail_arg("route_experts: score must be DYNB_SCORE_SOFTMAX or DYNB_SCORE_SIGMOID");
    if (!(in->scale >= 1e-30f && in->scale <= 1e30f)) return fail_arg("route_experts: scale must lie in [1e-30, 1e30]");
    *a = ReArgs{};
    a->logits = in->logits_dev; a->row = in->logits_row; a->bias = in->bias_dev; a->n = in->n_rows;
    a->count = in->experts; a->choices = in->choices; a->groups = in->groups; a->kept = in->kept_groups;
    a->sigmoid = in->score == DYNB_SCORE_SIGMOID; a->renormalize = in->renormalize != 0; a->scale = in->scale;
    return DYNB_OK;
}

// As few places in the list as the choices need: a longer one is entered more often (six choices of 64 experts, 200 k rows, with ten places 182 us, with eight 155).
template <typename T, int GROUPS>
static void (*rt_kernel(int choices))(ReArgs, int, int)
{
    if constexpr (GROUPS == 0)   // logits decide for good: nothing is looked at beside the choices
        return choices <= 1 ? rt_choose_kernel<T, 1, 0> : choices <= 2 ? rt_choose_kernel<T, 2, 0> : choices <= 4 ? rt_choose_kernel<T, 4, 0> :
               choices <= 6 ? rt_choose_kernel<T, 6, 0> : rt_choose_kernel<T, 8, 0>;
    else
        return choices <= 1 ? rt_choose_kernel<T, 3, GROUPS> : choices <= 2 ? rt_choose_kernel<T, 4, GROUPS> : choices <= 4 ? rt_choose_kernel<T, 6, GROUPS> :
               choices <= 6 ? rt_choose_kernel<T, 8, GROUPS> : rt_choose_kernel<T, 10, GROUPS>;
}

// Rows of `row` elements may be read, or written, by pieces of 16 bytes.
static bool re_wide(const void* p, int64_t row, int count, int size) { return starts_on(p, 16) && row * size % 16 == 0 && count * size % 16 == 0; }

// Bytes of shared memory.
static int rt_choose_shared(int count) { return (2 * count + 1 + RT_WARPS * 32 * (count | 1)) * 4; }
static int rt_backward_shared(int count) { return RT_WARPS * 32 * (count | 1) * 4; }
static int re_choose_shared(int count, int groups) { return ((count + 1) * 4 + 15) / 16 * 16 + (groups > 1 ? RE_WARPS * (count + groups) * 8 : 0); }

template <typename T>
static cudaError_t re_choose(const ReArgs& a, unsigned blocks, cudaStream_t s)
{
    if (rt_takes(a)) {
        const int pitch = a.count | 1, smem = rt_choose_shared(a.count);
        void (*const kernel)(ReArgs, int, int) = a.groups > 8 ? rt_kernel<T, 16>(a.choices) : a.groups > 1 ? rt_kernel<T, 8>(a.choices) :
                                                   a.bias != nullptr ? rt_kernel<T, 1>(a.choices) : rt_kernel<T, 0>(a.choices);
        const cudaError_t rc = allow_shared(reinterpret_cast<const void*>(kernel), rt_choose_shared(RT_MAX_EXPERTS));
        if (rc != cudaSuccess) return rc;
        kernel<<<blocks, RT_WARPS * 32, smem, s>>>(a, pitch, re_wide(a.logits, a.row, a.count, sizeof(T)));
        return cudaGetLastError();
    }
    const int smem = re_choose_shared(a.count, a.groups);
    void (*kernel)(ReArgs) = a.count <= 32 ? re_choose_kernel<T, 1> : a.count <= 64 ? re_choose_kernel<T, 2> : a.count <= 128 ? re_choose_kernel<T, 4> :
                             a.count <= 256 ? re_choose_kernel<T, 8> : a.count <= 512 ? re_choose_kernel<T, 16> : re_choose_kernel<T, 32>;
    const cudaError_t rc = allow_shared(reinterpret_cast<const void*>(kernel), re_choose_shared(DYNB_ROUTING_MAX_EXPERTS, DYNB_ROUTING_MAX_EXPERTS));
    if (rc != cudaSuccess) return rc;
    kernel<<<blocks, RE_WARPS * 32, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t re_backward(const ReArgs& a, const float* d_weights, void* d_logits, cudaStream_t s)
{
    if (rt_takes(a)) {
        const int pitch = a.count | 1, smem = rt_backward_shared(a.count);
        const cudaError_t rc = allow_shared(reinterpret_cast<const void*>(rt_backward_kernel<T>), rt_backward_shared(RT_MAX_EXPERTS));
        if (rc != cudaSuccess) return rc;
        const unsigned blocks = (unsigned)std::min<int64_t>((a.n + RT_WARPS * 32 - 1) / (RT_WARPS * 32), (int64_t)sm_count_cached() * 16);
        rt_backward_kernel<T><<<blocks, RT_WARPS * 32, smem, s>>>(a, d_weights, static_cast<T*>(d_logits), pitch, re_wide(a.logits, a.row, a.count, sizeof(T)),
                                                                  re_wide(d_logits, a.count, a.count, sizeof(T)));
        return cudaGetLastError();
    }
    void (*kernel)(ReArgs, const float*, T*) = a.count <= 32 ? re_backward_kernel<T, 1> : a.count <= 64 ? re_backward_kernel<T, 2> : a.count <= 128 ? re_backward_kernel<T, 4> :
                                               a.count <= 256 ? re_backward_kernel<T, 8> : a.count <= 512 ? re_backward_kernel<T, 16> : re_backward_kernel<T, 32>;
    const unsigned blocks = (unsigned)std::min<int64_t>((a.n + RE_WARPS - 1) / RE_WARPS, (int64_t)sm_count_cached() * 8);
    kernel<<<blocks, RE_WARPS * 32, 0, s>>>(a, d_weights, static_cast<T*>(d_logits));
    return cudaGetLastError();
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_route_experts_workspace_bytes(const dynb_routing* args, int64_t* bytes)
{
    ReArgs a;
    const int rc = re_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (bytes == nullptr) return fail_arg("null pointer");
    *bytes = re_layout(a).total;
    return DYNB_OK;
}

extern "C" int dynb_route_experts(const dynb_routing* args, int32_t* experts_dev, float* weights_dev, int32_t* order_dev, int32_t* start_dev,
                                  void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    ReArgs a;
    const int rc = re_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (!start_dev || !workspace_dev || (a.n > 0 && (!a.logits || !experts_dev || !weights_dev || !order_dev))) return fail_arg("null pointer");
    if (!starts_on(workspace_dev, 4)) return fail_arg("route_experts: the workspace must start on a 4-byte boundary");
    const ReLayout l = re_layout(a);
    if (workspace_bytes < l.total) return fail_arg("workspace too small");
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    a.experts = experts_dev; a.weights = weights_dev; a.order = order_dev; a.start = start_dev; a.chunk = l.chunk;
    a.counts = reinterpret_cast<int32_t*>(ws + l.counts);
    a.sums = reinterpret_cast<int32_t*>(ws + l.sums);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned blocks = (unsigned)l.blocks;
    if (args->dtype == DYNB_F32) DYNB_CUDA_OK(re_choose<float>(a, blocks, s));
    else if (args->dtype == DYNB_F16) DYNB_CUDA_OK(re_choose<__half>(a, blocks, s));
    else DYNB_CUDA_OK(re_choose<__nv_bfloat16>(a, blocks, s));
    DYNB_CUDA_OK(launch_chained(re_sums_kernel, a.count + 1, 256, 0, s, a.counts, a.sums, (int)blocks));
    DYNB_CUDA_OK(launch_chained(re_place_kernel, blocks, RE_WARPS * 32, (size_t)(a.count + 1) * 4 * (RE_WARPS + 1), s, a));
    return DYNB_OK;
}

extern "C" int dynb_route_experts_backward(const dynb_routing* args, const int32_t* experts_dev, const float* weights_dev, const float* d_weights_dev,
                                           void* d_logits_dev, void* stream)
{
    ReArgs a;
    const int rc = re_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (a.n == 0) return DYNB_OK;
    if (!a.logits || !experts_dev || !weights_dev || !d_weights_dev || !d_logits_dev) return fail_arg("null pointer");
    a.experts = const_cast<int32_t*>(experts_dev);
    a.weights = const_cast<float*>(weights_dev);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (args->dtype == DYNB_F32) DYNB_CUDA_OK(re_backward<float>(a, d_weights_dev, d_logits_dev, s));
    else if (args->dtype == DYNB_F16) DYNB_CUDA_OK(re_backward<__half>(a, d_weights_dev, d_logits_dev, s));
    else DYNB_CUDA_OK(re_backward<__nv_bfloat16>(a, d_weights_dev, d_logits_dev, s));
    return DYNB_OK;
}
