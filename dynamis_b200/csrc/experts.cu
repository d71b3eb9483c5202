// Rows times the matrices of their experts, and the weighted sums of the results (no counterpart in the reference, whose models leave it to
// their libraries).  Row i has the experts e_i1 ... e_ic (route_experts); pairs (i, j) are numbered i c + j, and `order` lists them by expert:
//     z_ij = act(x_i W[e_ij] + b[e_ij]),   y_i = r_i + sum_j w_ij z_ij.
//     back:  du = dz act'(u);  dx_i = sum_j du_ij W^T;  dW[e] = sum x^T du;  db[e] = sum du;   dz_ij = w_ij dy_i;  dw_ij = dy_i . z_ij.
// A place without an expert gives zeros and gets zero gradients.  Sums are in 32 bits, over pairs of an expert in stretches joined in their order: no atomics.

#include <algorithm>

#include "experts.cuh"

namespace dynb {

constexpr int EX_M = 64, EX_N = 64, EX_K = 16, EX_THREADS = 256;

// Rows of places without an expert are set to zero; `wide` bytes a row.
__device__ __forceinline__ void ex_clear_absent(const TlArgs& a, void* out, int64_t wide)
{
    const int64_t from = min(max((int64_t)a.start[a.types], (int64_t)0), a.n);
    for (int64_t at = from + blockIdx.x; at < a.n; at += gridDim.x) {
        const int32_t p = a.order[at];
        if ((uint32_t)p >= (uint64_t)a.n) continue;
        uint16_t* const row = reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(out) + p * wide);
        for (int64_t i = threadIdx.x; i < wide / 2; i += blockDim.x) row[i] = 0;
    }
}

// One tile of 64 gathered pairs times 64 columns, to results of type O.  `back`: the gradient du W^T of the pair's row instead.
template <typename T, typename O>
__global__ void __launch_bounds__(EX_THREADS)
ex_rows_kernel(const ExArgs e, int back)
{
    const TlArgs& a = e.t;
    __shared__ float sa[EX_K][EX_M + 4], sb[EX_K][EX_N + 4];
    __shared__ int32_t pairs[EX_M];
    const int kk = back ? a.outer : a.inner, nn = back ? a.inner : a.outer;
    O* const out = static_cast<O*>(back ? a.dx : a.y);
    if (blockIdx.y == 0) ex_clear_absent(a, out, (int64_t)nn * sizeof(O));
    const TlTile tile = tl_tile(a, blockIdx.x, EX_M);
    if (tile.type < 0) return;
    const T* const in = static_cast<const T*>(back ? a.dy : a.x);
    const T* const w = static_cast<const T*>(a.w) + (int64_t)tile.type * a.inner * a.outer;
    const int64_t in_row = back ? a.dy_row : a.x_row;
    const int fan = back ? 1 : e.fan;
    if (threadIdx.x < EX_M) {
        int32_t p = -1;
        if (tile.begin + threadIdx.x < tile.end) {
            p = a.order[tile.begin + threadIdx.x];
            if ((uint32_t)p >= (uint64_t)a.n) p = -1;
        }
        pairs[threadIdx.x] = p;
    }
    __syncthreads();
    const int col0 = blockIdx.y * EX_N, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < kk; k0 += EX_K) {
#pragma unroll
        for (int i = threadIdx.x; i < EX_M * EX_K; i += EX_THREADS) {
            const int m = i / EX_K, k = i % EX_K;
            sa[k][m] = pairs[m] >= 0 && k0 + k < kk ? tl_get(in + (pairs[m] / fan) * in_row + k0 + k) : 0.0f;
        }
#pragma unroll
        for (int i = threadIdx.x; i < EX_N * EX_K; i += EX_THREADS) {
            const int k = back ? i % EX_K : i / EX_N, n = back ? i / EX_K : i % EX_N;
            const bool ok = k0 + k < kk && col0 + n < nn;
            sb[k][n] = ok ? tl_get(back ? w + (int64_t)(col0 + n) * a.outer + k0 + k : w + (int64_t)(k0 + k) * a.outer + col0 + n) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EX_K; k++) {
            float fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                fa[i] = sa[k][ty * 4 + i];
                fb[i] = sb[k][tx * 4 + i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int32_t p = pairs[ty * 4 + i];
        if (p < 0) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = col0 + tx * 4 + j;
            if (n >= nn) continue;
            float v = acc[i][j];
            if (!back) {
                if (a.b != nullptr) v += tl_get(static_cast<const T*>(a.b) + (int64_t)tile.type * a.outer + n);
                float slope;
                v = ex_activate(v, e.activation, &slope);
                if (e.slope != nullptr) {
                    if constexpr (sizeof(T) == 4) static_cast<float*>(e.slope)[(int64_t)p * nn + n] = slope;
                    else static_cast<uint16_t*>(e.slope)[(int64_t)p * nn + n] = ex_slope_bits(slope);
                }
            }
            tl_put(out + (int64_t)p * nn + n, v);
        }
    }
}

// du = dz times the slope.
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_slope_kernel(const T* dz, int64_t dz_row, const void* slope, T* du, int64_t n, int wide)
{
    const int64_t all = n * wide;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const float s = sizeof(T) == 4 ? static_cast<const float*>(slope)[i] : ex_slope_of(static_cast<const uint16_t*>(slope)[i]);
        tl_put(du + i, tl_get(dz + i / wide * dz_row + i % wide) * s);
    }
}

// 64 x 64 elements of an expert's gradient over a stretch of its pairs; blockIdx.y 0 also sums the offsets' gradient.
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_weights_kernel(const ExArgs e)
{
    const TlArgs& a = e.t;
    __shared__ float sx[EX_K][EX_M + 4], sy[EX_K][EX_N + 4];
    const TlTile tile = tl_tile(a, blockIdx.x, a.stretch);
    if (tile.type < 0) return;
    const int row0 = blockIdx.y * EX_M, col0 = blockIdx.z * EX_N, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {}, sum[4] = {};
    for (int64_t p0 = tile.begin; p0 < tile.end; p0 += EX_K) {
#pragma unroll
        for (int i = threadIdx.x; i < EX_M * EX_K; i += EX_THREADS) {
            const int k = i / EX_M, m = i % EX_M;
            int32_t p = p0 + k < tile.end ? a.order[p0 + k] : -1;
            if ((uint32_t)p >= (uint64_t)a.n) p = -1;
            sx[k][m] = p >= 0 && row0 + m < a.inner ? tl_get(static_cast<const T*>(a.x) + (p / e.fan) * a.x_row + row0 + m) : 0.0f;
            sy[k][m] = p >= 0 && col0 + m < a.outer ? tl_get(static_cast<const T*>(a.dy) + p * a.dy_row + col0 + m) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EX_K; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v = sy[k][tx * 4 + j];
                sum[j] += v;
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i][j] = fmaf(sx[k][ty * 4 + i], v, acc[i][j]);
            }
        __syncthreads();
    }
    const int64_t cells = (int64_t)a.inner * a.outer;
    float* const mine = a.partial + blockIdx.x * (cells + a.outer);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = col0 + tx * 4 + j;
        if (n >= a.outer) continue;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (row0 + ty * 4 + i < a.inner) mine[(int64_t)(row0 + ty * 4 + i) * a.outer + n] = acc[i][j];
        if (row0 == 0 && ty == 0) mine[cells + n] = sum[j];
    }
}

// y_i = r_i + sum_j w_ij z_ij (w null: ones).  Z: type of z.
template <typename Z, typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_combine_kernel(const Z* z, const float* weights, const int32_t* experts, const T* residual, int64_t residual_row, T* y, int64_t n, int choices, int wide)
{
    const int64_t all = n * wide;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / wide, c = i % wide;
        float v = residual != nullptr ? tl_get(residual + row * residual_row + c) : 0.0f;
        for (int j = 0; j < choices; j++) {
            const int64_t p = row * choices + j;
            if (experts[p] >= 0) v = fmaf(weights != nullptr ? weights[p] : 1.0f, tl_get(z + p * wide + c), v);
        }
        tl_put(y + i, v);
    }
}

// A warp a row: dz_ij = w_ij dy_i, dw_ij = dy_i . z_ij.
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_combine_backward_kernel(const T* z, const float* weights, const int32_t* experts, const T* d_y, int64_t d_y_row, T* d_z, float* d_weights, int64_t n,
                           int choices, int wide)
{
    const int lane = threadIdx.x % 32;
    for (int64_t row = (int64_t)blockIdx.x * (EX_THREADS / 32) + threadIdx.x / 32; row < n; row += (int64_t)gridDim.x * (EX_THREADS / 32)) {
        for (int j = 0; j < choices; j++) {
            const int64_t p = row * choices + j;
            const bool live = experts[p] >= 0;
            const float w = weights[p];
            float dot = 0.0f;
            for (int c = lane; c < wide; c += 32) {
                const float g = tl_get(d_y + row * d_y_row + c);
                if (live && d_weights != nullptr) dot = fmaf(g, tl_get(z + p * wide + c), dot);
                if (d_z != nullptr) tl_put(d_z + p * wide + c, live ? w * g : 0.0f);
            }
            if (d_weights == nullptr) continue;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (lane == 0) d_weights[p] = dot;
        }
    }
}

// The stretches of an expert joined: blockIdx.y is the expert.
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_join_kernel(const TlArgs a, int64_t stretches)
{
    const int type = blockIdx.y;
    __shared__ int64_t first_of, count_of;
    if (threadIdx.x < 32) {
        int64_t first = 0;
        for (int t = threadIdx.x; t < type; t += 32) {
            int64_t s0, s1;
            tl_rows_of(a, t, &s0, &s1);
            first += (s1 - s0 + a.stretch - 1) / a.stretch;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
        if (threadIdx.x == 0) {
            int64_t s0, s1;
            tl_rows_of(a, type, &s0, &s1);
            first_of = first;
            count_of = (s1 - s0 + a.stretch - 1) / a.stretch;
        }
    }
    __syncthreads();
    const int64_t cells = (int64_t)a.inner * a.outer, all = cells + a.outer, first = first_of;
    const int64_t count = min(count_of, max(stretches - first, (int64_t)0));
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        double exact = 0.0;
#pragma unroll 8
        for (int64_t c = 0; c < count; c++) exact += (double)a.partial[(first + c) * all + i];
        const float sum = (float)exact;
        if (i < cells) {
            if (a.dw != nullptr) tl_put(static_cast<T*>(a.dw) + type * cells + i, sum);
        } else if (a.db != nullptr) {
            tl_put(static_cast<T*>(a.db) + (int64_t)type * a.outer + (i - cells), sum);
        }
    }
}

static unsigned ex_grid(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + EX_THREADS - 1) / EX_THREADS, (int64_t)sm_count_cached() * 16)); }

static int ex_args(const dynb_expert_linear_args* in, ExArgs* e)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("expert_linear: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->choices < 1 || in->choices > DYNB_ROUTING_MAX_CHOICES) return fail_arg("expert_linear: choices must lie in [1, 32]");
    if (in->n_rows < 0 || in->n_rows * in->choices >= INT32_MAX) return fail_arg("expert_linear: rows times choices must lie in [0, 2^31 - 1)");
    if (in->experts < 1 || in->experts > DYNB_ROUTING_MAX_EXPERTS) return fail_arg("expert_linear: experts must lie in [1, 1024]");
    if (in->inner < 1 || in->outer < 1 || in->inner > DYNB_TYPE_LINEAR_MAX_WIDTH || in->outer > DYNB_TYPE_LINEAR_MAX_WIDTH)
        return fail_arg("expert_linear: widths must lie in [1, 16384]");
    if (in->activation < DYNB_ACTIVATION_NONE || in->activation > DYNB_ACTIVATION_GELU) return fail_arg("expert_linear: unknown activation");
    if (!in->start_dev || !in->weight_dev || (in->n_rows > 0 && !in->order_dev)) return fail_arg("null pointer");
    *e = ExArgs{};
    TlArgs& a = e->t;
    a.w = in->weight_dev;
    a.order = in->order_dev;
    a.start = in->start_dev;
    a.n = in->n_rows * in->choices;
    a.types = in->experts;
    a.inner = in->inner;
    a.outer = in->outer;
    a.stretch = tl_stretch(a.n, in->inner, in->outer, in->dtype);
    a.status = in->status_dev;
    e->n_in = in->paired ? a.n : in->n_rows;
    e->fan = in->paired ? 1 : in->choices;
    e->activation = in->activation;
    return DYNB_OK;
}

// Workspace of the backward pass: du, the gradients of x by pairs, the sums of stretches.
struct ExLayout { int64_t du, by_pair, partial, total; };
static ExLayout ex_layout(const ExArgs& e, int dtype, bool dx, bool weights)
{
    const int size = dtype == DYNB_F32 ? 4 : 2;
    ExLayout l;
    l.du = 0;
    l.by_pair = align_up(e.activation != DYNB_ACTIVATION_NONE ? e.t.n * e.t.outer * size : 0, 256);
    l.partial = l.by_pair + align_up(dx && e.fan > 1 ? e.t.n * e.t.inner * 4 : 0, 256);
    l.total = l.partial + align_up(weights ? tl_stretches(e.t.n, e.t.types, e.t.stretch) * ((int64_t)e.t.inner * e.t.outer + e.t.outer) * 4 : 0, 256);
    return l;
}

template <typename T>
static cudaError_t ex_rows(const ExArgs& e, int back, cudaStream_t s)
{
    const int nn = back ? e.t.inner : e.t.outer;
    const dim3 grid((unsigned)((e.t.n + EX_M - 1) / EX_M + e.t.types), (nn + EX_N - 1) / EX_N);
    if (back && e.fan > 1) ex_rows_kernel<T, float><<<grid, EX_THREADS, 0, s>>>(e, back);   // summed over the choices before they are rounded
    else ex_rows_kernel<T, T><<<grid, EX_THREADS, 0, s>>>(e, back);
    return cudaGetLastError();
}

template <typename T>
static int ex_backward(ExArgs& e, int dtype, const int32_t* experts, void* d_x, unsigned char* ws, const ExLayout& l, cudaStream_t s)
{
    TlArgs& a = e.t;
    if (a.n > 0 && e.activation != DYNB_ACTIVATION_NONE) {
        T* const du = reinterpret_cast<T*>(ws + l.du);
        ex_slope_kernel<T><<<ex_grid(a.n * a.outer), EX_THREADS, 0, s>>>(static_cast<const T*>(a.dy), a.dy_row, e.slope, du, a.n, a.outer);
        DYNB_CUDA_OK(cudaGetLastError());
        a.dy = du;
        a.dy_row = a.outer;
    }
    if (d_x != nullptr && a.n > 0) {
        a.dx = e.fan > 1 ? ws + l.by_pair : static_cast<unsigned char*>(d_x);
        DYNB_CUDA_OK(ex_rows<T>(e, 1, s));
        if (e.fan > 1) {
            ex_combine_kernel<float, T><<<ex_grid(e.n_in * a.inner), EX_THREADS, 0, s>>>(reinterpret_cast<const float*>(ws + l.by_pair), nullptr, experts, static_cast<const T*>(nullptr), 0,
                                                                                 static_cast<T*>(d_x), e.n_in, e.fan, a.inner);
            DYNB_CUDA_OK(cudaGetLastError());
        }
    }
    if (a.dw != nullptr || a.db != nullptr) {
        const dim3 grid((unsigned)tl_stretches(a.n, a.types, a.stretch), (a.inner + EX_M - 1) / EX_M, (a.outer + EX_N - 1) / EX_N);
        ex_weights_kernel<T><<<grid, EX_THREADS, 0, s>>>(e);
        DYNB_CUDA_OK(cudaGetLastError());
        const int64_t all = (int64_t)a.inner * a.outer + a.outer;
        ex_join_kernel<T><<<dim3((unsigned)std::min<int64_t>((all + EX_THREADS - 1) / EX_THREADS, 1024), a.types), EX_THREADS, 0, s>>>(a, grid.x);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    return DYNB_OK;
}

static int ec_check(int64_t n_rows, int choices, int wide, int dtype)
{
    if (dtype != DYNB_F32 && dtype != DYNB_F16 && dtype != DYNB_BF16) return fail_arg("expert_combine: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (choices < 1 || choices > DYNB_ROUTING_MAX_CHOICES) return fail_arg("expert_combine: choices must lie in [1, 32]");
    if (n_rows < 0 || n_rows * choices >= INT32_MAX) return fail_arg("expert_combine: rows times choices must lie in [0, 2^31 - 1)");
    if (wide < 1 || wide > DYNB_TYPE_LINEAR_MAX_WIDTH) return fail_arg("expert_combine: the width must lie in [1, 16384]");
    return DYNB_OK;
}

template <typename T>
static cudaError_t ec_forward(const void* z, const float* weights, const int32_t* experts, const void* residual, int64_t residual_row, void* y, int64_t n, int choices,
                              int wide, cudaStream_t s)
{
    ex_combine_kernel<T, T><<<ex_grid(n * wide), EX_THREADS, 0, s>>>(static_cast<const T*>(z), weights, experts, static_cast<const T*>(residual), residual_row, static_cast<T*>(y), n,
                                                                  choices, wide);
    return cudaGetLastError();
}
template <typename T>
static cudaError_t ec_backward(const void* z, const float* weights, const int32_t* experts, const void* d_y, int64_t d_y_row, void* d_z, float* d_weights, int64_t n,
                               int choices, int wide, cudaStream_t s)
{
    ex_combine_backward_kernel<T><<<ex_grid(n * 32), EX_THREADS, 0, s>>>(static_cast<const T*>(z), weights, experts, static_cast<const T*>(d_y), d_y_row, static_cast<T*>(d_z), d_weights,
                                                                       n, choices, wide);
    return cudaGetLastError();
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_expert_linear(const dynb_expert_linear_args* args, const void* x_dev, int64_t x_row, const void* bias_dev, void* z_dev, void* slope_dev,
                                  void* stream)
{
    ExArgs e;
    const int rc = ex_args(args, &e);
    if (rc != DYNB_OK) return rc;
    if (e.t.n == 0) return DYNB_OK;
    if (!x_dev || !z_dev) return fail_arg("null pointer");
    e.t.x = x_dev; e.t.x_row = x_row; e.t.b = bias_dev; e.t.y = z_dev;
    e.slope = e.activation != DYNB_ACTIVATION_NONE ? slope_dev : nullptr;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (args->dtype == DYNB_F32) DYNB_CUDA_OK(ex_rows<float>(e, 0, s));
    else if (args->dtype == DYNB_F16) DYNB_CUDA_OK(ex_rows<__half>(e, 0, s));
    else DYNB_CUDA_OK(ex_rows<__nv_bfloat16>(e, 0, s));
    return DYNB_OK;
}

extern "C" int dynb_expert_linear_workspace_bytes(const dynb_expert_linear_args* args, int want_x, int want_weights, int64_t* bytes)
{
    ExArgs e;
    const int rc = ex_args(args, &e);
    if (rc != DYNB_OK) return rc;
    if (bytes == nullptr) return fail_arg("null pointer");
    *bytes = ex_layout(e, args->dtype, want_x != 0, want_weights != 0).total;
    return DYNB_OK;
}

extern "C" int dynb_expert_linear_backward(const dynb_expert_linear_args* args, const void* x_dev, int64_t x_row, const void* d_z_dev, int64_t d_z_row,
                                           const void* slope_dev, const int32_t* experts_dev, void* d_x_dev, void* d_weight_dev, void* d_bias_dev,
                                           void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    ExArgs e;
    const int rc = ex_args(args, &e);
    if (rc != DYNB_OK) return rc;
    const bool weights = d_weight_dev != nullptr || d_bias_dev != nullptr;
    if (!weights && (d_x_dev == nullptr || e.t.n == 0)) return DYNB_OK;
    if (e.t.n > 0 && (!x_dev || !d_z_dev || !experts_dev)) return fail_arg("null pointer");
    if (e.t.n > 0 && e.activation != DYNB_ACTIVATION_NONE && !slope_dev) return fail_arg("null pointer");
    const ExLayout l = ex_layout(e, args->dtype, d_x_dev != nullptr, weights);
    if (l.total > 0 && (workspace_dev == nullptr || !starts_on(workspace_dev, 16) || workspace_bytes < l.total)) return fail_arg("workspace too small");
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    e.t.x = x_dev; e.t.x_row = x_row; e.t.dy = d_z_dev; e.t.dy_row = d_z_row; e.t.dw = d_weight_dev; e.t.db = d_bias_dev;
    e.t.partial = reinterpret_cast<float*>(ws + l.partial);
    e.slope = const_cast<void*>(slope_dev);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (args->dtype == DYNB_F32) return ex_backward<float>(e, args->dtype, experts_dev, d_x_dev, ws, l, s);
    if (args->dtype == DYNB_F16) return ex_backward<__half>(e, args->dtype, experts_dev, d_x_dev, ws, l, s);
    return ex_backward<__nv_bfloat16>(e, args->dtype, experts_dev, d_x_dev, ws, l, s);
}

extern "C" int dynb_expert_combine(const void* z_dev, const float* weights_dev, const int32_t* experts_dev, const void* residual_dev, int64_t residual_row,
                                   int64_t n_rows, int choices, int width, int dtype, void* y_dev, void* stream)
{
    const int rc = ec_check(n_rows, choices, width, dtype);
    if (rc != DYNB_OK) return rc;
    if (n_rows == 0) return DYNB_OK;
    if (!z_dev || !weights_dev || !experts_dev || !y_dev) return fail_arg("null pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == DYNB_F32) DYNB_CUDA_OK(ec_forward<float>(z_dev, weights_dev, experts_dev, residual_dev, residual_row, y_dev, n_rows, choices, width, s));
    else if (dtype == DYNB_F16) DYNB_CUDA_OK(ec_forward<__half>(z_dev, weights_dev, experts_dev, residual_dev, residual_row, y_dev, n_rows, choices, width, s));
    else DYNB_CUDA_OK(ec_forward<__nv_bfloat16>(z_dev, weights_dev, experts_dev, residual_dev, residual_row, y_dev, n_rows, choices, width, s));
    return DYNB_OK;
}

extern "C" int dynb_expert_combine_backward(const void* z_dev, const float* weights_dev, const int32_t* experts_dev, const void* d_y_dev, int64_t d_y_row,
                                            int64_t n_rows, int choices, int width, int dtype, void* d_z_dev, float* d_weights_dev, void* stream)
{
    const int rc = ec_check(n_rows, choices, width, dtype);
    if (rc != DYNB_OK) return rc;
    if (n_rows == 0 || (d_z_dev == nullptr && d_weights_dev == nullptr)) return DYNB_OK;
    if (!z_dev || !weights_dev || !experts_dev || !d_y_dev) return fail_arg("null pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == DYNB_F32) DYNB_CUDA_OK(ec_backward<float>(z_dev, weights_dev, experts_dev, d_y_dev, d_y_row, d_z_dev, d_weights_dev, n_rows, choices, width, s));
    else if (dtype == DYNB_F16) DYNB_CUDA_OK(ec_backward<__half>(z_dev, weights_dev, experts_dev, d_y_dev, d_y_row, d_z_dev, d_weights_dev, n_rows, choices, width, s));
    else DYNB_CUDA_OK(ec_backward<__nv_bfloat16>(z_dev, weights_dev, experts_dev, d_y_dev, d_y_row, d_z_dev, d_weights_dev, n_rows, choices, width, s));
    return DYNB_OK;
}
