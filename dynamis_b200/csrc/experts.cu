// Rows times the matrices of their experts, and the weighted sums of the results (no counterpart in the reference, whose models leave it to
// their libraries).  Row i has the experts e_i1 ... e_ic (route_experts); pairs (i, j) are numbered i c + j, and `order` lists them by expert:
//     z_ij = act(x_i W[e_ij] + b[e_ij]),   y_i = r_i + sum_j w_ij z_ij.
//     back:  du = dz act'(u);  dx_i = sum_j du_ij W^T;  dW[e] = sum x^T du;  db[e] = sum du;   dz_ij = w_ij dy_i;  dw_ij = dy_i . z_ij.
// A place without an expert gives zeros and gets zero gradients.  Sums are in 32 bits, over pairs of an expert in stretches joined in their order: no atomics.

#include <algorithm>

#include "experts.cuh"

namespace dynb {

constexpr int EX_THREADS = 256;

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

// Workspace of the backward pass: the matrices as the kernel reads them, the gradients of x by pairs, the sums of stretches.
struct ExLayout { int64_t by_pair, partial, total; };
static ExLayout ex_layout(const ExArgs& e, int dtype, bool dx, bool weights)
{
    ExLayout l;
    l.by_pair = align_up(dx ? ex_packed_bytes(e, 1, dtype) : 0, 256);
    l.partial = l.by_pair + align_up(dx && e.fan > 1 ? e.t.n * e.t.inner * 4 : 0, 256);
    l.total = l.partial + align_up(weights ? ex_stretches(e) * ((int64_t)e.t.inner * e.t.outer + e.t.outer) * 4 : 0, 256);
    return l;
}

template <typename T>
static int ex_backward(ExArgs& e, int dtype, const int32_t* experts, void* d_x, unsigned char* ws, const ExLayout& l, cudaStream_t s)
{
    TlArgs& a = e.t;
    if (d_x != nullptr && a.n > 0) {
        a.dx = e.fan > 1 ? ws + l.by_pair : static_cast<unsigned char*>(d_x);
        DYNB_CUDA_OK(ex_mma_rows(e, 1, dtype, ws, s));
        if (e.fan > 1) {
            ex_combine_kernel<float, T><<<ex_grid(e.n_in * a.inner), EX_THREADS, 0, s>>>(reinterpret_cast<const float*>(ws + l.by_pair), nullptr, experts, static_cast<const T*>(nullptr), 0,
                                                                                     static_cast<T*>(d_x), e.n_in, e.fan, a.inner);
            DYNB_CUDA_OK(cudaGetLastError());
        }
    }
    if (a.dw != nullptr || a.db != nullptr) {
        DYNB_CUDA_OK(ex_mma_weights(e, dtype, s));
        const int64_t all = (int64_t)a.inner * a.outer + a.outer;
        ex_join_kernel<T><<<dim3((unsigned)std::min<int64_t>((all + EX_THREADS - 1) / EX_THREADS, 1024), a.types), EX_THREADS, 0, s>>>(a, ex_stretches(e));
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

extern "C" int dynb_expert_linear_workspace_bytes(const dynb_expert_linear_args* args, int backward, int want_x, int want_weights, int64_t* bytes)
{
    ExArgs e;
    const int rc = ex_args(args, &e);
    if (rc != DYNB_OK) return rc;
    if (bytes == nullptr) return fail_arg("null pointer");
    *bytes = backward ? ex_layout(e, args->dtype, want_x != 0, want_weights != 0).total : ex_packed_bytes(e, 0, args->dtype);
    return DYNB_OK;
}

extern "C" int dynb_expert_linear(const dynb_expert_linear_args* args, const void* x_dev, int64_t x_row, const void* bias_dev, void* z_dev, void* slope_dev,
                                  void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    ExArgs e;
    const int rc = ex_args(args, &e);
    if (rc != DYNB_OK) return rc;
    if (e.t.n == 0) return DYNB_OK;
    if (!x_dev || !z_dev) return fail_arg("null pointer");
    if (workspace_dev == nullptr || !starts_on(workspace_dev, 16) || workspace_bytes < ex_packed_bytes(e, 0, args->dtype)) return fail_arg("workspace too small");
    e.t.x = x_dev; e.t.x_row = x_row; e.t.b = bias_dev; e.t.y = z_dev;
    e.slope = e.activation != DYNB_ACTIVATION_NONE ? slope_dev : nullptr;
    DYNB_CUDA_OK(ex_mma_rows(e, 0, args->dtype, workspace_dev, static_cast<cudaStream_t>(stream)));
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
