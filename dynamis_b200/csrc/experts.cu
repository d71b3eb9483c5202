// Rows times the matrices of their experts, and the weighted sums of the results (no counterpart in the reference, whose models leave it to
// their libraries).  Row i has the experts e_i1 ... e_ic (route_experts); pairs (i, j) are numbered i c + j, and `order` lists them by expert:
//     z_ij = act(x_i W[e_ij] + b[e_ij]),   y_i = r_i + sum_j w_ij z_ij.
//     back:  du = dz act'(u);  dx_i = sum_j du_ij W^T;  dW[e] = sum x^T du;  db[e] = sum du;   dz_ij = w_ij dy_i;  dw_ij = dy_i . z_ij.
// A place without an expert gives zeros and gets zero gradients.  Sums are in 32 bits, over pairs of an expert in pieces joined in their order: no atomics.
//
// The weighted sums are bound by memory: 300 k rows of 4 x 256 bf16 with a residual 179 us (5.2 TB/s), gradients 285 us (4.9 TB/s); with an element a thread 471 and 496.

#include <algorithm>

#include "experts.cuh"

namespace dynb {

constexpr int EX_THREADS = 256;

template <typename T, int N> struct __align__(sizeof(T) * N) ExPack { T v[N]; };

// y_i = r_i + sum_j w_ij z_ij (w null: ones).  Z: type of z.  `lanes` threads (a power of two) a row, K pieces of N elements each at a time, four choices under way.
// Blocks an SM: four, for which 64 registers are enough but for 56 spilled bytes at most; 32-bit z by whole pieces six, with 8 to 36 spilled bytes (sums of 150 k rows of 2 x 256 back: 67
// us, with five blocks and no spills 75; of 4 x 256 forward 167 and 149).  Six for narrow 32-bit pieces spilled 448 bytes: 150 k rows of 4 x 102 121 us and now 80, of 4 x 101 176 and 113.
template <typename Z, typename T, int N, int K>
__global__ void __launch_bounds__(EX_THREADS, sizeof(Z) == 4 && K == 1 ? 6 : 4)
ex_combine_kernel(const Z* z, const float* weights, const int32_t* experts, const T* residual, int64_t residual_row, T* y, int64_t n, int choices, int wide, int lanes)
{
    const int in_row = threadIdx.x & (lanes - 1), rows = EX_THREADS / lanes, apart = lanes * N;
    for (int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x / lanes; row < n; row += (int64_t)gridDim.x * rows) {
        const int32_t* const es = experts + row * choices;
        for (int c = in_row * N; c < wide; c += K * apart) {
            float sum[K][N];
#pragma unroll
            for (int k = 0; k < K; k++) {
                ExPack<T, N> r = {};
                if (residual != nullptr && (K == 1 || c + k * apart < wide)) r = *reinterpret_cast<const ExPack<T, N>*>(residual + row * residual_row + c + k * apart);
#pragma unroll
                for (int i = 0; i < N; i++) sum[k][i] = residual != nullptr ? tl_get(&r.v[i]) : 0.0f;
            }
            const Z* at = z + row * choices * wide + c;
            for (int j0 = 0; j0 < choices; j0 += 4, at += (int64_t)4 * wide) {
                ExPack<Z, N> v[4][K];
                float w[4];
                bool live[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const bool here = j0 + j < choices;
                    live[j] = here && es[j0 + j] >= 0;
                    w[j] = here && weights != nullptr ? weights[row * choices + j0 + j] : 1.0f;
#pragma unroll
                    for (int k = 0; k < K; k++)   // also where there is no expert: it does not wait to be told
                        if (here && (K == 1 || c + k * apart < wide)) v[j][k] = *reinterpret_cast<const ExPack<Z, N>*>(at + (int64_t)j * wide + k * apart);
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (live[j]) {
#pragma unroll
                        for (int k = 0; k < K; k++)
#pragma unroll
                            for (int i = 0; i < N; i++) sum[k][i] = fmaf(w[j], tl_get(&v[j][k].v[i]), sum[k][i]);
                    }
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (K > 1 && c + k * apart >= wide) continue;
                ExPack<T, N> out;
#pragma unroll
                for (int i = 0; i < N; i++) tl_put(&out.v[i], sum[k][i]);
                *reinterpret_cast<ExPack<T, N>*>(y + row * wide + c + k * apart) = out;
            }
        }
    }
}

// dz_ij = w_ij dy_i, dw_ij = dy_i . z_ij: `lanes` lanes of a warp (a power of two) a row, N elements each, four choices at a time.
template <typename T, int N>
__global__ void __launch_bounds__(EX_THREADS)
ex_combine_backward_kernel(const T* z, const float* weights, const int32_t* experts, const T* d_y, int64_t d_y_row, T* d_z, float* d_weights, int64_t n,
                           int choices, int wide, int lanes)
{
    const int in_row = threadIdx.x & (lanes - 1), rows = EX_THREADS / lanes;
    const int64_t step = (int64_t)gridDim.x * rows, rounds = (n + step - 1) / step;
    int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x / lanes;
    for (int64_t round = 0; round < rounds; round++, row += step) {   // all lanes of a warp go as often
        const bool here = row < n;
        for (int j0 = 0; j0 < choices; j0 += 4) {
            float w[4], dot[4] = {};
            bool real[4], live[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                real[j] = here && j0 + j < choices;
                live[j] = real[j] && experts[row * choices + j0 + j] >= 0;
                w[j] = real[j] ? weights[row * choices + j0 + j] : 0.0f;
            }
            if (here) {
                const int64_t from = (row * choices + j0) * wide;
                for (int c = in_row * N; c < wide; c += lanes * N) {
                    const ExPack<T, N> g = *reinterpret_cast<const ExPack<T, N>*>(d_y + row * d_y_row + c);
                    ExPack<T, N> v[4];
                    if (d_weights != nullptr) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (real[j]) v[j] = *reinterpret_cast<const ExPack<T, N>*>(z + from + (int64_t)j * wide + c);
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (live[j]) {
#pragma unroll
                                for (int i = 0; i < N; i++) dot[j] = fmaf(tl_get(&g.v[i]), tl_get(&v[j].v[i]), dot[j]);
                            }
                    }
                    if (d_z != nullptr) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (real[j]) {
                                ExPack<T, N> out;
#pragma unroll
                                for (int i = 0; i < N; i++) tl_put(&out.v[i], live[j] ? w[j] * tl_get(&g.v[i]) : 0.0f);
                                *reinterpret_cast<ExPack<T, N>*>(d_z + from + (int64_t)j * wide + c) = out;
                            }
                    }
                }
            }
            if (d_weights == nullptr) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                for (int o = 1; o < lanes; o <<= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
                if (in_row == 0 && real[j]) d_weights[row * choices + j0 + j] = live[j] ? dot[j] : 0.0f;
            }
        }
    }
}

__host__ __device__ constexpr int ex_whole(int wide) { return (wide + 7) / 8 * 8; }

// Rows (times their slopes, or as they are where there are none) to rows of `out_row` elements, zeros behind `wide`: a warp a row.  For gradients of the matrices alone, where no
// pass of dx leaves du, and for rows that the products cannot read or store by whole pieces (120 k pairs of 129 x 131 bf16 with SiLU, forward, dx and dW: 354, 298 and 87 us by single
// elements; 48, 45 and 49 on copies, and 24 a copy).
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_copy_kernel(const T* in, int64_t in_row, const void* slope, T* out, int64_t n, int wide, int out_row)
{
    const int slope_row = ex_whole(wide);
    for (int64_t p = (int64_t)blockIdx.x * (EX_THREADS / 32) + threadIdx.x / 32; p < n; p += (int64_t)gridDim.x * (EX_THREADS / 32))
#pragma unroll 4
        for (int c = threadIdx.x % 32; c < out_row; c += 32) {
            float v = c < wide ? tl_get(in + p * in_row + c) : 0.0f;
            if (slope != nullptr && c < wide) v *= sizeof(T) == 4 ? static_cast<const float*>(slope)[p * slope_row + c] : ex_slopes_of(static_cast<const uint16_t*>(slope)[p * slope_row + c]).x;
            tl_put(out + p * out_row + c, v);
        }
}

// The sums of an expert joined (its pairs are cut at multiples of the stretch): blockIdx.y is the expert.
template <typename T>
__global__ void __launch_bounds__(EX_THREADS)
ex_join_kernel(const TlArgs a, int64_t stretches, int quads)   // quads: sums are read by 16 bytes
{
    const int type = blockIdx.y;
    __shared__ int64_t first_of, count_of;
    if (threadIdx.x < 32) {
        int64_t first = 0;
        for (int t = threadIdx.x; t < type; t += 32) {
            int64_t s0, s1;
            tl_rows_of(a, t, &s0, &s1);
            first += s1 > s0 ? (s1 + a.stretch - 1) / a.stretch - s0 / a.stretch : 0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
        if (threadIdx.x == 0) {
            int64_t s0, s1;
            tl_rows_of(a, type, &s0, &s1);
            first_of = first;
            count_of = s1 > s0 ? (s1 + a.stretch - 1) / a.stretch - s0 / a.stretch : 0;
        }
    }
    __syncthreads();
    const int64_t cells = (int64_t)a.inner * a.outer, all = cells + a.outer, first = first_of;
    const int64_t count = min(count_of, max(stretches - first, (int64_t)0));
    const auto put = [&](int64_t i, double v) {
        if (i < cells) {
            if (a.dw != nullptr) tl_put(static_cast<T*>(a.dw) + type * cells + i, (float)v);
        } else if (a.db != nullptr) {
            tl_put(static_cast<T*>(a.db) + (int64_t)type * a.outer + (i - cells), (float)v);
        }
    };
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    if (quads) {
        for (int64_t i = 4 * at; i < all; i += 4 * step) {
            double v[4] = {};
#pragma unroll 4
            for (int64_t c = 0; c < count; c++) {
                const float4 f = *reinterpret_cast<const float4*>(a.partial + (first + c) * all + i);
                v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) put(i + j, v[j]);
        }
        return;
    }
    for (int64_t i = at; i < all; i += step) {
        double v = 0.0;
#pragma unroll 8
        for (int64_t c = 0; c < count; c++) v += (double)a.partial[(first + c) * all + i];
        put(i, v);
    }
}

static unsigned ex_grid(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + EX_THREADS - 1) / EX_THREADS, (int64_t)sm_count_cached() * 16)); }

static int ex_args(const dynb_expert_linear_args* in, ExArgs* e)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("expert_linear: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->choices < 1 || in->choices > DYNB_ROUTING_MAX_CHOICES) return fail_arg("expert_linear: choices must lie in [1, 32]");
    if (in->n_rows < 0 || in->n_rows >= INT32_MAX || in->n_rows * in->choices >= INT32_MAX) return fail_arg("expert_linear: rows times choices must lie in [0, 2^31 - 1)");
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
    a.stretch = ex_stretch(a.n, in->inner, in->outer, in->dtype);
    a.status = in->status_dev;
    e->n_in = in->paired ? a.n : in->n_rows;
    e->fan = in->paired ? 1 : in->choices;
    e->activation = in->activation;
    return DYNB_OK;
}

// Pieces of `bytes` may be read and written at p and everywhere `row` elements on.
static bool ex_on(const void* p, int64_t row, int size, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && row * size % bytes == 0; }
// Threads of a row whose pieces are `pieces`, at most `most`.
static int ex_lanes(int pieces, int most)
{
    int lanes = 1;
    while (lanes < pieces && lanes < most) lanes *= 2;
    return lanes;
}

template <typename Z, typename T>
static cudaError_t ex_combine(const Z* z, const float* weights, const int32_t* experts, const T* residual, int64_t residual_row, T* y, int64_t n, int choices, int wide, cudaStream_t s)
{
    // the widest pieces that all addresses allow; narrow ones several at a time (150 k rows of 4 x 100 fp16 by single elements 178 us, of 4 x 256 by whole pieces 75)
    constexpr int MOST = 16 / (int)sizeof(Z);
    int piece = MOST;
    while (piece > 1 && !(wide % piece == 0 && ex_on(z, 0, 1, sizeof(Z) * piece) && ex_on(y, 0, 1, sizeof(T) * piece) && (residual == nullptr || ex_on(residual, residual_row, sizeof(T), sizeof(T) * piece))))
        piece /= 2;
    const auto start = [&](auto kernel, int at_once) {
        const int lanes = ex_lanes((wide / piece + at_once - 1) / at_once, EX_THREADS);
        kernel<<<ex_grid(n * lanes), EX_THREADS, 0, s>>>(z, weights, experts, residual, residual_row, y, n, choices, wide, lanes);
    };
    if (piece == MOST) {
        start(ex_combine_kernel<Z, T, MOST, 1>, 1);
        return cudaGetLastError();
    }
    if constexpr (MOST > 4) {
        if (piece == 4) {
            start(ex_combine_kernel<Z, T, 4, 2>, 2);
            return cudaGetLastError();
        }
    }
    if (piece == 2) start(ex_combine_kernel<Z, T, 2, 4>, 4);
    else start(ex_combine_kernel<Z, T, 1, 4>, 4);
    return cudaGetLastError();
}

// Whether rows are copied before the products read them: they do so by pieces of 8 elements on 16 bytes.
static bool ex_copies(const void* p, int64_t row, int wide, int size) { return wide % 8 != 0 || !ex_on(p, row, size, 16); }

template <typename T>
static cudaError_t ex_copy(const void* in, int64_t in_row, const void* slope, void* out, int64_t n, int wide, int out_row, cudaStream_t s)
{
    ex_copy_kernel<T><<<ex_grid(n * 32), EX_THREADS, 0, s>>>(static_cast<const T*>(in), in_row, slope, static_cast<T*>(out), n, wide, out_row);
    return cudaGetLastError();
}

// Workspaces: the matrices as the kernel reads them, rows of x that were copied, and of results that will be; backward also du, or copies of its rows, the gradients of x by pairs, the sums of pieces.
struct ExLayout { int64_t x, out, du, by_pair, partial, total; };
static ExLayout ex_layout(const ExArgs& e, int dtype, bool back, bool dx, bool weights, bool copy_x, bool copy_dy)
{
    const int size = dtype == DYNB_F32 ? 4 : 2;
    ExLayout l;
    l.x = align_up(!back || dx ? ex_packed_bytes(e, back, dtype) : 0, 256);
    l.out = l.x + align_up(copy_x && (!back || weights) ? e.n_in * ex_whole(e.t.inner) * size : 0, 256);
    l.du = l.out + align_up(!back && e.t.outer % 8 != 0 ? e.t.n * ex_whole(e.t.outer) * size : back && dx && e.t.inner % 8 != 0 ? e.n_in * ex_whole(e.t.inner) * size : 0, 256);
    l.by_pair = l.du + align_up(!back ? 0 : copy_dy ? e.t.n * ex_whole(e.t.outer) * size : weights && e.activation != DYNB_ACTIVATION_NONE ? e.t.n * e.t.outer * size : 0, 256);
    l.partial = l.by_pair + align_up(back && dx && e.fan > 1 ? e.t.n * ex_whole(e.t.inner) * 4 : 0, 256);
    l.total = l.partial + align_up(back && weights ? ex_stretches(e) * ((int64_t)e.t.inner * e.t.outer + e.t.outer) * 4 : 0, 256);
    return l;
}

template <typename T>
static int ex_forward(ExArgs& e, int dtype, unsigned char* ws, const ExLayout& l, bool copy_x, cudaStream_t s)
{
    TlArgs& a = e.t;
    if (copy_x) {
        DYNB_CUDA_OK(ex_copy<T>(a.x, a.x_row, nullptr, ws + l.x, e.n_in, a.inner, ex_whole(a.inner), s));
        a.x = ws + l.x;
        a.x_row = ex_whole(a.inner);
    }
    void* const z = a.y;
    e.out_row = ex_whole(a.outer);
    if (a.outer % 8 != 0) a.y = ws + l.out;   // whole pieces are stored; single elements by the copy alone
    DYNB_CUDA_OK(ex_mma_rows(e, 0, dtype, ws, s));
    if (a.outer % 8 != 0) DYNB_CUDA_OK(ex_copy<T>(a.y, e.out_row, nullptr, z, a.n, a.outer, a.outer, s));
    return DYNB_OK;
}

template <typename T>
static int ex_backward(ExArgs& e, int dtype, const int32_t* experts, void* d_x, unsigned char* ws, const ExLayout& l, bool copy_x, bool copy_dy, cudaStream_t s)
{
    TlArgs& a = e.t;
    const bool weights = a.dw != nullptr || a.db != nullptr, active = e.activation != DYNB_ACTIVATION_NONE;
    if (a.n > 0) {
        if (copy_dy) {   // times the slopes
            DYNB_CUDA_OK(ex_copy<T>(a.dy, a.dy_row, active ? e.slope : nullptr, ws + l.du, a.n, a.outer, ex_whole(a.outer), s));
            a.dy = ws + l.du;
            a.dy_row = ex_whole(a.outer);
            e.slope = nullptr;
        } else if (weights && active) {
            e.du = ws + l.du;
        }
        if (d_x != nullptr) {
            const bool copy = a.inner % 8 != 0;   // as forward
            void* const sums = copy ? ws + l.out : d_x;
            e.out_row = ex_whole(a.inner);
            a.dx = e.fan > 1 ? ws + l.by_pair : static_cast<unsigned char*>(sums);
            DYNB_CUDA_OK(ex_mma_rows(e, 1, dtype, ws, s));
            if (e.fan > 1) DYNB_CUDA_OK((ex_combine<float, T>(static_cast<const float*>(a.dx), nullptr, experts, nullptr, 0, static_cast<T*>(sums), e.n_in, e.fan, ex_whole(a.inner), s)));
            if (copy) DYNB_CUDA_OK(ex_copy<T>(sums, e.out_row, nullptr, d_x, e.n_in, a.inner, a.inner, s));
        } else if (e.du != nullptr) {
            DYNB_CUDA_OK(ex_copy<T>(a.dy, a.dy_row, e.slope, e.du, a.n, a.outer, a.outer, s));
        }
    }
    if (weights) {
        if (e.du != nullptr) { a.dy = e.du; a.dy_row = a.outer; }
        if (copy_x && a.n > 0) {
            DYNB_CUDA_OK(ex_copy<T>(a.x, a.x_row, nullptr, ws + l.x, e.n_in, a.inner, ex_whole(a.inner), s));
            a.x = ws + l.x;
            a.x_row = ex_whole(a.inner);
        }
        DYNB_CUDA_OK(ex_mma_weights(e, dtype, s));
        const int64_t all = (int64_t)a.inner * a.outer + a.outer;
        // enough blocks for all SMs, and no more: finding an expert's sums takes a block longer than adding a few (64 experts of 256 x 512: 129 blocks each 33 us, 37 blocks 22)
        const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((all + 4 * EX_THREADS - 1) / (4 * EX_THREADS), (int64_t)sm_count_cached() * 16 / a.types));
        ex_join_kernel<T><<<dim3(blocks, a.types), EX_THREADS, 0, s>>>(a, ex_stretches(e), all % 4 == 0);
        DYNB_CUDA_OK(cudaGetLastError());
    }
    return DYNB_OK;
}

static int ec_check(int64_t n_rows, int choices, int wide, int dtype)
{
    if (dtype != DYNB_F32 && dtype != DYNB_F16 && dtype != DYNB_BF16) return fail_arg("expert_combine: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (choices < 1 || choices > DYNB_ROUTING_MAX_CHOICES) return fail_arg("expert_combine: choices must lie in [1, 32]");
    if (n_rows < 0 || n_rows >= INT32_MAX || n_rows * choices >= INT32_MAX) return fail_arg("expert_combine: rows times choices must lie in [0, 2^31 - 1)");
    if (wide < 1 || wide > DYNB_TYPE_LINEAR_MAX_WIDTH) return fail_arg("expert_combine: the width must lie in [1, 16384]");
    return DYNB_OK;
}

template <typename T>
static cudaError_t ec_forward(const void* z, const float* weights, const int32_t* experts, const void* residual, int64_t residual_row, void* y, int64_t n, int choices,
                              int wide, cudaStream_t s)
{
    return ex_combine<T, T>(static_cast<const T*>(z), weights, experts, static_cast<const T*>(residual), residual_row, static_cast<T*>(y), n, choices, wide, s);
}
template <typename T>
static cudaError_t ec_backward(const void* z, const float* weights, const int32_t* experts, const void* d_y, int64_t d_y_row, void* d_z, float* d_weights, int64_t n,
                               int choices, int wide, cudaStream_t s)
{
    constexpr int MOST = 16 / (int)sizeof(T);
    int piece = MOST;
    while (piece > 1 && !(wide % piece == 0 && ex_on(z, 0, sizeof(T), sizeof(T) * piece) && ex_on(d_z, 0, sizeof(T), sizeof(T) * piece) && ex_on(d_y, d_y_row, sizeof(T), sizeof(T) * piece))) piece /= 2;
    const int lanes = ex_lanes(wide / piece, 32);
    const unsigned grid = ex_grid(n * lanes);
    void (*const kernel)(const T*, const float*, const int32_t*, const T*, int64_t, T*, float*, int64_t, int, int, int) =
        piece == MOST ? ex_combine_backward_kernel<T, MOST> : piece == 4 ? ex_combine_backward_kernel<T, 4> : piece == 2 ? ex_combine_backward_kernel<T, 2> : ex_combine_backward_kernel<T, 1>;
    kernel<<<grid, EX_THREADS, 0, s>>>(static_cast<const T*>(z), weights, experts, static_cast<const T*>(d_y), d_y_row, static_cast<T*>(d_z), d_weights, n, choices, wide, lanes);
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
    *bytes = ex_layout(e, args->dtype, backward != 0, want_x != 0, want_weights != 0, args->inner % 8 != 0 || (args->unaligned & 1), args->outer % 8 != 0 || (args->unaligned & 2)).total;
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
    const bool copy_x = ex_copies(x_dev, x_row, args->inner, args->dtype == DYNB_F32 ? 4 : 2);
    const ExLayout l = ex_layout(e, args->dtype, false, false, false, copy_x, false);
    if (workspace_dev == nullptr || !starts_on(workspace_dev, 16) || workspace_bytes < l.total) return fail_arg("workspace too small");
    e.t.x = x_dev; e.t.x_row = x_row; e.t.b = bias_dev; e.t.y = z_dev;
    e.slope = e.activation != DYNB_ACTIVATION_NONE ? slope_dev : nullptr;
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (args->dtype == DYNB_F32) return ex_forward<float>(e, args->dtype, ws, l, copy_x, s);
    if (args->dtype == DYNB_F16) return ex_forward<__half>(e, args->dtype, ws, l, copy_x, s);
    return ex_forward<__nv_bfloat16>(e, args->dtype, ws, l, copy_x, s);
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
    const int size = args->dtype == DYNB_F32 ? 4 : 2;
    const bool copy_x = ex_copies(x_dev, x_row, args->inner, size), copy_dy = ex_copies(d_z_dev, d_z_row, args->outer, size) || !ex_on(e.activation != DYNB_ACTIVATION_NONE ? slope_dev : nullptr, 0, size, 16);
    const ExLayout l = ex_layout(e, args->dtype, true, d_x_dev != nullptr, weights, copy_x, copy_dy);
    if (l.total > 0 && (workspace_dev == nullptr || !starts_on(workspace_dev, 16) || workspace_bytes < l.total)) return fail_arg("workspace too small");
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    e.t.x = x_dev; e.t.x_row = x_row; e.t.dy = d_z_dev; e.t.dy_row = d_z_row; e.t.dw = d_weight_dev; e.t.db = d_bias_dev;
    e.t.partial = reinterpret_cast<float*>(ws + l.partial);
    e.slope = const_cast<void*>(slope_dev);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (args->dtype == DYNB_F32) return ex_backward<float>(e, args->dtype, experts_dev, d_x_dev, ws, l, copy_x, copy_dy, s);
    if (args->dtype == DYNB_F16) return ex_backward<__half>(e, args->dtype, experts_dev, d_x_dev, ws, l, copy_x, copy_dy, s);
    return ex_backward<__nv_bfloat16>(e, args->dtype, experts_dev, d_x_dev, ws, l, copy_x, copy_dy, s);
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
