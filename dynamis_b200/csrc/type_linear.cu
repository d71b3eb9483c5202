// Rows times the matrix of their type (no counterpart in the reference, whose models leave it to their libraries):
//     y_i = x_i W[type_i] + b[type_i],   dx_i = dy_i W[type_i]^T,   dW[t] = sum over the rows i of type t of x_i^T dy_i,   db[t] = sum dy_i.
// The rows are not moved: `order` lists them by type (ascending inside a type), `start` where every type begins, and a tile gathers its
// rows as it loads them.  Products are summed in 32 bits and rounded once.  Sums over rows go in stretches of a fixed number of rows of a
// type, joined in their order: no atomics.

#include "clear.cuh"
#include "type_linear.cuh"

namespace dynb {

constexpr int TL_M = 64, TL_N = 64, TL_K = 16, TL_THREADS = 256;

// One tile of 64 gathered rows times 64 columns, for matrices that do not fit into shared memory (type_linear_mma.cu):
// bound by its multiply-adds, 200 k rows of 400 x 400 in fp32 4.2 ms (a loop over the types with library products: 1.9), 512 x 128 1.5 ms (0.85).
// `back`: dx = dy W^T instead of y = x W + b.
template <typename T>
__global__ void __launch_bounds__(TL_THREADS)
tl_rows_kernel(const TlArgs a, int back)
{
    __shared__ float sa[TL_K][TL_M + 4], sb[TL_K][TL_N + 4];
    __shared__ int32_t rows[TL_M];
    const TlTile tile = tl_tile(a, blockIdx.x, TL_M);
    if (tile.type < 0) return;
    const T* const in = static_cast<const T*>(back ? a.dy : a.x);
    const T* const w = static_cast<const T*>(a.w) + (int64_t)tile.type * a.inner * a.outer;
    T* const out = static_cast<T*>(back ? a.dx : a.y);
    const int64_t in_row = back ? a.dy_row : a.x_row;
    const int kk = back ? a.outer : a.inner, nn = back ? a.inner : a.outer;
    if (threadIdx.x < TL_M) {
        int32_t r = -1;
        if (tile.begin + threadIdx.x < tile.end) {
            r = a.order[tile.begin + threadIdx.x];
            if ((uint32_t)r >= (uint64_t)a.n) r = -1;
        }
        rows[threadIdx.x] = r;
    }
    __syncthreads();
    const int col0 = blockIdx.y * TL_N, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < kk; k0 += TL_K) {
#pragma unroll
        for (int i = threadIdx.x; i < TL_M * TL_K; i += TL_THREADS) {
            const int m = i / TL_K, k = i % TL_K;
            sa[k][m] = rows[m] >= 0 && k0 + k < kk ? tl_get(in + rows[m] * in_row + k0 + k) : 0.0f;
        }
#pragma unroll
        for (int i = threadIdx.x; i < TL_N * TL_K; i += TL_THREADS) {
            const int k = back ? i % TL_K : i / TL_N, n = back ? i / TL_K : i % TL_N;
            const bool ok = k0 + k < kk && col0 + n < nn;
            sb[k][n] = ok ? tl_get(back ? w + (int64_t)(col0 + n) * a.outer + k0 + k : w + (int64_t)(k0 + k) * a.outer + col0 + n) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TL_K; k++) {
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
        const int32_t r = rows[ty * 4 + i];
        if (r < 0) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = col0 + tx * 4 + j;
            if (n >= nn) continue;
            float v = acc[i][j];
            if (!back && a.b != nullptr) v += tl_get(static_cast<const T*>(a.b) + (int64_t)tile.type * a.outer + n);
            tl_put(out + (int64_t)r * nn + n, v);
        }
    }
}

// The stretches of a type joined: blockIdx.y is the type.
template <typename T>
__global__ void __launch_bounds__(TL_THREADS)
tl_join_kernel(const TlArgs a, int64_t stretches)
{
    const int type = blockIdx.y;
    __shared__ int64_t first_of, count_of;
    if (threadIdx.x < 32) {   // stretches of the types before
        int64_t first = 0;
        for (int t = threadIdx.x; t < type; t += 32) {
            const int64_t rows = min((int64_t)a.start[t + 1], a.n) - max(a.start[t], 0);
            first += rows > 0 ? (rows + a.stretch - 1) / a.stretch : 0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first += __shfl_xor_sync(0xffffffffu, first, o);
        if (threadIdx.x == 0) {
            const int64_t rows = min((int64_t)a.start[type + 1], a.n) - max(a.start[type], 0);
            first_of = first;
            count_of = rows > 0 ? (rows + a.stretch - 1) / a.stretch : 0;
        }
    }
    __syncthreads();
    const int64_t cells = (int64_t)a.inner * a.outer, all = cells + a.outer, first = first_of, count = min(count_of, stretches - first_of);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        double exact = 0.0;   // as many as a thousand stretches
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

// Types as sort keys; bit 0 of `words` where one lies outside [0, types).
__global__ void __launch_bounds__(TL_THREADS)
tl_keys_kernel(const int64_t* types, int64_t n, int n_types, uint64_t* keys, uint32_t* order, uint32_t* word)
{
    chain_begin();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        int64_t t = types[i];
        if (t < 0 || t >= n_types) {
            atomicOr(word, 1u);
            t = 0;
        }
        keys[i] = (uint64_t)t;
        order[i] = (uint32_t)i;
    }
}

// Where every type begins in the sorted keys; the word to the host.
__global__ void __launch_bounds__(TL_THREADS)
tl_start_kernel(const uint64_t* keys, int64_t n, int n_types, int32_t* start, const uint32_t* word, int64_t* host)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i <= n; i += (int64_t)gridDim.x * blockDim.x) {
        const int from = i == 0 ? 0 : (int)keys[i - 1] + 1, to = i == n ? n_types : (int)keys[i];
        for (int t = from; t <= to; t++) start[t] = (int32_t)i;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) host[0] = *word;
}

struct TiLayout { int64_t word, keys, sort, total; };
static TiLayout ti_layout(int64_t n)
{
    int64_t sort = 0;
    (void)dynb_radix_sort_workspace_bytes(n, &sort);
    TiLayout l;
    l.word = 0;
    l.keys = 256;
    l.sort = align_up(l.keys + 8 * n, 256);
    l.total = l.sort + align_up(sort, 256);
    return l;
}

static int tl_args(const dynb_type_linear_args* in, TlArgs* a)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("type_linear: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->n_rows < 0 || in->n_rows >= INT32_MAX) return fail_arg("type_linear: rows must lie in [0, 2^31 - 1)");
    if (in->types < 1 || in->types > DYNB_TYPE_LINEAR_MAX_TYPES) return fail_arg("type_linear: types must lie in [1, 4096]");
    if (in->inner < 1 || in->outer < 1 || in->inner > DYNB_TYPE_LINEAR_MAX_WIDTH || in->outer > DYNB_TYPE_LINEAR_MAX_WIDTH)
        return fail_arg("type_linear: widths must lie in [1, 16384]");
    if (!in->start_dev || !in->weight_dev || (in->n_rows > 0 && !in->order_dev)) return fail_arg("null pointer");
    *a = TlArgs{};
    a->w = in->weight_dev;
    a->order = in->order_dev;
    a->start = in->start_dev;
    a->n = in->n_rows;
    a->types = in->types;
    a->inner = in->inner;
    a->outer = in->outer;
    a->stretch = tl_stretch(in->n_rows, in->inner, in->outer, in->dtype);
    a->status = in->status_dev;
    return DYNB_OK;
}

template <typename T>
static cudaError_t tl_rows_plain(const TlArgs& a, int back, cudaStream_t s)
{
    const int nn = back ? a.inner : a.outer;
    const dim3 grid((unsigned)((a.n + TL_M - 1) / TL_M + a.types), (nn + TL_N - 1) / TL_N);
    tl_rows_kernel<T><<<grid, TL_THREADS, 0, s>>>(a, back);
    return cudaGetLastError();
}

static cudaError_t tl_rows(const TlArgs& a, int back, int dtype, cudaStream_t s)
{
    cudaError_t rc;
    if (tl_mma_rows(a, back, dtype, s, &rc)) return rc;
    return dtype == DYNB_F32 ? tl_rows_plain<float>(a, back, s) : dtype == DYNB_F16 ? tl_rows_plain<__half>(a, back, s) : tl_rows_plain<__nv_bfloat16>(a, back, s);
}

static cudaError_t tl_weights(const TlArgs& a, int dtype, cudaStream_t s)
{
    const cudaError_t rc = tl_mma_weights(a, dtype, s);
    if (rc != cudaSuccess) return rc;
    const int64_t stretches = tl_stretches(a.n, a.types, a.stretch), all = (int64_t)a.inner * a.outer + a.outer;
    const dim3 grid((unsigned)std::min<int64_t>((all + TL_THREADS - 1) / TL_THREADS, 1024), a.types);
    if (dtype == DYNB_F32) tl_join_kernel<float><<<grid, TL_THREADS, 0, s>>>(a, stretches);
    else if (dtype == DYNB_F16) tl_join_kernel<__half><<<grid, TL_THREADS, 0, s>>>(a, stretches);
    else tl_join_kernel<__nv_bfloat16><<<grid, TL_THREADS, 0, s>>>(a, stretches);
    return cudaGetLastError();
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_type_linear(const dynb_type_linear_args* args, const void* x_dev, int64_t x_row, const void* bias_dev, void* y_dev, void* stream)
{
    TlArgs a;
    const int rc = tl_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (a.n == 0) return DYNB_OK;
    if (!x_dev || !y_dev) return fail_arg("null pointer");
    a.x = x_dev; a.x_row = x_row; a.b = bias_dev; a.y = y_dev;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    DYNB_CUDA_OK(tl_rows(a, 0, args->dtype, s));
    return DYNB_OK;
}

extern "C" int dynb_type_linear_workspace_bytes(const dynb_type_linear_args* args, int64_t* bytes)
{
    TlArgs a;
    const int rc = tl_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (bytes == nullptr) return fail_arg("null pointer");
    *bytes = tl_stretches(a.n, a.types, a.stretch) * ((int64_t)a.inner * a.outer + a.outer) * 4;
    return DYNB_OK;
}

extern "C" int dynb_type_linear_backward(const dynb_type_linear_args* args, const void* x_dev, int64_t x_row, const void* d_y_dev, int64_t d_y_row,
                                         void* d_x_dev, void* d_weight_dev, void* d_bias_dev, void* workspace_dev, int64_t workspace_bytes,
                                         void* stream)
{
    TlArgs a;
    const int rc = tl_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (a.n > 0 && (!x_dev || !d_y_dev)) return fail_arg("null pointer");
    a.x = x_dev; a.x_row = x_row; a.dy = d_y_dev; a.dy_row = d_y_row; a.dx = d_x_dev; a.dw = d_weight_dev; a.db = d_bias_dev;
    a.partial = static_cast<float*>(workspace_dev);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d_x_dev != nullptr && a.n > 0)
        DYNB_CUDA_OK(tl_rows(a, 1, args->dtype, s));
    if (d_weight_dev != nullptr || d_bias_dev != nullptr) {
        int64_t need;
        (void)dynb_type_linear_workspace_bytes(args, &need);
        if (workspace_dev == nullptr || workspace_bytes < need) return fail_arg("workspace too small");
        DYNB_CUDA_OK(tl_weights(a, args->dtype, s));
    }
    return DYNB_OK;
}

extern "C" int dynb_type_index_workspace_bytes(int64_t n_rows, int64_t* bytes)
{
    if (n_rows < 0 || n_rows >= INT32_MAX || bytes == nullptr) return fail_arg("type_index: rows must lie in [0, 2^31 - 1)");
    *bytes = ti_layout(n_rows).total;
    return DYNB_OK;
}

extern "C" int dynb_type_index(const int64_t* types_dev, int64_t n_rows, int types, int32_t* order_dev, int32_t* start_dev, int64_t* word_host,
                               void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    if (n_rows < 0 || n_rows >= INT32_MAX) return fail_arg("type_index: rows must lie in [0, 2^31 - 1)");
    if (types < 1 || types > DYNB_TYPE_LINEAR_MAX_TYPES) return fail_arg("type_index: types must lie in [1, 4096]");
    if (!start_dev || !workspace_dev || !word_host || (n_rows > 0 && (!types_dev || !order_dev))) return fail_arg("null pointer");
    if (!starts_on(workspace_dev, 16)) return fail_arg("type_index: the workspace must start on a 16-byte boundary");
    const TiLayout l = ti_layout(n_rows);
    if (workspace_bytes < l.total) return fail_arg("workspace too small");
    void* const word_at = device_view_of_host(word_host);
    if (word_at == nullptr) return fail_arg("type_index: word_host must be pinned, on a 16-byte boundary");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    uint32_t* const word = reinterpret_cast<uint32_t*>(ws + l.word);
    uint64_t* const keys = reinterpret_cast<uint64_t*>(ws + l.keys);
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((n_rows + TL_THREADS) / TL_THREADS, (int64_t)sm_count_cached() * 8));
    DYNB_CUDA_OK(clear_ranges(s, {word, 4, 0}));
    DYNB_CUDA_OK(launch_chained(tl_keys_kernel, blocks, TL_THREADS, 0, s, types_dev, n_rows, types, keys, reinterpret_cast<uint32_t*>(order_dev), word));
    if (n_rows > 0) {
        const int rc = dynb_radix_sort_pairs(keys, reinterpret_cast<uint32_t*>(order_dev), n_rows, 0, types <= 256 ? 8 : 16, ws + l.sort, l.total - l.sort, stream);
        if (rc != DYNB_OK) return rc;
    }
    tl_start_kernel<<<blocks, TL_THREADS, 0, s>>>(keys, n_rows, types, start_dev, word, static_cast<int64_t*>(word_at));
    DYNB_CUDA_OK(cudaGetLastError());
    return DYNB_OK;
}
