// C entry points of neighbour attention: checks of the arguments, then the kernels of attention_forward.cu and attention_backward.cu.

#include <initializer_list>

#include "attention.cuh"

namespace dynb {

static int attn_args(const dynb_attention* in, AttnArgs* a)
{
    if (in == nullptr) return fail_arg("null pointer");
    if (in->dtype != DYNB_F32 && in->dtype != DYNB_F16 && in->dtype != DYNB_BF16) return fail_arg("neighbor_attention: dtype must be DYNB_F32, DYNB_F16 or DYNB_BF16");
    if (in->n_targets < 0 || in->n_sources < 0 || in->n_edges < 0) return fail_arg("neighbor_attention: sizes must be non-negative");
    if (in->n_targets >= INT32_MAX || in->n_sources >= INT32_MAX || in->n_edges >= DYNB_MAX_EDGES) return fail_arg("neighbor_attention: sizes must be below 2^31 - 1, edges below 2^31 - 2^16");
    if (in->heads < 1 || in->kv_heads < 1 || in->heads % in->kv_heads != 0 || in->heads > 65535) return fail_arg("neighbor_attention: heads must be a multiple of kv_heads");
    if (in->dim < 1 || in->dim > DYNB_ATTENTION_MAX_DIM) return fail_arg("neighbor_attention: dim must lie in [1, 256]");
    if (in->n_targets > 0 && (!in->rows_dev || !in->row_start_dev || !in->q_dev)) return fail_arg("null pointer");
    if (in->n_edges > 0 && (!in->src_dev || !in->k_dev || !in->v_dev)) return fail_arg("null pointer");
    for (const int64_t row : {in->q_row, in->k_row, in->v_row})
        if (row < 0 || row >= DYNB_ATTENTION_MAX_ROW) return fail_arg("neighbor_attention: row strides must lie in [0, 2^30)");
    *a = AttnArgs{};
    a->q = {in->q_dev, in->q_row, in->q_head};
    a->k = {in->k_dev, in->k_row, in->k_head};
    a->v = {in->v_dev, in->v_row, in->v_head};
    a->bias = in->bias_dev;
    a->rows = in->rows_dev;
    a->row_start = in->row_start_dev;
    a->src = in->src_dev;
    a->n_targets = in->n_targets;
    a->n_sources = in->n_sources;
    a->n_edges = in->n_targets > 0 && in->n_sources > 0 ? in->n_edges : 0;   // an edge has both ends
    a->heads = in->heads;
    a->kv_heads = in->kv_heads;
    a->shared = in->heads / in->kv_heads;
    a->dim = in->dim;
    a->scale = in->scale;
    return DYNB_OK;
}

// Whether the rows of a tensor lie in 128 GB.
static bool attn_narrow(const AttnRows& r, int64_t rows, int heads, int size) { return (rows * r.row + heads * r.head) * size / 32 < (1ll << 32); }

// Bytes on which the heads of all these tensors start and end.
static int attn_wide(int dim, int size, std::initializer_list<AttnRows> all, std::initializer_list<const void*> outputs)
{
    uint64_t bits = (uint64_t)dim * size;
    for (const AttnRows& r : all) bits |= reinterpret_cast<uintptr_t>(r.at) | (uint64_t)r.row * size | (uint64_t)r.head * size;
    for (const void* p : outputs) bits |= reinterpret_cast<uintptr_t>(p);
    return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : size;
}

}  // namespace dynb

using namespace dynb;

extern "C" int dynb_neighbor_attention(const dynb_attention* args, void* out_dev, float* out32_dev, float* stats_dev, void* stream)
{
    AttnArgs a;
    const int rc = attn_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (a.n_targets == 0) return DYNB_OK;
    if (out_dev == nullptr) return fail_arg("null pointer");
    const int size = args->dtype == DYNB_F32 ? 4 : 2;
    if (size == 2 && !starts_on(out32_dev, 8)) return fail_arg("neighbor_attention: out32 must start on an 8-byte boundary");
    a.out = out_dev;
    a.out32_w = out32_dev;
    a.stats_w = stats_dev;
    a.wide = attn_wide(a.dim, size, {a.q, a.k, a.v}, {out_dev});
    a.narrow = attn_narrow(a.k, a.n_sources, a.kv_heads, size) && attn_narrow(a.v, a.n_sources, a.kv_heads, size);
    DYNB_CUDA_OK(attn_forward(a, args->dtype, static_cast<cudaStream_t>(stream)));
    return DYNB_OK;
}

extern "C" int dynb_neighbor_attention_backward(const dynb_attention* args, const void* d_out_dev, int64_t d_out_row, int64_t d_out_head,
                                                const float* out32_dev, const float* stats_dev, const int32_t* cols_dev, const int32_t* col_start_dev,
                                                const int32_t* in_edge_dev, const int32_t* in_dst_dev, float* delta_dev, void* dq_dev, void* dk_dev,
                                                void* dv_dev, float* d_bias_dev, void* stream)
{
    AttnArgs a;
    const int rc = attn_args(args, &a);
    if (rc != DYNB_OK) return rc;
    if (d_out_row < 0 || d_out_row >= DYNB_ATTENTION_MAX_ROW) return fail_arg("neighbor_attention: row strides must lie in [0, 2^30)");
    const int size = args->dtype == DYNB_F32 ? 4 : 2;
    a.d_out = {d_out_dev, d_out_row, d_out_head};
    a.out32 = out32_dev;
    a.stats = stats_dev;
    a.delta = static_cast<float4*>(static_cast<void*>(delta_dev));
    a.cols = cols_dev;
    a.col_start = col_start_dev;
    a.in_edge = in_edge_dev;
    a.in_dst = in_dst_dev;
    a.dq = dq_dev;
    a.dk = dk_dev;
    a.dv = dv_dev;
    a.d_bias = d_bias_dev;
    if (d_bias_dev != nullptr && a.bias == nullptr) return fail_arg("neighbor_attention_backward: a gradient of a bias that is not there");
    a.wide = attn_wide(a.dim, size, {a.q, a.k, a.v, a.d_out}, {dq_dev, dk_dev, dv_dev});
    a.narrow = attn_narrow(a.k, a.n_sources, a.kv_heads, size) && attn_narrow(a.v, a.n_sources, a.kv_heads, size) &&
               attn_narrow(a.q, a.n_targets, a.heads, size) && attn_narrow(a.d_out, a.n_targets, a.heads, size);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool cols = (dk_dev != nullptr || dv_dev != nullptr) && a.n_sources > 0;
    if (a.n_targets > 0) {   // also for the sources' gradients, which read delta
        if (!d_out_dev || !out32_dev || !stats_dev || !delta_dev) return fail_arg("null pointer");
        if (!starts_on(delta_dev, 16)) return fail_arg("neighbor_attention_backward: delta must start on a 16-byte boundary");
        DYNB_CUDA_OK(attn_backward_rows(a, args->dtype, s));
    }
    if (cols) {
        if (!cols_dev || !col_start_dev || (a.n_edges > 0 && (!in_edge_dev || !in_dst_dev))) return fail_arg("null pointer");
        if (a.k.at == nullptr || a.v.at == nullptr) return fail_arg("null pointer");
        DYNB_CUDA_OK(attn_backward_cols(a, args->dtype, s));
    }
    return DYNB_OK;
}
