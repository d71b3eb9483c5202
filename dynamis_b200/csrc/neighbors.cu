// Lists of an edge list by target and by source (no counterpart in the reference, whose models gather and scatter along
// edge_index itself, dynamis_model/src/dynamis_model/nnp/mace.py:284-364).
//
//   rows, row_start   targets in the order of their runs in the edge list, those without edges behind them, ascending
//   cols, col_start   sources in the order of their first edge, those without edges behind them, ascending: sources that lie near one
//                     another stay together whatever their numbers are, because the runs are in cell order
//   src               sources of the edges in 32 bits
//   in_edge, in_dst   edges of a source in ascending order, and their targets
//
// Integer work, bound by memory and by atomics in L2: 16 B an edge in, 12 B out, one histogram entry and one minimum per edge.
// Everything is exact and independent of the order of the atomics: counts and minima commute, positions come from prefix sums.

#include <algorithm>

#include "clear.cuh"
#include "scan.cuh"

namespace dynb {

constexpr int NI_THREADS = 256;
constexpr int NI_ITEMS = 8;
constexpr int NI_TILE = NI_THREADS * NI_ITEMS;

struct NiLayout {
    int64_t run_of, count, first, place, sorted_count, tiles, scan, keys, total, total_sort;
    int64_t edge_tiles, node_tiles;
};

static NiLayout ni_layout(int64_t E, int64_t nt, int64_t ns)
{
    NiLayout l = {};
    l.edge_tiles = std::max<int64_t>((E + NI_TILE - 1) / NI_TILE, 1);
    l.node_tiles = std::max<int64_t>((std::max(nt, ns) + NI_TILE - 1) / NI_TILE, 1);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at = align_up(at + bytes, 256); return here; };
    l.run_of = take(4 * nt);                               // runs of a target
    l.count = take(4 * ns);                                // edges of a source
    l.first = take(4 * ns);                                // its first edge
    l.place = take(4 * ns);                                // its place in cols
    l.sorted_count = take(4 * (ns + 1));
    l.tiles = take(4 * (2 * l.edge_tiles + 2 * l.node_tiles + 8));  // run heads, first edges, empty targets, empty sources of a tile
    l.scan = take(8 * (std::max(l.edge_tiles, ns) / SCAN_TILE + 1 + 2));
    l.total = at;
    l.keys = take(8 * E);                                  // lists sorted by key
    l.total_sort = at;
    return l;
}

// Block-wide count of flags, one value a thread, and the exclusive prefix of the thread.
__device__ __forceinline__ uint32_t ni_prefix(uint32_t v, uint32_t* total)
{
    __shared__ uint32_t sums[NI_THREADS / 32];
    return block_excl_scan<uint32_t>(v, total, sums);
}

// Endpoints in range, targets in one run each, edges and first edge of every source, sources in 32 bits.
__global__ void __launch_bounds__(NI_THREADS)
ni_mark_kernel(const int64_t* src, const int64_t* dst, int64_t E, int64_t nt, int64_t ns, uint32_t* run_of, uint32_t* count,
               uint32_t* first, int32_t* src32, uint32_t* tile_heads, uint32_t* words)
{
    chain_begin();
    const int64_t base = (int64_t)blockIdx.x * NI_TILE;
    uint32_t heads = 0, status = 0;
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t e = base + k * NI_THREADS + threadIdx.x;
        if (e >= E) break;
        const int64_t s = src[e], d = dst[e];
        const bool head = e == 0 || dst[e - 1] != d;
        const bool ok = s >= 0 && s < ns && d >= 0 && d < nt;
        if (!ok) status |= 1u;
        if (ok && head) {
            heads++;
            if (atomicAdd(&run_of[d], 1u) != 0) status |= 2u;
        }
        if (ok) {
            atomicAdd(&count[s], 1u);
            atomicMin(&first[s], (uint32_t)e);
        }
        src32[e] = ok ? (int32_t)s : -1;
    }
    uint32_t total;
    (void)ni_prefix(heads, &total);
    if (threadIdx.x == 0) tile_heads[blockIdx.x] = total;
    if (status) atomicOr(&words[0], status);
}

// First edges of sources per tile of edges; targets and sources without edges per tile of nodes; longest list.
__global__ void __launch_bounds__(NI_THREADS)
ni_count_kernel(const int32_t* src32, int64_t E, int64_t nt, int64_t ns, const uint32_t* run_of, const uint32_t* count,
                const uint32_t* first, int edge_tiles, uint32_t* tile_firsts, uint32_t* tile_no_run, uint32_t* tile_no_edge, uint32_t* words)
{
    chain_begin();
    uint32_t total;
    if ((int)blockIdx.x < edge_tiles) {
        const int64_t base = (int64_t)blockIdx.x * NI_TILE;
        uint32_t firsts = 0;
#pragma unroll
        for (int k = 0; k < NI_ITEMS; k++) {
            const int64_t e = base + k * NI_THREADS + threadIdx.x;
            if (e < E && src32[e] >= 0 && first[src32[e]] == (uint32_t)e) firsts++;
        }
        (void)ni_prefix(firsts, &total);
        if (threadIdx.x == 0) tile_firsts[blockIdx.x] = total;
        return;
    }
    const int tile = blockIdx.x - edge_tiles;
    const int64_t base = (int64_t)tile * NI_TILE;
    uint32_t no_run = 0, no_edge = 0, longest = 0;
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t i = base + k * NI_THREADS + threadIdx.x;
        if (i < nt && run_of[i] == 0) no_run++;
        if (i < ns) {
            if (count[i] == 0) no_edge++;
            longest = max(longest, count[i]);
        }
    }
    (void)ni_prefix(no_run, &total);
    if (threadIdx.x == 0) tile_no_run[tile] = total;
    (void)ni_prefix(no_edge, &total);
    if (threadIdx.x == 0) tile_no_edge[tile] = total;
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((threadIdx.x & 31) == 0) atomicMax(&words[1], longest);
}

// One block: the four lists of tile counts become exclusive prefix sums, the empty nodes behind the others.
__global__ void __launch_bounds__(1024)
ni_tiles_kernel(uint32_t* heads, uint32_t* firsts, int edge_tiles, uint32_t* no_run, uint32_t* no_edge, int node_tiles)
{
    chain_begin();
    __shared__ uint32_t warp_sums[32];
    uint32_t carry_of[2] = {0, 0};
    for (int list = 0; list < 4; list++) {
        uint32_t* const at = list == 0 ? heads : list == 1 ? firsts : list == 2 ? no_run : no_edge;
        const int n = list < 2 ? edge_tiles : node_tiles;
        uint32_t carry = list < 2 ? 0 : carry_of[list - 2];
        for (int base = 0; base < n; base += 1024) {
            const int i = base + (int)threadIdx.x;
            const uint32_t v = i < n ? at[i] : 0;
            uint32_t x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
                if ((threadIdx.x & 31) >= o) x += y;
            }
            if ((threadIdx.x & 31) == 31) warp_sums[threadIdx.x >> 5] = x;
            __syncthreads();
            uint32_t before = 0, total = 0;
            for (int w = 0; w < 32; w++) {
                if (w < (int)(threadIdx.x >> 5)) before += warp_sums[w];
                total += warp_sums[w];
            }
            __syncthreads();
            if (i < n) at[i] = carry + before + x - v;
            carry += total;
        }
        if (list < 2) carry_of[list] = carry;
    }
}

// rows, row_start, cols, places and counts of the sources in that order.
__global__ void __launch_bounds__(NI_THREADS)
ni_rows_kernel(const int32_t* src32, const int64_t* dst, int64_t E, int64_t nt, int64_t ns, const uint32_t* run_of, const uint32_t* count,
               const uint32_t* first, int edge_tiles, const uint32_t* tile_heads, const uint32_t* tile_firsts, const uint32_t* tile_no_run,
               const uint32_t* tile_no_edge, int32_t* rows, int32_t* row_start, int32_t* cols, int32_t* place, uint32_t* sorted_count)
{
    chain_begin();
    uint32_t total;
    if ((int)blockIdx.x < edge_tiles) {
        const int64_t base = (int64_t)blockIdx.x * NI_TILE;
        uint32_t at_row = tile_heads[blockIdx.x], at_col = tile_firsts[blockIdx.x];
#pragma unroll 1
        for (int k = 0; k < NI_ITEMS; k++) {
            const int64_t e = base + k * NI_THREADS + threadIdx.x;
            const int32_t s = e < E ? src32[e] : -1;
            const int64_t d = s >= 0 ? dst[e] : -1;
            const bool head = s >= 0 && (e == 0 || dst[e - 1] != d);
            const bool is_first = s >= 0 && first[s] == (uint32_t)e;
            const uint32_t both = (head ? 1u : 0u) | (is_first ? 1u << 16 : 0u);
            const uint32_t before = ni_prefix(both, &total);
            const uint32_t r = at_row + (before & 0xffffu), c = at_col + (before >> 16);
            if (head && r < nt) {
                rows[r] = (int32_t)d;
                row_start[r] = (int32_t)e;
            }
            if (is_first && c < ns) {
                cols[c] = s;
                place[s] = (int32_t)c;
                sorted_count[c] = count[s];
            }
            at_row += total & 0xffffu;
            at_col += total >> 16;
        }
        return;
    }
    const int tile = blockIdx.x - edge_tiles;
    const int64_t base = (int64_t)tile * NI_TILE;
    uint32_t at_row = tile_no_run[tile], at_col = tile_no_edge[tile];
#pragma unroll 1
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t i = base + k * NI_THREADS + threadIdx.x;
        const bool no_run = i < nt && run_of[i] == 0, no_edge = i < ns && count[i] == 0;
        const uint32_t both = (no_run ? 1u : 0u) | (no_edge ? 1u << 16 : 0u);
        const uint32_t before = ni_prefix(both, &total);
        const uint32_t r = at_row + (before & 0xffffu), c = at_col + (before >> 16);
        if (no_run && r < nt) {
            rows[r] = (int32_t)i;
            row_start[r] = (int32_t)E;
        }
        if (no_edge && c < ns) {
            cols[c] = (int32_t)i;
            sorted_count[c] = 0;
        }
        at_row += total & 0xffffu;
        at_col += total >> 16;
    }
    if (tile == 0 && threadIdx.x == 0) {
        row_start[nt] = (int32_t)E;
        sorted_count[ns] = 0;
    }
}

__global__ void __launch_bounds__(1)
ni_words_kernel(const uint32_t* words, int64_t* host)
{
    chain_begin();
    host[0] = words[0];
    host[1] = words[1];
}

__global__ void __launch_bounds__(NI_THREADS)
ni_keys_kernel(const int32_t* src32, int64_t E, const int32_t* place, uint64_t* keys, uint32_t* edges)
{
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < E; e += (int64_t)gridDim.x * blockDim.x) {
        keys[e] = (uint32_t)place[src32[e]];
        edges[e] = (uint32_t)e;
    }
}

__global__ void __launch_bounds__(NI_THREADS)
ni_targets_kernel(const int32_t* in_edge, const int64_t* dst, int64_t E, int32_t* in_dst)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < E; i += (int64_t)gridDim.x * blockDim.x) in_dst[i] = (int32_t)dst[in_edge[i]];
}

}  // namespace dynb

using namespace dynb;

static int ni_check(int64_t E, int64_t nt, int64_t ns)
{
    if (E < 0 || nt < 0 || ns < 0) return fail_arg("neighbor_index: sizes must be non-negative");
    if (E >= DYNB_MAX_EDGES || nt >= INT32_MAX || ns >= INT32_MAX) return fail_arg("neighbor_index: sizes must be below 2^31 - 1, edges below 2^31 - 2^16");
    return DYNB_OK;
}

extern "C" int dynb_neighbor_index_workspace_bytes(int64_t n_edges, int64_t n_targets, int64_t n_sources, int64_t* bytes)
{
    if (bytes == nullptr) return fail_arg("null pointer");
    const int rc = ni_check(n_edges, n_targets, n_sources);
    if (rc != DYNB_OK) return rc;
    int64_t sort;
    const int rs = dynb_radix_sort_workspace_bytes(n_edges, &sort);
    if (rs != DYNB_OK) return rs;
    *bytes = ni_layout(n_edges, n_targets, n_sources).total_sort + align_up(sort, 256);
    return DYNB_OK;
}

extern "C" int dynb_neighbor_index_plan(const int64_t* src_dev, const int64_t* dst_dev, int64_t n_edges, int64_t n_targets, int64_t n_sources,
                                        int32_t* rows_dev, int32_t* row_start_dev, int32_t* src32_dev, int32_t* cols_dev,
                                        int32_t* col_start_dev, int64_t* words_host, void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    const int rc = ni_check(n_edges, n_targets, n_sources);
    if (rc != DYNB_OK) return rc;
    if (row_start_dev == nullptr || col_start_dev == nullptr || workspace_dev == nullptr || words_host == nullptr) return fail_arg("null pointer");
    if ((n_edges > 0 && (!src_dev || !dst_dev || !src32_dev)) || (n_targets > 0 && !rows_dev) || (n_sources > 0 && !cols_dev))
        return fail_arg("null pointer");
    const NiLayout l = ni_layout(n_edges, n_targets, n_sources);
    if (workspace_bytes < l.total) return fail_arg("workspace too small");
    void* const words_at = device_view_of_host(words_host);
    if (words_at == nullptr) return fail_arg("neighbor_index: words_host must be pinned");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    uint32_t* const run_of = reinterpret_cast<uint32_t*>(ws + l.run_of);
    uint32_t* const count = reinterpret_cast<uint32_t*>(ws + l.count);
    uint32_t* const first = reinterpret_cast<uint32_t*>(ws + l.first);
    int32_t* const place = reinterpret_cast<int32_t*>(ws + l.place);
    uint32_t* const sorted_count = reinterpret_cast<uint32_t*>(ws + l.sorted_count);
    uint32_t* const heads = reinterpret_cast<uint32_t*>(ws + l.tiles);
    uint32_t* const firsts = heads + l.edge_tiles;
    uint32_t* const no_run = firsts + l.edge_tiles;
    uint32_t* const no_edge = no_run + l.node_tiles;
    uint32_t* const words = no_edge + l.node_tiles;
    const int et = (int)l.edge_tiles, nt = (int)l.node_tiles;
    DYNB_CUDA_OK(clear_ranges(s, {run_of, 4 * n_targets, 0}, {count, 4 * n_sources, 0}, {first, 4 * n_sources, 0xff}, {words, 32, 0}));
    DYNB_CUDA_OK(launch_chained(ni_mark_kernel, et, NI_THREADS, 0, s, src_dev, dst_dev, n_edges, n_targets, n_sources, run_of, count, first,
                                src32_dev, heads, words));
    DYNB_CUDA_OK(launch_chained(ni_count_kernel, et + nt, NI_THREADS, 0, s, src32_dev, n_edges, n_targets, n_sources, run_of, count, first, et,
                                firsts, no_run, no_edge, words));
    DYNB_CUDA_OK(launch_chained(ni_tiles_kernel, 1, 1024, 0, s, heads, firsts, et, no_run, no_edge, nt));
    DYNB_CUDA_OK(launch_chained(ni_rows_kernel, et + nt, NI_THREADS, 0, s, src32_dev, dst_dev, n_edges, n_targets, n_sources, run_of, count,
                                first, et, heads, firsts, no_run, no_edge, rows_dev, row_start_dev, cols_dev, place, sorted_count));
    DYNB_CUDA_OK(exclusive_scan(sorted_count, reinterpret_cast<uint32_t*>(col_start_dev), nullptr, n_sources + 1,
                                reinterpret_cast<uint32_t*>(ws + l.scan), static_cast<uint32_t*>(nullptr), s));
    DYNB_CUDA_OK(launch_chained(ni_words_kernel, 1, 1, 0, s, words, static_cast<int64_t*>(words_at)));
    return DYNB_OK;
}

extern "C" int dynb_neighbor_index_fill(const int64_t* dst_dev, int64_t n_edges, int64_t n_targets, int64_t n_sources, const int32_t* src32_dev,
                                        const int32_t* col_start_dev, int64_t longest, int32_t* in_edge_dev, int32_t* in_dst_dev,
                                        void* workspace_dev, int64_t workspace_bytes, void* stream)
{
    const int rc = ni_check(n_edges, n_targets, n_sources);
    if (rc != DYNB_OK) return rc;
    if (n_edges == 0) return DYNB_OK;
    if (!dst_dev || !src32_dev || !col_start_dev || !in_edge_dev || !in_dst_dev || !workspace_dev) return fail_arg("null pointer");
    const NiLayout l = ni_layout(n_edges, n_targets, n_sources);
    int64_t sort;
    (void)dynb_radix_sort_workspace_bytes(n_edges, &sort);
    if (workspace_bytes < l.total_sort + sort) return fail_arg("workspace too small");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    const int32_t* const place = reinterpret_cast<const int32_t*>(ws + l.place);
    (void)longest;
    uint64_t* const keys = reinterpret_cast<uint64_t*>(ws + l.keys);
    const unsigned blocks = (unsigned)std::min<int64_t>((n_edges + NI_THREADS - 1) / NI_THREADS, (int64_t)sm_count_cached() * 8);
    int bits = 8;
    while (bits < 32 && (n_sources >> bits) != 0) bits += 8;
    ni_keys_kernel<<<blocks, NI_THREADS, 0, s>>>(src32_dev, n_edges, place, keys, reinterpret_cast<uint32_t*>(in_edge_dev));
    DYNB_CUDA_OK(cudaGetLastError());
    const int rs = dynb_radix_sort_pairs(keys, reinterpret_cast<uint32_t*>(in_edge_dev), n_edges, 0, bits, ws + l.total_sort, sort, stream);
    if (rs != DYNB_OK) return rs;
    ni_targets_kernel<<<blocks, NI_THREADS, 0, s>>>(in_edge_dev, dst_dev, n_edges, in_dst_dev);
    DYNB_CUDA_OK(cudaGetLastError());
    return DYNB_OK;
}
