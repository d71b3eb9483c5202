// Lists of an edge list by target and by source (no counterpart in the reference, whose models gather and scatter along
// edge_index itself, dynamis_model/src/dynamis_model/nnp/mace.py:284-364).
//
//   rows, row_start   targets in the order of their runs in the edge list, those without edges behind them, ascending
//   cols, col_start   sources in the order of their first edge, those without edges behind them, ascending: sources that lie near one
//                     another stay together whatever their numbers are, because the runs are in cell order
//   src               sources of the edges in 32 bits
//   in_edge, in_dst   edges of a source in ascending order, and their targets
//
// Integer work, bound by atomics and scattered accesses in L2: an edge counts itself at its source and so gets a number inside the source's list, in
// whatever order the atomics came; it is put at that place, and every list is then sorted by a warp.  The result does not depend on the order
// of the atomics.  Lists too long for a warp's registers (a hub) go through a radix sort of all edges.
// 154 k targets, 200 k sources, 8.1 M edges: 358 us, of which the numbers take 132, the places 58 and the sorting of the lists 99 (radix sort of all edges: 641 us in all).

#include <algorithm>

#include "clear.cuh"
#include "scan.cuh"

namespace dynb {

constexpr int NI_THREADS = 256;
constexpr int NI_ITEMS = 8;
constexpr int NI_TILE = NI_THREADS * NI_ITEMS;

struct NiLayout {
    int64_t run_of, count, first, place, sorted_count, bits, tiles, words, scan, keys, total, total_fill, total_sort;
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
    l.bits = take(8 * l.edge_tiles * (NI_TILE / 32));      // a bit an edge: first of its target's run; first of its source
    l.tiles = take(4 * (2 * l.edge_tiles + 2 * l.node_tiles));   // run heads, first edges, empty targets, empty sources of a tile
    l.words = take(64);
    l.scan = take(8 * (std::max(l.edge_tiles, ns) / SCAN_TILE + 1 + 2));
    l.total = at;
    l.keys = take(8 * E);                                  // edges and targets at their places; keys of the sort
    l.total_fill = at;
    l.total_sort = at;
    return l;
}

// Block-wide count of flags, one value a thread, and the exclusive prefix of the thread.
__device__ __forceinline__ uint32_t ni_prefix(uint32_t v, uint32_t* total)
{
    __shared__ uint32_t sums[NI_THREADS / 32];
    return block_excl_scan<uint32_t>(v, total, sums);
}

// Endpoints in range, targets in one run each, edges and first edge of every source, numbers of the edges at their source, sources in 32 bits.
__global__ void __launch_bounds__(NI_THREADS)
ni_mark_kernel(const int64_t* src, const int64_t* dst, int64_t E, int64_t nt, int64_t ns, uint32_t* run_of, uint32_t* count,
               uint32_t* first, int32_t* src32, int32_t* number, uint32_t* head_bits, uint32_t* tile_heads, uint32_t* words)
{
    chain_begin();
    const int64_t base = (int64_t)blockIdx.x * NI_TILE + threadIdx.x;
    uint32_t heads = 0, status = 0;
    int64_t s[NI_ITEMS], d[NI_ITEMS], before[NI_ITEMS];
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t e = base + k * NI_THREADS;
        s[k] = d[k] = before[k] = -1;
        if (e < E) {
            s[k] = src[e];
            d[k] = dst[e];
            if (e > 0) before[k] = dst[e - 1];
        }
    }
    uint32_t seen[NI_ITEMS], mine[NI_ITEMS];
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t e = base + k * NI_THREADS;
        const bool ok = s[k] >= 0 && s[k] < ns && d[k] >= 0 && d[k] < nt, head = ok && (e == 0 || before[k] != d[k]);
        if (e < E && !ok) status |= 1u;
        const uint32_t bits = __ballot_sync(0xffffffffu, head);
        if ((threadIdx.x & 31) == 0) head_bits[(base + k * NI_THREADS) >> 5] = bits;
        if (head) {
            heads++;
            if (atomicAdd(&run_of[d[k]], 1u) != 0) status |= 2u;
        }
        if (!ok) s[k] = -1;
        seen[k] = mine[k] = 0;
        if (ok) {
            mine[k] = atomicAdd(&count[s[k]], 1u);
            seen[k] = __ldcg(first + s[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t e = base + k * NI_THREADS;
        if (e >= E) break;
        src32[e] = (int32_t)s[k];
        number[e] = (int32_t)mine[k];
        if (s[k] >= 0 && (uint32_t)e < seen[k]) atomicMin(&first[s[k]], (uint32_t)e);   // few edges: the earlier ones mostly come first
    }
    uint32_t total;
    (void)ni_prefix(heads, &total);
    if (threadIdx.x == 0) tile_heads[blockIdx.x] = total;
    if (status) atomicOr(&words[0], status);
}

// First edges of sources per tile of edges; targets and sources without edges per tile of nodes; longest list.
__global__ void __launch_bounds__(NI_THREADS)
ni_count_kernel(const int32_t* src32, int64_t E, int64_t nt, int64_t ns, const uint32_t* run_of, const uint32_t* count,
                const uint32_t* first, int edge_tiles, uint32_t* first_bits, uint32_t* tile_firsts, uint32_t* tile_no_run, uint32_t* tile_no_edge,
                uint32_t* words)
{
    chain_begin();
    uint32_t total;
    if ((int)blockIdx.x < edge_tiles) {
        const int64_t base = (int64_t)blockIdx.x * NI_TILE + threadIdx.x;
        uint32_t firsts = 0, at[NI_ITEMS];
        int32_t s[NI_ITEMS];
#pragma unroll
        for (int k = 0; k < NI_ITEMS; k++) s[k] = base + k * NI_THREADS < E ? src32[base + k * NI_THREADS] : -1;
#pragma unroll
        for (int k = 0; k < NI_ITEMS; k++) at[k] = s[k] >= 0 ? first[s[k]] : 0xffffffffu;
#pragma unroll
        for (int k = 0; k < NI_ITEMS; k++) {
            const bool is_first = s[k] >= 0 && at[k] == (uint32_t)(base + k * NI_THREADS);
            const uint32_t bits = __ballot_sync(0xffffffffu, is_first);
            if ((threadIdx.x & 31) == 0) first_bits[(base + k * NI_THREADS) >> 5] = bits;
            firsts += is_first ? 1u : 0u;
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
            const uint32_t n = count[i];
            if (n == 0) no_edge++;
            longest = max(longest, n);
        }
    }
    (void)ni_prefix(no_run, &total);
    if (threadIdx.x == 0) tile_no_run[tile] = total;
    (void)ni_prefix(no_edge, &total);
    if (threadIdx.x == 0) tile_no_edge[tile] = total;
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((threadIdx.x & 31) == 0) atomicMax(&words[1], longest);
}

// Two blocks, of targets and of sources: the tile counts of their edges become exclusive prefix sums, those of the empty nodes go on behind.
__global__ void __launch_bounds__(1024)
ni_tiles_kernel(uint32_t* heads, uint32_t* firsts, int edge_tiles, uint32_t* no_run, uint32_t* no_edge, int node_tiles)
{
    chain_begin();
    __shared__ uint32_t warp_sums[32];
    uint32_t carry = 0;
    for (int list = 0; list < 2; list++) {
        uint32_t* const at = list == 0 ? (blockIdx.x == 0 ? heads : firsts) : (blockIdx.x == 0 ? no_run : no_edge);
        const int n = list == 0 ? edge_tiles : node_tiles;
        for (int base = 0; base < n; base += 4096) {
            const int i = base + 4 * (int)threadIdx.x;
            uint32_t v[4], own = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[k] = i + k < n ? at[i + k] : 0;
                own += v[k];
            }
            int total;
            uint32_t excl = (uint32_t)warp_excl_scan((int)own, threadIdx.x & 31, &total);
            __syncthreads();
            if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = (uint32_t)total;
            __syncthreads();
            int all;
            const int mine = warp_excl_scan((int)warp_sums[threadIdx.x & 31], threadIdx.x & 31, &all);
            excl += carry + (uint32_t)__shfl_sync(0xffffffffu, mine, threadIdx.x >> 5);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (i + k < n) at[i + k] = excl;
                excl += v[k];
            }
            carry += (uint32_t)all;
        }
    }
}

// rows, row_start, cols, places and counts of the sources in that order, from the bits.
__global__ void __launch_bounds__(NI_THREADS)
ni_rows_kernel(const int32_t* src32, const int64_t* dst, int64_t E, int64_t nt, int64_t ns, const uint32_t* run_of, const uint32_t* count,
               int edge_tiles, const uint32_t* head_bits, const uint32_t* first_bits, const uint32_t* tile_heads, const uint32_t* tile_firsts,
               const uint32_t* tile_no_run, const uint32_t* tile_no_edge, int32_t* rows, int32_t* row_start, int32_t* cols, int32_t* place,
               uint32_t* sorted_count)
{
    chain_begin();
    uint32_t total;
    if ((int)blockIdx.x < edge_tiles) {
        // a word of 32 edges each for the first threads of the block, 64 words a tile
        constexpr int WORDS = NI_TILE / 32;
        __shared__ uint32_t before_of[2][WORDS], bits_of[2][WORDS];
        const int64_t word0 = (int64_t)blockIdx.x * WORDS;
        const int t = threadIdx.x;
        const uint32_t hb = t < WORDS ? head_bits[word0 + t] : 0, fb = t < WORDS ? first_bits[word0 + t] : 0;
        const uint32_t both = ni_prefix((uint32_t)__popc(hb) | (uint32_t)__popc(fb) << 16, &total);
        if (t < WORDS) {
            before_of[0][t] = tile_heads[blockIdx.x] + (both & 0xffffu);
            before_of[1][t] = tile_firsts[blockIdx.x] + (both >> 16);
            bits_of[0][t] = hb;
            bits_of[1][t] = fb;
        }
        __syncthreads();
        const uint32_t lower = lanemask_lt();
        for (int w = t >> 5; w < WORDS; w += NI_THREADS / 32) {
            const uint32_t bit = 1u << (t & 31);
            const int64_t e = (word0 + w) * 32 + (t & 31);
            if (bits_of[0][w] & bit) {
                const uint32_t r = before_of[0][w] + __popc(bits_of[0][w] & lower);
                if (r < nt) {
                    rows[r] = (int32_t)dst[e];
                    row_start[r] = (int32_t)e;
                }
            }
            if (bits_of[1][w] & bit) {
                const uint32_t c = before_of[1][w] + __popc(bits_of[1][w] & lower);
                const int32_t s = src32[e];
                if (c < ns) {
                    cols[c] = s;
                    place[s] = (int32_t)c;
                    sorted_count[c] = count[s];
                }
            }
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
ni_words_kernel(const uint4* words, uint4* host)
{
    chain_begin();
    host[0] = words[0];
}

// Edges and their targets to the places of their sources' lists, in the order of their numbers there.
__global__ void __launch_bounds__(NI_THREADS)
ni_place_kernel(const int32_t* src32, const int32_t* number, const int64_t* dst, int64_t E, const int32_t* place, const int32_t* col_start, uint2* out)
{
    chain_begin();
    const int64_t base = (int64_t)blockIdx.x * NI_TILE + threadIdx.x;
    int32_t s[NI_ITEMS], at[NI_ITEMS];
    uint32_t t[NI_ITEMS];
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) {
        const int64_t e = base + k * NI_THREADS;
        s[k] = e < E ? src32[e] : -1;
        at[k] = e < E ? number[e] : 0;
        t[k] = e < E ? (uint32_t)dst[e] : 0;
    }
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++) s[k] = s[k] >= 0 ? place[s[k]] : -1;
#pragma unroll
    for (int k = 0; k < NI_ITEMS; k++)
        if (s[k] >= 0) out[col_start[s[k]] + at[k]] = make_uint2((uint32_t)(base + k * NI_THREADS), t[k]);
}

// A warp sorts a list by edge: the place of an edge is the number of smaller ones, which go round the lanes.  R: edges a lane.
constexpr int NI_LONGEST = 256;
template <int R>
__device__ __forceinline__ void ni_sort_list(const uint2* in, int n, int lane, int32_t* in_edge, int32_t* in_dst)
{
    uint32_t e[R], t[R];
    int at[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        const uint2 v = k * 32 + lane < n ? in[k * 32 + lane] : make_uint2(0xffffffffu, 0);
        e[k] = v.x;
        t[k] = v.y;
        at[k] = 0;
    }
#pragma unroll
    for (int j = 0; j < R; j++) {
        const int have = min(n - j * 32, 32);
#pragma unroll 4
        for (int l = 0; l < have; l++) {
            const uint32_t other = __shfl_sync(0xffffffffu, e[j], l);
#pragma unroll
            for (int k = 0; k < R; k++) at[k] += other < e[k] ? 1 : 0;
        }
    }
#pragma unroll
    for (int k = 0; k < R; k++)
        if (k * 32 + lane < n) {
            in_edge[at[k]] = (int32_t)e[k];
            in_dst[at[k]] = (int32_t)t[k];
        }
}
__global__ void __launch_bounds__(NI_THREADS)
ni_sort_kernel(const uint2* in, const int32_t* col_start, int64_t ns, int32_t* in_edge, int32_t* in_dst)
{
    chain_begin();
    const int lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * (NI_THREADS / 32) + (threadIdx.x >> 5);
    if (c >= ns) return;
    const int32_t begin = col_start[c];
    const int n = col_start[c + 1] - begin;
    if (n <= 0) return;
    if (n <= 32) ni_sort_list<1>(in + begin, n, lane, in_edge + begin, in_dst + begin);
    else if (n <= 64) ni_sort_list<2>(in + begin, n, lane, in_edge + begin, in_dst + begin);
    else if (n <= 128) ni_sort_list<4>(in + begin, n, lane, in_edge + begin, in_dst + begin);
    else ni_sort_list<8>(in + begin, n, lane, in_edge + begin, in_dst + begin);
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

extern "C" int dynb_neighbor_index_workspace_bytes(int64_t n_edges, int64_t n_targets, int64_t n_sources, int64_t longest, int64_t* bytes)
{
    if (bytes == nullptr) return fail_arg("null pointer");
    const int rc = ni_check(n_edges, n_targets, n_sources);
    if (rc != DYNB_OK) return rc;
    int64_t sort;
    const int rs = dynb_radix_sort_workspace_bytes(n_edges, &sort);
    if (rs != DYNB_OK) return rs;
    const NiLayout l = ni_layout(n_edges, n_targets, n_sources);
    *bytes = longest <= NI_LONGEST ? l.total_fill : l.total_sort + align_up(sort, 256);
    return DYNB_OK;
}

extern "C" int dynb_neighbor_index_plan(const int64_t* src_dev, const int64_t* dst_dev, int64_t n_edges, int64_t n_targets, int64_t n_sources,
                                        int32_t* rows_dev, int32_t* row_start_dev, int32_t* src32_dev, int32_t* cols_dev,
                                        int32_t* col_start_dev, int32_t* in_edge_dev, int64_t* words_host, void* workspace_dev,
                                        int64_t workspace_bytes, void* stream)
{
    const int rc = ni_check(n_edges, n_targets, n_sources);
    if (rc != DYNB_OK) return rc;
    if (row_start_dev == nullptr || col_start_dev == nullptr || workspace_dev == nullptr || words_host == nullptr) return fail_arg("null pointer");
    if ((n_edges > 0 && (!src_dev || !dst_dev || !src32_dev || !in_edge_dev)) || (n_targets > 0 && !rows_dev) || (n_sources > 0 && !cols_dev))
        return fail_arg("null pointer");
    if (!starts_on(workspace_dev, 16)) return fail_arg("neighbor_index: the workspace must start on a 16-byte boundary");
    const NiLayout l = ni_layout(n_edges, n_targets, n_sources);
    if (workspace_bytes < l.total) return fail_arg("workspace too small");
    void* const words_at = device_view_of_host(words_host);
    if (words_at == nullptr) return fail_arg("neighbor_index: words_host must be pinned, on a 16-byte boundary");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    uint32_t* const run_of = reinterpret_cast<uint32_t*>(ws + l.run_of);
    uint32_t* const count = reinterpret_cast<uint32_t*>(ws + l.count);
    uint32_t* const first = reinterpret_cast<uint32_t*>(ws + l.first);
    int32_t* const place = reinterpret_cast<int32_t*>(ws + l.place);
    uint32_t* const sorted_count = reinterpret_cast<uint32_t*>(ws + l.sorted_count);
    uint32_t* const head_bits = reinterpret_cast<uint32_t*>(ws + l.bits);
    uint32_t* const first_bits = head_bits + l.edge_tiles * (NI_TILE / 32);
    uint32_t* const heads = reinterpret_cast<uint32_t*>(ws + l.tiles);
    uint32_t* const firsts = heads + l.edge_tiles;
    uint32_t* const no_run = firsts + l.edge_tiles;
    uint32_t* const no_edge = no_run + l.node_tiles;
    uint32_t* const words = reinterpret_cast<uint32_t*>(ws + l.words);
    const int et = (int)l.edge_tiles, nt = (int)l.node_tiles;
    DYNB_CUDA_OK(clear_ranges(s, {run_of, 4 * n_targets, 0}, {count, 4 * n_sources, 0}, {first, 4 * n_sources, 0xff}, {words, 64, 0}));
    DYNB_CUDA_OK(launch_chained(ni_mark_kernel, et, NI_THREADS, 0, s, src_dev, dst_dev, n_edges, n_targets, n_sources, run_of, count, first,
                                src32_dev, in_edge_dev, head_bits, heads, words));
    DYNB_CUDA_OK(launch_chained(ni_count_kernel, et + nt, NI_THREADS, 0, s, src32_dev, n_edges, n_targets, n_sources, run_of, count, first, et,
                                first_bits, firsts, no_run, no_edge, words));
    DYNB_CUDA_OK(launch_chained(ni_tiles_kernel, 2, 1024, 0, s, heads, firsts, et, no_run, no_edge, nt));
    DYNB_CUDA_OK(launch_chained(ni_rows_kernel, et + nt, NI_THREADS, 0, s, src32_dev, dst_dev, n_edges, n_targets, n_sources, run_of, count,
                                et, head_bits, first_bits, heads, firsts, no_run, no_edge, rows_dev, row_start_dev, cols_dev, place, sorted_count));
    const bool publish = scan_publishes(n_sources + 1);
    DYNB_CUDA_OK(exclusive_scan(sorted_count, reinterpret_cast<uint32_t*>(col_start_dev), nullptr, n_sources + 1, reinterpret_cast<uint32_t*>(ws + l.scan),
                                reinterpret_cast<uint32_t*>(words) + 2, s,
                                publish ? ScanPublish{reinterpret_cast<const uint4*>(words), static_cast<uint4*>(words_at), true} : ScanPublish{}));
    if (!publish)
        DYNB_CUDA_OK(launch_chained(ni_words_kernel, 1, 1, 0, s, reinterpret_cast<const uint4*>(words), static_cast<uint4*>(words_at)));
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
    if (!starts_on(workspace_dev, 16)) return fail_arg("neighbor_index: the workspace must start on a 16-byte boundary");
    const NiLayout l = ni_layout(n_edges, n_targets, n_sources);
    int64_t sort;
    (void)dynb_radix_sort_workspace_bytes(n_edges, &sort);
    if (workspace_bytes < (longest <= NI_LONGEST ? l.total_fill : l.total_sort + sort)) return fail_arg("workspace too small");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace_dev);
    const int32_t* const place = reinterpret_cast<const int32_t*>(ws + l.place);
    if (longest <= NI_LONGEST) {
        uint2* const pairs = reinterpret_cast<uint2*>(ws + l.keys);
        DYNB_CUDA_OK(launch_chained(ni_place_kernel, (unsigned)l.edge_tiles, NI_THREADS, 0, s, src32_dev, in_edge_dev, dst_dev, n_edges, place, col_start_dev, pairs));
        DYNB_CUDA_OK(launch_chained(ni_sort_kernel, (unsigned)((n_sources + NI_THREADS / 32 - 1) / (NI_THREADS / 32)), NI_THREADS, 0, s, pairs, col_start_dev,
                                    n_sources, in_edge_dev, in_dst_dev));
        return DYNB_OK;
    }
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
