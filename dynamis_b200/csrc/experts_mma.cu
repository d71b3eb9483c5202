// The products by expert on the tensor cores.
//
// z = act(x W + b) and dx = du W^T, du = dz act'(u): tiles of 128 pairs of one expert by up to 256 columns (fp32: 128).  Eight warps gather the rows of x (or of dz, times
// the slope) into stages of 64 summed columns, one warp brings the matrix, one issues the products, four, eight or sixteen take the sums out of tensor memory, which holds two tiles, and
// apply offset and activation.  The matrices are laid out once per call as the multipliers read them (ex_pack_kernel: both products read them along the summed
// index, fp32 in its three parts), so that a piece of 64 summed columns is one copy of a run of bytes.  A matrix that fits beside four stages of rows (two in fp32 and with slopes) stays for
// all tiles of its expert; a larger one comes anew with every stage, from L2.
//
// dW = sum x^T du: a block takes a stretch of an expert's pairs, 128 x up to 256 elements of the matrix; both operands are the gathered rows as they
// are, read along their columns.  db is summed by threads from the stages as they stand in shared memory.
//
// fp32 operands are three bf16 parts, six of nine products (mma_parts.cuh).
//
// 300 k pairs of 64 experts in bf16: 512 x 256 101 us (4.6 TB/s), 256 x 512 with SiLU and its slopes 184 us (3.8 TB/s), dx 242 us (5.1 TB/s, du for the weights' pass among it), dW 152 us.
// 200 k pairs of 16 experts in fp32, 512 x 128: 163, 163 and 216 us (0.58, 0.58 and 0.44 of the six products' time).  In 16 bits the rows' passes are bound by the latency of gathered
// rows and what they write, in fp32 by the chain of a stage from memory through the conversion to the multipliers.  Tiles of 64 x 64 with fused multiply-adds took
// 4549 us for the first, 14 483 for the next three together and 5502 for the last three.

#include "experts.cuh"
#include "mma_parts.cuh"

namespace dynb {

// Warps that gather, and that store results.  An SM's four schedulers have room for five warps of 96 registers each, or four of 128: rows in fp32 wait in the registers of
// their threads and need the latter.
template <typename T> constexpr int EM_FEED = sizeof(T) == 4 ? 16 : 8;
constexpr int EM_COLUMNS = 16;                                       // columns that a warp takes out of tensor memory at a time
template <typename T> __host__ __device__ constexpr int em_threads(int out) { return (out + 2 + EM_FEED<T>) * 32; }
constexpr int EM_MAX_STAGES = 8;
constexpr int EM_SMEM = 220 * 1024;                                  // beside 4 KB of offsets and barriers
constexpr int EM_RAW = 3;                                            // stages of rows and slopes on their way beside those of the products

enum EmPath { EM_ASYNC, EM_REGISTERS, EM_SLOPE, EM_ASYNC_SLOPE };

struct EmPlan {
    int back, columns, column_stride, chunks, stages, tensor_columns, resident, b_bytes, stage_bytes, store, slope_store, smem;   // b_bytes: matrix of one stage
    const unsigned char* packed;
};

struct EmBars { uint64_t full[EM_MAX_STAGES], empty[EM_MAX_STAGES], b_full[EM_MAX_STAGES], panel_full, panel_free, sums_full[2], sums_free[2]; uint32_t tensor; };

__device__ __forceinline__ void bulk_expect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(to)), "l"(from), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}
// 16 bytes, zeros where `live` is false (nothing is read then).
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
// The barrier gets this thread's arrival when all its copies so far are there.  What they wrote is made visible to the tensor cores by the thread that waits.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory"); }
__device__ __forceinline__ void load_16(uint32_t from, uint4& v)
{
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last `left` groups of this thread have arrived.
__device__ __forceinline__ void copies_wait(int left)
{
    if (left >= 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Matrices in the order of the multipliers: [expert][tile of columns][64 summed columns][part][column][128 bytes, 16-byte pieces swizzled], zeros beyond the matrix.
// WIDE: rows of the matrix are read by 16 bytes; forward a thread turns a piece of 8 rows by that many columns round.  What is written lies side by side for 8 threads.
// (64 matrices of 512 x 256 bf16: 8.6 us, by single elements 12.7.)
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256)
ex_pack_kernel(const T* w, int64_t experts, int inner, int outer, int back, int columns, int tiles, int chunks, unsigned char* packed)
{
    constexpr int PARTS = TmParts<T>::N, N = 16 / (int)sizeof(T);
    const int kk = back ? outer : inner, nn = back ? inner : outer, group = WIDE && !back ? N : 1, groups = columns / group;
    const int64_t all = experts * tiles * chunks * groups * 8;
    for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < all; u += (int64_t)gridDim.x * blockDim.x) {
        const int64_t block = u / (groups * 8);
        const int inside = (int)(u - block * (groups * 8)), piece = inside % 8, n = inside / 8 * group;
        const int64_t run = block / chunks, e = run / tiles;
        const int chunk = (int)(block - run * chunks), tile = (int)(run - e * tiles);
        const int k = chunk * 64 + piece * 8, col = tile * columns + n;
        const int have = col < nn ? min(8, kk - k) : 0;
        const T* const from = w + e * inner * outer + (back ? (int64_t)col * outer + k : (int64_t)k * outer + col);
        unsigned char* const to = packed + block * ((int64_t)PARTS * columns * 128);
        TmRaw<T> v[N];
        if constexpr (WIDE) {
            if (!back) {
                uint4 row[8];
#pragma unroll
                for (int j = 0; j < 8; j++) row[j] = j < have ? __ldg(reinterpret_cast<const uint4*>(from + (int64_t)j * outer)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < 8; j++) reinterpret_cast<T*>(&v[i])[j] = reinterpret_cast<const T*>(&row[j])[i];
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const TmRaw<T> one[1] = {v[i]};
                    if (tm_odd(one)) tm_store<true>(v[i], to + tile_piece(n + i, piece), columns * 128);
                    else tm_store<false>(v[i], to + tile_piece(n + i, piece), columns * 128);
                }
                continue;
            }
        }
        v[0] = back && WIDE ? tm_load<true>(have > 0 ? from : w, 1, have) : tm_load<false>(have > 0 ? from : w, back ? 1 : outer, have);
        const TmRaw<T> one[1] = {v[0]};
        if (tm_odd(one)) tm_store<true>(v[0], to + tile_piece(n, piece), columns * 128);
        else tm_store<false>(v[0], to + tile_piece(n, piece), columns * 128);
    }
}

// The warps that gather by way of registers in fp32 are two teams, which take the stages by turns: what a warp does for a stage is one long chain (wait, conversion, stores,
// fence, addresses of the next), and while one team is in it the other is, too (200 k pairs 512 x 128: one team with two stages ahead 174 us, two teams 166, rows' pass).
template <typename T, EmPath PATH> constexpr int EM_TEAMS = sizeof(T) == 4 && PATH == EM_REGISTERS ? 2 : 1;

// Eight elements times their slopes.  In 16 bits the product is rounded to the type: it is an operand of the tensor cores, as a 16-bit gradient of a step by step
// program would be (two operands, rounded and rest, would double the products of dx and dW).
template <typename T>
__device__ __forceinline__ void em_times(TmRaw<T>& v, const TmRaw<T>& slope)
{
    if constexpr (sizeof(T) == 4) {
        uint32_t* const a = reinterpret_cast<uint32_t*>(&v);
        const uint32_t* const s = reinterpret_cast<const uint32_t*>(&slope);
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = __float_as_uint(__uint_as_float(a[i]) * __uint_as_float(s[i]));
    } else {
        uint32_t* const a = reinterpret_cast<uint32_t*>(&v);
        const uint32_t* const s = reinterpret_cast<const uint32_t*>(&slope);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 by = ex_slopes_of(s[i]);
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(a + i));
                const __half2 h = __floats2half2_rn(f.x * by.x, f.y * by.y);
                a[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(a[i] << 16) * by.x, __uint_as_float(a[i] & 0xffff0000u) * by.y);
                a[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
}

// Eight elements from p, where there are any (behind them, zeros are in memory); WIDE 2: fp32 on 32 bytes, by one load.
template <int WIDE, typename T>
__device__ __forceinline__ TmRaw<T> em_load(const T* p, int64_t step, int have)
{
    if constexpr (WIDE == 2) {
        TmRaw<T> r = {};
        if (have > 0)
            asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(r.v[0].x), "=r"(r.v[0].y), "=r"(r.v[0].z), "=r"(r.v[0].w), "=r"(r.v[1].x), "=r"(r.v[1].y), "=r"(r.v[1].z), "=r"(r.v[1].w)
                         : "l"(p));
        return r;
    } else {
        return tm_load<true>(p, step, have);
    }
}

// WORDS words of a row, the first `bytes` bytes of them real, in stores of 32 or 16 bytes or of elements of `size`.  Every lane stores its own row: a store of 32 bytes a lane fills
// whole sectors, and what goes through shared memory to lie side by side costs more steps than that saves (300 k pairs 256 x 512 bf16 with slopes: 250 against 227 us).
template <int WORDS>
__device__ __forceinline__ void em_put(unsigned char* to, const uint32_t (&w)[WORDS], int bytes, int store, int size)
{
    if (store == 32) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8)
            if (4 * i < bytes)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + 4 * i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                             "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                             : "memory");
    } else if (store == 16) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            if (4 * i < bytes) *reinterpret_cast<uint4*>(to + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else if (size == 4) {
#pragma unroll
        for (int i = 0; i < WORDS; i++)
            if (4 * i < bytes) reinterpret_cast<uint32_t*>(to)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 2 * WORDS; i++)
            if (2 * i < bytes) reinterpret_cast<uint16_t*>(to)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
}

// The activation of a row's sums, and their slopes.
template <typename T, int ACTIVATION>
__device__ __forceinline__ void em_activate(uint32_t (&bits)[EM_COLUMNS], uint32_t (&slopes)[EM_COLUMNS * sizeof(T) / 4])
{
#pragma unroll
    for (int i = 0; i < EM_COLUMNS; i += 2) {
        float s0, s1;
        const float v0 = ex_activate<ACTIVATION>(__uint_as_float(bits[i]), &s0), v1 = ex_activate<ACTIVATION>(__uint_as_float(bits[i + 1]), &s1);
        bits[i] = __float_as_uint(v0);
        bits[i + 1] = __float_as_uint(v1);
        if constexpr (sizeof(T) == 4) {
            slopes[i] = __float_as_uint(s0);
            slopes[i + 1] = __float_as_uint(s1);
        } else {
            slopes[i / 2] = ex_slopes_bits(s0, s1);
        }
    }
}

// Rows are read by pieces of 8 elements on 16 bytes, with WIDE 2 in fp32 on 32.  O: type of the results (fp32 for gradients that are summed over the choices before they are rounded).
template <typename T, typename O, EmPath PATH, int WIDE, int OUT>
__global__ void __launch_bounds__(em_threads<T>(OUT), 1)
em_rows_kernel(const ExArgs e, const EmPlan plan)
{
    constexpr int PARTS = TmParts<T>::N, A_BYTES = PARTS * TM_ROWS * 128, SIZE = (int)sizeof(O), COLUMNS = EM_COLUMNS, WORDS = COLUMNS * SIZE / 4;   // columns that a warp takes at a time
    constexpr int SHARES = OUT / 4, FEED = EM_FEED<T>;
    constexpr int TEAMS = EM_TEAMS<T, PATH>, TEAM = FEED / TEAMS;
    const TlArgs& a = e.t;
    extern __shared__ unsigned char raw_smem[];
    __shared__ EmBars bars;
    __shared__ __align__(16) float offsets[OUT][256 / SHARES];
    unsigned char* const panel = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    unsigned char* const stage0 = panel + (plan.resident ? plan.chunks * plan.b_bytes : 0);
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int kk = plan.back ? a.outer : a.inner, nn = plan.back ? a.inner : a.outer;
    const int col0 = blockIdx.y * plan.columns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; s++) {
            bar_init(&bars.full[s], PATH == EM_ASYNC ? FEED * 32 : TEAM);
            bar_init(&bars.empty[s], 1);
            bar_init(&bars.b_full[s], 1);
        }
        bar_init(&bars.panel_full, 1);
        bar_init(&bars.panel_free, 1);
        for (int b = 0; b < 2; b++) {
            bar_init(&bars.sums_full[b], 1);
            bar_init(&bars.sums_free[b], OUT);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tensor_alloc(&bars.tensor, plan.tensor_columns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = bars.tensor;

    int64_t pieces = 0;
    (void)tl_tile(a, INT64_MAX, TM_ROWS, &pieces);
    const int64_t per = (pieces + gridDim.x - 1) / gridDim.x, first = blockIdx.x * per;
    TmCursor cursor;
    cursor.start(a, first, min(per, pieces - first));

    if (warp < OUT) {
        // sums to results: the warps of the rows 32 (warp % 4) on take the groups of columns in turn
        unsigned char* const out = static_cast<unsigned char*>(plan.back ? a.dx : a.y);
        const int have = min(plan.columns, nn - col0), share = warp >> 2;
        const bool with_offset = !plan.back && a.b != nullptr;
        const int activation = plan.back ? DYNB_ACTIVATION_NONE : e.activation;
        const bool with_slope = activation != DYNB_ACTIVATION_NONE && e.slope != nullptr;
        ex_clear_absent(a, out, e.out_row * SIZE, plan.store >= 16 ? 16 : 2, ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * OUT + warp, (int64_t)gridDim.x * gridDim.y * OUT);
        float* const offset = offsets[warp];
        int buffer = 0, offset_type = -1;
        uint32_t phase = 0;
        for (; cursor.tile.type >= 0; cursor.next(a)) {
            const int64_t place = cursor.tile.begin + (warp & 3) * 32 + lane;
            int32_t r = place < cursor.tile.end ? __ldg(a.order + place) : -1;
            if (with_offset && cursor.tile.type != offset_type) {
                offset_type = cursor.tile.type;
                __syncwarp();
                for (int i = lane; i < (have + SHARES * COLUMNS - 1) / (SHARES * COLUMNS) * COLUMNS; i += 32) {   // of this warp's columns, one group behind the other
                    const int c = i / COLUMNS * SHARES * COLUMNS + share * COLUMNS + i % COLUMNS;
                    offset[i] = c < have ? tl_get(static_cast<const T*>(a.b) + (int64_t)offset_type * a.outer + col0 + c) : 0.0f;
                }
                __syncwarp();
            }
            if (!bar_wait(&bars.sums_full[buffer], phase)) { tm_ran_out(a); break; }
            tensor_fence_after();
            if ((uint32_t)r >= (uint64_t)a.n) r = -1;
            const uint32_t from = tensor + ((uint32_t)((warp & 3) * 32) << 16) + buffer * plan.column_stride;
            for (int c = share * COLUMNS; c < have; c += SHARES * COLUMNS) {
                uint32_t bits[COLUMNS];
                __syncwarp();
                tensor_load(from + c, bits);
                if constexpr (PARTS > 1) {   // the small products' sums
                    uint32_t small[COLUMNS];
                    tensor_load(from + 2 * plan.column_stride + c, small);
                    tensor_wait_loads();
#pragma unroll
                    for (int i = 0; i < COLUMNS; i++) bits[i] = __float_as_uint(__uint_as_float(bits[i]) + __uint_as_float(small[i]));
                } else {
                    tensor_wait_loads();
                }
                if (with_offset) {
#pragma unroll
                    for (int i = 0; i < COLUMNS; i += 4) {
                        const float4 o = *reinterpret_cast<const float4*>(offset + c / (SHARES * COLUMNS) * COLUMNS + i);
                        bits[i] = __float_as_uint(__uint_as_float(bits[i]) + o.x);
                        bits[i + 1] = __float_as_uint(__uint_as_float(bits[i + 1]) + o.y);
                        bits[i + 2] = __float_as_uint(__uint_as_float(bits[i + 2]) + o.z);
                        bits[i + 3] = __float_as_uint(__uint_as_float(bits[i + 3]) + o.w);
                    }
                }
                uint32_t words[WORDS], slopes[COLUMNS * sizeof(T) / 4];
                if constexpr (std::is_same<T, O>::value) {   // one choice for all elements: with one at each, they wait for one another (300 k pairs 256 x 512 with slopes: 421 in place of 250 us)
                    if (activation == DYNB_ACTIVATION_SILU) em_activate<T, DYNB_ACTIVATION_SILU>(bits, slopes);
                    else if (activation == DYNB_ACTIVATION_GELU) em_activate<T, DYNB_ACTIVATION_GELU>(bits, slopes);
                }
#pragma unroll
                for (int i = 0; i < COLUMNS; i += 4) {
                    const float v[4] = {__uint_as_float(bits[i]), __uint_as_float(bits[i + 1]), __uint_as_float(bits[i + 2]), __uint_as_float(bits[i + 3])};
                    tm_words<O>(v, words + i * SIZE / 4);
                }
                if (r < 0) continue;
                em_put(out + (r * e.out_row + col0 + c) * SIZE, words, (have - c) * SIZE, plan.store, SIZE);
                if (with_slope) em_put(static_cast<unsigned char*>(e.slope) + (r * e.out_row + col0 + c) * SIZE, slopes, (have - c) * SIZE, plan.slope_store, SIZE);
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars.sums_free[buffer]);
            buffer ^= 1;
            if (buffer == 0) phase ^= 1;
        }
    } else if (warp == OUT) {
        // products
        const bool bf16 = !std::is_same<T, __half>::value;
        const uint32_t what = mma_what(bf16, plan.columns, false, false);
        const int b_part = plan.columns * 128 / 16;
        int stage = 0, buffer = 0, panel_type = -1;
        uint32_t phase = 0, panel_phase = 0, sums_phase = 1;
        bool ok = true;
        while (ok && cursor.tile.type >= 0) {
            if (plan.resident && cursor.tile.type != panel_type) {
                if (!bar_wait(&bars.panel_full, panel_phase)) { ok = false; break; }
                panel_phase ^= 1;
                panel_type = cursor.tile.type;
            }
            if (!bar_wait(&bars.sums_free[buffer], sums_phase)) { ok = false; break; }
            tensor_fence_after();
            const uint32_t sums = tensor + buffer * plan.column_stride;
            for (int chunk = 0; chunk < plan.chunks; chunk++) {
                if (!bar_wait(&bars.full[stage], phase)) { ok = false; break; }
                if constexpr (PATH == EM_ASYNC) fence_to_tensor();
                if (!plan.resident && !bar_wait(&bars.b_full[stage], phase)) { ok = false; break; }
                tensor_fence_after();
                if (elected()) {
                    const int steps = min(4, (kk - chunk * 64 + 15) / 16);
                    unsigned char* const at = stage0 + stage * plan.stage_bytes;
                    const uint64_t at_a = tile_descriptor(smem_addr(at), 16, 1024);
                    const uint64_t at_b = tile_descriptor(smem_addr(plan.resident ? panel + chunk * plan.b_bytes : at + A_BYTES), 16, 1024);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (k < steps) tm_step<PARTS>(sums, sums + 2 * plan.column_stride, at_a + 2 * k, TM_ROWS * 128 / 16, at_b + 2 * k, b_part, what, chunk > 0 || k > 0);
                    tensor_commit(&bars.empty[stage]);
                    if (chunk == plan.chunks - 1) tensor_commit(&bars.sums_full[buffer]);
                }
                __syncwarp();
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            cursor.next(a);
            if (plan.resident && cursor.tile.type >= 0 && cursor.tile.type != panel_type && elected()) tensor_commit(&bars.panel_free);
            __syncwarp();
            buffer ^= 1;
            if (buffer == 0) sums_phase ^= 1;
        }
        if (!ok) tm_ran_out(a);
    } else if (warp == OUT + 1) {
        // matrices
        const int64_t tiles = gridDim.y;
        if (plan.resident) {
            int panel_type = -1;
            uint32_t free_phase = 0, asked = 0;
            for (; cursor.tile.type >= 0; cursor.next(a)) {
                if (cursor.tile.type == panel_type) continue;
                if (panel_type >= 0) {
                    if (!bar_wait(&bars.panel_free, free_phase)) { tm_ran_out(a); break; }
                    free_phase ^= 1;
                }
                panel_type = cursor.tile.type;
                if (elected()) {
                    const unsigned char* const from = plan.packed + ((int64_t)panel_type * tiles + blockIdx.y) * plan.chunks * plan.b_bytes;
                    bulk_expect(&bars.panel_full, plan.chunks * plan.b_bytes);
                    for (int chunk = 0; chunk < plan.chunks; chunk++) bulk_copy(panel + chunk * plan.b_bytes, from + (int64_t)chunk * plan.b_bytes, plan.b_bytes, &bars.panel_full);
                }
                __syncwarp();
                asked++;
            }
            if (asked > 0) (void)bar_wait(&bars.panel_full, (asked - 1) & 1);   // a block does not end before its copies
        } else {
            int stage = 0;
            uint32_t phase = 1;
            int64_t asked = 0;
            bool ok = true;
            for (; ok && cursor.tile.type >= 0; cursor.next(a)) {
                const unsigned char* from = plan.packed + ((int64_t)cursor.tile.type * tiles + blockIdx.y) * plan.chunks * plan.b_bytes;
                for (int chunk = 0; chunk < plan.chunks; chunk++, from += plan.b_bytes) {
                    if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); ok = false; break; }
                    if (elected()) {
                        bulk_expect(&bars.b_full[stage], plan.b_bytes);
                        bulk_copy(stage0 + stage * plan.stage_bytes + A_BYTES, from, plan.b_bytes, &bars.b_full[stage]);
                    }
                    __syncwarp();
                    asked++;
                    if (++stage == plan.stages) { stage = 0; phase ^= 1; }
                }
            }
            // the last copy of every stage: number c of stage c % stages
            for (int64_t c = max(asked - plan.stages, (int64_t)0); c < asked; c++) (void)bar_wait(&bars.b_full[c % plan.stages], (uint32_t)(c / plan.stages) & 1);
        }
    } else {
        // rows to shared memory
        const T* const in = static_cast<const T*>(plan.back ? a.dy : a.x);
        const int64_t in_row = plan.back ? a.dy_row : a.x_row;
        const int fan = plan.back ? 1 : e.fan;
        const uint32_t rows_in = (uint32_t)(plan.back ? a.n : e.n_in);
        constexpr int UNITS = TM_ROWS * 8 / (TEAM * 32);
        const int team = (warp - OUT - 2) / TEAM, tid = threadIdx.x - (OUT + 2 + team * TEAM) * 32, piece = tid & 7;
        int32_t rows[UNITS], rows_next[UNITS];      // of the next tile to ask for, and the one behind it
        auto rows_of = [&](const TlTile& t, int32_t (&r)[UNITS]) {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int64_t place = t.begin + (tid >> 3) + (TEAM * 4) * i;
                r[i] = t.type >= 0 && place < t.end ? __ldg(a.order + place) : -1;   // looked at a tile later
            }
        };
        // the pair's row, or a number that is no row
        auto row_in = [&](int32_t p) { return (uint32_t)p >= (uint64_t)a.n ? 0xffffffffu : fan == 1 ? (uint32_t)p : (uint32_t)p / (uint32_t)fan; };
        int stage = 0;
        uint32_t phase = 1;
        if constexpr (PATH == EM_ASYNC) {
            rows_of(cursor.tile, rows);
            bool ok = true;
            while (ok && cursor.tile.type >= 0) {
                uint32_t at[UNITS];
#pragma unroll
                for (int i = 0; i < UNITS; i++) at[i] = row_in(rows[i]);
                cursor.next(a);
                rows_of(cursor.tile, rows);
                for (int chunk = 0; chunk < plan.chunks; chunk++) {
                    if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); ok = false; break; }
                    const uint32_t to = smem_addr(stage0) + stage * plan.stage_bytes + tile_piece(tid >> 3, piece);   // TEAM * 4 rows on: the same place among eight
                    const int k = chunk * 64 + piece * 8;
#pragma unroll
                    for (int i = 0; i < UNITS; i++) {
                        const bool live = at[i] < rows_in && k < kk;
                        copy_16(to + i * TEAM * 512, in + (live ? at[i] * in_row + k : 0), live);
                    }
                    copies_arrive(&bars.full[stage]);
                    if (++stage == plan.stages) { stage = 0; phase ^= 1; }
                }
            }
            copies_commit();
            copies_wait(0);
        } else if constexpr (PATH == EM_ASYNC_SLOPE) {
            // Rows and slopes come to places that are this thread's own, EM_RAW stages of them, and go from there, multiplied, to the stages of the products
            const uint32_t raw = smem_addr(stage0) + plan.stages * plan.stage_bytes + tid * 16;
            constexpr uint32_t UNIT = TEAM * 512, SLOT = 2 * UNITS * UNIT;
            const bool keep_du = e.du != nullptr && blockIdx.y == 0;
            TmCursor behind = cursor;               // of the stage that is multiplied, for du
            int chunk = 0, behind_chunk = 0, slot = 0, behind_slot = 0;
            int32_t behind_rows[UNITS];
            if (keep_du) rows_of(behind.tile, behind_rows);
            rows_of(cursor.tile, rows);
            uint32_t at[UNITS];
            int64_t left = 0;                       // stages asked for and not yet multiplied
            auto ask = [&] {
                if (chunk == 0 && cursor.tile.type >= 0) {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) at[i] = row_in(rows[i]);
                }
                if (cursor.tile.type >= 0) {
                    const int k = chunk * 64 + piece * 8;
#pragma unroll
                    for (int i = 0; i < UNITS; i++) {
                        const bool ok = at[i] < rows_in && k < kk;
                        copy_16(raw + slot * SLOT + i * UNIT, in + (ok ? at[i] * in_row + k : 0), ok);
                        copy_16(raw + slot * SLOT + (UNITS + i) * UNIT, static_cast<const T*>(e.slope) + (ok ? (int64_t)at[i] * kk + k : 0), ok);
                    }
                    left++;
                    if (++slot == EM_RAW) slot = 0;
                    if (++chunk == plan.chunks) {
                        chunk = 0;
                        cursor.next(a);
                        rows_of(cursor.tile, rows);
                    }
                }
                copies_commit();                    // an empty group behind the last stage: the number of those under way stays the same
            };
#pragma unroll
            for (int i = 0; i < EM_RAW - 1; i++) ask();
            while (left > 0) {
                ask();
                copies_wait(EM_RAW - 1);
                TmRaw<T> v[UNITS];
#pragma unroll
                for (int i = 0; i < UNITS; i++) {
                    TmRaw<T> slope;
                    load_16(raw + behind_slot * SLOT + i * UNIT, v[i].v[0]);
                    load_16(raw + behind_slot * SLOT + (UNITS + i) * UNIT, slope.v[0]);
                    em_times(v[i], slope);
                    const int k = behind_chunk * 64 + piece * 8;
                    if (keep_du && (uint32_t)behind_rows[i] < rows_in && k < kk) *reinterpret_cast<uint4*>(static_cast<T*>(e.du) + (int64_t)behind_rows[i] * kk + k) = v[i].v[0];
                }
                if (++behind_slot == EM_RAW) behind_slot = 0;
                if (keep_du && ++behind_chunk == plan.chunks) {
                    behind_chunk = 0;
                    behind.next(a);
                    rows_of(behind.tile, behind_rows);
                }
                left--;
                if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); break; }
                unsigned char* const to = stage0 + stage * plan.stage_bytes + tile_piece(tid >> 3, piece);
#pragma unroll
                for (int i = 0; i < UNITS; i++) *reinterpret_cast<uint4*>(to + i * UNIT) = v[i].v[0];
                fence_to_tensor();
                __syncwarp();
                if (lane == 0) bar_arrive(&bars.full[stage]);
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
            }
            copies_wait(0);
        } else {
            constexpr int SLOPES = PATH == EM_SLOPE ? UNITS : 1;
            TlTile next = cursor.tile;
            int chunk = 0;
            TmRaw<T> v[UNITS], slope[SLOPES];       // of the next stage, under way
            bool more = false;
            uint32_t row_du[SLOPES];                // pair whose du is kept, or a number that is none; its first column
            int k_du = 0;
            const bool keep_du = PATH == EM_SLOPE && e.du != nullptr && blockIdx.y == 0;
            auto step = [&](int stages) {           // on to a stage behind the next
                for (int i = 0; i < stages && next.type >= 0; i++) {
                    if (++chunk < plan.chunks) continue;
                    chunk = 0;
                    next = cursor.tile;
#pragma unroll
                    for (int j = 0; j < UNITS; j++) rows[j] = rows_next[j];
                    if (next.type >= 0) {
                        cursor.next(a);
                        rows_of(cursor.tile, rows_next);
                    }
                }
            };
            auto ask = [&] {
                more = next.type >= 0;
                if (!more) return;
                const int k = chunk * 64 + piece * 8, have = min(8, kk - k);
                k_du = k;
#pragma unroll
                for (int i = 0; i < UNITS; i++) {
                    const uint32_t at = row_in(rows[i]);
                    const bool ok = at < rows_in;
                    if constexpr (PATH == EM_SLOPE) row_du[i] = keep_du && have > 0 ? at : 0xffffffffu;
                    v[i] = em_load<WIDE>(in + (ok ? at * in_row + k : 0), 1, ok ? have : 0);
                    if constexpr (PATH == EM_SLOPE) slope[i] = em_load<WIDE>(static_cast<const T*>(e.slope) + (ok ? (int64_t)at * kk + k : 0), 1, ok ? have : 0);
                }
                step(TEAMS);
            };
            rows_of(next, rows);
            if (next.type >= 0) cursor.next(a);
            rows_of(cursor.tile, rows_next);
            step(team);
            stage = team;
            ask();
            while (more) {
                if constexpr (PATH == EM_SLOPE) {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) {
                        em_times(v[i], slope[i]);
                        if (row_du[i] < rows_in) {
                            uint4* const to = reinterpret_cast<uint4*>(static_cast<T*>(e.du) + (int64_t)row_du[i] * kk + k_du);
#pragma unroll
                            for (int h = 0; h < (int)(sizeof(TmRaw<T>) / 16); h++) to[h] = v[i].v[h];
                        }
                    }
                }
                if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); break; }
                unsigned char* const to = stage0 + stage * plan.stage_bytes + tile_piece(tid >> 3, piece);
                if (tm_odd(v)) {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) tm_store<true>(v[i], to + i * TEAM * 512, TM_ROWS * 128);
                } else {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) tm_store<false>(v[i], to + i * TEAM * 512, TM_ROWS * 128);
                }
                fence_to_tensor();
                __syncwarp();
                if (lane == 0) bar_arrive(&bars.full[stage]);
                stage += TEAMS;
                if (stage >= plan.stages) { stage -= plan.stages; phase ^= 1; }
                ask();
            }
        }
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, plan.tensor_columns);
}

// ------------------------------------------------------------------------------------------------ gradients of the matrices
// Warps that store sums, issue products, sum up the offsets' gradient, and gather.
constexpr int EW_OUT = 4, EW_FEED = 16, EW_MAX_STAGES = 8;
template <typename T> constexpr int EW_SUM = sizeof(T) == 4 ? 2 : 4;
template <typename T> constexpr int EW_THREADS = (EW_OUT + 1 + EW_SUM<T> + EW_FEED) * 32;
template <typename T> constexpr int EW_ROWS = sizeof(T) == 4 ? 32 : 64;   // pairs of a stage
constexpr int EW_SMEM = 222 * 1024;

struct EwPlan { int64_t most; int columns, column_stride, x_blocks, y_blocks, row_tiles, column_tiles, stages, tensor_columns, store; };   // most: sums that there is room for
struct EwBars { uint64_t full[EW_MAX_STAGES], empty[EW_MAX_STAGES], sums_full[2], sums_free[2]; uint32_t tensor; };

// The pairs in the order of their experts are cut at multiples of `stretch` and where experts begin; a block takes the pieces of its slice one after the other.
struct EwCursor {
    int type;                       // -1 behind the last
    int64_t begin, end, end_of_type, end_of_slice, index;   // index: number of the piece among all

    __device__ __forceinline__ void cut(int stretch) { end = min(min(end_of_type, end_of_slice), (begin / stretch + 1) * stretch); }
    __device__ __forceinline__ void start(const TlArgs& a, int64_t first, int64_t last)   // all lanes of a warp
    {
        const int lane = threadIdx.x & 31;
        type = -1;
        end_of_slice = last;
        index = 0;
        begin = first;
        if (first >= last) return;
        for (int t0 = 0; t0 < a.types; t0 += 32) {
            int64_t s0 = 0, s1 = 0;
            if (t0 + lane < a.types) tl_rows_of(a, t0 + lane, &s0, &s1);
            const int mine = s1 > s0 ? (int)((s1 + a.stretch - 1) / a.stretch - s0 / a.stretch) : 0;
            int total;
            const int before = warp_excl_scan(mine, lane, &total);
            const uint32_t found = __ballot_sync(0xffffffffu, s0 <= first && first < s1);
            if (found != 0) {
                const int from = __ffs(found) - 1;
                type = t0 + from;
                end_of_type = __shfl_sync(0xffffffffu, s1, from);
                index += __shfl_sync(0xffffffffu, before, from) + first / a.stretch - __shfl_sync(0xffffffffu, s0, from) / a.stretch;
                cut(a.stretch);
                return;
            }
            index += total;
        }
    }
    __device__ __forceinline__ void next(const TlArgs& a)
    {
        begin = end;
        index++;
        if (begin >= end_of_slice) { type = -1; return; }
        while (begin >= end_of_type) {
            if (++type >= a.types) { type = -1; return; }
            int64_t s0;
            tl_rows_of(a, type, &s0, &end_of_type);
        }
        cut(a.stretch);
    }
};

template <typename T, EmPath PATH, int WIDE>
__global__ void __launch_bounds__(EW_THREADS<T>, 1)
em_weights_kernel(const ExArgs e, const EwPlan plan)
{
    constexpr int PARTS = TmParts<T>::N, TEAMS = EM_TEAMS<T, PATH>, TEAM = EW_FEED / TEAMS, FEED_THREADS = TEAM * 32, ROWS = EW_ROWS<T>, BLOCK = ROWS * 128;
    constexpr int SUMS = PARTS == 1 ? 1 : 2;    // sums of a buffer: leading parts, small ones
    constexpr int UNITS = PARTS == 1 ? 6 : 2 * TEAMS;   // pieces of 8 elements a thread and stage: 64 pairs x (128 + 256) elements, or 32 x (128 + 128)
    const TlArgs& a = e.t;
    extern __shared__ unsigned char raw_smem[];
    __shared__ EwBars bars;
    unsigned char* const stage0 = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    const int warp = warp_number(), lane = threadIdx.x & 31;
    // the tiles of a slice are neighbours: what they share comes from L2
    const int tiles = plan.row_tiles * plan.column_tiles, of_tile = blockIdx.x % tiles, slices = gridDim.x / tiles;
    const int row0 = of_tile / plan.column_tiles * TM_ROWS, col0 = of_tile % plan.column_tiles * plan.columns;
    const int blocks = plan.x_blocks + plan.y_blocks, stage_bytes = blocks * PARTS * BLOCK;
    const bool sums_wanted = row0 == 0 && a.db != nullptr;
    const int64_t cells = (int64_t)a.inner * a.outer;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; s++) {
            bar_init(&bars.full[s], PATH == EM_ASYNC ? EW_FEED * 32 : TEAM);
            bar_init(&bars.empty[s], sums_wanted ? 1 + EW_SUM<T> : 1);
        }
        for (int b = 0; b < 2; b++) {
            bar_init(&bars.sums_full[b], 1);
            bar_init(&bars.sums_free[b], EW_OUT);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tensor_alloc(&bars.tensor, plan.tensor_columns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = bars.tensor;
    const int64_t all = min(max((int64_t)a.start[a.types], (int64_t)0), a.n), pieces = (all + a.stretch - 1) / a.stretch;
    const int64_t slice = ((pieces + slices - 1) / slices) * a.stretch, first = min((int64_t)(blockIdx.x / tiles) * slice, all);
    EwCursor cursor;
    cursor.start(a, first, min(first + slice, all));

    if (warp < EW_OUT) {
        int buffer = 0;
        uint32_t phase = 0;
        const int m = row0 + threadIdx.x, have = min(plan.columns, a.outer - col0);
        for (; cursor.type >= 0; cursor.next(a)) {
            if (!bar_wait(&bars.sums_full[buffer], phase)) { tm_ran_out(a); break; }
            tensor_fence_after();
            unsigned char* const at = reinterpret_cast<unsigned char*>(a.partial + cursor.index * (cells + a.outer) + (int64_t)m * a.outer + col0);
            const uint32_t from = tensor + ((uint32_t)(warp * 32) << 16) + buffer * SUMS * plan.column_stride;
            for (int c = 0; c < have; c += 16) {
                uint32_t bits[16];
                __syncwarp();
                tensor_load(from + c, bits);
                if constexpr (PARTS > 1) {
                    uint32_t small[16];
                    tensor_load(from + plan.column_stride + c, small);
                    tensor_wait_loads();
#pragma unroll
                    for (int i = 0; i < 16; i++) bits[i] = __float_as_uint(__uint_as_float(bits[i]) + __uint_as_float(small[i]));
                } else {
                    tensor_wait_loads();
                }
                if (m < a.inner && cursor.index < plan.most) em_put(at + 4 * c, bits, 4 * (have - c), plan.store, 4);
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars.sums_free[buffer]);
            buffer ^= 1;
            if (buffer == 0) phase ^= 1;
        }
    } else if (warp == EW_OUT) {
        const bool bf16 = !std::is_same<T, __half>::value;
        const uint32_t what = mma_what(bf16, plan.columns, true, true);
        const uint32_t stage_at = smem_addr(stage0);
        const uint32_t lead = PARTS * BLOCK, lead_x = plan.x_blocks > 1 ? lead : 0;   // one block: the upper 64 rows repeat the lower
        int stage = 0, buffer = 0;
        uint32_t phase = 0, sums_phase = 1;
        bool ok = true;
        for (; ok && cursor.type >= 0; cursor.next(a)) {
            const int steps = (int)((cursor.end - cursor.begin + ROWS - 1) / ROWS);
            if (!bar_wait(&bars.sums_free[buffer], sums_phase)) { ok = false; break; }
            tensor_fence_after();
            const uint32_t sums = tensor + buffer * SUMS * plan.column_stride;
            for (int step = 0; step < steps; step++) {
                if (!bar_wait(&bars.full[stage], phase)) { ok = false; break; }
                if constexpr (PATH == EM_ASYNC) fence_to_tensor();
                tensor_fence_after();
                if (elected()) {
                    const uint32_t at = stage_at + stage * stage_bytes;
                    const uint64_t at_x = tile_descriptor(at, lead_x, 1024), at_y = tile_descriptor(at + plan.x_blocks * PARTS * BLOCK, lead, 1024);
#pragma unroll
                    for (int k = 0; k < ROWS / 16; k++) tm_step<PARTS>(sums, sums + plan.column_stride, at_x + k * 128, BLOCK / 16, at_y + k * 128, BLOCK / 16, what, step > 0 || k > 0);
                    tensor_commit(&bars.empty[stage]);
                    if (step == steps - 1) tensor_commit(&bars.sums_full[buffer]);
                }
                __syncwarp();
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
            }
            buffer ^= 1;
            if (buffer == 0) sums_phase ^= 1;
        }
        if (!ok) tm_ran_out(a);
    } else if (warp < EW_OUT + 1 + EW_SUM<T>) {
        // the offsets' gradient: a thread sums two columns of the stages as they stand in shared memory, all parts
        if (sums_wanted) {
            const int c = (threadIdx.x - (EW_OUT + 1) * 32) * 2, have = min(plan.columns, a.outer - col0);
            const uint32_t at = smem_addr(stage0) + (plan.x_blocks + c / 64) * PARTS * BLOCK + (c & 7) * 2;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (; ok && cursor.type >= 0; cursor.next(a)) {
                const int steps = (int)((cursor.end - cursor.begin + ROWS - 1) / ROWS);
                float lo = 0.0f, hi = 0.0f;
                for (int step = 0; step < steps; step++) {
                    if (!bar_wait(&bars.full[stage], phase)) { tm_ran_out(a); ok = false; break; }
                    if (c < plan.columns) {
                        float l = 0.0f, h = 0.0f;
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll 16
                            for (int r = 0; r < ROWS; r++) {
                                uint32_t v;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at + stage * stage_bytes + p * BLOCK + tile_piece(r, (c >> 3) & 7)));
                                if constexpr (std::is_same<T, __half>::value) {
                                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
                                    l += f.x;
                                    h += f.y;
                                } else {
                                    l += __uint_as_float(v << 16);
                                    h += __uint_as_float(v & 0xffff0000u);
                                }
                            }
                        lo += l;
                        hi += h;
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(&bars.empty[stage]);
                    if (++stage == plan.stages) { stage = 0; phase ^= 1; }
                }
                float* const to = a.partial + cursor.index * (cells + a.outer) + cells + col0 + c;
                if (ok && c < have && cursor.index < plan.most) to[0] = lo;
                if (ok && c + 1 < have && cursor.index < plan.most) to[1] = hi;
            }
        }
    } else {
        // a thread takes pieces of one pair's rows, piece `piece` of every block (of every other one): number, division and addresses of the pair are its own, once a stage
        constexpr int GROUPS = FEED_THREADS / (ROWS * 8);
        const int team = (warp - EW_OUT - 1 - EW_SUM<T>) / TEAM, tid = threadIdx.x - (EW_OUT + 1 + EW_SUM<T> + team * TEAM) * 32, piece = tid & 7, group = (tid >> 3) % GROUPS, r = tid / (8 * GROUPS);
        const int at0 = group * PARTS * BLOCK + (int)tile_piece(r, piece), y_limit = min(a.outer, col0 + plan.columns);
        // the pair of the next stage
        int64_t place = cursor.begin;
        auto step = [&](int stages) {
            for (int i = 0; i < stages && cursor.type >= 0; i++) {
                place += ROWS;
                if (place < cursor.end) continue;
                cursor.next(a);
                place = cursor.begin;
            }
        };
        auto row_of = [&](int32_t& p) {
            p = cursor.type >= 0 && place + r < cursor.end ? __ldg(a.order + place + r) : -1;   // looked at a stage later
            if (cursor.type < 0) return false;
            step(TEAMS);
            return true;
        };
        // f(unit, address, elements there are) for every unit of pair p
        auto units_of = [&](int32_t p, auto&& f) {
            const bool live = (uint32_t)p < (uint64_t)a.n;
            const T* const x = static_cast<const T*>(a.x) + (live ? (int64_t)(e.fan == 1 ? (uint32_t)p : (uint32_t)p / (uint32_t)e.fan) * a.x_row : 0);
            const T* const y = static_cast<const T*>(a.dy) + (live ? p * a.dy_row : 0);
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int block = i * GROUPS + group;
                if (block >= blocks) continue;
                const bool of_y = block >= plan.x_blocks;
                const int c = (of_y ? col0 + (block - plan.x_blocks) * 64 : row0 + block * 64) + piece * 8, have = live ? min(8, (of_y ? y_limit : a.inner) - c) : 0;
                f(i, (of_y ? y : x) + (have > 0 ? c : 0), have);
            }
        };
        int32_t id;
        int stage = team;
        uint32_t phase = 1;
        step(team);
        bool more = row_of(id);
        if constexpr (PATH == EM_ASYNC) {
            auto ask = [&](int32_t p) {
                if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); return false; }
                const uint32_t to = smem_addr(stage0) + stage * stage_bytes + at0;
                units_of(p, [&](int i, const T* from, int have) { copy_16(to + i * GROUPS * BLOCK, from, have > 0); });
                copies_arrive(&bars.full[stage]);
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
                return true;
            };
            // numbers of two stages by turns, each asked for two stages ahead (copied from one place to another they would be waited for at once)
            int32_t other_id;
            bool other = row_of(other_id);
            while (more) {
                if (!ask(id)) break;
                more = row_of(id);
                if (!other || !ask(other_id)) break;
                other = row_of(other_id);
            }
            copies_commit();
            copies_wait(0);
        } else {
            // the rows of the next stage are under way in registers, the number of the pair behind it
            TmRaw<T> v[UNITS] = {};
            bool live = false;
            auto fetch = [&] {
                units_of(id, [&](int i, const T* from, int have) { v[i] = em_load<WIDE>(from, 1, have); });
                live = more;
                more = row_of(id);
            };
            fetch();
            while (live) {
                if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); break; }
                unsigned char* const to = stage0 + stage * stage_bytes + at0;
                if (tm_odd(v)) {
#pragma unroll
                    for (int i = 0; i < UNITS; i++)
                        if (i * GROUPS + group < blocks) tm_store<true>(v[i], to + i * GROUPS * PARTS * BLOCK, BLOCK);
                } else {
#pragma unroll
                    for (int i = 0; i < UNITS; i++)
                        if (i * GROUPS + group < blocks) tm_store<false>(v[i], to + i * GROUPS * PARTS * BLOCK, BLOCK);
                }
                fence_to_tensor();
                __syncwarp();
                if (lane == 0) bar_arrive(&bars.full[stage]);
                stage += TEAMS;
                if (stage >= plan.stages) { stage -= plan.stages; phase ^= 1; }
                fetch();   // behind the last stage: zeros
            }
        }
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, plan.tensor_columns);
}

// ------------------------------------------------------------------------------------------------ host
template <typename T>
static EmPlan em_plan(const ExArgs& e, int back, bool slopes, int* tiles)   // slopes: they are brought beside the rows
{
    constexpr int PARTS = TmParts<T>::N, A_BYTES = PARTS * TM_ROWS * 128, MOST = PARTS == 1 ? 256 : 128;
    const int kk = back ? e.t.outer : e.t.inner, nn = back ? e.t.inner : e.t.outer;
    EmPlan p = {};
    p.back = back;
    p.chunks = (kk + 63) / 64;
    const int raw = slopes ? EM_RAW * 2 * A_BYTES : 0, room = EM_SMEM - 1024 - raw;
    // As few tiles of columns as there is room for sums: every tile gathers the rows anew, which costs more than a matrix that comes from L2 with every tile of
    // rows (300 k pairs 512 x 256 bf16 in one tile, from L2: 101 us; in two whose halves of the matrix stay: 131).
    *tiles = (nn + MOST - 1) / MOST;
    p.columns = tm_round((nn + *tiles - 1) / *tiles, 16);
    *tiles = (nn + p.columns - 1) / p.columns;
    p.b_bytes = PARTS * p.columns * 128;
    p.resident = (int64_t)p.chunks * p.b_bytes + (PARTS == 1 && !slopes ? 4 : 2) * A_BYTES <= room;
    p.stage_bytes = A_BYTES + (p.resident ? 0 : p.b_bytes);
    p.stages = std::min(EM_MAX_STAGES, (room - (p.resident ? p.chunks * p.b_bytes : 0)) / p.stage_bytes);
    p.column_stride = tm_round(p.columns, 32);
    p.tensor_columns = tm_tensor_columns((PARTS == 1 ? 2 : 4) * p.column_stride);
    p.smem = 1024 + (p.resident ? p.chunks * p.b_bytes : 0) + p.stages * p.stage_bytes + raw;
    return p;
}

template <typename T>
static int64_t em_packed(const ExArgs& e, int back)
{
    int tiles;
    const EmPlan p = em_plan<T>(e, back, false, &tiles);
    return (int64_t)e.t.types * tiles * p.chunks * p.b_bytes;
}

int64_t ex_packed_bytes(const ExArgs& e, int back, int dtype) { return dtype == DYNB_F32 ? em_packed<float>(e, back) : em_packed<__nv_bfloat16>(e, back); }

template <typename T, typename O>
static cudaError_t em_rows(const ExArgs& e, int back, void* packed, cudaStream_t s)
{
    constexpr int SIZE = (int)sizeof(T);
    const TlArgs& a = e.t;
    const int kk = back ? a.outer : a.inner;
    const void* const in = back ? a.dy : a.x;
    const void* const out = back ? a.dx : a.y;
    const bool slope = back && e.activation != DYNB_ACTIVATION_NONE && e.slope != nullptr;   // rows that were copied have met theirs
    int tiles;
    EmPlan p = em_plan<T>(e, back, SIZE == 2 && slope, &tiles);
    p.packed = static_cast<const unsigned char*>(packed);
    p.store = tm_on(out, e.out_row, sizeof(O), 32) ? 32 : tm_on(out, e.out_row, sizeof(O), 16) ? 16 : (int)sizeof(O);
    p.slope_store = tm_on(e.slope, e.out_row, SIZE, 32) ? 32 : tm_on(e.slope, e.out_row, SIZE, 16) ? 16 : SIZE;
    const bool wide_w = tm_on(a.w, a.outer, SIZE, 16) && a.outer % 8 == 0;
    const int64_t units = (int64_t)a.types * tiles * p.chunks * (p.columns / (wide_w && !back ? 16 / SIZE : 1)) * 8;
    (wide_w ? ex_pack_kernel<T, true> : ex_pack_kernel<T, false>)<<<(unsigned)std::min<int64_t>((units + 255) / 256, (int64_t)sm_count_cached() * 8), 256, 0, s>>>(
        static_cast<const T*>(a.w), a.types, a.inner, a.outer, back, p.columns, tiles, p.chunks, static_cast<unsigned char*>(packed));
    cudaError_t rc = cudaGetLastError();
    if (rc != cudaSuccess) return rc;
    // Warps that store results: activations in 16 bits keep sixteen busy (300 k pairs 256 x 512 with slopes: 196 us, with eight 227); without them eight leave the others more registers.
    constexpr int FEW = SIZE == 4 ? 4 : 8, MANY = SIZE == 4 ? 4 : 16;
    const bool many = MANY != FEW && std::is_same<T, O>::value && !back && e.activation != DYNB_ACTIVATION_NONE;
    void (*kernel)(ExArgs, EmPlan);
    if constexpr (SIZE == 4) {   // by 32 bytes half as many steps to the same lines (200 k pairs 512 x 128: 166 -> 163 us, the weights' pass 224 -> 216)
        const bool all = tm_on(in, back ? a.dy_row : a.x_row, SIZE, 32) && (!slope || tm_on(e.slope, kk, SIZE, 32));
        if (slope) kernel = all ? em_rows_kernel<T, O, EM_SLOPE, 2, FEW> : em_rows_kernel<T, O, EM_SLOPE, 1, FEW>;
        else kernel = all ? em_rows_kernel<T, O, EM_REGISTERS, 2, FEW> : em_rows_kernel<T, O, EM_REGISTERS, 1, FEW>;
    } else {
        kernel = slope ? em_rows_kernel<T, O, EM_ASYNC_SLOPE, 1, FEW> : em_rows_kernel<T, O, EM_ASYNC, 1, FEW>;
        if constexpr (std::is_same<T, O>::value)
            if (many) kernel = em_rows_kernel<T, O, EM_ASYNC, 1, MANY>;
    }
    const int64_t most = (a.n + TM_ROWS - 1) / TM_ROWS + a.types;
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(most, sm_count_cached() / std::min(tiles, sm_count_cached()))), tiles);
    rc = allow_shared(reinterpret_cast<const void*>(kernel), EM_SMEM);
    if (rc != cudaSuccess) return rc;
    kernel<<<grid, em_threads<T>(many ? MANY : FEW), p.smem, s>>>(e, p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t em_rows_of(const ExArgs& e, int back, void* packed, cudaStream_t s)
{
    if constexpr (sizeof(T) == 2) {
        if (back && e.fan > 1) return em_rows<T, float>(e, back, packed, s);
    }
    return em_rows<T, T>(e, back, packed, s);
}

cudaError_t ex_mma_rows(const ExArgs& e, int back, int dtype, void* packed, cudaStream_t s)
{
    if (dtype == DYNB_F32) return em_rows_of<float>(e, back, packed, s);
    if (dtype == DYNB_F16) return em_rows_of<__half>(e, back, packed, s);
    return em_rows_of<__nv_bfloat16>(e, back, packed, s);
}

int64_t ex_stretches(const ExArgs& e) { return e.t.n / e.t.stretch + 1 + std::min<int64_t>(e.t.n, e.t.types); }   // cuts at multiples, and where experts begin

template <typename T>
static cudaError_t em_weights(const ExArgs& e, cudaStream_t s)
{
    constexpr int PARTS = TmParts<T>::N, BLOCK = EW_ROWS<T> * 128, SIZE = (int)sizeof(T);
    const TlArgs& a = e.t;
    EwPlan p = {};
    p.most = ex_stretches(e);
    const int most = PARTS == 1 ? 256 : 128, tiles = (a.outer + most - 1) / most;
    p.columns = tm_round((a.outer + tiles - 1) / tiles, 16);
    p.column_stride = tm_round(p.columns, 32);
    p.x_blocks = a.inner > 64 ? 2 : 1;
    p.y_blocks = (p.columns + 63) / 64;
    p.row_tiles = (a.inner + TM_ROWS - 1) / TM_ROWS;
    p.column_tiles = (a.outer + p.columns - 1) / p.columns;
    const int stage = (p.x_blocks + p.y_blocks) * PARTS * BLOCK;
    p.stages = std::min(EW_MAX_STAGES, (EW_SMEM - 1024) / stage);
    p.tensor_columns = tm_tensor_columns((PARTS == 1 ? 2 : 4) * p.column_stride);
    p.store = tm_on(a.partial, a.outer, 4, 32) && (int64_t)a.inner * a.outer % 8 == 0 ? 32 : tm_on(a.partial, a.outer, 4, 16) ? 16 : 4;
    void (*kernel)(ExArgs, EwPlan);
    if constexpr (SIZE == 4) kernel = tm_on(a.x, a.x_row, SIZE, 32) && tm_on(a.dy, a.dy_row, SIZE, 32) ? em_weights_kernel<T, EM_REGISTERS, 2> : em_weights_kernel<T, EM_REGISTERS, 1>;
    else kernel = em_weights_kernel<T, EM_ASYNC, 1>;
    const int smem = 1024 + p.stages * stage, tiles_of = p.row_tiles * p.column_tiles;
    const cudaError_t rc = allow_shared(reinterpret_cast<const void*>(kernel), EW_SMEM);
    if (rc != cudaSuccess) return rc;
    kernel<<<(unsigned)(std::max(1, ex_slices(a.inner, a.outer, sizeof(T))) * tiles_of), EW_THREADS<T>, smem, s>>>(e, p);
    return cudaGetLastError();
}

cudaError_t ex_mma_weights(const ExArgs& e, int dtype, cudaStream_t s)
{
    if (dtype == DYNB_F32) return em_weights<float>(e, s);
    if (dtype == DYNB_F16) return em_weights<__half>(e, s);
    return em_weights<__nv_bfloat16>(e, s);
}

}  // namespace dynb
