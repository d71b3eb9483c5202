// The products by type on the tensor cores.
//
// y = x W + b and dx = dy W^T: a block keeps the whole matrix of a type for its columns in shared memory (laid out once per type) and takes
// tiles of 128 rows one after the other: eight or sixteen warps gather the rows into stages of 64 columns, one thread issues the products, four
// warps take the sums out of tensor memory, which holds two of them, turn them in shared memory and store the rows by whole lines.  What bounds
// it is the chain of a stage from memory to the multipliers, and shared memory, which rows, matrix and results share.
//
// dW = sum x_i^T dy_i: a block takes a stretch of rows of one type, 128 x up to 256 elements of the matrix; both operands are the gathered
// rows as they are, read along their columns.  db is a product too, with a tile of ones.
//
// 1 M rows, 128 x 128 fp32, 5 types: y 268 us, dx 271 (3.8 TB/s), the weights' gradient 384 us; bf16: 148, 150 and 325.  400 k rows, 256 x 256 bf16,
// 89 types: 142 us (2.9 TB/s).  Kernels of fused multiply-adds on 64 x 64 tiles took 6.6 ms for the three in fp32, and 3.3 ms.
//
// The whole summed dimension of a matrix has to stand in shared memory beside two stages of rows.  So y sums at most 256 columns in fp32 and 1344 in 16 bits, dx
// 1088 and 5376; wider ones go to tl_rows_kernel.  Columns that do not fit beside one another are tiles, each of which reads all rows (fp32, 129 to 256 summed
// columns: tiles of 64).  200 k rows in fp32: 256 x 128 151 us, 257 x 128 778 us; the weights' gradient has no such limit.
//
// fp32 operands are split into three bf16 parts (8 bits each, together all 24): v = p0 + p1 + p2 (below
// 2^-109 the last parts meet the smallest steps of bf16 and v is kept to within 2^-133).  Six of the nine products are formed,
// those left out are below 2^-25 of the whole; the small ones are added first.  Sums are in fp32.

#include <type_traits>

#include "type_linear.cuh"
#include "umma.cuh"

namespace dynb {

constexpr int TM_ROWS = 128;
// Warps that gather, and stages whose rows are on their way in their registers beside the one that is being stored.  Sixteen warps are ahead of one
// another; rows in fp32 need the registers of eight (1 M rows 128 x 128, both passes: 519 us, sixteen 543; the weights' gradient 308 and 284).
template <typename T> constexpr int TM_FEED = sizeof(T) == 4 ? 8 : 16;
template <typename T> constexpr int TM_AHEAD = sizeof(T) == 4 ? 2 : 1;
constexpr int TW_FEED = 16;
__host__ __device__ constexpr int tm_threads(int feed) { return (4 + 1 + feed) * 32; }
constexpr int TM_MAX_STAGES = 8;
constexpr int TM_SMEM = 202 * 1024;        // beside 23 KB of offsets, results under way and barriers
constexpr int TW_ROWS = 32;                 // rows of a stage of the weights' gradient

template <typename T> struct TmParts { static constexpr int N = 1; };
template <> struct TmParts<float> { static constexpr int N = 3; };
template <typename T> struct TmRaw { uint4 v[sizeof(T) == 4 ? 2 : 1]; };   // 8 elements as loaded

// Eight elements `step` apart from p, the first `have` of them real, zeros behind.  WIDE: 16-byte boundaries, step 1 and have 0 or 8.  (Chosen
// at run time, the two ways meet in copies of what was loaded, and each load is waited for before the next.)
template <bool WIDE, typename T>
__device__ __forceinline__ TmRaw<T> tm_load(const T* p, int64_t step, int have)
{
    TmRaw<T> r;
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(r) / 16); i++) {
            r.v[i] = make_uint4(0, 0, 0, 0);
            if (have > 0) r.v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        }
        return r;
    }
    using W = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    union { TmRaw<T> r; W w[8]; } u;
#pragma unroll
    for (int i = 0; i < 8; i++) u.w[i] = i < have ? *reinterpret_cast<const W*>(p + i * step) : (W)0;
    return u.r;
}

// Two elements one of which may not split by rounding, part by part: an infinity becomes (1, 0, itself), whose products with finite elements and
// with another infinity are what they should be; where rounding to 8 bits gives an infinity, the largest number of 8 bits leads; a NaN leads itself.
__device__ __forceinline__ void tm_split_odd(uint32_t lo, uint32_t hi, uint32_t (&part)[3])
{
    uint32_t p[2][3];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t bits = k == 0 ? lo : hi, size = bits & 0x7fffffffu, sign = bits & 0x80000000u;
        if (size >= 0x7f800000u) {
            p[k][0] = size == 0x7f800000u ? sign | 0x3f800000u : 0x7fc00000u;
            p[k][1] = 0;
            p[k][2] = size == 0x7f800000u ? bits : 0;
        } else {
            const float v = __uint_as_float(bits);
            p[k][0] = size >= 0x7f7f8000u ? sign | 0x7f7f0000u : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) << 16;
            const float rest = v - __uint_as_float(p[k][0]);
            p[k][1] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(rest)) << 16;
            p[k][2] = __float_as_uint(rest - __uint_as_float(p[k][1]));
        }
    }
#pragma unroll
    for (int i = 0; i < 3; i++) part[i] = __byte_perm(p[0][i], p[1][i], 0x7632);
}

// Whether one of these elements is among them (of a NaN this says nothing: it comes through by rounding, too).  Asked once for all pieces of a stage, which costs 8
// of the 1028 us of all passes over 1 M rows of 128 x 128; a branch at every piece cost 17.
template <typename T, int N>
__device__ __forceinline__ bool tm_odd(const TmRaw<T> (&r)[N])
{
    if constexpr (sizeof(T) == 2) {
        return false;
    } else {
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(__uint_as_float(reinterpret_cast<const uint32_t*>(&r[k])[i])));
        return most >= __uint_as_float(0x7f7f8000u);
    }
}

// The parts of eight elements, 16 bytes each, to `at`, `at + apart`, ...  ODD: see above.
template <bool ODD, typename T>
__device__ __forceinline__ void tm_store(const TmRaw<T>& r, unsigned char* at, int apart)
{
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(at) = r.v[0];
    } else {
        const uint32_t* const bits = reinterpret_cast<const uint32_t*>(&r);
        uint32_t part[3][4];
        if constexpr (ODD) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t p[3];
                tm_split_odd(bits[2 * i], bits[2 * i + 1], p);
#pragma unroll
                for (int k = 0; k < 3; k++) *reinterpret_cast<uint32_t*>(at + k * apart + 4 * i) = p[k];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[2] = {__uint_as_float(bits[2 * i]), __uint_as_float(bits[2 * i + 1])};
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[0], v[1]);
                const uint32_t w = *reinterpret_cast<const uint32_t*>(&b);
                part[p][i] = w;
                v[0] -= __uint_as_float(w << 16);          // exact
                v[1] -= __uint_as_float(w & 0xffff0000u);
            }
            part[2][i] = __byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x7632);   // eight bits at most are left
        }
#pragma unroll
        for (int p = 0; p < 3; p++) *reinterpret_cast<uint4*>(at + p * apart) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
    }
}

// Adds the products of one step of 16 summed elements: the parts of `a` are `a_part` apart, those of `b` `b_part` (units of 16 bytes).  A part of `a`
// stays at the multipliers for its products.  The products of the leading parts go to d, the small ones to `small`.  The tensor cores cut sums off
// where they do not fit 24 bits, towards zero, every step: with six additions a step to one sum, operands of one sign lost 4.1e-6 of a weights' gradient over
// 1024 rows and 1.4e-6 of y over 256 columns (means); with one addition a step to a sum of its own 1.7e-6 and 3.1e-7.
template <int PARTS>
__device__ __forceinline__ void tm_step(uint32_t d, uint32_t small, uint64_t a, int a_part, uint64_t b, int b_part, uint32_t what, bool add)
{
    if constexpr (PARTS == 1) {
        tensor_mma(d, a, b, what, add);
    } else {
        tensor_mma(small, a + 2 * a_part, b, what, add);
        tensor_mma_keep<1>(small, a + a_part, b + b_part, what, true);
        tensor_mma_keep<3>(small, a + a_part, b, what, true);
        tensor_mma_keep<1>(small, a, b + 2 * b_part, what, true);
        tensor_mma_keep<2>(small, a, b + b_part, what, true);
        tensor_mma_keep<3>(d, a, b, what, add);
    }
}

// Walks the pieces [first, first + count) of TM_ROWS rows.
struct TmCursor {
    TlTile tile;
    int64_t end_of_type;
    int64_t left;

    __device__ __forceinline__ void start(const TlArgs& a, int64_t first, int64_t count)   // all lanes of a warp
    {
        left = count;
        tile = {-1, 0, 0};
        if (count <= 0) return;
        tile = tl_tile(a, first, TM_ROWS);
        if (tile.type < 0) { left = 0; return; }
        int64_t s0;
        tl_rows_of(a, tile.type, &s0, &end_of_type);
    }
    __device__ __forceinline__ void next(const TlArgs& a)
    {
        if (--left <= 0) { tile.type = -1; return; }
        tile.begin += TM_ROWS;
        if (tile.begin >= end_of_type) {
            do {
                if (++tile.type >= a.types) { tile.type = -1; left = 0; return; }
                tl_rows_of(a, tile.type, &tile.begin, &end_of_type);
            } while (tile.begin >= end_of_type);
        }
        tile.end = min(tile.begin + TM_ROWS, end_of_type);
    }
};

struct TmPlan {
    int back, columns, column_stride, chunks, stages, tensor_columns, panel_bytes, b_chunk, b_part, b_step, wide_w, store;   // store: bytes of a store of results, 16 or one element
};

struct TmBars { uint64_t full[TM_MAX_STAGES], empty[TM_MAX_STAGES], panel_full, panel_free, sums_full[2], sums_free[2]; uint32_t tensor; };

__device__ __forceinline__ void tm_ran_out(const TlArgs& a)
{
    if (a.status != nullptr) {
        *reinterpret_cast<volatile uint32_t*>(a.status) = 1u;
        __threadfence_system();
    }
}

// Four results as words of the type.
template <typename T>
__device__ __forceinline__ void tm_words(const float (&v)[4], uint32_t* w)
{
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
    }
}

// `n` sums of a row, in stores of 16 bytes or of one element.
__device__ __forceinline__ void tm_put_row(float* at, const uint32_t (&v)[32], int n, bool wide)
{
    if (wide && n >= 32) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(at + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; i++)
        if (i < n) at[i] = __uint_as_float(v[i]);
}

// The matrix of a type, its rows as they are.  y = x W reads them along columns: blocks of 64 columns by all summed rows.  dx = dy W^T reads them along
// rows: blocks of 64 summed columns by all rows.
template <typename T, bool WIDE>
__device__ __forceinline__ void tm_panel(const TmPlan& plan, const T* w, unsigned char* panel, int tid, int kk, int nn, int col0, int outer)
{
    const int across = plan.back ? plan.chunks * 8 : (plan.columns + 63) / 64 * 8, down = plan.back ? plan.columns : plan.chunks * 64;
    const int row0 = plan.back ? col0 : 0, piece0 = plan.back ? 0 : col0;
    const int rows = plan.back ? min(nn - col0, plan.columns) : kk, columns = plan.back ? kk : min(nn, col0 + plan.columns);
    const int block = plan.back ? TmParts<T>::N * down * 128 : down * 128, apart = plan.b_part * 16;
    constexpr int threads = TM_FEED<T> * 32;
#pragma unroll (sizeof(T) == 4 ? 1 : 8)
    for (int u = tid; u < across * down; u += threads) {
        const int piece = u % across, r = u / across, c = piece0 + piece * 8;
        const int have = r < rows ? min(8, columns - c) : 0;
        const TmRaw<T> m = tm_load<WIDE>(have > 0 ? w + (int64_t)(row0 + r) * outer + c : w, 1, have);
        const TmRaw<T> one[1] = {m};
        unsigned char* const to = panel + (piece / 8) * block + tile_piece(r, piece & 7);
        if (tm_odd(one)) tm_store<true>(m, to, apart);
        else tm_store<false>(m, to, apart);
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(tm_threads(TM_FEED<T>), 1)
tm_rows_kernel(const TlArgs a, const TmPlan plan)
{
    constexpr int FEED = TM_FEED<T>, FEED_THREADS = FEED * 32, PARTS = TmParts<T>::N, STAGE = PARTS * TM_ROWS * 128, COLUMNS = 128 / (int)sizeof(T);
    extern __shared__ unsigned char raw_smem[];
    __shared__ TmBars bars;
    __shared__ __align__(16) float offsets[4][256];
    __shared__ __align__(16) unsigned char turned[4][32 * 144];
    unsigned char* const panel = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    unsigned char* const stage0 = panel + plan.panel_bytes;
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const T* const in = static_cast<const T*>(plan.back ? a.dy : a.x);
    T* const out = static_cast<T*>(plan.back ? a.dx : a.y);
    const int64_t in_row = plan.back ? a.dy_row : a.x_row;
    const int kk = plan.back ? a.outer : a.inner, nn = plan.back ? a.inner : a.outer;
    const int col0 = blockIdx.y * plan.columns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; s++) {
            bar_init(&bars.full[s], FEED);
            bar_init(&bars.empty[s], 1);
        }
        bar_init(&bars.panel_full, FEED);
        bar_init(&bars.panel_free, 1);
        for (int b = 0; b < 2; b++) {
            bar_init(&bars.sums_full[b], 1);
            bar_init(&bars.sums_free[b], 4);
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

    if (warp < 4) {
        // sums to the rows
        const bool with_offset = !plan.back && a.b != nullptr;
        float* const offset = offsets[warp];
        int buffer = 0, offset_type = -1;
        uint32_t phase = 0;
        for (; cursor.tile.type >= 0; cursor.next(a)) {
            const int64_t place = cursor.tile.begin + threadIdx.x;
            int32_t r = place < cursor.tile.end ? __ldg(a.order + place) : -1;
            const int have = min(plan.columns, nn - col0);
            if (with_offset && cursor.tile.type != offset_type) {
                offset_type = cursor.tile.type;
                __syncwarp();
                for (int c = lane; c < have; c += 32) offset[c] = tl_get(static_cast<const T*>(a.b) + (int64_t)offset_type * a.outer + col0 + c);
                __syncwarp();
            }
            if (!bar_wait(&bars.sums_full[buffer], phase)) { tm_ran_out(a); break; }
            tensor_fence_after();
            if ((uint32_t)r >= (uint64_t)a.n) r = -1;
            // 32 words of every row at a time: out of tensor memory by rows, through shared memory, to memory by pieces of 16 bytes of whole lines
            const uint32_t from = tensor + ((uint32_t)(warp * 32) << 16) + buffer * plan.column_stride;
            for (int c = 0; c < have; c += COLUMNS) {
                uint32_t words[32];
#pragma unroll
                for (int half = 0; half < COLUMNS / 32; half++) {
                    uint32_t bits[32];
                    __syncwarp();
                    tensor_load_32(from + min(c + 32 * half, plan.column_stride - 32), bits);
                    tensor_wait_loads();
                    if constexpr (PARTS > 1) {   // the small products' sums
                        uint32_t small[32];
                        tensor_load_32(from + 2 * plan.column_stride + min(c + 32 * half, plan.column_stride - 32), small);
                        tensor_wait_loads();
#pragma unroll
                        for (int i = 0; i < 32; i++) bits[i] = __float_as_uint(__uint_as_float(bits[i]) + __uint_as_float(small[i]));
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float v[4] = {__uint_as_float(bits[i]), __uint_as_float(bits[i + 1]), __uint_as_float(bits[i + 2]), __uint_as_float(bits[i + 3])};
                        if (with_offset) {   // behind `have`: not stored
                            const float4 o = *reinterpret_cast<const float4*>(offset + min(c + 32 * half, 224) + i);
                            v[0] += o.x; v[1] += o.y; v[2] += o.z; v[3] += o.w;
                        }
                        tm_words<T>(v, words + (COLUMNS / 32 == 1 ? i : 16 * half + i / 2));
                    }
                }
                unsigned char* const mine = turned[warp];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; i++) *reinterpret_cast<uint4*>(mine + lane * 144 + 16 * i) = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
                __syncwarp();
                constexpr int PER = 16 / (int)sizeof(T);
                const int at = c + (lane & 7) * PER;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int row = 4 * j + (lane >> 3);
                    const int32_t to = __shfl_sync(0xffffffffu, r, row);
                    const uint4 piece = *reinterpret_cast<const uint4*>(mine + row * 144 + 16 * (lane & 7));
                    if (to < 0 || at >= have) continue;
                    T* const p = out + (int64_t)to * nn + col0 + at;
                    if (plan.store == 16) {
                        *reinterpret_cast<uint4*>(p) = piece;
                    } else {
                        const T* const e = reinterpret_cast<const T*>(&piece);
#pragma unroll
                        for (int i = 0; i < PER; i++)
                            if (at + i < have) p[i] = e[i];
                    }
                }
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars.sums_free[buffer]);
            buffer ^= 1;
            if (buffer == 0) phase ^= 1;
        }
    } else if (warp == 4) {
        // products
        const bool bf16 = !std::is_same<T, __half>::value;
        const uint32_t what = mma_what(bf16, plan.columns, false, !plan.back);
        const uint32_t stage_at = smem_addr(stage0);
        const uint64_t panel_from = tile_descriptor(smem_addr(panel), plan.back ? 16 : plan.chunks * 8192, 1024);
        int stage = 0, buffer = 0, panel_type = -1;
        uint32_t phase = 0, panel_phase = 0, sums_phase = 1;
        bool ok = true;
        while (ok && cursor.tile.type >= 0) {
            if (cursor.tile.type != panel_type) {
                if (!bar_wait(&bars.panel_full, panel_phase)) { ok = false; break; }
                panel_phase ^= 1;
                panel_type = cursor.tile.type;
            }
            if (!bar_wait(&bars.sums_free[buffer], sums_phase)) { ok = false; break; }
            tensor_fence_after();
            const uint32_t sums = tensor + buffer * plan.column_stride;
            for (int chunk = 0; chunk < plan.chunks; chunk++) {
                if (!bar_wait(&bars.full[stage], phase)) { ok = false; break; }
                tensor_fence_after();
                if (elected()) {
                    const int steps = min(4, (kk - chunk * 64 + 15) / 16);
                    // descriptors are in units of 16 bytes: steps and parts are additions
                    const uint64_t at_a = tile_descriptor(stage_at + stage * STAGE, 16, 1024), at_b = panel_from + (uint32_t)(chunk * plan.b_chunk);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (k < steps) tm_step<PARTS>(sums, sums + 2 * plan.column_stride, at_a + 2 * k, TM_ROWS * 128 / 16, at_b + (uint32_t)(k * plan.b_step), plan.b_part, what, chunk > 0 || k > 0);
                    tensor_commit(&bars.empty[stage]);
                    if (chunk == plan.chunks - 1) tensor_commit(&bars.sums_full[buffer]);
                }
                __syncwarp();
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            cursor.next(a);
            if (cursor.tile.type >= 0 && cursor.tile.type != panel_type && elected()) tensor_commit(&bars.panel_free);
            __syncwarp();
            buffer ^= 1;
            if (buffer == 0) sums_phase ^= 1;
        }
        if (!ok) tm_ran_out(a);
    } else {
        // rows and matrices to shared memory: stages are asked for AHEAD of their turn
        constexpr int AHEAD = TM_AHEAD<T>, UNITS = TM_ROWS * 8 / FEED_THREADS;
        const int tid = threadIdx.x - 5 * 32, piece = tid & 7;
        int panel_type = -1, stage = 0, chunk = 0;
        uint32_t phase = 1, free_phase = 0;
        TlTile next = cursor.tile;                  // of the next stage to ask for
        int32_t rows[UNITS], rows_next[UNITS];      // of that tile and the one behind it
        auto rows_of = [&](const TlTile& t, int32_t (&r)[UNITS]) {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int64_t place = t.begin + (tid >> 3) + (FEED_THREADS / 8) * i;
                r[i] = t.type >= 0 && place < t.end ? __ldg(a.order + place) : -1;   // looked at a tile later
            }
        };
        TmRaw<T> v[AHEAD][UNITS];
        int type_of[AHEAD];
        auto ask = [&](TmRaw<T> (&to)[UNITS], int& type) {
            type = next.type;
            if (next.type < 0) return;
            const int k = chunk * 64 + piece * 8, have = min(8, kk - k);
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const bool ok = (uint32_t)rows[i] < (uint64_t)a.n;
                to[i] = tm_load<WIDE>(in + (ok ? rows[i] * in_row + k : 0), 1, ok ? have : 0);
            }
            if (++chunk == plan.chunks) {
                chunk = 0;
                next = cursor.tile;
#pragma unroll
                for (int i = 0; i < UNITS; i++) rows[i] = rows_next[i];
                if (next.type >= 0) {
                    cursor.next(a);
                    rows_of(cursor.tile, rows_next);
                }
            }
        };
        rows_of(next, rows);
        if (next.type >= 0) cursor.next(a);
        rows_of(cursor.tile, rows_next);
#pragma unroll
        for (int s = 0; s < AHEAD; s++) ask(v[s], type_of[s]);
        bool more = true;
        while (more) {
#pragma unroll
            for (int s = 0; s < AHEAD; s++) {
                if (type_of[s] < 0) { more = false; break; }
                if (type_of[s] != panel_type) {
                    if (panel_type >= 0) {
                        if (!bar_wait(&bars.panel_free, free_phase)) { tm_ran_out(a); more = false; break; }
                        free_phase ^= 1;
                    }
                    panel_type = type_of[s];
                    const T* const w = static_cast<const T*>(a.w) + (int64_t)panel_type * a.inner * a.outer;
                    if (plan.wide_w) tm_panel<T, true>(plan, w, panel, tid, kk, nn, col0, a.outer);
                    else tm_panel<T, false>(plan, w, panel, tid, kk, nn, col0, a.outer);
                    fence_to_tensor();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&bars.panel_full);
                }
                if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); more = false; break; }
                unsigned char* const to = stage0 + stage * STAGE + tile_piece(tid >> 3, piece);   // FEED_THREADS / 8 rows on: the same place among eight
                if (tm_odd(v[s])) {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) tm_store<true>(v[s][i], to + i * FEED_THREADS * 16, TM_ROWS * 128);
                } else {
#pragma unroll
                    for (int i = 0; i < UNITS; i++) tm_store<false>(v[s][i], to + i * FEED_THREADS * 16, TM_ROWS * 128);
                }
                fence_to_tensor();
                __syncwarp();
                if (lane == 0) bar_arrive(&bars.full[stage]);
                if (++stage == plan.stages) { stage = 0; phase ^= 1; }
                ask(v[s], type_of[s]);
            }
        }
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, plan.tensor_columns);
}

struct TwPlan { int columns, column_stride, x_blocks, y_blocks, stages, tensor_columns, vec; };

template <typename T, bool WIDE>
__global__ void __launch_bounds__(tm_threads(TW_FEED), 1)
tm_weights_kernel(const TlArgs a, const TwPlan plan)
{
    constexpr int FIRST = TmParts<T>::N == 1 ? 1 : 2;   // sums of the matrix: leading parts, small ones; those of the rows behind them
    constexpr int FEED = TW_FEED, FEED_THREADS = FEED * 32, PARTS = TmParts<T>::N, BLOCK = TW_ROWS * 128;
    constexpr int UNITS = PARTS == 1 ? 3 : 2;   // pieces of 8 elements a thread and stage: 32 rows x (128 + 256 or 128) elements
    extern __shared__ unsigned char raw_smem[];
    __shared__ TmBars bars;
    unsigned char* const ones = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    unsigned char* const stage0 = ones + TM_ROWS * 128;
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int row0 = blockIdx.y * TM_ROWS, col0 = blockIdx.z * plan.columns;
    const int blocks = plan.x_blocks + plan.y_blocks, stage_bytes = blocks * PARTS * BLOCK;
    const TlTile tile = tl_tile(a, blockIdx.x, a.stretch);
    if (tile.type < 0) return;   // the whole block
    const int steps = (int)((tile.end - tile.begin + TW_ROWS - 1) / TW_ROWS);
    const bool sums_wanted = blockIdx.y == 0 && a.db != nullptr;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; s++) {
            bar_init(&bars.full[s], FEED);
            bar_init(&bars.empty[s], 1);
        }
        bar_init(&bars.sums_full[0], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const uint32_t one = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
    for (int i = threadIdx.x; i < TM_ROWS * 8; i += tm_threads(FEED)) reinterpret_cast<uint4*>(ones)[i] = make_uint4(one, one, one, one);
    fence_to_tensor();
    if (warp == 0) tensor_alloc(&bars.tensor, plan.tensor_columns);
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = bars.tensor;

    if (warp < 4) {
        if (!bar_wait(&bars.sums_full[0], 0)) {
            tm_ran_out(a);
        } else {
            tensor_fence_after();
            const int64_t cells = (int64_t)a.inner * a.outer;
            float* const mine = a.partial + blockIdx.x * (cells + a.outer);
            const int m = row0 + threadIdx.x, have = min(plan.columns, a.outer - col0);
            for (int which = 0; which < (sums_wanted ? 2 : 1); which++) {
                float* const at = which == 0 ? mine + (int64_t)m * a.outer + col0 : mine + cells + col0;
                const bool write = which == 0 ? m < a.inner : threadIdx.x == 0;
                const uint32_t from = tensor + ((uint32_t)(warp * 32) << 16) + which * FIRST * plan.column_stride;
                for (int c = 0; c < have; c += 32) {
                    uint32_t bits[32];
                    __syncwarp();
                    tensor_load_32(from + c, bits);
                    tensor_wait_loads();
                    if constexpr (PARTS > 1) {
                        uint32_t small[32];
                        tensor_load_32(from + plan.column_stride + c, small);
                        tensor_wait_loads();
#pragma unroll
                        for (int i = 0; i < 32; i++) bits[i] = __float_as_uint(__uint_as_float(bits[i]) + __uint_as_float(small[i]));
                    }
                    if (write) tm_put_row(at + c, bits, have - c, plan.vec != 0);
                }
            }
        }
    } else if (warp == 4) {
        const bool bf16 = !std::is_same<T, __half>::value;
        const uint32_t what = mma_what(bf16, plan.columns, true, true), what_sum = mma_what(bf16, plan.columns, false, true);
        const uint32_t stage_at = smem_addr(stage0);
        const uint64_t ones_desc = tile_descriptor(smem_addr(ones), 16, 1024);
        const uint32_t lead = PARTS * BLOCK, lead_x = plan.x_blocks > 1 ? lead : 0;   // one block: the upper 64 rows repeat the lower
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int step = 0; step < steps; step++) {
            if (!bar_wait(&bars.full[stage], phase)) { ok = false; break; }
            tensor_fence_after();
            if (elected()) {
                const uint32_t at = stage_at + stage * stage_bytes;
                const uint64_t at_x = tile_descriptor(at, lead_x, 1024), at_y = tile_descriptor(at + plan.x_blocks * PARTS * BLOCK, lead, 1024);
#pragma unroll
                for (int k = 0; k < TW_ROWS / 16; k++) tm_step<PARTS>(tensor, tensor + plan.column_stride, at_x + k * 128, BLOCK / 16, at_y + k * 128, BLOCK / 16, what, step > 0 || k > 0);
                if (sums_wanted) {
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
                        for (int k = 0; k < TW_ROWS / 16; k++)
                            tensor_mma(tensor + (p == 0 ? FIRST : FIRST + 1) * plan.column_stride, ones_desc, at_y + (p * BLOCK + k * 2048) / 16, what_sum,
                                       step > 0 || k > 0 || (p > 0 && p < PARTS - 1));
                }
                tensor_commit(&bars.empty[stage]);
                if (step == steps - 1) tensor_commit(&bars.sums_full[0]);
            }
            __syncwarp();
            if (++stage == plan.stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) tm_ran_out(a);
    } else {
        const int tid = threadIdx.x - 5 * 32;
        const int per_row = blocks * 8, units = TW_ROWS * per_row;
        // this thread's pieces are the same ones in every stage: row, place in the stage, operand, column
        int row[UNITS], at[UNITS], col[UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            const int u = tid + i * FEED_THREADS, r = u / per_row, piece = u % per_row;
            const int block = piece >> 3;
            const bool of_y = block >= plan.x_blocks;
            row[i] = u < units ? r : -1;
            at[i] = block * PARTS * BLOCK + (int)tile_piece(r, piece & 7);
            const int c = (of_y ? col0 + (block - plan.x_blocks) * 64 : row0 + block * 64) + (piece & 7) * 8;
            const int limit = of_y ? min(a.outer, col0 + plan.columns) : a.inner;
            col[i] = c < limit ? (of_y ? c | (1 << 30) : c) : -1;
        }
        auto rows_of = [&](int step, int32_t (&r)[UNITS]) {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int64_t place = tile.begin + (int64_t)step * TW_ROWS + row[i];
                r[i] = row[i] >= 0 && col[i] >= 0 && place < tile.end ? __ldg(a.order + place) : -1;   // looked at a stage later
            }
        };
        auto fetch = [&](const int32_t (&r)[UNITS], TmRaw<T> (&v)[UNITS]) {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const bool of_y = (col[i] >> 30) & 1;
                const int c = col[i] & ((1 << 30) - 1);
                const T* const p = of_y ? static_cast<const T*>(a.dy) + r[i] * a.dy_row + c : static_cast<const T*>(a.x) + r[i] * a.x_row + c;
                const bool ok = (uint32_t)r[i] < (uint64_t)a.n;
                v[i] = tm_load<WIDE>(ok ? p : static_cast<const T*>(a.x), 1, ok ? min(8, (of_y ? a.outer : a.inner) - c) : 0);
            }
        };
        // the rows of the next stage are asked for behind this one, their numbers a stage earlier
        int32_t ids[UNITS];
        TmRaw<T> v[UNITS];
        rows_of(0, ids);
        fetch(ids, v);
        rows_of(1, ids);
        int stage = 0;
        uint32_t phase = 1;
        for (int step = 0; step < steps; step++) {
            if (!bar_wait(&bars.empty[stage], phase)) { tm_ran_out(a); break; }
            if (tm_odd(v)) {
#pragma unroll
                for (int i = 0; i < UNITS; i++)
                    if (row[i] >= 0) tm_store<true>(v[i], stage0 + stage * stage_bytes + at[i], BLOCK);
            } else {
#pragma unroll
                for (int i = 0; i < UNITS; i++)
                    if (row[i] >= 0) tm_store<false>(v[i], stage0 + stage * stage_bytes + at[i], BLOCK);
            }
            fence_to_tensor();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars.full[stage]);
            if (++stage == plan.stages) { stage = 0; phase ^= 1; }
            fetch(ids, v);   // behind the stretch: zeros
            rows_of(step + 2, ids);
        }
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (warp == 0) tensor_free(tensor, plan.tensor_columns);
}

static int tm_round(int v, int to) { return (v + to - 1) / to * to; }
static int tm_tensor_columns(int need)
{
    int c = 32;
    while (c < need) c *= 2;
    return c;
}
static bool tm_on(const void* p, int64_t row, int size, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && row * size % bytes == 0; }

template <typename T>
static bool tm_rows(const TlArgs& a, int back, cudaStream_t s, cudaError_t* rc)
{
    constexpr int PARTS = TmParts<T>::N, STAGE = PARTS * TM_ROWS * 128, SIZE = (int)sizeof(T);
    const int kk = back ? a.outer : a.inner, nn = back ? a.inner : a.outer;
    TmPlan p = {};
    p.back = back;
    p.chunks = (kk + 63) / 64;
    // as few column tiles as leave room for the matrix beside two stages (the rows are read once for each)
    int tiles = 1;
    for (;; tiles++) {
        p.columns = tm_round((nn + tiles - 1) / tiles, 16);
        p.panel_bytes = back ? p.chunks * PARTS * p.columns * 128 : PARTS * ((p.columns + 63) / 64) * p.chunks * 8192;
        if (p.columns <= (PARTS == 1 ? 256 : 128) && p.panel_bytes + 2 * STAGE + 1024 <= TM_SMEM) break;
        if (p.columns == 16) return false;
    }
    tiles = (nn + p.columns - 1) / p.columns;
    p.b_part = (back ? p.columns * 128 : p.panel_bytes / PARTS) / 16;
    p.b_chunk = (back ? PARTS * p.columns * 128 : 8192) / 16;
    p.b_step = (back ? 32 : 2048) / 16;
    p.stages = std::min(TM_MAX_STAGES, (TM_SMEM - 1024 - p.panel_bytes) / STAGE);
    p.column_stride = tm_round(p.columns, 32);
    p.tensor_columns = tm_tensor_columns((PARTS == 1 ? 2 : 4) * p.column_stride);
    const void* const in = back ? a.dy : a.x;
    const void* const out = back ? a.dx : a.y;
    const bool wide = tm_on(in, back ? a.dy_row : a.x_row, SIZE, 16) && kk % 8 == 0;
    p.wide_w = tm_on(a.w, a.outer, SIZE, 16) && a.outer % 8 == 0;
    p.store = tm_on(out, nn, SIZE, 16) && nn * SIZE % 16 == 0 ? 16 : SIZE;
    const int64_t most = (a.n + TM_ROWS - 1) / TM_ROWS + a.types;
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(most, sm_count_cached() / std::min(tiles, sm_count_cached()))), tiles);
    const int smem = 1024 + p.panel_bytes + p.stages * STAGE;
    void (*const kernel)(TlArgs, TmPlan) = wide ? tm_rows_kernel<T, true> : tm_rows_kernel<T, false>;
    *rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (*rc != cudaSuccess) return true;
    kernel<<<grid, tm_threads(TM_FEED<T>), smem, s>>>(a, p);
    *rc = cudaGetLastError();
    return true;
}

bool tl_mma_rows(const TlArgs& a, int back, int dtype, cudaStream_t s, cudaError_t* rc)
{
    if (dtype == DYNB_F32) return tm_rows<float>(a, back, s, rc);
    if (dtype == DYNB_F16) return tm_rows<__half>(a, back, s, rc);
    return tm_rows<__nv_bfloat16>(a, back, s, rc);
}

template <typename T>
static cudaError_t tm_weights(const TlArgs& a, cudaStream_t s)
{
    constexpr int PARTS = TmParts<T>::N, BLOCK = TW_ROWS * 128, SIZE = (int)sizeof(T);
    TwPlan p = {};
    const int most = PARTS == 1 ? 256 : 128, tiles = (a.outer + most - 1) / most;
    p.columns = tm_round((a.outer + tiles - 1) / tiles, 16);
    p.column_stride = tm_round(p.columns, 32);
    p.x_blocks = a.inner > 64 ? 2 : 1;
    p.y_blocks = (p.columns + 63) / 64;
    const int stage = (p.x_blocks + p.y_blocks) * PARTS * BLOCK;
    p.stages = std::min(TM_MAX_STAGES, (TM_SMEM - 1024 - TM_ROWS * 128) / stage);
    p.tensor_columns = tm_tensor_columns((PARTS == 1 ? 2 : 4) * p.column_stride);
    const bool wide = tm_on(a.x, a.x_row, SIZE, 16) && a.inner % 8 == 0 && tm_on(a.dy, a.dy_row, SIZE, 16) && a.outer % 8 == 0;
    p.vec = a.outer % 4 == 0 && tm_on(a.partial, 0, 4, 16);
    const dim3 grid((unsigned)tl_stretches(a.n, a.types, a.stretch), (a.inner + TM_ROWS - 1) / TM_ROWS, (a.outer + p.columns - 1) / p.columns);
    const int smem = 1024 + TM_ROWS * 128 + p.stages * stage;
    void (*const kernel)(TlArgs, TwPlan) = wide ? tm_weights_kernel<T, true> : tm_weights_kernel<T, false>;
    const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    kernel<<<grid, tm_threads(TW_FEED), smem, s>>>(a, p);
    return cudaGetLastError();
}

cudaError_t tl_mma_weights(const TlArgs& a, int dtype, cudaStream_t s)
{
    if (dtype == DYNB_F32) return tm_weights<float>(a, s);
    if (dtype == DYNB_F16) return tm_weights<__half>(a, s);
    return tm_weights<__nv_bfloat16>(a, s);
}

}  // namespace dynb
