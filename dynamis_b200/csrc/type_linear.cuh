// What the kernels of the products by type share: arguments, pieces of rows by type, loads and stores of the three types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace dynb {

struct TlArgs {
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *db;
    float* partial;
    const int32_t *order, *start;
    uint32_t* status;
    int64_t n, x_row, dy_row;
    int types, inner, outer;
    int stretch;               // rows of a type whose products one block sums
};

__device__ __forceinline__ float tl_get(const float* p) { return *p; }
__device__ __forceinline__ float tl_get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float tl_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void tl_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void tl_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void tl_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

struct TlTile { int type; int64_t begin, end; };   // places in `order`

// The rows of type t: places [s0, s1) of `order`, inside it whatever `start` holds.
__device__ __forceinline__ void tl_rows_of(const TlArgs& a, int t, int64_t* s0, int64_t* s1)
{
    *s0 = max(a.start[t], 0);
    *s1 = max(min((int64_t)a.start[t + 1], a.n), *s0);
}

// The tile-th piece of `per` rows when every type's rows are cut into such pieces; type < 0 behind the last.  All lanes of a warp call it.
// `pieces` (optional): their number, when `tile` is behind the last.
__device__ __forceinline__ TlTile tl_tile(const TlArgs& a, int64_t tile, int per, int64_t* pieces = nullptr)
{
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int t0 = 0; t0 < a.types; t0 += 32) {
        const int t = t0 + lane;
        int64_t s0 = 0, s1 = 0;
        if (t < a.types) tl_rows_of(a, t, &s0, &s1);
        const int mine = (int)((s1 - s0 + per - 1) / per);
        int total;
        const int excl = warp_excl_scan(mine, lane, &total);
        const bool here = tile >= before + excl && tile < before + excl + mine;
        const uint32_t found = __ballot_sync(0xffffffffu, here);
        if (found != 0) {
            const int from = __ffs(found) - 1;
            const int64_t begin = s0 + (tile - before - excl) * per;
            TlTile r;
            r.type = t0 + from;
            r.begin = __shfl_sync(0xffffffffu, begin, from);
            r.end = min(r.begin + per, __shfl_sync(0xffffffffu, s1, from));
            return r;
        }
        before += total;
    }
    if (pieces != nullptr) *pieces = before;
    return {-1, 0, 0};
}

// Rows of a stretch: four blocks an SM where there are as many rows, no fewer than 256, and no more than 1024 (a sum in tensor memory is one chain of
// additions that are cut off), unless the stretches' sums would take more than twice the room of the rows.
static inline int tl_stretch(int64_t n, int inner, int outer, int dtype)
{
    const int64_t tiles = (int64_t)((inner + 127) / 128) * ((outer + (dtype == DYNB_F32 ? 127 : 255)) / (dtype == DYNB_F32 ? 128 : 256));
    const int64_t rows = n * tiles / (148 * 4) + 1, most = std::max<int64_t>(1024, (int64_t)inner * outer / (2 * ((int64_t)inner + outer)));
    return (int)((std::min<int64_t>(most, std::max<int64_t>(256, rows)) + 31) / 32 * 32);
}
// An upper bound: every type with rows has one stretch that is not full.
static inline int64_t tl_stretches(int64_t n, int types, int stretch) { return n / stretch + std::min<int64_t>(n, types) + 1; }

// type_linear_mma.cu: the products on the tensor cores.  False: the widths are too large for it (nothing was launched).
bool tl_mma_rows(const TlArgs& a, int back, int dtype, cudaStream_t s, cudaError_t* rc);
cudaError_t tl_mma_weights(const TlArgs& a, int dtype, cudaStream_t s);

}  // namespace dynb
