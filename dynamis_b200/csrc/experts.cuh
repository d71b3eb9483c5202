// What the kernels of the products by expert share.
#pragma once

#include <algorithm>

#include "type_linear.cuh"

namespace dynb {

// Pairs p = (row, choice), numbered row * choices + choice.  A pair reads row p / fan of x (fan = choices, or 1 where x is of pairs).
struct ExArgs {
    TlArgs t;                  // x, w, b, dy, order, start; n: pairs; y: result, dx: gradient of x by pairs
    void* slope;               // the activation's slope, [pairs, outer rounded up to 8], or null
    void* du;                  // room for dz times the slope, [pairs, outer], or null
    int64_t n_in;              // rows of x
    int64_t out_row;           // elements from row to row of the results of a rows' pass, and forward of the slopes
    int fan, activation;
};

// The activation's slope beside 16-bit results, in 16 bits (slopes lie in [-0.129, 1.13]).  From 1/8 on: steps of 2^-14, the numbers 0x3000 and on, off by 2^-15 at most (a 16-bit
// float would be off by as much as the result's own rounding, and the gradient with it); 0 and 1 are kept as they are.  Below: an fp16 number, 31/32 of the slope, so that no negative one
// reaches 1/8, where its steps would be twice as wide; off by 2^-11 of the slope, or 2^-25 where that is more.  (In steps of 2^-14 throughout, SiLU's slopes
// from u = -13 on were zero, and 7 % off at -10.)  NaN stays one: arithmetic gives 0x7fff, behind the steps.
constexpr float EX_SLOPE_SCALE = 31.0f / 32.0f;
__device__ __forceinline__ uint32_t ex_slopes_bits(float v0, float v1)
{
    const __half2 h = __floats2half2_rn(v0 * EX_SLOPE_SCALE, v1 * EX_SLOPE_SCALE);
    const uint32_t small = *reinterpret_cast<const uint32_t*>(&h);
    // the lowest bits of 2^23 + a whole number are that number
    const uint32_t s0 = __float_as_uint(fmaf(v0, 16384.0f, 8388608.0f + 12288.0f - 2048.0f)), s1 = __float_as_uint(fmaf(v1, 16384.0f, 8388608.0f + 12288.0f - 2048.0f));
    return __byte_perm(v0 >= 0.125f ? s0 : small, v1 >= 0.125f ? s1 : small >> 16, 0x5410);
}
__device__ __forceinline__ float2 ex_slopes_of(uint32_t pair)
{
    const float2 small = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    const uint32_t b0 = pair & 0xffffu, b1 = pair >> 16;
    const float s0 = fmaf(__uint_as_float(0x4b000000u | b0), 1.0f / 16384.0f, -512.625f), s1 = fmaf(__uint_as_float(0x4b000000u | b1), 1.0f / 16384.0f, -512.625f);
    return make_float2(b0 - 0x3000u < 0x4800u ? s0 : small.x * (1.0f / EX_SLOPE_SCALE), b1 - 0x3000u < 0x4800u ? s1 : small.y * (1.0f / EX_SLOPE_SCALE));
}

__device__ __forceinline__ float ex_inverse(float v)   // to within an unit in the last place; 0 of an infinity
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// The activation and its slope.  Exponentials by the fast route: off by 2 + |u| units in the last place of 1 + e^-u.  The normal distribution function by formula
// 7.1.26 of Abramowitz and Stegun, off by 7.5e-8, whose exponential the slope shares.
template <int ACTIVATION>
__device__ __forceinline__ float ex_activate(float u, float* slope)
{
    if constexpr (ACTIVATION == DYNB_ACTIVATION_SILU) {
        const float p = ex_inverse(1.0f + __expf(-u));
        const float z = u * p;
        *slope = fmaf(z, 1.0f - p, p);
        return z;
    } else {
        const float x = fabsf(u) * 0.70710678118654752f, t = ex_inverse(fmaf(0.3275911f, x, 1.0f)), e = __expf(-x * x);
        const float tail = 0.5f * e * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        const float p = u < 0.0f ? tail : 1.0f - tail;
        *slope = fmaf(u * 0.3989422804014327f, e, p);
        return u * p;
    }
}

// Rows of places without an expert are set to zero, `wide` bytes a row (16: whole pieces of 16 bytes), by warp `warp` of `warps`: it looks at 32 places at a time.
__device__ __forceinline__ void ex_clear_absent(const TlArgs& a, void* out, int64_t wide, int piece, int64_t warp, int64_t warps)
{
    const int lane = threadIdx.x & 31;
    for (int64_t at = min(max((int64_t)a.start[a.types], (int64_t)0), a.n) + 32 * warp; at < a.n; at += 32 * warps) {
        const int32_t mine = at + lane < a.n ? a.order[at + lane] : -1;
        for (int i = 0; i < 32; i++) {
            const int32_t p = __shfl_sync(0xffffffffu, mine, i);
            if ((uint32_t)p >= (uint64_t)a.n) continue;
            unsigned char* const row = static_cast<unsigned char*>(out) + p * wide;
            if (piece == 16) {
                for (int64_t c = 16 * lane; c < wide; c += 512) *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
            } else {
                for (int64_t c = 2 * lane; c < wide; c += 64) *reinterpret_cast<uint16_t*>(row + c) = 0;
            }
        }
    }
}

// experts_mma.cu: the products on the tensor cores.  `packed`: room for the matrices as the kernel reads them, on 16 bytes.
int64_t ex_packed_bytes(const ExArgs& e, int back, int dtype);
cudaError_t ex_mma_rows(const ExArgs& e, int back, int dtype, void* packed, cudaStream_t s);   // back: du goes to e.du as well, where it is not null
cudaError_t ex_mma_weights(const ExArgs& e, int dtype, cudaStream_t s);
int64_t ex_stretches(const ExArgs& e);

// The weights' gradient: slices of the pairs that run beside one another, as many as its tiles leave SMs for.
static inline int ex_slices(int inner, int outer, int size)
{
    const int most = size == 4 ? 128 : 256;
    return std::max(1, sm_count_cached() / std::max(1, ((inner + 127) / 128) * ((outer + most - 1) / most)));
}
// Pairs that one sum takes: a slice, or an equal part of it, of at most 1024 pairs in fp32 (a sum in tensor memory is one chain of additions that are cut off: operands of one sign
// lose 1.7e-6 of it) and 8192 in 16 bits, unless the sums would take more than twice the room of the rows.  In 16 bits the products are cut, too, where they end below the sum's last place:
// 7500 pairs lose 4.5e-5 in fp16 and 2.8e-5 in bf16, a tenth and a hundredth of half a step of the results.
static inline int ex_stretch(int64_t n, int inner, int outer, int dtype)
{
    const int64_t most = std::max<int64_t>(dtype == DYNB_F32 ? 1024 : 8192, (int64_t)inner * outer / (2 * ((int64_t)inner + outer)));
    const int slices = ex_slices(inner, outer, dtype == DYNB_F32 ? 4 : 2);
    const int64_t slice = std::max<int64_t>(256, (n + slices - 1) / slices), parts = (slice + most - 1) / most;
    return (int)(((slice + parts - 1) / parts + 31) / 32 * 32);
}

}  // namespace dynb
