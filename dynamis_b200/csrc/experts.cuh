// What the kernels of the products by expert share.
#pragma once

#include "type_linear.cuh"

namespace dynb {

// Pairs p = (row, choice), numbered row * choices + choice.  A pair reads row p / fan of x (fan = choices, or 1 where x is of pairs).
struct ExArgs {
    TlArgs t;                  // x, w, b, dy, order, start; n: pairs; y: result, dx: gradient of x by pairs
    void* slope;               // the activation's slope, [pairs, outer], or null
    int64_t n_in;              // rows of x
    int fan, activation;
};

// The activation's slope beside 16-bit results: steps of 2^-14 from -0.5 on, as 16 bits (slopes lie in [-0.13, 1.13]); all bits set for NaN.  It is off by
// 2^-15 at most, and 0 and 1 are kept as they are.  (As a 16-bit float it would be off by as much as the result's own rounding, and the gradient with it.)
__device__ __forceinline__ uint16_t ex_slope_bits(float v) { return isnan(v) ? 0xffffu : (uint16_t)__float2int_rn(fmaf(v, 16384.0f, 8192.0f)); }
__device__ __forceinline__ float ex_slope_of(uint32_t bits) { return bits == 0xffffu ? NAN : fmaf(__uint_as_float(0x4b000000u | bits), 1.0f / 16384.0f, -512.5f); }   // 2^23 + bits, exactly

__device__ __forceinline__ float ex_activate(float u, int activation, float* slope)
{
    if (activation == DYNB_ACTIVATION_SILU) {
        const float p = 1.0f / (1.0f + expf(-u));
        *slope = p * (1.0f + u * (1.0f - p));
        return u * p;
    }
    if (activation == DYNB_ACTIVATION_GELU) {
        const float p = normcdff(u);
        *slope = fmaf(u, 0.3989422804014327f * expf(-0.5f * u * u), p);
        return u * p;
    }
    *slope = 1.0f;
    return u;
}

}  // namespace dynb
