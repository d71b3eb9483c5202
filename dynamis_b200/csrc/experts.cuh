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
// The lowest bits of 2^23 + a whole number are that number; of a NaN that arithmetic makes they are all set.
__device__ __forceinline__ uint32_t ex_slope_bits(float v) { return __float_as_uint(fmaf(v, 16384.0f, 8388608.0f + 8192.0f)); }   // the lower 16
__device__ __forceinline__ float ex_slope_of(uint32_t bits) { return bits == 0xffffu ? NAN : fmaf(__uint_as_float(0x4b000000u | bits), 1.0f / 16384.0f, -512.5f); }

// The activation and its slope.  Exponentials by the fast route: off by 2 + |u| units in the last place of 1 + e^-u.  The normal distribution function by formula
// 7.1.26 of Abramowitz and Stegun, off by 7.5e-8, whose exponential the slope shares.
__device__ __forceinline__ float ex_activate(float u, int activation, float* slope)
{
    if (activation == DYNB_ACTIVATION_SILU) {
        const float p = __fdividef(1.0f, 1.0f + __expf(-u));
        const float z = u * p;
        *slope = fmaf(z, 1.0f - p, p);
        return z;
    }
    if (activation == DYNB_ACTIVATION_GELU) {
        const float x = fabsf(u) * 0.70710678118654752f, t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f)), e = __expf(-x * x);
        const float tail = 0.5f * e * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        const float p = u < 0.0f ? tail : 1.0f - tail;
        *slope = fmaf(u * 0.3989422804014327f, e, p);
        return u * p;
    }
    *slope = 1.0f;
    return u;
}

// Rows of places without an expert are set to zero, `wide` bytes a row, by `threads` threads of every block of row `blockIdx.y` 0.
__device__ __forceinline__ void ex_clear_absent(const TlArgs& a, void* out, int64_t wide, int thread, int threads)
{
    const int64_t from = min(max((int64_t)a.start[a.types], (int64_t)0), a.n);
    for (int64_t at = from + blockIdx.x; at < a.n; at += gridDim.x) {
        const int32_t p = a.order[at];
        if ((uint32_t)p >= (uint64_t)a.n) continue;
        uint16_t* const row = reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(out) + p * wide);
        for (int64_t i = thread; i < wide / 2; i += threads) row[i] = 0;
    }
}

// experts_mma.cu: the products on the tensor cores.  `packed`: room for the matrices as the kernel reads them, on 16 bytes.
int64_t ex_packed_bytes(const ExArgs& e, int back, int dtype);
cudaError_t ex_mma_rows(const ExArgs& e, int back, int dtype, void* packed, cudaStream_t s);
cudaError_t ex_mma_weights(const ExArgs& e, int dtype, cudaStream_t s);
int64_t ex_stretches(const ExArgs& e);

}  // namespace dynb
