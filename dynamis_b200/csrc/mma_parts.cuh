// What the products of gathered rows on the tensor cores share: operands in parts, their way into the tiles, the walk over pieces of rows by type.
#pragma once

#include <type_traits>

#include "type_linear.cuh"
#include "umma.cuh"

namespace dynb {

constexpr int TM_ROWS = 128;

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

static inline int tm_round(int v, int to) { return (v + to - 1) / to * to; }
static inline int tm_tensor_columns(int need)
{
    int c = 32;
    while (c < need) c *= 2;
    return c;
}
static inline bool tm_on(const void* p, int64_t row, int size, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && row * size % bytes == 0; }

}  // namespace dynb
