// Numbers as 8-bit integers with a scale: q = rint(x / scale) in [-127, 127], scale = max |x| / 127, both in 32 bits, ties to even.
#pragma once

#include "frame_columns.cuh"

namespace bb200 {

__device__ __forceinline__ float quant_scale(uint32_t abs_bits)
{
    return abs_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(__uint_as_float(abs_bits), 127.0f);
}

__device__ __forceinline__ int quantize(float x, float scale)
{
    if (!(scale > 0.0f)) return 0;                        // zeros, or not finite
    return max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale))));
}

// Four numbers of a frame as a word of q.  x / scale comes through the reciprocal, off by less than 1e-4, and is rounded by adding 1.5 * 2^23, which
// leaves the integer in the lowest byte; where that could have decided the rounding, and for scales without a normal reciprocal, the quotient is divided
// out.  (The kernels are bound by their instructions, and the division costs more than all the rest.)
struct Quantizer {
    float scale, inv;
    bool plain;
    __device__ explicit Quantizer(float s) : scale(s), inv(1.0f / s), plain(s > 1e-36f && s < 1e36f) {}
    __device__ uint32_t operator()(float x0, float x1, float x2, float x3) const
    {
        constexpr float kRound = 12582912.0f;
        const float x[4] = {x0, x1, x2, x3};
        float worst = 0.0f;
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = x[i] * inv, n = t + kRound;
            worst = fmaxf(worst, fabsf(t - (n - kRound)));
            r[i] = __float_as_uint(n);
        }
        if (worst > 0.4999f || !plain) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (uint32_t)quantize(x[i], scale);
        }
        return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    }
};

// the larger of the magnitudes of packed numbers, as integers: infinities and NaN are on top
template <typename T> __device__ __forceinline__ uint32_t packed_abs_max(uint32_t a, uint32_t b)
{
    return sizeof(T) == 4 ? max(a, b & 0x7fffffffu) : __vmaxu2(a, b & 0x7fff7fffu);
}

}   // namespace bb200
