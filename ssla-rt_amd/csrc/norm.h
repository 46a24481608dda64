// norm.h -- what the norms' kernels share: a group's mean and scale as three
// floats, and sums over the lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>

namespace ssla {

// A group's mean and 1 / sqrt(var + eps), of which
//     (x - mean) / sqrt(var + eps) = (2^-16 x - hi) scale - lo scale.
// hi + lo is the mean to 48 bits: hi alone would be off by up to 2^-25 of the
// mean, which is 0.03 standard deviations where the mean is 10^6 of them.
// 2^-16 x - hi, one fused operation, is finite for all finite x and mean; what it and lo
// lose of the smallest x lies below 2^-133.  scale, 2^16 / sqrt(var + eps), is a normal number
// for any larger spread, and overflows where sqrt(var + eps) is 2^-112 (1.9e-34) or less.
struct alignas(16) Norm {
    float hi, lo, scale;
};
constexpr float kDown = 0x1p-16f;

__device__ __forceinline__ Norm norm_of(double mean, double var, float eps) {
    const double s = var + (double)eps, m = mean * (double)kDown;
    // the instruction's root is good to some 2^-24; a Newton step doubles that,
    // except for 0 and infinity, where it gives a NaN
    const double r0 = __builtin_amdgcn_rsq(s), r1 = r0 * fma(-0.5 * s * r0, r0, 1.5);
    const double r = (r1 == r1 ? r1 : r0) / (double)kDown;
    const float hi = (float)m;
    return Norm{hi, (float)(m - (double)hi), (float)r};
}

// x + x of the lane that the DPP pattern names.
template <int CTRL>
__device__ __forceinline__ double plus_dpp(double x) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    u2 v = __builtin_bit_cast(u2, x);
    v[0] = __builtin_amdgcn_mov_dpp(v[0], CTRL, 0xf, 0xf, true);
    v[1] = __builtin_amdgcn_mov_dpp(v[1], CTRL, 0xf, 0xf, true);
    return x + __builtin_bit_cast(double, v);
}
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
    const int v = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
    return x + __builtin_bit_cast(float, v);
}
// Sum over the w lanes (a power of two up to 64) that share a group, in each of them,
// the first steps without LDS (30000 rows of 512 gated fp32 channels in 8 groups: 42 us, by
// shuffles alone 44).
template <class F>
__device__ __forceinline__ F lanes_sum(F x, int w) {
    if (w > 1) x = plus_dpp<0xb1>(x);            // lanes 1, 0, 3, 2 of four
    if (w > 2) x = plus_dpp<0x4e>(x);            // lanes 2, 3, 0, 1
    if (w > 4) x = plus_dpp<0x141>(x);           // eight lanes reversed
    if (w > 8) x = plus_dpp<0x140>(x);           // sixteen
    if (w > 16) x += __shfl_xor(x, 16);
    if (w > 32) x += __shfl_xor(x, 32);
    return x;
}

}  // namespace ssla
