// The rotation of the appends to a paged cache.
#pragma once

#include "common.hpp"

namespace muyo
{
/// cos and sin of the angle 2 pi (position * turns), times the magnitude. Far positions turn a pair
/// many times over, and only the fraction of a turn counts: the product and the fraction are in 64
/// bits (in 32, position 100000 would leave two digits less), cos and sin of the fraction in 32.
__device__ __forceinline__ void PairAngle(double turns, int32_t position, float magnitude, float& c, float& s)
{
    const double t = static_cast<double>(position) * turns;
    float sn, cs;
    sincospif(static_cast<float>(2.0 * (t - rint(t))), &sn, &cs);
    c = cs * magnitude;
    s = sn * magnitude;
}

__device__ __forceinline__ void Rotate(float x0, float x1, float c, float s, float& y0, float& y1)
{
    y0 = fmaf(x0, c, -(x1 * s));
    y1 = fmaf(x0, s, x1 * c);
}
}  // namespace muyo
