// The order of a row of logits: falling, equal ones by rising index.
#pragma once

#include "common.hpp"

namespace muyo
{
/// The order's upper word: rises with the value. -0 counts as +0, NaN comes before -inf.
__device__ __forceinline__ uint32_t OrderBits(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t ordered = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return v != v ? 0u : ordered;
}

/// A 64-bit key whose descending order is (value descending, index ascending). 0 is below every key.
__device__ __forceinline__ uint64_t OrderKey(float v, uint32_t index)
{
    return (static_cast<uint64_t>(OrderBits(v)) << 32) | static_cast<uint64_t>(~index);
}

__device__ __forceinline__ float KeyValue(uint64_t key)
{
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);  // 0 is a NaN
}
}  // namespace muyo
