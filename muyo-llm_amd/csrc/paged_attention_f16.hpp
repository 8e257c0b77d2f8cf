// The fp16 cache's attention over each query's own keys, for the one that joins it with a shared prefix.
#pragma once

#include "paged_attention_core.hpp"

namespace muyo
{
// Softmax weights over own keys are held in two planes of f16, which ends at 2^16: the weight of the maximum is
// 2^kWeightBias, and 2^15 when a later one has run kLag binary orders ahead.
constexpr float kLag = 4.0f;
constexpr float kWeightBias = 15.0f - kLag;

struct PagedAttentionF16Args : PagedAttentionArgs
{
    const uint16_t* kcache;
    const uint16_t* vcache;
};

/// muyo_paged_attention_decode_f16kv's launches but for the join of what shares cut: OwnKeysSplit says if there is any.
/// What no share cut is in `out` and `stats`.
template <int kHd>
hipError_t LaunchOwnKeys(hipStream_t s, const PagedAttentionF16Args& a);

bool OwnKeysSplit(const PagedAttentionF16Args& a);

extern template hipError_t LaunchOwnKeys<64>(hipStream_t, const PagedAttentionF16Args&);
extern template hipError_t LaunchOwnKeys<128>(hipStream_t, const PagedAttentionF16Args&);
}  // namespace muyo
