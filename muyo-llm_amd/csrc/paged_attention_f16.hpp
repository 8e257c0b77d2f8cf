// The fp16 cache's attention over each query's own keys, for the one that joins it with a shared prefix.
#pragma once

#include "paged_attention_core.hpp"

namespace muyo
{
struct PagedAttentionF16Args : PagedAttentionArgs
{
    const uint16_t* kcache;
    const uint16_t* vcache;
};

/// muyo_paged_attention_decode_f16kv's launches, with `stats` written.
template <int kHd>
hipError_t LaunchOwnKeys(hipStream_t s, const PagedAttentionF16Args& a);

extern template hipError_t LaunchOwnKeys<64>(hipStream_t, const PagedAttentionF16Args&);
extern template hipError_t LaunchOwnKeys<128>(hipStream_t, const PagedAttentionF16Args&);
}  // namespace muyo
