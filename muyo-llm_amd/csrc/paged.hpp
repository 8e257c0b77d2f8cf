// What the operators over a paged cache share on the host.
#pragma once

#include <cstdint>

#include "common.hpp"

namespace muyo
{
constexpr uint32_t kMinPageSize = 16;
constexpr uint32_t kMaxPageSize = 1024;

/// MUYO_OK for a power-of-two page size in kMinPageSize..kMaxPageSize and fewer than 2^31 slots,
/// else the failure's status.
int CheckPages(const char* name, uint32_t pages, uint32_t pageSize);

/// The arguments that the appends have in common.
struct AppendCall
{
    const float* q;
    const float* k;
    const float* v;
    uint64_t qStride, kStride, vStride;
    float* qOut;
    const int32_t* positions;
    const int32_t* slots;
    uint32_t tokens, heads, kvHeads, headDim;
    uint32_t pages, pageSize;
    uint32_t layout;
    uint32_t rotary;
    const double* turns;
    float magnitude;
    uint64_t threads;  // of its launch
};

/// MUYO_OK, or the status of the first part of an append's contract that the call breaks. `caches`: what it
/// writes besides q_out.
int CheckAppend(const char* name, const AppendCall& call, const Range* caches, int cacheCount);
}  // namespace muyo
