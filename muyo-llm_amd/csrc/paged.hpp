// What the operators over a paged cache share on the host.
#pragma once

#include <cstdint>

namespace muyo
{
constexpr uint32_t kMinPageSize = 16;
constexpr uint32_t kMaxPageSize = 1024;

/// MUYO_OK for a power-of-two page size in kMinPageSize..kMaxPageSize and fewer than 2^31 slots,
/// else the failure's status.
int CheckPages(const char* name, uint32_t pages, uint32_t pageSize);

/// One buffer of a call, for the overlap check.
struct Range
{
    const void* at;
    uint64_t bytes;
    const char* name;
};

inline bool Overlap(const Range& a, const Range& b)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at);
    const uintptr_t y = reinterpret_cast<uintptr_t>(b.at);
    return x < y + b.bytes && y < x + a.bytes;
}

/// A call's rows of `bytes` each, `stride` bytes apart: other buffers may lie between them.
struct Rows
{
    const void* at;
    uint64_t bytes;
    uint64_t stride;
    uint64_t count;
    const char* name;
};

inline bool Overlap(const Range& a, const Rows& b)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at);
    const uintptr_t y = reinterpret_cast<uintptr_t>(b.at);
    // The first row that ends behind the range's begin: it overlaps, or none does.
    const uint64_t row = x < y + b.bytes ? 0 : (x - y - b.bytes) / b.stride + 1;
    return row < b.count && y + row * b.stride < x + a.bytes;
}
}  // namespace muyo
