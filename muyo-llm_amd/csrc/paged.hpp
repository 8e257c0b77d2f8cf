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
}  // namespace muyo
