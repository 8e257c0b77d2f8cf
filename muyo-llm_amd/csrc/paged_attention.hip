// Attention of single tokens over a paged fp16 cache, many sequences of any lengths in one call.
#include <cmath>

#include "paged_attention_f16.hpp"

namespace muyo
{
namespace
{
template <int kHd, bool kSplit>
__global__ __launch_bounds__(kBlock, kHd == 64 ? (kSplit ? 3 : 4) : 2) void PagedAttentionKernel(
    PagedAttentionF16Args a)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kOwnKeysBytes<kHd>];
    __shared__ OwnKeysSpace space;
    OwnKeys<kHd, kSplit, false>(a, blockIdx.x, blockIdx.y, lds, space);
}
}  // namespace

int CheckAttention(const char* name, const AttentionCall& c, const Range* more, int moreCount, int aligned)
{
    bool missing = c.q == nullptr || c.out == nullptr || c.tables == nullptr || c.querySequence == nullptr ||
                   c.positions == nullptr;
    bool wide = Aligned16(c.q) && Aligned16(c.out);
    for (int i = 0; i < moreCount; ++i)
    {
        missing = missing || more[i].at == nullptr;
        wide = wide && (i >= aligned || Aligned16(more[i].at));
    }
    if (missing)
    {
        return Fail(MUYO_E_NULL, "%s: every buffer is required", name);
    }
    const int checked = CheckPages(name, c.pages, c.pageSize);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    if (!AttentionShape(c.queries, c.heads, c.kvHeads, c.headDim))
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: needs 1..65535 queries, heads %% kv_heads == 0, at most 16 heads per kv "
                                        "head and 1024 in all, head_dim 64 or 128",
                    name);
    }
    if (c.sequences == 0 || c.tablePages == 0 || static_cast<uint64_t>(c.tablePages) * c.pageSize > 0x7FFFFFFFull)
    {
        return Fail(MUYO_E_RANGE, "%s: needs sequences >= 1 and table_pages * page_size in 1..2^31 - 1", name);
    }
    if (!wide || !std::isfinite(c.scale))
    {
        return Fail(MUYO_E_CONTRACT, "%s: q, out and the caches must be 16-byte aligned, and scale finite", name);
    }
    if (c.workspace == nullptr || !Aligned16(c.workspace) || c.workspaceBytes < c.need)
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a 16-byte aligned workspace of %llu bytes (got %llu)", name,
                    static_cast<unsigned long long>(c.need), static_cast<unsigned long long>(c.workspaceBytes));
    }
    const uint64_t rowsBytes = 4ull * c.queries * c.heads * c.headDim;
    const Range out{c.out, rowsBytes, "out"};
    const Range space{c.workspace, c.need, "workspace"};
    // The positions, sequences and tables are read again while other workgroups write.
    const Range lists[] = {{c.q, rowsBytes, "q"},
                           {c.tables, 4ull * c.sequences * c.tablePages, "tables"},
                           {c.querySequence, 4ull * c.queries, "query_sequence"},
                           {c.positions, 4ull * c.queries, "positions"}};
    if (Overlap(out, space))
    {
        return Fail(MUYO_E_CONTRACT, "%s: out overlaps workspace", name);
    }
    for (const Range* w : {&out, &space})
    {
        for (const Range& r : lists)
        {
            // In place a workgroup has read its (query, kv head)'s q when it writes its output there, and one that
            // is cut is written by the join.
            const bool inPlace = w == &out && &r == lists && c.q == c.out;
            if (!inPlace && Overlap(*w, r))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w->name, r.name);
            }
        }
        for (int i = 0; i < moreCount; ++i)
        {
            if (Overlap(*w, more[i]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w->name, more[i].name);
            }
        }
    }
    return MUYO_OK;
}
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_paged_attention_decode_f16kv_workspace_bytes(uint32_t queries, uint32_t heads,
                                                                    uint32_t kv_heads, uint32_t head_dim)
{
    if (!AttentionShape(queries, heads, kv_heads, head_dim))
    {
        return 0;
    }
    return DecodeWorkspaceBytes(queries, heads, kv_heads, head_dim);
}

extern "C" int muyo_paged_attention_decode_f16kv(const float* q, const void* kcache, const void* vcache, float* out,
                                                 const int32_t* tables, uint32_t sequences, uint32_t table_pages,
                                                 const int32_t* query_sequence, const int32_t* positions,
                                                 uint32_t queries, uint32_t heads, uint32_t kv_heads,
                                                 uint32_t head_dim, uint32_t pages, uint32_t page_size,
                                                 uint32_t window, float scale, void* workspace,
                                                 uint64_t workspace_bytes, void* stream)
{
    const char* name = "paged_attention_decode_f16kv";
    const uint64_t cacheBytes = 2ull * pages * page_size * kv_heads * head_dim;
    const Range caches[] = {{kcache, cacheBytes, "kcache"}, {vcache, cacheBytes, "vcache"}};
    const AttentionCall call{q, out, tables, sequences, table_pages, query_sequence, positions, queries, heads,
                             kv_heads, head_dim, pages, page_size, scale, workspace, workspace_bytes,
                             muyo_paged_attention_decode_f16kv_workspace_bytes(queries, heads, kv_heads, head_dim)};
    const int checked = CheckAttention(name, call, caches, 2, 2);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    PagedAttentionF16Args a{};
    FillAttentionArgs(a, call, window);
    a.kcache = static_cast<const uint16_t*>(kcache);
    a.vcache = static_cast<const uint16_t*>(vcache);
    const hipError_t launched =
        head_dim == 64 ? LaunchPagedAttention<64, kTile>(AsStream(stream), a, PagedAttentionKernel<64, false>,
                                                                PagedAttentionKernel<64, true>)
                       : LaunchPagedAttention<128, kTile>(AsStream(stream), a,
                                                                 PagedAttentionKernel<128, false>,
                                                                 PagedAttentionKernel<128, true>);
    return launched == hipSuccess ? MUYO_OK : HipStatus(launched, name);
}
