// Attention of one new token per sequence over a paged fp16 cache.
#include <cmath>

#include "common.hpp"
#include "paged.hpp"

namespace muyo
{
namespace
{
constexpr int kBlock = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttentionArgs
{
    const float* q;
    const uint16_t* kcache;
    const uint16_t* vcache;
    float* out;
    const int32_t* tables;
    uint32_t sequences;
    uint32_t tablePages;
    const int32_t* querySequence;
    const int32_t* positions;
    uint32_t queries, heads, kvHeads;
    uint32_t pages, pageShift;
    uint32_t window;
    float scale;
};

/// One workgroup per (head, query): slices of kHd / 8 lanes own a key each, an online softmax a
/// slice, joined in LDS.
template <int kHd>
__global__ __launch_bounds__(kBlock) void PagedAttentionKernel(PagedAttentionArgs a)
{
    constexpr int kRC = kHd / 8;
    constexpr int kSlices = kBlock / kRC;
    __shared__ float sliceMax[kSlices];
    __shared__ float sliceSum[kSlices];
    __shared__ float sliceAcc[kSlices][kHd];

    const uint32_t head = blockIdx.x;
    const uint32_t query = blockIdx.y;
    const int32_t row = a.querySequence[query];
    if (row < 0 || static_cast<uint32_t>(row) >= a.sequences)
    {
        return;  // padding
    }
    const uint32_t g = head / (a.heads / a.kvHeads);
    const uint32_t slice = threadIdx.x / kRC;
    const uint32_t part = threadIdx.x % kRC;
    const uint32_t pageSize = 1u << a.pageShift;
    const uint32_t capacity = a.tablePages << a.pageShift;
    const int32_t position = a.positions[query];
    const uint32_t end = position < 0 ? 0 : min(static_cast<uint32_t>(position) + 1, capacity);
    const uint32_t begin = a.window != 0 && position >= 0 && static_cast<uint32_t>(position) + 1 > a.window
                               ? static_cast<uint32_t>(position) + 1 - a.window
                               : 0;
    float qv[8];
    const float* qh = a.q + (static_cast<uint64_t>(query) * a.heads + head) * kHd + part * 8;
#pragma unroll
    for (int c = 0; c < 8; ++c)
    {
        qv[c] = qh[c];
    }
    float m = -INFINITY;
    float l = 0.0f;
    float acc[8] = {};
    const int32_t* table = a.tables + static_cast<uint64_t>(row) * a.tablePages;
    for (uint32_t key = begin + slice; key < end; key += kSlices)
    {
        const uint32_t page = static_cast<uint32_t>(table[key >> a.pageShift]);
        if (page >= a.pages)
        {
            continue;
        }
        const uint64_t at =
            ((((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + (key & (pageSize - 1))) * kHd) + part * 8;
        float kv[8], vv[8];
        LoadHalf8(a.kcache + at, kv);
        LoadHalf8(a.vcache + at, vv);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c)
        {
            s = fmaf(qv[c], kv[c], s);
        }
        s = GroupSum<kRC>(s) * (a.scale * kLog2e);
        const float top = fmaxf(m, s);
        const float factor = m == top ? 1.0f : exp2f(m - top);
        const float p = s == top ? 1.0f : exp2f(s - top);
        l = fmaf(l, factor, p);
        m = top;
#pragma unroll
        for (int c = 0; c < 8; ++c)
        {
            acc[c] = fmaf(p, vv[c], acc[c] * factor);
        }
    }
    if (part == 0)
    {
        sliceMax[slice] = m;
        sliceSum[slice] = l;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
    {
        sliceAcc[slice][part * 8 + c] = acc[c];
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < kHd; d += kBlock)
    {
        float top = -INFINITY;
        for (int s = 0; s < kSlices; ++s)
        {
            top = fmaxf(top, sliceMax[s]);
        }
        float num = 0.0f;
        float den = 0.0f;
        for (int s = 0; s < kSlices; ++s)
        {
            const float w = sliceMax[s] == top ? 1.0f : exp2f(sliceMax[s] - top);
            if (sliceSum[s] != 0.0f)  // a slice without keys; NaN counts
            {
                num = fmaf(w, sliceAcc[s][d], num);
                den = fmaf(w, sliceSum[s], den);
            }
        }
        a.out[(static_cast<uint64_t>(query) * a.heads + head) * kHd + d] = den == 0.0f ? 0.0f : num / den;
    }
}

bool AttentionShape(uint32_t queries, uint32_t heads, uint32_t kvHeads, uint32_t headDim)
{
    return queries >= 1 && queries <= 65535 && kvHeads >= 1 && heads >= 1 && heads % kvHeads == 0 &&
           heads / kvHeads <= 16 && heads <= 1024 && (headDim == 64 || headDim == 128);
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_paged_attention_decode_f16kv_workspace_bytes(uint32_t queries, uint32_t heads,
                                                                    uint32_t kv_heads, uint32_t head_dim)
{
    return AttentionShape(queries, heads, kv_heads, head_dim) ? 16 : 0;
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
    if (q == nullptr || kcache == nullptr || vcache == nullptr || out == nullptr || tables == nullptr ||
        query_sequence == nullptr || positions == nullptr)
    {
        return Fail(MUYO_E_NULL, "%s: every buffer is required", name);
    }
    const int checked = CheckPages(name, pages, page_size);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    if (!AttentionShape(queries, heads, kv_heads, head_dim))
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: needs 1..65535 queries, heads %% kv_heads == 0, at most 16 heads per kv "
                                        "head and 1024 in all, head_dim 64 or 128",
                    name);
    }
    if (sequences == 0 || table_pages == 0 || static_cast<uint64_t>(table_pages) * page_size > 0x7FFFFFFFull)
    {
        return Fail(MUYO_E_RANGE, "%s: needs sequences >= 1 and table_pages * page_size in 1..2^31 - 1", name);
    }
    if (!Aligned16(q) || !Aligned16(kcache) || !Aligned16(vcache) || !Aligned16(out))
    {
        return Fail(MUYO_E_CONTRACT, "%s: q, out and the caches must be 16-byte aligned", name);
    }
    const size_t need = muyo_paged_attention_decode_f16kv_workspace_bytes(queries, heads, kv_heads, head_dim);
    if (workspace == nullptr || !Aligned16(workspace) || workspace_bytes < need)
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a 16-byte aligned workspace of %zu bytes (got %llu)", name, need,
                    static_cast<unsigned long long>(workspace_bytes));
    }
    PagedAttentionArgs a{q, static_cast<const uint16_t*>(kcache), static_cast<const uint16_t*>(vcache), out, tables,
                         sequences, table_pages, query_sequence, positions, queries, heads, kv_heads, pages, 0, window,
                         scale};
    while ((1u << a.pageShift) < page_size)
    {
        ++a.pageShift;
    }
    if (head_dim == 64)
    {
        hipLaunchKernelGGL(PagedAttentionKernel<64>, dim3(heads, queries), dim3(kBlock), 0, AsStream(stream), a);
    }
    else
    {
        hipLaunchKernelGGL(PagedAttentionKernel<128>, dim3(heads, queries), dim3(kBlock), 0, AsStream(stream), a);
    }
    return LaunchStatus(name);
}
