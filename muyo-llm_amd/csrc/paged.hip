// A cache in pages: the plan of a step (block tables, the ring of free pages, slots of new tokens)
// and rope + append into the slots. The attention over the pages is in paged_attention.hip.
//
// A cache is [pages][kv_heads][page_size][head_dim] fp16; slot s is row s % page_size of page
// s / page_size; row b of a table [sequences][table_pages] names sequence b's pages in order.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "paged.hpp"

namespace muyo
{
namespace
{
constexpr uint32_t kMaxPlanSequences = 4096;
constexpr uint32_t kMaxPlanTokens = 1u << 24;
constexpr uint32_t kSmallPlan = 1024;  // sequences that workgroups of 256 threads plan

struct PlanArgs
{
    const int32_t* lengths;
    const int32_t* targets;
    uint32_t sequences;
    int32_t* tables;
    uint32_t tablePages;
    int32_t* freePages;
    const int32_t* pool;  // head of the ring, free pages in it
    uint32_t pages;
    uint32_t pageShift;
    uint32_t tokens;
    int32_t* granted;
    int32_t* poolOut;
    int32_t* starts;
    int32_t* tokenSequence;
    int32_t* positions;
    int32_t* slots;
    uint32_t lists;  // write tables, ring, starts and the tokens' lists
    uint32_t state;  // write granted and poolOut
};

/// Inclusive sums over the workgroup's threads of N 64-bit values each, in thread order.
template <int kThreads, int N>
__device__ __forceinline__ void BlockInclusiveSum(uint64_t (&v)[N], uint64_t (*waveSum)[N])
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
    const uint32_t wave = threadIdx.x / kWave;
#pragma unroll
    for (uint32_t step = 1; step < kWave; step *= 2)
    {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            const uint64_t other = __shfl_up(static_cast<unsigned long long>(v[n]), step);
            v[n] += lane >= step ? other : 0;
        }
    }
    __syncthreads();  // the previous sums' readers are done
    if (lane == kWave - 1)
    {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            waveSum[wave][n] = v[n];
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / kWave; ++w)
    {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            v[n] += w < wave ? waveSum[w][n] : 0;
        }
    }
}

/// The b with sums[b] <= i < sums[b + 1] (sums[0] = 0, i < sums[n]).
__device__ __forceinline__ uint32_t OwnerOf(const uint32_t* sums, uint32_t n, uint32_t i)
{
    uint32_t low = 0;
    uint32_t high = n;
    while (high - low > 1)
    {
        const uint32_t mid = (low + high) / 2;
        if (sums[mid] <= i)
        {
            low = mid;
        }
        else
        {
            high = mid;
        }
    }
    return low;
}

/// The plan of a step. Sequences are served in order; with l and t their length and target, P the
/// page size, one gets what it asks for if its new tokens fit in the lists behind those of all before it
/// (sum max(0, t - l) <= tokens) and its new pages, need = max(0, ceil(t/P) - ceil(l/P)), in what the
/// sums of the needs before leave of the ring. Both sums only grow, so those that get pages are the
/// first ones that ask for any.
///
/// Every workgroup makes the sums over all the sequences itself (three dependent ones, kPer sequences a
/// thread, in 64 bits) and then takes its share of the tokens, pages taken and pages given back,
/// finding an item's sequence in the sums by bisection: nothing passes between workgroups. A new
/// token's page comes from the ring when it is a new one (the table's entry may not be there yet).
/// Pages given back go behind the ring's last free page, apart from all that are read from it.
template <int kThreads, int kPer>
__global__ __launch_bounds__(kThreads) void PagedPlanKernel(PlanArgs p)
{
    constexpr uint32_t kMost = kThreads * kPer;
    __shared__ uint32_t startOf[kMost + 1];
    __shared__ uint32_t takeOf[kMost + 1];
    __shared__ uint32_t backOf[kMost + 1];
    __shared__ uint64_t waveSum2[kThreads / kWave][2];
    __shared__ uint64_t waveSum1[kThreads / kWave][1];

    const uint32_t pageSize = 1u << p.pageShift;
    const uint32_t capacity = p.tablePages << p.pageShift;  // the host keeps it below 2^31
    uint32_t head = static_cast<uint32_t>(p.pool[0]);
    uint32_t count = static_cast<uint32_t>(p.pool[1]);
    const bool ring = head < p.pages && count <= p.pages;  // negative values are large here
    if (!ring)
    {
        head = 0;
        count = 0;
    }

    uint32_t len[kPer], tgt[kPer], fresh[kPer], need[kPer];
    bool fits[kPer];
    uint64_t one[1] = {0};
#pragma unroll
    for (int e = 0; e < kPer; ++e)
    {
        const uint32_t s = threadIdx.x * kPer + e;
        const int32_t l = s < p.sequences ? p.lengths[s] : -1;
        const int32_t t = s < p.sequences ? p.targets[s] : -1;
        len[e] = static_cast<uint32_t>(l);
        tgt[e] = static_cast<uint32_t>(t);
        fits[e] = l >= 0 && t >= 0 && len[e] <= capacity && tgt[e] <= capacity;
        fresh[e] = fits[e] && t > l ? tgt[e] - len[e] : 0;
        one[0] += fresh[e];
    }
    uint64_t mine = one[0];
    BlockInclusiveSum<kThreads>(one, waveSum1);
    uint64_t before = one[0] - mine;
    mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
    {
        before += fresh[e];
        fits[e] = fits[e] && before <= p.tokens;
        const uint32_t have = (len[e] + pageSize - 1) >> p.pageShift;
        const uint32_t want = (tgt[e] + pageSize - 1) >> p.pageShift;
        need[e] = fits[e] && want > have ? want - have : 0;
        mine += need[e];
    }
    one[0] = mine;
    BlockInclusiveSum<kThreads>(one, waveSum1);
    before = one[0] - mine;
    // New tokens in the low word, pages taken in the high one (both below 2^31), then pages given back.
    uint64_t two[2] = {0, 0};
    bool ok[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
    {
        before += need[e];
        ok[e] = fits[e] && (need[e] == 0 || before <= count);
        const uint32_t have = (len[e] + pageSize - 1) >> p.pageShift;
        const uint32_t want = (tgt[e] + pageSize - 1) >> p.pageShift;
        two[0] += ok[e] ? fresh[e] + (static_cast<uint64_t>(need[e]) << 32) : 0;
        two[1] += ok[e] && have > want ? have - want : 0;
    }
    uint64_t own[2] = {two[0], two[1]};
    BlockInclusiveSum<kThreads>(two, waveSum2);
    uint64_t at = two[0] - own[0];
    uint64_t back = two[1] - own[1];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
    {
        const uint32_t s = threadIdx.x * kPer + e;
        const uint32_t have = (len[e] + pageSize - 1) >> p.pageShift;
        const uint32_t want = (tgt[e] + pageSize - 1) >> p.pageShift;
        startOf[s] = static_cast<uint32_t>(at);
        takeOf[s] = static_cast<uint32_t>(at >> 32);
        backOf[s] = static_cast<uint32_t>(back);
        at += ok[e] ? fresh[e] + (static_cast<uint64_t>(need[e]) << 32) : 0;
        back += ok[e] && have > want ? have - want : 0;
    }
    if (threadIdx.x == kThreads - 1)
    {
        startOf[kMost] = static_cast<uint32_t>(at);
        takeOf[kMost] = static_cast<uint32_t>(at >> 32);
        backOf[kMost] = static_cast<uint32_t>(back);
    }
    __syncthreads();
    const uint32_t fresh0 = startOf[p.sequences];
    const uint32_t taken = takeOf[p.sequences];
    // More pages than the ring has places left were given back twice or never taken: the rest is dropped.
    const uint32_t given = ring ? min(backOf[p.sequences], p.pages - count) : 0;
    auto ringAt = [&](uint32_t i) {
        const uint32_t place = head + i;  // below 2 * pages
        return place < p.pages ? place : place - p.pages;
    };

    const uint32_t first = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t stride = gridDim.x * kThreads;
    if (p.lists != 0)
    {
        for (uint32_t t = first; t < p.tokens; t += stride)
        {
            int32_t sequence = -1;
            int32_t position = -1;
            int32_t slot = -1;
            if (t < fresh0)
            {
                const uint32_t b = OwnerOf(startOf, p.sequences, t);
                const uint32_t held = static_cast<uint32_t>(p.lengths[b]);
                const uint32_t have = (held + pageSize - 1) >> p.pageShift;
                const uint32_t pos = held + t - startOf[b];
                const uint32_t block = pos >> p.pageShift;
                const int32_t page = block < have ? p.tables[static_cast<uint64_t>(b) * p.tablePages + block]
                                                  : p.freePages[ringAt(takeOf[b] + block - have)];
                sequence = static_cast<int32_t>(b);
                position = static_cast<int32_t>(pos);
                if (static_cast<uint32_t>(page) < p.pages)
                {
                    slot = static_cast<int32_t>((static_cast<uint32_t>(page) << p.pageShift) + (pos & (pageSize - 1)));
                }
            }
            p.tokenSequence[t] = sequence;
            p.positions[t] = position;
            p.slots[t] = slot;
        }
        for (uint32_t i = first; i < taken; i += stride)
        {
            const uint32_t b = OwnerOf(takeOf, p.sequences, i);
            const uint32_t have = (static_cast<uint32_t>(p.lengths[b]) + pageSize - 1) >> p.pageShift;
            p.tables[static_cast<uint64_t>(b) * p.tablePages + have + i - takeOf[b]] = p.freePages[ringAt(i)];
        }
        for (uint32_t i = first; i < given; i += stride)
        {
            const uint32_t b = OwnerOf(backOf, p.sequences, i);
            const uint32_t want = (static_cast<uint32_t>(p.targets[b]) + pageSize - 1) >> p.pageShift;
            // count + i < pages, so head + count + i is below 2 * pages too.
            p.freePages[ringAt(count + i)] = p.tables[static_cast<uint64_t>(b) * p.tablePages + want + i - backOf[b]];
        }
        for (uint32_t s = first; s <= p.sequences; s += stride)
        {
            p.starts[s] = static_cast<int32_t>(startOf[s]);
        }
    }
    if (p.state != 0 && blockIdx.x == 0)
    {
        // granted may be lengths and poolOut pool: then this is the only workgroup (or a launch of its
        // own), and all its reads of them are done here.
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; ++e)
        {
            const uint32_t s = threadIdx.x * kPer + e;
            if (s < p.sequences)
            {
                p.granted[s] = static_cast<int32_t>(ok[e] ? tgt[e] : len[e]);
            }
        }
        if (threadIdx.x == 0)
        {
            p.poolOut[0] = ring ? static_cast<int32_t>(ringAt(taken)) : p.pool[0];
            p.poolOut[1] = ring ? static_cast<int32_t>(count - taken + given) : p.pool[1];
        }
    }
}

hipError_t LaunchPlan(hipStream_t s, PlanArgs p, uint32_t blocks)
{
    if (p.sequences <= 256)
    {
        hipLaunchKernelGGL((PagedPlanKernel<256, 1>), dim3(blocks), dim3(256), 0, s, p);
    }
    else if (p.sequences <= kSmallPlan)
    {
        hipLaunchKernelGGL((PagedPlanKernel<256, 4>), dim3(blocks), dim3(256), 0, s, p);
    }
    else
    {
        hipLaunchKernelGGL((PagedPlanKernel<1024, 4>), dim3(blocks), dim3(1024), 0, s, p);
    }
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// Rope and append.

struct AppendArgs
{
    const float* q;
    const float* k;
    const float* v;
    uint64_t qStride, kStride, vStride;
    float* qOut;
    uint16_t* kcache;
    uint16_t* vcache;
    const int32_t* positions;
    const int32_t* slots;
    uint32_t tokens, heads, kvHeads, headDim;
    uint32_t pageShift;
    uint32_t slotCount;
    uint32_t interleaved;
    uint32_t rotary;
    const double* turns;
    float magnitude;
};

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

/// Row r of a token: a head of q, then of k, then of v.
__device__ __forceinline__ const float* AppendSource(const AppendArgs& a, uint64_t token, uint32_t r)
{
    if (r < a.heads)
    {
        return a.q + token * a.qStride + static_cast<uint64_t>(r) * a.headDim;
    }
    r -= a.heads;
    return r < a.kvHeads ? a.k + token * a.kStride + static_cast<uint64_t>(r) * a.headDim
                         : a.v + token * a.vStride + static_cast<uint64_t>(r - a.kvHeads) * a.headDim;
}

__device__ __forceinline__ uint16_t* AppendTarget(const AppendArgs& a, uint32_t slot, uint32_t r)
{
    r -= a.heads;
    uint16_t* cache = r < a.kvHeads ? a.kcache : a.vcache;
    const uint32_t g = r < a.kvHeads ? r : r - a.kvHeads;
    const uint32_t page = slot >> a.pageShift;
    const uint32_t row = slot & ((1u << a.pageShift) - 1);
    return cache + ((((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + row) * a.headDim);
}

typedef _Float16 half4 __attribute__((ext_vector_type(4)));

/// One thread per (token, row, eight values) for rotary dimensions that are multiples of 8: four pairs, or
/// eight values behind the rotated ones, as two loads of 16 bytes and two stores (8 bytes of f16). v's
/// values go the same way without the rotation.
///
/// What bounds it: memory. 8191 tokens of 28 / 4 heads of 128, 64 values rotated: 285 MB in 54 us, 5.3 TB/s,
/// at the rate of a large copy (5.1); in pairs, by the kernel below, 109 us. Several rows a thread, so that
/// an angle serves them all, measured the same there (two, three or four: 53 to 54 us) and slower for few
/// tokens (253: 4.4 us with one, 5.2 with four), non-temporal loads 58 us: q was just written.
template <bool kInterleaved>
__global__ __launch_bounds__(256) void PagedAppendOctets(AppendArgs a)
{
    const uint32_t octets = a.headDim / 8;
    const uint32_t rows = a.heads + 2 * a.kvHeads;
    const uint32_t perToken = rows * octets;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t token = item / perToken;
    if (token >= a.tokens)
    {
        return;
    }
    const uint32_t rest = static_cast<uint32_t>(item - token * perToken);
    const uint32_t r = rest / octets;
    const uint32_t o = rest - r * octets;
    const int32_t position = a.positions[token];
    const int32_t slot = a.slots[token];
    const bool turned = 8 * o < a.rotary;
    // Two quads of values: halves of four pairs, or one behind the other.
    const uint32_t lo = turned && !kInterleaved ? 4 * o : 8 * o;
    const uint32_t hi = turned && !kInterleaved ? 4 * o + a.rotary / 2 : 8 * o + 4;
    const float* from = AppendSource(a, token, r);
    const float4v x0 = *reinterpret_cast<const float4v*>(from + lo);
    const float4v x1 = *reinterpret_cast<const float4v*>(from + hi);
    const bool stored = slot >= 0 && static_cast<uint32_t>(slot) < a.slotCount;
    if (position < 0 || (r >= a.heads && !stored))
    {
        return;
    }
    float4v y0 = x0;
    float4v y1 = x1;
    if (turned && r < a.heads + a.kvHeads)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            float c, s;
            PairAngle(a.turns[4 * o + e], position, a.magnitude, c, s);
            float u, w;
            if (kInterleaved)
            {
                Rotate((e < 2 ? x0 : x1)[e % 2 * 2], (e < 2 ? x0 : x1)[e % 2 * 2 + 1], c, s, u, w);
                (e < 2 ? y0 : y1)[e % 2 * 2] = u;
                (e < 2 ? y0 : y1)[e % 2 * 2 + 1] = w;
            }
            else
            {
                Rotate(x0[e], x1[e], c, s, u, w);
                y0[e] = u;
                y1[e] = w;
            }
        }
    }
    if (r < a.heads)
    {
        float* to = a.qOut + (token * a.heads + r) * a.headDim;
        *reinterpret_cast<float4v*>(to + lo) = y0;
        *reinterpret_cast<float4v*>(to + hi) = y1;
    }
    else
    {
        // The cache's type: half a step of f16, 2^-11 of the value.
        uint16_t* to = AppendTarget(a, static_cast<uint32_t>(slot), r);
        *reinterpret_cast<half4*>(to + lo) = __builtin_convertvector(y0, half4);
        *reinterpret_cast<half4*>(to + hi) = __builtin_convertvector(y1, half4);
    }
}

/// One thread per (token, row, pair of values): any even rotary dimension.
__global__ __launch_bounds__(256) void PagedAppendPairs(AppendArgs a)
{
    const uint32_t pairs = a.headDim / 2;
    const uint32_t rows = a.heads + 2 * a.kvHeads;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t token = item / (static_cast<uint64_t>(pairs) * rows);
    if (token >= a.tokens)
    {
        return;
    }
    const uint32_t rest = static_cast<uint32_t>(item - token * pairs * rows);
    const uint32_t r = rest / pairs;
    const uint32_t j = rest - r * pairs;
    const int32_t position = a.positions[token];
    const int32_t slot = a.slots[token];
    const bool stored = slot >= 0 && static_cast<uint32_t>(slot) < a.slotCount;
    if (position < 0 || (r >= a.heads && !stored))
    {
        return;
    }
    const uint32_t half = a.rotary / 2;
    const bool turned = j < half;
    const uint32_t i0 = turned && a.interleaved == 0 ? j : 2 * j;
    const uint32_t i1 = turned && a.interleaved == 0 ? j + half : 2 * j + 1;
    const float* from = AppendSource(a, token, r);
    float y0 = from[i0];
    float y1 = from[i1];
    if (turned && r < a.heads + a.kvHeads)
    {
        float c, s;
        PairAngle(a.turns[j], position, a.magnitude, c, s);
        Rotate(y0, y1, c, s, y0, y1);
    }
    if (r < a.heads)
    {
        float* to = a.qOut + (token * a.heads + r) * a.headDim;
        to[i0] = y0;
        to[i1] = y1;
    }
    else
    {
        uint16_t* to = AppendTarget(a, static_cast<uint32_t>(slot), r);
        to[i0] = FloatToHalfBits(y0);  // the cache's type: half a step of f16, 2^-11 of the value
        to[i1] = FloatToHalfBits(y1);
    }
}

int Launched(hipError_t status, const char* name)
{
    return status == hipSuccess ? MUYO_OK : HipStatus(status, name);
}
}  // namespace

int CheckPages(const char* name, uint32_t pages, uint32_t pageSize)
{
    if (pageSize < kMinPageSize || pageSize > kMaxPageSize || (pageSize & (pageSize - 1)) != 0)
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: page_size must be a power of two in %u..%u (got %u)", name, kMinPageSize,
                    kMaxPageSize, pageSize);
    }
    if (pages == 0 || static_cast<uint64_t>(pages) * pageSize > 0x7FFFFFFFull)
    {
        return Fail(MUYO_E_RANGE, "%s: needs 1 <= pages and pages * page_size < 2^31 (got %u pages of %u)", name, pages,
                    pageSize);
    }
    return MUYO_OK;
}
}  // namespace muyo

using namespace muyo;

extern "C" int muyo_paged_plan(const int32_t* lengths, const int32_t* targets, uint32_t sequences, int32_t* tables,
                               uint32_t table_pages, int32_t* free_pages, const int32_t* pool, uint32_t pages,
                               uint32_t page_size, uint32_t tokens, int32_t* granted, int32_t* pool_out,
                               int32_t* starts, int32_t* token_sequence, int32_t* positions, int32_t* slots,
                               void* stream)
{
    const char* name = "paged_plan";
    if (lengths == nullptr || targets == nullptr || tables == nullptr || free_pages == nullptr || pool == nullptr ||
        granted == nullptr || pool_out == nullptr || starts == nullptr ||
        (tokens > 0 && (token_sequence == nullptr || positions == nullptr || slots == nullptr)))
    {
        return Fail(MUYO_E_NULL, "%s: every buffer is required (the tokens' lists when tokens > 0)", name);
    }
    const int checked = CheckPages(name, pages, page_size);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    if (sequences == 0 || sequences > kMaxPlanSequences || tokens > kMaxPlanTokens)
    {
        return Fail(MUYO_E_RANGE, "%s: takes 1..%u sequences and at most %u tokens (got %u and %u)", name,
                    kMaxPlanSequences, kMaxPlanTokens, sequences, tokens);
    }
    if (table_pages == 0 || static_cast<uint64_t>(table_pages) * page_size > 0x7FFFFFFFull ||
        static_cast<uint64_t>(table_pages) * sequences > 0x7FFFFFFFull)
    {
        return Fail(MUYO_E_RANGE, "%s: table_pages * page_size and table_pages * sequences must be in 1..2^31 - 1 (got "
                                  "%u pages a row)",
                    name, table_pages);
    }
    const Range ranges[] = {{granted, 4ull * sequences, "granted"},
                            {pool_out, 8, "pool_out"},
                            {tables, 4ull * sequences * table_pages, "tables"},
                            {free_pages, 4ull * pages, "free_pages"},
                            {starts, 4ull * sequences + 4, "starts"},
                            {token_sequence, 4ull * tokens, "token_sequence"},
                            {positions, 4ull * tokens, "positions"},
                            {slots, 4ull * tokens, "slots"},
                            {lengths, 4ull * sequences, "lengths"},
                            {targets, 4ull * sequences, "targets"},
                            {pool, 8, "pool"}};
    constexpr int kOutputs = 8;
    constexpr int kRanges = static_cast<int>(sizeof ranges / sizeof ranges[0]);
    const bool inPlace = granted == lengths || pool_out == pool;
    for (int i = 0; i < kOutputs; ++i)
    {
        for (int j = i + 1; j < kRanges; ++j)
        {
            const bool same = (i == 0 && j == kOutputs && granted == lengths) ||
                              (i == 1 && j == kRanges - 1 && pool_out == pool);
            if (ranges[i].bytes != 0 && ranges[j].bytes != 0 && !same && Overlap(ranges[i], ranges[j]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, ranges[i].name, ranges[j].name);
            }
        }
    }
    PlanArgs p{lengths, targets, sequences, tables, table_pages, free_pages, pool, pages, 0, tokens, granted, pool_out,
               starts, token_sequence, positions, slots, 1, 1};
    while ((1u << p.pageShift) < page_size)
    {
        ++p.pageShift;
    }
    // A thread has one token (of a workgroup of 1024, two): its chain of loads (sequence, length, page) is what
    // takes long. 131104 tokens of 256 sequences take 11.8 us at eight a thread, 7.2 at two, 6.5 at one. A
    // list that one workgroup goes through twice is one launch still.
    const uint32_t threads = sequences <= kSmallPlan ? 256 : 1024;
    const uint32_t blocks =
        tokens <= 2 * threads ? 1 : std::min(1024u, CeilDiv(tokens, threads == 256 ? threads : 2 * threads));
    if (blocks > 1 && inPlace)
    {
        // The state is overwritten only when every workgroup has read it.
        p.state = 0;
        const hipError_t first = LaunchPlan(AsStream(stream), p, blocks);
        if (first != hipSuccess)
        {
            return HipStatus(first, name);
        }
        p.lists = 0;
        p.state = 1;
        return Launched(LaunchPlan(AsStream(stream), p, 1), name);
    }
    return Launched(LaunchPlan(AsStream(stream), p, blocks), name);
}

extern "C" int muyo_rope_frequencies(double base, uint32_t rotary_dim, const MuyoRopeScaling* scaling,
                                     const float* pair_divisors, double* turns, float* magnitude)
{
    const char* name = "rope_frequencies";
    if (turns == nullptr || magnitude == nullptr)
    {
        return Fail(MUYO_E_NULL, "%s: turns and magnitude are required", name);
    }
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || !(base > 1.0) || !std::isfinite(base))
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs an even rotary_dim >= 2 and a finite base above 1", name);
    }
    const uint32_t kind = scaling != nullptr ? scaling->kind : static_cast<uint32_t>(MUYO_ROPE_SCALING_NONE);
    const double factor = kind != MUYO_ROPE_SCALING_NONE ? scaling->factor : 1.0;
    if (kind > MUYO_ROPE_SCALING_WAVELENGTH)
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: unknown scaling kind %u", name, kind);
    }
    if (!(factor > 0.0) || !std::isfinite(factor) || (kind == MUYO_ROPE_SCALING_BASE && rotary_dim == 2))
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a positive factor (and rotary_dim > 2 to stretch the base)", name);
    }
    const double pi2 = 6.283185307179586476925;
    double low = 0.0;
    double high = 0.0;
    float scale = 1.0f;
    if (kind == MUYO_ROPE_SCALING_YARN)
    {
        if (scaling->trainedContext == 0 || !(scaling->low > 0.0f) || !(scaling->high >= scaling->low) ||
            !std::isfinite(scaling->high))
        {
            return Fail(MUYO_E_CONTRACT, "%s: YaRN needs trainedContext and 0 < low <= high", name);
        }
        // The pairs that turn `high` and `low` times in the trained context bound the ramp.
        auto pairOf = [&](double turning) {
            return rotary_dim * std::log(scaling->trainedContext / (turning * pi2)) / (2.0 * std::log(base));
        };
        low = std::max(0.0, std::floor(pairOf(scaling->high)));
        high = std::min(rotary_dim - 1.0, std::ceil(pairOf(scaling->low)));
        scale = static_cast<float>(scaling->attnFactor * (1.0 + 0.1 * std::log(factor)));
        if (!(scale > 0.0f) || !std::isfinite(scale))
        {
            return Fail(MUYO_E_CONTRACT, "%s: YaRN's magnitude attnFactor * (1 + ln(factor) / 10) must be finite and "
                                         "above 0",
                        name);
        }
    }
    if (kind == MUYO_ROPE_SCALING_WAVELENGTH &&
        (scaling->trainedContext == 0 || !(scaling->low > 0.0f) || !(scaling->high > scaling->low) ||
         !std::isfinite(scaling->high)))
    {
        return Fail(MUYO_E_CONTRACT, "%s: scaling by wavelength needs trainedContext and 0 < low < high", name);
    }
    for (uint32_t j = 0; pair_divisors != nullptr && j < rotary_dim / 2; ++j)
    {
        if (!(pair_divisors[j] > 0.0f) || !std::isfinite(pair_divisors[j]))
        {
            return Fail(MUYO_E_CONTRACT, "%s: pair_divisors must be positive and finite", name);
        }
    }
    if (kind == MUYO_ROPE_SCALING_BASE)
    {
        base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
        if (!std::isfinite(base))
        {
            return Fail(MUYO_E_CONTRACT, "%s: the stretched base is not finite", name);
        }
    }
    for (uint32_t j = 0; j < rotary_dim / 2; ++j)
    {
        double radians = std::pow(base, -2.0 * j / rotary_dim);
        if (pair_divisors != nullptr)
        {
            radians /= pair_divisors[j];
        }
        if (kind == MUYO_ROPE_SCALING_LINEAR)
        {
            radians /= factor;
        }
        else if (kind == MUYO_ROPE_SCALING_YARN)
        {
            const double ramp = std::min(1.0, std::max(0.0, (j - low) / std::max(0.001, high - low)));
            radians = radians * (1.0 - ramp) + radians / factor * ramp;
        }
        else if (kind == MUYO_ROPE_SCALING_WAVELENGTH)
        {
            const double turning = scaling->trainedContext * radians / pi2;  // in the trained context
            const double keep = std::min(1.0, std::max(0.0, (turning - scaling->low) / (scaling->high - scaling->low)));
            radians = radians * keep + radians / factor * (1.0 - keep);
        }
        turns[j] = radians / pi2;
    }
    *magnitude = scale;
    return MUYO_OK;
}

extern "C" int muyo_paged_rope_append_f16kv(const float* q, const float* k, const float* v, uint64_t q_stride,
                                            uint64_t k_stride, uint64_t v_stride, float* q_out, void* kcache,
                                            void* vcache, const int32_t* positions, const int32_t* slots,
                                            uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                            uint32_t pages, uint32_t page_size, uint32_t rope_layout,
                                            uint32_t rotary_dim, const double* turns, float magnitude, void* stream)
{
    const char* name = "paged_rope_append_f16kv";
    if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || kcache == nullptr || vcache == nullptr ||
        positions == nullptr || slots == nullptr || turns == nullptr)
    {
        return Fail(MUYO_E_NULL, "%s: every buffer is required", name);
    }
    const int checked = CheckPages(name, pages, page_size);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    if (tokens == 0 || tokens > kMaxPlanTokens || heads == 0 || kv_heads == 0 || heads > 1024 || kv_heads > 1024)
    {
        return Fail(MUYO_E_RANGE, "%s: takes 1..%u tokens, 1..1024 heads and kv_heads (got %u, %u and %u)", name,
                    kMaxPlanTokens, tokens, heads, kv_heads);
    }
    if (head_dim == 0 || head_dim % 8 != 0 || head_dim > 1024 || rotary_dim < 2 || rotary_dim % 2 != 0 ||
        rotary_dim > head_dim || rope_layout > MUYO_ROPE_INTERLEAVED)
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: needs head_dim a multiple of 8 up to 1024, an even rotary_dim of at most "
                                        "that, and a known rope_layout (got %u, %u, %u)",
                    name, head_dim, rotary_dim, rope_layout);
    }
    const uint32_t rows = heads + 2 * kv_heads;
    const bool octets = rotary_dim % 8 == 0;
    const uint64_t items = static_cast<uint64_t>(tokens) * rows * (octets ? head_dim / 8 : head_dim / 2);
    if (items > 1ull << 31)  // a launch has fewer than 2^32 threads
    {
        return Fail(MUYO_E_RANGE, "%s: %u tokens of %u heads of %u values are too many for one call", name, tokens,
                    rows, head_dim);
    }
    const uint64_t qdim = static_cast<uint64_t>(heads) * head_dim;
    const uint64_t kdim = static_cast<uint64_t>(kv_heads) * head_dim;
    if (q_stride < qdim || k_stride < kdim || v_stride < kdim || q_stride % 4 != 0 || k_stride % 4 != 0 ||
        v_stride % 4 != 0 || q_stride > 0xFFFFFFFFull || k_stride > 0xFFFFFFFFull || v_stride > 0xFFFFFFFFull)
    {
        return Fail(MUYO_E_CONTRACT, "%s: token strides must be multiples of 4 that hold a token's heads", name);
    }
    if (!Aligned16(q) || !Aligned16(k) || !Aligned16(v) || !Aligned16(q_out) || !Aligned16(kcache) ||
        !Aligned16(vcache) || (reinterpret_cast<uintptr_t>(turns) & 7u) != 0 || !std::isfinite(magnitude))
    {
        return Fail(MUYO_E_CONTRACT, "%s: q, k, v, q_out and the caches must be 16-byte aligned, turns 8-byte aligned, "
                                     "magnitude finite",
                    name);
    }
    const uint64_t cacheBytes = 2 * kdim * pages * page_size;
    const Range written[] = {{kcache, cacheBytes, "kcache"},
                             {vcache, cacheBytes, "vcache"},
                             {q_out, 4 * qdim * tokens, "q_out"}};
    const Range lists[] = {{positions, 4ull * tokens, "positions"},
                           {slots, 4ull * tokens, "slots"},
                           {turns, 4ull * rotary_dim, "turns"}};
    const Rows sources[] = {{q, 4 * qdim, 4 * q_stride, tokens, "q"},
                            {k, 4 * kdim, 4 * k_stride, tokens, "k"},
                            {v, 4 * kdim, 4 * v_stride, tokens, "v"}};
    for (int i = 0; i < 3; ++i)
    {
        const Range& w = written[i];
        for (int j = i + 1; j < 3; ++j)
        {
            if (Overlap(w, written[j]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w.name, written[j].name);
            }
        }
        for (const Range& r : lists)
        {
            if (Overlap(w, r))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w.name, r.name);
            }
        }
        for (const Rows& r : sources)
        {
            if (i < 2 && Overlap(w, r))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w.name, r.name);
            }
        }
    }
    const Range& out = written[2];
    const Range in[] = {{q, 4 * (q_stride * (tokens - 1) + qdim), "q"},
                        {k, 4 * (k_stride * (tokens - 1) + kdim), "k"},
                        {v, 4 * (v_stride * (tokens - 1) + kdim), "v"}};
    for (const Range& r : in)
    {
        // In place over a dense q each thread writes what it alone has read.
        const bool inPlace = &r == in && q == q_out && q_stride == qdim;
        if (!inPlace && Overlap(out, r))
        {
            return Fail(MUYO_E_CONTRACT, "%s: q_out overlaps %s", name, r.name);
        }
    }
    AppendArgs a{q, k, v, q_stride, k_stride, v_stride, q_out, static_cast<uint16_t*>(kcache),
                 static_cast<uint16_t*>(vcache), positions, slots, tokens, heads, kv_heads, head_dim, 0,
                 pages * page_size, rope_layout, rotary_dim, turns, magnitude};
    while ((1u << a.pageShift) < page_size)
    {
        ++a.pageShift;
    }
    const dim3 grid(static_cast<uint32_t>((items + 255) / 256));
    if (octets && rope_layout == MUYO_ROPE_INTERLEAVED)
    {
        hipLaunchKernelGGL(PagedAppendOctets<true>, grid, dim3(256), 0, AsStream(stream), a);
    }
    else if (octets)
    {
        hipLaunchKernelGGL(PagedAppendOctets<false>, grid, dim3(256), 0, AsStream(stream), a);
    }
    else
    {
        hipLaunchKernelGGL(PagedAppendPairs, grid, dim3(256), 0, AsStream(stream), a);
    }
    return LaunchStatus(name);
}
