// What the attentions of single tokens over a paged cache share: the keys that a query sees, the equal shares of a
// batch that workgroups take, and the join of what shares cut.
#pragma once

#include <algorithm>

#include "common.hpp"
#include "paged.hpp"

namespace muyo
{
struct PagedAttentionArgs
{
    const float* q;
    float* out;
    const int32_t* tables;
    uint32_t sequences;
    uint32_t tablePages;
    const int32_t* querySequence;
    const int32_t* positions;
    uint32_t queries, group, kvHeads;
    uint32_t pages, pageShift;
    uint32_t window;
    float scale;
    uint32_t* costSums;  // [queries + 1]: CostOf of one kv head of the queries before
    uint4* cuts;         // what to join: query, kv head, first share, pieces (0: nothing)
    uint32_t cutsByUnit; // cuts has an entry per (query, kv head); else one per share
    float* wholes;       // of kPieces: [queries][heads], as partials, of what no share cut
    float* partials;     // [2 * shares][group][4 + headDim]: base, sum, a score's log2 units, -, weighted values
};

/// The arguments that the attentions have in common.
struct AttentionCall
{
    const float* q;
    float* out;
    const int32_t* tables;
    uint32_t sequences, tablePages;
    const int32_t* querySequence;
    const int32_t* positions;
    uint32_t queries, heads, kvHeads, headDim;
    uint32_t pages, pageSize;
    float scale;
    void* workspace;
    uint64_t workspaceBytes;
    uint64_t need;  // of it
};

/// MUYO_OK, or the status of the first part of the contract that the call breaks. `more`: what it reads
/// besides, the first `aligned` of them 16-byte aligned.
int CheckAttention(const char* name, const AttentionCall& call, const Range* more, int moreCount, int aligned);

namespace
{
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kMaxGroup = 16;        // query heads per kv head: the columns of a matrix operation
constexpr uint32_t kScanQueries = 1024;   // batches up to this many queries: each workgroup makes the sums itself
// Tables or windows of at most this many keys are not split: 16 sequences of 1 to 1000 keys (28 / 4 heads of
// 128) take 13.4 us whole, 9.8 and 3.8 for the join split; one of 1000 8.2, 6.7 and 4.4; 250 of 1 to 1000 at
// 14 / 2 heads of 64 14.7, 17.9 and 4.9.
constexpr uint32_t kWholeKeys = 1024;
constexpr uint32_t kMinShare = kWaves;    // a share is at least a tile a wave
constexpr uint32_t kSplitBlocks = 512;    // workgroups of a split launch: two on each of 256 CUs

/// *p for a p that is the same in the whole wave, of memory that nothing writes while the kernel runs: a
/// scalar load. (Through a vector register the wait for it would also be one for every load before it:
/// that took a third longer.)
__device__ __forceinline__ int32_t ScalarLoad(const int32_t* p)
{
    return *(const __attribute__((address_space(4))) int32_t*)reinterpret_cast<uintptr_t>(p);
}

/// The keys begin..end - 1 that a query sees, and the tiles they lie in. A query without any has one
/// tile of which it sees nothing (its output is 0), one without a sequence none.
struct KeyRange
{
    uint32_t begin, end, firstTile, tiles;
    uint32_t row;  // of the tables
};

/// In tiles of kTile keys.
template <uint32_t kTile>
__device__ __forceinline__ KeyRange RangeOf(const PagedAttentionArgs& a, uint32_t query)
{
    const int32_t row = a.querySequence[query];
    const int32_t position = a.positions[query];
    const uint32_t capacity = a.tablePages << a.pageShift;  // the host keeps it below 2^31
    const uint32_t count = position < 0 ? 0 : static_cast<uint32_t>(position) + 1;
    KeyRange r;
    r.end = min(count, capacity);
    r.begin = a.window != 0 && count > a.window ? count - a.window : 0;
    if (r.begin >= r.end)
    {
        r.begin = 0;
        r.end = 0;
    }
    r.firstTile = r.begin / kTile;
    r.row = static_cast<uint32_t>(row);
    r.tiles = r.row < a.sequences ? max((r.end + kTile - 1) / kTile - r.firstTile, 1u) : 0;
    return r;
}

/// What a (query, kv head) of `tiles` tiles counts in the shares. A change to it (its q, its first tile's
/// round trips, joining the waves) takes 3 to 4 us, a tile of each wave about one: dealt out by tiles alone,
/// shares of short sequences had up to four of them. 28 / 4 heads of 128, with a cost of 0, 4, 8 and 12 tiles of
/// 32 keys: 64 sequences of 1 to 500 keys 27, 15.7, 14.4 and 15.2 us; 250 of 1 to 2000, most short, -, 41, 38 and 43.
template <uint32_t kTile>
inline constexpr uint32_t kSetupTiles = 256 / kTile;

template <uint32_t kTile>
__host__ __device__ constexpr uint32_t CostOf(uint32_t tiles)
{
    return tiles != 0 ? tiles + kSetupTiles<kTile> : 0;
}

/// Inclusive sum over the workgroup's threads, in thread order; `total` is the last one's.
template <int kThreads>
__device__ __forceinline__ uint32_t BlockSums(uint32_t v, uint32_t* waveSum, uint32_t& total)
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (uint32_t step = 1; step < kWave; step *= 2)
    {
        const uint32_t other = __shfl_up(v, step);
        v += lane >= step ? other : 0;
    }
    __syncthreads();
    if (lane == kWave - 1)
    {
        waveSum[threadIdx.x / kWave] = v;
    }
    __syncthreads();
    total = 0;
    uint32_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / kWave; ++w)
    {
        before += w < threadIdx.x / kWave ? waveSum[w] : 0;
        total += waveSum[w];
    }
    return v + before;
}

/// v plus that of the lane a DPP control names, in the given rows of 16 lanes; 0 from no lane.
template <int kControl, int kRows>
__device__ __forceinline__ uint32_t PlusLane(uint32_t v)
{
    return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, kRows, 0xF, false));
}

/// Inclusive sum over the wave's lanes: shifts inside rows of 16 lanes, then the last lanes of rows to the
/// rows behind them.
__device__ __forceinline__ uint32_t WaveSums(uint32_t v)
{
    v = PlusLane<0x111, 0xF>(v);  // row_shr:1
    v = PlusLane<0x112, 0xF>(v);
    v = PlusLane<0x114, 0xF>(v);
    v = PlusLane<0x118, 0xF>(v);
    v = PlusLane<0x142, 0xA>(v);     // row_bcast:15
    return PlusLane<0x143, 0xC>(v);  // row_bcast:31
}

/// The i with sums[i] <= at < sums[i + 1] (sums[0] = 0, at < sums[n]).
__device__ __forceinline__ uint32_t OwnerOf(const uint32_t* sums, uint32_t n, uint32_t at)
{
    uint32_t low = 0;
    uint32_t high = n;
    while (high - low > 1)
    {
        const uint32_t mid = (low + high) / 2;
        if (sums[mid] <= at)
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

/// The sums of batches of more than kScanQueries queries, by one workgroup before the others start.
template <uint32_t kTile>
__global__ __launch_bounds__(1024) void PagedCostSumsKernel(PagedAttentionArgs a)
{
    __shared__ uint32_t waveSum[1024 / kWave];
    uint32_t before = 0;
    for (uint32_t first = 0; first < a.queries; first += 1024)
    {
        const uint32_t i = first + threadIdx.x;
        const uint32_t cost = i < a.queries ? CostOf<kTile>(RangeOf<kTile>(a, i).tiles) : 0;
        uint32_t total;
        const uint32_t sum = BlockSums<1024>(cost, waveSum, total);
        if (i < a.queries)
        {
            a.costSums[i] = before + sum - cost;
        }
        before += total;
    }
    if (threadIdx.x == 0)
    {
        a.costSums[a.queries] = before;
    }
}

/// Where a workgroup's share begins and ends in the row of all costs (the host keeps that below 2^31), and the
/// first query that it has a part of.
struct Share
{
    uint32_t share, at, stop;
    uint32_t query, queryAt;  // where the query begins in that row
    KeyRange range;
};

/// What the workgroup's threads tell each other of it, in LDS.
struct ShareSpace
{
    uint32_t waveSum[kWaves];
    KeyRange firstRange;
    uint32_t firstAt[2];  // the share's first query, and the costs before it
};

/// Share `block`; one that is empty has at >= stop.
template <uint32_t kTile>
__device__ __forceinline__ Share FirstShare(const PagedAttentionArgs& a, uint32_t block, uint32_t lane,
                                            ShareSpace& space)
{
    Share first;
    uint32_t total;
    if (a.queries <= kWave)
    {
        // Every wave makes the sums, a query a lane.
        KeyRange mine = RangeOf<kTile>(a, min(lane, a.queries - 1));
        mine.tiles = lane < a.queries ? mine.tiles : 0;
        const uint32_t cost = CostOf<kTile>(mine.tiles);
        const uint32_t sum = WaveSums(cost);
        total = __builtin_amdgcn_readlane(sum, kWave - 1);
        first.share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
        first.at = block * first.share;
        const uint64_t has = __ballot((sum - cost) * a.kvHeads <= first.at && first.at < sum * a.kvHeads);
        first.query = has != 0 ? static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(has)) - 1) : 0;
        first.queryAt = __builtin_amdgcn_readlane(sum - cost, first.query) * a.kvHeads;
        first.range.begin = __builtin_amdgcn_readlane(mine.begin, first.query);
        first.range.end = __builtin_amdgcn_readlane(mine.end, first.query);
        first.range.firstTile = __builtin_amdgcn_readlane(mine.firstTile, first.query);
        first.range.tiles = __builtin_amdgcn_readlane(mine.tiles, first.query);
        first.range.row = __builtin_amdgcn_readlane(mine.row, first.query);
    }
    else if (a.queries <= kScanQueries)
    {
        // Every workgroup makes the sums; the thread that has the share's first query says so.
        constexpr uint32_t kPer = kScanQueries / kBlock;
        KeyRange ranges[kPer];
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t e = 0; e < kPer; ++e)
        {
            const uint32_t i = threadIdx.x * kPer + e;
            ranges[e] = RangeOf<kTile>(a, min(i, a.queries - 1));  // no condition: all loads at once
            ranges[e].tiles = i < a.queries ? ranges[e].tiles : 0;
            sum += CostOf<kTile>(ranges[e].tiles);
        }
        const uint32_t all = sum;
        sum = BlockSums<kBlock>(sum, space.waveSum, total) - all;
        first.share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
        first.at = block * first.share;
#pragma unroll
        for (uint32_t e = 0; e < kPer; ++e)
        {
            const uint32_t i = threadIdx.x * kPer + e;
            if (sum * a.kvHeads <= first.at && first.at < (sum + CostOf<kTile>(ranges[e].tiles)) * a.kvHeads)
            {
                space.firstRange = ranges[e];
                space.firstAt[0] = i;
                space.firstAt[1] = sum;
            }
            sum += CostOf<kTile>(ranges[e].tiles);
        }
        __syncthreads();
        first.query = space.firstAt[0];
        first.queryAt = space.firstAt[1] * a.kvHeads;
        first.range = space.firstRange;
    }
    else
    {
        total = a.costSums[a.queries];
        first.share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
        first.at = block * first.share;
        first.query = OwnerOf(a.costSums, a.queries, min(first.at / a.kvHeads, total - 1));
        first.queryAt = a.costSums[first.query] * a.kvHeads;
        first.range = RangeOf<kTile>(a, first.query);
    }
    total *= a.kvHeads;
    first.stop = min(first.at + first.share, total);
    return first;
}

/// Joins the pieces of a (query, kv head) that shares cut: blockIdx.x goes over those, or over the shares,
/// whichever are fewer (a share's end cuts at most one that begins in it). A workgroup per head,
/// kHd / 4 lanes over the channels of a piece, and kThreads / (kHd / 4) pieces side by side in slices,
/// kDeep of each in flight. A slice's sums are relative to its own running base, so that nothing waits for
/// a first pass over the maxima. The order is fixed.
///
/// 256 threads have 32 pieces of 128 channels in flight, 512 have 128: one sequence of 32749 keys (28 / 4
/// heads, 28 workgroups of 128 pieces) takes 4.9 us with 512 threads and 7.6 with 256; 64 sequences (1792
/// workgroups, most with three pieces) take 8.4 us with 512, whose waves start no faster, and 4.7 with 256.
template <int kHd, uint32_t kTile, int kThreads>
__global__ __launch_bounds__(kThreads) void PagedAttentionMergeKernel(PagedAttentionArgs a)
{
    constexpr uint32_t kLanes = kHd / 4;
    constexpr uint32_t kSlices = kThreads / kLanes;
    constexpr uint32_t kDeep = kThreads / 64;
    __shared__ float4v sliceNum[kSlices][kLanes];
    __shared__ float sliceBase[kSlices];
    __shared__ float sliceDen[kSlices];
    const uint4 cut = a.cuts[blockIdx.x];
    const uint32_t pieces = cut.w;
    // By unit, padding has no entry.
    if ((a.cutsByUnit != 0 && RangeOf<kTile>(a, blockIdx.x / a.kvHeads).tiles == 0) || pieces == 0)
    {
        return;
    }
    const uint32_t h = blockIdx.y;
    const uint32_t lane = threadIdx.x % kLanes;
    const uint32_t slice = threadIdx.x / kLanes;
    float top = -INFINITY;
    float den = 0.0f;
    float scaleLog2 = 1.0f;  // the head's, in every piece
    float4v num = float4v{};
    for (uint32_t p0 = slice; p0 < pieces; p0 += kDeep * kSlices)
    {
        float4v head[kDeep], x[kDeep];
        float best = top;
#pragma unroll
        for (uint32_t i = 0; i < kDeep; ++i)
        {
            // Piece 0 begins the (query, kv head), the others are their shares' first.
            const uint32_t p = min(p0 + i * kSlices, pieces - 1);
            const float* from = a.partials + (static_cast<uint64_t>(2 * (cut.z + p) + (p == 0 ? 1 : 0)) * a.group +
                                              h) * (kHd + 4);
            head[i] = *reinterpret_cast<const float4v*>(from);
            x[i] = *reinterpret_cast<const float4v*>(from + 4 + 4 * lane);
        }
#pragma unroll
        for (uint32_t i = 0; i < kDeep; ++i)
        {
            best = p0 + i * kSlices < pieces ? fmaxf(best, head[i][0]) : best;
        }
        scaleLog2 = head[0][2];
        const float factor = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((top - best) * scaleLog2);
        top = best;
        den *= factor;
        num *= factor;
#pragma unroll
        for (uint32_t i = 0; i < kDeep; ++i)
        {
            if (p0 + i * kSlices < pieces)
            {
                // A piece without keys is all 0; one of NaN scores has this base too, and stays NaN.
                const float w = head[i][0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((head[i][0] - best) * scaleLog2);
                den = fmaf(w, head[i][1], den);
                num += w * x[i];
            }
        }
    }
    sliceNum[slice][lane] = num;
    if (lane == 0)
    {
        sliceBase[slice] = top;
        sliceDen[slice] = den;
    }
    __syncthreads();
    if (slice == 0)
    {
        float best = -INFINITY;
#pragma unroll
        for (uint32_t s = 0; s < kSlices; ++s)
        {
            best = fmaxf(best, sliceBase[s]);
        }
        num = float4v{};
        den = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSlices; ++s)
        {
            const float w = sliceBase[s] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((sliceBase[s] - best) * scaleLog2);
            den = fmaf(w, sliceDen[s], den);
            num += w * sliceNum[s][lane];
        }
        const float4v result = den == 0.0f ? float4v{} : num / den;
        const uint64_t head = (static_cast<uint64_t>(cut.x) * a.kvHeads + cut.y) * a.group + h;
        *reinterpret_cast<float4v*>(a.out + head * kHd + 4 * lane) = result;
    }
}

bool AttentionShape(uint32_t queries, uint32_t heads, uint32_t kvHeads, uint32_t headDim)
{
    return queries >= 1 && queries <= 65535 && kvHeads >= 1 && heads >= 1 && heads % kvHeads == 0 &&
           heads / kvHeads <= kMaxGroup && heads <= 1024 && (headDim == 64 || headDim == 128);
}

/// The workspace's parts: the sums of batches that the workgroups do not sum themselves, the cuts, the
/// partials.
size_t CostSumBytes(uint32_t queries)
{
    return queries <= kScanQueries ? 0 : (4 * (static_cast<size_t>(queries) + 1) + 15) & ~static_cast<size_t>(15);
}

constexpr size_t kCutBytes = kSplitBlocks * sizeof(uint4);

/// The common fields of `a`, of a call that CheckAttention has passed.
inline void FillAttentionArgs(PagedAttentionArgs& a, const AttentionCall& c, uint32_t window)
{
    a.q = c.q;
    a.out = c.out;
    a.tables = c.tables;
    a.sequences = c.sequences;
    a.tablePages = c.tablePages;
    a.querySequence = c.querySequence;
    a.positions = c.positions;
    a.queries = c.queries;
    a.group = c.heads / c.kvHeads;
    a.kvHeads = c.kvHeads;
    a.pages = c.pages;
    a.pageShift = 0;
    while ((1u << a.pageShift) < c.pageSize)
    {
        ++a.pageShift;
    }
    a.window = window;
    a.scale = c.scale;
    char* const space = static_cast<char*>(c.workspace);
    a.costSums = reinterpret_cast<uint32_t*>(space);
    a.cuts = reinterpret_cast<uint4*>(space + CostSumBytes(c.queries));
    a.cutsByUnit = 0;
    a.wholes = nullptr;
    a.partials = reinterpret_cast<float*>(space + CostSumBytes(c.queries) + kCutBytes);
}

/// Bytes of the workspace of a decode attention.
inline size_t DecodeWorkspaceBytes(uint32_t queries, uint32_t heads, uint32_t kvHeads, uint32_t headDim)
{
    return CostSumBytes(queries) + kCutBytes + sizeof(float) * 2 * kSplitBlocks * (heads / kvHeads) * (headDim + 4);
}

/// Whether a call's keys are dealt out in shares: not those of tables or windows of at most kWholeKeys keys.
template <uint32_t kTile>
bool SplitKeys(const PagedAttentionArgs& a)
{
    const uint64_t keys = std::min<uint64_t>(static_cast<uint64_t>(a.tablePages) << a.pageShift,
                                             a.window != 0 ? a.window : 0xFFFFFFFFull);
    const uint64_t units = static_cast<uint64_t>(a.queries) * a.kvHeads;
    return keys > kWholeKeys && units * (keys / kTile + 2 + kSetupTiles<kTile>) <= 0x7FFFFFFFull;
}

/// Split launches take `split` and the join, others `whole`.
template <int kHd, uint32_t kTile, typename Args>
hipError_t LaunchPagedAttention(hipStream_t s, Args a, void (*whole)(Args), void (*split)(Args))
{
    const uint64_t units = static_cast<uint64_t>(a.queries) * a.kvHeads;
    if (!SplitKeys<kTile>(a))
    {
        hipLaunchKernelGGL(whole, dim3(a.kvHeads, a.queries), dim3(kBlock), 0, s, a);
        return hipGetLastError();
    }
    if (a.queries > kScanQueries)
    {
        hipLaunchKernelGGL(PagedCostSumsKernel<kTile>, dim3(1), dim3(1024), 0, s, a);
    }
    a.cutsByUnit = units < kSplitBlocks ? 1 : 0;
    const uint32_t joins = a.cutsByUnit != 0 ? static_cast<uint32_t>(units) : kSplitBlocks - 1;
    hipLaunchKernelGGL(split, dim3(kSplitBlocks), dim3(kBlock), 0, s, a);
    if (joins * a.group <= 256)
    {
        hipLaunchKernelGGL((PagedAttentionMergeKernel<kHd, kTile, 512>), dim3(joins, a.group), dim3(512), 0, s, a);
    }
    else
    {
        hipLaunchKernelGGL((PagedAttentionMergeKernel<kHd, kTile, 256>), dim3(joins, a.group), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}
}  // namespace
}  // namespace muyo
