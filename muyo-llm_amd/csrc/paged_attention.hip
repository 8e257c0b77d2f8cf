// Attention of single tokens over a paged fp16 cache, many sequences of any lengths in one call.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "paged.hpp"

namespace muyo
{
namespace
{
typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kTile = 32;            // keys of a tile: what a wave takes at a time
constexpr int kHalves = kTile / 16;       // matrix operands of 16 keys
constexpr uint32_t kMaxGroup = 16;        // query heads per kv head: the columns of a matrix operation
constexpr uint32_t kScanQueries = 1024;   // batches up to this many queries: each workgroup makes the sums itself
// Tables or windows of at most this many keys are not split: 16 sequences of 1 to 1000 keys (28 / 4 heads of
// 128) take 13.4 us whole, 9.8 and 3.8 for the join split; one of 1000 8.2, 6.7 and 4.4; 250 of 1 to 1000 at
// 14 / 2 heads of 64 14.7, 17.9 and 4.9.
constexpr uint32_t kWholeKeys = 1024;
constexpr uint32_t kMinShare = kWaves;    // a share is at least a tile a wave
constexpr uint32_t kSetupTiles = 8;       // what a share's change to another (query, kv head) costs, in tiles
constexpr uint32_t kSplitBlocks = 512;    // workgroups of a split launch: two on each of 256 CUs
// Softmax weights are held in two planes of f16, which ends at 2^16: the weight of the maximum is 2^kWeightBias, and
// 2^15 when a later one has run kLag binary orders ahead.
constexpr float kLag = 4.0f;
constexpr float kWeightBias = 15.0f - kLag;
constexpr float kLowScale = 2048.0f;      // of the low plane: what 11 bits of the high one leave, in f16's range again

/// *p for a p that is the same in the whole wave, of memory that nothing writes while the kernel runs: a
/// scalar load. (Through a vector register the wait for it would also be one for every load before it:
/// that took a third longer.)
__device__ __forceinline__ int32_t ScalarLoad(const int32_t* p)
{
    return *(const __attribute__((address_space(4))) int32_t*)reinterpret_cast<uintptr_t>(p);
}

template <bool kOnce>
__device__ __forceinline__ half8 LoadRow(const uint16_t* p)
{
    return kOnce ? __builtin_nontemporal_load(reinterpret_cast<const half8*>(p)) : *reinterpret_cast<const half8*>(p);
}

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
    uint32_t queries, group, kvHeads;
    uint32_t pages, pageShift;
    uint32_t window;
    float scale;
    uint32_t* costSums;  // [queries + 1]: CostOf of one kv head of the queries before
    uint4* cuts;         // what to join: query, kv head, first share, pieces (0: nothing)
    uint32_t cutsByUnit; // cuts has an entry per (query, kv head); else one per share
    float* partials;     // [2 * shares][group][4 + headDim]: base, sum, a score's log2 units, -, weighted values
};

/// The keys begin..end - 1 that a query sees, and the tiles they lie in. A query without any has one
/// tile of which it sees nothing (its output is 0), one without a sequence none.
struct KeyRange
{
    uint32_t begin, end, firstTile, tiles;
    uint32_t row;  // of the tables
};

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
/// shares of short sequences had up to four of them. 28 / 4 heads of 128, with a cost of 0, 4, 8 and 12 tiles:
/// 64 sequences of 1 to 500 keys 27, 15.7, 14.4 and 15.2 us; 250 of 1 to 2000, most short, -, 41, 38 and 43.
__host__ __device__ constexpr uint32_t CostOf(uint32_t tiles) { return tiles != 0 ? tiles + kSetupTiles : 0; }

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
__global__ __launch_bounds__(1024) void PagedCostSumsKernel(PagedAttentionArgs a)
{
    __shared__ uint32_t waveSum[1024 / kWave];
    uint32_t before = 0;
    for (uint32_t first = 0; first < a.queries; first += 1024)
    {
        const uint32_t i = first + threadIdx.x;
        const uint32_t cost = i < a.queries ? CostOf(RangeOf(a, i).tiles) : 0;
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

/// LDS byte of 16-byte chunk `chunk` of V row `row`: chunks are permuted by the row so that the eight
/// rows by two chunks that half a wave's transposing read takes lie in different banks.
template <int kHd>
__device__ __forceinline__ uint32_t ValueAt(uint32_t row, uint32_t chunk)
{
    const uint32_t by = kHd == 128 ? 2 * (row & 7u) : 2 * ((row >> 1) & 3u);
    return row * (2 * kHd) + (chunk ^ by) * 16;
}

/// The cache is read once: all the query heads of a kv head are columns of the same matrix operations
/// (v_mfma_f32_16x16x32_f16: D = A.B with lane l supplying A[l % 16][8 (l / 16) .. +8] and
/// B[8 (l / 16) .. +8][l % 16], receiving D[4 (l / 16) + r][l % 16]). Per tile a wave
///   - takes K rows straight from memory as A operands (of 16 keys each) and forms S^T (keys x heads) =
///     K . q^T, q in registers as two planes of f16 (hi + lo, of q times the power of two that takes the head's
///     largest value to 2^13 .. 2^14: 22 bits down to 2^-16 of that value, and 2^-38 of it below);
///   - passes the V rows through its own part of LDS, to read them back transposed
///     (ds_read_b64_tr_b16: 16 lanes give 4 rows of 16 channels, each gets a channel of 4 rows);
///   - requests the next tile's K and V into the registers that are now free;
///   - makes the softmax weights of the running maximum and from them, in two planes again, the B operand:
///     lane l's weights are keys 4 (l / 16) + r of each 16, and the products sum over keys in any order,
///     so the V^T operand just takes its rows in the same order: O^T (channels x heads) += V^T . P^T.
/// f16 products are exact in f32 and the sums are f32 throughout; the planes keep what one f16 operand
/// would lose (1e-4 of the result).
///
/// Weights are relative to `base`, a raw score that follows the maximum only once that is 2^kLag past it: rescaling
/// the accumulators is rare. They are made of differences of raw scores, in the joins too, so that those of scaled
/// scores of any size are 1 where scores are equal (scaled scores past 2^29 are rounded by more than f16 holds, and
/// weights of them were infinite or 0). Where one key has most of the weight and a small value row, the result is
/// that of the small weights, so these need their bits too: f16 has 11 down to 2^-14, and the low plane, times
/// kLowScale in accumulators of its own, the next 11. A weight keeps 22 bits down to 2^-25 of the largest
/// (17 nats), and 2^-47 of the largest below. (With a key 20 nats above the others and a value row of 0, both planes
/// in the same accumulators lose 3e-4 of the result, and a third of it with weights of at most 1.) The
/// accumulators cost no time for long caches (64 sequences of 1 to 16384 keys 167.5 us, without 167.3) and
/// 0.1 us for short ones.
///
/// Only tiles that reach over an end of the key range, or into a page that is not there, are masked: their scores to
/// -inf, and their V rows to 0, since 0 * NaN would be NaN.
///
/// kSplit: the tiles of all queries and kv heads in a row, each with its setup's cost before it, are dealt
/// out in equal shares, whatever the sequences' lengths. A share may begin and end inside a (query, kv
/// head); those pieces go to `partials` (a share has at most one that does not begin its (query, kv head)
/// and one that does) for PagedAttentionMergeKernel, which finds in `cuts` what to join. Otherwise a
/// workgroup has one (query, kv head). Either way the workgroup's four waves take every fourth tile and join
/// in LDS.
///
/// What bounds it: the cache's arrival. 64 sequences of 1 to 16384 keys (28 / 4 heads of 128, pages of 16,
/// 1.07 GB of K and V): 168 us, 6.4 TB/s, where the best streaming read here has 6.9; 14 / 2 heads of 64,
/// 0.27 GB: 45 us, 6.0 TB/s; one sequence of 32749 keys, 67 MB: 16 us, 4.2 TB/s, of which the way to the
/// first tile and the joins take about five. Past the caches' size, loads without the non-temporal hint took 190 us; a
/// split launch is for long caches, and loads K and V with it. Short ones are a chain of round trips
/// (position, page, rows), 5.2 us: 8 or 16 waves a workgroup, tiles of 64 keys, and two or three tiles in
/// flight at head_dim 64 all measured no better or worse.
template <int kHd, bool kSplit>
__global__ __launch_bounds__(kBlock, kHd == 64 ? (kSplit ? 3 : 4) : 2) void PagedAttentionKernel(PagedAttentionArgs a)
{
    constexpr int kSteps = kHd / 32;               // matrix operations over a head's channels
    constexpr int kChannels = kHd / 16;            // 16-channel blocks of the output
    constexpr uint32_t kChunks = kHd / 8;          // 16-byte chunks of a row
    constexpr uint32_t kRows = kWave / kChunks;    // V rows of one load of the wave
    constexpr int kHalfLoads = 16 / kRows;         // V loads of 16 keys
    constexpr uint32_t kWaveBytes = kTile * 2 * kHd;  // V of a tile; later O^T of 16 heads in f32
    static_assert(kWaveBytes >= kMaxGroup * kHd * 4, "O^T fits where V was");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kWaveBytes];
    __shared__ float waveBase[kWaves][kMaxGroup];
    __shared__ float waveTotal[kWaves][kMaxGroup];
    __shared__ float headScale[kMaxGroup];  // scaleLog2
    __shared__ uint32_t waveSum[kWaves];
    __shared__ KeyRange firstRange;
    __shared__ uint32_t firstAt[2];  // the share's first query, and the costs before it

    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t column = lane % 16;  // the head (of the kv head's group) in operands and results
    const uint32_t quad = lane / 16;
    const uint32_t pageSize = 1u << a.pageShift;

    uint32_t query, g;
    KeyRange range;
    uint32_t at = 0;        // where this share goes on in the row of all costs (the host keeps that below 2^31)
    uint32_t stop = 0;
    uint32_t share = 0;
    uint32_t queryAt = 0;   // where the query begins there, and its kv head
    uint32_t unitAt = 0;
    uint4 cut = make_uint4(0, 0, 0, 0);
    if constexpr (kSplit)
    {
        uint32_t total;
        if (a.queries <= kWave)
        {
            // Every wave makes the sums, a query a lane.
            KeyRange mine = RangeOf(a, min(lane, a.queries - 1));
            mine.tiles = lane < a.queries ? mine.tiles : 0;
            const uint32_t cost = CostOf(mine.tiles);
            const uint32_t sum = WaveSums(cost);
            total = __builtin_amdgcn_readlane(sum, kWave - 1);
            share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
            at = blockIdx.x * share;
            const uint64_t has = __ballot((sum - cost) * a.kvHeads <= at && at < sum * a.kvHeads);
            query = has != 0 ? static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(has)) - 1) : 0;
            queryAt = __builtin_amdgcn_readlane(sum - cost, query) * a.kvHeads;
            range.begin = __builtin_amdgcn_readlane(mine.begin, query);
            range.end = __builtin_amdgcn_readlane(mine.end, query);
            range.firstTile = __builtin_amdgcn_readlane(mine.firstTile, query);
            range.tiles = __builtin_amdgcn_readlane(mine.tiles, query);
            range.row = __builtin_amdgcn_readlane(mine.row, query);
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
                ranges[e] = RangeOf(a, min(i, a.queries - 1));  // no condition: all loads at once
                ranges[e].tiles = i < a.queries ? ranges[e].tiles : 0;
                sum += CostOf(ranges[e].tiles);
            }
            const uint32_t all = sum;
            sum = BlockSums<kBlock>(sum, waveSum, total) - all;
            share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
            at = blockIdx.x * share;
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e)
            {
                const uint32_t i = threadIdx.x * kPer + e;
                if (sum * a.kvHeads <= at && at < (sum + CostOf(ranges[e].tiles)) * a.kvHeads)
                {
                    firstRange = ranges[e];
                    firstAt[0] = i;
                    firstAt[1] = sum;
                }
                sum += CostOf(ranges[e].tiles);
            }
            __syncthreads();
            query = firstAt[0];
            queryAt = firstAt[1] * a.kvHeads;
            range = firstRange;
        }
        else
        {
            total = a.costSums[a.queries];
            share = max((total * a.kvHeads + kSplitBlocks - 1) / kSplitBlocks, kMinShare);
            at = blockIdx.x * share;
            query = OwnerOf(a.costSums, a.queries, min(at / a.kvHeads, total - 1));
            queryAt = a.costSums[query] * a.kvHeads;
            range = RangeOf(a, query);
        }
        total *= a.kvHeads;
        stop = min(at + share, total);
        if (at >= total)
        {
            if (a.cutsByUnit == 0 && threadIdx.x == 0)
            {
                a.cuts[blockIdx.x] = cut;
            }
            return;
        }
        g = 0;
    }
    else
    {
        query = blockIdx.y;
        g = blockIdx.x;
        range = RangeOf(a, query);
    }

    uint8_t* const mine = lds + wave * kWaveBytes;
    const uint32_t readAt = ValueAt<kHd>(4 * quad + column / 4, column % 4 / 2) + column % 2 * 8;
    do
    {
        if constexpr (kSplit)
        {
            // The same for the whole workgroup, but read from LDS or counted up: scalars again.
            query = __builtin_amdgcn_readfirstlane(query);
            range.begin = __builtin_amdgcn_readfirstlane(range.begin);
            range.end = __builtin_amdgcn_readfirstlane(range.end);
            range.firstTile = __builtin_amdgcn_readfirstlane(range.firstTile);
            range.tiles = __builtin_amdgcn_readfirstlane(range.tiles);
            range.row = __builtin_amdgcn_readfirstlane(range.row);
        }
        uint32_t tile0 = 0;
        uint32_t tile1 = range.tiles;
        if constexpr (kSplit)
        {
            if (range.tiles == 0)  // padding
            {
                ++query;
                range = RangeOf(a, query);
                continue;
            }
            const uint32_t cost = CostOf(range.tiles);
            g = __builtin_amdgcn_readfirstlane((at - queryAt) / cost);
            unitAt = __builtin_amdgcn_readfirstlane(queryAt + g * cost);
            const uint32_t from = __builtin_amdgcn_readfirstlane(at - unitAt);
            const uint32_t to = __builtin_amdgcn_readfirstlane(min(cost, from + (stop - at)));
            at = unitAt + to;
            tile0 = from > kSetupTiles ? from - kSetupTiles : 0;
            tile1 = to > kSetupTiles ? to - kSetupTiles : 0;
            if (tile0 >= tile1)  // its setup alone: the tiles are the next share's
            {
                continue;
            }
        }
        else if (range.tiles == 0)
        {
            return;
        }
        const bool whole = tile0 == 0 && tile1 == range.tiles;
        const int32_t* table = a.tables + static_cast<uint64_t>(range.row) * a.tablePages;

        // q is requested before the first tile and made into operands while that arrives.
        float4v qv[kSteps][2];
        {
            const float* from =
                a.q + ((static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + min(column, a.group - 1)) * kHd +
                8 * quad;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                qv[s][0] = *reinterpret_cast<const float4v*>(from + 32 * s);
                qv[s][1] = *reinterpret_cast<const float4v*>(from + 32 * s + 4);
            }
        }
        __builtin_amdgcn_sched_barrier(0);

        struct Pages
        {
            uint32_t of[kHalves];
        };
        // The part of a tile behind the table's end, if any, has the last page's id: its keys are past the
        // range, and so masked.
        auto pagesOf = [&](uint32_t tile) {
            Pages ids;
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
                const uint32_t entry = ((range.firstTile + tile) * kTile + 16 * half) >> a.pageShift;
                ids.of[half] = static_cast<uint32_t>(ScalarLoad(table + min(entry, a.tablePages - 1)));
            }
            return ids;
        };
        struct Tile
        {
            Pages pages;
            half8 k[kHalves][kSteps];
            half8 v[kHalves][kHalfLoads];
        };
        Tile now;
        // A tile's K, then its V: loads complete in order, and the scores wait only for K. Pages outside the
        // cache are read as page 0, whose rows are then masked.
        auto request = [&](uint32_t tile, const Pages& pages) {
            now.pages = pages;
            uint64_t base[kHalves];
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
                const uint32_t page = pages.of[half] < a.pages ? pages.of[half] : 0;
                const uint32_t row = ((range.firstTile + tile) * kTile + 16 * half) & (pageSize - 1);
                base[half] = (((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + row) * kHd;
            }
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                {
                    now.k[half][s] = LoadRow<kSplit>(a.kcache + base[half] + (column * kHd + 8 * quad) + 32 * s);
                }
            }
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
#pragma unroll
                for (int j = 0; j < kHalfLoads; ++j)
                {
                    now.v[half][j] = LoadRow<kSplit>(a.vcache + base[half] + lane * 8 + j * kRows * kHd);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };

        float4v o[kChannels], oLow[kChannels];  // from the weights' planes; oLow times kLowScale
#pragma unroll
        for (int c = 0; c < kChannels; ++c)
        {
            o[c] = float4v{};
            oLow[c] = float4v{};
        }
        float base = -INFINITY;  // the raw score that weights are relative to; -inf: none yet
        float runSum = 0.0f;     // of this lane's keys
        // A wave without a tile requests the last one and leaves it: a request under a condition would make
        // the wait for q one for everything.
        request(min(tile0 + wave, tile1 - 1), pagesOf(min(tile0 + wave, tile1 - 1)));
        Pages next = pagesOf(min(tile0 + wave + kWaves, tile1 - 1));  // of the next tile to request

        // The group's heads as columns; columns past it are 0. Planes of q / 2^e, whose largest value is below 2^14:
        // f16 then holds any q, and its small values with their bits where K makes them count.
        half8 qhi[kSteps], qlo[kSteps];
        float scaleLog2;
        {
            float largest = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                {
                    largest = fmaxf(largest, fabsf(qv[s][c / 4][c % 4]));
                }
            }
            largest = fmaxf(largest, PartnerLane<16>(largest));
            largest = fmaxf(largest, PartnerLane<32>(largest));
            int e = 0;
            if (largest > 0.0f && largest < INFINITY)
            {
                (void)frexpf(largest, &e);
            }
            e -= 14;
            // A negative scale turns q's sign, and 0 clears q, so that scores are scaled by a positive number.
            const float sign = column >= a.group || a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
            // Finite and above 0: no difference of raw scores makes a NaN of it.
            scaleLog2 = a.scale == 0.0f ? 1.0f
                                        : fminf(fmaxf(ldexpf(fabsf(a.scale), e) * kLog2e, 0x1p-126f), 0x1.fffffep127f);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                {
                    const float x = column >= a.group ? 0.0f : ldexpf(qv[s][c / 4][c % 4], -e) * sign;
                    qhi[s][c] = static_cast<_Float16>(x);
                    qlo[s][c] = static_cast<_Float16>(x - static_cast<float>(qhi[s][c]));
                }
            }
        }

        for (uint32_t tile = tile0 + wave; tile < tile1; tile += kWaves)
        {
            const Pages afterNext = pagesOf(min(tile + 2 * kWaves, tile1 - 1));
            float4v score[kHalves];
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
            {
                score[half] = float4v{};
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
                {
                    score[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now.k[half][s], qlo[s], score[half], 0, 0, 0);
                }
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
#pragma unroll
                for (int half = 0; half < kHalves; ++half)
                {
                    score[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now.k[half][s], qhi[s], score[half], 0, 0, 0);
                }
            }
            const uint32_t key0 = (range.firstTile + tile) * kTile;
            bool inside = key0 >= range.begin && key0 + kTile <= range.end;
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
                inside = inside && now.pages.of[half] < a.pages;
            }
            if (!inside)
            {
#pragma unroll
                for (uint32_t half = 0; half < kHalves; ++half)
                {
                    const bool there = now.pages.of[half] < a.pages;
#pragma unroll
                    for (int j = 0; j < kHalfLoads; ++j)
                    {
                        const uint32_t key = key0 + 16 * half + j * kRows + lane / kChunks;
                        if (!there || key < range.begin || key >= range.end)
                        {
                            now.v[half][j] = half8{};
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                    {
                        const uint32_t key = key0 + 16 * half + 4 * quad + r;
                        if (!there || key < range.begin || key >= range.end)
                        {
                            score[half][r] = -INFINITY;
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t half = 0; half < kHalves; ++half)
            {
#pragma unroll
                for (int j = 0; j < kHalfLoads; ++j)
                {
                    const uint32_t row = 16 * half + j * kRows + lane / kChunks;
                    *reinterpret_cast<half8*>(mine + ValueAt<kHd>(row, lane % kChunks)) = now.v[half][j];
                }
            }
            // The wave's LDS operations complete in order; this keeps the compiler's order too.
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (tile + kWaves < tile1)
            {
                request(tile + kWaves, next);
                next = afterNext;
            }

            float tileMax = -INFINITY;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
            {
                tileMax = fmaxf(tileMax, fmaxf(fmaxf(score[half][0], score[half][1]),
                                               fmaxf(score[half][2], score[half][3])));
            }
            tileMax = fmaxf(tileMax, PartnerLane<16>(tileMax));
            tileMax = fmaxf(tileMax, PartnerLane<32>(tileMax));
            const bool rises =
                tileMax != -INFINITY && (base == -INFINITY || (tileMax - base) * scaleLog2 > kLag);
            if (__any(rises))
            {
                const float factor =
                    rises ? (base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((base - tileMax) * scaleLog2)) : 1.0f;
                base = rises ? tileMax : base;
                runSum *= factor;
#pragma unroll
                for (int c = 0; c < kChannels; ++c)
                {
                    o[c] *= factor;
                    oLow[c] *= factor;
                }
            }
            half8 phi[kHalves / 2], plo[kHalves / 2];
            const float from = base == -INFINITY ? 0.0f : base;  // without keys so far every score is -inf
            float sum = 0.0f;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
            {
                float4v p;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    p[r] = __builtin_amdgcn_exp2f(fmaf(score[half][r] - from, scaleLog2, kWeightBias));
                    const _Float16 hi = static_cast<_Float16>(p[r]);
                    phi[half / 2][4 * (half % 2) + r] = hi;
                    plo[half / 2][4 * (half % 2) + r] =
                        static_cast<_Float16>(kLowScale * (p[r] - static_cast<float>(hi)));
                }
                sum += (p[0] + p[1]) + (p[2] + p[3]);
            }
            runSum += sum;
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
            {
#pragma unroll
                for (int pair = 0; pair < kHalves / 2; ++pair)
                {
                    uint8_t* row = mine + ((readAt ^ (32u * c)) + pair * 32 * 2 * kHd);
                    const half4 first = __builtin_bit_cast(
                        half4,
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)row));
                    const half4 second = __builtin_bit_cast(
                        half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                   (__attribute__((address_space(3))) short4v*)(row + 16 * 2 * kHd)));
                    const half8 vt = __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7);
                    oLow[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, plo[pair], oLow[c], 0, 0, 0);
                    o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, phi[pair], o[c], 0, 0, 0);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }

        // The four waves' results meet in LDS.
        runSum += PartnerLane<16>(runSum);
        runSum += PartnerLane<32>(runSum);
        if (quad == 0)
        {
            waveBase[wave][column] = base;
            headScale[column] = scaleLog2;  // the same in every wave
        }
        __syncthreads();
        float top = waveBase[0][column];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
        {
            top = fmaxf(top, waveBase[w][column]);
        }
        // A wave without keys has nothing to add: its weight is 0, not that of -inf - -inf.
        const float factor = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((base - top) * scaleLog2);
        if (quad == 0)
        {
            waveTotal[wave][column] = runSum * factor;
        }
        // [16 heads][kHd], 16-byte chunks permuted by the head: eight heads' writes go to different banks.
        float* const acc = reinterpret_cast<float*>(mine);
        if (column < a.group)
        {
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
            {
                // NaN scores leave the base at -inf and NaN in the sums: they are kept.
                const float4v x = base == -INFINITY && runSum == 0.0f ? float4v{}
                                                                      : (o[c] + oLow[c] * (1.0f / kLowScale)) * factor;
                *reinterpret_cast<float4v*>(acc + column * kHd + 4 * ((4 * c + quad) ^ (column & 7u))) = x;
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.group * kHd / 4; i += kBlock)
        {
            const uint32_t h = i / (kHd / 4);
            float4v num = float4v{};
            float den = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
            {
                num += *reinterpret_cast<const float4v*>(lds + w * kWaveBytes + 16 * (i ^ (h & 7u)));
                den += waveTotal[w][h];
            }
            const uint32_t channel = 4 * (i % (kHd / 4));
            if (!kSplit || whole)
            {
                const float inv = 1.0f / den;
                const float4v x = den == 0.0f ? float4v{} : num * inv;
                *reinterpret_cast<float4v*>(
                    a.out + ((static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + h) * kHd + channel) = x;
            }
            else
            {
                float* slot = a.partials +
                              (static_cast<uint64_t>(2 * blockIdx.x + (tile0 == 0 ? 1 : 0)) * a.group + h) * (kHd + 4);
                *reinterpret_cast<float4v*>(slot + 4 + channel) = num;
                if (channel == 0)
                {
                    float best = waveBase[0][h];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w)
                    {
                        best = fmaxf(best, waveBase[w][h]);
                    }
                    slot[0] = best;
                    slot[1] = den;
                    slot[2] = headScale[h];
                }
            }
        }
        if constexpr (kSplit)
        {
            __syncthreads();  // the next piece overwrites the results
            if (tile0 == 0)
            {
                const uint32_t last = (unitAt + CostOf(range.tiles) - 1) / share;
                const uint32_t pieces = whole ? 0 : last - blockIdx.x + 1;
                const uint4 join = make_uint4(query, g, blockIdx.x, pieces);
                if (a.cutsByUnit == 0)
                {
                    cut = join;  // only the last piece is not whole
                }
                else if (threadIdx.x == 0)
                {
                    a.cuts[query * a.kvHeads + g] = join;
                }
            }
            if (at < stop && g + 1 == a.kvHeads)
            {
                queryAt = at;
                ++query;
                range = RangeOf(a, query);
            }
        }
    } while (kSplit && at < stop);
    if constexpr (kSplit)
    {
        if (a.cutsByUnit == 0 && threadIdx.x == 0)
        {
            a.cuts[blockIdx.x] = cut;
        }
    }
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
template <int kHd, int kThreads>
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
    if ((a.cutsByUnit != 0 && RangeOf(a, blockIdx.x / a.kvHeads).tiles == 0) || pieces == 0)
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
        *reinterpret_cast<float4v*>(
            a.out + ((static_cast<uint64_t>(cut.x) * a.kvHeads + cut.y) * a.group + h) * kHd + 4 * lane) = result;
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

template <int kHd>
hipError_t LaunchPagedAttention(hipStream_t s, PagedAttentionArgs a)
{
    const uint64_t keys = std::min<uint64_t>(static_cast<uint64_t>(a.tablePages) << a.pageShift,
                                             a.window != 0 ? a.window : 0xFFFFFFFFull);
    const uint64_t units = static_cast<uint64_t>(a.queries) * a.kvHeads;
    if (keys <= kWholeKeys || units * (keys / kTile + 2 + kSetupTiles) > 0x7FFFFFFFull)
    {
        hipLaunchKernelGGL((PagedAttentionKernel<kHd, false>), dim3(a.kvHeads, a.queries), dim3(kBlock), 0, s, a);
        return hipGetLastError();
    }
    if (a.queries > kScanQueries)
    {
        hipLaunchKernelGGL(PagedCostSumsKernel, dim3(1), dim3(1024), 0, s, a);
    }
    a.cutsByUnit = units < kSplitBlocks ? 1 : 0;
    const uint32_t joins = a.cutsByUnit != 0 ? static_cast<uint32_t>(units) : kSplitBlocks - 1;
    hipLaunchKernelGGL((PagedAttentionKernel<kHd, true>), dim3(kSplitBlocks), dim3(kBlock), 0, s, a);
    if (joins * a.group <= 256)
    {
        hipLaunchKernelGGL((PagedAttentionMergeKernel<kHd, 512>), dim3(joins, a.group), dim3(512), 0, s, a);
    }
    else
    {
        hipLaunchKernelGGL((PagedAttentionMergeKernel<kHd, 256>), dim3(joins, a.group), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_paged_attention_decode_f16kv_workspace_bytes(uint32_t queries, uint32_t heads,
                                                                    uint32_t kv_heads, uint32_t head_dim)
{
    if (!AttentionShape(queries, heads, kv_heads, head_dim))
    {
        return 0;
    }
    return CostSumBytes(queries) + kCutBytes +
           sizeof(float) * 2 * kSplitBlocks * (heads / kv_heads) * (head_dim + 4);
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
    if (!Aligned16(q) || !Aligned16(kcache) || !Aligned16(vcache) || !Aligned16(out) || !std::isfinite(scale))
    {
        return Fail(MUYO_E_CONTRACT, "%s: q, out and the caches must be 16-byte aligned, and scale finite", name);
    }
    const size_t need = muyo_paged_attention_decode_f16kv_workspace_bytes(queries, heads, kv_heads, head_dim);
    if (workspace == nullptr || !Aligned16(workspace) || workspace_bytes < need)
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a 16-byte aligned workspace of %zu bytes (got %llu)", name, need,
                    static_cast<unsigned long long>(workspace_bytes));
    }
    const uint64_t rowsBytes = 4ull * queries * heads * head_dim;
    const uint64_t cacheBytes = 2ull * pages * page_size * kv_heads * head_dim;
    // The positions, sequences and tables are read again while other workgroups write.
    const Range ranges[] = {{out, rowsBytes, "out"},
                            {workspace, need, "workspace"},
                            {q, rowsBytes, "q"},
                            {kcache, cacheBytes, "kcache"},
                            {vcache, cacheBytes, "vcache"},
                            {tables, 4ull * sequences * table_pages, "tables"},
                            {query_sequence, 4ull * queries, "query_sequence"},
                            {positions, 4ull * queries, "positions"}};
    constexpr int kOutputs = 2;
    constexpr int kRanges = static_cast<int>(sizeof ranges / sizeof ranges[0]);
    for (int i = 0; i < kOutputs; ++i)
    {
        for (int j = i + 1; j < kRanges; ++j)
        {
            // In place a workgroup has read its (query, kv head)'s q when it writes its output there, and one that
            // is cut is written by the join.
            const bool inPlace = i == 0 && j == kOutputs && q == out;
            if (!inPlace && Overlap(ranges[i], ranges[j]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, ranges[i].name, ranges[j].name);
            }
        }
    }
    PagedAttentionArgs a{q,
                         static_cast<const uint16_t*>(kcache),
                         static_cast<const uint16_t*>(vcache),
                         out,
                         tables,
                         sequences,
                         table_pages,
                         query_sequence,
                         positions,
                         queries,
                         heads / kv_heads,
                         kv_heads,
                         pages,
                         0,
                         window,
                         scale,
                         static_cast<uint32_t*>(workspace),
                         reinterpret_cast<uint4*>(static_cast<char*>(workspace) + CostSumBytes(queries)),
                         0,
                         reinterpret_cast<float*>(static_cast<char*>(workspace) + CostSumBytes(queries) + kCutBytes)};
    while ((1u << a.pageShift) < page_size)
    {
        ++a.pageShift;
    }
    const hipError_t launched = head_dim == 64 ? LaunchPagedAttention<64>(AsStream(stream), a)
                                               : LaunchPagedAttention<128>(AsStream(stream), a);
    return launched == hipSuccess ? MUYO_OK : HipStatus(launched, name);
}
