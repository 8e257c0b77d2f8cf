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
constexpr uint32_t kMaxGroup = 16;        // query heads per kv head: the columns of a matrix operation
constexpr uint32_t kScanQueries = 1024;   // batches up to this many queries: each workgroup makes the sums itself
constexpr uint32_t kWholeTiles = 32;      // caches of at most this many tiles are not split
constexpr uint32_t kMinTiles = 16;        // a workgroup's share of the tiles is at least this long

/// Workgroups of a split launch: as many as run at once on 256 CUs.
constexpr uint32_t SplitBlocks(uint32_t headDim) { return headDim == 64 ? 1024 : 512; }

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
    uint64_t* tileSums;  // [queries + 1]: tiles of one kv head of the queries before
    float* partials;     // [2 * blocks][group][2 + headDim]: max (log2 units), sum, weighted values
};

/// The keys begin..end - 1 that a query sees, and the tiles they lie in. A query without any has one
/// tile of which it sees nothing (its output is 0), one without a sequence none.
struct KeyRange
{
    uint32_t begin, end, firstTile, tiles;
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
    r.tiles = max((r.end + kTile - 1) / kTile - r.firstTile, 1u);
    if (row < 0 || static_cast<uint32_t>(row) >= a.sequences)
    {
        r.tiles = 0;
    }
    return r;
}

/// Inclusive sum over the workgroup's threads, in thread order; `total` is the last one's.
template <int kThreads>
__device__ __forceinline__ uint64_t BlockSums(uint64_t v, uint64_t* waveSum, uint64_t& total)
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (uint32_t step = 1; step < kWave; step *= 2)
    {
        const uint64_t other = __shfl_up(static_cast<unsigned long long>(v), step);
        v += lane >= step ? other : 0;
    }
    __syncthreads();
    if (lane == kWave - 1)
    {
        waveSum[threadIdx.x / kWave] = v;
    }
    __syncthreads();
    total = 0;
    uint64_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / kWave; ++w)
    {
        before += w < threadIdx.x / kWave ? waveSum[w] : 0;
        total += waveSum[w];
    }
    return v + before;
}

/// The i with sums[i] <= at < sums[i + 1] (sums[0] = 0, at < sums[n]).
__device__ __forceinline__ uint32_t OwnerOf(const uint64_t* sums, uint32_t n, uint64_t at)
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

/// A workgroup's share of `total` tiles: the same for all but the last.
__device__ __forceinline__ uint64_t ShareOf(uint64_t total, uint32_t blocks)
{
    return max((total + blocks - 1) / blocks, static_cast<uint64_t>(kMinTiles));
}

/// The sums of batches of more than kScanQueries queries, by one workgroup before the others start.
__global__ __launch_bounds__(1024) void PagedTileSumsKernel(PagedAttentionArgs a)
{
    __shared__ uint64_t waveSum[1024 / kWave];
    uint64_t before = 0;
    for (uint32_t first = 0; first < a.queries; first += 1024)
    {
        const uint32_t i = first + threadIdx.x;
        const uint32_t tiles = i < a.queries ? RangeOf(a, i).tiles : 0;
        uint64_t total;
        const uint64_t sum = BlockSums<1024>(tiles, waveSum, total);
        if (i < a.queries)
        {
            a.tileSums[i] = before + sum - tiles;
        }
        before += total;
    }
    if (threadIdx.x == 0)
    {
        a.tileSums[a.queries] = before;
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
/// B[8 (l / 16) .. +8][l % 16], receiving D[4 (l / 16) + r][l % 16]). Per tile of 32 keys a wave
///   - takes K rows straight from memory as A operands (two of 16 keys) and forms S^T (keys x heads) =
///     K . q^T, q in registers as two planes of f16 (hi + lo: 22 bits, of q over its largest value's
///     power of two);
///   - passes the V rows through its own part of LDS, to read them back transposed
///     (ds_read_b64_tr_b16: 16 lanes give 4 rows of 16 channels, each gets a channel of 4 rows);
///   - requests the next tile's K and V into the registers that are now free;
///   - makes the softmax weights of the running maximum and from them, in two planes again, the B operand:
///     lane l's weights are keys 4 (l / 16) + r and 16 more, and the products sum over keys in any order,
///     so the V^T operand just takes its rows in the same order: O^T (channels x heads) += V^T . P^T.
/// f16 products are exact in f32 and the sums are f32 throughout; the planes keep what one f16 operand
/// would lose (1e-4 of the result).
///
/// Weights are relative to `shift`, which follows the maximum only once that is 2^8 past it: rescaling
/// the accumulators is rare. Only tiles that reach over an end of the key range, or into a page that is
/// not there, are masked: their scores to -inf, and their V rows to 0, since 0 * NaN would be NaN.
///
/// kSplit: the tiles of all queries and kv heads in a row are dealt out in equal shares, whatever the
/// sequences' lengths. A share may begin and end inside a (query, kv head); those pieces go to
/// `partials` (a share has at most one that does not begin its (query, kv head) and one that does) for
/// PagedAttentionMergeKernel. Otherwise a workgroup has one (query, kv head). Either way the
/// workgroup's four waves take every fourth tile and join in LDS.
template <int kHd, bool kSplit>
__global__ __launch_bounds__(kBlock, kHd == 64 ? 4 : 2) void PagedAttentionKernel(PagedAttentionArgs a)
{
    constexpr int kSteps = kHd / 32;               // matrix operations over a head's channels
    constexpr int kChannels = kHd / 16;            // 16-channel blocks of the output
    constexpr uint32_t kChunks = kHd / 8;          // 16-byte chunks of a row
    constexpr uint32_t kRows = kWave / kChunks;    // V rows of one load of the wave
    constexpr int kHalfLoads = 16 / kRows;         // V loads of 16 keys
    constexpr uint32_t kWaveBytes = kTile * 2 * kHd;  // V of a tile; later O^T of 16 heads in f32
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kWaveBytes];
    __shared__ float waveMax[kWaves][kMaxGroup];
    __shared__ float waveTotal[kWaves][kMaxGroup];
    __shared__ uint64_t tileSums[kSplit ? kScanQueries + 1 : 1];
    __shared__ uint64_t waveSum[kWaves];

    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t column = lane % 16;  // the head (of the kv head's group) in operands and results
    const uint32_t quad = lane / 16;
    const uint32_t pageSize = 1u << a.pageShift;

    uint32_t query, g;
    uint64_t at = 0;   // this share's tiles, in the row of all
    uint64_t stop = 0;
    const uint64_t* sums = tileSums;
    if constexpr (kSplit)
    {
        if (a.queries <= kScanQueries)
        {
            constexpr uint32_t kPer = kScanQueries / kBlock;
            uint32_t tiles[kPer];
            uint64_t mine = 0;
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e)
            {
                const uint32_t i = threadIdx.x * kPer + e;
                tiles[e] = i < a.queries ? RangeOf(a, i).tiles : 0;
                mine += tiles[e];
            }
            uint64_t total;
            uint64_t sum = BlockSums<kBlock>(mine, waveSum, total) - mine;
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e)
            {
                const uint32_t i = threadIdx.x * kPer + e;
                tileSums[i] = sum;
                if (blockIdx.x == 0 && i < a.queries)
                {
                    a.tileSums[i] = sum;  // for the merge
                }
                sum += tiles[e];
            }
            if (threadIdx.x == 0)
            {
                tileSums[kScanQueries] = total;
                if (blockIdx.x == 0)
                {
                    a.tileSums[a.queries] = total;
                }
            }
            __syncthreads();
        }
        else
        {
            sums = a.tileSums;
        }
        const uint64_t total = sums[a.queries] * a.kvHeads;
        const uint64_t share = ShareOf(total, gridDim.x);
        at = blockIdx.x * share;
        stop = min(at + share, total);
        if (at >= stop)
        {
            return;
        }
        query = OwnerOf(sums, a.queries, at / a.kvHeads);
        g = 0;
    }
    else
    {
        query = blockIdx.x / a.kvHeads;
        g = blockIdx.x % a.kvHeads;
    }

    uint8_t* const mine = lds + wave * kWaveBytes;
    const uint32_t readAt = ValueAt<kHd>(4 * quad + column / 4, column % 4 / 2) + column % 2 * 8;
    do
    {
        query = __builtin_amdgcn_readfirstlane(query);
        const KeyRange range = RangeOf(a, query);
        if (range.tiles == 0)
        {
            if constexpr (kSplit)
            {
                ++query;  // padding has no tiles
                continue;
            }
            else
            {
                return;
            }
        }
        uint32_t tile0 = 0;
        uint32_t tile1 = range.tiles;
        if constexpr (kSplit)
        {
            const uint64_t inQuery = at - sums[query] * a.kvHeads;
            g = static_cast<uint32_t>(inQuery / range.tiles);
            tile0 = static_cast<uint32_t>(inQuery - static_cast<uint64_t>(g) * range.tiles);
            tile1 = static_cast<uint32_t>(min(static_cast<uint64_t>(range.tiles), tile0 + (stop - at)));
        }
        const bool whole = tile0 == 0 && tile1 == range.tiles;
        const int32_t* table = a.tables + static_cast<uint64_t>(a.querySequence[query]) * a.tablePages;

        // The group's heads as columns; columns past it are 0. Planes of q / 2^e with 2^e above the head's
        // largest value: f16 then holds any q.
        half8 qhi[kSteps], qlo[kSteps];
        float scaleLog2;
        {
            float v[kSteps][8];
            float largest = 0.0f;
            const float* from =
                a.q + ((static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + min(column, a.group - 1)) * kHd +
                8 * quad;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                *reinterpret_cast<float4*>(v[s]) = *reinterpret_cast<const float4*>(from + 32 * s);
                *reinterpret_cast<float4*>(v[s] + 4) = *reinterpret_cast<const float4*>(from + 32 * s + 4);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                {
                    largest = fmaxf(largest, fabsf(v[s][c]));
                }
            }
            largest = fmaxf(largest, PartnerLane<16>(largest));
            largest = fmaxf(largest, PartnerLane<32>(largest));
            int e = 0;
            if (largest > 0.0f && largest < INFINITY)
            {
                (void)frexpf(largest, &e);
            }
            // A negative scale turns q's sign, and 0 clears q, so that scores are scaled by a positive number.
            const float sign = column >= a.group || a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
            scaleLog2 = a.scale == 0.0f ? 1.0f : fmaxf(ldexpf(fabsf(a.scale) * kLog2e, e), 0x1p-126f);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                {
                    const float x = column >= a.group ? 0.0f : ldexpf(v[s][c], -e) * sign;
                    const float hi = __uint_as_float(__float_as_uint(x) & 0xFFFFE000u);  // 11 bits: exact in f16
                    qhi[s][c] = static_cast<_Float16>(hi);
                    qlo[s][c] = static_cast<_Float16>(x - hi);
                }
            }
        }

        auto pageOf = [&](uint32_t tile, uint32_t half) {
            const uint32_t column = ((range.firstTile + tile) * kTile + 16 * half) >> a.pageShift;
            return column < a.tablePages ? static_cast<uint32_t>(table[column]) : 0xFFFFFFFFu;
        };
        half8 k[2][kSteps], v[2][kHalfLoads];
        // A tile's K and V. Pages outside the cache are read as page 0, whose rows are then masked.
        auto request = [&](uint32_t tile, uint32_t page0, uint32_t page1) {
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half)
            {
                const uint32_t page = half == 0 ? page0 : page1;
                const uint32_t row = ((range.firstTile + tile) * kTile + 16 * half) & (pageSize - 1);
                const uint64_t base =
                    (((static_cast<uint64_t>(page < a.pages ? page : 0) * a.kvHeads + g) << a.pageShift) + row) * kHd;
                const uint16_t* kFrom = a.kcache + base + (column * kHd + 8 * quad);
                const uint16_t* vFrom = a.vcache + base + lane * 8;
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                {
                    k[half][s] = *reinterpret_cast<const half8*>(kFrom + 32 * s);
                }
#pragma unroll
                for (int j = 0; j < kHalfLoads; ++j)
                {
                    v[half][j] = *reinterpret_cast<const half8*>(vFrom + j * kRows * kHd);
                }
            }
        };

        float4v o[kChannels];
#pragma unroll
        for (int c = 0; c < kChannels; ++c)
        {
            o[c] = float4v{};
        }
        float runMax = -INFINITY;  // of the raw scores
        float shift = 0.0f;        // in log2 units
        float runSum = 0.0f;       // of this lane's keys
        uint32_t page0 = 0, page1 = 0;  // of the tile in registers
        uint32_t next0 = 0, next1 = 0;  // of the one to request
        if (tile0 + wave < tile1)
        {
            page0 = pageOf(tile0 + wave, 0);
            page1 = pageOf(tile0 + wave, 1);
            request(tile0 + wave, page0, page1);
            const uint32_t later = min(tile0 + wave + kWaves, tile1 - 1);
            next0 = pageOf(later, 0);
            next1 = pageOf(later, 1);
        }
        for (uint32_t tile = tile0 + wave; tile < tile1; tile += kWaves)
        {
            float4v score[2] = {float4v{}, float4v{}};
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                score[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0][s], qlo[s], score[0], 0, 0, 0);
                score[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[1][s], qlo[s], score[1], 0, 0, 0);
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                score[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0][s], qhi[s], score[0], 0, 0, 0);
                score[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[1][s], qhi[s], score[1], 0, 0, 0);
            }
            const uint32_t key0 = (range.firstTile + tile) * kTile;
            const bool inside =
                key0 >= range.begin && key0 + kTile <= range.end && page0 < a.pages && page1 < a.pages;
            if (!inside)
            {
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                {
                    const bool there = (half == 0 ? page0 : page1) < a.pages;
#pragma unroll
                    for (int j = 0; j < kHalfLoads; ++j)
                    {
                        const uint32_t key = key0 + 16 * half + j * kRows + lane / kChunks;
                        if (!there || key < range.begin || key >= range.end)
                        {
                            v[half][j] = half8{};
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
            for (uint32_t half = 0; half < 2; ++half)
            {
#pragma unroll
                for (int j = 0; j < kHalfLoads; ++j)
                {
                    const uint32_t row = 16 * half + j * kRows + lane / kChunks;
                    *reinterpret_cast<half8*>(mine + ValueAt<kHd>(row, lane % kChunks)) = v[half][j];
                }
            }
            // The wave's LDS operations complete in order; this keeps the compiler's order too.
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (tile + kWaves < tile1)
            {
                page0 = next0;
                page1 = next1;
                request(tile + kWaves, page0, page1);
                const uint32_t later = min(tile + 2 * kWaves, tile1 - 1);
                next0 = pageOf(later, 0);
                next1 = pageOf(later, 1);
            }

            float tileMax = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                tileMax = fmaxf(tileMax, fmaxf(score[0][r], score[1][r]));
            }
            tileMax = fmaxf(tileMax, PartnerLane<16>(tileMax));
            tileMax = fmaxf(tileMax, PartnerLane<32>(tileMax));
            const float top = tileMax * scaleLog2;
            const bool rises = tileMax != -INFINITY && (runMax == -INFINITY || top > shift + 8.0f);
            if (__any(rises))
            {
                const float newShift = rises ? top : shift;
                const float factor =
                    rises ? (runMax == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(shift - newShift)) : 1.0f;
                runMax = rises ? tileMax : runMax;
                shift = newShift;
                runSum *= factor;
#pragma unroll
                for (int c = 0; c < kChannels; ++c)
                {
                    o[c] *= factor;
                }
            }
            half8 phi, plo;
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    const float p = __builtin_amdgcn_exp2f(fmaf(score[half][r], scaleLog2, -shift));
                    sum[half] += p;
                    const _Float16 hi = static_cast<_Float16>(p);
                    phi[4 * half + r] = hi;
                    plo[4 * half + r] = static_cast<_Float16>(p - static_cast<float>(hi));
                }
            }
            runSum += sum[0] + sum[1];
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
            {
                uint8_t* from = mine + (readAt ^ (32u * c));
                const half4 first = __builtin_bit_cast(
                    half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)from));
                const half4 second = __builtin_bit_cast(
                    half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (__attribute__((address_space(3))) short4v*)(from + 16 * 2 * kHd)));
                const half8 vt = __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7);
                o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, plo, o[c], 0, 0, 0);
                o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, phi, o[c], 0, 0, 0);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }

        // The four waves' results meet in LDS.
        runSum += PartnerLane<16>(runSum);
        runSum += PartnerLane<32>(runSum);
        if (quad == 0)
        {
            waveMax[wave][column] = runMax == -INFINITY ? -INFINITY : shift;
            waveTotal[wave][column] = runSum;
        }
        __syncthreads();
        float top = waveMax[0][column];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
        {
            top = fmaxf(top, waveMax[w][column]);
        }
        // A wave without keys has nothing to add: its weight is 0, not that of -inf - -inf.
        const float factor = runMax == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(shift - top);
        float* const acc = reinterpret_cast<float*>(mine);  // [16 heads][kHd]
        if (column < a.group)
        {
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
            {
                // NaN scores leave the maximum at -inf and NaN in the sums: they are kept.
                const float4v x = runMax == -INFINITY && runSum == 0.0f ? float4v{} : o[c] * factor;
                *reinterpret_cast<float4v*>(acc + column * kHd + 16 * c + 4 * quad) = x;
            }
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.group * kHd / 4; i += kBlock)
        {
            const uint32_t h = i / (kHd / 4);
            float best = waveMax[0][h];
#pragma unroll
            for (int w = 1; w < kWaves; ++w)
            {
                best = fmaxf(best, waveMax[w][h]);
            }
            float4v num = float4v{};
            float den = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
            {
                num += *reinterpret_cast<const float4v*>(lds + w * kWaveBytes + 16 * i);
                const float share = waveTotal[w][h];
                den += waveMax[w][h] == -INFINITY ? share * 0.0f
                                                  : share * __builtin_amdgcn_exp2f(waveMax[w][h] - best);
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
                    slot[0] = best;
                    slot[1] = den;
                }
            }
        }
        if constexpr (kSplit)
        {
            __syncthreads();  // the next piece overwrites the results
            at += tile1 - tile0;
            if (tile1 == range.tiles && g + 1 == a.kvHeads)
            {
                ++query;
            }
        }
    } while (kSplit && at < stop);
}

/// Joins the pieces of the (query, kv head) that the end of share blockIdx.x cuts, if no earlier share's
/// end does: a workgroup per head, threads side by side over the channels and over every
/// (256 / kHd)th piece. The pieces are added in their order.
template <int kHd>
__global__ __launch_bounds__(kBlock) void PagedAttentionMergeKernel(PagedAttentionArgs a, uint32_t blocks)
{
    constexpr uint32_t kSlices = kBlock / kHd;
    __shared__ float sliceNum[kSlices][kHd];
    __shared__ float sliceDen[kSlices];
    const uint64_t total = a.tileSums[a.queries] * a.kvHeads;
    const uint64_t share = ShareOf(total, blocks);
    const uint64_t cut = (blockIdx.x + 1) * share;  // the end of share blockIdx.x
    if (cut >= total)
    {
        return;
    }
    const uint32_t query = OwnerOf(a.tileSums, a.queries, cut / a.kvHeads);
    const uint64_t tiles = a.tileSums[query + 1] - a.tileSums[query];
    const uint64_t g = (cut - a.tileSums[query] * a.kvHeads) / tiles;
    const uint64_t first = a.tileSums[query] * a.kvHeads + g * tiles;
    if (cut == first || blockIdx.x * share > first)
    {
        return;
    }
    const uint32_t pieces = static_cast<uint32_t>((first + tiles - 1) / share) - blockIdx.x + 1;
    const uint32_t h = blockIdx.y;
    // Piece 0 begins the (query, kv head), the others are their shares' first.
    auto piece = [&](uint32_t p) {
        return a.partials + (static_cast<uint64_t>(2 * (blockIdx.x + p) + (p == 0 ? 1 : 0)) * a.group + h) * (kHd + 4);
    };
    const uint32_t channel = threadIdx.x % kHd;
    const uint32_t slice = threadIdx.x / kHd;
    float top = -INFINITY;
    for (uint32_t p = 0; p < pieces; ++p)
    {
        top = fmaxf(top, piece(p)[0]);
    }
    float num = 0.0f;
    float den = 0.0f;
    for (uint32_t p = slice; p < pieces; p += kSlices)
    {
        const float* from = piece(p);
        const float w = from[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(from[0] - top);
        num = fmaf(w, from[4 + channel], num);
        den = fmaf(w, from[1], den);
    }
    sliceNum[slice][channel] = num;
    if (channel == 0)
    {
        sliceDen[slice] = den;
    }
    __syncthreads();
    if (slice == 0)
    {
#pragma unroll
        for (uint32_t s = 1; s < kSlices; ++s)
        {
            num += sliceNum[s][channel];
            den += sliceDen[s];
        }
        a.out[((static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + h) * kHd + channel] =
            den == 0.0f ? 0.0f : num / den;
    }
}

bool AttentionShape(uint32_t queries, uint32_t heads, uint32_t kvHeads, uint32_t headDim)
{
    return queries >= 1 && queries <= 65535 && kvHeads >= 1 && heads >= 1 && heads % kvHeads == 0 &&
           heads / kvHeads <= kMaxGroup && heads <= 1024 && (headDim == 64 || headDim == 128);
}

size_t TileSumBytes(uint32_t queries) { return (8 * (static_cast<size_t>(queries) + 1) + 15) & ~static_cast<size_t>(15); }

template <int kHd>
hipError_t LaunchPagedAttention(hipStream_t s, const PagedAttentionArgs& a)
{
    const uint64_t keys = std::min<uint64_t>(static_cast<uint64_t>(a.tablePages) << a.pageShift,
                                             a.window != 0 ? a.window : 0xFFFFFFFFull);
    if (keys <= kWholeTiles * kTile)
    {
        hipLaunchKernelGGL((PagedAttentionKernel<kHd, false>), dim3(a.queries * a.kvHeads), dim3(kBlock), 0, s, a);
        return hipGetLastError();
    }
    if (a.queries > kScanQueries)
    {
        hipLaunchKernelGGL(PagedTileSumsKernel, dim3(1), dim3(1024), 0, s, a);
    }
    const uint32_t blocks = SplitBlocks(kHd);
    hipLaunchKernelGGL((PagedAttentionKernel<kHd, true>), dim3(blocks), dim3(kBlock), 0, s, a);
    hipLaunchKernelGGL(PagedAttentionMergeKernel<kHd>, dim3(blocks - 1, a.group), dim3(kBlock), 0, s, a, blocks);
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
    return TileSumBytes(queries) + sizeof(float) * 2 * SplitBlocks(head_dim) * (heads / kv_heads) * (head_dim + 4);
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
                         static_cast<uint64_t*>(workspace),
                         reinterpret_cast<float*>(static_cast<char*>(workspace) + TileSumBytes(queries))};
    while ((1u << a.pageShift) < page_size)
    {
        ++a.pageShift;
    }
    const hipError_t launched = head_dim == 64 ? LaunchPagedAttention<64>(AsStream(stream), a)
                                               : LaunchPagedAttention<128>(AsStream(stream), a);
    return launched == hipSuccess ? MUYO_OK : HipStatus(launched, name);
}
