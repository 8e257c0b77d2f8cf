// The fp16 cache's attention over each query's own keys.
#pragma once

#include "paged_attention_core.hpp"

namespace muyo
{
struct PagedAttentionF16Args : PagedAttentionArgs
{
    const uint16_t* kcache;
    const uint16_t* vcache;
};

namespace
{
typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

// Softmax weights are held in two planes of f16, which ends at 2^16: the weight of the maximum is 2^kWeightBias, and
// 2^15 when a later one has run kLag binary orders ahead.
constexpr float kLag = 4.0f;
constexpr float kWeightBias = 15.0f - kLag;
constexpr uint32_t kTile = 32;            // keys of a tile: what a wave takes at a time
constexpr int kHalves = kTile / 16;       // matrix operands of 16 keys
constexpr float kLowScale = 2048.0f;      // of the low plane: what 11 bits of the high one leave, in f16's range again

template <bool kOnce>
__device__ __forceinline__ half8 LoadRow(const uint16_t* p)
{
    return kOnce ? __builtin_nontemporal_load(reinterpret_cast<const half8*>(p)) : *reinterpret_cast<const half8*>(p);
}

/// LDS byte of 16-byte chunk `chunk` of V row `row`: chunks are permuted by the row so that the eight
/// rows by two chunks that half a wave's transposing read takes lie in different banks.
template <int kHd>
__device__ __forceinline__ uint32_t ValueAt(uint32_t row, uint32_t chunk)
{
    const uint32_t by = kHd == 128 ? 2 * (row & 7u) : 2 * ((row >> 1) & 3u);
    return row * (2 * kHd) + (chunk ^ by) * 16;
}

/// LDS of OwnKeys: V of a wave's tile, and what its waves tell each other.
template <int kHd>
inline constexpr uint32_t kOwnKeysBytes = kWaves * kTile * 2 * kHd;

struct OwnKeysSpace
{
    float waveBase[kWaves][kMaxGroup];
    float waveTotal[kWaves][kMaxGroup];
    float headScale[kMaxGroup];  // scaleLog2
    ShareSpace share;
};

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
///
/// kPieces: nothing is joined here, what is not cut goes to `wholes`. `block` is the share, or the kv head of
/// `wholeQuery`.
template <int kHd, bool kSplit, bool kPieces>
__device__ __forceinline__ void OwnKeys(const PagedAttentionF16Args& a, uint32_t block, uint32_t wholeQuery,
                                        uint8_t* lds, OwnKeysSpace& shared)
{
    constexpr int kSteps = kHd / 32;               // matrix operations over a head's channels
    constexpr int kChannels = kHd / 16;            // 16-channel blocks of the output
    constexpr uint32_t kChunks = kHd / 8;          // 16-byte chunks of a row
    constexpr uint32_t kRows = kWave / kChunks;    // V rows of one load of the wave
    constexpr int kHalfLoads = 16 / kRows;         // V loads of 16 keys
    constexpr uint32_t kWaveBytes = kOwnKeysBytes<kHd> / kWaves;  // V of a tile; later O^T of 16 heads in f32
    static_assert(kWaveBytes >= kMaxGroup * kHd * 4, "O^T fits where V was");
    auto& waveBase = shared.waveBase;
    auto& waveTotal = shared.waveTotal;
    auto& headScale = shared.headScale;

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
        const Share first = FirstShare<kTile>(a, block, lane, shared.share);
        share = first.share;
        at = first.at;
        stop = first.stop;
        if (at >= stop)
        {
            if (a.cutsByUnit == 0 && threadIdx.x == 0)
            {
                a.cuts[block] = cut;
            }
            return;
        }
        query = first.query;
        queryAt = first.queryAt;
        range = first.range;
        g = 0;
    }
    else
    {
        query = wholeQuery;
        g = block;
        range = RangeOf<kTile>(a, query);
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
                range = RangeOf<kTile>(a, query);
                continue;
            }
            const uint32_t cost = CostOf<kTile>(range.tiles);
            g = __builtin_amdgcn_readfirstlane((at - queryAt) / cost);
            unitAt = __builtin_amdgcn_readfirstlane(queryAt + g * cost);
            const uint32_t from = __builtin_amdgcn_readfirstlane(at - unitAt);
            const uint32_t to = __builtin_amdgcn_readfirstlane(min(cost, from + (stop - at)));
            at = unitAt + to;
            tile0 = from > kSetupTiles<kTile> ? from - kSetupTiles<kTile> : 0;
            tile1 = to > kSetupTiles<kTile> ? to - kSetupTiles<kTile> : 0;
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
        auto bestOf = [&](uint32_t h) {
            float best = waveBase[0][h];
#pragma unroll
            for (int w = 1; w < kWaves; ++w)
            {
                best = fmaxf(best, waveBase[w][h]);
            }
            return best;
        };
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
            const uint64_t head = (static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + h;
            const bool isWhole = !kSplit || whole;
            if (!kPieces && isWhole)
            {
                const float inv = 1.0f / den;
                const float4v x = den == 0.0f ? float4v{} : num * inv;
                *reinterpret_cast<float4v*>(a.out + head * kHd + channel) = x;
            }
            else
            {
                const uint64_t piece = 2 * block + (tile0 == 0 ? 1 : 0);
                float* slot = kPieces && isWhole ? a.wholes + head * (kHd + 4)
                                                 : a.partials + (piece * a.group + h) * (kHd + 4);
                *reinterpret_cast<float4v*>(slot + 4 + channel) = num;
                if (channel == 0)
                {
                    slot[0] = bestOf(h);
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
                const uint32_t last = (unitAt + CostOf<kTile>(range.tiles) - 1) / share;
                const uint32_t pieces = whole ? 0 : last - block + 1;
                const uint4 join = make_uint4(query, g, block, pieces);
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
                range = RangeOf<kTile>(a, query);
            }
        }
    } while (kSplit && at < stop);
    if constexpr (kSplit)
    {
        if (a.cutsByUnit == 0 && threadIdx.x == 0)
        {
            a.cuts[block] = cut;
        }
    }
}
}  // namespace
}  // namespace muyo
