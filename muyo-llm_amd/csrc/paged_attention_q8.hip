// Attention of single tokens over a paged cache of 8-bit values with a scale per row and kv head.
#include <cmath>

#include "paged_attention_core.hpp"

namespace muyo
{
namespace
{
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr uint32_t kTile = 32;       // keys of a tile
constexpr int kParts = kTile / 16;   // matrix operands of 16 keys
constexpr int kPlanes = 3;           // of weights, 8 bits each: what f32 holds
constexpr float kLag = 8.0f;         // binary orders that a weight may be above 1: with 4 a long batch takes 2 % more

struct PagedAttentionQ8Args : PagedAttentionArgs
{
    const uint8_t* kcache;
    const uint8_t* vcache;
    const float* kscales;
    const float* vscales;
};

template <bool kOnce, typename T>
__device__ __forceinline__ T LoadOnce(const void* p)
{
    return kOnce ? __builtin_nontemporal_load(reinterpret_cast<const T*>(p)) : *reinterpret_cast<const T*>(p);
}

/// The upper halves of two f32, `first`'s in the lower half.
__device__ __forceinline__ uint32_t UpperHalves(float first, float second)
{
    return __builtin_amdgcn_perm(__float_as_uint(second), __float_as_uint(first), 0x07060302u);
}

/// Eight codes as bf16, which holds each: whole numbers of 7 bits, or 4 bits and an exponent.
template <int kFormat>
__device__ __forceinline__ bf8 ToBf16(uint32_t lo, uint32_t hi)
{
    uint4v words;
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        const uint32_t codes = i == 0 ? lo : hi;
        if constexpr (kFormat == MUYO_KV_INT8)
        {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                x[e] = static_cast<float>(static_cast<int8_t>(codes >> (8 * e)));
            }
            words[2 * i] = UpperHalves(x[0], x[1]);
            words[2 * i + 1] = UpperHalves(x[2], x[3]);
        }
        else
        {
            words[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
            words[2 * i + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true));
        }
    }
    return __builtin_bit_cast(bf8, words);
}

/// Eight codes as f16, which holds each too.
template <int kFormat>
__device__ __forceinline__ half8 ToF16(uint32_t lo, uint32_t hi)
{
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    uint4v words;
#pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        const uint32_t codes = i == 0 ? lo : hi;
        if constexpr (kFormat == MUYO_KV_INT8)
        {
            // 128 above the code, below f16's upper byte of 1024: 1152 above it.
            const uint32_t above = codes ^ 0x80808080u;
            const half2v by = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
            const half2v first =
                __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, above, 0x04010400u)) + by;
            const half2v second =
                __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, above, 0x04030402u)) + by;
            words[2 * i] = __builtin_bit_cast(uint32_t, first);
            words[2 * i + 1] = __builtin_bit_cast(uint32_t, second);
        }
        else
        {
            words[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false));
            words[2 * i + 1] =
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true));
        }
    }
    return __builtin_bit_cast(half8, words);
}

/// Planes of eight f32, each the first 8 bits of what the ones before leave: together exactly the value.
__device__ __forceinline__ void Split(const float (&x)[8], bf8 (&planes)[kPlanes])
{
    float left[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
    {
        left[c] = x[c];
    }
#pragma unroll
    for (int p = 0; p < kPlanes; ++p)
    {
        uint4v words;
#pragma unroll
        for (int c = 0; c < 8; c += 2)
        {
            words[c / 2] = UpperHalves(left[c], left[c + 1]);
        }
        planes[p] = __builtin_bit_cast(bf8, words);
#pragma unroll
        for (int c = 0; c < 8; ++c)
        {
            left[c] -= __uint_as_float(__float_as_uint(left[c]) & 0xFFFF0000u);
        }
    }
}

/// LDS byte of 16-byte chunk `chunk` of V row `row` in bf16: chunks are permuted by the row so that the eight
/// rows by two chunks that half a wave's transposing read takes lie in different banks.
template <int kHd>
__device__ __forceinline__ uint32_t ValueAt(uint32_t row, uint32_t chunk)
{
    const uint32_t by = kHd == 128 ? 2 * (row & 7u) : 2 * ((row >> 1) & 3u);
    return row * (2 * kHd) + (chunk ^ by) * 16;
}

/// The fp16 cache's attention (paged_attention_f16.hpp) with codes for K and V: the same shares, masks and joins, and
/// operands in the same places. What differs:
///   - K's codes are widened to f16, which holds them exactly, in registers on the way to the matrix cores, where they
///     meet the same two planes of q; a key's scale multiplies its score;
///   - V's are widened to bf16, as exact, on the way to LDS; a key's weight is multiplied by its scale before it meets
///     them, in three planes of bf16, whose exponent is f32's: all 24 bits of weights down to 2^-31 with scales down to
///     2^-79. (Two planes of f16 would want those products kept in f16's range, a second running maximum.) Three matrix
///     operations for the fp16 cache's two;
///   - f32 ends: raw scores are below 2^30 (q / 2^e below 2^14, codes of up to 448, 128 channels) before a K scale of up
///     to 2^96, and a sum over n keys is of weights of up to 2^kLag, codes and V scales of up to 2^110 / n;
///   - a tile is half the bytes, so two are on their way.
///
/// What bounds it: two waves of a SIMD taking turns at the codes' widening (176 vector operations of 390 for a tile of
/// 128 channels), the matrix cores and the wait for either. 64 sequences of 1 to 16384 keys (28 / 4 heads of 128, pages
/// of 16, 554 MB): 97 us and 5 for the join, 5.7 TB/s where the best streaming read here has 6.9; the vector units are
/// busy for 42 us of it, the matrix cores for 17. Three waves, of one tile each, spill their registers (168) and take
/// 147 us in all, two waves of one tile 125. One sequence of 32749 keys 13 us and 5
/// for the join; 16 of up to 500 keys 6.1.
template <int kHd, int kFormat, bool kSplit>
__global__ __launch_bounds__(kBlock, kHd == 64 ? 3 : 2) void PagedAttentionQ8Kernel(PagedAttentionQ8Args a)
{
    constexpr int kSteps = kHd / 32;             // matrix operations over a head's channels
    constexpr int kChunksK = kHd / 64;           // 16-byte loads of a lane from a K row
    constexpr int kChannels = kHd / 16;          // 16-channel blocks of the output
    constexpr int kAtOnce = 4;                   // of them
    constexpr uint32_t kLanesV = kHd / 16;       // lanes of a V row
    constexpr uint32_t kRows = kWave / kLanesV;  // V rows of one load of the wave
    constexpr int kPartLoads = 16 / kRows;       // V loads of 16 keys
    constexpr uint32_t kWaveBytes = kTile * 2 * kHd;  // V of a tile; later O^T of 16 heads in f32
    static_assert(kWaveBytes >= kMaxGroup * kHd * 4, "O^T fits where V was");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kWaveBytes];
    __shared__ __attribute__((aligned(16))) float waveScales[kWaves][2 * kTile];  // of a tile: K's, V's
    __shared__ float waveBase[kWaves][kMaxGroup];
    __shared__ float waveTotal[kWaves][kMaxGroup];
    __shared__ float headScale[kMaxGroup];  // scaleLog2
    __shared__ ShareSpace space;

    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t column = lane % 16;  // the head (of the kv head's group) in operands and results
    const uint32_t quad = lane / 16;
    const uint32_t pageSize = 1u << a.pageShift;

    uint32_t query, g;
    KeyRange range;
    uint32_t at = 0;
    uint32_t stop = 0;
    uint32_t share = 0;
    uint32_t queryAt = 0;
    uint32_t unitAt = 0;
    uint4 cut = make_uint4(0, 0, 0, 0);
    if constexpr (kSplit)
    {
        const Share first = FirstShare<kTile>(a, blockIdx.x, lane, space);
        share = first.share;
        at = first.at;
        stop = first.stop;
        if (at >= stop)
        {
            if (a.cutsByUnit == 0 && threadIdx.x == 0)
            {
                a.cuts[blockIdx.x] = cut;
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
        query = blockIdx.y;
        g = blockIdx.x;
        range = RangeOf<kTile>(a, query);
    }

    uint8_t* const mine = lds + wave * kWaveBytes;
    float* const scales = waveScales[wave];
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

        // q is requested before the first tile and made into operands while that arrives. A lane's chunk of a K row
        // is 16 channels, two matrix operations' of 8 each: q's are taken in that order.
        float4v qv[kSteps][2];
        {
            const float* from =
                a.q + ((static_cast<uint64_t>(query) * a.kvHeads + g) * a.group + min(column, a.group - 1)) * kHd +
                16 * quad;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                qv[s][0] = *reinterpret_cast<const float4v*>(from + 64 * (s / 2) + 8 * (s % 2));
                qv[s][1] = *reinterpret_cast<const float4v*>(from + 64 * (s / 2) + 8 * (s % 2) + 4);
            }
        }
        __builtin_amdgcn_sched_barrier(0);

        struct Pages
        {
            uint32_t of[kParts];
        };
        // The part of a tile behind the table's end, if any, has the last page's id: its keys are past the
        // range, and so masked.
        auto pagesOf = [&](uint32_t tile) {
            Pages ids;
            tile = min(tile, tile1 - 1);
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
                const uint32_t entry = ((range.firstTile + tile) * kTile + 16 * part) >> a.pageShift;
                ids.of[part] = static_cast<uint32_t>(ScalarLoad(table + min(entry, a.tablePages - 1)));
            }
            return ids;
        };
        struct Tile
        {
            Pages pages;
            uint4v k[kParts][kChunksK];
            float scale;  // of K's row lane % 32, or of V's in the wave's upper half
            uint4v v[kParts][kPartLoads];
        };
        Tile even, odd;  // two tiles are on their way
        // A tile's K, then its V: loads complete in order, and the scores wait only for K. Pages outside the
        // cache are read as page 0, whose rows are then masked. Tiles past the last are requests for one row of it:
        // a request under a condition would make the waits for the other tile ones for everything.
        auto request = [&](Tile& now, uint32_t tile, const Pages& pages) {
            const uint32_t lanes = tile < tile1 ? ~0u : 0u;
            tile = min(tile, tile1 - 1);
            now.pages = pages;
            uint64_t base[kParts];
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
                const uint32_t page = now.pages.of[part] < a.pages ? now.pages.of[part] : 0;
                const uint32_t row = ((range.firstTile + tile) * kTile + 16 * part) & (pageSize - 1);
                base[part] = ((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + row;
            }
            const uint32_t keyAt = (column * kHd + 16 * quad) & lanes;
            const uint32_t valueAt = (lane * 16) & lanes;
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
#pragma unroll
                for (int i = 0; i < kChunksK; ++i)
                {
                    now.k[part][i] = LoadOnce<kSplit, uint4v>(a.kcache + base[part] * kHd + keyAt + 64 * i);
                }
            }
            static_assert(kTile == 32 && kParts == 2, "a lane for each scale");
            const uint64_t first = base[0];
            const uint64_t second = base[1];
            now.scale = LoadOnce<kSplit, float>((lane < 32 ? a.kscales : a.vscales) +
                                                (quad % 2 == 0 ? first : second) + column);
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
#pragma unroll
                for (int j = 0; j < kPartLoads; ++j)
                {
                    now.v[part][j] = LoadOnce<kSplit, uint4v>(a.vcache + base[part] * kHd + valueAt + j * kRows * kHd);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };

        float4v o[kChannels];
#pragma unroll
        for (int c = 0; c < kChannels; ++c)
        {
            o[c] = float4v{};
        }
        float base = -INFINITY;  // the raw score that weights are relative to; -inf: none yet
        float runSum = 0.0f;     // of this lane's keys
        {
            const Pages first = pagesOf(tile0 + wave);
            const Pages second = pagesOf(tile0 + wave + kWaves);
            request(even, tile0 + wave, first);
            request(odd, tile0 + wave + kWaves, second);
        }

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

        auto take = [&](Tile& now, uint32_t tile) {
            const Pages next = pagesOf(tile + 2 * kWaves);  // on their way while the scores are made
            __builtin_amdgcn_sched_barrier(0);
            float4v score[kParts];
#pragma unroll
            for (int part = 0; part < kParts; ++part)
            {
                score[part] = float4v{};
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                half8 k[kParts];
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                {
                    k[part] = ToF16<kFormat>(now.k[part][s / 2][2 * (s % 2)], now.k[part][s / 2][2 * (s % 2) + 1]);
                    score[part] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[part], qlo[s], score[part], 0, 0, 0);
                }
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                {
                    score[part] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[part], qhi[s], score[part], 0, 0, 0);
                }
            }
            const uint32_t key0 = (range.firstTile + tile) * kTile;
            bool inside = key0 >= range.begin && key0 + kTile <= range.end;
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
                inside = inside && now.pages.of[part] < a.pages;
            }
            if (!inside && lane >= 32)
            {
                const uint32_t key = key0 + lane % 32;
                const bool first = now.pages.of[0] < a.pages;
                const bool second = now.pages.of[1] < a.pages;
                const bool there = quad % 2 == 0 ? first : second;
                now.scale = there && key >= range.begin && key < range.end ? now.scale : 0.0f;
            }
            scales[lane] = now.scale;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int part = 0; part < kParts; ++part)
            {
                score[part] *= *reinterpret_cast<const float4v*>(scales + 16 * part + 4 * quad);
            }
            if (!inside)
            {
#pragma unroll
                for (uint32_t part = 0; part < kParts; ++part)
                {
                    const bool there = now.pages.of[part] < a.pages;
#pragma unroll
                    for (int j = 0; j < kPartLoads; ++j)
                    {
                        const uint32_t key = key0 + 16 * part + j * kRows + lane / kLanesV;
                        if (!there || key < range.begin || key >= range.end)
                        {
                            now.v[part][j] = uint4v{};
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                    {
                        const uint32_t key = key0 + 16 * part + 4 * quad + r;
                        if (!there || key < range.begin || key >= range.end)
                        {
                            score[part][r] = -INFINITY;
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t part = 0; part < kParts; ++part)
            {
#pragma unroll
                for (int j = 0; j < kPartLoads; ++j)
                {
                    const uint32_t row = 16 * part + j * kRows + lane / kLanesV;
                    const uint32_t chunk = 2 * (lane % kLanesV);
                    const uint4v codes = now.v[part][j];
                    *reinterpret_cast<bf8*>(mine + ValueAt<kHd>(row, chunk)) = ToBf16<kFormat>(codes[0], codes[1]);
                    *reinterpret_cast<bf8*>(mine + ValueAt<kHd>(row, chunk + 1)) =
                        ToBf16<kFormat>(codes[2], codes[3]);
                }
            }
            // The wave's LDS operations complete in order; this keeps the compiler's order too.
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            request(now, tile + 2 * kWaves, next);
            // V of some channels, transposed; the first are on their way while the weights are made.
            auto valuesOf = [&](int group, bf8 (&vt)[kAtOnce]) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                {
                    uint8_t* row = mine + (readAt ^ (32u * (group * kAtOnce + i)));
                    const short4v first = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) short4v*)row);
                    const short4v second = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) short4v*)(row + 16 * 2 * kHd));
                    vt[i] = __builtin_bit_cast(bf8, __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7));
                }
            };
            bf8 vt[kAtOnce];
            valuesOf(0, vt);
            __builtin_amdgcn_sched_barrier(0);

            float tileMax = -INFINITY;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
            {
                tileMax = fmaxf(tileMax, fmaxf(fmaxf(score[part][0], score[part][1]),
                                               fmaxf(score[part][2], score[part][3])));
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
                }
            }
            bf8 weights[kPlanes];
            const float from = base == -INFINITY ? 0.0f : base;  // without keys so far every score is -inf
            float sum = 0.0f;
            float scaled[8];
#pragma unroll
            for (int part = 0; part < kParts; ++part)
            {
                float4v p;
                const float4v vscale = *reinterpret_cast<const float4v*>(scales + 32 + 16 * part + 4 * quad);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    p[r] = __builtin_amdgcn_exp2f((score[part][r] - from) * scaleLog2);
                    scaled[4 * part + r] = p[r] * vscale[r];
                }
                sum += (p[0] + p[1]) + (p[2] + p[3]);
            }
            Split(scaled, weights);
            runSum += sum;
            // A group's planes in turn over its channels: sums that do not wait for one another.
#pragma unroll
            for (int group = 0; group < kChannels / kAtOnce; ++group)
            {
                bf8 later[kAtOnce];
                if (group + 1 < kChannels / kAtOnce)
                {
                    valuesOf(group + 1, later);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int p = kPlanes - 1; p >= 0; --p)
                {
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                    {
                        const int c = group * kAtOnce + i;
                        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[i], weights[p], o[c], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                {
                    vt[i] = later[i];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        uint32_t tile = tile0 + wave;
        // In pairs: a way out between them would meet the way round, where the compiler then waits for both.
        for (; tile + kWaves < tile1; tile += 2 * kWaves)
        {
            take(even, tile);
            take(odd, tile + kWaves);
        }
        if (tile < tile1)
        {
            take(even, tile);
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
                const float4v x = base == -INFINITY && runSum == 0.0f ? float4v{} : o[c] * factor;
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
                const uint32_t last = (unitAt + CostOf<kTile>(range.tiles) - 1) / share;
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
                range = RangeOf<kTile>(a, query);
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

template <int kHd, int kFormat>
hipError_t LaunchQ8(hipStream_t s, const PagedAttentionQ8Args& a)
{
    return LaunchPagedAttention<kHd, kTile>(s, a, PagedAttentionQ8Kernel<kHd, kFormat, false>,
                                                   PagedAttentionQ8Kernel<kHd, kFormat, true>);
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_paged_attention_decode_q8kv_workspace_bytes(uint32_t queries, uint32_t heads,
                                                                   uint32_t kv_heads, uint32_t head_dim)
{
    if (!AttentionShape(queries, heads, kv_heads, head_dim))
    {
        return 0;
    }
    return DecodeWorkspaceBytes(queries, heads, kv_heads, head_dim);
}

extern "C" int muyo_paged_attention_decode_q8kv(const float* q, const void* kcache, const void* vcache,
                                                const float* kscales, const float* vscales, float* out,
                                                const int32_t* tables, uint32_t sequences, uint32_t table_pages,
                                                const int32_t* query_sequence, const int32_t* positions,
                                                uint32_t queries, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                                uint32_t pages, uint32_t page_size, uint32_t format, uint32_t window,
                                                float scale, void* workspace, uint64_t workspace_bytes, void* stream)
{
    const char* name = "paged_attention_decode_q8kv";
    if (format > MUYO_KV_E4M3)
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: unknown format %u", name, format);
    }
    const uint64_t scaleBytes = 4ull * pages * page_size * kv_heads;
    const uint64_t cacheBytes = scaleBytes / 4 * head_dim;
    const Range caches[] = {{kcache, cacheBytes, "kcache"},
                            {vcache, cacheBytes, "vcache"},
                            {kscales, scaleBytes, "kscales"},
                            {vscales, scaleBytes, "vscales"}};
    const AttentionCall call{q, out, tables, sequences, table_pages, query_sequence, positions, queries, heads,
                             kv_heads, head_dim, pages, page_size, scale, workspace, workspace_bytes,
                             muyo_paged_attention_decode_q8kv_workspace_bytes(queries, heads, kv_heads, head_dim)};
    const int checked = CheckAttention(name, call, caches, 4, 4);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    PagedAttentionQ8Args a{};
    FillAttentionArgs(a, call, window);
    a.kcache = static_cast<const uint8_t*>(kcache);
    a.vcache = static_cast<const uint8_t*>(vcache);
    a.kscales = kscales;
    a.vscales = vscales;
    const hipStream_t s = AsStream(stream);
    const hipError_t launched = head_dim == 64
                                    ? (format == MUYO_KV_INT8 ? LaunchQ8<64, MUYO_KV_INT8>(s, a)
                                                              : LaunchQ8<64, MUYO_KV_E4M3>(s, a))
                                    : (format == MUYO_KV_INT8 ? LaunchQ8<128, MUYO_KV_INT8>(s, a)
                                                              : LaunchQ8<128, MUYO_KV_E4M3>(s, a));
    return launched == hipSuccess ? MUYO_OK : HipStatus(launched, name);
}
