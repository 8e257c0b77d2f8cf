// Attention of single tokens over a paged fp16 cache whose sequences go on from the same first keys: those are read
// once for many queries, and joined with each query's own (paged_attention.hip).
#include <algorithm>

#include "paged_attention_f16.hpp"
#include "prefill_core.hpp"

namespace muyo
{
namespace
{
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr uint32_t kStep = 64;            // keys of one step: an LDS buffer of K and V rows
constexpr uint32_t kStepPages = kStep / 16;
constexpr uint32_t kRowsOfWave = 32;      // rows are (query, head of a kv head's group)
constexpr uint32_t kRowsOfBlock = kRowsOfWave * kWaves;
constexpr uint32_t kMaxChunks = 128;
constexpr uint32_t kFewChunks = 8;
constexpr uint32_t kTurn = 256;           // workgroups of a kind in turn: one on each CU

struct PagedPrefixArgs
{
    const float* q;
    const uint16_t* kcache;
    const uint16_t* vcache;
    float* out;
    const int32_t* tables;
    uint32_t sequences, tablePages;
    const int32_t* querySequence;
    uint32_t queries, group, kvHeads;
    const int32_t* prefix;  // its row of tables, its keys
    uint32_t pages, pageShift;
    float scale;
    uint32_t chunks;        // of the prefix, at most
    // The own keys': what no share cut, and where shares are dealt out those of each (query, kv head) and their pieces.
    const float* wholes;
    const uint4* cuts;
    const float* pieces;
    float* partials;        // [kv_heads][queries * group][chunks][4 + headDim], as the own keys' partials
};

/// The prefix's keys, and the steps of a chunk of them.
struct PrefixKeys
{
    uint32_t row, keys, perChunk, chunks;
};

__device__ __forceinline__ PrefixKeys KeysOf(const PagedPrefixArgs& a)
{
    const int32_t row = a.prefix[0];
    const int32_t keys = a.prefix[1];
    PrefixKeys p;
    p.row = static_cast<uint32_t>(row);
    p.keys = p.row < a.sequences && keys > 0 ? min(static_cast<uint32_t>(keys), a.tablePages << a.pageShift) : 0;
    const uint32_t steps = (p.keys + kStep - 1) / kStep;
    p.perChunk = max((steps + a.chunks - 1) / a.chunks, 1u);
    p.chunks = (steps + p.perChunk - 1) / p.perChunk;
    return p;
}

template <int kHd>
inline constexpr int kPrefixStages = kHd == 128 ? 2 : 3;

/// LDS of PrefixKeysOfRows: K and V of its steps, and later the rows' results.
template <int kHd>
inline constexpr uint32_t kPrefixBytes = kPrefixStages<kHd> * 2 * kStep * 2 * kHd;

/// A wave has 32 rows, the columns of its matrix operations; a workgroup's four waves share each step of 64 keys of K
/// and V through LDS, where they go straight from memory a step ahead. Per step a wave
///   - forms S^T (keys x rows) = K . q^T, K from LDS, q in registers as two planes of f16 (of q / 2^e, e by the row's
///     largest value, as in the attention over own keys: the two are joined by their raw scores);
///   - makes the softmax weights of a row's 32 keys in a lane, one exchange with the lane 32 away, in two planes that
///     keep the bits of own keys' weights (accumulators that follow a maximum only 2^10 ahead would save 1.5 % of the
///     time and cost 1e-4 of a result 20 nats below a key with a value of 0);
///   - O^T (channels x rows) += V^T . P^T, V^T by transposing LDS reads, keys in the order that the scores have.
/// The weights' low plane, times 2048, has sums of its own, so that small weights count beside a key that has most of
/// the weight: at head_dim 64 accumulators beside the others, at 128, where these would not fit the registers, sums of
/// the step that are added to the others by a multiply-add.
///
/// What bounds it: vector work, matrix work and LDS reads, which a SIMD's two waves overlap little: each wave reads all
/// of a step's K and V for its 32 rows. 250 queries of 28 / 4 heads of 128 with 16381 keys: 137 us with one own key
/// each, 146 with up to 500, of which at 2.4 GHz the vector units are busy for 57, the matrix cores for 49 and LDS for
/// 26 (24 of them K's and V's reads at 128 bytes a clock), and 12 more in bank conflicts (the clock is below that
/// here). 32 keys at a time took 2 % more, without V's reads ahead of the weights 2 to 4; one wave a SIMD, with the
/// next step's matrix operations between this one's weights, 200 us; other orders of the chunks in LDS, with fewer bank
/// conflicts, and a wave's priority in either kind of work, no less.
///
/// Steps that reach past the prefix, or into a page that is not there, are masked: scores to -inf, and V's rows to 0 in
/// LDS, since 0 * NaN would be NaN.
///
/// `block` goes over (kv head, chunk) fastest, then blocks of 128 rows.
template <int kHd>
__device__ __forceinline__ void PrefixKeysOfRows(const PagedPrefixArgs& a, uint32_t block, uint8_t* lds)
{
    constexpr int kStages = kPrefixStages<kHd>;
    constexpr bool kKeepLow = kHd == 64;
    constexpr uint32_t kRowBytes = 2 * kHd;
    constexpr uint32_t kChunks = kHd / 8;                // 16-byte chunks of a row
    constexpr uint32_t kRowsPerLoad = kWave / kChunks;
    constexpr uint32_t kMatrixBytes = kStep * kRowBytes;  // K or V of a step
    constexpr int kMatrixLoads = kMatrixBytes / 1024 / kWaves;  // of a wave
    constexpr int kLoads = 2 * kMatrixLoads;
    constexpr int kChannels = kHd / 32;                  // 32-channel blocks of the output
    constexpr int kHalves = kStep / 32;                  // matrix operands of 32 keys
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t h = lane / 32;
    const uint32_t g = block % a.kvHeads;
    const uint32_t chunk = block / a.kvHeads % a.chunks;
    const PrefixKeys prefix = KeysOf(a);
    if (chunk >= prefix.chunks)
    {
        return;
    }
    const uint32_t rows = a.queries * a.group;
    const uint32_t row0 = block / (a.kvHeads * a.chunks) * kRowsOfBlock + wave * kRowsOfWave;
    const bool active = row0 < rows;  // a wave past the rows only loads
    const uint32_t row = min(row0 + lane % 32, rows - 1);
    const uint32_t firstStep = chunk * prefix.perChunk;
    const uint32_t steps = min(prefix.perChunk, (prefix.keys + kStep - 1) / kStep - firstStep);
    const uint32_t pageSize = 1u << a.pageShift;
    const int32_t* table = a.tables + static_cast<uint64_t>(prefix.row) * a.tablePages;

    // Load i of a wave: 1 KB of K (the first kMatrixLoads of a step) or V, rows of one 16-key part of the step. Chunks
    // of 16 bytes are permuted by the row: K's by row % 8, V's by 2 (row % 4).
    const uint32_t ldsBase =
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
    const uint32_t laneRow = lane / kChunks;
    const uint32_t kAt = (lane % kChunks ^ ((wave * kRowsPerLoad + laneRow) & 7u)) * 16 + laneRow * kRowBytes;
    const uint32_t vAtLoad = (lane % kChunks ^ (laneRow & 3u) * 2) * 16 + laneRow * kRowBytes;
    // Pages of a step's parts; those behind the table's end have the last one's id, and are past the prefix.
    struct Pages
    {
        uint32_t of[kStepPages];
    };
    auto pagesOf = [&](uint32_t step) {
        Pages ids;
#pragma unroll
        for (uint32_t part = 0; part < kStepPages; ++part)
        {
            const uint32_t entry = ((firstStep + min(step, steps - 1)) * kStep + 16 * part) >> a.pageShift;
            ids.of[part] = static_cast<uint32_t>(ScalarLoad(table + min(entry, a.tablePages - 1)));
        }
        return ids;
    };
    auto request = [&](uint32_t stage, uint32_t step, const Pages& ids) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
        {
            const bool isV = i >= kMatrixLoads;
            const uint32_t first = (wave + i % kMatrixLoads * kWaves) * kRowsPerLoad;  // row of the step
            // The part is known up to the wave's half of 32 rows.
            const int part = i % kMatrixLoads;
            const uint32_t id =
                kHd == 128 ? ids.of[part] : wave < 2 ? ids.of[2 * part] : ids.of[2 * part + 1];
            const uint32_t page = id < a.pages ? id : 0;  // read, and masked
            const uint32_t at = ((firstStep + step) * kStep + first) & (pageSize - 1);
            const uint16_t* base = (isV ? a.vcache : a.kcache) +
                                   (((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + at) * kHd;
            LoadToLds(ldsBase + stage * 2 * kMatrixBytes + wave * 1024,
                      isV * kMatrixBytes + i % kMatrixLoads * kWaves * 1024, isV ? vAtLoad : kAt, base);
        }
    };

    // q's planes and a score's log2 units, as in the attention over own keys.
    half8 qhi[kHd / 16], qlo[kHd / 16];
    float scaleLog2;
    {
        float4v qv[kHd / 16][2];
        const float* from = a.q + (static_cast<uint64_t>(row / a.group) * a.kvHeads * a.group + g * a.group +
                                   row % a.group) * kHd + 8 * h;
#pragma unroll
        for (int s = 0; s < kHd / 16; ++s)
        {
            qv[s][0] = *reinterpret_cast<const float4v*>(from + 16 * s);
            qv[s][1] = *reinterpret_cast<const float4v*>(from + 16 * s + 4);
        }
        float largest = 0.0f;
#pragma unroll
        for (int s = 0; s < kHd / 16; ++s)
        {
#pragma unroll
            for (int c = 0; c < 8; ++c)
            {
                largest = fmaxf(largest, fabsf(qv[s][c / 4][c % 4]));
            }
        }
        largest = fmaxf(largest, PartnerLane<32>(largest));
        int e = 0;
        if (largest > 0.0f && largest < INFINITY)
        {
            (void)frexpf(largest, &e);
        }
        e -= 14;
        const float sign = a.scale == 0.0f ? 0.0f : a.scale < 0.0f ? -1.0f : 1.0f;
        scaleLog2 =
            a.scale == 0.0f ? 1.0f : fminf(fmaxf(ldexpf(fabsf(a.scale), e) * kLog2e, 0x1p-126f), 0x1.fffffep127f);
#pragma unroll
        for (int s = 0; s < kHd / 16; ++s)
        {
#pragma unroll
            for (int c = 0; c < 8; ++c)
            {
                const float x = ldexpf(qv[s][c / 4][c % 4], -e) * sign;
                qhi[s][c] = static_cast<_Float16>(x);
                qlo[s][c] = static_cast<_Float16>(x - static_cast<float>(qhi[s][c]));
            }
        }
        // Waited for here, outside the loop: the compiler's own wait would also cover the loads to LDS.
#pragma unroll
        for (int s = 0; s < kHd / 16; ++s)
        {
            asm volatile("" : "+v"(qhi[s]), "+v"(qlo[s]));
        }
    }

    floatx16 o[kChannels], oLow[kChannels];
#pragma unroll
    for (int c = 0; c < kChannels; ++c)
    {
        o[c] = floatx16{};
        oLow[c] = floatx16{};
    }
    float base = -INFINITY;
    float runSum = 0.0f;
    const uint32_t kRow = lane % 32;
    const uint32_t vRow = 4 * h + lane % 16 / 4;
    const uint32_t vChunk = (lane / 16 % 2 * 2 + lane % 4 / 2) ^ (vRow & 3u) * 2;
    const uint32_t vAt = vRow * kRowBytes + lane % 2 * 8;

    Pages now = pagesOf(0);
    Pages ahead[kStages - 1];  // of the steps on their way
#pragma unroll
    for (uint32_t s = 0; s < kStages - 1; ++s)
    {
        ahead[s] = s == 0 ? now : pagesOf(s);
        if (s < steps)
        {
            request(s, s, ahead[s]);
        }
    }
    uint32_t stage = 0;
    for (uint32_t t = 0; t < steps; ++t, stage = stage + 1 == kStages ? 0 : stage + 1)
    {
        const Pages next = pagesOf(t + kStages - 1);
        now = ahead[0];
#pragma unroll
        for (uint32_t s = 0; s + 1 < kStages - 1; ++s)
        {
            ahead[s] = ahead[s + 1];
        }
        ahead[kStages - 2] = next;
        if (kStages <= 2 || t + 1 >= steps)
        {
            WaitAndMeet<0>();
        }
        else
        {
            WaitAndMeet<kLoads>();
        }
        if (t + kStages - 1 < steps)
        {
            request(stage == 0 ? kStages - 1 : stage - 1, t + kStages - 1, next);
        }
        const uint32_t key0 = (firstStep + t) * kStep;
        bool inside = key0 + kStep <= prefix.keys;
#pragma unroll
        for (uint32_t part = 0; part < kStepPages; ++part)
        {
            inside = inside && now.of[part] < a.pages;
        }
        uint8_t* const kRows = lds + stage * 2 * kMatrixBytes;
        uint8_t* const vRows = kRows + kMatrixBytes;
        if (!inside)
        {
            for (uint32_t i = threadIdx.x; i < kStep * kChunks; i += kBlock)
            {
                const uint32_t r = i / kChunks;
                const uint32_t first = r / 16 % 2 == 0 ? now.of[0] : now.of[1];
                const uint32_t second = r / 16 % 2 == 0 ? now.of[2] : now.of[3];
                if (key0 + r >= prefix.keys || (r < 32 ? first : second) >= a.pages)
                {
                    *reinterpret_cast<half8*>(vRows + r * kRowBytes + i % kChunks * 16) = half8{};
                }
            }
            __syncthreads();
        }
        if (!active)
        {
            continue;
        }
        floatx16 score[kHalves];
#pragma unroll
        for (int half = 0; half < kHalves; ++half)
        {
            const uint8_t* keys = kRows + half * 32 * kRowBytes;
            score[half] = floatx16{};
#pragma unroll
            for (int s = 0; s < kHd / 16; ++s)
            {
                const half8 k = *reinterpret_cast<const half8*>(keys + kRow * kRowBytes +
                                                                ((2 * s + h) ^ (kRow & 7u)) * 16);
                score[half] = Mfma(k, qlo[s], score[half]);
                score[half] = Mfma(k, qhi[s], score[half]);
            }
            if (!inside)
            {
                const bool there0 = now.of[2 * half] < a.pages;
                const bool there1 = now.of[2 * half + 1] < a.pages;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                {
                    const uint32_t key = key0 + 32 * half + 8 * (r / 4) + 4 * h + r % 4;
                    if (key >= prefix.keys || !(r < 8 ? there0 : there1))
                    {
                        score[half][r] = -INFINITY;
                    }
                }
            }
        }
        // V of 32 channels, transposed; the first are on their way while the weights are made.
        auto valuesOf = [&](int c, half8 (&vt)[2 * kHalves]) {
#pragma unroll
            for (int s = 0; s < 2 * kHalves; ++s)
            {
                const uint8_t* at = vRows + vAt + 16 * s * kRowBytes + (vChunk ^ (4u * c)) * 16;
                const half4 one = __builtin_bit_cast(
                    half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (__attribute__((address_space(3))) short4v*)(const_cast<uint8_t*>(at))));
                const half4 two = __builtin_bit_cast(
                    half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(
                               const_cast<uint8_t*>(at + 8 * kRowBytes))));
                vt[s] = __builtin_shufflevector(one, two, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        };
        half8 vt[2 * kHalves];
        valuesOf(0, vt);
        __builtin_amdgcn_sched_barrier(0);
        float stepMax = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r)
        {
            stepMax = fmaxf(stepMax, fmaxf(score[0][r], score[1][r]));
        }
        stepMax = fmaxf(stepMax, PartnerLane<32>(stepMax));
        const bool rises = stepMax != -INFINITY && (base == -INFINITY || (stepMax - base) * scaleLog2 > kLag);
        if (__any(rises))
        {
            const float factor =
                rises ? (base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((base - stepMax) * scaleLog2)) : 1.0f;
            base = rises ? stepMax : base;
            runSum *= factor;
#pragma unroll
            for (int c = 0; c < kChannels; ++c)
            {
                o[c] *= factor;
                if (kKeepLow)
                {
                    oLow[c] *= factor;
                }
            }
        }
        const float from = base == -INFINITY ? 0.0f : base;  // without keys so far every score is -inf
        half8 phi[2 * kHalves], plo[2 * kHalves];
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16 * kHalves; i += 2)
        {
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                p[e] = __builtin_amdgcn_exp2f(fmaf(score[i / 16][i % 16 + e] - from, scaleLog2, kWeightBias));
                sum[(i + e) % 4] += p[e];
            }
            // The high plane is cut off, the low one has what that leaves: one operation a pair and one a weight.
            const half2v hi = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(p[0], p[1]));
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                phi[i / 8][i % 8 + e] = hi[e];
                plo[i / 8][i % 8 + e] = static_cast<_Float16>(
                    fmaf(static_cast<float>(hi[e]), -kLowScale, kLowScale * p[e]));
            }
        }
        runSum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int c = 0; c < kChannels; ++c)
        {
            half8 later[2 * kHalves];
            if (c + 1 < kChannels)
            {
                valuesOf(c + 1, later);
            }
            __builtin_amdgcn_sched_barrier(0);
            floatx16 add = kKeepLow ? oLow[c] : floatx16{};
#pragma unroll
            for (int s = 0; s < 2 * kHalves; ++s)
            {
                add = Mfma(vt[s], plo[s], add);
                o[c] = Mfma(vt[s], phi[s], o[c]);
                if (c + 1 < kChannels)
                {
                    vt[s] = later[s];
                }
            }
            if (kKeepLow)
            {
                oLow[c] = add;
            }
            else
            {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                {
                    o[c][r] = fmaf(add[r], 1.0f / kLowScale, o[c][r]);
                }
            }
        }
    }

    // Out through LDS: a row's channels side by side.
    __syncthreads();
    if (!active)
    {
        return;
    }
    runSum += PartnerLane<32>(runSum);
    constexpr uint32_t kOutBytes = kRowsOfWave * kHd * 4;
    float* const mine = reinterpret_cast<float*>(lds + wave * kOutBytes);
#pragma unroll
    for (int c = 0; c < kChannels; ++c)
    {
        if (kKeepLow)
        {
            o[c] += oLow[c] * (1.0f / kLowScale);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            const uint32_t quad = 8 * c + 2 * r + h;  // of channels
            *reinterpret_cast<float4v*>(mine + kRow * kHd + 4 * (quad ^ (kRow & 7u))) =
                float4v{o[c][4 * r], o[c][4 * r + 1], o[c][4 * r + 2], o[c][4 * r + 3]};
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t here = min(rows - row0, kRowsOfWave);
    float* const to = a.partials + (static_cast<uint64_t>(g) * rows + row0) * a.chunks * (kHd + 4) +
                      static_cast<uint64_t>(chunk) * (kHd + 4);
    const uint64_t stride = static_cast<uint64_t>(a.chunks) * (kHd + 4);
    for (uint32_t i = lane; i < here * (kHd / 4); i += kWave)
    {
        const uint32_t r = i / (kHd / 4);
        const uint32_t quad = i % (kHd / 4);
        *reinterpret_cast<float4v*>(to + r * stride + 4 + 4 * quad) =
            *reinterpret_cast<const float4v*>(mine + r * kHd + 4 * (quad ^ (r & 7u)));
    }
    if (h == 0 && lane < here)
    {
        *reinterpret_cast<float4v*>(to + lane * stride) = float4v{base, runSum, scaleLog2, 0.0f};
    }
}

/// Both kinds of keys in one launch: workgroups for the prefix, whose matrix operations bound them, and for own keys,
/// which wait for memory, in turns of a CU each. The q of a workgroup may be read when others have ended, so none
/// writes `out`.
///
/// When both were built, two launches, the prefix's before the own keys', took 14.3 us for 3 queries (1009 keys and up
/// to 100 own, 14 / 2 heads of 64) and one 10.3; for 64 queries (8190 and up to 2000, 28 / 4 of 128) 53 and 45; for 250
/// (16381 and up to 500) 183 and 172. One takes 10.3, 39.4 and 157 now (each with 4 to 10 for the join); in turns of 8,
/// 128 and 512 workgroups the latter two take 49, 44 and 39, and 216, 178 and 167, with the own keys first 41 and 155.
template <int kHd, bool kSplit>
__global__ __launch_bounds__(kBlock, 2) void PagedPrefixKernel(PagedPrefixArgs a, PagedAttentionF16Args own,
                                                               uint32_t prefixBlocks, uint32_t ownBlocks)
{
    static_assert(kPrefixBytes<kHd> >= kOwnKeysBytes<kHd> && kPrefixBytes<kHd> >= kRowsOfBlock * kHd * 4,
                  "own keys' V and all results fit");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kPrefixBytes<kHd>];
    __shared__ OwnKeysSpace space;
    const uint32_t turns = min(prefixBlocks, ownBlocks) / kTurn * kTurn;  // of each kind
    uint32_t at = blockIdx.y * gridDim.x + blockIdx.x;
    if (at >= prefixBlocks + ownBlocks)
    {
        return;
    }
    bool isOwn;
    if (at < 2 * turns)
    {
        isOwn = at / kTurn % 2 != 0;
        at = at / (2 * kTurn) * kTurn + at % kTurn;
    }
    else
    {
        at -= turns;
        isOwn = at >= prefixBlocks;
        at -= isOwn ? prefixBlocks - turns : 0;
    }
    if (!isOwn)
    {
        PrefixKeysOfRows<kHd>(a, at, lds);
    }
    else
    {
        OwnKeys<kHd, kSplit, true>(own, kSplit ? at : at % a.kvHeads, at / a.kvHeads, lds, space);
    }
}

/// Joins a row's chunks with its own keys' pieces: kThreads threads a row, kHd / 4 of them over the channels, so many
/// pieces side by side, kDeep of each on their way. In a fixed order.
template <int kHd, int kThreads>
__global__ __launch_bounds__(256) void PagedPrefixJoinKernel(PagedPrefixArgs a)
{
    constexpr uint32_t kLanes = kHd / 4;
    constexpr uint32_t kSlices = kThreads / kLanes;
    constexpr uint32_t kDeep = 4;
    __shared__ float4v sliceNum[256 / kLanes][kLanes];
    __shared__ float4v sliceHead[256 / kLanes];
    const uint32_t heads = a.kvHeads * a.group;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * (256 / kThreads) + threadIdx.x / kThreads;
    const uint64_t items = static_cast<uint64_t>(a.queries) * heads;
    const PrefixKeys prefix = KeysOf(a);
    const uint32_t lane = threadIdx.x % kLanes;
    const uint32_t slice = threadIdx.x % kThreads / kLanes;
    const uint32_t at = threadIdx.x / kLanes;
    const uint32_t query = static_cast<uint32_t>(min(item, items - 1) / heads);
    const uint32_t head = static_cast<uint32_t>(min(item, items - 1) % heads);
    const bool is = item < items && static_cast<uint32_t>(a.querySequence[query]) < a.sequences;
    uint32_t first = 0;  // share of the own keys
    uint32_t pieces = 0;
    if (a.cuts != nullptr && is)
    {
        const uint4 cut = a.cuts[query * a.kvHeads + head / a.group];
        first = cut.z;
        pieces = cut.w;
    }
    const uint32_t parts = prefix.chunks + max(pieces, 1u);
    float base = -INFINITY;
    float den = 0.0f;
    float scaleLog2 = 1.0f;
    float4v num = float4v{};
    float* const out = a.out + (static_cast<uint64_t>(query) * heads + head) * kHd + 4 * lane;
    if (is)
    {
        const uint64_t rows = static_cast<uint64_t>(a.queries) * a.group;
        const float* const from = a.partials +
                                  ((head / a.group) * rows + static_cast<uint64_t>(query) * a.group + head % a.group) *
                                      a.chunks * (kHd + 4);
        const float* const whole = a.wholes + (static_cast<uint64_t>(query) * heads + head) * (kHd + 4);
        for (uint32_t p0 = slice; p0 < parts; p0 += kDeep * kSlices)
        {
            float4v of[kDeep], x[kDeep];
            float best = base;
#pragma unroll
            for (uint32_t i = 0; i < kDeep; ++i)
            {
                const uint32_t p = min(p0 + i * kSlices, parts - 1);
                // Piece 0 begins the own keys, the others are their shares' first.
                const uint32_t own = p - prefix.chunks;
                const uint64_t piece = 2 * (first + own) + (own == 0 ? 1 : 0);
                const float* at = p < prefix.chunks ? from + static_cast<uint64_t>(p) * (kHd + 4)
                                  : pieces == 0     ? whole
                                                    : a.pieces + (piece * a.group + head % a.group) * (kHd + 4);
                of[i] = *reinterpret_cast<const float4v*>(at);
                x[i] = *reinterpret_cast<const float4v*>(at + 4 + 4 * lane);
            }
#pragma unroll
            for (uint32_t i = 0; i < kDeep; ++i)
            {
                best = p0 + i * kSlices < parts ? fmaxf(best, of[i][0]) : best;
            }
            scaleLog2 = of[0][2];
            const float factor = base == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((base - best) * scaleLog2);
            base = best;
            den *= factor;
            num *= factor;
#pragma unroll
            for (uint32_t i = 0; i < kDeep; ++i)
            {
                if (p0 + i * kSlices < parts)
                {
                    // A piece without keys is all 0; one of NaN scores has this base too, and stays NaN.
                    const float w =
                        of[i][0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((of[i][0] - best) * scaleLog2);
                    den = fmaf(w, of[i][1], den);
                    num += w * x[i];
                }
            }
        }
    }
    sliceNum[at][lane] = num;
    if (lane == 0)
    {
        sliceHead[at] = float4v{base, den, scaleLog2, 0.0f};
    }
    __syncthreads();
    if (is && slice == kSlices - 1)
    {
        const uint32_t slice0 = at - (kSlices - 1);
        scaleLog2 = sliceHead[slice0][2];  // slice 0 has a part
        float best = -INFINITY;
#pragma unroll
        for (uint32_t s = 0; s < kSlices; ++s)
        {
            best = fmaxf(best, sliceHead[slice0 + s][0]);
        }
        num = float4v{};
        den = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kSlices; ++s)
        {
            const float b = sliceHead[slice0 + s][0];
            const float w = b == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((b - best) * scaleLog2);
            den = fmaf(w, sliceHead[slice0 + s][1], den);
            num += w * sliceNum[slice0 + s][lane];
        }
        *reinterpret_cast<float4v*>(out) = den == 0.0f ? float4v{} : num / den;
    }
}

/// Chunks of the prefix: workgroups for one on each of 256 CUs, beside one of own keys; two where that would be few
/// chunks, so that rounding their number down leaves many CUs without. 28 / 4 heads of 128: 64 queries, 8190 keys in 16
/// chunks 40.1 us, in 32 44.5; 16 queries, 16000 keys in 64 chunks 29.7 us, in 128 36.6; 250 queries, 16381 keys in 9
/// chunks 157 us, in 4 182. (A number of workgroups of the same rows that is a multiple of eight, which keeps those of
/// the same keys on one XCD, gained nothing: the last in 8 chunks 5 us slower, when it took 187.)
uint32_t PrefixChunks(uint32_t queries, uint32_t heads, uint32_t kvHeads)
{
    const uint32_t blocks = kvHeads * CeilDiv(static_cast<uint64_t>(queries) * (heads / kvHeads), kRowsOfBlock);
    const uint32_t chunks = kTurn / blocks;
    return std::max(1u, std::min(kMaxChunks, chunks < kFewChunks ? 2 * kTurn / blocks : chunks));
}

size_t CutBytes(uint32_t queries, uint32_t kvHeads) { return sizeof(uint4) * static_cast<size_t>(queries) * kvHeads; }

size_t WholeBytes(uint32_t queries, uint32_t heads, uint32_t headDim)
{
    return sizeof(float) * static_cast<size_t>(queries) * heads * (headDim + 4);
}

template <int kHd>
hipError_t LaunchPrefix(hipStream_t s, const PagedPrefixArgs& a, const PagedAttentionF16Args& own)
{
    const uint32_t rowBlocks = CeilDiv(static_cast<uint64_t>(a.queries) * a.group, kRowsOfBlock);
    const uint32_t prefixBlocks = a.kvHeads * a.chunks * rowBlocks;
    auto grid = [](uint32_t blocks) {  // a dimension's threads are below 2^32
        constexpr uint32_t kMost = 1u << 23;
        return dim3(std::min(blocks, kMost), CeilDiv(blocks, kMost));
    };
    if (a.cuts != nullptr)
    {
        if (a.queries > kScanQueries)
        {
            hipLaunchKernelGGL(PagedCostSumsKernel<kTile>, dim3(1), dim3(1024), 0, s, own);
        }
        hipLaunchKernelGGL((PagedPrefixKernel<kHd, true>), grid(prefixBlocks + kSplitBlocks), dim3(kBlock), 0, s, a,
                           own, prefixBlocks, kSplitBlocks);
    }
    else
    {
        const uint32_t ownBlocks = a.queries * a.kvHeads;
        hipLaunchKernelGGL((PagedPrefixKernel<kHd, false>), grid(prefixBlocks + ownBlocks), dim3(kBlock), 0, s, a, own,
                           prefixBlocks, ownBlocks);
    }
    const uint64_t items = static_cast<uint64_t>(a.queries) * a.kvHeads * a.group;
    // 256 threads have 32 parts of 128 channels on their way, 64 have 8: 16 queries of 28 heads with 64 chunks take
    // 29.7 us in all with 256 and 37.5 with 64, 64 queries with 16 chunks 40.0 and 41.2, 250 with 9 164 and 157.
    if (a.chunks >= 16)
    {
        hipLaunchKernelGGL((PagedPrefixJoinKernel<kHd, 256>), dim3(static_cast<uint32_t>(items)), dim3(256), 0, s, a);
    }
    else
    {
        hipLaunchKernelGGL((PagedPrefixJoinKernel<kHd, 64>), dim3(CeilDiv(items, 4)), dim3(256), 0, s, a);
    }
    return hipGetLastError();
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_paged_attention_prefix_f16kv_workspace_bytes(uint32_t queries, uint32_t heads,
                                                                    uint32_t kv_heads, uint32_t head_dim)
{
    if (!AttentionShape(queries, heads, kv_heads, head_dim))
    {
        return 0;
    }
    return DecodeWorkspaceBytes(queries, heads, kv_heads, head_dim) + WholeBytes(queries, heads, head_dim) +
           CutBytes(queries, kv_heads) +
           sizeof(float) * static_cast<size_t>(queries) * heads * PrefixChunks(queries, heads, kv_heads) *
               (head_dim + 4);
}

extern "C" int muyo_paged_attention_prefix_f16kv(const float* q, const void* kcache, const void* vcache, float* out,
                                                 const int32_t* tables, uint32_t sequences, uint32_t table_pages,
                                                 const int32_t* query_sequence, const int32_t* positions,
                                                 uint32_t queries, const int32_t* prefix, uint32_t heads,
                                                 uint32_t kv_heads, uint32_t head_dim, uint32_t pages,
                                                 uint32_t page_size, float scale, void* workspace,
                                                 uint64_t workspace_bytes, void* stream)
{
    const char* name = "paged_attention_prefix_f16kv";
    const uint64_t cacheBytes = 2ull * pages * page_size * kv_heads * head_dim;
    const Range more[] = {{kcache, cacheBytes, "kcache"}, {vcache, cacheBytes, "vcache"}, {prefix, 8, "prefix"}};
    const AttentionCall call{q, out, tables, sequences, table_pages, query_sequence, positions, queries, heads,
                             kv_heads, head_dim, pages, page_size, scale, workspace, workspace_bytes,
                             muyo_paged_attention_prefix_f16kv_workspace_bytes(queries, heads, kv_heads, head_dim)};
    const int checked = CheckAttention(name, call, more, 3, 2);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    PagedAttentionF16Args own{};
    FillAttentionArgs(own, call, 0);
    own.kcache = static_cast<const uint16_t*>(kcache);
    own.vcache = static_cast<const uint16_t*>(vcache);
    char* const behind = static_cast<char*>(workspace) + DecodeWorkspaceBytes(queries, heads, kv_heads, head_dim);
    own.wholes = reinterpret_cast<float*>(behind);
    own.cutsByUnit = 1;
    own.cuts = reinterpret_cast<uint4*>(behind + WholeBytes(queries, heads, head_dim));
    const PagedPrefixArgs a{q, own.kcache, own.vcache, out, tables, sequences, table_pages, query_sequence, queries,
                            heads / kv_heads, kv_heads, prefix, pages, own.pageShift, scale,
                            PrefixChunks(queries, heads, kv_heads), own.wholes,
                            SplitKeys<kTile>(own) ? own.cuts : nullptr, own.partials,
                            reinterpret_cast<float*>(behind + WholeBytes(queries, heads, head_dim) +
                                                     CutBytes(queries, kv_heads))};
    const hipError_t launched =
        head_dim == 64 ? LaunchPrefix<64>(AsStream(stream), a, own) : LaunchPrefix<128>(AsStream(stream), a, own);
    return launched == hipSuccess ? MUYO_OK : HipStatus(launched, name);
}
