// Log probabilities of given tokens, their ranks, the entropy and the most likely tokens of rows of
// logits.
//
// With m the row's largest logit, s = sum e^(x - m) and t = sum e^(x - m) (x - m): a token's log
// probability is x - m - log s and the row's entropy log s - t / s. Parts of a row join exactly: over a
// larger maximum m' = m - d, s becomes s e^d and t becomes (t + d s) e^d (d <= 0).
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace muyo
{
namespace
{
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kQuads = 8;                           // 16-byte loads of a lane's batch
constexpr uint32_t kBatch = kWave * 4 * kQuads;     // logits a wave takes at a time
constexpr uint32_t kMaxTop = 64;                    // a lane of a wave each
constexpr uint32_t kMaxParts = 64;                  // workgroups of a row
constexpr uint32_t kTargetBlocks = 2048;            // workgroups wanted of a call: eight for each of 256 CUs
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobArgs
{
    const float* logits;
    uint64_t stride;
    uint32_t rows, vocab;
    const int32_t* tokens;
    float* logprobs;
    int32_t* ranks;
    float* entropy;
    uint32_t top;
    int32_t* topIds;
    float* topLogprobs;
    uint32_t parts;   // workgroups of a row
    float4* sums;     // [rows][parts]: m, s, t, tokens before the given one (bits)
    uint64_t* keys;   // [rows][parts][top]
};

/// The order's upper word: rises with the value. -0 counts as +0, NaN comes before -inf.
__device__ __forceinline__ uint32_t OrderBits(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t ordered = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return v != v ? 0u : ordered;
}

/// A 64-bit key whose descending order is (value descending, index ascending). 0 is below every key.
__device__ __forceinline__ uint64_t OrderKey(float v, uint32_t index)
{
    return (static_cast<uint64_t>(OrderBits(v)) << 32) | static_cast<uint64_t>(~index);
}

__device__ __forceinline__ float KeyValue(uint64_t key)
{
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);  // 0 is a NaN
}

/// `key` of lane `lane` (the same in every lane), in every lane.
__device__ __forceinline__ uint64_t KeyOfLane(uint64_t key, uint32_t lane)
{
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(key), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(key >> 32), lane);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ uint32_t CountLanes(bool is) { return static_cast<uint32_t>(__popcll(__ballot(is))); }

/// The sums of a lane, a wave, a workgroup or a row.
struct Sums
{
    float m, s, t;
    uint32_t above;
};

/// `x` over the maximum `m` (at least its own).
__device__ __forceinline__ void Rebase(Sums& x, float m)
{
    // Differences of the type's lowest value or of -inf: their weight is 0, and 0 times them shall be 0. (NaN
    // stays in s.)
    const float d = x.m == m ? 0.0f : fmaxf(x.m - m, -1e4f);
    const float f = exp2f(d * kLog2e);
    x.t = (x.t + d * x.s) * f;
    x.s *= f;
    x.m = m;
}

/// One row's answers from its sums and the keys of its first `top` tokens. By the calling threads,
/// `thread` of `threads`.
__device__ __forceinline__ void WriteRow(const LogprobArgs& a, uint32_t row, const Sums& x, const uint64_t* best,
                                         uint32_t thread, uint32_t threads)
{
    const bool empty = x.s == 0.0f;  // no logit above -inf
    const float logSum = empty ? 0.0f : logf(x.s);
    for (uint32_t k = thread; k < a.top; k += threads)
    {
        const uint64_t at = static_cast<uint64_t>(row) * a.top + k;
        a.topIds[at] = static_cast<int32_t>(~static_cast<uint32_t>(best[k]));
        a.topLogprobs[at] = empty ? -INFINITY : KeyValue(best[k]) - x.m - logSum;
    }
    if (thread == 0)
    {
        const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
        const bool given = token >= 0 && static_cast<uint32_t>(token) < a.vocab;
        if (a.logprobs != nullptr)
        {
            a.logprobs[row] =
                !given || empty ? -INFINITY : a.logits[row * a.stride + static_cast<uint32_t>(token)] - x.m - logSum;
        }
        if (a.ranks != nullptr)
        {
            a.ranks[row] = given ? static_cast<int32_t>(x.above) : -1;
        }
        if (a.entropy != nullptr)
        {
            a.entropy[row] = empty ? 0.0f : logSum - x.t / x.s;
        }
    }
}

/// The `top` largest of keys[0..count) (different ones, in LDS), into best[0..top) in falling order: a
/// key's place is the number of keys above it.
__device__ __forceinline__ void RankKeys(const uint64_t* keys, uint32_t count, uint32_t top, uint64_t* best)
{
    for (uint32_t i = threadIdx.x; i < count; i += blockDim.x)
    {
        const uint64_t key = keys[i];
        uint32_t place = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < count; ++j)
        {
            place += keys[j] > key ? 1u : 0u;
        }
        if (place < top)
        {
            best[place] = key;
        }
    }
}

/// One pass over the row: a wave takes batches of 2048 logits into registers, the next one on its way
/// meanwhile, and each lane keeps the sums of its own.
///
/// The first `top` tokens: the wave's best so far lie in order across its lanes (lane i has the i-th), and
/// a batch is looked through only if some lane's largest logit reaches the last of them. Then a lower bound
/// of the batch's own `top`-th is found first, by bisection: a value that the largest ones of `top` lanes
/// reach. What reaches both bounds, a few more than `top` in the first batch and hardly any later, is
/// inserted one by one. Equal logits are told apart by their index in the key, so nothing overflows.
///
/// The rank is counted on the way: the tokens before a given one have a larger logit, or the same at
/// a lower index, which is a different comparison on each side of its batch.
template <bool kOnce>
__global__ __launch_bounds__(kBlock, 3) void TokenLogprobsKernel(LogprobArgs a)
{
    __shared__ Sums waveSums[kWaves];
    __shared__ uint64_t waveKeys[kWaves * kMaxTop];
    __shared__ uint64_t best[kMaxTop];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t row = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x - row * a.parts;
    const float* x = a.logits + row * a.stride;
    // Loads are 16-byte aligned: the row begins `lead` values into the first.
    const uint32_t lead = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) / 4 % 4);
    const uint64_t span = static_cast<uint64_t>(lead) + a.vocab;
    const uint32_t batches = static_cast<uint32_t>((span + kBatch - 1) / kBatch);
    const uint32_t stride = a.parts * kWaves;

    // A batch's logits, and a bit for each that is the row's (the others are -inf).
    float4v next[kQuads];
    uint32_t nextThere = ~0u;
    auto request = [&](uint32_t batch) {
        const uint64_t first = static_cast<uint64_t>(batch) * kBatch;
        nextThere = ~0u;
        if (first >= lead && first + kBatch <= span)
        {
            const float4v* from = reinterpret_cast<const float4v*>(x - lead + first) + lane;
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
                next[j] = kOnce ? __builtin_nontemporal_load(from + j * kWave) : from[j * kWave];
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                const uint64_t at = first + 4 * (j * kWave + lane) + c;
                const bool there = at >= lead && at < span;
                next[j][c] = there ? x[at - lead] : -INFINITY;
                nextThere = there ? nextThere : nextThere & ~(1u << (4 * j + c));
            }
        }
    };

    uint32_t batch = part * kWaves + wave;
    if (batch < batches)
    {
        request(batch);
    }
    const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
    const bool given = token >= 0 && static_cast<uint32_t>(token) < a.vocab;
    const float own = given ? x[token] : INFINITY;
    const uint64_t ownKey = given ? OrderKey(own, static_cast<uint32_t>(token)) : ~0ull;
    const bool plain = own > -INFINITY;  // not -inf, not NaN
    const float below = nextafterf(own, -INFINITY);

    Sums sums{-INFINITY, 0.0f, 0.0f, 0};
    uint64_t mine = 0;       // lane i: the i-th best so far
    uint64_t least = 0;      // the last of the first `top`
    for (; batch < batches; batch += stride)
    {
        float4v v[kQuads];
        const uint32_t there = nextThere;
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
            v[j] = next[j];
        }
        if (batch + stride < batches)
        {
            request(batch + stride);
        }

        float largest = -INFINITY;
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
            largest = fmaxf(largest, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
        }
        if (largest > sums.m)
        {
            Rebase(sums, largest);
        }
        const float base = sums.m == -INFINITY ? 0.0f : sums.m;
        float s[4] = {}, t[4] = {};
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                const float d = v[j][c] - base;
                const float e = __builtin_amdgcn_exp2f(d * kLog2e);
                s[c] += e;
                t[c] = fmaf(e, fmaxf(d, -1e4f), t[c]);  // 0 times -inf would be NaN
            }
        }
        sums.s += (s[0] + s[1]) + (s[2] + s[3]);
        sums.t += (t[0] + t[1]) + (t[2] + t[3]);

        // Index of v[j][c]: at0 + 256 j + c.
        const uint32_t at0 = static_cast<uint32_t>(static_cast<uint64_t>(batch) * kBatch - lead) + 4 * lane;
        if (given)
        {
            const bool after = static_cast<int64_t>(batch) * kBatch - lead > token;
            const bool before = static_cast<int64_t>(batch) * kBatch - lead + kBatch <= token;
            if (plain && (after || before))
            {
                const float over = after ? own : below;
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        sums.above += v[j][c] > over ? 1u : 0u;
                    }
                }
            }
            else
            {
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        const bool is = (there >> (4 * j + c) & 1u) != 0;
                        sums.above += is && OrderKey(v[j][c], at0 + 256 * j + c) > ownKey ? 1u : 0u;
                    }
                }
            }
        }

        if (a.top > 0)
        {
            uint32_t high = OrderBits(largest);
            if (__any(there != ~0u || sums.s != sums.s))
            {
                // Of a lane with NaN, or without logits: not that of the -inf that `largest` begins with.
                high = 0;
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        high = (there >> (4 * j + c) & 1u) != 0 ? max(high, OrderBits(v[j][c])) : high;
                    }
                }
            }
            uint32_t floor = static_cast<uint32_t>(least >> 32);
            const uint32_t reach = CountLanes(high >= floor);
            if (reach != 0)
            {
                if (reach >= a.top)
                {
                    uint32_t bound = 0;
#pragma unroll 1
                    for (uint32_t bit = 1u << 31; bit > 1u << 11; bit >>= 1)
                    {
                        bound = CountLanes(high >= (bound | bit)) >= a.top ? bound | bit : bound;
                    }
                    floor = max(floor, bound);
                }
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        const uint32_t bits = OrderBits(v[j][c]);
                        const bool is = bits >= floor && (there >> (4 * j + c) & 1u) != 0;
                        const uint64_t key = (static_cast<uint64_t>(bits) << 32) | ~(at0 + 256 * j + c);
                        uint64_t mask = __ballot(is && key > least);
                        while (mask != 0)
                        {
                            const uint32_t from = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(mask)) - 1);
                            const uint64_t one = KeyOfLane(key, from);
                            const uint32_t place = CountLanes(mine > one);
                            const uint64_t left = __shfl_up(static_cast<unsigned long long>(mine), 1);
                            mine = lane < place ? mine : lane == place ? one : left;
                            least = KeyOfLane(mine, a.top - 1);
                            mask &= mask - 1;
                            mask &= __ballot(key > least);
                        }
                    }
                }
            }
        }
    }

    // Lanes, then waves.
    const float top = GroupMax<kWave>(sums.m);
    Rebase(sums, top);
    sums.s = GroupSum<kWave>(sums.s);
    sums.t = GroupSum<kWave>(sums.t);
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        sums.above += __shfl_xor(sums.above, step);
    }
    if (lane == 0)
    {
        waveSums[wave] = sums;
    }
    if (lane < a.top)
    {
        waveKeys[wave * a.top + lane] = mine;
    }
    if (wave == 0)
    {
        best[lane] = 0;  // a part may have fewer tokens
    }
    __syncthreads();
    float most = waveSums[0].m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
    {
        most = fmaxf(most, waveSums[w].m);
    }
    Sums all{most, 0.0f, 0.0f, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
    {
        Sums one = waveSums[w];
        Rebase(one, most);
        all.s += one.s;
        all.t += one.t;
        all.above += one.above;
    }
    RankKeys(waveKeys, kWaves * a.top, a.top, best);
    __syncthreads();
    if (a.parts == 1)
    {
        WriteRow(a, row, all, best, threadIdx.x, kBlock);
        return;
    }
    if (threadIdx.x == 0)
    {
        a.sums[blockIdx.x] = make_float4(all.m, all.s, all.t, __uint_as_float(all.above));
    }
    for (uint32_t k = threadIdx.x; k < a.top; k += kBlock)
    {
        a.keys[static_cast<uint64_t>(blockIdx.x) * a.top + k] = best[k];
    }
}

/// Joins a row's parts: a workgroup a row. The last of a part's keys is a lower bound of the row's
/// last, so only keys that reach the largest of those are ranked.
__global__ __launch_bounds__(kBlock) void TokenLogprobsJoinKernel(LogprobArgs a)
{
    __shared__ uint64_t held[kMaxParts * kMaxTop];
    __shared__ uint64_t best[kMaxTop];
    __shared__ uint32_t count;
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % kWave;
    const uint64_t first = static_cast<uint64_t>(row) * a.parts;
    // Lane p of every wave has part p.
    const float4 own = a.sums[first + min(lane, a.parts - 1)];
    uint64_t floor = a.top > 0 ? a.keys[(first + min(lane, a.parts - 1)) * a.top + a.top - 1] : 0;
    Sums sums{own.x, own.y, own.z, __float_as_uint(own.w)};
    if (lane >= a.parts)
    {
        sums = Sums{-INFINITY, 0.0f, 0.0f, 0};
    }
    const float most = GroupMax<kWave>(sums.m);
    Rebase(sums, most);
    sums.s = GroupSum<kWave>(sums.s);
    sums.t = GroupSum<kWave>(sums.t);
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        sums.above += __shfl_xor(sums.above, step);
        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(floor), step);
        floor = floor > other ? floor : other;
    }
    if (a.top > 0)
    {
        if (threadIdx.x == 0)
        {
            count = 0;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.parts * a.top; i += kBlock)
        {
            const uint64_t key = a.keys[first * a.top + i];
            if (key >= floor)
            {
                held[atomicAdd(&count, 1u)] = key;  // the order does not matter: keys are ranked
            }
        }
        __syncthreads();
        RankKeys(held, count, a.top, best);
        __syncthreads();
    }
    WriteRow(a, row, sums, best, threadIdx.x, kBlock);
}

/// Workgroups of a row: enough for kTargetBlocks in all, a batch for each wave at least.
uint32_t RowParts(uint32_t rows, uint32_t vocab)
{
    const uint32_t most = std::min(kMaxParts, CeilDiv(CeilDiv(static_cast<uint64_t>(vocab) + 3, kBatch), kWaves));
    return std::max(1u, std::min(most, CeilDiv(kTargetBlocks, rows)));
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_token_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top)
{
    if (rows == 0 || vocab == 0 || vocab > 0x7FFFFFFFu || top > kMaxTop || top > vocab)
    {
        return 0;
    }
    return (sizeof(float4) + 8 * static_cast<size_t>(top)) * rows * RowParts(rows, vocab) + 16;
}

extern "C" int muyo_token_logprobs_f32(const float* logits, uint64_t row_stride, uint32_t rows, uint32_t vocab,
                                       const int32_t* tokens, float* logprobs, int32_t* ranks, float* entropy,
                                       uint32_t top, int32_t* top_ids, float* top_logprobs, void* workspace,
                                       uint64_t workspace_bytes, void* stream)
{
    const char* name = "token_logprobs_f32";
    if (logits == nullptr || ((logprobs != nullptr || ranks != nullptr) && tokens == nullptr) ||
        (top > 0 && (top_ids == nullptr || top_logprobs == nullptr)))
    {
        return Fail(MUYO_E_NULL, "%s: logits are required, tokens for logprobs or ranks, top_ids and top_logprobs when "
                                 "top > 0",
                    name);
    }
    const size_t need = muyo_token_logprobs_workspace_bytes(rows, vocab, top);
    if (need == 0)
    {
        return Fail(MUYO_E_RANGE, "%s: needs rows >= 1, 1 <= vocab < 2^31, top <= %u and top <= vocab (got %u, %u, %u)",
                    name, kMaxTop, rows, vocab, top);
    }
    if (row_stride < vocab)
    {
        return Fail(MUYO_E_CONTRACT, "%s: row_stride %llu is below vocab %u", name,
                    static_cast<unsigned long long>(row_stride), vocab);
    }
    if (workspace == nullptr || !Aligned16(workspace) || workspace_bytes < need)
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a 16-byte aligned workspace of %zu bytes (got %llu)", name, need,
                    static_cast<unsigned long long>(workspace_bytes));
    }
    const uint32_t parts = RowParts(rows, vocab);
    float4* sums = static_cast<float4*>(workspace);
    LogprobArgs a{logits,  row_stride, rows,  vocab, tokens,  logprobs, ranks,
                  entropy, top,        top_ids, top_logprobs, parts, sums,
                  reinterpret_cast<uint64_t*>(sums + static_cast<size_t>(rows) * parts)};
    const uint64_t blocks = static_cast<uint64_t>(rows) * parts;
    if (blocks > 0x7FFFFFFFull)
    {
        return Fail(MUYO_E_RANGE, "%s: %u rows are too many for one launch", name, rows);
    }
    hipLaunchKernelGGL(TokenLogprobsKernel<false>, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, AsStream(stream), a);
    if (parts > 1)
    {
        hipLaunchKernelGGL(TokenLogprobsJoinKernel, dim3(rows), dim3(kBlock), 0, AsStream(stream), a);
    }
    return LaunchStatus(name);
}
