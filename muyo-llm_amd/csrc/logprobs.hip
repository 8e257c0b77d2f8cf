// Log probabilities of given tokens, their ranks, the entropy and the most likely tokens of rows of
// logits.
//
// With m the row's largest logit, y = (x - m) log2 e, s = sum 2^y and t = sum 2^y y, a token's log
// probability is (x - m) - ln s and the row's entropy ln s - ln 2 t / s. Parts of a row join exactly: over
// a larger m, with d = (m - larger) log2 e, s becomes s 2^d and t becomes (t + d s) 2^d.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace muyo
{
namespace
{
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kQuads = 4;                           // 16-byte loads of a lane's batch
constexpr uint32_t kBatch = kWave * 4 * kQuads;     // logits a wave takes at a time
constexpr int kKept = 3;                            // batches with its largest logits that a lane knows
constexpr uint32_t kTooMany = 1u << 20;             // candidates
constexpr int kFewLanes = 4;                        // looked at one by one
constexpr uint32_t kMaxTop = 64;                    // a lane of a wave each
constexpr uint32_t kMaxParts = 64;                  // workgroups of a row
constexpr int kPerCu = 5;                           // workgroups of a CU
constexpr uint32_t kBlocksAtOnce = 256 * kPerCu;    // workgroups that 256 CUs run at once
constexpr uint32_t kMaxRows = (1u << 24) - 1;       // a launch has fewer than 2^32 threads
constexpr uint64_t kOnceBytes = 256ull << 20;       // logits that no cache holds: read without caching them
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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

/// `key` of the lane before (wave_shr:1; lane 0 keeps its own).
__device__ __forceinline__ uint64_t KeyOfLaneBefore(uint64_t key)
{
    const int lo = static_cast<int>(static_cast<uint32_t>(key));
    const int hi = static_cast<int>(static_cast<uint32_t>(key >> 32));
    const uint32_t high = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(hi, hi, 0x138, 0xF, 0xF, false));
    const uint32_t low = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(lo, lo, 0x138, 0xF, 0xF, false));
    return (static_cast<uint64_t>(high) << 32) | low;
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
    // Differences to the type's lowest value overflow: the weight is 0, and 0 times them shall be 0. (A
    // part without logits above -inf has sums of 0, and NaN stays in s.)
    const float d = x.m == m || x.m == -INFINITY ? 0.0f : fmaxf((x.m - m) * kLog2e, -1e4f);
    const float f = exp2f(d);
    x.t = (x.t + d * x.s) * f;
    x.s *= f;
    x.m = m;
}

/// The given token of a row, and its logit.
struct Given
{
    bool is;
    uint32_t token;
    float logit;
};

__device__ __forceinline__ Given GivenOf(const LogprobArgs& a, uint32_t row)
{
    const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
    Given g;
    g.is = token >= 0 && static_cast<uint32_t>(token) < a.vocab;
    g.token = static_cast<uint32_t>(token);
    g.logit = g.is ? a.logits[row * a.stride + g.token] : INFINITY;
    return g;
}

/// One row's answers from its sums and the keys of its first `top` tokens.
__device__ __forceinline__ void WriteRow(const LogprobArgs& a, uint32_t row, const Sums& x, const Given& given,
                                         const uint64_t* best)
{
    const bool empty = x.s == 0.0f;  // no logit above -inf
    const float logSum = empty ? 0.0f : logf(x.s);
    for (uint32_t k = threadIdx.x; k < a.top; k += kBlock)
    {
        const uint64_t at = static_cast<uint64_t>(row) * a.top + k;
        a.topIds[at] = static_cast<int32_t>(~static_cast<uint32_t>(best[k]));
        a.topLogprobs[at] = empty ? -INFINITY : KeyValue(best[k]) - x.m - logSum;
    }
    if (threadIdx.x == 0)
    {
        if (a.logprobs != nullptr)
        {
            a.logprobs[row] = !given.is || empty ? -INFINITY : given.logit - x.m - logSum;
        }
        if (a.ranks != nullptr)
        {
            a.ranks[row] = given.is ? static_cast<int32_t>(x.above) : -1;
        }
        if (a.entropy != nullptr)
        {
            a.entropy[row] = empty ? 0.0f : logSum - kLn2 * (x.t / x.s);
        }
    }
}

/// The `top` largest of keys[0..count) (different ones, in LDS), into best[0..top) in falling order: a
/// key's place is the number of keys above it. Up to 256 keys are counted against by four threads each (64
/// keys), two or one; `places` has room for 256.
__device__ __forceinline__ void RankKeys(const uint64_t* keys, uint32_t count, uint32_t top, uint64_t* best,
                                         uint32_t* places)
{
    if (count <= kBlock)
    {
        const uint32_t span = count <= 64 ? 64 : count <= 128 ? 128 : 256;
        const uint32_t i = threadIdx.x & (span - 1);
        places[threadIdx.x] = 0;
        __syncthreads();
        const uint64_t key = i < count ? keys[i] : 0;
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = threadIdx.x / span; j < count; j += kBlock / span)
        {
            above += keys[j] > key ? 1u : 0u;
        }
        if (i < count)
        {
            atomicAdd(places + i, above);
        }
        __syncthreads();
        if (threadIdx.x < count && places[threadIdx.x] < top)
        {
            best[places[threadIdx.x]] = key;
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < count; i += kBlock)
    {
        const uint64_t key = keys[i];
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < count; ++j)
        {
            above += keys[j] > key ? 1u : 0u;
        }
        if (above < top)
        {
            best[above] = key;
        }
    }
}

/// A value that `high` reaches in lanes that count for `top` together, `each` apiece (0: fewer do): the
/// largest one of 16 bits.
__device__ __forceinline__ uint32_t LowerBound(uint32_t high, uint32_t each, uint32_t top)
{
    uint32_t bound = 0;
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit > 1u << 15; bit >>= 1)
    {
        bound = CountLanes(high >= (bound | bit)) * each >= top ? bound | bit : bound;
    }
    return bound;
}

/// The row's values begin `lead` values into a 16-byte load, and end at `span`.
struct RowSpan
{
    const float* x;
    uint32_t lead, span;
};

__device__ __forceinline__ RowSpan SpanOf(const LogprobArgs& a, uint32_t row)
{
    RowSpan s;
    s.x = a.logits + row * a.stride;
    s.lead = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s.x) / 4 % 4);
    s.span = s.lead + a.vocab;
    return s;
}

/// The lane's kQuads * 4 values of a batch, with a bit of `there` for each that is the row's.
template <bool kOnce>
__device__ __forceinline__ void LoadBatch(const RowSpan& s, uint32_t batch, uint32_t lane, float4v (&v)[kQuads],
                                          uint32_t& there)
{
    there = ~0u;
    const uint32_t first = batch * kBatch;
    if (first >= s.lead && first + kBatch <= s.span)
    {
        const float4v* from = reinterpret_cast<const float4v*>(s.x - s.lead + first) + lane;
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
            v[j] = kOnce ? __builtin_nontemporal_load(from + j * kWave) : from[j * kWave];
        }
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < kQuads; ++j)
    {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c)
        {
            const uint32_t at = first + 4 * (j * kWave + lane) + c;
            const bool is = at >= s.lead && at < s.span;
            v[j][c] = is ? s.x[at - s.lead] : -INFINITY;
            there = is ? there : there & ~(1u << (4 * j + c));
        }
    }
}

/// What a workgroup needs to find the first tokens of its part.
struct TopSpace
{
    __attribute__((aligned(16))) uint32_t places[kBlock];
    uint32_t bound;
    uint32_t found;
    uint32_t waveHeld[kWaves];
    uint64_t keys[kWaves * kWave];
    uint64_t best[kMaxTop];
    float4v staged[kWaves][kQuads][kWave];
    uint64_t candidates[kWaves][kWave];
};

/// A lane's batches with its largest logits: the largest of each, in falling order, and which of the wave's
/// batches it is. Of the others only the largest logit is kept.
struct LaneBatches
{
    float most[kKept + 1];
    uint32_t nth[kKept];

    __device__ __forceinline__ void Clear()
    {
#pragma unroll
        for (int i = 0; i < kKept; ++i)
        {
            most[i] = -INFINITY;
            nth[i] = 0;
        }
        most[kKept] = -INFINITY;
    }

    __device__ __forceinline__ void Add(float largest, uint32_t which)
    {
        if (!__any(largest > most[kKept - 1]))
        {
            most[kKept] = fmaxf(most[kKept], largest);
            return;
        }
        most[kKept] = largest > most[kKept - 1] ? most[kKept - 1] : fmaxf(most[kKept], largest);
#pragma unroll
        for (int i = kKept - 1; i > 0; --i)
        {
            const bool here = largest > most[i];
            const bool before = largest > most[i - 1];
            most[i] = before ? most[i - 1] : here ? largest : most[i];
            nth[i] = before ? nth[i - 1] : here ? which : nth[i];
        }
        const bool first = largest > most[0];
        most[0] = first ? largest : most[0];
        nth[0] = first ? which : nth[0];
    }

    __device__ __forceinline__ void Drop()
    {
#pragma unroll
        for (int i = 0; i + 1 < kKept; ++i)
        {
            most[i] = most[i + 1];
            nth[i] = nth[i + 1];
        }
        most[kKept - 1] = -INFINITY;
    }
};

/// The first a.top tokens of a part, for any number of logits that reach `floor`: wave by wave, batch by
/// batch (from the wave's first, `stride` apart).
///
/// A wave's best so far lie in order across its lanes (lane i has the i-th). Few lanes of a batch reach the
/// last of them: their logits are looked at lane by lane and inserted one by one. Otherwise a lower bound
/// of the batch's own `top`-th is found first, by bisection: a value that the largest ones of `top` lanes
/// reach. The candidates (a few more than `top`) are gathered, with the best so far, and ranked: a candidate's
/// place is the number of those above it. More than 64 are inserted too. Equal logits are told apart by
/// their index in the key, so nothing overflows. The batch goes through LDS: the registers are free for
/// the next one at once, and loops over its logits need not be unrolled. Batches that no lane knows to
/// reach the last are left out: of a row with few logits above -inf, or of equal ones, most (a call on 300 rows with
/// ten above -inf and 20 alternatives: 66 us, 202 through all batches, where one on ordinary rows takes 49).
__device__ __forceinline__ void TopByWaves(const LogprobArgs& a, const RowSpan& s, uint32_t firstBatch,
                                           uint32_t batches, uint32_t stride, uint32_t floorBits,
                                           const LaneBatches& own, TopSpace& space)
{
    const uint64_t floorKey = static_cast<uint64_t>(floorBits) << 32;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    float4v v[kQuads];
    uint32_t there = 0;
    uint64_t mine = 0;          // lane i: the i-th best so far
    uint64_t least = floorKey;  // the last of the first `top`, or what they reach
    auto lastOf = [&]() {
        const uint64_t last = KeyOfLane(mine, a.top - 1);
        return last > floorKey ? last : floorKey;
    };
    // What counts in a batch: the last's value too while it is a bound, and more than the last's once that is one of
    // the wave's own, as the batches rise in index.
    auto floorOf = [&]() { return static_cast<uint32_t>(least >> 32) + (static_cast<uint32_t>(least) != 0 ? 1u : 0u); };
    uint32_t most[kKept + 1];
#pragma unroll
    for (int i = 0; i <= kKept; ++i)
    {
        most[i] = OrderBits(own.most[i]);
    }
    const uint32_t count = firstBatch < batches ? (batches - 1 - firstBatch) / stride + 1 : 0;
    auto after = [&](uint32_t nth) {
        const uint32_t floor = floorOf();
        while (++nth < count)
        {
            bool reaches = most[kKept] >= floor;
#pragma unroll
            for (int i = 0; i < kKept; ++i)
            {
                reaches = reaches || (own.nth[i] == nth && most[i] >= floor);
            }
            if (__any(reaches))
            {
                break;
            }
        }
        return nth;
    };
    if (count != 0)
    {
        LoadBatch<false>(s, firstBatch, lane, v, there);
    }
    uint32_t following;
    for (uint32_t nth = 0; nth < count; nth = following)
    {
        const uint32_t batch = firstBatch + nth * stride;
        const uint32_t at0 = batch * kBatch - s.lead;  // index of v[j][c]: at0 + 256 j + 4 lane + c
        const uint32_t is = there;
        uint32_t high = 0;
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
        {
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                high = max(high, (is >> (4 * j + c) & 1u) != 0 ? OrderBits(v[j][c]) : 0u);
            }
        }
        uint32_t floor = floorOf();
        const bool any = is != 0;
        if (CountLanes(any && high >= floor) >= a.top)
        {
            floor = max(floor, LowerBound(high, 1, a.top));
        }
        uint64_t lanes = __ballot(any && high >= floor);
        if (lanes != 0)
        {
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
                space.staged[wave][j][lane] = v[j];
            }
        }
        following = after(nth);
        if (following < count)
        {
            LoadBatch<false>(s, firstBatch + following * stride, lane, v, there);
        }
        if (lanes == 0)
        {
            continue;
        }
        // The wave's LDS operations complete in order; the fences keep the compiler's order too.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        uint32_t found = kWave + 1;
        if (__popcll(lanes) > kFewLanes)
        {
            uint32_t take = 0;  // a bit for each of the lane's candidates
#pragma unroll 1
            for (int j = 0; j < kQuads; ++j)
            {
                const float4v x4 = space.staged[wave][j][lane];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    take |= OrderBits(x4[c]) >= floor ? 1u << (4 * j + c) : 0u;
                }
            }
            take &= is;
            found = 0;
            for (uint64_t mask = __ballot(take != 0); mask != 0; mask = __ballot(take != 0))
            {
                const uint32_t place =
                    found + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
                if (take != 0 && place < kWave)
                {
                    const uint32_t e = static_cast<uint32_t>(__ffs(static_cast<int>(take)) - 1);
                    space.candidates[wave][place] = OrderKey(space.staged[wave][e / 4][lane][e % 4],
                                                             at0 + 256 * (e / 4) + 4 * lane + e % 4);
                }
                take &= take - 1;
                found += static_cast<uint32_t>(__popcll(mask));
            }
            const uint32_t kept = min(CountLanes(mine != 0), a.top);
            if (found + kept <= kWave && lane < kept)
            {
                space.candidates[wave][found + lane] = mine;
            }
            found += kept;
        }
        if (found <= kWave)
        {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const uint64_t key = lane < found ? space.candidates[wave][lane] : 0;
            mine = key;
            if (following >= count)
            {
                continue;  // the workgroup ranks them
            }
            uint32_t place = 0;
#pragma unroll 4
            for (uint32_t i = 0; i < found; ++i)
            {
                place += KeyOfLane(key, i) > key ? 1u : 0u;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (lane < found)
            {
                space.candidates[wave][place] = key;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            mine = lane < found ? space.candidates[wave][lane] : 0;
            least = lastOf();
        }
        else
        {
            // Lane l looks at the l-th of their values. `best` is above any of its own's keys.
            const uint32_t index = at0 + 4 * lane;
            const uint64_t best =
                (static_cast<uint64_t>(high) << 32) | ~(static_cast<int32_t>(index) < 0 ? 0u : index);
            while (lanes != 0)
            {
                const uint32_t from = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(lanes)) - 1);
                lanes &= lanes - 1;
                const uint32_t j = lane / 4 % kQuads;
                const float value = space.staged[wave][j][from][lane % 4];
                const uint32_t theirs = __builtin_amdgcn_readlane(is, from);
                const uint64_t key = OrderKey(value, at0 + 256 * j + 4 * from + lane % 4);
                const bool take = lane < 4 * kQuads && (theirs >> lane & 1u) != 0 &&
                                  static_cast<uint32_t>(key >> 32) >= floor;
                uint64_t mask = __ballot(take && key > least);
                while (mask != 0)
                {
                    const uint64_t one =
                        KeyOfLane(key, static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(mask)) - 1));
                    const uint32_t place = CountLanes(mine > one);
                    const uint64_t left = KeyOfLaneBefore(mine);
                    mine = lane < place ? mine : lane == place ? one : left;
                    least = lastOf();
                    mask &= mask - 1;
                    mask &= __ballot(key > least);
                }
                lanes &= __ballot(best > least);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    const uint32_t held = CountLanes(mine != 0);
    if (lane == 0)
    {
        space.waveHeld[wave] = held;
    }
    __syncthreads();
    uint32_t keys = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w)
    {
        if (w == wave && lane < held)
        {
            space.keys[keys + lane] = mine;  // none of them is 0, and they come first
        }
        keys += space.waveHeld[w];
    }
    __syncthreads();
    RankKeys(space.keys, keys, a.top, space.best, space.places);
    __syncthreads();
}

/// The first a.top tokens of a workgroup's part into space.best, in order (0 behind the last).
///
/// The a.top-th of the 256 threads' largest logits is a lower bound of the part's a.top-th. Threads look again
/// at those of their batches that reach it, mostly one of a few threads (the last one is in v still), and what
/// reaches it, a few more than a.top logits, is gathered and ranked. Where that does not do (a thread has more
/// such batches than it knows, or there are more than 256 such logits, or fewer threads than a.top have any)
/// the waves go through the part once more.
__device__ __forceinline__ void TopOfPart(const LogprobArgs& a, const RowSpan& s, uint32_t firstBatch, uint32_t batches,
                                          uint32_t stride, float4v (&v)[kQuads], uint32_t there, const LaneBatches& own,
                                          TopSpace& space)
{
    const uint32_t lane = threadIdx.x % kWave;
    space.places[threadIdx.x] = own.most[0] > -INFINITY ? OrderBits(own.most[0]) : 0;  // -inf: NaN, or none
    if (threadIdx.x < kMaxTop)
    {
        space.best[threadIdx.x] = 0;
    }
    __syncthreads();
    if (threadIdx.x < kWave)
    {
        // Four threads' a lane. The bound's upper 16 bits are enough. (In every wave at once it would keep the
        // scalar unit, which a CU's waves share, busy for 2 us.)
        const uint4 four = *reinterpret_cast<const uint4*>(space.places + 4 * lane);
        uint32_t bound = 0;
#pragma unroll 1
        for (uint32_t bit = 1u << 31; bit > 1u << 15; bit >>= 1)
        {
            const uint32_t next = bound | bit;
            const uint32_t reach = CountLanes(four.x >= next) + CountLanes(four.y >= next) +
                                   CountLanes(four.z >= next) + CountLanes(four.w >= next);
            bound = reach >= a.top ? next : bound;
        }
        if (lane == 0)
        {
            space.bound = bound;
            space.found = 0;
        }
    }
    __syncthreads();
    const uint32_t floor = __builtin_amdgcn_readfirstlane(space.bound);
    if (floor == 0 || OrderBits(own.most[kKept]) >= floor)
    {
        space.found = kTooMany;
    }
    else
    {
        uint32_t held = (batches - 1 - firstBatch) / stride;
        LaneBatches left = own;
        while (OrderBits(left.most[0]) >= floor)
        {
            const uint32_t batch = firstBatch + left.nth[0] * stride;
            if (left.nth[0] != held)
            {
                LoadBatch<false>(s, batch, lane, v, there);
            }
            held = ~0u;
            left.Drop();
            uint32_t take = there;
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    take = OrderBits(v[j][c]) >= floor ? take : take & ~(1u << (4 * j + c));
                }
            }
            take &= (1u << 4 * kQuads) - 1;
            while (take != 0)
            {
                const uint32_t e = static_cast<uint32_t>(__ffs(static_cast<int>(take)) - 1);
                take &= take - 1;
                float value = v[0][0];
#pragma unroll
                for (uint32_t i = 1; i < 4 * kQuads; ++i)
                {
                    value = e == i ? v[i / 4][i % 4] : value;
                }
                const uint32_t place = atomicAdd(&space.found, 1u);
                if (place < kBlock)
                {
                    // The order does not matter: they are ranked.
                    space.keys[place] = OrderKey(value, batch * kBatch - s.lead + 256 * (e / 4) + 4 * lane + e % 4);
                }
            }
        }
    }
    __syncthreads();
    const uint32_t found = space.found;
    __syncthreads();
    if (found <= kBlock)
    {
        RankKeys(space.keys, found, a.top, space.best, space.places);
        __syncthreads();
        return;
    }
    TopByWaves(a, s, firstBatch, batches, stride, floor, own, space);
}

/// One pass over the row: a wave takes batches of kBatch logits into registers, and each lane keeps the sums
/// of its own, and which of its batches have its largest logits: enough to find the part's first `top` tokens
/// when all of it has been read.
///
/// The rank is counted on the way: the tokens before a given one have a larger logit, or the same at
/// a lower index, which is a different comparison on each side of its batch. That batch itself goes through
/// LDS, so that the loop over its logits need not be unrolled (one wave of a row runs it, and its instructions
/// come from memory).
///
/// What bounds it: for many rows, the logits' arrival. 1000 rows of 151936, 608 MB: 96 to 100 us, 6.2 TB/s, where the
/// best streaming read here has 6.9; read without the non-temporal hint (they fit no cache) 111 us. For
/// few rows, a chain: the batches' round trips, then two barriers and a bisection to the bound, another round
/// trip and the ranking. One row with 20 alternatives takes 8.2 us and 4.3 for the join (4.5 of the first
/// without alternatives), 61 rows with 5 14.4 and 4.0 (10.1), 300 rows with 20 42 and 5 (36). Looking for
/// candidates in every batch as it comes took 7.7, 16.3 and 59 us; knowing only the largest logit of
/// each batch, and reading those that reach the bound whole, 7.4, 15.9 and 49; keeping two batches a
/// lane instead of three, and so going through more parts again, 48 for the last.
template <bool kOnce>
__global__ __launch_bounds__(kBlock, kPerCu) void TokenLogprobsKernel(LogprobArgs a)
{
    __shared__ Sums waveSums[kWaves];
    __shared__ TopSpace space;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t row = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x - row * a.parts;
    const RowSpan s = SpanOf(a, row);
    const uint32_t stride = a.parts * kWaves;

    float4v v[kQuads];
    uint32_t there = ~0u;  // a bit for each that is the row's (the others are -inf)
    const uint32_t batches = (s.span + kBatch - 1) / kBatch;
    const uint32_t firstBatch = part * kWaves + wave;
    if (firstBatch < batches)
    {
        LoadBatch<kOnce>(s, firstBatch, lane, v, there);
    }
    const Given given = GivenOf(a, row);
    const uint64_t ownKey = given.is ? OrderKey(given.logit, given.token) : ~0ull;
    const bool plain = given.logit > -INFINITY;  // not -inf, not NaN
    const float below = nextafterf(given.logit, -INFINITY);

    Sums sums{-INFINITY, 0.0f, 0.0f, 0};
    uint32_t above = 0;     // the wave's
    LaneBatches own;
    own.Clear();
    uint32_t nth = 0;
    for (uint32_t batch = firstBatch; batch < batches; batch += stride, ++nth)
    {
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
        {
            float es[4] = {}, ts[4] = {};
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    const float y = (v[j][c] - base) * kLog2e;
                    const float e = __builtin_amdgcn_exp2f(y);
                    es[c] += e;
                    ts[c] = fmaf(e, y, ts[c]);
                }
            }
            float more = (ts[0] + ts[1]) + (ts[2] + ts[3]);
            if (__any(more != more))
            {
                // 0 times the -inf of a masked logit. (NaN logits stay in s.)
                more = 0.0f;
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        const float y = (v[j][c] - base) * kLog2e;
                        more = fmaf(__builtin_amdgcn_exp2f(y), fmaxf(y, -1e4f), more);
                    }
                }
            }
            sums.s += (es[0] + es[1]) + (es[2] + es[3]);
            sums.t += more;
        }

        // Index of v[j][c]: begin + 256 j + 4 lane + c.
        const int64_t begin = static_cast<int64_t>(batch) * kBatch - s.lead;
        const bool after = begin > given.token;
        const bool before = begin + kBatch <= given.token;
        const bool single = given.is && !(plain && (after || before));
        if (given.is && !single)
        {
            const float over = after ? given.logit : below;
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    above += CountLanes(v[j][c] > over);
                }
            }
        }
        if (a.top > 0)
        {
            own.Add(largest, nth);
        }
        const uint32_t is = there;
        if (single)
        {
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
            {
                space.staged[wave][j][lane] = v[j];
            }
        }
        if (batch + stride < batches)
        {
            LoadBatch<kOnce>(s, batch + stride, lane, v, there);
        }
        if (single)
        {
            const uint32_t at = static_cast<uint32_t>(begin) + 4 * lane;
#pragma unroll 1
            for (int j = 0; j < kQuads; ++j)
            {
                const float4v x4 = space.staged[wave][j][lane];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    const bool counts = (is >> (4 * j + c) & 1u) != 0 && OrderKey(x4[c], at + 256 * j + c) > ownKey;
                    sums.above += counts ? 1u : 0u;
                }
            }
        }
    }

    // Lanes, then waves.
    Rebase(sums, GroupMax<kWave>(sums.m));
    sums.s = GroupSum<kWave>(sums.s);
    sums.t = GroupSum<kWave>(sums.t);
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        sums.above += __shfl_xor(sums.above, step);
    }
    sums.above += above;
    if (lane == 0)
    {
        waveSums[wave] = sums;
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
    if (a.top > 0)
    {
        TopOfPart(a, s, firstBatch, batches, stride, v, there, own, space);
    }
    if (a.parts == 1)
    {
        WriteRow(a, row, all, given, space.best);
        return;
    }
    if (threadIdx.x == 0)
    {
        a.sums[blockIdx.x] = make_float4(all.m, all.s, all.t, __uint_as_float(all.above));
    }
    for (uint32_t k = threadIdx.x; k < a.top; k += kBlock)
    {
        a.keys[static_cast<uint64_t>(blockIdx.x) * a.top + k] = space.best[k];
    }
}

/// Joins a row's parts: a workgroup a row. The last of a part's keys is a lower bound of the row's
/// last, so only keys that reach the largest of those are ranked.
__global__ __launch_bounds__(kBlock) void TokenLogprobsJoinKernel(LogprobArgs a)
{
    __shared__ uint64_t held[kMaxParts * kMaxTop];
    __shared__ uint64_t best[kMaxTop];
    __shared__ uint32_t places[kBlock];
    __shared__ uint32_t count;
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % kWave;
    const uint64_t first = static_cast<uint64_t>(row) * a.parts;
    const Given given = GivenOf(a, row);
    const uint32_t keys = a.parts * a.top;
    uint64_t early[2];  // most calls' keys, on their way together with the sums
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e)
    {
        const uint32_t i = e * kBlock + threadIdx.x;
        early[e] = i < keys ? a.keys[first * a.top + i] : 0;
    }
    // Lane p of every wave has part p. Its `deep`-th key counts for `deep` keys: where the lanes with one that
    // reaches a value have `top` together, that value is a lower bound too.
    const uint32_t deep = a.top > 0 ? (a.top + a.parts - 1) / a.parts : 1;
    const uint64_t part = first + min(lane, a.parts - 1);
    const uint32_t reach =
        a.top > 0 && lane < a.parts ? static_cast<uint32_t>(a.keys[part * a.top + deep - 1] >> 32) : 0;
    const float4 own = a.sums[part];
    uint64_t floor = a.top > 0 ? a.keys[part * a.top + a.top - 1] : 0;
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
        const uint64_t lower = static_cast<uint64_t>(LowerBound(reach, deep, a.top)) << 32;
        floor = floor > lower ? floor : lower;
        if (threadIdx.x == 0)
        {
            count = 0;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < keys; i += kBlock)
        {
            const uint64_t key = i < kBlock ? early[0] : i < 2 * kBlock ? early[1] : a.keys[first * a.top + i];
            if (key >= floor)
            {
                held[atomicAdd(&count, 1u)] = key;  // the order does not matter: keys are ranked
            }
        }
        __syncthreads();
        RankKeys(held, count, a.top, best, places);
        __syncthreads();
    }
    WriteRow(a, row, sums, given, best);
}

/// Workgroups of a row: the fewest estimated batches after one another, when 1280 workgroups run at once
/// (five on each of 256 CUs), each round of them costs as much as three batches besides its own, and so
/// does the join.
uint32_t RowParts(uint32_t rows, uint32_t vocab)
{
    const uint32_t batches = CeilDiv(static_cast<uint64_t>(vocab) + 3, kBatch);
    const uint32_t most = std::min(kMaxParts, CeilDiv(batches, kWaves));
    uint32_t best = 1;
    uint64_t least = ~0ull;
    for (uint32_t parts = 1; parts <= most; ++parts)
    {
        const uint64_t rounds = CeilDiv(static_cast<uint64_t>(rows) * parts, kBlocksAtOnce);
        const uint64_t after = CeilDiv(batches, static_cast<uint64_t>(parts) * kWaves);
        const uint64_t cost = rounds * (after + 3) + (parts > 1 ? 3 : 0);
        if (cost < least)
        {
            least = cost;
            best = parts;
        }
    }
    return best;
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_token_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top)
{
    if (rows == 0 || rows > kMaxRows || vocab == 0 || vocab > 0x7FFFFFFFu || top > kMaxTop || top > vocab)
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
        return Fail(MUYO_E_RANGE, "%s: needs 1..%u rows, 1 <= vocab < 2^31, top <= %u and top <= vocab (got %u, "
                                  "%u, %u)",
                    name, kMaxRows, kMaxTop, rows, vocab, top);
    }
    if (row_stride < vocab || (reinterpret_cast<uintptr_t>(logits) & 3u) != 0)
    {
        return Fail(MUYO_E_CONTRACT, "%s: row_stride %llu is below vocab %u, or logits are not 4-byte aligned", name,
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
    if (blocks > kMaxRows)
    {
        return Fail(MUYO_E_RANGE, "%s: %u rows of %u are too many for one call", name, rows, vocab);
    }
    const Range ranges[] = {{logprobs, 4ull * rows, "logprobs"},
                            {ranks, 4ull * rows, "ranks"},
                            {entropy, 4ull * rows, "entropy"},
                            {top_ids, 4ull * rows * top, "top_ids"},
                            {top_logprobs, 4ull * rows * top, "top_logprobs"},
                            {workspace, need, "workspace"},
                            {tokens, 4ull * rows, "tokens"}};
    constexpr int kOutputs = 6;
    const Rows read{logits, 4ull * vocab, 4 * std::min<uint64_t>(row_stride, 1ull << 60), rows, "logits"};
    for (int i = 0; i < kOutputs; ++i)
    {
        const Range& w = ranges[i];
        if (w.at == nullptr || w.bytes == 0)
        {
            continue;
        }
        // The join reads a row's given token and its logit again when other rows' results are written.
        if (Overlap(w, read))
        {
            return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w.name, read.name);
        }
        for (int j = i + 1; j <= kOutputs; ++j)
        {
            if (ranges[j].at != nullptr && ranges[j].bytes != 0 && Overlap(w, ranges[j]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, w.name, ranges[j].name);
            }
        }
    }
    const dim3 grid(static_cast<uint32_t>(blocks));
    if (4ull * rows * vocab > kOnceBytes)
    {
        hipLaunchKernelGGL(TokenLogprobsKernel<true>, grid, dim3(kBlock), 0, AsStream(stream), a);
    }
    else
    {
        hipLaunchKernelGGL(TokenLogprobsKernel<false>, grid, dim3(kBlock), 0, AsStream(stream), a);
    }
    if (parts > 1)
    {
        hipLaunchKernelGGL(TokenLogprobsJoinKernel, dim3(rows), dim3(kBlock), 0, AsStream(stream), a);
    }
    return LaunchStatus(name);
}
