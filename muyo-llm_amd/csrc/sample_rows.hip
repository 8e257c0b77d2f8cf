// The next token of rows of logits: temperature, top-k, top-p and min-p of each row, and one given random number.
//
// A logit x has a place on a grid of eighths of an octave of weight, y = x 8 log2(e) / temperature = g + f, g whole
// and f within half a step of 0: its weight is 2^(g / 8) 2^(f / 8). The second factor, near 1, is held as a whole
// number of 2^-38, so that the mass of all logits in the same step is an exact sum in any order, and weights of
// different steps meet as 64-bit floating-point numbers in a fixed order: the same call gives the same bits.
#include <algorithm>
#include <cmath>

#include "logit_order.hpp"

namespace muyo
{
namespace
{
constexpr int kBlock = 256;                    // threads that count a part of a row
constexpr int kWaves = kBlock / kWave;
constexpr int kSteps = 512;                    // of the grid, from the row's largest logit down: 64 octaves
constexpr int kSlack = 8;                      // steps above the largest logit so far
constexpr int kLoads = 16;                     // of a lane at a time
constexpr uint32_t kBatch = kWave * kLoads;    // logits a wave takes at a time
constexpr int kPickBlock = 1024;               // threads that decide a row
constexpr int kPickWaves = kPickBlock / kWave;
constexpr int kPickLoads = 8;
constexpr uint32_t kGroup = kWave * kPickLoads;  // logits of a sum on the way to the token
constexpr uint32_t kListed = 4096;             // logits of a step that are listed
constexpr uint32_t kMaxParts = 64;             // workgroups of a row
constexpr uint32_t kMaxRows = (1u << 22) - 1;  // a launch has fewer than 2^32 threads
constexpr uint32_t kMaxVocab = 1u << 24;       // masses of so many logits fit in 63 bits
constexpr uint32_t kBlocksAtOnce = 256 * 6;    // workgroups that 256 CUs run at once
constexpr double kLog2e = 1.44269504088896340736;
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kUnit = 0x1p-38;              // of a mass

/// What a part of a row says besides its counts.
struct PartHead
{
    double top;    // the grid's place of its first step, -inf: it has none
    float most;    // its largest logit
    uint32_t at;   // the first place of that
};

struct SampleArgs
{
    const float* logits;
    uint64_t stride;
    uint32_t rows, vocab;
    const float* temperatures;
    const int32_t* topKs;
    const float* topPs;
    const float* minPs;
    const double* randoms;
    int32_t* tokens;
    float* logprobs;
    uint32_t parts, partLength;
    PartHead* heads;     // [rows][parts]
    uint64_t* masses;    // [rows][parts][kSteps]
    uint32_t* counts;    // [rows][parts][kSteps]
};

/// A logit as it counts: -inf for NaN, the largest finite one for +inf.
__device__ __forceinline__ float Counted(float x) { return x == x ? fminf(x, 0x1.fffffep127f) : -INFINITY; }

/// Steps of the grid per unit of a logit, 0 for a greedy row.
__device__ __forceinline__ double StepsPerUnit(const SampleArgs& a, uint32_t row)
{
    const float t = a.temperatures != nullptr ? a.temperatures[row] : 1.0f;
    return t > 0.0f ? 8.0 * kLog2e / static_cast<double>(t) : -1.0;
}

/// A logit's place on the grid.
struct Place
{
    double step;  // whole
    double rest;  // from its middle
};

/// The same bits wherever it is computed: nothing is contracted.
__device__ __forceinline__ Place PlaceOf(float x, double perUnit)
{
#pragma clang fp contract(off)
    // The product and what its rounding left out: differences of far places keep their bits.
    const double y = static_cast<double>(x);
    const double p = y * perUnit;
    const double left = fma(y, perUnit, -p);
    Place at;
    at.step = rint(p);
    // Places past 2^50 are whole steps apart, if they differ at all.
    at.rest = fmin(fmax((p - at.step) + left, -0.75), 0.75);
    return at;
}

/// 2^(rest / 8) in units of 2^-38: a power series, whose next term is below 2^-49 (|rest / 8 ln 2| <= 0.065).
__device__ __forceinline__ uint64_t MassOf(double rest)
{
    const double z = rest * (kLn2 / 8.0);
    double s = 1.0 / 5040.0;
    s = fma(s, z, 1.0 / 720.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, 1.0 / 24.0);
    s = fma(s, z, 1.0 / 6.0);
    s = fma(s, z, 0.5);
    s = fma(s, z, 1.0);
    s = fma(s, z, 1.0);
    // Rounded to a whole number by 2^52, whose bits then go.
    return static_cast<uint64_t>(__double_as_longlong(fma(s, 1.0 / kUnit, 0x1p52))) & 0xFFFFFFFFFFFFFull;
}

/// The weight of a mass in the `d`-th step from the top, relative to that.
__device__ __forceinline__ double WeightOf(uint64_t mass, uint32_t d)
{
    return static_cast<double>(mass) * exp2(-38.0 - static_cast<double>(d) * 0.125);
}

/// Counts the logits of a part of a row in steps of the grid, and their masses. A wave has counters of its own in
/// LDS, from a step above the largest logit that it has met; a larger one moves them down, which is rare.
__global__ __launch_bounds__(kBlock) void SampleCountKernel(SampleArgs a)
{
    __shared__ uint64_t massOf[kWaves][kSteps];
    __shared__ uint32_t countOf[kWaves][kSteps];
    __shared__ double topOf[kWaves];
    __shared__ float mostOf[kWaves];
    __shared__ uint32_t atOf[kWaves];
    const uint32_t row = blockIdx.x / a.parts;
    const uint32_t part = blockIdx.x - row * a.parts;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = threadIdx.x / kWave;
    const uint32_t begin = part * a.partLength;
    const uint32_t end = min(begin + a.partLength, a.vocab);
    const float* const x = a.logits + row * a.stride;
    const double perUnit = StepsPerUnit(a, row);
    uint64_t* const masses = massOf[wave];
    uint32_t* const counts = countOf[wave];
    for (int i = lane; i < kSteps; i += kWave)
    {
        masses[i] = 0;
        counts[i] = 0;
    }
    double top = -INFINITY;
    float most = -INFINITY;
    uint32_t at = 0;
    for (uint32_t first = begin + wave * kBatch; first < end; first += kWaves * kBatch)
    {
        float v[kLoads];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i)
        {
            const uint32_t index = first + i * kWave + lane;
            v[i] = x[min(index, end - 1)];
        }
        float batchMost = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i)
        {
            const uint32_t index = first + i * kWave + lane;
            v[i] = index < end ? Counted(v[i]) : -INFINITY;
            batchMost = fmaxf(batchMost, v[i]);
            if (v[i] > most)
            {
                most = v[i];
                at = index;
            }
        }
        batchMost = GroupMax<kWave>(batchMost);
        if (perUnit < 0.0 || batchMost == -INFINITY)
        {
            continue;
        }
        const double highest = PlaceOf(batchMost, perUnit).step;
        if (highest > top)
        {
            const double moved = highest + kSlack;
            if (top != -INFINITY)
            {
                const double by = moved - top;
                const uint32_t shift = by < kSteps ? static_cast<uint32_t>(by) : kSteps;
                uint64_t m[kSteps / kWave];
                uint32_t c[kSteps / kWave];
#pragma unroll
                for (uint32_t i = 0; i < kSteps / kWave; ++i)
                {
                    const uint32_t to = i * kWave + lane;
                    m[i] = to >= shift ? masses[to - shift] : 0;
                    c[i] = to >= shift ? counts[to - shift] : 0;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (uint32_t i = 0; i < kSteps / kWave; ++i)
                {
                    masses[i * kWave + lane] = m[i];
                    counts[i * kWave + lane] = c[i];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            top = moved;
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i)
        {
            const Place place = PlaceOf(v[i], perUnit);
            const double d = top - place.step;
            if (v[i] > -INFINITY && d < kSteps)
            {
                const uint32_t step = static_cast<uint32_t>(d);
                atomicAdd(reinterpret_cast<unsigned long long*>(masses + step), MassOf(place.rest));
                atomicAdd(counts + step, 1u);
            }
        }
    }
    // The wave's largest and its first place.
    const float waveMost = GroupMax<kWave>(most);
    uint32_t first = most == waveMost && most > -INFINITY ? at : ~0u;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        first = min(first, static_cast<uint32_t>(__shfl_xor(first, step)));
    }
    if (lane == 0)
    {
        topOf[wave] = top;
        mostOf[wave] = waveMost;
        atOf[wave] = first;
    }
    __syncthreads();
    double partTop = topOf[0];
    float partMost = mostOf[0];
    uint32_t partAt = atOf[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
    {
        partTop = fmax(partTop, topOf[w]);
        partAt = mostOf[w] > partMost ? atOf[w] : mostOf[w] == partMost ? min(partAt, atOf[w]) : partAt;
        partMost = fmaxf(partMost, mostOf[w]);
    }
    const uint64_t slot = blockIdx.x;
    if (threadIdx.x == 0)
    {
        a.heads[slot] = PartHead{partTop, partMost, partAt};
    }
    if (partTop == -INFINITY)
    {
        return;
    }
    for (uint32_t i = threadIdx.x; i < kSteps; i += kBlock)
    {
        uint64_t mass = 0;
        uint32_t count = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
        {
            const double by = partTop - topOf[w];
            if (by <= static_cast<double>(i))
            {
                const uint32_t from = i - static_cast<uint32_t>(by);
                mass += massOf[w][from];
                count += countOf[w][from];
            }
        }
        a.masses[slot * kSteps + i] = mass;
        a.counts[slot * kSteps + i] = count;
    }
}

/// Inclusive sums over the workgroup's threads, in thread order.
template <typename T>
__device__ __forceinline__ T PickSums(T v, T* waveSum)
{
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = threadIdx.x / kWave;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        const T other = __shfl_up(v, step);
        v += lane >= static_cast<uint32_t>(step) ? other : T{};
    }
    __syncthreads();
    if (lane == kWave - 1)
    {
        waveSum[wave] = v;
    }
    __syncthreads();
    T before{};
    for (uint32_t w = 0; w < wave; ++w)
    {
        before += waveSum[w];
    }
    return before + v;
}

template <typename T>
__device__ __forceinline__ T WaveSum(T v)
{
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        v += __shfl_xor(v, step);
    }
    return v;
}

/// A key and the counts of those above it.
struct Cut
{
    uint64_t key;    // what is kept of a step has at least this key
    uint64_t mass;   // of what is kept
};

struct PickSpace
{
    uint64_t keys[kListed];
    uint64_t steps[kSteps];      // masses of a step, of digits; weights up to a step (as double)
    uint32_t counts[kSteps];     // logits up to a step
    uint32_t digitCounts[256];
    double waveWeights[kPickWaves];
    uint32_t waveCounts[kPickWaves];
    uint64_t waveMasses[kPickWaves];
    double groupWeights[kPickBlock];
    uint32_t partShift[kMaxParts];
    uint64_t partMass[kMaxParts];
    double partWeight[kMaxParts];
    uint64_t digitMasses[256];
    uint32_t listed;
    uint32_t stepK, stepP;
    uint32_t last, lastAbove;  // a digit of the cut, and the logits above it
    uint64_t lastMasses[2];    // above it, and its own
};

/// A row's grid and its threshold.
struct RowGrid
{
    const float* x;
    uint32_t vocab;
    double perUnit, top;
    Place largest;
    double lowest;  // of y - largest, by min-p; -inf: none
};

__device__ __forceinline__ bool Reaches(const RowGrid& r, const Place& at)
{
    return (at.step - r.largest.step) + (at.rest - r.largest.rest) >= r.lowest;
}

/// Calls use(key, mass) for the logits of step d that reach min-p, by all threads (a barrier before and after is
/// the caller's).
template <typename Use>
__device__ __forceinline__ void ForStep(const RowGrid& r, uint32_t d, Use use)
{
    for (uint32_t first = 0; first < r.vocab; first += kPickBlock * kPickLoads)
    {
        float v[kPickLoads];
#pragma unroll
        for (uint32_t i = 0; i < kPickLoads; ++i)
        {
            v[i] = r.x[min(first + i * kPickBlock + threadIdx.x, r.vocab - 1)];
        }
#pragma unroll
        for (uint32_t i = 0; i < kPickLoads; ++i)
        {
            const uint32_t index = first + i * kPickBlock + threadIdx.x;
            const float x = Counted(v[i]);
            const Place at = PlaceOf(x, r.perUnit);
            if (index < r.vocab && x > -INFINITY && r.top - at.step == static_cast<double>(d) && Reaches(r, at))
            {
                use(OrderKey(x, index), MassOf(at.rest));
            }
        }
    }
}

/// The cut in step d: the first keys, `most` at most, and no more than it takes to have `limit` of mass (a key is
/// kept where those above it have less). Digit by digit of the keys, from the highest: the digit in which the cut
/// lies is found from counts and masses of all digits. Steps of up to kListed logits are listed first.
__device__ Cut CutStep(const RowGrid& r, uint32_t d, uint32_t count, uint32_t most, double limit, PickSpace& s)
{
    const bool list = count <= kListed;
    __syncthreads();
    if (list)
    {
        if (threadIdx.x == 0)
        {
            s.listed = 0;
        }
        __syncthreads();
        ForStep(r, d, [&](uint64_t key, uint64_t) { s.keys[atomicAdd(&s.listed, 1u)] = key; });
        __syncthreads();
    }
    uint64_t prefix = 0;     // of the cut's key
    uint64_t aboveMass = 0;  // of keys above those with the prefix
    uint32_t above = 0;
    for (int shift = 56; shift >= 0; shift -= 8)
    {
        for (uint32_t i = threadIdx.x; i < 256; i += kPickBlock)
        {
            s.digitCounts[i] = 0;
            s.digitMasses[i] = 0;
        }
        if (threadIdx.x == 0)
        {
            s.last = 0;
        }
        __syncthreads();
        auto use = [&](uint64_t key, uint64_t mass) {
            if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
            {
                const uint32_t digit = 255u - (static_cast<uint32_t>(key >> shift) & 255u);
                atomicAdd(&s.digitCounts[digit], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.digitMasses[digit]), mass);
            }
        };
        if (list)
        {
            for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
            {
                use(s.keys[i], MassOf(PlaceOf(KeyValue(s.keys[i]), r.perUnit).rest));
            }
        }
        else
        {
            ForStep(r, d, use);
        }
        __syncthreads();
        // In falling order of digits; those of a key that is kept begin before both limits.
        const uint32_t c = threadIdx.x < 256 ? s.digitCounts[threadIdx.x] : 0;
        const uint64_t m = threadIdx.x < 256 ? s.digitMasses[threadIdx.x] : 0;
        const uint32_t counts = above + PickSums(c, s.waveCounts) - c;
        const uint64_t masses = aboveMass + PickSums(m, s.waveMasses) - m;
        const bool begins = c > 0 && counts < most && static_cast<double>(masses) < limit;
        if (begins)
        {
            atomicMax(&s.last, threadIdx.x + 1);  // the last digit of which something is kept
        }
        __syncthreads();
        const uint32_t last = s.last;
        if (last == 0)  // nothing in the step reaches min-p
        {
            return Cut{~0ull, aboveMass};
        }
        if (threadIdx.x == last - 1)
        {
            s.lastAbove = counts;
            s.lastMasses[0] = masses;
            s.lastMasses[1] = m;
        }
        __syncthreads();
        above = s.lastAbove;
        aboveMass = s.lastMasses[0];
        prefix |= static_cast<uint64_t>(256u - last) << shift;
        if (shift == 0)
        {
            aboveMass += s.lastMasses[1];  // keys differ: one
        }
        __syncthreads();
    }
    return Cut{prefix, aboveMass};
}

/// Decides a row: where the cuts lie in the steps' counts and masses, in which part the token lies, and which it is.
__global__ __launch_bounds__(kPickBlock) void SamplePickKernel(SampleArgs a)
{
    __shared__ PickSpace s;
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = threadIdx.x / kWave;
    const uint64_t slot = static_cast<uint64_t>(row) * a.parts;

    // Every wave looks at the parts, a lane each.
    static_assert(kMaxParts == kWave, "a lane for each part");
    PartHead head = a.heads[slot + min(lane, a.parts - 1)];
    if (lane >= a.parts)
    {
        head = PartHead{-INFINITY, -INFINITY, ~0u};
    }
    const float most = GroupMax<kWave>(head.most);
    uint32_t at = head.most == most ? head.at : ~0u;
    double top = head.top;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2)
    {
        at = min(at, static_cast<uint32_t>(__shfl_xor(at, step)));
        top = fmax(top, __shfl_xor(top, step));
    }
    const double perUnit = StepsPerUnit(a, row);
    if (most == -INFINITY || perUnit < 0.0)
    {
        if (threadIdx.x == 0)
        {
            a.tokens[row] = most == -INFINITY ? -1 : static_cast<int32_t>(at);
            if (a.logprobs != nullptr)
            {
                a.logprobs[row] = most == -INFINITY ? -INFINITY : 0.0f;
            }
        }
        return;
    }
    RowGrid r;
    r.x = a.logits + row * a.stride;
    r.vocab = a.vocab;
    r.perUnit = perUnit;
    r.top = top;
    r.largest = PlaceOf(most, perUnit);
    const float minP = a.minPs != nullptr ? a.minPs[row] : 0.0f;
    r.lowest = minP > 0.0f ? 8.0 * log2(static_cast<double>(minP)) : -INFINITY;
    if (threadIdx.x < kWave)
    {
        const double by = top - head.top;
        s.partShift[lane] = by < kSteps ? static_cast<uint32_t>(by) : kSteps;  // a part with nothing: all
        s.partMass[lane] = 0;
    }
    __syncthreads();

    // The row's steps, and what they add up to.
    const uint32_t d = threadIdx.x;
    uint64_t mass = 0;
    uint32_t count = 0;
    if (d < kSteps)
    {
        for (uint32_t p = 0; p < a.parts; ++p)
        {
            const uint32_t shift = s.partShift[p];
            if (d >= shift)
            {
                mass += a.masses[(slot + p) * kSteps + d - shift];
                count += a.counts[(slot + p) * kSteps + d - shift];
            }
        }
    }
    const double weight = WeightOf(mass, d);
    const uint32_t counts = PickSums(count, s.waveCounts);
    const double weights = PickSums(weight, s.waveWeights);
    double* const upTo = reinterpret_cast<double*>(s.steps);
    if (d < kSteps)
    {
        s.counts[d] = counts;
        upTo[d] = weights;
    }
    if (threadIdx.x == 0)
    {
        s.stepK = kSteps - 1;
        s.stepP = kSteps - 1;
    }
    __syncthreads();
    const uint32_t all = s.counts[kSteps - 1];
    const int32_t topK = a.topKs != nullptr ? a.topKs[row] : 0;
    const float topP = a.topPs != nullptr ? a.topPs[row] : 1.0f;
    const uint32_t k = topK > 0 ? min(static_cast<uint32_t>(topK), all) : all;
    // The step in which the first k end.
    if (d < kSteps && counts >= k)
    {
        atomicMin(&s.stepK, d);
    }
    __syncthreads();
    const uint32_t stepK = s.stepK;
    const uint32_t beforeK = stepK > 0 ? s.counts[stepK - 1] : 0;
    const bool wholeK = s.counts[stepK] == k;
    // The step in which top-p's share of their weight is reached.
    uint32_t stepP = kSteps;
    double share = INFINITY;
    if (topP < 1.0f)
    {
        double ofK = upTo[stepK];
        if (!wholeK)
        {
            RowGrid whole = r;
            whole.lowest = -INFINITY;
            const Cut cut = CutStep(whole, stepK, s.counts[stepK] - beforeK, k - beforeK, INFINITY, s);
            ofK = (stepK > 0 ? upTo[stepK - 1] : 0.0) + WeightOf(cut.mass, stepK);
        }
        share = static_cast<double>(topP) * ofK;
        if (d <= stepK && counts > 0 && weights >= share)
        {
            atomicMin(&s.stepP, d);
        }
        __syncthreads();
        stepP = min(s.stepP, stepK);
    }
    // The step in which min-p's bound lies.
    uint32_t stepM = kSteps;
    if (minP > 0.0f)
    {
        const double by = top - rint(r.largest.step + r.largest.rest + r.lowest);
        const double first = top - r.largest.step;
        stepM = by < kSteps ? static_cast<uint32_t>(fmax(by, first)) : kSteps;
    }
    const uint32_t step = min(min(stepK, stepP), stepM);
    const double before = step > 0 ? upTo[step - 1] : 0.0;
    const uint32_t countBefore = step > 0 ? s.counts[step - 1] : 0;
    Cut cut{0, 0};
    const bool whole = step != stepP && step != stepM && (step != stepK || wholeK);
    double total = upTo[step];
    if (!whole)
    {
        const uint32_t left = step == stepK ? k - countBefore : ~0u;
        // A share that is reached before this step's first, by a rounding, still keeps that one.
        const double limit =
            step == stepP ? fmax((share - before) * exp2(38.0 + static_cast<double>(step) * 0.125), 0x1p-30) : INFINITY;
        RowGrid bounded = r;
        bounded.lowest = step == stepM ? r.lowest : -INFINITY;
        // The first logit is always kept.
        bounded.lowest = fmin(bounded.lowest, 0.0);
        cut = CutStep(bounded, step, s.counts[step] - countBefore, minP > 1.0f ? min(left, 1u) : left, limit, s);
        total = before + WeightOf(cut.mass, step);
    }
    // Kept: the steps before, and of this one the keys from the cut on.
    auto weightAt = [&](float v, uint32_t index) {
        const float x = Counted(v);
        const Place place = PlaceOf(x, perUnit);
        const double dist = top - place.step;
        const bool kept = x > -INFINITY && (dist < static_cast<double>(step) ||
                                            (dist == static_cast<double>(step) && OrderKey(x, index) >= cut.key));
        return kept ? WeightOf(MassOf(place.rest), static_cast<uint32_t>(dist)) : 0.0;
    };

    // What each part has of it: the steps before from its counts, this one's kept logits by a look at them.
    __syncthreads();
    constexpr uint32_t kLanesOfPart = kPickBlock / kMaxParts;
    {
        const uint32_t p = threadIdx.x / kLanesOfPart;
        double sum = 0.0;
        if (p < a.parts)
        {
            const uint32_t shift = s.partShift[p];
            const uint32_t until = whole ? step + 1 : step;
            for (uint32_t i = shift + threadIdx.x % kLanesOfPart; i < until; i += kLanesOfPart)
            {
                sum += WeightOf(a.masses[(slot + p) * kSteps + i - shift], i);
            }
        }
#pragma unroll
        for (uint32_t i = 1; i < kLanesOfPart; i *= 2)
        {
            sum += __shfl_xor(sum, i);
        }
        if (threadIdx.x % kLanesOfPart == 0)
        {
            s.partWeight[p] = sum;
        }
    }
    __syncthreads();
    if (!whole)
    {
        auto use = [&](uint64_t key, uint64_t ofKey) {
            if (key >= cut.key)
            {
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.partMass[~static_cast<uint32_t>(key) / a.partLength]),
                          ofKey);
            }
        };
        if (s.counts[step] - countBefore <= kListed)
        {
            for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
            {
                use(s.keys[i], MassOf(PlaceOf(KeyValue(s.keys[i]), perUnit).rest));
            }
        }
        else
        {
            RowGrid bounded = r;
            bounded.lowest = -INFINITY;
            ForStep(bounded, step, use);
        }
    }
    __syncthreads();
    const double random = a.randoms[row];
    const double reach = (random > 0.0 ? random : 0.0) * total;
    // The first part that reaches past the number's share, else the last with anything kept.
    uint32_t part = 0;
    double passed = 0.0;
    {
        double upToPart = 0.0;
        for (uint32_t p = 0; p < a.parts; ++p)
        {
            const double of = s.partWeight[p] + WeightOf(s.partMass[p], step);
            if (of > 0.0)
            {
                part = p;
                passed = upToPart;
                upToPart += of;
                if (upToPart > reach)
                {
                    break;
                }
            }
        }
    }
    // Sums of its groups of logits, and the first group that reaches past it, else the last with anything kept.
    const uint32_t begin = part * a.partLength;
    const uint32_t end = min(begin + a.partLength, a.vocab);
    const uint32_t groups = (end - begin + kGroup - 1) / kGroup;
    uint32_t group = 0;
    double sum = passed;
    bool past = false;
    for (uint32_t first = 0; first < groups && !past; first += kPickBlock)
    {
        const uint32_t here = min(groups - first, static_cast<uint32_t>(kPickBlock));
        __syncthreads();
        for (uint32_t i = wave; i < here; i += kPickWaves)
        {
            float v[kPickLoads];
            const uint32_t from = begin + (first + i) * kGroup + lane;
#pragma unroll
            for (uint32_t j = 0; j < kPickLoads; ++j)
            {
                v[j] = r.x[min(from + j * kWave, end - 1)];
            }
            double own = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < kPickLoads; ++j)
            {
                own += from + j * kWave < end ? weightAt(v[j], from + j * kWave) : 0.0;
            }
            own = WaveSum(own);
            if (lane == 0)
            {
                s.groupWeights[i] = own;
            }
        }
        __syncthreads();
        for (uint32_t i = 0; i < here && !past; ++i)
        {
            const double of = s.groupWeights[i];
            if (of > 0.0)
            {
                group = first + i;
                passed = sum;
                sum += of;
                past = sum > reach;
            }
        }
    }
    if (wave != 0)
    {
        return;
    }
    // The first of its logits that reaches past it, else its last that is kept.
    uint32_t token = ~0u;
    double of = 0.0;
    const uint32_t from = begin + group * kGroup;
    for (uint32_t j = 0; j < kPickLoads; ++j)
    {
        const uint32_t index = from + j * kWave + lane;
        const double own = index < end ? weightAt(r.x[index], index) : 0.0;
        double sum = own;
#pragma unroll
        for (int i = 1; i < kWave; i *= 2)
        {
            const double other = __shfl_up(sum, i);
            sum += lane >= static_cast<uint32_t>(i) ? other : 0.0;
        }
        const uint64_t kept = __ballot(own > 0.0);
        const uint64_t past = __ballot(own > 0.0 && passed + sum > reach);
        if (kept != 0)
        {
            const int which = past != 0 ? __ffsll(static_cast<unsigned long long>(past)) - 1
                                        : 63 - __clzll(static_cast<long long>(kept));
            token = from + j * kWave + which;
            of = __shfl(own, which);
        }
        if (past != 0)
        {
            break;
        }
        passed += __shfl(sum, kWave - 1);
    }
    if (lane == 0)
    {
        a.tokens[row] = static_cast<int32_t>(token);
        if (a.logprobs != nullptr)
        {
            a.logprobs[row] = static_cast<float>(log(of / total));
        }
    }
}

/// Workgroups of a row, and its logits that one counts.
struct Parts
{
    uint32_t count, length;
};

Parts PartsOf(uint32_t rows, uint32_t vocab)
{
    const uint32_t batches = CeilDiv(vocab, kBatch);
    const uint32_t most = std::min(kMaxParts, CeilDiv(batches, kWaves));
    const uint32_t wanted = std::max(1u, std::min(most, kBlocksAtOnce / std::max(rows, 1u)));
    const uint32_t length = CeilDiv(batches, wanted) * kBatch;
    return Parts{CeilDiv(vocab, length), length};
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_sample_rows_workspace_bytes(uint32_t rows, uint32_t vocab)
{
    if (rows == 0 || rows > kMaxRows || vocab == 0 || vocab > kMaxVocab)
    {
        return 0;
    }
    return (sizeof(PartHead) + 12ull * kSteps) * rows * PartsOf(rows, vocab).count;
}

extern "C" int muyo_sample_rows_f32(const float* logits, uint64_t row_stride, uint32_t rows, uint32_t vocab,
                                    const float* temperatures, const int32_t* top_ks, const float* top_ps,
                                    const float* min_ps, const double* randoms, int32_t* tokens, float* logprobs,
                                    void* workspace, uint64_t workspace_bytes, void* stream)
{
    const char* name = "sample_rows_f32";
    if (logits == nullptr || randoms == nullptr || tokens == nullptr)
    {
        return Fail(MUYO_E_NULL, "%s: logits, randoms and tokens are required", name);
    }
    const size_t need = muyo_sample_rows_workspace_bytes(rows, vocab);
    if (need == 0)
    {
        return Fail(MUYO_E_RANGE, "%s: needs 1..%u rows of 1..%u logits (got %u of %u)", name, kMaxRows, kMaxVocab, rows,
                    vocab);
    }
    if (row_stride < vocab || (reinterpret_cast<uintptr_t>(logits) & 3u) != 0 ||
        (reinterpret_cast<uintptr_t>(randoms) & 7u) != 0)
    {
        return Fail(MUYO_E_CONTRACT, "%s: row_stride %llu is below vocab %u, or logits are not 4-byte or randoms not "
                                     "8-byte aligned",
                    name, static_cast<unsigned long long>(row_stride), vocab);
    }
    if (workspace == nullptr || !Aligned16(workspace) || workspace_bytes < need)
    {
        return Fail(MUYO_E_CONTRACT, "%s: needs a 16-byte aligned workspace of %zu bytes (got %llu)", name, need,
                    static_cast<unsigned long long>(workspace_bytes));
    }
    const Range ranges[] = {{tokens, 4ull * rows, "tokens"},
                            {workspace, need, "workspace"},
                            {logprobs, 4ull * rows, "logprobs"},
                            {temperatures, 4ull * rows, "temperatures"},
                            {top_ks, 4ull * rows, "top_ks"},
                            {top_ps, 4ull * rows, "top_ps"},
                            {min_ps, 4ull * rows, "min_ps"},
                            {randoms, 8ull * rows, "randoms"}};
    constexpr int kOutputs = 3;
    constexpr int kRanges = static_cast<int>(sizeof ranges / sizeof ranges[0]);
    const Rows read{logits, 4ull * vocab, 4 * std::min<uint64_t>(row_stride, 1ull << 60), rows, "logits"};
    for (int i = 0; i < kOutputs; ++i)
    {
        if (ranges[i].at == nullptr)
        {
            continue;
        }
        if (Overlap(ranges[i], read))
        {
            return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, ranges[i].name, read.name);
        }
        for (int j = i + 1; j < kRanges; ++j)
        {
            if (ranges[j].at != nullptr && Overlap(ranges[i], ranges[j]))
            {
                return Fail(MUYO_E_CONTRACT, "%s: %s overlaps %s", name, ranges[i].name, ranges[j].name);
            }
        }
    }
    const Parts parts = PartsOf(rows, vocab);
    const uint64_t blocks = static_cast<uint64_t>(rows) * parts.count;
    char* space = static_cast<char*>(workspace);
    SampleArgs a{logits, row_stride, rows, vocab, temperatures, top_ks, top_ps, min_ps, randoms, tokens, logprobs,
                 parts.count, parts.length, nullptr, nullptr, nullptr};
    a.masses = reinterpret_cast<uint64_t*>(space);
    a.heads = reinterpret_cast<PartHead*>(space + 8ull * kSteps * blocks);
    a.counts = reinterpret_cast<uint32_t*>(space + (8ull * kSteps + sizeof(PartHead)) * blocks);
    hipLaunchKernelGGL(SampleCountKernel, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, AsStream(stream), a);
    hipLaunchKernelGGL(SamplePickKernel, dim3(rows), dim3(kPickBlock), 0, AsStream(stream), a);
    return LaunchStatus(name);
}
