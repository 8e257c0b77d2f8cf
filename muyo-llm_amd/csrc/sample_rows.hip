// The next token of rows of logits: temperature, top-k, top-p and min-p of each row, and one given random number.
//
// A logit x has a place on a grid of eighths of an octave of weight, y = x 8 log2(e) / temperature = g + f, g whole
// and f within half a step of 0: its weight is 2^(g / 8) 2^(f / 8). The second factor, near 1, is held as a whole
// number of 2^-38, so that the mass of all logits in the same step is an exact sum in any order, and weights of
// different steps meet as 64-bit floating-point numbers in a fixed order: the same call gives the same bits. Sums in
// 32 bits would not do: a number lands on another token where the sums before it are off, which of 151936 tokens of
// similar weight one row in ten would see.
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
constexpr int kQuads = 4;                      // 16-byte loads of a lane's batch
constexpr uint32_t kBatch = kWave * 4 * kQuads;  // logits a wave takes at a time
constexpr int kPickBlock = 512;                // threads that decide a row
constexpr int kPickWaves = kPickBlock / kWave;
constexpr int kPickLoads = 8;
constexpr uint32_t kGroup = kWave * kPickLoads;  // logits of a sum on the way to the token
constexpr uint32_t kGroups = 32;               // such sums at a time, four of each wave: half a part on average
constexpr uint32_t kListed = 4096;             // logits that are listed
constexpr int32_t kListedK = 2048;             // a top-k up to which listing the tokens is likely to do
constexpr uint32_t kDigits = 256;
constexpr uint32_t kFew = kWave;               // candidates that a wave looks at one by one
constexpr uint32_t kMaxParts = 64;             // workgroups of a row
constexpr uint32_t kMaxRows = (1u << 22) - 1;  // a launch has fewer than 2^32 threads
constexpr uint32_t kMaxVocab = 1u << 24;       // masses of so many logits fit in 63 bits
constexpr uint32_t kCountBlocks = 1024;        // workgroups to aim at that count
constexpr uint32_t kFewestParts = 4;           // of a row, if it has the batches
constexpr double kLog2e = 1.44269504088896340736;
constexpr uint32_t kListRows = 4096;           // rows whose lists get workgroups of their own
constexpr uint32_t kListAtOnce = 16384;        // waves of those that fit the GPU at about once
constexpr double kFar = 0x1p48;                // places past which steps are not whole numbers apart
constexpr double kWhole = 0x1.8p52;            // added, the whole part's last 32 bits come last
constexpr double kFixed = 0x1p50;              // units of the top step's weight, for sums of listed logits

/// What a part of a row says besides its counts.
struct PartHead
{
    double top;    // the grid's place of its first step, -inf: it has none
    float most;    // its largest logit
    uint32_t at;   // the first place of that, of a greedy row
};

/// What is known of a row's steps before its token is chosen, and which are listed.
struct RowSteps
{
    double upTo[kSteps];
    uint32_t counts[kSteps];
    double top, perUnit;
    uint32_t first, last;  // steps that are listed: none if first > last
    float low, high;       // bounds of their logits
    uint32_t listed;
    uint32_t unused;
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
    float* batchMost;    // [rows][parts][batches]: the largest logit of each
    uint32_t batches;    // of a part, at most
    RowSteps* steps;     // [rows], of at most kListRows; where the workspace begins
    uint64_t* listKeys;  // [rows][listRoom] of these
    uint32_t listRoom;
};

/// What a row asks for.
struct RowMode
{
    double perUnit;  // steps of the grid per unit of a logit; below 0: the largest logit is taken
    int32_t topK;    // 0: all
    bool counted;    // logits of a step are counted, for top-k
    bool weighed;    // their masses are summed; where few tokens are kept at most, these are listed instead
};

__device__ __forceinline__ RowMode ModeOf(const SampleArgs& a, uint32_t row)
{
    const float t = a.temperatures != nullptr ? a.temperatures[row] : 1.0f;
    RowMode mode;
    // Above 0 also where the temperature is infinite, so that a logit of -inf is as far away as elsewhere.
    mode.perUnit = t > 0.0f ? fmax(8.0 * kLog2e / static_cast<double>(t), 1e-290) : -1.0;
    mode.topK = a.topKs != nullptr ? max(a.topKs[row], 0) : 0;
    mode.counted = mode.topK > 0;
    mode.weighed = mode.topK == 0 || mode.topK > kListedK;
    return mode;
}

/// move(word) of each 32-bit word of v.
template <typename T, typename Move>
__device__ __forceinline__ T ByWords(T v, Move move)
{
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "words");
    if constexpr (sizeof(T) == 4)
    {
        return __builtin_bit_cast(T, move(__builtin_bit_cast(int, v)));
    }
    else
    {
        const uint64_t bits = __builtin_bit_cast(uint64_t, v);
        const uint32_t low = static_cast<uint32_t>(move(static_cast<int>(static_cast<uint32_t>(bits))));
        const uint32_t high = static_cast<uint32_t>(move(static_cast<int>(static_cast<uint32_t>(bits >> 32))));
        return __builtin_bit_cast(T, static_cast<uint64_t>(high) << 32 | low);
    }
}

/// The same of all of a wave's lanes: join(a, b) of all, in pairs, pairs of pairs and so on.
template <typename T, typename Join>
__device__ __forceinline__ T WaveJoin(T v, Join join)
{
    v = join(v, ByWords(v, [](int w) { return PartnerLane<1>(w); }));
    v = join(v, ByWords(v, [](int w) { return PartnerLane<2>(w); }));
    v = join(v, ByWords(v, [](int w) { return PartnerLane<4>(w); }));
    v = join(v, ByWords(v, [](int w) { return PartnerLane<8>(w); }));
    v = join(v, ByWords(v, [](int w) { return PartnerLane<16>(w); }));
    return join(v, ByWords(v, [](int w) { return PartnerLane<32>(w); }));
}

template <typename T>
__device__ __forceinline__ T WaveSum(T v)
{
    return WaveJoin(v, [](T a, T b) { return a + b; });
}

/// The smallest of a wave's values.
template <typename T>
__device__ __forceinline__ T WaveLeast(T v)
{
    return WaveJoin(v, [](T a, T b) { return a < b ? a : b; });
}

/// v plus that of the lane a DPP control names, in the given rows of 16 lanes; 0 from no lane.
template <int kControl, int kRows, typename T>
__device__ __forceinline__ T PlusLane(T v)
{
    return v + ByWords(v, [](int w) { return __builtin_amdgcn_update_dpp(0, w, kControl, kRows, 0xF, false); });
}

/// Inclusive sum over the wave's lanes: shifts inside rows of 16 lanes, then the last lanes of rows to those behind.
template <typename T>
__device__ __forceinline__ T WaveInclusive(T v)
{
    v = PlusLane<0x111, 0xF>(v);  // row_shr:1
    v = PlusLane<0x112, 0xF>(v);
    v = PlusLane<0x114, 0xF>(v);
    v = PlusLane<0x118, 0xF>(v);
    v = PlusLane<0x142, 0xA>(v);     // row_bcast:15
    return PlusLane<0x143, 0xC>(v);  // row_bcast:31
}

/// A lane's value, the lane the same in the whole wave.
template <typename T>
__device__ __forceinline__ T OfLane(T v, int lane)
{
    return ByWords(v, [&](int w) { return __builtin_amdgcn_readlane(w, lane); });
}

/// `x`, of a signalling NaN the quiet one: the larger of that and a number is the number, of a signalling one and a
/// number a quiet NaN, so that the number would be lost.
__device__ __forceinline__ float Quiet(float x) { return __builtin_canonicalizef(x); }

/// A logit as it counts: -inf for NaN, the largest finite one for +inf.
__device__ __forceinline__ float Counted(float x) { return fminf(fmaxf(Quiet(x), -INFINITY), 0x1.fffffep127f); }

/// A logit's place on the grid.
struct Place
{
    double step;  // whole
    double rest;  // from its middle
};

/// The whole number next to y * perUnit, as its sum with kWhole: for products below 2^51.
__device__ __forceinline__ double WholeOf(double y, double perUnit) { return fma(y, perUnit, kWhole); }

/// The same bits wherever it is computed.
__device__ __forceinline__ Place PlaceOf(float x, double perUnit)
{
    // A product is rounded once, what is left of it too: differences of far places keep their bits.
    const double y = static_cast<double>(x);
    Place at;
    at.step = fabs(y * perUnit) < 0x1p50 ? WholeOf(y, perUnit) - kWhole : rint(y * perUnit);
    // Far places are whole steps apart, if they differ at all, and have any remainder.
    at.rest = fmin(fmax(fma(y, perUnit, -at.step), -0.75), 0.75);
    return at;
}

/// 2^52 and 2^(rest / 8) in units of 2^-38, by a polynomial (the fit of least error over half a step each way:
/// 2^-41.6), to a whole number. kCount side by side.
template <int kCount>
__device__ __forceinline__ void MassSums(const double (&rest)[kCount], double (&m)[kCount])
{
    constexpr double kOne = 0x1p38;
    constexpr double c0 = 4.069392558613428e-08 * kOne;
    constexpr double c1 = 2.3483963990465326e-06 * kOne;
    constexpr double c2 = 0.00010840646184941278 * kOne;
    constexpr double c3 = 0.0037535391505790455 * kOne;
    constexpr double c4 = 0.08664339757000515 * kOne;
    constexpr double c5 = 1.0000000000002864 * kOne + 0x1p52;
    // As it stands, with the summands in scalar registers: the compiler would take the form that overwrites its
    // summand, and copy each first.
    if constexpr (kCount == 4)
    {
        asm("v_fma_f64 %0, %8, %4, %9\n\tv_fma_f64 %1, %8, %5, %9\n\t"
            "v_fma_f64 %2, %8, %6, %9\n\tv_fma_f64 %3, %8, %7, %9\n\t"
            "v_fma_f64 %0, %0, %4, %10\n\tv_fma_f64 %1, %1, %5, %10\n\t"
            "v_fma_f64 %2, %2, %6, %10\n\tv_fma_f64 %3, %3, %7, %10\n\t"
            "v_fma_f64 %0, %0, %4, %11\n\tv_fma_f64 %1, %1, %5, %11\n\t"
            "v_fma_f64 %2, %2, %6, %11\n\tv_fma_f64 %3, %3, %7, %11\n\t"
            "v_fma_f64 %0, %0, %4, %12\n\tv_fma_f64 %1, %1, %5, %12\n\t"
            "v_fma_f64 %2, %2, %6, %12\n\tv_fma_f64 %3, %3, %7, %12\n\t"
            "v_fma_f64 %0, %0, %4, %13\n\tv_fma_f64 %1, %1, %5, %13\n\t"
            "v_fma_f64 %2, %2, %6, %13\n\tv_fma_f64 %3, %3, %7, %13"
            : "=&v"(m[0]), "=&v"(m[1]), "=&v"(m[2]), "=&v"(m[3])
            : "v"(rest[0]), "v"(rest[1]), "v"(rest[2]), "v"(rest[3]), "v"(c0), "s"(c1), "s"(c2), "s"(c3), "s"(c4),
              "s"(c5));
    }
    else
    {
        static_assert(kCount == 1, "one, or four");
        asm("v_fma_f64 %0, %2, %1, %3\n\tv_fma_f64 %0, %0, %1, %4\n\tv_fma_f64 %0, %0, %1, %5\n\t"
            "v_fma_f64 %0, %0, %1, %6\n\tv_fma_f64 %0, %0, %1, %7"
            : "=&v"(m[0])
            : "v"(rest[0]), "v"(c0), "s"(c1), "s"(c2), "s"(c3), "s"(c4), "s"(c5));
    }
}

/// The mass of a sum with 2^52.
__device__ __forceinline__ uint64_t MassIn(double sum)
{
    return static_cast<uint64_t>(__double_as_longlong(sum)) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ uint64_t MassOf(double rest)
{
    double sum[1];
    MassSums<1>({rest}, sum);
    return MassIn(sum[0]);
}

/// Weight of a unit of mass in step d, relative to the top's.
__device__ __forceinline__ double UnitOf(uint32_t d) { return exp2(-38.0 - static_cast<double>(d) * 0.125); }

/// Whether places of logits that are at least `least` are near the top step's, so that steps are whole numbers of 32
/// bits apart; `least` lies past the last step.
__device__ __forceinline__ bool NearPlaces(double top, double perUnit, float& least)
{
    const double bound = (top - (kSteps + 2)) / perUnit;
    // Down: at small temperatures all steps are less than a unit in the last place of the largest logit, and the f32
    // nearest to the bound is that logit itself.
    least = __double2float_rd(bound);
    // (At huge temperatures the bound is below all numbers, and does not tell -inf from them.)
    return fabs(top) < kFar && bound > -0x1p127;
}

/// Adds a lane's logit to the counters of steps below `top`.
__device__ __forceinline__ void AddOne(float v, double top, double perUnit, uint64_t* masses, uint32_t* counts)
{
    const float x = Counted(v);
    const Place place = PlaceOf(x, perUnit);
    const double d = top - place.step;
    if (x > -INFINITY && d < kSteps)
    {
        const uint32_t step = static_cast<uint32_t>(d);
        atomicAdd(reinterpret_cast<unsigned long long*>(masses + step), MassOf(place.rest));
        atomicAdd(counts + step, 1u);
    }
}

/// The same of a batch, for places below kFar, with fewer operations: a step is the last 32 bits of a place's sum with
/// kWhole. Logits below `least`, past the last step, count as that, as does a NaN, so that no place is far; none is
/// past the top, infinite or a signalling NaN.
template <bool kCount, bool kMass>
__device__ __forceinline__ void AddNearBatch(const float4v (&v)[kQuads], double top, float least, double perUnit,
                                             uint64_t* masses, uint32_t* counts)
{
    const uint32_t topStep = static_cast<uint32_t>(__double_as_longlong(top + kWhole));
#pragma unroll
    for (int q = 0; q < kQuads; ++q)
    {
        // Four at a time, side by side up to the counters.
        uint32_t step[4];
        double rest[4], mass[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            // As it stands: the compiler would make both quiet again.
            float x;
            asm("v_max_f32 %0, %1, %2" : "=v"(x) : "v"(v[q][e]), "v"(least));
            const double y = static_cast<double>(x);
            const double whole = WholeOf(y, perUnit);
            step[e] = topStep - static_cast<uint32_t>(__double_as_longlong(whole));
            rest[e] = fma(y, perUnit, -(whole - kWhole));
        }
        if (kMass)
        {
            MassSums<4>(rest, mass);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            if (step[e] < kSteps)
            {
                if (kMass)
                {
                    atomicAdd(reinterpret_cast<unsigned long long*>(masses + step[e]), MassIn(mass[e]));
                }
                if (kCount)
                {
                    atomicAdd(counts + step[e], 1u);
                }
            }
        }
    }
}

/// A part of a row in batches of kBatch logits from the last 16-byte address at or before its first one on.
struct PartRange
{
    uint32_t begin, end;
    uint32_t before;   // logits of the first batch that are the part's before
    uint32_t batches;
};

__device__ __forceinline__ PartRange RangeOf(const float* x, uint32_t begin, uint32_t end)
{
    PartRange r{begin, end, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x + begin) / 4 % 4), 0};
    r.batches = (end - begin + r.before + kBatch - 1) / kBatch;
    return r;
}

/// A lane's i-th logit of a batch: four in a row from each quad. Before the part's first logit it wraps or is too
/// small.
__device__ __forceinline__ uint32_t IndexOf(const PartRange& r, uint32_t batch, uint32_t i)
{
    return r.begin - r.before + batch * kBatch + (i / 4 * kWave + threadIdx.x % kWave) * 4 + i % 4;
}

/// Whether a batch lies in the part as a whole.
__device__ __forceinline__ bool IsWhole(const PartRange& r, uint32_t batch)
{
    const uint32_t first = batch * kBatch;
    return first >= r.before && first + kBatch <= r.end - r.begin + r.before;
}

/// A batch logit by logit, -inf outside of the part.
__device__ __forceinline__ void LoadOneByOne(const float* x, const PartRange& r, uint32_t batch, float4v (&v)[kQuads])
{
#pragma unroll
    for (uint32_t i = 0; i < 4 * kQuads; ++i)
    {
        const uint32_t index = IndexOf(r, batch, i);
        const bool inside = index >= r.begin && index < r.end;
        const float one = x[inside ? index : r.begin];
        v[i / 4][i % 4] = inside ? one : -INFINITY;
    }
}

/// A batch in 16-byte loads, logit by logit where it reaches over an end of the part.
__device__ __forceinline__ void LoadBatch(const float* x, const PartRange& r, uint32_t batch, float4v (&v)[kQuads])
{
    if (IsWhole(r, batch))
    {
#pragma unroll
        for (uint32_t q = 0; q < kQuads; ++q)
        {
            v[q] = *reinterpret_cast<const float4v*>(x + IndexOf(r, batch, 4 * q));
        }
    }
    else if (batch < r.batches)
    {
        LoadOneByOne(x, r, batch, v);
    }
}

/// Counts the logits of a part of a row in steps of the grid, and their masses. A wave has counters of its own in
/// LDS, from a step above the largest logit that it has met; a larger one moves them down, which is rare.
///
/// What bounds it: some 20 vector operations a logit, ten of them in 64 bits, beside the logits' arrival: 500 rows of
/// 151936 in 70 us, 4.4 TB/s, the vector units busy for 0.65 of that at 2.4 GHz, and 0.6 of the LDS operations' time in
/// bank conflicts. Two batches on their way, or three or five waves a SIMD, were slower.
__global__ __launch_bounds__(kBlock, 4) void SampleCountKernel(SampleArgs a)
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
    const RowMode mode = ModeOf(a, row);
    const bool greedy = mode.perUnit < 0.0;
    uint64_t* const masses = massOf[wave];
    uint32_t* const counts = countOf[wave];
    for (int i = lane; i < kSteps; i += kWave)
    {
        masses[i] = 0;
        counts[i] = 0;
    }
    double top = -INFINITY;
    float least = -INFINITY;  // NearPlaces
    bool near = false;
    float most = -INFINITY;   // of the wave; of a greedy row's lane
    uint32_t at = 0;
    const PartRange range = RangeOf(x, begin, end);
    // The next batch is on its way, always in as many loads: under a condition they would all be waited for at once.
    // What lies outside the part's whole quads is read as the nearest of these, and again one by one; without any, as
    // what the workspace begins with.
    const uint32_t firstQuad = range.before != 0 ? 1 : 0;
    const uint32_t quads = (end - begin + range.before) / 4;
    const float4v* const wide = quads > firstQuad ? reinterpret_cast<const float4v*>(x + begin - range.before)
                                                  : reinterpret_cast<const float4v*>(a.steps);
    const uint32_t low = quads > firstQuad ? firstQuad : 0;
    const uint32_t high = quads > firstQuad ? quads - 1 : 0;
    auto request = [&](uint32_t batch, float4v (&to)[kQuads]) {
#pragma unroll
        for (uint32_t q = 0; q < kQuads; ++q)
        {
            to[q] = wide[min(max(batch * (kBatch / 4) + q * kWave + lane, low), high)];
        }
    };
    float4v v[kQuads], next[kQuads];
    request(wave, next);
    for (uint32_t batch = wave; batch < range.batches; batch += kWaves)
    {
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
        {
            v[q] = next[q];
        }
        request(batch + kWaves, next);
        if (!IsWhole(range, batch))
        {
            LoadOneByOne(x, range, batch, v);
        }
        float batchMost = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < 4 * kQuads; ++i)
        {
            v[i / 4][i % 4] = Quiet(v[i / 4][i % 4]);
            batchMost = fmaxf(batchMost, v[i / 4][i % 4]);
        }
        batchMost = fminf(batchMost, 0x1.fffffep127f);
        if (greedy)
        {
            if (batchMost > most)
            {
                most = batchMost;
#pragma unroll
                for (int i = 4 * kQuads - 1; i >= 0; --i)
                {
                    at = Counted(v[i / 4][i % 4]) == batchMost ? IndexOf(range, batch, i) : at;
                }
            }
            continue;
        }
        batchMost = GroupMax<kWave>(batchMost);
        most = fmaxf(most, batchMost);
        if (lane == 0)
        {
            a.batchMost[static_cast<uint64_t>(blockIdx.x) * a.batches + batch] = batchMost;
        }
        if (batchMost == -INFINITY)
        {
            continue;
        }
        const double highest = PlaceOf(batchMost, mode.perUnit).step;
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
            near = NearPlaces(top, mode.perUnit, least);
        }
        // What counts as the largest number may be an infinity.
        if (!near || batchMost == 0x1.fffffep127f)
        {
#pragma unroll 1
            for (uint32_t i = 0; i < 4 * kQuads; ++i)
            {
                const uint32_t index = IndexOf(range, batch, i);
                const bool inside = index >= begin && index < end;
                AddOne(inside ? x[index] : -INFINITY, top, mode.perUnit, masses, counts);
            }
        }
        else if (!mode.weighed)
        {
            AddNearBatch<true, false>(v, top, least, mode.perUnit, masses, counts);
        }
        else if (mode.counted)
        {
            AddNearBatch<true, true>(v, top, least, mode.perUnit, masses, counts);
        }
        else
        {
            AddNearBatch<false, true>(v, top, least, mode.perUnit, masses, counts);
        }
    }
    if (greedy)
    {
        // The wave's largest and its first place.
        const float waveMost = GroupMax<kWave>(most);
        at = most == waveMost && most > -INFINITY ? at : ~0u;
        at = WaveLeast(at);
        most = waveMost;
    }
    if (lane == 0)
    {
        topOf[wave] = top;
        mostOf[wave] = most;
        atOf[wave] = at;
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
        if (mode.weighed)
        {
            a.masses[slot * kSteps + i] = mass;
        }
        if (mode.counted)
        {
            a.counts[slot * kSteps + i] = count;
        }
    }
}

struct PickSpace
{
    uint64_t keys[kListed];
    double unit[kSteps];         // UnitOf
    double upTo[kSteps];         // weights of the steps up to each
    uint64_t masses[kSteps];
    uint32_t counts[kSteps];     // logits up to each, or a bound of them
    uint64_t digitMasses[kDigits];
    uint32_t digitCounts[kDigits];
    uint64_t fewKeys[kFew];
    uint64_t fewMasses[kFew];
    double waveWeights[kPickWaves];
    uint32_t waveCounts[kPickWaves];
    double groupWeights[kGroups];
    uint32_t partShift[kMaxParts];
    unsigned long long partMass[kMaxParts];
    double partWeight[kMaxParts];
    unsigned long long low, high, sum;
    uint32_t listed, few;
    uint32_t stepK, stepP;
};

/// Inclusive sums of both over the threads, in their order.
__device__ __forceinline__ void StepSums(uint32_t& count, double& weight, PickSpace& s)
{
    const uint32_t wave = threadIdx.x / kWave;
    count = WaveInclusive(count);
    weight = WaveInclusive(weight);
    __syncthreads();
    if (threadIdx.x % kWave == kWave - 1)
    {
        s.waveCounts[wave] = count;
        s.waveWeights[wave] = weight;
    }
    __syncthreads();
    uint32_t counts = 0;
    double weights = 0.0;
    for (uint32_t w = 0; w < wave; ++w)
    {
        counts += s.waveCounts[w];
        weights += s.waveWeights[w];
    }
    count += counts;
    weight += weights;
}

/// A row's grid and its threshold.
struct RowGrid
{
    const float* x;
    uint32_t vocab;
    double perUnit, top;
    Place largest;
    double lowest;  // of y - largest, by min-p; -inf: none
};

/// Keys from low to high.
struct KeyRange
{
    uint64_t low, high;
};

constexpr KeyRange kAllKeys{0, ~0ull};

__device__ __forceinline__ bool Reaches(const RowGrid& r, const Place& at)
{
    return (at.step - r.largest.step) + (at.rest - r.largest.rest) >= r.lowest;
}

/// Bounds in f32, a little wide, of the logits in steps first..last.
__device__ __forceinline__ void BoundsOf(const RowGrid& r, uint32_t first, uint32_t last, float& low, float& high)
{
    const double wide = 0.5 + 1e-6 + 1e-9 * fabs(r.top);
    low = __double2float_rd((r.top - last - wide) / r.perUnit);
    high = __double2float_ru((r.top - first + wide) / r.perUnit);
    // +inf is not above the last number, as which it counts.
    high = high >= 0x1.fffffep127f ? INFINITY : high;
}

/// Calls use(key, step, mass) for a row's logits in steps first..last with keys in keys.low..high, by all threads.
/// Bounds in f32, a little wide, tell which of a thread's logits of a round may be meant; those are placed one by one
/// (a copy of that for each of them filled the instruction cache). kAhead: 16-byte loads of a thread in a round.
template <uint32_t kAhead, typename Use>
__device__ __forceinline__ void ForSteps(const RowGrid& r, uint32_t first, uint32_t last, KeyRange keys, Use use)
{
    float low, high;
    BoundsOf(r, first, last, low, high);
    low = fmaxf(low, KeyValue(keys.low));
    high = KeyValue(keys.high) < 0x1.fffffep127f ? fminf(high, KeyValue(keys.high)) : high;
    const uint32_t head = min((4u - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(r.x) / 4 % 4)) % 4u, r.vocab);
    const uint32_t quads = (r.vocab - head) / 4;
    const uint32_t edges = r.vocab - 4 * quads;  // before the first quad and behind the last
    float4v v[kAhead], next[kAhead];  // quads of a round; the next round's are on their way
    auto load = [&](uint32_t from) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
        {
            const uint32_t quad = min(from + i * kPickBlock + threadIdx.x, quads - 1);
            next[i] = *reinterpret_cast<const float4v*>(r.x + head + 4 * quad);
        }
    };
    if (quads > 0)
    {
        load(0);
    }
    // The first round is that of the edges.
    uint32_t may = threadIdx.x < edges ? 1u : 0u;
    bool edge = true;
    const uint32_t edgeIndex = threadIdx.x < head ? threadIdx.x : threadIdx.x + 4 * quads;
    v[0][0] = r.x[threadIdx.x < edges ? edgeIndex : 0];
    uint32_t from = 0;
    while (true)
    {
        while (may != 0)
        {
            const uint32_t bit = __ffs(static_cast<int>(may)) - 1;
            may &= may - 1;
            float logit = v[0][0];
#pragma unroll
            for (uint32_t i = 1; i < 4 * kAhead; ++i)
            {
                logit = bit == i ? v[i / 4][i % 4] : logit;
            }
            const uint32_t at = edge ? edgeIndex : head + 4 * (from + bit / 4 * kPickBlock + threadIdx.x) + bit % 4;
            const float x = Counted(logit);
            const Place place = PlaceOf(x, r.perUnit);
            const double d = r.top - place.step;
            const uint64_t key = OrderKey(x, at);
            if (x > -INFINITY && d >= first && d <= last && key >= keys.low && key <= keys.high)
            {
                use(key, static_cast<uint32_t>(d), MassOf(place.rest));
            }
        }
        from += edge ? 0 : kPickBlock * kAhead;
        edge = false;
        if (from >= quads)
        {
            break;
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
        {
            v[i] = next[i];
        }
        load(from + kPickBlock * kAhead);
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
        {
            const bool there = from + i * kPickBlock + threadIdx.x < quads;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
            {
                may |= there && v[i][e] >= low && v[i][e] <= high ? 1u << (4 * i + e) : 0u;
            }
        }
    }
}

/// Lists the keys of those (at most kListed, as the caller has seen).
template <uint32_t kAhead>
__device__ __forceinline__ void ListSteps(const RowGrid& r, uint32_t first, uint32_t last, KeyRange keys, PickSpace& s)
{
    __syncthreads();
    if (threadIdx.x == 0)
    {
        s.listed = 0;
    }
    __syncthreads();
    ForSteps<kAhead>(r, first, last, keys, [&](uint64_t key, uint32_t, uint64_t) {
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < kListed)
        {
            s.keys[at] = key;
        }
    });
    __syncthreads();
}

/// The last of what is kept, and the mass of all of it.
struct Cut
{
    uint64_t key;
    uint64_t mass;
};

/// Of 256 equal ranges from the high end of keys down, `shift` says how many bits of a distance they leave.
__device__ __forceinline__ int DigitShift(KeyRange keys)
{
    return max(56 - __clzll(static_cast<long long>(keys.high - keys.low)), 0);
}

__device__ __forceinline__ KeyRange DigitOf(KeyRange keys, uint32_t which, int shift)
{
    keys.high -= static_cast<uint64_t>(which) << shift;
    const uint64_t span = (1ull << shift) - 1;
    keys.low = keys.high - keys.low > span ? keys.high - span : keys.low;
    return keys;
}

/// The last such range that begins before both limits, by the counts and masses of all (the first after `above` items
/// of `aboveMass`), and what it begins after; ~0: none. Every wave finds the same, four ranges a lane.
struct Digit
{
    uint32_t which, count, above;
    uint64_t aboveMass;
};

__device__ __forceinline__ Digit LastDigit(uint32_t most, uint64_t limit, uint32_t above, uint64_t aboveMass,
                                           const PickSpace& s)
{
    const uint32_t lane = threadIdx.x % kWave;
    constexpr uint32_t kPer = kDigits / kWave;
    uint32_t c[kPer];
    uint64_t m[kPer];
    uint32_t ofLane = 0;
    uint64_t massOfLane = 0;
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e)
    {
        c[e] = s.digitCounts[lane * kPer + e];
        m[e] = s.digitMasses[lane * kPer + e];
        ofLane += c[e];
        massOfLane += m[e];
    }
    uint32_t before = above + WaveInclusive(ofLane) - ofLane;
    uint64_t massBefore = aboveMass + WaveInclusive(massOfLane) - massOfLane;
    Digit last{~0u, 0, above, aboveMass};
#pragma unroll
    for (uint32_t e = 0; e < kPer; ++e)
    {
        if (c[e] > 0 && before < most && massBefore < limit)
        {
            last = Digit{lane * kPer + e, c[e], before, massBefore};
        }
        before += c[e];
        massBefore += m[e];
    }
    const uint64_t has = __ballot(last.which != ~0u);
    const int owner = has != 0 ? 63 - __clzll(static_cast<long long>(has)) : 0;
    return Digit{OfLane(last.which, owner), OfLane(last.count, owner), OfLane(last.above, owner),
                 OfLane(last.aboveMass, owner)};
}

/// Of `n` items in falling order of their keys (which differ), those that have fewer than `most` before them and
/// less than `limit` of mass: the last one's key, and their mass. item(i, key, mass) says whether there is one; there
/// are `some` at most.
///
/// All keys are in `keys`. That is taken apart into 256 equal ranges, the one with the last item is found from
/// counts and masses of all, and so on between the smallest and the largest there, until a wave can look at the rest
/// one by one.
template <typename Item>
__device__ __forceinline__ Cut LastKept(uint32_t n, uint32_t some, Item item, uint32_t most, uint64_t limit,
                                        KeyRange keys, PickSpace& s)
{
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t above = 0;
    uint64_t aboveMass = 0;
    bool few = min(n, some) <= kFew;
    bool narrow = true;  // the range is not worth a look for its ends
    while (true)
    {
        __syncthreads();
        if (threadIdx.x == 0)
        {
            s.low = ~0ull;
            s.high = 0;
            s.few = 0;
        }
        for (uint32_t i = threadIdx.x; i < kDigits; i += kPickBlock)
        {
            s.digitCounts[i] = 0;
            s.digitMasses[i] = 0;
        }
        __syncthreads();
        if (!few && !narrow)
        {
            uint64_t least = ~0ull;
            uint64_t largest = 0;
            for (uint32_t i = threadIdx.x; i < n; i += kPickBlock)
            {
                uint64_t key, mass;
                if (item(i, key, mass) && key >= keys.low && key <= keys.high)
                {
                    least = least < key ? least : key;
                    largest = largest > key ? largest : key;
                }
            }
            least = WaveLeast(least);
            largest = ~WaveLeast(~largest);
            if (lane == 0 && least <= largest)
            {
                atomicMin(&s.low, static_cast<unsigned long long>(least));
                atomicMax(&s.high, static_cast<unsigned long long>(largest));
            }
            __syncthreads();
            keys = KeyRange{s.low, s.high};
        }
        narrow = false;
        if (few)
        {
            for (uint32_t i = threadIdx.x; i < n; i += kPickBlock)
            {
                uint64_t key, mass;
                if (item(i, key, mass) && key >= keys.low && key <= keys.high)
                {
                    const uint32_t at = atomicAdd(&s.few, 1u);
                    s.fewKeys[at] = key;
                    s.fewMasses[at] = mass;
                }
            }
            __syncthreads();
            // Every wave finds the same.
            const uint32_t count = s.few;
            const uint64_t key = lane < count ? s.fewKeys[lane] : 0;
            const uint64_t mass = lane < count ? s.fewMasses[lane] : 0;
            uint32_t before = above;
            uint64_t massBefore = aboveMass;
            for (uint32_t j = 0; j < count; ++j)
            {
                const bool is = s.fewKeys[j] > key;
                before += is ? 1u : 0u;
                massBefore += is ? s.fewMasses[j] : 0;
            }
            const bool kept = lane < count && before < most && massBefore < limit;
            // The last one kept is the smallest of them.
            const uint64_t last = WaveLeast(kept ? key : ~0ull);
            const uint64_t is = __ballot(kept && key == last);
            if (is == 0)
            {
                return Cut{~0ull, aboveMass};
            }
            return Cut{last, OfLane(massBefore + mass, __ffsll(static_cast<unsigned long long>(is)) - 1)};
        }
        const int shift = DigitShift(keys);
        for (uint32_t i = threadIdx.x; i < n; i += kPickBlock)
        {
            uint64_t key, mass;
            if (item(i, key, mass) && key >= keys.low && key <= keys.high)
            {
                const uint32_t digit = static_cast<uint32_t>((keys.high - key) >> shift);
                atomicAdd(&s.digitCounts[digit], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.digitMasses[digit]), mass);
            }
        }
        __syncthreads();
        const Digit digit = LastDigit(most, limit, above, aboveMass, s);
        if (digit.which == ~0u)
        {
            return Cut{~0ull, aboveMass};
        }
        few = digit.count <= kFew;
        above = digit.above;
        aboveMass = digit.aboveMass;
        keys = DigitOf(keys, digit.which, shift);
    }
}

/// In a step of more logits than are listed: takes `keys` to a range that has the last of what is kept, of few enough
/// to list, and returns what that begins after (which ~0: nothing is kept). Range by range of 256 and between the
/// smallest and the largest key there, with a pass over the row for each.
template <uint32_t kAhead>
__device__ __forceinline__ Digit NarrowStep(const RowGrid& r, uint32_t d, uint32_t most, uint64_t limit, KeyRange& keys,
                                            PickSpace& s)
{
    Digit last{0, ~0u, 0, 0};
    while (last.count > kListed)
    {
        __syncthreads();
        if (threadIdx.x == 0)
        {
            s.low = ~0ull;
            s.high = 0;
        }
        for (uint32_t i = threadIdx.x; i < kDigits; i += kPickBlock)
        {
            s.digitCounts[i] = 0;
            s.digitMasses[i] = 0;
        }
        __syncthreads();
        const int shift = DigitShift(keys);
        uint64_t least = ~0ull;
        uint64_t largest = 0;
        ForSteps<kAhead>(r, d, d, keys, [&](uint64_t key, uint32_t, uint64_t mass) {
            if (Reaches(r, PlaceOf(KeyValue(key), r.perUnit)))
            {
                const uint32_t digit = static_cast<uint32_t>((keys.high - key) >> shift);
                atomicAdd(&s.digitCounts[digit], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.digitMasses[digit]), mass);
                least = least < key ? least : key;
                largest = largest > key ? largest : key;
            }
        });
        least = WaveLeast(least);
        largest = ~WaveLeast(~largest);
        if (threadIdx.x % kWave == 0 && least <= largest)
        {
            atomicMin(&s.low, static_cast<unsigned long long>(least));
            atomicMax(&s.high, static_cast<unsigned long long>(largest));
        }
        __syncthreads();
        last = LastDigit(most, limit, last.above, last.aboveMass, s);
        if (last.which == ~0u)
        {
            return last;
        }
        keys = DigitOf(keys, last.which, shift);
        keys.low = keys.low > s.low ? keys.low : s.low;
        keys.high = keys.high < s.high ? keys.high : s.high;
    }
    return last;
}

/// What the launches of a row's end do: everything; or the steps and what of them is to be listed, and then, with the
/// list made by workgroups all over the GPU, the rest.
enum PickPhase
{
    kPickAll,
    kPickSteps,
    kPickToken
};

/// Decides a row: where the cuts lie in the steps' counts and masses, and which token the number lands on. Where the
/// logits of the steps down to the cut are few they are listed, in one pass over the row; else the step of the cut is,
/// and the token is looked for in the part of the row that the parts' masses name.
///
/// What bounds it: a workgroup's chain of searches, each some passes over the list between barriers (1.3 us where a
/// wave can look at all, 4 for thousands); where the list does not do, 64-bit work for half a part of the row (10 us of
/// 30, where 500 rows have 4 parts); and where a cut's step is not to be listed, a pass over the row for each range of
/// it (500 rows of 151936 of standard deviation 0.75 take 311 us in all, of 2.5 with some that stand out 131; by digits
/// of the keys, eight passes, the former took 980). Two workgroups fit a CU at 123 registers: with more loads on their
/// way in such passes, 169 and one, 500 rows with lists take 143 us.
template <PickPhase kPhase>
__global__ __launch_bounds__(kPickBlock, kPhase == kPickAll ? 1 : 4) void SamplePickKernel(SampleArgs a)
{
    __shared__ PickSpace s;
    // Without lists made before, passes over the row are the rule; else the registers of more loads on their way would
    // take the second workgroup's place on a CU.
    constexpr uint32_t kAhead = kPhase == kPickAll ? 4 : 1;
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = threadIdx.x / kWave;
    const uint64_t slot = static_cast<uint64_t>(row) * a.parts;

    // Every wave looks at the parts, a lane each.
    static_assert(kMaxParts == kWave, "a lane for each part");
    PartHead head = a.heads[slot + min(lane, a.parts - 1)];
    const RowMode mode = ModeOf(a, row);
    const float topP = a.topPs != nullptr ? a.topPs[row] : 1.0f;
    const float minP = a.minPs != nullptr ? a.minPs[row] : 0.0f;
    const double given = a.randoms[row];
    const double number = given > 0.0 ? given : 0.0;
    if (lane >= a.parts)
    {
        head = PartHead{-INFINITY, -INFINITY, ~0u};
    }
    const float most = GroupMax<kWave>(head.most);
    double top = head.top;
    top = WaveJoin(top, [](double x, double y) { return fmax(x, y); });
    RowSteps* const kept = kPhase == kPickAll ? nullptr : a.steps + row;
    if (kPhase == kPickSteps && threadIdx.x == 0)
    {
        kept->top = top;
        kept->first = 1;
        kept->last = 0;
        kept->listed = 0;
    }
    if (kPhase == kPickSteps && (most == -INFINITY || mode.perUnit < 0.0))
    {
        return;
    }
    if (most == -INFINITY || mode.perUnit < 0.0)
    {
        uint32_t at = head.most == most ? head.at : ~0u;
        at = WaveLeast(at);
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
    r.perUnit = mode.perUnit;
    r.top = top;
    r.largest = PlaceOf(most, mode.perUnit);
    r.lowest = -INFINITY;
    static_assert(kPickBlock == kSteps, "a thread a step");
    const uint32_t d = threadIdx.x;
    if (wave == 0)
    {
        const double by = top - head.top;
        s.partShift[lane] = by < kSteps ? static_cast<uint32_t>(by) : kSteps;  // a part with nothing: all
        s.partMass[lane] = 0;
        if (lane == 0)
        {
            s.stepK = kSteps - 1;
            s.stepP = kSteps - 1;
        }
    }
    s.unit[d] = UnitOf(d);
    __syncthreads();

    uint32_t count = 0;
    double weight = 0.0;
    if constexpr (kPhase == kPickToken)
    {
        count = kept->counts[d];
        weight = kept->upTo[d];
    }
    else
    {
        // The row's steps, a thread each, several parts' on their way at a time.
        uint64_t mass = 0;
        constexpr uint32_t kDeep = 20;
        for (uint32_t p0 = 0; p0 < a.parts; p0 += kDeep)
        {
            uint64_t m[kDeep];
            uint32_t c[kDeep];
    #pragma unroll
            for (uint32_t i = 0; i < kDeep; ++i)
            {
                const uint32_t p = min(p0 + i, a.parts - 1);
                const uint32_t shift = s.partShift[p];
                const uint64_t from = (slot + p) * kSteps + (d >= shift ? d - shift : 0);
                const bool is = p0 + i < a.parts && d >= shift;
                m[i] = is && mode.weighed ? a.masses[from] : 0;
                c[i] = is && mode.counted ? a.counts[from] : 0;
            }
    #pragma unroll
            for (uint32_t i = 0; i < kDeep; ++i)
            {
                mass += m[i];
                count += c[i];
            }
        }
        weight = static_cast<double>(mass) * s.unit[d];
        if (!mode.counted)
        {
            // A bound: a logit's mass is at least 2^(-3/32) of a unit's.
            count = static_cast<uint32_t>(static_cast<double>(mass) * (0x1p-38 * 1.0672)) + (mass != 0 ? 1u : 0u);
        }
        StepSums(count, weight, s);
    }
    s.counts[d] = count;
    s.upTo[d] = weight;
    if (kPhase == kPickSteps)
    {
        kept->counts[d] = count;
        kept->upTo[d] = weight;
    }
    __syncthreads();
    // The step in which the first k end.
    uint32_t stepK = kSteps - 1;
    uint32_t left = ~0u;  // of the first k in that step
    bool wholeK = true;
    if (mode.counted)
    {
        const uint32_t k = min(static_cast<uint32_t>(mode.topK), s.counts[kSteps - 1]);
        if (count >= k && (d == 0 || s.counts[d - 1] < k))  // one thread
        {
            s.stepK = d;
        }
        __syncthreads();
        stepK = s.stepK;
        left = k - (stepK > 0 ? s.counts[stepK - 1] : 0);
        wholeK = s.counts[stepK] == k;
    }
    auto countOf = [&](uint32_t step) { return s.counts[step] - (step > 0 ? s.counts[step - 1] : 0); };
    auto weightBefore = [&](uint32_t step) { return step > 0 ? s.upTo[step - 1] : 0.0; };
    if (kPhase != kPickSteps && !mode.weighed && s.counts[stepK] > kListed)
    {
        // Counted alone, and too many for the list after all: the masses by a pass of their own.
        s.masses[d] = 0;
        __syncthreads();
        ForSteps<kAhead>(r, 0, stepK, kAllKeys, [&](uint64_t, uint32_t step, uint64_t one) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.masses[step]), one);
        });
    }

    // In turn, where each is needed: the masses of a list that has all of the first k; the cut of these; the cut of
    // all that is kept; and the token among what is listed.
    enum Task
    {
        kMassesOfK,
        kCutOfK,
        kCutOfAll,
        kToken
    };
    const bool narrow = topP < 1.0f;
    Task task = !mode.weighed ? kMassesOfK : narrow && !wholeK ? kCutOfK : kCutOfAll;
    uint32_t listFirst = 1;  // steps that are listed: none
    uint32_t listLast = 0;
    if constexpr (kPhase == kPickToken)
    {
        listFirst = kept->first;
        listLast = kept->last;
        const uint32_t listed = listFirst <= listLast ? min(kept->listed, a.listRoom) : 0;
        const uint64_t* const keys = a.listKeys + static_cast<uint64_t>(row) * a.listRoom;
        for (uint32_t i = threadIdx.x; i < listed; i += kPickBlock)
        {
            s.keys[i] = keys[i];
        }
        if (threadIdx.x == 0)
        {
            s.listed = listed;
        }
        __syncthreads();
    }
    uint32_t step = 0;       // of the cut of all
    bool whole = false;      // nothing of that step is cut off
    bool all = false;        // all that is kept is listed
    double ofK = 0.0;
    double share = INFINITY;
    double total = 0.0;
    uint32_t stepP = kSteps;
    Cut cut{0, 0};
    Cut token{0, 0};
    while (true)
    {
        uint32_t from = 1;  // to be listed
        uint32_t to = 0;
        if (task == kMassesOfK)
        {
            to = s.counts[stepK] <= kListed ? stepK : 0;
            from = s.counts[stepK] <= kListed ? 0 : 1;
        }
        else if (task == kCutOfK)
        {
            to = countOf(stepK) <= kListed ? stepK : 0;
            from = countOf(stepK) <= kListed ? stepK : 1;
        }
        else if (task == kCutOfAll)
        {
            if (narrow)
            {
                // The step in which top-p's share of the first k's weight is reached.
                share = static_cast<double>(topP) * (wholeK ? s.upTo[stepK] : ofK);
                auto reached = [&](double sum) { return sum > 0.0 && sum >= share; };
                if (reached(weight) && (d == 0 || !reached(s.upTo[d - 1])))
                {
                    s.stepP = d;
                }
                __syncthreads();
                stepP = min(s.stepP, stepK);
            }
            // The step in which min-p's bound lies; the largest always reaches it.
            uint32_t stepM = kSteps;
            if (minP > 0.0f)
            {
                const double lowest = fmin(8.0 * log2(static_cast<double>(minP)), 0.0);
                const double by = top - rint(r.largest.step + r.largest.rest + lowest);
                stepM = by < kSteps ? static_cast<uint32_t>(fmax(by, top - r.largest.step)) : kSteps;
                r.lowest = stepM <= min(stepK, stepP) ? lowest : -INFINITY;
            }
            step = min(min(stepK, stepP), stepM);
            whole = step != stepP && step != stepM && (step != stepK || wholeK);
            const bool have = listFirst == 0 && step <= listLast;
            all = have || s.counts[step] <= kListed;
            if (!have && (all || (!whole && countOf(step) <= kListed)))
            {
                from = all ? 0 : step;
                to = step;
            }
            total = s.upTo[step];
        }
        if constexpr (kPhase == kPickSteps)
        {
            if (threadIdx.x == 0)
            {
                kept->perUnit = r.perUnit;
                BoundsOf(r, from, to, kept->low, kept->high);
                kept->first = from;
                kept->last = to;
            }
            return;
        }
        if (from <= to && !(listFirst <= from && to <= listLast))
        {
            ListSteps<kAhead>(r, from, to, kAllKeys, s);
            listFirst = from;
            listLast = to;
        }
        if (task == kMassesOfK)
        {
            if (from <= to)
            {
                s.masses[d] = 0;
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
                {
                    const Place place = PlaceOf(KeyValue(s.keys[i]), r.perUnit);
                    atomicAdd(reinterpret_cast<unsigned long long*>(&s.masses[static_cast<uint32_t>(top - place.step)]),
                              MassOf(place.rest));
                }
            }
            __syncthreads();
            uint32_t unused = 0;
            weight = static_cast<double>(s.masses[d]) * s.unit[d];
            StepSums(unused, weight, s);
            s.upTo[d] = weight;
            __syncthreads();
            task = narrow && !wholeK ? kCutOfK : kCutOfAll;
            continue;
        }
        // What is looked for: items of step `of` (or, for the token, all that are kept).
        const uint32_t of = task == kCutOfK ? stepK : step;
        uint32_t atMost = ~0u;
        double limit = INFINITY;
        bool needed = true;
        if (task == kCutOfK)
        {
            atMost = left;
        }
        else if (task == kCutOfAll)
        {
            needed = !whole;
            atMost = minP > 1.0f ? 1u : step == stepK ? left : ~0u;
            // A share that is reached before this step's first, by a rounding, still keeps that one.
            limit = step == stepP ? fmax((share - weightBefore(step)) / s.unit[step], 0x1p-30) : INFINITY;
        }
        auto item = [&](uint32_t i, uint64_t& key, uint64_t& ofKey) {
            key = s.keys[i];
            const Place place = PlaceOf(KeyValue(key), r.perUnit);
            const uint32_t dist = static_cast<uint32_t>(top - place.step);
            ofKey = MassOf(place.rest);
            if (task != kToken)
            {
                return dist == of && Reaches(r, place);
            }
            // By falling ~index, weights as whole numbers, whose sums are exact.
            const bool kept = dist < of || (dist == of && key >= cut.key);
            ofKey = static_cast<uint64_t>(rint(static_cast<double>(ofKey) * (s.unit[dist] * kFixed)));
            key &= 0xFFFFFFFFull;
            return kept && ofKey != 0;
        };
        if (task == kToken)
        {
            __syncthreads();
            if (threadIdx.x == 0)
            {
                s.sum = 0;
            }
            __syncthreads();
            uint64_t sum = 0;
            for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
            {
                uint64_t key, fixed;
                sum += item(i, key, fixed) ? fixed : 0;
            }
            sum = WaveSum(sum);
            if (lane == 0 && sum != 0)
            {
                atomicAdd(&s.sum, static_cast<unsigned long long>(sum));
            }
            __syncthreads();
            // The first token whose sum is past the number's share is the last that begins at or before it.
            limit = floor(number * static_cast<double>(s.sum)) + 1.0;
        }
        Cut found{0, 0};
        if (needed)
        {
            const uint64_t below = limit < 0x1p63 ? static_cast<uint64_t>(ceil(limit)) : ~0ull;
            // Of the token's search keys are indices, else those of the step's logits.
            uint32_t some = task != kToken ? countOf(of)
                            : mode.counted ? min(s.counts[of], static_cast<uint32_t>(mode.topK))
                                           : s.counts[of];
            KeyRange keys{static_cast<uint32_t>(~(a.vocab - 1)), 0xFFFFFFFFull};
            const bool inList = task == kToken || (listFirst <= of && of <= listLast);
            if (task != kToken && inList && min(s.listed, some) <= kFew)
            {
                keys = kAllKeys;
            }
            else if (task != kToken)
            {
                float least, largest;
                BoundsOf(r, of, of, least, largest);
                keys.low = static_cast<uint64_t>(OrderBits(least)) << 32;
                keys.high |= static_cast<uint64_t>(OrderBits(largest)) << 32;
            }
            Digit before{0, 0, 0, 0};
            if (!inList)
            {
                before = NarrowStep<kAhead>(r, of, atMost, below, keys, s);
                some = before.count;
                listFirst = 1;
                listLast = 0;
                if (before.which != ~0u)
                {
                    ListSteps<kAhead>(r, of, of, keys, s);
                }
            }
            found = Cut{~0ull, 0};
            if (before.which != ~0u)
            {
                found = LastKept(s.listed, some, item, atMost - before.above, below - before.aboveMass, keys, s);
            }
            found.mass += before.aboveMass;
        }
        if (task == kCutOfK)
        {
            ofK = weightBefore(stepK) + static_cast<double>(found.mass) * s.unit[stepK];
            task = kCutOfAll;
        }
        else if (task == kCutOfAll)
        {
            cut = found;
            total = whole ? total : weightBefore(step) + static_cast<double>(cut.mass) * s.unit[step];
            if (!all)
            {
                break;
            }
            task = kToken;
        }
        else
        {
            token = found;
            break;
        }
    }

    uint32_t index = ~static_cast<uint32_t>(token.key);
    double ofToken = 0.0;  // its weight, in one thread
    bool writes = false;
    if (all)
    {
        for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
        {
            if ((s.keys[i] & 0xFFFFFFFFull) == token.key)
            {
                const Place place = PlaceOf(KeyValue(s.keys[i]), r.perUnit);
                ofToken = static_cast<double>(MassOf(place.rest)) * s.unit[static_cast<uint32_t>(top - place.step)];
                writes = true;
            }
        }
    }
    else
    {
        // Kept: the steps before, and of this one the keys from the cut on.
        auto weightAt = [&](float v, uint32_t at) {
            const float x = Counted(v);
            const Place place = PlaceOf(x, r.perUnit);
            const double dist = top - place.step;
            const bool kept = dist < static_cast<double>(step) ||
                              (dist == static_cast<double>(step) && OrderKey(x, at) >= cut.key);
            return kept ? static_cast<double>(MassOf(place.rest)) * s.unit[static_cast<uint32_t>(dist)] : 0.0;
        };
        // The same of logits of which none is far, with fewer operations (AddNearBatch): by the cut's own logit.
        float least;
        const bool near = NearPlaces(top, r.perUnit, least);
        const uint32_t topStep = static_cast<uint32_t>(__double_as_longlong(top + kWhole));
        const bool none = cut.key == ~0ull;  // of the step of the cut
        const uint32_t lastStep = none ? step - 1 : step;
        const float cutLogit = whole || none ? -INFINITY : KeyValue(cut.key);
        const uint32_t cutIndex = ~static_cast<uint32_t>(cut.key);
        uint32_t begin = 0;
        uint32_t end = a.vocab;
        // Adds those of four logits, kWave apart.
        auto nearWeights = [&](const float (&v)[4], uint32_t at, double& sum) {
            float x[4];
            uint32_t dist[4];
            double rest[4], mass[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
            {
                x[e] = Counted(v[e]);
                const double y = static_cast<double>(fmaxf(x[e], least));
                const double place = WholeOf(y, r.perUnit);
                dist[e] = topStep - static_cast<uint32_t>(__double_as_longlong(place));
                rest[e] = fma(y, r.perUnit, -(place - kWhole));
            }
            MassSums<4>(rest, mass);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
            {
                const uint32_t index = at + e * kWave;
                const bool kept = index < end && dist[e] <= lastStep &&
                                  (x[e] > cutLogit || (x[e] == cutLogit && index <= cutIndex));
                const double weight = (mass[e] - 0x1p52) * s.unit[min(dist[e], static_cast<uint32_t>(kSteps - 1))];
                sum += kept ? weight : 0.0;
            }
        };
        const double reach = number * total;
        double passed = 0.0;
        if (mode.weighed)
        {
            // What each part has of it: the steps before from its masses, this one's kept logits by a look at them.
            __syncthreads();
            const uint32_t until = whole ? step + 1 : step;
            for (uint32_t p0 = wave; p0 < a.parts; p0 += 2 * kPickWaves)
            {
                // Two parts' at a time.
                uint64_t m[2][kSteps / kWave];
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
                {
                    const uint32_t p = min(p0 + h * kPickWaves, a.parts - 1);
                    const uint32_t shift = s.partShift[p];
#pragma unroll
                    for (uint32_t j = 0; j < kSteps / kWave; ++j)
                    {
                        const uint32_t i = j * kWave + lane;
                        m[h][j] = i >= shift && i < until ? a.masses[(slot + p) * kSteps + i - shift] : 0;
                    }
                }
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
                {
                    double sum = 0.0;
#pragma unroll
                    for (uint32_t j = 0; j < kSteps / kWave; ++j)
                    {
                        sum += static_cast<double>(m[h][j]) * s.unit[j * kWave + lane];
                    }
                    sum = WaveSum(sum);
                    if (lane == 0 && p0 + h * kPickWaves < a.parts)
                    {
                        s.partWeight[p0 + h * kPickWaves] = sum;
                    }
                }
            }
            if (!whole)
            {
                auto use = [&](uint64_t key, uint64_t one) {
                    if (key >= cut.key)
                    {
                        atomicAdd(&s.partMass[~static_cast<uint32_t>(key) / a.partLength],
                                  static_cast<unsigned long long>(one));
                    }
                };
                if (listFirst <= step && step <= listLast)
                {
                    for (uint32_t i = threadIdx.x; i < s.listed; i += kPickBlock)
                    {
                        const Place place = PlaceOf(KeyValue(s.keys[i]), r.perUnit);
                        if (top - place.step == static_cast<double>(step))
                        {
                            use(s.keys[i], MassOf(place.rest));
                        }
                    }
                }
                else
                {
                    ForSteps<kAhead>(r, step, step, KeyRange{cut.key, ~0ull},
                                     [&](uint64_t key, uint32_t, uint64_t one) { use(key, one); });
                }
            }
            __syncthreads();
            // The first part that reaches past the number's share, else the last with anything kept.
            uint32_t part = 0;
            double upToPart = 0.0;
            for (uint32_t p = 0; p < a.parts; ++p)
            {
                const double ofPart = s.partWeight[p] + static_cast<double>(s.partMass[p]) * s.unit[step];
                if (ofPart > 0.0)
                {
                    part = p;
                    passed = upToPart;
                    upToPart += ofPart;
                    if (upToPart > reach)
                    {
                        break;
                    }
                }
            }
            begin = part * a.partLength;
            end = min(begin + a.partLength, a.vocab);
        }
        // Sums of groups of logits, and the first group that reaches past it, else the last with anything kept.
        constexpr uint32_t kAtOnce = 4;  // groups of a wave
        const uint32_t groups = (end - begin + kGroup - 1) / kGroup;
        uint32_t group = 0;
        double sum = passed;
        bool past = false;
        for (uint32_t first = 0; first < groups && !past; first += kGroups)
        {
            const uint32_t here = min(groups - first, kGroups);
            __syncthreads();
            for (uint32_t i0 = wave; i0 < here; i0 += kAtOnce * kPickWaves)
            {
                float v[kAtOnce][kPickLoads];
#pragma unroll
                for (uint32_t b = 0; b < kAtOnce; ++b)
                {
#pragma unroll
                    for (uint32_t j = 0; j < kPickLoads; ++j)
                    {
                        const uint32_t at = begin + (first + i0 + b * kPickWaves) * kGroup + lane + j * kWave;
                        v[b][j] = r.x[min(at, end - 1)];
                    }
                }
                double own[kAtOnce];
#pragma unroll
                for (uint32_t b = 0; b < kAtOnce; ++b)
                {
                    const uint32_t i = i0 + b * kPickWaves;
                    const uint32_t at = begin + (first + i) * kGroup + lane;
                    own[b] = 0.0;
                    if (near)
                    {
                        if (i < here)
                        {
#pragma unroll
                            for (uint32_t j = 0; j < kPickLoads; j += 4)
                            {
                                nearWeights({v[b][j], v[b][j + 1], v[b][j + 2], v[b][j + 3]}, at + j * kWave, own[b]);
                            }
                        }
                    }
                    else
                    {
#pragma unroll 1
                        for (uint32_t j = 0; j < kPickLoads; ++j)
                        {
                            const uint32_t here1 = at + j * kWave;
                            own[b] += i < here && here1 < end ? weightAt(r.x[here1], here1) : 0.0;
                        }
                    }
                }
#pragma unroll
                for (uint32_t b = 0; b < kAtOnce; ++b)
                {
                    const double ofGroup = WaveSum(own[b]);
                    if (lane == 0 && i0 + b * kPickWaves < here)
                    {
                        s.groupWeights[i0 + b * kPickWaves] = ofGroup;
                    }
                }
            }
            __syncthreads();
            // Every wave finds the same, a group a lane.
            for (uint32_t i0 = 0; i0 < here && !past; i0 += kWave)
            {
                const double ofGroup = i0 + lane < here ? s.groupWeights[i0 + lane] : 0.0;
                const double upToGroup = WaveInclusive(ofGroup);
                const uint64_t kept = __ballot(ofGroup > 0.0);
                const uint64_t over = __ballot(ofGroup > 0.0 && sum + upToGroup > reach);
                if (kept != 0)
                {
                    const int which = over != 0 ? __ffsll(static_cast<unsigned long long>(over)) - 1
                                                : 63 - __clzll(static_cast<long long>(kept));
                    group = first + i0 + which;
                    passed = sum + OfLane(upToGroup - ofGroup, which);
                }
                past = over != 0;
                sum += OfLane(upToGroup, kWave - 1);
            }
        }
        if (wave != 0)
        {
            return;
        }
        // The first of its logits that reaches past it, else its last that is kept.
        const uint32_t first = begin + group * kGroup;
#pragma unroll 1
        for (uint32_t j = 0; j < kPickLoads; ++j)
        {
            const uint32_t at = first + j * kWave + lane;
            const double own = at < end ? weightAt(r.x[at], at) : 0.0;
            const double upToOwn = WaveInclusive(own);
            const uint64_t kept = __ballot(own > 0.0);
            const uint64_t over = __ballot(own > 0.0 && passed + upToOwn > reach);
            if (kept != 0)
            {
                const int which = over != 0 ? __ffsll(static_cast<unsigned long long>(over)) - 1
                                            : 63 - __clzll(static_cast<long long>(kept));
                index = first + j * kWave + which;
                ofToken = OfLane(own, which);
            }
            if (over != 0)
            {
                break;
            }
            passed += OfLane(upToOwn, kWave - 1);
        }
        writes = lane == 0;
    }
    if (writes)
    {
        a.tokens[row] = static_cast<int32_t>(index);
        if (a.logprobs != nullptr)
        {
            a.logprobs[row] = static_cast<float>(log(ofToken / total));
        }
    }
}

/// Lists the logits of the rows' chosen steps, kBatches batches a wave. Batches whose largest logit is below the
/// steps are not read: tokens that stand out of a row are in few of them.
///
/// What bounds it: the arrival of the others, at one CU if the workgroup that decides the row listed them (608 KB in
/// 13 us). A batch a wave where all fit the GPU at about once, else two: one row 27.5 us in all with one and 28.6 with
/// two, 61 rows 53.3 and 54.5, 500 134.3 and 131.2 (with four 135.2).
template <uint32_t kBatches>
__global__ __launch_bounds__(kBlock) void SampleListKernel(SampleArgs a)
{
    const uint32_t row = blockIdx.y;
    RowSteps* const kept = a.steps + row;
    const uint32_t first = kept->first;
    const uint32_t last = kept->last;
    if (first > last)
    {
        return;
    }
    const uint32_t wave = blockIdx.x * kWaves + threadIdx.x / kWave;
    const uint32_t perPart = (a.batches + kBatches - 1) / kBatches;  // waves
    const uint32_t part = wave / perPart;
    if (part >= a.parts)
    {
        return;
    }
    const float* const x = a.logits + row * a.stride;
    uint64_t* const keys = a.listKeys + static_cast<uint64_t>(row) * a.listRoom;
    const double perUnit = kept->perUnit;
    const double top = kept->top;
    const float low = kept->low;
    const float high = kept->high;
    const uint64_t slot = static_cast<uint64_t>(row) * a.parts + part;
    const uint32_t begin = part * a.partLength;
    const PartRange range = RangeOf(x, begin, min(begin + a.partLength, a.vocab));
    const uint32_t batch0 = (wave - part * perPart) * kBatches;
    bool reads[kBatches];
    float4v v[kBatches][kQuads];
#pragma unroll
    for (uint32_t b = 0; b < kBatches; ++b)
    {
        reads[b] = batch0 + b < range.batches && a.batchMost[slot * a.batches + batch0 + b] >= low;
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatches; ++b)
    {
        if (reads[b])
        {
            LoadBatch(x, range, batch0 + b, v[b]);
        }
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatches; ++b)
    {
        if (!reads[b])
        {
            continue;
        }
        uint32_t may = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4 * kQuads; ++i)
        {
            may |= v[b][i / 4][i % 4] >= low && v[b][i / 4][i % 4] <= high ? 1u << i : 0u;
        }
        while (may != 0)
        {
            const uint32_t bit = __ffs(static_cast<int>(may)) - 1;
            may &= may - 1;
            float logit = v[b][0][0];
#pragma unroll
            for (uint32_t i = 1; i < 4 * kQuads; ++i)
            {
                logit = bit == i ? v[b][i / 4][i % 4] : logit;
            }
            const float counted = Counted(logit);
            const double d = top - PlaceOf(counted, perUnit).step;
            if (counted > -INFINITY && d >= first && d <= last)
            {
                const uint32_t at = atomicAdd(&kept->listed, 1u);
                if (at < a.listRoom)
                {
                    // In any order: what is made of them goes by their own.
                    keys[at] = OrderKey(counted, IndexOf(range, batch0 + b, bit));
                }
            }
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
    // Four batches a wave, where that leaves workgroups enough; the end of a row looks through a part of it.
    const uint32_t wanted = std::min(most, std::max(kCountBlocks / rows, kFewestParts));
    const uint32_t length = CeilDiv(batches, wanted) * kBatch;
    return Parts{CeilDiv(vocab, length), length};
}

/// Batches of a part: one more than its logits fill, since they may begin anywhere.
uint32_t BatchesOf(const Parts& parts) { return parts.length / kBatch + 1; }

/// Keys of a row's list.
uint32_t ListRoom(uint32_t vocab) { return std::min(vocab, kListed); }
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_sample_rows_workspace_bytes(uint32_t rows, uint32_t vocab)
{
    if (rows == 0 || rows > kMaxRows || vocab == 0 || vocab > kMaxVocab)
    {
        return 0;
    }
    const Parts parts = PartsOf(rows, vocab);
    return (sizeof(PartHead) + 12ull * kSteps + 4ull * BatchesOf(parts)) * rows * parts.count +
           (rows <= kListRows ? (sizeof(RowSteps) + sizeof(uint64_t) * ListRoom(vocab)) * rows : 0);
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
        return Fail(MUYO_E_RANGE, "%s: needs 1..%u rows of 1..%u logits (got %u of %u)", name, kMaxRows, kMaxVocab,
                    rows, vocab);
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
                 parts.count, parts.length, nullptr, nullptr, nullptr, nullptr, BatchesOf(parts), nullptr, nullptr,
                 ListRoom(vocab)};
    const bool lists = rows <= kListRows;
    a.steps = reinterpret_cast<RowSteps*>(space);
    space += lists ? sizeof(RowSteps) * rows : 0;
    a.listKeys = reinterpret_cast<uint64_t*>(space);
    space += lists ? sizeof(uint64_t) * a.listRoom * rows : 0;
    a.masses = reinterpret_cast<uint64_t*>(space);
    a.heads = reinterpret_cast<PartHead*>(space + 8ull * kSteps * blocks);
    a.counts = reinterpret_cast<uint32_t*>(space + (8ull * kSteps + sizeof(PartHead)) * blocks);
    a.batchMost = reinterpret_cast<float*>(space + (12ull * kSteps + sizeof(PartHead)) * blocks);
    const hipStream_t s = AsStream(stream);
    hipLaunchKernelGGL(SampleCountKernel, dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, a);
    if (lists)
    {
        hipLaunchKernelGGL(SamplePickKernel<kPickSteps>, dim3(rows), dim3(kPickBlock), 0, s, a);
        const auto waves = [&](uint32_t each) { return CeilDiv(a.batches, each) * parts.count; };
        if (static_cast<uint64_t>(waves(1)) * rows <= kListAtOnce)
        {
            hipLaunchKernelGGL(SampleListKernel<1>, dim3(CeilDiv(waves(1), kWaves), rows), dim3(kBlock), 0, s, a);
        }
        else
        {
            hipLaunchKernelGGL(SampleListKernel<2>, dim3(CeilDiv(waves(2), kWaves), rows), dim3(kBlock), 0, s, a);
        }
        hipLaunchKernelGGL(SamplePickKernel<kPickToken>, dim3(rows), dim3(kPickBlock), 0, s, a);
    }
    else
    {
        hipLaunchKernelGGL(SamplePickKernel<kPickAll>, dim3(rows), dim3(kPickBlock), 0, s, a);
    }
    return LaunchStatus(name);
}
