// Rope + append into a paged cache of 8-bit values with an f32 scale per row and kv head. The attention over
// it is in paged_attention_q8.hip.
//
// A cache is [pages][kv_heads][page_size][head_dim] bytes and [pages][kv_heads][page_size] scales; a value is
// scale * code.
#include <cmath>

#include "common.hpp"
#include "paged.hpp"
#include "paged_rope.hpp"

namespace muyo
{
namespace
{
struct AppendQ8Args
{
    const float* q;
    const float* k;
    const float* v;
    uint64_t qStride, kStride, vStride;
    float* qOut;
    uint8_t* kcache;
    uint8_t* vcache;
    float* kscales;
    float* vscales;
    const int32_t* positions;
    const int32_t* slots;
    uint32_t tokens, heads, kvHeads;
    uint32_t pageShift;
    uint32_t slotCount;
    uint32_t interleaved;
    uint32_t rotary;
    const double* turns;
    float magnitude;
};

/// The largest of `value` in groups of kLanes lanes.
template <int kLanes>
__device__ __forceinline__ uint64_t GroupLargest(uint64_t value)
{
    auto step = [&](auto partner) {
        const uint32_t lo = static_cast<uint32_t>(partner(static_cast<int>(static_cast<uint32_t>(value))));
        const uint32_t hi = static_cast<uint32_t>(partner(static_cast<int>(static_cast<uint32_t>(value >> 32))));
        const uint64_t other = (static_cast<uint64_t>(hi) << 32) | lo;
        value = value > other ? value : other;
    };
    step([](int v) { return PartnerLane<1>(v); });
    step([](int v) { return PartnerLane<2>(v); });
    step([](int v) { return PartnerLane<4>(v); });
    if constexpr (kLanes == 16)
    {
        step([](int v) { return PartnerLane<8>(v); });
    }
    return value;
}

/// `x` rounded to f32 so that a later rounding to a shorter type is that of `x` itself: towards 0, with the last
/// bit set where something was left out.
__device__ __forceinline__ float ToOdd(double x)
{
    const float f = __double2float_rz(x);
    return static_cast<double>(f) == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

/// The codes of four scaled values, the first in the lowest byte.
template <int kFormat>
__device__ __forceinline__ uint32_t Codes(const double (&x)[4])
{
    if constexpr (kFormat == MUYO_KV_INT8)
    {
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            const int code = static_cast<int>(rint(x[e]));
            word |= (static_cast<uint32_t>(code) & 0xFFu) << (8 * e);
        }
        return word;
    }
    else
    {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(ToOdd(x[0]), ToOdd(x[1]), 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(ToOdd(x[2]), ToOdd(x[3]), word, true);
        return static_cast<uint32_t>(word);
    }
}

/// The fraction, about 0, of the turns of a pair at a position: the product is rounded before its whole turns are
/// taken off it, as it is when turns are counted in 64 bits anywhere else.
__device__ __forceinline__ double TurnFraction(double turns, int32_t position)
{
#pragma clang fp contract(off)
    const double t = static_cast<double>(position) * turns;
    return t - rint(t);
}

/// kHd / 8 lanes a row (a head of q, then of k, then of v) of a token, four pairs of values a lane: kOctets
/// (rotary dimensions that are multiples of 8) as two loads of 16 bytes, else value by value.
///
/// A row's scale is its largest size over the type's, rounded to f32, and its codes are the values over that
/// scale, rounded once (half steps to even): k is rotated in 64 bits and scaled in 64 bits, so that a value next
/// to the border between two codes gets the one that is nearer (from f32, about one value in 2^16 would get the
/// other). q stays f32, as in the fp16 cache's append. (Two heads of q a lane, which share their angles, take 62 us
/// instead of 63.5 for 8191 tokens of 28 / 4 heads of 128, and 7.2 instead of 5.8 for 253.)
///
/// What bounds it: round trips for few tokens; for many, reads and writes together (277 MB, 4.4 TB/s, where a copy has
/// 5.1) beside vector work: angles, and codes in 64 bits.
template <int kHd, int kFormat, bool kOctets, bool kInterleaved>
__global__ __launch_bounds__(256) void PagedAppendQ8Kernel(AppendQ8Args a)
{
    constexpr uint32_t kLanes = kHd / 8;
    const uint32_t rows = a.heads + 2 * a.kvHeads;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint64_t token = item / (static_cast<uint64_t>(rows) * kLanes);
    if (token >= a.tokens)
    {
        return;
    }
    const uint32_t rest = static_cast<uint32_t>(item - token * rows * kLanes);
    const uint32_t r = rest / kLanes;
    const uint32_t o = rest % kLanes;
    const int32_t position = a.positions[token];
    const int32_t slot = a.slots[token];
    const uint32_t half = a.rotary / 2;
    const bool isQ = r < a.heads;
    const bool isK = !isQ && r < a.heads + a.kvHeads;
    const uint32_t g = isQ ? 0 : isK ? r - a.heads : r - a.heads - a.kvHeads;
    const float* from = isQ   ? a.q + token * a.qStride + r * kHd
                        : isK ? a.k + token * a.kStride + g * kHd
                              : a.v + token * a.vStride + g * kHd;
    // Pair e's places: those of rotated pair 4 o + e, or two values behind the rotated ones.
    uint32_t i0[4], i1[4];
    float x0[4], x1[4];
    const bool turned = 8 * o < a.rotary;  // kOctets: the lane's pairs
    const uint32_t lo = turned && !kInterleaved ? 4 * o : 8 * o;
    const uint32_t hi = turned && !kInterleaved ? 4 * o + half : 8 * o + 4;
    if constexpr (kOctets)
    {
        const float4v u = *reinterpret_cast<const float4v*>(from + lo);
        const float4v w = *reinterpret_cast<const float4v*>(from + hi);
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            x0[e] = kInterleaved ? (e < 2 ? u : w)[e % 2 * 2] : u[e];
            x1[e] = kInterleaved ? (e < 2 ? u : w)[e % 2 * 2 + 1] : w[e];
        }
    }
    else
    {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
        {
            const uint32_t p = 4 * o + e;
            i0[e] = p < half && !kInterleaved ? p : 2 * p;
            i1[e] = p < half && !kInterleaved ? p + half : 2 * p + 1;
            x0[e] = from[i0[e]];
            x1[e] = from[i1[e]];
        }
    }
    // The same for all of a row's lanes.
    if (position < 0 || (!isQ && (slot < 0 || static_cast<uint32_t>(slot) >= a.slotCount)))
    {
        return;
    }
    if (isQ)
    {
        float* to = a.qOut + (token * a.heads + r) * kHd;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
        {
            if (kOctets ? turned : 4 * o + e < half)
            {
                float c, s;
                PairAngle(a.turns[4 * o + e], position, a.magnitude, c, s);
                Rotate(x0[e], x1[e], c, s, x0[e], x1[e]);
            }
        }
        if constexpr (kOctets)
        {
            *reinterpret_cast<float4v*>(to + lo) =
                kInterleaved ? float4v{x0[0], x1[0], x0[1], x1[1]} : float4v{x0[0], x0[1], x0[2], x0[3]};
            *reinterpret_cast<float4v*>(to + hi) =
                kInterleaved ? float4v{x0[2], x1[2], x0[3], x1[3]} : float4v{x1[0], x1[1], x1[2], x1[3]};
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                to[i0[e]] = x0[e];
                to[i1[e]] = x1[e];
            }
        }
        return;
    }
    double y0[4], y1[4];
    uint64_t largest = 0;  // of the sizes' bits: those of an infinity or NaN are above all others
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
    {
        y0[e] = x0[e];
        y1[e] = x1[e];
        if (isK && (kOctets ? turned : 4 * o + e < half))
        {
            double sn, cs;
            sincospi(2.0 * TurnFraction(a.turns[4 * o + e], position), &sn, &cs);
            cs *= a.magnitude;
            sn *= a.magnitude;
            const double u = y0[e];
            y0[e] = fma(u, cs, -(y1[e] * sn));
            y1[e] = fma(u, sn, y1[e] * cs);
        }
        const uint64_t b0 = static_cast<uint64_t>(__double_as_longlong(fabs(y0[e])));
        const uint64_t b1 = static_cast<uint64_t>(__double_as_longlong(fabs(y1[e])));
        largest = largest > b0 ? largest : b0;
        largest = largest > b1 ? largest : b1;
    }
    largest = GroupLargest<kLanes>(largest);
    constexpr double kMost = kFormat == MUYO_KV_INT8 ? 127.0 : 448.0;
    const double size = __longlong_as_double(static_cast<long long>(largest));
    const bool finite = size < INFINITY;
    // A row that is not finite, or that a magnitude has taken past f32, is told by its scale.
    const float scale = finite ? static_cast<float>(size / kMost) : NAN;
    const bool codes = scale > 0.0f && scale < INFINITY;
    // Quotients by the reciprocal and a step from what is left, which rounds them as a division does (Markstein).
    const double wide = codes ? static_cast<double>(scale) : 1.0;
    const double per = 1.0 / wide;
    auto scaled = [&](double y) {
        const double x = y * per;
        // A scale next to f32's end is rounded by more than half a code.
        return codes ? fmin(fmax(fma(fma(-x, wide, y), per, x), -kMost), kMost) : 0.0;
    };
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        y0[e] = scaled(y0[e]);
        y1[e] = scaled(y1[e]);
    }
    const uint32_t page = static_cast<uint32_t>(slot) >> a.pageShift;
    const uint32_t row = static_cast<uint32_t>(slot) & ((1u << a.pageShift) - 1);
    const uint64_t at = ((static_cast<uint64_t>(page) * a.kvHeads + g) << a.pageShift) + row;
    uint8_t* to = (isK ? a.kcache : a.vcache) + at * kHd;
    if constexpr (kOctets && !kInterleaved)
    {
        *reinterpret_cast<uint32_t*>(to + lo) = Codes<kFormat>(y0);
        *reinterpret_cast<uint32_t*>(to + hi) = Codes<kFormat>(y1);
    }
    else if constexpr (kOctets)
    {
        const double first[4] = {y0[0], y1[0], y0[1], y1[1]};
        const double second[4] = {y0[2], y1[2], y0[3], y1[3]};
        *reinterpret_cast<uint2*>(to + lo) = make_uint2(Codes<kFormat>(first), Codes<kFormat>(second));
    }
    else
    {
        const uint32_t c0 = Codes<kFormat>(y0);
        const uint32_t c1 = Codes<kFormat>(y1);
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            to[i0[e]] = static_cast<uint8_t>(c0 >> (8 * e));
            to[i1[e]] = static_cast<uint8_t>(c1 >> (8 * e));
        }
    }
    if (o == 0)
    {
        (isK ? a.kscales : a.vscales)[at] = scale;
    }
}

template <int kHd, int kFormat>
void LaunchAppendQ8(hipStream_t s, const AppendQ8Args& a, dim3 grid)
{
    const bool octets = a.rotary % 8 == 0;
    if (octets && a.interleaved != 0)
    {
        hipLaunchKernelGGL((PagedAppendQ8Kernel<kHd, kFormat, true, true>), grid, dim3(256), 0, s, a);
    }
    else if (octets)
    {
        hipLaunchKernelGGL((PagedAppendQ8Kernel<kHd, kFormat, true, false>), grid, dim3(256), 0, s, a);
    }
    else if (a.interleaved != 0)
    {
        hipLaunchKernelGGL((PagedAppendQ8Kernel<kHd, kFormat, false, true>), grid, dim3(256), 0, s, a);
    }
    else
    {
        hipLaunchKernelGGL((PagedAppendQ8Kernel<kHd, kFormat, false, false>), grid, dim3(256), 0, s, a);
    }
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" int muyo_paged_rope_append_q8kv(const float* q, const float* k, const float* v, uint64_t q_stride,
                                           uint64_t k_stride, uint64_t v_stride, float* q_out, void* kcache,
                                           void* vcache, float* kscales, float* vscales, const int32_t* positions,
                                           const int32_t* slots, uint32_t tokens, uint32_t heads, uint32_t kv_heads,
                                           uint32_t head_dim, uint32_t pages, uint32_t page_size, uint32_t format,
                                           uint32_t rope_layout, uint32_t rotary_dim, const double* turns,
                                           float magnitude, void* stream)
{
    const char* name = "paged_rope_append_q8kv";
    if ((head_dim != 64 && head_dim != 128) || format > MUYO_KV_E4M3)
    {
        return Fail(MUYO_E_UNSUPPORTED, "%s: needs head_dim 64 or 128 and a known format (got %u, %u)", name, head_dim,
                    format);
    }
    const uint64_t scaleBytes = 4ull * kv_heads * pages * page_size;
    const uint64_t cacheBytes = scaleBytes / 4 * head_dim;
    const Range caches[] = {{kcache, cacheBytes, "kcache"},
                            {vcache, cacheBytes, "vcache"},
                            {kscales, scaleBytes, "kscales"},
                            {vscales, scaleBytes, "vscales"}};
    const uint64_t items = static_cast<uint64_t>(tokens) * (heads + 2ull * kv_heads) * (head_dim / 8);
    const AppendCall call{q, k, v, q_stride, k_stride, v_stride, q_out, positions, slots, tokens, heads, kv_heads,
                          head_dim, pages, page_size, rope_layout, rotary_dim, turns, magnitude, items};
    const int checked = CheckAppend(name, call, caches, 4);
    if (checked != MUYO_OK)
    {
        return checked;
    }
    AppendQ8Args a{q, k, v, q_stride, k_stride, v_stride, q_out, static_cast<uint8_t*>(kcache),
                   static_cast<uint8_t*>(vcache), kscales, vscales, positions, slots, tokens, heads, kv_heads, 0,
                   pages * page_size, rope_layout, rotary_dim, turns, magnitude};
    while ((1u << a.pageShift) < page_size)
    {
        ++a.pageShift;
    }
    const dim3 grid(CeilDiv(items, 256));
    if (head_dim == 64)
    {
        format == MUYO_KV_INT8 ? LaunchAppendQ8<64, MUYO_KV_INT8>(AsStream(stream), a, grid)
                               : LaunchAppendQ8<64, MUYO_KV_E4M3>(AsStream(stream), a, grid);
    }
    else
    {
        format == MUYO_KV_INT8 ? LaunchAppendQ8<128, MUYO_KV_INT8>(AsStream(stream), a, grid)
                               : LaunchAppendQ8<128, MUYO_KV_E4M3>(AsStream(stream), a, grid);
    }
    return LaunchStatus(name);
}
