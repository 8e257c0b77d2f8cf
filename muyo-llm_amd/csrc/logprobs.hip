// Log probabilities of given tokens, their ranks, the entropy and the most likely tokens of rows of
// logits.
//
// With m the row's largest logit, s = sum e^(x - m) and t = sum e^(x - m) (x - m): a token's log
// probability is x - m - log s and the row's entropy log s - t / s.
#include <cmath>

#include "common.hpp"

namespace muyo
{
namespace
{
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr uint32_t kMaxTop = 64;
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
};

/// A 64-bit key whose descending order is (value descending, index ascending). -0 counts as +0, NaN
/// comes after -inf.
__device__ __forceinline__ uint64_t OrderKey(float v, uint32_t index)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t ordered = v != v ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (static_cast<uint64_t>(ordered) << 32) | static_cast<uint64_t>(~index);
}

template <class Op, class T>
__device__ __forceinline__ T BlockReduce(T v, T* shared)
{
    for (int step = 1; step < kWave; step *= 2)
    {
        v = Op()(v, __shfl_xor(v, step));
    }
    __syncthreads();
    if (threadIdx.x % kWave == 0)
    {
        shared[threadIdx.x / kWave] = v;
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
    {
        v = w == 0 ? shared[0] : Op()(v, shared[w]);
    }
    return v;
}

struct MaxF
{
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumF
{
    __device__ float operator()(float a, float b) const { return a + b; }
};
struct SumU
{
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a + b; }
};
struct MaxU64
{
    __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a > b ? a : b; }
};

/// A workgroup a row: the maximum, then the sums and the rank, then one pass per alternative.
__global__ __launch_bounds__(kBlock) void TokenLogprobsKernel(LogprobArgs a)
{
    __shared__ float sharedF[kWaves];
    __shared__ uint32_t sharedU[kWaves];
    __shared__ unsigned long long sharedK[kWaves];
    const uint32_t row = blockIdx.x;
    const float* x = a.logits + row * a.stride;
    const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
    const bool given = token >= 0 && static_cast<uint32_t>(token) < a.vocab;
    const float own = given ? x[token] : 0.0f;
    const uint64_t ownKey = given ? OrderKey(own, static_cast<uint32_t>(token)) : ~0ull;
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kBlock)
    {
        m = fmaxf(m, x[i]);
    }
    m = BlockReduce<MaxF>(m, sharedF);
    float s = 0.0f;
    float t = 0.0f;
    uint32_t above = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kBlock)
    {
        const float v = x[i];
        const float d = v - m;
        const float e = v == -INFINITY ? 0.0f : exp2f(d * kLog2e);
        s += e;
        t = e == 0.0f ? t : fmaf(e, d, t);
        above += OrderKey(v, i) > ownKey ? 1u : 0u;
    }
    s = BlockReduce<SumF>(s, sharedF);
    t = BlockReduce<SumF>(t, sharedF);
    above = BlockReduce<SumU>(above, sharedU);
    const bool empty = s == 0.0f;  // no logit above -inf
    const float logSum = empty ? 0.0f : logf(s);
    if (threadIdx.x == 0)
    {
        if (a.logprobs != nullptr)
        {
            a.logprobs[row] = !given || empty ? -INFINITY : own - m - logSum;
        }
        if (a.ranks != nullptr)
        {
            a.ranks[row] = given ? static_cast<int32_t>(above) : -1;
        }
        if (a.entropy != nullptr)
        {
            a.entropy[row] = empty ? 0.0f : logSum - t / s;
        }
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top; ++k)
    {
        unsigned long long best = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += kBlock)
        {
            const uint64_t key = OrderKey(x[i], i);
            best = key < last && key > best ? key : best;
        }
        best = BlockReduce<MaxU64>(best, sharedK);
        last = best;
        if (threadIdx.x == 0)
        {
            const uint32_t id = ~static_cast<uint32_t>(best);
            a.topIds[static_cast<uint64_t>(row) * a.top + k] = static_cast<int32_t>(id);
            a.topLogprobs[static_cast<uint64_t>(row) * a.top + k] = empty ? -INFINITY : x[id] - m - logSum;
        }
    }
}
}  // namespace
}  // namespace muyo

using namespace muyo;

extern "C" size_t muyo_token_logprobs_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t top)
{
    return rows == 0 || vocab == 0 || vocab > 0x7FFFFFFFu || top > kMaxTop || top > vocab ? 0 : 16;
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
    LogprobArgs a{logits, row_stride, rows, vocab, tokens, logprobs, ranks, entropy, top, top_ids, top_logprobs};
    hipLaunchKernelGGL(TokenLogprobsKernel, dim3(rows), dim3(kBlock), 0, AsStream(stream), a);
    return LaunchStatus(name);
}
