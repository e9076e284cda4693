// Routing: the k largest logits of each token's row with their softmax
// weights, and the assignments (token, choice) sorted by expert.
//
// The choice is a CSR matrix of k entries per row; what is built here is its
// CSC pattern: offsets[e] (the column pointers), row_tokens (the row of each
// entry, in column order) and places (where entry (t, j) went).  Columns keep
// the order of the rows (a stable counting sort), so every result is the same
// from run to run.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "experts_device.h"
#include "experts_internal.h"

namespace aclsp {
namespace {

constexpr int kRouteThreads = 1024;
constexpr int kRouteWaves = kRouteThreads / 64;
constexpr int64_t kTokensPerTurn = kRouteThreads / 16;  // a quarter of that beyond 256 experts

// A logit as an unsigned key of the same order.  NaN is above everything, as
// in torch.topk; -0 and +0 are one value; 0 is below every value.
__device__ __forceinline__ uint32_t OrderKey(float v)
{
    if (v != v) return 0xFFFFFFFFU;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFU : 0x80000000U);
}
constexpr uint32_t kKeyMinusInf = 0x007FFFFFU;

__device__ __forceinline__ float KeyValue(uint32_t key)
{
    return key == 0xFFFFFFFFU ? __uint_as_float(0x7FC00000U)
                              : __uint_as_float(key ^ ((key >> 31) ? 0x80000000U : 0xFFFFFFFFU));
}

// The choices of a wave's tokens, L = 16 lanes each (64 beyond 256 experts,
// whose values would not fit the registers): lane l of a token holds its
// logits l*V to l*V + V - 1.  Each of the k rounds takes the largest key of
// the L lanes and, among equal ones, the lowest lane and its lowest value,
// which is the lowest index; that lane notes the choice in LDS and drops the
// value.  The rounds are a chain of dependent steps, which four tokens share.
struct Choice {
    uint32_t key;
    int32_t index;
};

template <typename T, int V, int L>
__device__ __forceinline__ void GateTokens(const RouteLaunch& p, int64_t t, bool valid, Choice* choices)
{
    const int lane = threadIdx.x & 63, sub = lane & (L - 1), row = lane / L;
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    const T* logits = static_cast<const T*>(p.logits) + (valid ? t : 0) * p.ld;
    uint32_t key[V];
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = sub * V + i;
        v[i] = valid && e < experts ? ToFloat(logits[e]) : -INFINITY;
        key[i] = e < experts ? OrderKey(v[i]) : 0U;
    }
    uint32_t top = 0;
    int32_t count = 0;
    for (int j = 0; j < k; ++j) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < V; ++i) {
            at = key[i] > best ? i : at;
            best = key[i] > best ? key[i] : best;
        }
        const uint32_t most = L == 16 ? RowMaxU32(best) : WaveMaxU32(best);
        if (__all(most <= kKeyMinusInf)) break;
        const uint64_t who = __ballot(best == most) >> (row * L) & (~uint64_t{0} >> (64 - L));
        if (most > kKeyMinusInf) {
            if (j == 0) top = most;
            count = j + 1;
            if (sub == __builtin_ctzll(who)) {
                choices[j] = {most, sub * V + at};
#pragma unroll
                for (int i = 0; i < V; ++i) key[i] = i == at ? 0U : key[i];
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the choices of other lanes
    const float peak = KeyValue(top);
    float sum = 0.0f;
    if (p.normalize) {
        for (int j = sub; j < count; j += L) sum += expf(KeyValue(choices[j].key) - peak);
    } else if (count > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += v[i] != -INFINITY ? expf(v[i] - peak) : 0.0f;
    }
    sum = L == 16 ? RowSum(sum) : WaveSum(sum);
    if (!valid) return;
    for (int j = sub; j < k; j += L) {
        const bool chosen = j < count;
        p.weights[t * k + j] = chosen ? expf(KeyValue(choices[j].key) - peak) / sum : 0.0f;
        p.ids[t * k + j] = chosen ? choices[j].index : -1;
    }
}

// Counts of one workgroup's assignments by expert, with their choice where
// logits are given.
template <typename T, int V, int L>
__device__ __forceinline__ void GateAndCount(const RouteLaunch& p, int64_t t0, int64_t t1, int32_t* hist)
{
    constexpr int kTokens = kRouteThreads / L;
    __shared__ Choice choices[kTokens][kMaxRouteK];
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) hist[e] = 0;
    if (p.logits != nullptr) {
        for (int64_t t = t0; t < t1; t += kTokens) {
            const int slot = threadIdx.x / L;
            GateTokens<T, V, L>(p, t + slot, t + slot < t1, choices[slot]);
        }
    }
    __syncthreads();
    for (int64_t a = t0 * k + threadIdx.x; a < t1 * k; a += kRouteThreads) {
        const int id = p.ids[a];
        if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
    }
    __syncthreads();
}

// Places of one workgroup's assignments.  base[e] starts as the place of the
// workgroup's first assignment of expert e; 1024 assignments a turn are ranked
// within their wave (lanes of the same expert below this one) and over the
// waves: waveCount[w][e] holds wave w's count, then that of the waves before
// it, and its last row the turn's count.
using WaveCounts = uint16_t[kRouteWaves + 1][kMaxRouteExperts];

__device__ void PlaceAssignments(const RouteLaunch& p, int64_t a0, int64_t a1, int32_t* base, WaveCounts& waveCount,
                                 int bits)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int experts = static_cast<int>(p.experts);
    const uint32_t k = static_cast<uint32_t>(p.k);
    for (int64_t first = a0; first < a1; first += kRouteThreads) {
        for (int e = lane; e < experts; e += 64) waveCount[wave][e] = 0;
        __syncthreads();
        const int64_t a = first + threadIdx.x;
        int id = a < a1 ? p.ids[a] : -1;
        if (id >= experts) id = -1;
        uint64_t same = __ballot(id >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((id >> b) & 1);
            same &= ((id >> b) & 1) ? m : ~m;
        }
        const int rank = __popcll(same & ((uint64_t{1} << lane) - 1));
        if (id >= 0 && rank == 0) waveCount[wave][id] = static_cast<uint16_t>(__popcll(same));
        __syncthreads();
        for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
            uint32_t at = 0;
            for (int w = 0; w < kRouteWaves; ++w) {
                const uint32_t c = waveCount[w][e];
                waveCount[w][e] = static_cast<uint16_t>(at);
                at += c;
            }
            waveCount[kRouteWaves][e] = static_cast<uint16_t>(at);
        }
        __syncthreads();
        if (a < a1) {
            const int32_t place = id >= 0 ? base[id] + waveCount[wave][id] + rank : -1;
            p.places[a] = place;
            if (place >= 0) p.row_tokens[place] = static_cast<int32_t>(static_cast<uint32_t>(a) / k);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < experts; e += kRouteThreads) base[e] += waveCount[kRouteWaves][e];
    }
}

// base[e] = the exclusive sum over experts of total[e], by the first wave.
// Returns the total of all experts in every thread of that wave.
__device__ int32_t ScanExperts(const int32_t* total, int32_t* base, int experts)
{
    const int lane = threadIdx.x & 63;
    int32_t before = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int32_t c = e0 + lane < experts ? total[e0 + lane] : 0;
        const int32_t incl = WaveInclusiveSum(c);
        if (e0 + lane < experts) base[e0 + lane] = before + incl - c;
        before += __shfl(incl, 63);
    }
    return before;
}

// The plan from every expert's total and, in before[e], its assignments in
// earlier workgroups.
__device__ void PlacePart(const RouteLaunch& p, int64_t t0, int64_t t1, const int32_t* total, int32_t* before, int bits)
{
    __shared__ WaveCounts waveCount;
    __shared__ int32_t first[kMaxRouteExperts];
    __shared__ int32_t used;
    const int experts = static_cast<int>(p.experts);
    if (threadIdx.x < 64) {
        const int32_t n = ScanExperts(total, first, experts);
        if (threadIdx.x == 0) used = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
        before[e] += first[e];
        if (blockIdx.x == 0) p.offsets[e] = first[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[experts] = used;
    // rows that no assignment took (dropped ones) read -1
    for (int64_t r = used + static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x; r < p.tokens * p.k;
         r += static_cast<int64_t>(gridDim.x) * kRouteThreads) {
        p.row_tokens[r] = -1;
    }
    __syncthreads();
    PlaceAssignments(p, t0 * p.k, t1 * p.k, before, waveCount, bits);
}

// Few tokens: everything in one workgroup and one launch, bound by its
// latency: one token of 64 experts, 8 chosen, 5.1 us (an empty launch 3.5).
template <typename T, int V, int L>
__global__ __launch_bounds__(kRouteThreads) void RouteOneKernel(RouteLaunch p, int bits)
{
    __shared__ int32_t total[kMaxRouteExperts], before[kMaxRouteExperts];
    GateAndCount<T, V, L>(p, 0, p.tokens, total);
    for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) before[e] = 0;
    PlacePart(p, 0, p.tokens, total, before, bits);
}

// The first of two launches: the choices, and each workgroup's counts.  Bound
// by the chain of a token's k rounds rather than by its bytes: 16384 tokens of
// 128 experts, 8 chosen, fp32, 10.2 us.
template <typename T, int V, int L>
__global__ __launch_bounds__(kRouteThreads) void RouteGateKernel(RouteLaunch p, int64_t tokensPerBlock)
{
    __shared__ int32_t hist[kMaxRouteExperts];
    const int64_t t0 = blockIdx.x * tokensPerBlock;
    GateAndCount<T, V, L>(p, t0, t0 + tokensPerBlock < p.tokens ? t0 + tokensPerBlock : p.tokens, hist);
    for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) p.hist[blockIdx.x * p.experts + e] = hist[e];
}

// Every workgroup sums the histograms itself (at most 256 of them, from L2):
// those before it give its base within each expert, all of them the experts'
// totals.  The threads of one expert take turns at the histograms.  The same
// tokens: 7 us (with the counting launch of a given choice, in a graph, 9.7).
__global__ __launch_bounds__(kRouteThreads) void RoutePlaceKernel(RouteLaunch p, int64_t tokensPerBlock, int bits)
{
    __shared__ int32_t total[kMaxRouteExperts], before[kMaxRouteExperts];
    const int experts = static_cast<int>(p.experts), blocks = static_cast<int>(gridDim.x);
    const int width = 1 << (bits < 6 ? 6 : bits);  // whole waves per histogram
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) total[e] = before[e] = 0;
    __syncthreads();
    const int e = threadIdx.x & (width - 1);
    if (e < experts) {
        int32_t mine = 0, all = 0;
#pragma unroll 8
        for (int b = static_cast<int>(threadIdx.x) / width; b < blocks; b += kRouteThreads / width) {
            const int32_t c = p.hist[static_cast<int64_t>(b) * experts + e];
            mine += b < static_cast<int>(blockIdx.x) ? c : 0;
            all += c;
        }
        atomicAdd(&before[e], mine);
        atomicAdd(&total[e], all);
    }
    __syncthreads();
    const int64_t t0 = blockIdx.x * tokensPerBlock;
    PlacePart(p, t0, t0 + tokensPerBlock < p.tokens ? t0 + tokensPerBlock : p.tokens, total, before, bits);
}

// Gradient of the weights with respect to the logits of one token, by one
// wave: the row is put together in LDS, which the chosen entries enter by index.
// The formulas: with weights normalised over the chosen, dl_j = w_j (g_j -
// sum_i w_i g_i) there and 0 elsewhere; else dl_e = p_e (g_e - sum_i w_i g_i)
// for every expert, g_e = 0 off the chosen.  The same tokens, normalised, where
// the logits are not read: 5.1 us, 10 MB.
template <typename T, int V>
__global__ __launch_bounds__(256) void RouteGradKernel(RouteGradLaunch p)
{
    __shared__ float rows[4][V * 64];
    const int lane = threadIdx.x & 63;
    const int64_t t = static_cast<int64_t>(BlockNumber()) * 4 + (threadIdx.x >> 6);
    if (t >= p.tokens) return;  // whole waves
    float* row = rows[threadIdx.x >> 6];
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    const float w = lane < k ? p.weights[t * k + lane] : 0.0f;
    const float g = lane < k ? p.grad_weights[t * k + lane] : 0.0f;
    const int id = lane < k ? p.ids[t * k + lane] : -1;
    const float dot = WaveSum(id >= 0 ? w * g : 0.0f);
    if (p.normalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) row[64 * i + lane] = 0.0f;
    } else {
        float prob[V];
        const T* logits = static_cast<const T*>(p.logits) + t * p.ld;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            prob[i] = 64 * i + lane < experts ? ToFloat(logits[64 * i + lane]) : -INFINITY;
            top = fmaxf(top, prob[i]);
        }
        top = WaveMax(top);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            prob[i] = prob[i] == -INFINITY ? 0.0f : expf(prob[i] - top);
            s += prob[i];
        }
        s = WaveSum(s);
#pragma unroll
        for (int i = 0; i < V; ++i) row[64 * i + lane] = s == 0.0f ? 0.0f : -(prob[i] / s) * dot;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (id >= 0 && id < experts) row[id] = w * (g - dot);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    T* out = static_cast<T*>(p.grad_logits) + t * p.ld_grad;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (64 * i + lane < experts) out[64 * i + lane] = FromFloat<T>(row[64 * i + lane]);
    }
}

// Whole turns of 64 tokens, and no more than 256 workgroups.
int64_t TokensPerBlock(int64_t tokens)
{
    const int64_t turns = (tokens + 256 * kTokensPerTurn - 1) / (256 * kTokensPerTurn);
    return (turns > 0 ? turns : 1) * kTokensPerTurn;
}

int Bits(int64_t experts)
{
    int b = 0;
    while ((int64_t{1} << b) < experts) ++b;
    return b;
}

template <typename T, int V, int L>
int RouteTyped(const RouteLaunch& l, hipStream_t s)
{
    const int64_t per = TokensPerBlock(l.tokens);
    const int64_t blocks = RouteBlocks(l.tokens);
    if (blocks == 1) {
        RouteOneKernel<T, V, L><<<1, kRouteThreads, 0, s>>>(l, Bits(l.experts));
        return 0;
    }
    RouteGateKernel<T, V, L><<<static_cast<uint32_t>(blocks), kRouteThreads, 0, s>>>(l, per);
    RoutePlaceKernel<<<static_cast<uint32_t>(blocks), kRouteThreads, 0, s>>>(l, per, Bits(l.experts));
    return 0;
}

template <typename T, int V>
int RouteGradTyped(const RouteGradLaunch& l, hipStream_t s)
{
    RouteGradKernel<T, V><<<GridOf((l.tokens + 3) / 4), 256, 0, s>>>(l);
    return 0;
}

template <typename T>
int RouteByExperts(const RouteLaunch& l, hipStream_t s)
{
    if (l.experts <= 64) return RouteTyped<T, 4, 16>(l, s);
    if (l.experts <= 128) return RouteTyped<T, 8, 16>(l, s);
    if (l.experts <= 256) return RouteTyped<T, 16, 16>(l, s);
    return RouteTyped<T, 16, 64>(l, s);
}

template <typename T>
int RouteGradByExperts(const RouteGradLaunch& l, hipStream_t s)
{
    if (l.experts <= 64) return RouteGradTyped<T, 1>(l, s);
    if (l.experts <= 128) return RouteGradTyped<T, 2>(l, s);
    if (l.experts <= 256) return RouteGradTyped<T, 4>(l, s);
    return RouteGradTyped<T, 16>(l, s);
}

}  // namespace

int64_t RouteBlocks(int64_t tokens)
{
    const int64_t per = TokensPerBlock(tokens);
    const int64_t b = (tokens + per - 1) / per;
    return b > 0 ? b : 1;
}

int LaunchRoute(const RouteLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.logits == nullptr || l.type == ACL_FLOAT) return RouteByExperts<float>(l, s);
    return l.type == ACL_FLOAT16 ? RouteByExperts<Half>(l, s) : RouteByExperts<Bf16>(l, s);
}

int LaunchRouteGrad(const RouteGradLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.type == ACL_FLOAT) return RouteGradByExperts<float>(l, s);
    return l.type == ACL_FLOAT16 ? RouteGradByExperts<Half>(l, s) : RouteGradByExperts<Bf16>(l, s);
}

}  // namespace aclsp
