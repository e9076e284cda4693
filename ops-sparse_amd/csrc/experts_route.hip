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

// A logit as an unsigned key of the same order.  NaN is above everything, as
// in torch.topk; -0 and +0 are one value; 0 is below every value.
__device__ __forceinline__ uint32_t OrderKey(float v)
{
    if (v != v) return 0xFFFFFFFFU;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFU : 0x80000000U);
}
constexpr uint32_t kKeyMinusInf = 0x007FFFFFU;

// One token's choice by one wave: lane j < k ends with the j-th largest logit
// and its index (-1 when the row has no j-th logit above -inf).  Each of the
// k rounds takes the wave's largest key and, among equal ones, the lowest
// index: value i of lane l is expert 64 i + l.
template <int V>
__device__ __forceinline__ void ChooseTopK(const float (&v)[V], int experts, int k, int lane, float& value, int& index)
{
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = 64 * i + lane < experts ? OrderKey(v[i]) : 0U;
    value = -INFINITY;
    index = -1;
    for (int j = 0; j < k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = best > key[i] ? best : key[i];
        best = WaveMaxU32(best);
        if (best <= kKeyMinusInf) break;  // uniform
        int who = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint64_t m = __ballot(key[i] == best);
            if (who < 0 && m != 0) {
                who = 64 * i + __builtin_ctzll(m);
                if (lane == (who & 63)) key[i] = 0U;
            }
        }
        if (lane == j) {
            index = who;
            const uint32_t u = best == 0xFFFFFFFFU ? 0x7FC00000U
                                                   : best ^ ((best >> 31) ? 0x80000000U : 0xFFFFFFFFU);
            value = __uint_as_float(u);
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void LoadRow(const T* row, int experts, int lane, float (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 64 * i + lane < experts ? ToFloat(row[64 * i + lane]) : -INFINITY;
}

// Weights and ids of one token by one wave: w_j = exp(l_j - m) / sum, the sum
// over the chosen or over the whole row, all in 32 bits.
template <typename T, int V>
__device__ __forceinline__ int GateToken(const RouteLaunch& p, int64_t t, int lane)
{
    float v[V];
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    LoadRow<T, V>(static_cast<const T*>(p.logits) + t * p.ld, experts, lane, v);
    float value;
    int index;
    ChooseTopK<V>(v, experts, k, lane, value, index);
    const float top = __shfl(value, 0);
    const float e = index >= 0 ? expf(value - top) : 0.0f;
    float sum;
    if (p.normalize) {
        sum = WaveSum(e);
    } else {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += 64 * i + lane < experts && v[i] != -INFINITY ? expf(v[i] - top) : 0.0f;
        sum = WaveSum(s);
    }
    if (lane < k) {
        p.weights[t * k + lane] = index >= 0 ? e / sum : 0.0f;
        p.ids[t * k + lane] = index;
    }
    return index;
}

// The experts' assignment counts of one workgroup's tokens, with their choice
// where logits are given.
template <typename T, int V>
__global__ __launch_bounds__(kRouteThreads) void RouteGateKernel(RouteLaunch p, int64_t tokensPerBlock)
{
    __shared__ int32_t hist[kMaxRouteExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) hist[e] = 0;
    __syncthreads();
    const int64_t t0 = blockIdx.x * tokensPerBlock;
    const int64_t t1 = t0 + tokensPerBlock < p.tokens ? t0 + tokensPerBlock : p.tokens;
    if (p.logits != nullptr) {
        for (int64_t t = t0 + wave; t < t1; t += kRouteWaves) {
            const int index = GateToken<T, V>(p, t, lane);
            if (lane < k && index >= 0) atomicAdd(&hist[index], 1);
        }
    } else {
        for (int64_t a = t0 * k + threadIdx.x; a < t1 * k; a += kRouteThreads) {
            const int id = p.ids[a];
            if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) p.hist[blockIdx.x * p.experts + e] = hist[e];
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

// Rows of row_tokens that no assignment took (dropped ones) read -1.
__device__ void FillTail(const RouteLaunch& p, int32_t used, int64_t start, int64_t step)
{
    for (int64_t r = used + start; r < p.tokens * p.k; r += step) p.row_tokens[r] = -1;
}

// Every workgroup sums the histograms itself (at most 256 of them, from L2):
// those before it give its base within each expert, all of them the experts' totals.
__global__ __launch_bounds__(kRouteThreads) void RoutePlaceKernel(RouteLaunch p, int64_t tokensPerBlock, int blocks,
                                                                  int bits)
{
    __shared__ WaveCounts waveCount;
    __shared__ int32_t base[kMaxRouteExperts], total[kMaxRouteExperts], first[kMaxRouteExperts];
    __shared__ int32_t used;
    const int experts = static_cast<int>(p.experts);
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
        int32_t before = 0, all = 0;
        for (int b = 0; b < blocks; ++b) {
            const int32_t c = p.hist[static_cast<int64_t>(b) * experts + e];
            before += b < static_cast<int>(blockIdx.x) ? c : 0;
            all += c;
        }
        base[e] = before;
        total[e] = all;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int32_t n = ScanExperts(total, first, experts);
        if (threadIdx.x == 0) used = n;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kRouteThreads) {
        base[e] += first[e];
        if (blockIdx.x == 0) p.offsets[e] = first[e];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[experts] = used;
    __syncthreads();
    FillTail(p, used, static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x,
             static_cast<int64_t>(blocks) * kRouteThreads);
    const int64_t t0 = blockIdx.x * tokensPerBlock;
    const int64_t t1 = t0 + tokensPerBlock < p.tokens ? t0 + tokensPerBlock : p.tokens;
    PlaceAssignments(p, t0 * p.k, t1 * p.k, base, waveCount, bits);
}

// Gradient of the weights with respect to the logits of one token, by one wave.
template <typename T, int V>
__global__ __launch_bounds__(256) void RouteGradKernel(RouteGradLaunch p)
{
    const int lane = threadIdx.x & 63;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= p.tokens) return;
    const int experts = static_cast<int>(p.experts), k = static_cast<int>(p.k);
    const float w = lane < k ? p.weights[t * k + lane] : 0.0f;
    const float g = lane < k ? p.grad_weights[t * k + lane] : 0.0f;
    const int id = lane < k ? p.ids[t * k + lane] : -1;
    const float dot = WaveSum(id >= 0 ? w * g : 0.0f);
    float d[V];
    float prob[V];
    if (p.normalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = 0.0f;
    } else {
        LoadRow<T, V>(static_cast<const T*>(p.logits) + t * p.ld, experts, lane, prob);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) top = fmaxf(top, prob[i]);
        top = WaveMax(top);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            prob[i] = prob[i] == -INFINITY ? 0.0f : expf(prob[i] - top);
            s += prob[i];
        }
        s = WaveSum(s);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            prob[i] = s == 0.0f ? 0.0f : prob[i] / s;
            d[i] = -prob[i] * dot;
        }
    }
    // the k chosen entries: those of lane l are taken up by the lane that holds expert id
    for (int j = 0; j < k; ++j) {
        const int idj = __shfl(id, j);
        const float wj = __shfl(w, j), gj = __shfl(g, j);
        if (idj >= 0 && lane == (idj & 63)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (i == (idj >> 6)) d[i] = wj * (gj - dot);
            }
        }
    }
    T* out = static_cast<T*>(p.grad_logits) + t * p.ld_grad;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (64 * i + lane < experts) out[64 * i + lane] = FromFloat<T>(d[i]);
    }
}

int64_t TokensPerBlock(int64_t tokens, int64_t k)
{
    // 16 tokens at least (one per wave), and no more than 256 workgroups
    const int64_t even = (tokens + 255) / 256;
    const int64_t least = (kRouteThreads + k - 1) / k;
    return even > least ? even : least;
}

int Bits(int64_t experts)
{
    int b = 0;
    while ((int64_t{1} << b) < experts) ++b;
    return b;
}

template <typename T, int V>
int RouteTyped(const RouteLaunch& l, hipStream_t s)
{
    const int64_t per = TokensPerBlock(l.tokens, l.k);
    const int64_t blocks = RouteBlocks(l.tokens, l.experts, l.k);
    RouteGateKernel<T, V><<<static_cast<uint32_t>(blocks), kRouteThreads, 0, s>>>(l, per);
    RoutePlaceKernel<<<static_cast<uint32_t>(blocks), kRouteThreads, 0, s>>>(l, per, static_cast<int>(blocks),
                                                                            Bits(l.experts));
    return 0;
}

template <typename T, int V>
int RouteGradTyped(const RouteGradLaunch& l, hipStream_t s)
{
    RouteGradKernel<T, V><<<static_cast<uint32_t>((l.tokens + 3) / 4), 256, 0, s>>>(l);
    return 0;
}

}  // namespace

int64_t RouteBlocks(int64_t tokens, int64_t experts, int64_t k)
{
    (void)experts;
    const int64_t per = TokensPerBlock(tokens, k);
    const int64_t b = (tokens + per - 1) / per;
    return b > 0 ? b : 1;
}

#define ROUTE_BY_EXPERTS(T, FN)                         \
    if (l.experts <= 64) return FN<T, 1>(l, s);         \
    if (l.experts <= 128) return FN<T, 2>(l, s);        \
    if (l.experts <= 256) return FN<T, 4>(l, s);        \
    if (l.experts <= 512) return FN<T, 8>(l, s);        \
    return FN<T, 16>(l, s);

int LaunchRoute(const RouteLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.logits == nullptr) return RouteTyped<float, 1>(l, s);  // the choice is given: V is not used
    if (l.type == ACL_FLOAT16) { ROUTE_BY_EXPERTS(Half, RouteTyped) }
    if (l.type == ACL_BF16) { ROUTE_BY_EXPERTS(Bf16, RouteTyped) }
    ROUTE_BY_EXPERTS(float, RouteTyped)
}

int LaunchRouteGrad(const RouteGradLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.type == ACL_FLOAT16) { ROUTE_BY_EXPERTS(Half, RouteGradTyped) }
    if (l.type == ACL_BF16) { ROUTE_BY_EXPERTS(Bf16, RouteGradTyped) }
    ROUTE_BY_EXPERTS(float, RouteGradTyped)
}

}  // namespace aclsp
