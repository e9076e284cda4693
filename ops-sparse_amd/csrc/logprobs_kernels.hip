// Log probabilities of given tokens under rows of logits, with each row's
// entropy and its largest alternatives, and their gradient.
//
//   log p_v = (l_v - M) - log S,  S = sum exp(l_v - M),  M the row's largest
//   H = log S - W / S,            W = sum exp(l_v - M) (l_v - M)
//   dl_v = g_t [v = t] - p_v (g_t + gH (log p_v + H))
//
// One pass over a row keeps M, S and W per thread; where the largest grows,
// S and W are moved to it.  With few rows several workgroups share one, and
// another launch joins what they found.  Bound by memory: the logits are read
// once, those of few threads a second time for alternatives.  8192 rows of 65536
// bf16 logits with the entropy: 192 us (5.6 TB/s), their gradient 358 us (6.0
// TB/s read and written).  One row of 131072 with 20 alternatives, 64 segments:
// 4.8 us and 4.8 to join them, latency alone; 37 rows of 32003 fp32 with 5, a
// workgroup each: 7.5 us, its exponentials and what is around them.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "experts_device.h"
#include "experts_internal.h"
#include "model_ops_internal.h"

namespace aclsp {
namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;         // logits that a thread loads at a time
constexpr int kBatch = 4;        // units between two looks at the largest
constexpr int kMaxSegments = 64; // of a row: one for each lane of the wave that joins them
constexpr int kCandidates = 1024;

constexpr float kLog2E = 1.44269504f;
constexpr float kLowest = -3.402823466e38f;  // stands for no logit yet: finite, so that differences from it are not NaN
constexpr float kFar = -1e4f;                // log p of what has p = 0, in products with it: 2^kFar is 0

__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float Infinity() { return __uint_as_float(0x7F800000U); }

// What a part of a row comes to; s and w relative to m, w in units of log 2.
struct Part {
    float m, s, w;
    __device__ __forceinline__ void MoveTo(float to)
    {
        const float by = fmaxf((m - to) * kLog2E, kFar), c = Exp2(by);
        w = c * (w + s * by);
        s *= c;
        m = to;
    }
};

// f over the lanes of each G, in all of them
template <int G, typename F>
__device__ __forceinline__ uint32_t OverLanes(uint32_t x, F f)
{
    static_assert(G == 2 || G == 4 || G == 8 || G == 16, "");
    x = f(x, Dpp<0xB1, 0xF>(x, x));
    if constexpr (G > 2) x = f(x, Dpp<0x4E, 0xF>(x, x));
    if constexpr (G > 4) x = f(x, Dpp<0x141, 0xF>(x, x));  // mirrored in each 8
    if constexpr (G > 8) x = f(x, Dpp<0x140, 0xF>(x, x));  // and in each 16
    return x;
}
template <int G>
__device__ __forceinline__ float MaxOverLanes(float x)
{
    return __uint_as_float(OverLanes<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int G>
__device__ __forceinline__ uint32_t SumOverLanes(uint32_t x)
{
    return OverLanes<G>(x, [](uint32_t a, uint32_t b) { return a + b; });
}

// The parts of a wave's lanes as one, in all lanes
__device__ __forceinline__ Part WavePart(Part p)
{
    p.MoveTo(WaveMax(p.m));
    return {p.m, WaveSum(p.s), WaveSum(p.w)};
}

// A logit as an unsigned key of the same order, NaN above all, and with the
// index behind it, the lower the greater: what comes first is the larger number.
// No pair has all bits set, which stands for what is before the first.
constexpr uint32_t kKeyNan = 0xFFFFFFFEU;
__device__ __forceinline__ uint32_t OrderKey(float v)
{
    if (v != v) return kKeyNan;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFU : 0x80000000U);
}
constexpr uint32_t kKeyMinusInf = 0x007FFFFFU;
__device__ __forceinline__ float KeyValue(uint32_t key)
{
    return key == kKeyNan ? __uint_as_float(0x7FC00000U)
                          : __uint_as_float(key ^ ((key >> 31) ? 0x80000000U : 0xFFFFFFFFU));
}
__device__ __forceinline__ uint64_t Pair(float v, int32_t index)
{
    return static_cast<uint64_t>(OrderKey(v)) << 32 | ~static_cast<uint32_t>(index);
}
__device__ __forceinline__ int32_t PairIndex(uint64_t pair) { return static_cast<int32_t>(~static_cast<uint32_t>(pair)); }
__device__ __forceinline__ float PairValue(uint64_t pair) { return KeyValue(static_cast<uint32_t>(pair >> 32)); }

// The largest of a wave's lanes: of the high halves, then of the low ones of the lanes that have it.
__device__ __forceinline__ uint64_t WaveMaxU64(uint64_t x)
{
    const uint32_t high = WaveMaxU32(static_cast<uint32_t>(x >> 32));
    const uint32_t low = WaveMaxU32(static_cast<uint32_t>(x >> 32) == high ? static_cast<uint32_t>(x) : 0U);
    return static_cast<uint64_t>(high) << 32 | low;
}

// Logits [c, c + 8) of a row's first `end`; -inf past them.
template <typename T>
__device__ __forceinline__ void LoadUnit(const T* row, int32_t c, int32_t end, T (&v)[kUnit])
{
    if (c + kUnit <= end) {
        __builtin_memcpy(v, row + c, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = c + i < end ? row[c + i] : FromFloat<T>(-Infinity());
    }
}

// Adds N units to a thread's part.
template <bool kEntropy, int N, typename T>
__device__ __forceinline__ void AddUnits(Part& p, const T (&v)[N][kUnit])
{
    float most = p.m;
#pragma unroll
    for (int i = 0; i < N * kUnit; ++i) most = fmaxf(most, ToFloat(v[i / kUnit][i % kUnit]));
    if (most > p.m) p.MoveTo(most);
#pragma unroll
    for (int i = 0; i < N * kUnit; ++i) {
        const float d = (ToFloat(v[i / kUnit][i % kUnit]) - p.m) * kLog2E, e = Exp2(d);
        p.s += e;
        if constexpr (kEntropy) p.w += e * fmaxf(d, kFar);
    }
}

// A thread's logits of [begin, end), for a workgroup of W threads: H units that it holds where they fit, none for H = 0.
template <typename T, int H, int W>
struct Held {
    T v[H > 0 ? H : 1][kUnit];

    template <bool kEntropy>
    __device__ __forceinline__ Part Read(const T* row, int32_t begin, int32_t end)
    {
        const int32_t c = begin + static_cast<int32_t>(threadIdx.x) * kUnit;
        Part p{kLowest, 0.0f, 0.0f};
        if constexpr (H > 0) {
#pragma unroll
            for (int b = 0; b < H; ++b) LoadUnit(row, c + b * W * kUnit, end, v[b]);
            AddUnits<kEntropy>(p, v);
        } else {
            for (int32_t at = c; at < end; at += W * kUnit * kBatch) {
                T u[kBatch][kUnit];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) LoadUnit(row, at + b * W * kUnit, end, u[b]);
                AddUnits<kEntropy>(p, u);
            }
        }
        return p;
    }

    // f(value, index) for each of them, -inf past the end
    template <typename F>
    __device__ __forceinline__ void ForEach(const T* row, int32_t begin, int32_t end, F f) const
    {
        const int32_t c = begin + static_cast<int32_t>(threadIdx.x) * kUnit;
        if constexpr (H > 0) {
#pragma unroll
            for (int i = 0; i < H * kUnit; ++i) {
                f(ToFloat(v[i / kUnit][i % kUnit]), c + i / kUnit * W * kUnit + i % kUnit);
            }
        } else {
            for (int32_t at = c; at < end; at += W * kUnit) {
                T u[kUnit];
                LoadUnit(row, at, end, u);
#pragma unroll
                for (int i = 0; i < kUnit; ++i) f(ToFloat(u[i]), at + i);
            }
        }
    }
};

// What a row's parts come to
struct RowResult {
    float m, logs;  // M and log S; 0 and infinity for a row of nothing but -inf
    bool none;
};
__device__ __forceinline__ RowResult Finish(const Part& p)
{
    if (p.s == 0.0f) return {0.0f, Infinity(), true};
    return {p.m, logf(p.s), false};
}

__device__ __forceinline__ int64_t Target(const void* targets, bool wide, int64_t row)
{
    return wide ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
}

template <typename T>
__device__ __forceinline__ void WriteRow(const LogprobsLaunch& p, int64_t row, const Part& part, const RowResult& r)
{
    if (p.logprobs != nullptr) {
        const int64_t t = Target(p.targets, p.wide, row);
        float value = 0.0f;
        if (t >= 0 && t < p.vocab) value = (ToFloat(static_cast<const T*>(p.logits)[row * p.ld + t]) - r.m) - r.logs;
        p.logprobs[row] = value;
    }
    if (p.entropy != nullptr) p.entropy[row] = r.none ? 0.0f : r.logs - part.w / part.s * 0.693147181f;
    if (p.stats != nullptr) {
        p.stats[row * 2] = r.m;
        p.stats[row * 2 + 1] = r.logs;
    }
}

template <int W>
struct Shared {
    Part part[W / 64];
    uint64_t pair[kCandidates];  // candidates; before that each group's largest
    uint64_t best[W / 64];
    uint16_t looking[W];  // threads that hold candidates
    uint32_t count, lookers;
    float threshold;
};

// The k largest of logits [begin, end), first ones first; write(rank, pair)
// for each, fewer than k where fewer are above -inf.  m: the thread's largest.
//
// The k-th largest of 64 or 128 groups' largest is a bound below which the answer
// has nothing: those groups of threads hold k logits at or above it.  (128 where
// 64 leave some empty: rows of 1025 to 2048 logits, more than the candidates, else
// had no bound; its ranks cost 0.6 us more of 256 threads.)  What is
// at or above the bound is listed, mostly little more than k logits, out of what
// the threads have seen whose largest is, and each finds its rank by comparing
// itself with all.  A row with NaN, or with more logits
// at the bound than fit (equal ones), goes through k passes instead.
template <typename T, int H, int W, typename Write>
__device__ __forceinline__ void TakeTop(Shared<W>& sh, const Held<T, H, W>& held, const T* row, int32_t begin, int32_t end,
                                        int32_t k, float m, bool nan, Write write)
{
    const int tid = threadIdx.x;
    if (tid == 0) sh.count = sh.lookers = 0;
    auto setBound = [&](auto lanes) {
        constexpr int G = decltype(lanes)::value;
        const int group = tid / G, lane = tid % G;
        const float most = MaxOverLanes<G>(m);
        if (lane == 0) sh.pair[group] = Pair(most, group);
        __syncthreads();
        // each lane of a group compares the group's with its share of the others
        uint32_t rank = 0;
        const uint64_t mine = sh.pair[group];
#pragma unroll
        for (int i = 0; i < W / G / G; ++i) rank += sh.pair[i * G + lane] > mine ? 1 : 0;
        rank = SumOverLanes<G>(rank);
        if (rank == static_cast<uint32_t>(k) - 1 && lane == 0) sh.threshold = most;
    };
    constexpr int kLanes = W / kMaxTop;
    if ((end - begin) / (kLanes * kUnit) >= k) setBound(std::integral_constant<int, kLanes>{});
    else setBound(std::integral_constant<int, kLanes / 2>{});
    __syncthreads();
    const float threshold = sh.threshold;
    if (!nan) {
        auto add = [&](float x, int32_t index) {
            if (x >= threshold) {
                const uint32_t at = atomicAdd(&sh.count, 1U);
                if (at < kCandidates) sh.pair[at] = Pair(x, index);
            }
        };
        if constexpr (H > 0) {
            if (m >= threshold) held.ForEach(row, begin, end, add);
        } else {
            // Few threads have seen any.  What they have read is read again, by all threads (1024 rows of 131072 fp32 with 5
            // alternatives 94 us, by those threads alone 103, the whole row again 180; with none 91).
            if (m >= threshold) sh.looking[atomicAdd(&sh.lookers, 1U)] = static_cast<uint16_t>(tid);
            __syncthreads();
            const uint32_t lookers = sh.lookers, rounds = (end - begin + W * kUnit - 1) / (W * kUnit);
            const uint32_t units = lookers * rounds;
            for (uint32_t first = tid; first < units; first += W * kBatch) {
                T u[kBatch][kUnit];
                int32_t at[kBatch];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const uint32_t n = first + b * W, round = n / lookers;
                    at[b] = n < units ? begin + static_cast<int32_t>((round * W + sh.looking[n - round * lookers]) * kUnit)
                                      : end;
                    LoadUnit(row, at[b], end, u[b]);
                }
#pragma unroll
                for (int i = 0; i < kBatch * kUnit; ++i) add(ToFloat(u[i / kUnit][i % kUnit]), at[i / kUnit] + i % kUnit);
            }
        }
        __syncthreads();
        const uint32_t count = sh.count;
        if (count <= kCandidates) {
            for (uint32_t c = tid; c < count; c += W) {
                const uint64_t pair = sh.pair[c];
                int above = 0;
#pragma unroll 8
                for (uint32_t i = 0; i < count; ++i) above += sh.pair[i] > pair ? 1 : 0;
                if (above < k) write(above, pair);
            }
            for (int32_t r = static_cast<int32_t>(count) + tid; r < k; r += W) write(r, uint64_t{0});
            return;
        }
    }
    uint64_t last = ~uint64_t{0};
    for (int32_t r = 0; r < k; ++r) {
        uint64_t best = 0;
        held.ForEach(row, begin, end, [&](float x, int32_t index) {
            const uint64_t pair = Pair(x, index);
            if (static_cast<uint32_t>(pair >> 32) > kKeyMinusInf && pair < last && pair > best) best = pair;
        });
        best = WaveMaxU64(best);
        __syncthreads();
        if ((tid & 63) == 0) sh.best[tid >> 6] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W / 64; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        if (tid == 0) write(r, best);
        last = best;  // 0: nothing is left, nor will be
    }
}

// pair 0: none
__device__ __forceinline__ void WriteTop(const LogprobsLaunch& p, int64_t row, int32_t rank, uint64_t pair, float m,
                                         float logs)
{
    p.top_ids[row * p.top + rank] = pair == 0 ? -1 : PairIndex(pair);
    p.top_logprobs[row * p.top + rank] = pair == 0 ? -Infinity() : (PairValue(pair) - m) - logs;
}

// The buffer: a part for each segment of each row, then the k largest of each.
__device__ __forceinline__ Part* PartOf(const LogprobsLaunch& p, int64_t at)
{
    return reinterpret_cast<Part*>(static_cast<char*>(p.buffer) + at * 16);
}
__device__ __forceinline__ uint64_t* PairsOf(const LogprobsLaunch& p, int64_t at, int32_t segments)
{
    return reinterpret_cast<uint64_t*>(static_cast<char*>(p.buffer) + p.rows * segments * 16) + at * p.top;
}

// A workgroup's part of a row, or all of it.  Where it is short enough a thread
// keeps its logits for the alternatives, in H units (one row of 131072 with 20:
// 11.2 us at the time; 12.3 read twice).  The target's logit is two loads, one
// after the other, at the end; loaded first, it was no sooner there.
template <typename T, bool kEntropy, int H, int W>
__global__ __launch_bounds__(W) void LogprobsKernel(LogprobsLaunch p, int32_t segments, int32_t length)
{
    __shared__ Shared<W> sh;
    const uint32_t number = BlockNumber();
    const int64_t row = number / static_cast<uint32_t>(segments);
    if (row >= p.rows) return;
    const int32_t segment = static_cast<int32_t>(number % static_cast<uint32_t>(segments));
    const T* logits = static_cast<const T*>(p.logits) + row * p.ld;
    const int32_t vocab = static_cast<int32_t>(p.vocab);
    const int32_t begin = segment * length, end = vocab - begin < length ? vocab : begin + length;
    Held<T, H, W> held;
    const Part mine = held.template Read<kEntropy>(logits, begin, end);
    const Part wave = WavePart(mine);
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = wave;
    __syncthreads();
    float most = kLowest;
#pragma unroll
    for (int w = 0; w < W / 64; ++w) most = fmaxf(most, sh.part[w].m);
    Part all{most, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W / 64; ++w) {
        Part one = sh.part[w];
        one.MoveTo(most);
        all.s += one.s;
        all.w += one.w;
    }
    if (segments == 1) {
        const RowResult r = Finish(all);
        if (threadIdx.x == 0) WriteRow<T>(p, row, all, r);
        if (p.top > 0) {
            TakeTop(sh, held, logits, begin, end, static_cast<int32_t>(p.top), mine.m, all.s != all.s,
                    [&](int32_t rank, uint64_t pair) { WriteTop(p, row, rank, pair, r.m, r.logs); });
        }
        return;
    }
    const int64_t at = row * segments + segment;
    if (threadIdx.x == 0) *PartOf(p, at) = all;
    if (p.top > 0) {
        uint64_t* pairs = PairsOf(p, at, segments);
        TakeTop(sh, held, logits, begin, end, static_cast<int32_t>(p.top), mine.m, all.s != all.s,
                [&](int32_t rank, uint64_t pair) { pairs[rank] = pair; });
    }
}

// Joins a row's segments, one per lane of the first wave, and their sorted lists.
//
// Of the k-th of all, a bound: where r = ceil(k / segments), the ceil(k / r)-th
// largest of the lists' r-th ones has k at or above it.  What is at or above the
// bound finds its rank by comparing itself with all of it, as in TakeTop.  Few
// alternatives, or too many at the bound, are taken one after another, the
// largest head of all lists each time: a lane holds its list's and the one behind
// it, so that a step waits for no memory.  Both launches with 5 alternatives of
// 32000 one after another 8.0 us, by the bound 9.1; 20 of 131072 11 and 10.4, 50
// 17.9 and 13.2.
constexpr int32_t kOneByOne = 12;
template <typename T>
__global__ __launch_bounds__(kThreads) void LogprobsJoinKernel(LogprobsLaunch p, int32_t segments)
{
    __shared__ uint64_t list[kMaxSegments * kMaxTop], candidate[kCandidates], bound;
    __shared__ uint32_t count;
    __shared__ RowResult result;
    const int64_t row = BlockNumber();
    if (row >= p.rows) return;
    const int tid = threadIdx.x;
    const int32_t k = static_cast<int32_t>(p.top);
    const bool mine = tid < segments;
    Part part{kLowest, 0.0f, 0.0f};
    if (mine) part = *PartOf(p, row * segments + tid);
    constexpr int kEach = kMaxSegments * kMaxTop / kThreads;
    uint64_t held[kEach] = {};
    if (k > 0) {
        const uint64_t* pairs = PairsOf(p, row * segments, segments);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * kThreads + tid < segments * k) held[i] = pairs[i * kThreads + tid];
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * kThreads + tid < segments * k) list[i * kThreads + tid] = held[i];
        }
        if (tid == 64) {
            bound = 1;  // 0 stands for none
            count = 0;
        }
        __syncthreads();
    }
    if (k > kOneByOne) {
        // four lanes compare a list's with a quarter of the others
        constexpr int G = kThreads / kMaxSegments;
        const int32_t r = (k + segments - 1) / segments, place = (k + r - 1) / r - 1;
        const int32_t own = tid / G, lane = tid % G;
        const uint64_t x = own < segments ? list[own * k + r - 1] : 0;
        uint32_t above = 0;
#pragma unroll
        for (int i = 0; i < kMaxSegments / G; ++i) {
            const int32_t s = i * G + lane;
            above += s < segments && list[s * k + r - 1] > x ? 1 : 0;
        }
        above = SumOverLanes<G>(above);
        if (above == static_cast<uint32_t>(place) && x != 0 && lane == 0) bound = x;
    }
    if (tid < 64) {
        part = WavePart(part);
        const RowResult r = Finish(part);
        if (tid == 0) {
            WriteRow<T>(p, row, part, r);
            result = r;
        }
    }
    if (k == 0) return;
    __syncthreads();
    const RowResult r = result;
    uint32_t found = kCandidates + 1;
    if (k > kOneByOne) {
        const uint64_t least = bound;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (held[i] >= least) {
                const uint32_t at = atomicAdd(&count, 1U);
                if (at < kCandidates) candidate[at] = held[i];
            }
        }
        __syncthreads();
        found = count;
    }
    if (found <= kCandidates) {
        for (uint32_t c = tid; c < found; c += kThreads) {
            const uint64_t pair = candidate[c];
            int32_t above = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < found; ++i) above += candidate[i] > pair ? 1 : 0;
            if (above < k) WriteTop(p, row, above, pair, r.m, r.logs);
        }
        for (int32_t rank = static_cast<int32_t>(found) + tid; rank < k; rank += kThreads) {
            WriteTop(p, row, rank, 0, r.m, r.logs);
        }
        return;
    }
    if (tid >= 64) return;
    int32_t at = tid * k + 1;
    const int32_t end = mine ? tid * k + k : 0;
    uint64_t head = mine ? list[tid * k] : 0, next = at < end ? list[at] : 0, taken = 0;
    for (int32_t rank = 0; rank < k; ++rank) {
        const uint64_t best = WaveMaxU64(head);
        if (tid == rank) taken = best;
        if (head == best) {  // one lane's, unless nothing is left
            head = next;
            ++at;
            next = at < end ? list[at] : 0;
        }
    }
    if (tid < k) WriteTop(p, row, tid, taken, r.m, r.logs);
}

constexpr int32_t kGradLength = kThreads * kUnit * kBatch;  // of a row that a workgroup takes

// The gradient of one part of a row, which may take the logits' place.  Columns
// that a token or an alternative names are written again, after the others, with
// what they have besides; their logits are read before any is written over.
template <typename T>
__global__ __launch_bounds__(kThreads) void LogprobsGradKernel(LogprobsGradLaunch p, int32_t segments)
{
    __shared__ int32_t column[kMaxTop + 1];
    __shared__ float weight[kMaxTop + 1];
    const uint32_t number = BlockNumber();
    const int64_t row = number / static_cast<uint32_t>(segments);
    if (row >= p.rows) return;
    const int32_t segment = static_cast<int32_t>(number % static_cast<uint32_t>(segments));
    const int32_t vocab = static_cast<int32_t>(p.vocab), k = p.grad_top != nullptr ? static_cast<int32_t>(p.top) : 0;
    const int32_t begin = segment * kGradLength, end = vocab - begin < kGradLength ? vocab : begin + kGradLength;
    const T* logits = static_cast<const T*>(p.logits) + row * p.ld;
    T* grad = static_cast<T*>(p.grad) + row * p.ld_grad;
    const int tid = threadIdx.x;
    T v[kBatch][kUnit];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) LoadUnit(logits, begin + (b * kThreads + tid) * kUnit, end, v[b]);
    float mine = 0.0f;  // the logit of this thread's named column
    if (tid <= k) {
        int64_t c = -1;
        float g = 0.0f;
        if (tid < k) {
            c = p.top_ids[row * p.top + tid];
            g = p.grad_top[row * p.top + tid];
        } else if (p.grad_logprobs != nullptr) {
            c = Target(p.targets, p.wide, row);
            g = p.grad_logprobs[row];
        }
        // a row of nothing but -inf has no gradient
        const bool named = c >= 0 && c < vocab && p.stats[row * 2 + 1] != Infinity();
        column[tid] = named ? static_cast<int32_t>(c) : -1;
        weight[tid] = named ? g : 0.0f;
        if (named && c >= begin && c < end) mine = ToFloat(logits[c]);
    }
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i <= k; ++i) total += weight[i];
    const float m = p.stats[row * 2], logs = p.stats[row * 2 + 1];
    const float gh = p.grad_entropy != nullptr ? p.grad_entropy[row] : 0.0f;
    const float h = p.grad_entropy != nullptr ? p.entropy[row] : 0.0f;
    auto one = [&](float x) {
        const float d = (x - m) - logs;
        return -Exp2(d * kLog2E) * (total + gh * (fmaxf(d, kFar) + h));
    };
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
        const int32_t c = begin + (b * kThreads + tid) * kUnit;
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[b][i] = FromFloat<T>(one(ToFloat(v[b][i])));
        if (c + kUnit <= end) {
            StoreStreaming<sizeof(v[b])>(grad + c, v[b]);
        } else {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) {
                if (c + i < end) grad[c + i] = v[b][i];
            }
        }
    }
    __syncthreads();  // the stores above come before those below
    if (tid <= k) {
        const int32_t c = column[tid];
        bool first = c >= begin && c < end;
        float g = 0.0f;
        for (int i = 0; i <= k; ++i) {
            if (column[i] != c) continue;
            if (i < tid) first = false;
            g += weight[i];
        }
        if (first) grad[c] = FromFloat<T>(g + one(mine));
    }
}

// How the rows are cut: segments of a row, their length (a multiple of a unit), threads of a workgroup.
//
// Up to 4096 logits are one workgroup's, and so are up to 32768 of up to 512 rows, with 1024 threads that hold them: 37
// rows of 32000 fp32 with 5 alternatives take 8.2 us, in segments and joined 10.1; 8000 with none 4.3 and 5.2; 512 rows
// of 32000 with 5 21 and 26, 1024 39 and 29 (of 8000 15 and 11).  Few rows without alternatives are joined faster, 16 of
// 32000 in 5.1 us where one workgroup each takes 5.5, but a row's sum should not change with what else is asked for.
// Longer rows are cut into as many segments as make a thousand workgroups, none shorter than a unit for each thread.
struct Cut {
    int32_t segments, length;
    bool wide;
};
Cut CutOf(int64_t rows, int64_t vocab)
{
    auto whole = [](int64_t n) { return static_cast<int32_t>((n + kUnit - 1) / kUnit * kUnit); };
    const bool wide = vocab > 4096 && vocab <= 1024 * kUnit * kBatch && rows <= 512;
    if (vocab <= 4096 || wide) return {1, whole(vocab), wide};
    const int64_t units = (vocab + kThreads * kUnit - 1) / (kThreads * kUnit), want = rows > 0 ? 1024 / rows : 1;
    int64_t s = want < units ? want : units;
    s = s > kMaxSegments ? kMaxSegments : s < 1 ? 1 : s;
    const int32_t length = whole((vocab + s - 1) / s);
    return {static_cast<int32_t>((vocab + length - 1) / length), length, false};
}

template <typename T>
int LaunchTyped(const LogprobsLaunch& l, hipStream_t s)
{
    const Cut cut = CutOf(l.rows, l.vocab);
    if (l.rows > INT32_MAX / cut.segments) return kTooLarge;
    auto launch = [&](auto held, auto threads) {
        constexpr int H = decltype(held)::value, W = decltype(threads)::value;
        const dim3 grid = GridOf(l.rows * cut.segments);
        if (l.entropy != nullptr) LogprobsKernel<T, true, H, W><<<grid, W, 0, s>>>(l, cut.segments, cut.length);
        else LogprobsKernel<T, false, H, W><<<grid, W, 0, s>>>(l, cut.segments, cut.length);
    };
    constexpr std::integral_constant<int, 0> none{};
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, kBatch> batch{};
    constexpr std::integral_constant<int, kThreads> threads{};
    constexpr std::integral_constant<int, 1024> many{};
    if (cut.wide) {
        if (cut.length <= 1024 * kUnit) launch(one, many);
        else launch(batch, many);
    } else if (cut.length <= kThreads * kUnit) {
        launch(one, threads);
    } else if (cut.length <= kThreads * kUnit * kBatch) {
        launch(batch, threads);
    } else {
        launch(none, threads);
    }
    if (cut.segments > 1) LogprobsJoinKernel<T><<<GridOf(l.rows), kThreads, 0, s>>>(l, cut.segments);
    return 0;
}

template <typename T>
int LaunchGradTyped(const LogprobsGradLaunch& l, hipStream_t s)
{
    const int64_t segments = (l.vocab + kGradLength - 1) / kGradLength;
    if (l.rows > INT32_MAX / segments) return kTooLarge;
    LogprobsGradKernel<T><<<GridOf(l.rows * segments), kThreads, 0, s>>>(l, static_cast<int32_t>(segments));
    return 0;
}

}  // namespace

size_t LogprobsBytes(int64_t rows, int64_t vocab, int64_t top)
{
    const int32_t segments = CutOf(rows, vocab).segments;
    return segments > 1 ? static_cast<size_t>(rows) * segments * (16 + 8 * top) : 0;
}

int LaunchLogprobs(const LogprobsLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.type == ACL_FLOAT) return LaunchTyped<float>(l, s);
    return l.type == ACL_FLOAT16 ? LaunchTyped<Half>(l, s) : LaunchTyped<Bf16>(l, s);
}

int LaunchLogprobsGrad(const LogprobsGradLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.type == ACL_FLOAT) return LaunchGradTyped<float>(l, s);
    return l.type == ACL_FLOAT16 ? LaunchGradTyped<Half>(l, s) : LaunchGradTyped<Bf16>(l, s);
}

}  // namespace aclsp
