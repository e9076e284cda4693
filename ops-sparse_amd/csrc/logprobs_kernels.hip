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
// once, for alternatives a second time out of the caches.  8192 rows of 65536
// bf16 logits with the entropy: 192 us (5.6 TB/s), their gradient 351 us (6.1
// TB/s read and written).  One row of 131072 with 20 alternatives, 64 segments:
// 4.6 us and 5.8 to join them, latency alone.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "experts_device.h"
#include "experts_internal.h"
#include "model_ops_internal.h"

namespace aclsp {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
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

constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E;
__device__ __forceinline__ float QuadMax(float x)
{
    x = fmaxf(x, __uint_as_float(Dpp<kQuadXor1, 0xF>(__float_as_uint(x), __float_as_uint(x))));
    return fmaxf(x, __uint_as_float(Dpp<kQuadXor2, 0xF>(__float_as_uint(x), __float_as_uint(x))));
}
__device__ __forceinline__ uint32_t QuadSum(uint32_t x)
{
    x += Dpp<kQuadXor1, 0xF>(x, x);
    return x + Dpp<kQuadXor2, 0xF>(x, x);
}

// The parts of a wave's lanes as one, in all lanes
__device__ __forceinline__ Part WavePart(Part p)
{
    p.MoveTo(WaveMax(p.m));
    return {p.m, WaveSum(p.s), WaveSum(p.w)};
}

// A logit as an unsigned key of the same order, NaN above all, and with the
// index behind it, the lower the greater: what comes first is the larger number.
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

// A thread's logits of [begin, end): H units that it holds where they fit, none for H = 0.
template <typename T, int H>
struct Held {
    T v[H > 0 ? H : 1][kUnit];

    template <bool kEntropy>
    __device__ __forceinline__ Part Read(const T* row, int32_t begin, int32_t end)
    {
        const int32_t c = begin + static_cast<int32_t>(threadIdx.x) * kUnit;
        Part p{kLowest, 0.0f, 0.0f};
        if constexpr (H > 0) {
#pragma unroll
            for (int b = 0; b < H; ++b) LoadUnit(row, c + b * kThreads * kUnit, end, v[b]);
            AddUnits<kEntropy>(p, v);
        } else {
            for (int32_t at = c; at < end; at += kThreads * kUnit * kBatch) {
                T u[kBatch][kUnit];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) LoadUnit(row, at + b * kThreads * kUnit, end, u[b]);
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
                f(ToFloat(v[i / kUnit][i % kUnit]), c + i / kUnit * kThreads * kUnit + i % kUnit);
            }
        } else {
            for (int32_t at = c; at < end; at += kThreads * kUnit) {
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

struct Shared {
    Part part[kWaves];
    uint64_t pair[kCandidates];  // candidates; before that each quad's largest
    uint64_t best[kWaves];
    uint32_t count;
    float threshold;
};

// The k largest of logits [begin, end), first ones first; write(rank, pair)
// for each, fewer than k where fewer are above -inf.  m: the thread's largest.
//
// The k-th largest of 64 quads' largest is a bound below which the answer has
// nothing: those quads hold k logits at or above it.  A second pass lists
// what is at or above the bound, mostly little more than k logits, and each finds
// its rank by comparing itself with all.  A row with NaN, or with more logits
// at the bound than fit (equal ones), goes through k passes instead.
template <typename T, int H, typename Write>
__device__ __forceinline__ void TakeTop(Shared& sh, const Held<T, H>& held, const T* row, int32_t begin, int32_t end,
                                        int32_t k, float m, bool nan, Write write)
{
    static_assert(kThreads == 4 * kMaxTop, "as many quads as there can be alternatives");
    const int tid = threadIdx.x;
    m = QuadMax(m);
    if ((tid & 3) == 0) sh.pair[tid >> 2] = Pair(m, tid >> 2);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    // each lane of a quad compares the quad's with a quarter of the others
    uint32_t rank = 0;
    const uint64_t mine = sh.pair[tid >> 2];
#pragma unroll
    for (int i = 0; i < kMaxTop / 4; ++i) rank += sh.pair[(tid & 3) * (kMaxTop / 4) + i] > mine ? 1 : 0;
    rank = QuadSum(rank);
    if (rank == static_cast<uint32_t>(k) - 1 && (tid & 3) == 0) sh.threshold = m;
    __syncthreads();
    const float threshold = sh.threshold;
    if (!nan) {
        held.ForEach(row, begin, end, [&](float x, int32_t index) {
            if (x >= threshold) {
                const uint32_t at = atomicAdd(&sh.count, 1U);
                if (at < kCandidates) sh.pair[at] = Pair(x, index);
            }
        });
        __syncthreads();
        const uint32_t count = sh.count;
        if (count <= kCandidates) {
            for (uint32_t c = tid; c < count; c += kThreads) {
                const uint64_t pair = sh.pair[c];
                int above = 0;
                for (uint32_t i = 0; i < count; ++i) above += sh.pair[i] > pair ? 1 : 0;
                if (above < k) write(above, pair);
            }
            for (int32_t r = static_cast<int32_t>(count) + tid; r < k; r += kThreads) write(r, uint64_t{0});
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
        for (int w = 0; w < kWaves; ++w) best = sh.best[w] > best ? sh.best[w] : best;
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

// Where a row's part is short enough a thread keeps its logits for the
// alternatives, in H units (one row of 131072 with 20: 11.2 us; 12.3 read twice).
template <typename T, bool kEntropy, int H>
__global__ __launch_bounds__(kThreads) void LogprobsKernel(LogprobsLaunch p, int32_t segments, int32_t length)
{
    __shared__ Shared sh;
    const uint32_t number = BlockNumber();
    const int64_t row = number / static_cast<uint32_t>(segments);
    if (row >= p.rows) return;
    const int32_t segment = static_cast<int32_t>(number % static_cast<uint32_t>(segments));
    const T* logits = static_cast<const T*>(p.logits) + row * p.ld;
    const int32_t vocab = static_cast<int32_t>(p.vocab);
    const int32_t begin = segment * length, end = vocab - begin < length ? vocab : begin + length;
    Held<T, H> held;
    const Part mine = held.template Read<kEntropy>(logits, begin, end);
    const Part wave = WavePart(mine);
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = wave;
    __syncthreads();
    float most = kLowest;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = fmaxf(most, sh.part[w].m);
    Part all{most, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
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

// Joins a row's segments, one per lane of the first wave; of the sorted lists the
// largest head is taken k times.  All waves bring the lists to LDS, and a lane
// holds its head and the one behind it: a step waits for no memory.
template <typename T>
__global__ __launch_bounds__(kThreads) void LogprobsJoinKernel(LogprobsLaunch p, int32_t segments)
{
    __shared__ uint64_t list[kMaxSegments * kMaxTop];
    const int64_t row = BlockNumber();
    if (row >= p.rows) return;
    const int tid = threadIdx.x;
    const int32_t k = static_cast<int32_t>(p.top);
    const bool mine = tid < segments;
    Part part{kLowest, 0.0f, 0.0f};
    if (mine) part = *PartOf(p, row * segments + tid);
    if (k > 0) {
        const uint64_t* pairs = PairsOf(p, row * segments, segments);
        constexpr int kEach = kMaxSegments * kMaxTop / kThreads;
        uint64_t held[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * kThreads + tid < segments * k) held[i] = pairs[i * kThreads + tid];
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * kThreads + tid < segments * k) list[i * kThreads + tid] = held[i];
        }
        __syncthreads();
    }
    if (tid >= 64) return;
    part = WavePart(part);
    const RowResult r = Finish(part);
    if (tid == 0) WriteRow<T>(p, row, part, r);
    if (k == 0) return;
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

// The gradient of one part of a row.  Columns that a token or an alternative
// names are written again, after the others, with what they have besides.
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
    T v[kBatch][kUnit];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) LoadUnit(logits, begin + (b * kThreads + tid) * kUnit, end, v[b]);
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
        if (first) grad[c] = FromFloat<T>(g + one(ToFloat(logits[c])));
    }
}

// Segments of a row: as many as make a thousand workgroups, none shorter than a unit for each thread.
int32_t Segments(int64_t rows, int64_t vocab)
{
    const int64_t units = (vocab + kThreads * kUnit - 1) / (kThreads * kUnit), want = rows > 0 ? 1024 / rows : 1;
    int64_t s = want < units ? want : units;
    s = s < kMaxSegments ? s : kMaxSegments;
    return static_cast<int32_t>(s < 1 ? 1 : s);
}

// Of a segment, a multiple of a unit
int32_t Length(int64_t vocab, int32_t segments)
{
    const int64_t each = (vocab + segments - 1) / segments;
    return static_cast<int32_t>((each + kUnit - 1) / kUnit * kUnit);
}

template <typename T>
int LaunchTyped(const LogprobsLaunch& l, hipStream_t s)
{
    int32_t segments = Segments(l.rows, l.vocab);
    const int32_t length = Length(l.vocab, segments);
    segments = static_cast<int32_t>((l.vocab + length - 1) / length);
    if (l.rows > INT32_MAX / segments) return kTooLarge;
    const dim3 grid = GridOf(l.rows * segments);
    auto launch = [&](auto held) {
        constexpr int H = decltype(held)::value;
        if (l.entropy != nullptr) LogprobsKernel<T, true, H><<<grid, kThreads, 0, s>>>(l, segments, length);
        else LogprobsKernel<T, false, H><<<grid, kThreads, 0, s>>>(l, segments, length);
    };
    if (length <= kThreads * kUnit) launch(std::integral_constant<int, 1>{});
    else if (length <= kThreads * kUnit * kBatch) launch(std::integral_constant<int, kBatch>{});
    else launch(std::integral_constant<int, 0>{});
    if (segments > 1) LogprobsJoinKernel<T><<<GridOf(l.rows), kThreads, 0, s>>>(l, segments);
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
    const int32_t segments = Segments(rows, vocab);
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
