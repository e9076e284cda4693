// Combination of the experts' rows: out_t = sum_j w[t,j] * y[places[t,j]],
// a product with the routing matrix, and its gradients dy[places[t,j]] =
// w[t,j] * dout_t and dw[t,j] = <dout_t, y[places[t,j]]>.  Both pass over
// every row once and are bound by memory.  Sums are in 32 bits in the order
// of j (of the lanes for dw), without atomics.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "experts_device.h"
#include "experts_internal.h"

namespace aclsp {
namespace {

constexpr int kThreads = 256;  // as GridOf takes them

template <typename T, int N>
struct Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> LoadPack(const T* p)
{
    Pack<T, N> out;
    __builtin_memcpy(&out, __builtin_assume_aligned(p, sizeof(out)), sizeof(out));
    return out;
}

template <typename T, int N>
__device__ __forceinline__ void StorePack(T* p, const Pack<T, N>& v)
{
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(v)), &v, sizeof(v));
}

// The lists of the assignments that name each row, for gradients of any places: head[r] is one of row r's and next[a]
// another of the row that a names, or whatever the memory held: neither array is cleared before.  An entry counts only
// where it is an assignment that names the row (Names).  That is enough, as every assignment of a
// row enters its list: what the first to enter finds in head[r] is either no assignment of the row or one that the
// list holds as well.
struct Lists {
    int32_t* head;
    int32_t* next;
};
// Enters assignments [first, end), one per thread at a time, `threads` of them apart.
__device__ __forceinline__ void EnterPlaces(const Lists& l, const int32_t* places, int64_t rows, int64_t first,
                                            int64_t end, int64_t threads)
{
    for (int64_t a = first; a < end; a += threads) {
        const int32_t place = places[a];
        if (place >= 0 && place < rows) l.next[a] = atomicExch(&l.head[place], static_cast<int32_t>(a));
    }
}

// VEC columns of one token per thread, 16 bytes of the output: a row's parts
// are read whole wherever they lie.  With lists a token's first workgroup in
// every kListed tokens enters the assignments of all of them: the exchanges come
// back late, and a workgroup waits for them.  Bound by memory: 16384 tokens of 8
// rows of 2048, bfloat16, 136 us for 604 MB, 4.4 TB/s (a copy reaches 5.05,
// reading alone 3.9); with the lists 138 (142 where every token's workgroup
// enters its own, 158 where kListed is 32 and one die gets all that wait).
constexpr int kListed = 31;  // odd, so that they are dealt to all dies
template <typename TIn, typename TOut, int VEC>
__global__ __launch_bounds__(kThreads) void CombineKernel(CombineLaunch p, int32_t chunks)
{
    const uint32_t block = BlockNumber();
    const int64_t t = block / static_cast<uint32_t>(chunks);
    const int64_t c = (static_cast<int64_t>(block % static_cast<uint32_t>(chunks)) * kThreads + threadIdx.x) * VEC;
    if (t >= p.tokens) return;
    const int k = static_cast<int>(p.k);
    if (p.head != nullptr && t % kListed == 0 && block % static_cast<uint32_t>(chunks) == 0) {
        const int64_t end = t + kListed < p.tokens ? t + kListed : p.tokens;
        EnterPlaces({p.head, p.next}, p.places, p.rows, t * k + threadIdx.x, end * k, kThreads);
    }
    if (c >= p.width) return;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    for (int j = 0; j < k; ++j) {
        const int32_t place = p.places[t * k + j];
        if (place < 0 || place >= p.rows) continue;  // a dropped assignment adds nothing
        const float w = p.weights != nullptr ? p.weights[t * k + j] : 1.0f;
        const auto y = LoadPack<TIn, VEC>(static_cast<const TIn*>(p.y) + place * p.ldy + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w, ToFloat(y.v[i]), acc[i]);
    }
    Pack<TOut, VEC> out;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out.v[i] = FromFloat<TOut>(acc[i]);
    StorePack<TOut, VEC>(static_cast<TOut*>(p.out) + t * p.ldo + c, out);
}

// The lists alone, where the product did not make them.  The same assignments: 5.5 us.
__global__ __launch_bounds__(kThreads) void ListPlacesKernel(CombineGradLaunch p)
{
    EnterPlaces({p.head, p.next}, p.places, p.rows, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x,
                p.tokens * p.k, static_cast<int64_t>(gridDim.x) * kThreads);
}

struct CombineGradLists {
    const CombineGradLaunch& p;
    int64_t assignments;

    // without a branch, so that what follows need not wait for the load
    __device__ __forceinline__ bool Names(int32_t a, int64_t row) const
    {
        const bool in = a >= 0 && a < assignments;
        return (p.places[in ? a : 0] == row) & in;
    }
};

// dy of a row that several assignments name, a at the head of their list, by one wave: the sum of their parts in
// fp32 in the order of the assignments, whatever the list's.  A list of more than a wave's lanes is left, and the
// places are searched for its assignments.
template <typename T, int VEC>
__device__ void SumSharedRow(const CombineGradLaunch& p, const CombineGradLists& lists, int32_t a, int32_t place)
{
    const int lane = threadIdx.x & 63;
    int32_t mine = -1, count = 0, at = a;
    bool searched = false;
    while (true) {
        if (lane == count) mine = at;
        ++count;
        at = p.next[at];
        if (!lists.Names(at, place) || __any(mine == at)) break;
        if (count == 64) {
            searched = true;
            break;
        }
    }
    int32_t rank = 0;
    for (int i = 0; i < count; ++i) rank += __builtin_amdgcn_readlane(mine, i) < mine ? 1 : 0;
    if (lane >= count) rank = -1;
    for (int64_t c0 = 0; c0 < p.width; c0 += 64 * VEC) {
        const int64_t c = c0 + lane * VEC;
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        auto add = [&](int64_t other) {
            if (c >= p.width) return;
            const float w = p.weights != nullptr ? p.weights[other] : 1.0f;
            const auto g = LoadPack<T, VEC>(static_cast<const T*>(p.grad_out) + other / p.k * p.ldo + c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w, ToFloat(g.v[i]), acc[i]);
        };
        if (searched) {
            for (int64_t first = 0; first < lists.assignments; first += 64) {
                const bool named = first + lane < lists.assignments && p.places[first + lane] == place;
                for (uint64_t left = __ballot(named); left != 0; left &= left - 1) add(first + __builtin_ctzll(left));
            }
        } else {
            for (int i = 0; i < count; ++i) add(__builtin_amdgcn_readlane(mine, __builtin_ctzll(__ballot(rank == i))));
        }
        if (c < p.width) {
            Pack<T, VEC> d;
#pragma unroll
            for (int i = 0; i < VEC; ++i) d.v[i] = FromFloat<T>(acc[i]);
            StorePack<T, VEC>(static_cast<T*>(p.grad_y) + place * p.ld_grad_y + c, d);
        }
    }
}

// One wave per assignment, which reads its token's dout (from L2 after the
// first of the token's k), its own row of y once, and writes its row of dy; dw
// is the wave's own sum, so nothing is added across waves.  Wave number r also
// clears row r of dy where the row has no assignment.  With kAny those are the
// rows that no place names, and the head of a row's list writes it; without,
// the rows past the last group, as in a plan whose places name each row before
// them once.  Bound by memory: 16384 tokens of 8 rows of 2048, bfloat16, 211 to
// 218 us with kAny for 1.14 GB, 5.3 TB/s (with the list looked up before the
// row's first loads 236 to 241 us: a chain of three dependent loads of each wave
// that nothing hid).
template <typename T, int VEC, bool kAny>
__global__ __launch_bounds__(kThreads) void CombineGradKernel(CombineGradLaunch p)
{
    const int lane = threadIdx.x & 63;
    const int64_t a = static_cast<int64_t>(BlockNumber()) * (kThreads / 64) + (threadIdx.x >> 6);
    const int64_t assignments = p.tokens * p.k;
    const CombineGradLists lists{p, assignments};
    T* gy = static_cast<T*>(p.grad_y);
    bool unnamed = false;  // row a has no assignment
    if (gy != nullptr && a < p.rows) {
        if constexpr (kAny) {
            unnamed = assignments == 0 || !lists.Names(p.head[a], a);
        } else {
            unnamed = a >= p.offsets[p.groups];
        }
    }
    if (a < assignments) {
        const int32_t place = p.places[a];
        float dot = 0.0f;
        if (place >= 0 && place < p.rows) {
            const float w = p.weights != nullptr ? p.weights[a] : 1.0f;
            const T* go =
                static_cast<const T*>(p.grad_out) + static_cast<uint32_t>(a) / static_cast<uint32_t>(p.k) * p.ldo;
            const T* y = p.grad_weights != nullptr ? static_cast<const T*>(p.y) + place * p.ldy : nullptr;
            // the row's first part is asked for before anything is known of its list, each next one before the last
            // one's store
            int64_t c = lane * VEC;
            Pack<T, VEC> g{}, v{};
            auto load = [&] {
                if (c >= p.width) return;
                g = LoadPack<T, VEC>(go + c);
                if (y != nullptr) v = LoadPack<T, VEC>(y + c);
            };
            load();
            bool only = gy != nullptr, first = false;
            if constexpr (kAny) {
                if (gy != nullptr) {
                    const int32_t other = p.next[a];
                    const bool listed = p.head[place] == a;
                    const bool shared = lists.Names(other, place) & (other != a);
                    only = listed & !shared;
                    first = listed & shared;
                }
            } else {
                only = gy != nullptr && place < p.offsets[p.groups];
            }
            while (c < p.width) {
                const auto g0 = g, v0 = v;
                T* to = gy + place * p.ld_grad_y + c;
                c += 64 * VEC;
                load();
                if (y != nullptr) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) dot = fmaf(ToFloat(g0.v[i]), ToFloat(v0.v[i]), dot);
                }
                if (only) {
                    Pack<T, VEC> d;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) d.v[i] = FromFloat<T>(w * ToFloat(g0.v[i]));
                    StorePack<T, VEC>(to, d);
                }
            }
            if constexpr (kAny) {
                if (__any(first)) SumSharedRow<T, VEC>(p, lists, static_cast<int32_t>(a), place);
            }
        }
        if (p.grad_weights != nullptr) {
            dot = WaveSum(dot);
            if (lane == 0) p.grad_weights[a] = dot;
        }
    }
    if (unnamed) {
        Pack<T, VEC> zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.v[i] = FromFloat<T>(0.0f);
        for (int64_t c = lane * VEC; c < p.width; c += 64 * VEC) StorePack<T, VEC>(gy + a * p.ld_grad_y + c, zero);
    }
}

bool Aligned(const void* p, int64_t ld, size_t bytes, size_t pack)
{
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % pack == 0 && static_cast<size_t>(ld) * bytes % pack == 0);
}

template <typename TIn, typename TOut>
int CombineTyped(const CombineLaunch& l, hipStream_t s)
{
    constexpr int VEC = 16 / sizeof(TOut);
    const bool wide = l.width % VEC == 0 && Aligned(l.y, l.ldy, sizeof(TIn), VEC * sizeof(TIn)) &&
                      Aligned(l.out, l.ldo, sizeof(TOut), 16);
    const int64_t per = static_cast<int64_t>(kThreads) * (wide ? VEC : 1);
    const int64_t chunks = (l.width + per - 1) / per;
    if (l.tokens > INT32_MAX / chunks) return kTooLarge;
    const dim3 grid = GridOf(l.tokens * chunks);
    if (wide) {
        CombineKernel<TIn, TOut, VEC><<<grid, kThreads, 0, s>>>(l, static_cast<int32_t>(chunks));
    } else {
        CombineKernel<TIn, TOut, 1><<<grid, kThreads, 0, s>>>(l, static_cast<int32_t>(chunks));
    }
    return 0;
}

template <typename T, bool kAny>
int CombineGradTyped(const CombineGradLaunch& l, hipStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = l.width % VEC == 0 && Aligned(l.y, l.ldy, sizeof(T), 16) &&
                      Aligned(l.grad_out, l.ldo, sizeof(T), 16) && Aligned(l.grad_y, l.ld_grad_y, sizeof(T), 16);
    const int64_t count = l.tokens * l.k > l.rows ? l.tokens * l.k : l.rows;
    const dim3 grid = GridOf((count + kThreads / 64 - 1) / (kThreads / 64));
    if (kAny && !l.listed && l.grad_y != nullptr && l.tokens > 0) {
        const int64_t blocks = (l.tokens * l.k + kThreads - 1) / kThreads;
        ListPlacesKernel<<<static_cast<uint32_t>(blocks < 4096 ? blocks : 4096), kThreads, 0, s>>>(l);
    }
    if (wide) {
        CombineGradKernel<T, VEC, kAny><<<grid, kThreads, 0, s>>>(l);
    } else {
        CombineGradKernel<T, 1, kAny><<<grid, kThreads, 0, s>>>(l);
    }
    return 0;
}

}  // namespace

int LaunchCombine(const CombineLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.out_type == ACL_FLOAT16) {
        return l.y_type == ACL_FLOAT ? CombineTyped<float, Half>(l, s) : CombineTyped<Half, Half>(l, s);
    }
    return l.y_type == ACL_FLOAT ? CombineTyped<float, Bf16>(l, s) : CombineTyped<Bf16, Bf16>(l, s);
}

int LaunchCombineGrad(const CombineGradLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.offsets == nullptr) {
        return l.type == ACL_FLOAT16 ? CombineGradTyped<Half, true>(l, s) : CombineGradTyped<Bf16, true>(l, s);
    }
    return l.type == ACL_FLOAT16 ? CombineGradTyped<Half, false>(l, s) : CombineGradTyped<Bf16, false>(l, s);
}

}  // namespace aclsp
