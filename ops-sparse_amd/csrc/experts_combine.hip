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

constexpr int kThreads = 256;

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

// VEC columns of one token per thread, 16 bytes of the output: a row's parts
// are read whole wherever they lie.  Bound by memory: 16384 tokens of 8 rows of
// 2048, bfloat16, 137 us for 604 MB, 4.4 TB/s (a copy reaches 5.05, reading
// alone 3.9).
template <typename TIn, typename TOut, int VEC>
__global__ __launch_bounds__(kThreads) void CombineKernel(CombineLaunch p, int32_t chunks)
{
    const int64_t t = blockIdx.x / static_cast<uint32_t>(chunks);
    const int64_t c = (static_cast<int64_t>(blockIdx.x % static_cast<uint32_t>(chunks)) * kThreads + threadIdx.x) * VEC;
    if (c >= p.width) return;
    const int k = static_cast<int>(p.k);
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

// One wave per assignment, which reads its token's dout (from L2 after the
// first of the token's k), its own row of y once, and writes its row of dy; dw
// is the wave's own sum, so nothing is added across waves.  Assignment number
// a also clears row a of dy when that row belongs to no group.  Bound by
// memory: 16384 tokens of 8 rows of 2048, bfloat16, 214 us for 1.14 GB, 5.3
// TB/s.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void CombineGradKernel(CombineGradLaunch p)
{
    const int lane = threadIdx.x & 63;
    const int64_t a = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    const int64_t assignments = p.tokens * p.k;
    T* gy = static_cast<T*>(p.grad_y);
    if (a < assignments) {
        const int32_t place = p.places[a];
        float dot = 0.0f;
        if (place >= 0 && place < p.rows) {
            const float w = p.weights != nullptr ? p.weights[a] : 1.0f;
            const T* go =
                static_cast<const T*>(p.grad_out) + static_cast<uint32_t>(a) / static_cast<uint32_t>(p.k) * p.ldo;
            const T* y = p.grad_weights != nullptr ? static_cast<const T*>(p.y) + place * p.ldy : nullptr;
            for (int64_t c = lane * VEC; c < p.width; c += 64 * VEC) {
                const auto g = LoadPack<T, VEC>(go + c);
                if (y != nullptr) {
                    const auto v = LoadPack<T, VEC>(y + c);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) dot = fmaf(ToFloat(g.v[i]), ToFloat(v.v[i]), dot);
                }
                if (gy != nullptr) {
                    Pack<T, VEC> d;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) d.v[i] = FromFloat<T>(w * ToFloat(g.v[i]));
                    StorePack<T, VEC>(gy + place * p.ld_grad_y + c, d);
                }
            }
        }
        if (p.grad_weights != nullptr) {
            dot = WaveSum(dot);
            if (lane == 0) p.grad_weights[a] = dot;
        }
    }
    if (gy != nullptr && a < p.rows && a >= p.offsets[p.groups]) {
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
    const uint32_t grid = static_cast<uint32_t>(l.tokens * chunks);
    if (wide) {
        CombineKernel<TIn, TOut, VEC><<<grid, kThreads, 0, s>>>(l, static_cast<int32_t>(chunks));
    } else {
        CombineKernel<TIn, TOut, 1><<<grid, kThreads, 0, s>>>(l, static_cast<int32_t>(chunks));
    }
    return 0;
}

template <typename T>
int CombineGradTyped(const CombineGradLaunch& l, hipStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = l.width % VEC == 0 && Aligned(l.y, l.ldy, sizeof(T), 16) &&
                      Aligned(l.grad_out, l.ldo, sizeof(T), 16) && Aligned(l.grad_y, l.ld_grad_y, sizeof(T), 16);
    const int64_t count = l.tokens * l.k > l.rows ? l.tokens * l.k : l.rows;
    const uint32_t grid = static_cast<uint32_t>((count + kThreads / 64 - 1) / (kThreads / 64));
    if (wide) {
        CombineGradKernel<T, VEC><<<grid, kThreads, 0, s>>>(l);
    } else {
        CombineGradKernel<T, 1><<<grid, kThreads, 0, s>>>(l);
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
    return l.type == ACL_FLOAT16 ? CombineGradTyped<Half>(l, s) : CombineGradTyped<Bf16>(l, s);
}

}  // namespace aclsp
