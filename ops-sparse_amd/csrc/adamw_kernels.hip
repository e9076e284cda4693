// One AdamW step over many tensors, by the formulas of decoupled weight decay:
//   m = beta1 m + (1 - beta1) g           v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
// with m and v kept in fp32, or in 8 bits with a power of two for each block of
// 32 values.
//
// Bound by memory: every value that is kept is read once and written once.
// The moments' arithmetic is in fp32, each operation rounded by itself, so that
// 8-bit moments are the same as any other program's that takes the same steps.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "experts_device.h"
#include "model_ops_internal.h"

namespace aclsp {
namespace {

constexpr int kThreads = 256;
static_assert(kAdamWChunk == kThreads * 8, "eight values per thread");

// 8-bit floating point of a block that shares the exponent of its largest
// value: m has a sign, 4 bits of exponent and 3 behind the point, v, which is
// never negative, 5 and 3.  The least exponents leave room above the largest
// value, which lies under 2: rounding up from it never leaves the format.
// Codes under 8 are subnormal.
constexpr int kLeastM = -13, kLeastV = -29;

template <int kLeast>
__device__ __forceinline__ float Decode8(uint32_t magnitude)
{
    const float small = static_cast<float>(magnitude) * __uint_as_float((127U + kLeast - 3) << 23);
    const float normal = __uint_as_float((magnitude << 20) + ((126U + kLeast) << 23));
    return magnitude < 8 ? small : normal;
}

// The code of a in [0, 2), rounded up with the probability of what lies behind
// its bits, by 16 random ones.  Rounding to the nearest would lose the slow
// changes that the moments are made of: beta2 = 0.999 moves v by a hundredth of
// the distance between two codes.
template <int kLeast>
__device__ __forceinline__ uint32_t Encode8(float a, uint32_t random)
{
    constexpr uint32_t kFirst = static_cast<uint32_t>(kLeast + 127) << 3;
    const uint32_t add = (random << 4) + 8;
    const float least = __uint_as_float((127U + kLeast) << 23);
    const uint32_t normal = ((__float_as_uint(a) + add) >> 20) - kFirst + 8;
    const uint32_t small = ((__float_as_uint(a + least) + add) >> 20) - kFirst;
    return a < least ? small : normal;
}

__device__ __forceinline__ float Power(uint32_t e)  // 2^(e - 127), NaN for 255
{
    return __uint_as_float(e == 0 ? 0x00400000U : e == 255 ? 0x7FC00000U : e << 23);
}

constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E;
__device__ __forceinline__ uint32_t QuadMax(uint32_t x)
{
    const uint32_t y = Dpp<kQuadXor1, 0xF>(x, x);
    x = x > y ? x : y;
    const uint32_t z = Dpp<kQuadXor2, 0xF>(x, x);
    return x > z ? x : z;
}

// Scrambles 32 bits; the factors are the first bits of the roots of 13 and 19.
__device__ __forceinline__ uint32_t Mix(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x9B05688DU;
    x ^= x >> 15;
    x *= 0x5BE0CD19U;
    return x ^ (x >> 16);
}

// What all values of a launch share
struct Factors {
    float beta1, rest1, beta2, rest2, decay, size, root, eps, scale;
};

__device__ __forceinline__ double IntPower(double base, int32_t n)
{
    double r = 1.0;
    for (; n > 0; n >>= 1) {
        if (n & 1) r *= base;
        base *= base;
    }
    return r;
}

// Eight elements from `at` on, of which `left` are the tensor's.
template <typename T>
__device__ __forceinline__ void Load8(const T* from, int64_t left, float (&v)[8])
{
    T t[8];
    if (left >= 8) {
        __builtin_memcpy(t, from, sizeof(t));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ToFloat(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? ToFloat(from[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void Store8(T* to, int64_t left, const float (&v)[8])
{
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = FromFloat<T>(v[i]);
    if (left >= 8) {
        __builtin_memcpy(to, t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) to[i] = t[i];
        }
    }
}

template <int kLeast, bool kSigned>
__device__ __forceinline__ void Unpack(const uint8_t* codes, uint32_t e, float (&v)[8])
{
    uint8_t c[8];
    __builtin_memcpy(c, __builtin_assume_aligned(codes, 8), 8);
    const float scale = Power(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (kSigned) {
            const float a = Decode8<kLeast>(c[i] & 127U);
            v[i] = (c[i] >= 128 ? -a : a) * scale;
        } else {
            v[i] = Decode8<kLeast>(c[i]) * scale;
        }
    }
}

// shift: of the random bits
template <int kLeast, bool kSigned>
__device__ __forceinline__ void Pack(const float (&v)[8], const uint32_t (&random)[8], int shift, uint8_t* codes,
                                     uint8_t* exponent)
{
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7FFFFFFFU;
        most = bits > most ? bits : most;
    }
    const uint32_t e = QuadMax(most) >> 23;
    // a block that holds infinity or NaN is NaN
    const float inverse = e == 255 ? 0.0f : e == 254 ? __uint_as_float(0x00400000U) : __uint_as_float((254U - e) << 23);
    uint8_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = __uint_as_float(__float_as_uint(v[i]) & 0x7FFFFFFFU) * inverse;
        uint32_t code = Encode8<kLeast>(a, random[i] >> shift & 0xFFFF);
        if constexpr (kSigned) {
            code |= __float_as_uint(v[i]) >> 31 << 7;
        } else {
            if (code == 0 && a > 0.0f) code = 1;  // a v of zero under an m that is none would make the step m / eps
        }
        c[i] = static_cast<uint8_t>(e == 255 ? 0 : code);
    }
    __builtin_memcpy(__builtin_assume_aligned(codes, 8), c, 8);
    if ((threadIdx.x & 3) == 0) *exponent = static_cast<uint8_t>(e);
}

// A thread takes eight neighbouring values, so a quad a block; a workgroup
// 2048 at a time.  The chunks of all tensors are numbered in one row, and each
// wave finds a chunk's tensor by one comparison per lane.
//
// The step is counted on the device, so that a captured step counts with each
// replay: every workgroup reads it first, and the last to finish writes it.
template <typename TP, typename TG, int kBits, bool kMaster>
__global__ __launch_bounds__(kThreads) void AdamWKernel(AdamWTable table, AdamWScalars s)
{
#pragma clang fp contract(off)
    const int32_t step = s.step[0] + 1;
    Factors f;
    {
        const double lr = s.lr_device != nullptr ? static_cast<double>(*s.lr_device) : s.lr;
        f.beta1 = static_cast<float>(s.beta1);
        f.rest1 = static_cast<float>(1.0 - s.beta1);
        f.beta2 = static_cast<float>(s.beta2);
        f.rest2 = static_cast<float>(1.0 - s.beta2);
        f.decay = static_cast<float>(1.0 - lr * s.weight_decay);
        f.size = static_cast<float>(lr / (1.0 - IntPower(s.beta1, step)));
        f.root = static_cast<float>(sqrt(1.0 - IntPower(s.beta2, step)));
        f.eps = static_cast<float>(s.eps);
        f.scale = s.grad_scale != nullptr ? *s.grad_scale : 1.0f;
    }
    const uint32_t key = Mix(Mix(s.seed) + static_cast<uint32_t>(step));
    const int lane = threadIdx.x & 63;
    const uint32_t first = table.first[lane];
    for (uint32_t chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const int which = __popcll(__ballot(first <= chunk)) - 1;
        const AdamWTensor& t = table.tensor[which];
        const int64_t at = static_cast<int64_t>(chunk - table.first[which]) * kAdamWChunk + threadIdx.x * 8;
        const int64_t left = t.count - at, padded = (t.count + 31) / 32 * 32;
        if (at >= padded) continue;  // whole quads
        float g[8], p[8], m[8], v[8];
        Load8(static_cast<const TG*>(t.grad) + at, left, g);
        if constexpr (kMaster) {
            Load8(t.master + at, left, p);
        } else {
            Load8(static_cast<const TP*>(t.param) + at, left, p);
        }
        uint8_t *codesM = nullptr, *codesV = nullptr, *expM = nullptr, *expV = nullptr;
        float *heldM = nullptr, *heldV = nullptr;
        if constexpr (kBits == 8) {
            codesM = static_cast<uint8_t*>(t.moments) + at;
            codesV = codesM + padded;
            expM = t.exponents + at / 32;
            expV = expM + padded / 32;
            Unpack<kLeastM, true>(codesM, *expM, m);
            Unpack<kLeastV, false>(codesV, *expV, v);
        } else {
            heldM = static_cast<float*>(t.moments) + at;
            heldV = heldM + padded;
            __builtin_memcpy(m, heldM, sizeof(m));
            __builtin_memcpy(v, heldV, sizeof(v));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float grad = g[i] * f.scale;
            const float keptM = m[i] * f.beta1, newM = grad * f.rest1;
            m[i] = keptM + newM;
            const float keptV = v[i] * f.beta2, square = grad * grad, newV = square * f.rest2;
            v[i] = keptV + newV;
            const float denominator = sqrtf(v[i]) / f.root + f.eps;
            const float kept = p[i] * f.decay, change = f.size * (m[i] / denominator);
            p[i] = kept - change;
        }
        if constexpr (kBits == 8) {
            // past the tensor's end the block holds zeros
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= left) m[i] = v[i] = 0.0f;
            }
            uint32_t random[8];
            const uint32_t low = static_cast<uint32_t>(at);
            const uint32_t seed = Mix(key + static_cast<uint32_t>(table.place[which]) +
                                      static_cast<uint32_t>(static_cast<uint64_t>(at) >> 32));
#pragma unroll
            for (int i = 0; i < 8; ++i) random[i] = Mix(low + i + seed);
            Pack<kLeastM, true>(m, random, 0, codesM, expM);
            Pack<kLeastV, false>(v, random, 16, codesV, expV);
        } else {
            Store8(heldM, left, m);
            Store8(heldV, left, v);
        }
        if constexpr (kMaster) Store8(t.master + at, left, p);
        Store8(static_cast<TP*>(t.param) + at, left, p);
    }
    if (!s.last) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        const int32_t done = __hip_atomic_fetch_add(&s.step[1], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (done == static_cast<int32_t>(gridDim.x) - 1) {
            __hip_atomic_store(&s.step[0], step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(&s.step[1], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

__global__ __launch_bounds__(kThreads) void AdamWMomentsKernel(AdamWTable table)
{
    const int lane = threadIdx.x & 63;
    const uint32_t first = table.first[lane];
    for (uint32_t chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const int which = __popcll(__ballot(first <= chunk)) - 1;
        const AdamWTensor& t = table.tensor[which];
        const int64_t at = static_cast<int64_t>(chunk - table.first[which]) * kAdamWChunk + threadIdx.x * 8;
        const int64_t left = t.count - at, padded = (t.count + 31) / 32 * 32;
        if (left <= 0) continue;
        const uint8_t* codes = static_cast<const uint8_t*>(t.moments) + at;
        const uint8_t* exponent = t.exponents + at / 32;
        float m[8], v[8];
        Unpack<kLeastM, true>(codes, *exponent, m);
        Unpack<kLeastV, false>(codes + padded, exponent[padded / 32], v);
        Store8(t.master + at, left, m);
        Store8(t.master + t.count + at, left, v);
    }
}

uint32_t Grid(uint32_t chunks)
{
    // as many workgroups as the chip holds: each takes several chunks where there are more
    constexpr uint32_t kMost = 256 * 8;
    return chunks < kMost ? chunks : kMost;
}

template <typename TP, typename TG>
void Launch(const AdamWTable& t, const AdamWScalars& s, int bits, bool master, hipStream_t stream)
{
    const uint32_t grid = Grid(t.chunks > 0 ? t.chunks : 1);
    if (bits == 8) {
        if (master) AdamWKernel<TP, TG, 8, true><<<grid, kThreads, 0, stream>>>(t, s);
        else AdamWKernel<TP, TG, 8, false><<<grid, kThreads, 0, stream>>>(t, s);
    } else {
        if (master) AdamWKernel<TP, TG, 32, true><<<grid, kThreads, 0, stream>>>(t, s);
        else AdamWKernel<TP, TG, 32, false><<<grid, kThreads, 0, stream>>>(t, s);
    }
}

template <typename TP>
void LaunchParam(const AdamWTable& t, const AdamWScalars& s, aclDataType grad, int bits, bool master, hipStream_t stream)
{
    if (grad == ACL_FLOAT) Launch<TP, float>(t, s, bits, master, stream);
    else if (grad == ACL_FLOAT16) Launch<TP, Half>(t, s, bits, master, stream);
    else Launch<TP, Bf16>(t, s, bits, master, stream);
}

}  // namespace

int LaunchAdamW(const AdamWTable& t, const AdamWScalars& s, aclDataType param, aclDataType grad, int bits, bool master,
                void* stream)
{
    hipStream_t q = static_cast<hipStream_t>(stream);
    if (param == ACL_FLOAT) LaunchParam<float>(t, s, grad, bits, master, q);
    else if (param == ACL_FLOAT16) LaunchParam<Half>(t, s, grad, bits, master, q);
    else LaunchParam<Bf16>(t, s, grad, bits, master, q);
    return 0;
}

int LaunchAdamWMoments(const AdamWTable& t, void* stream)
{
    AdamWMomentsKernel<<<Grid(t.chunks), kThreads, 0, static_cast<hipStream_t>(stream)>>>(t);
    return 0;
}

}  // namespace aclsp
