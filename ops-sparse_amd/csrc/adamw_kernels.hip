// One AdamW step over many tensors, by the formulas of decoupled weight decay:
//   m = beta1 m + (1 - beta1) g           v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
// with m and v kept in fp32, or in 8 bits with a power of two for each block of
// 32 values.
//
// Bound by memory: every value that is kept is read once and written once.
// 201 M values in bf16 with fp32 masters and moments: 1.08 ms, 5.2 TB/s, the
// rate of a copy; 67 M with 8-bit moments and no masters: 123 us (680 MB, 5.5
// TB/s), and 105 us to take the moments out in fp32 (675 MB, 6.4 TB/s).
// The moments' arithmetic is in fp32, each operation rounded by itself, so that
// 8-bit moments are the same as any other program's that takes the same steps.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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
//
// A magnitude's bits, moved to the last three of fp32's exponent's bits and
// the first three behind it, are a float 2^(126 + least) times too small,
// subnormal where the code is: one product decodes or aligns both kinds.
constexpr int kLeastM = -13, kLeastV = -29;

template <int kLeast>
__device__ __forceinline__ float Decode8(uint32_t bits)  // of the magnitude, from bit 20 on, and the sign
{
    return __uint_as_float(bits) * __uint_as_float(static_cast<uint32_t>(253 + kLeast) << 23);
}

// The code of a in [0, 2), rounded up with the probability of what lies behind
// its bits, by 16 random ones (at bit 4; with 8 they are the middle of their
// range).  Rounding to the nearest would lose the slow changes that the moments
// are made of: beta2 = 0.999 moves v by a hundredth of the distance between two
// codes.
template <int kLeast>
__device__ __forceinline__ uint32_t Encode8(float a, uint32_t random)
{
    const float aligned = a * __uint_as_float(static_cast<uint32_t>(1 - kLeast) << 23);
    return (__float_as_uint(aligned) + random + 8) >> 20;
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

// Scrambles 32 bits.
__device__ __forceinline__ uint32_t Mix(uint32_t x, const AdamWMix& by)
{
    x ^= x >> 16;
    x *= by.first;
    x ^= x >> 15;
    x *= by.second;
    return x ^ (x >> 16);
}

// What all values of a step share, in the caller's buffer
struct Factors {
    float beta1, rest1, beta2, rest2, decay, size, inverse_root, eps, scale;
    uint32_t key;
    AdamWMix mix;
};
static_assert(sizeof(Factors) <= kAdamWBufferBytes, "");

// size * m / (sqrt(v) / root + eps), to 11 roundings: the square root and the
// reciprocal are the instructions' (one unit in the last place each).  They
// take no subnormal numbers, so v is at least the least normal one: its root is
// under 2^-62, which an eps of 1e-8 does not see.  By a comparison, which NaN
// passes: the larger of NaN and a number would be the number, and the change
// m / eps.
__device__ __forceinline__ float Change(const Factors& f, float m, float v)
{
    constexpr float kLeast = 1.17549435e-38f;
    const float root = __builtin_amdgcn_sqrtf(v < kLeast ? kLeast : v);
    return f.size * (m * __builtin_amdgcn_rcpf(root * f.inverse_root + f.eps));
}

// 1 / x and 1 / sqrt(x) to about a unit in the last place, by Newton's steps from the instructions' estimates.
__device__ __forceinline__ double Reciprocal(double x)
{
    double r = __builtin_amdgcn_rcp(x);
    for (int i = 0; i < 2; ++i) r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
    return r;
}
__device__ __forceinline__ double InverseRoot(double x)
{
    double r = __builtin_amdgcn_rsq(x);
    for (int i = 0; i < 2; ++i) r = __builtin_fma(__builtin_fma(-x * r, r, 1.0), 0.5 * r, r);
    return r;
}

// Counts the step and works out its factors, in 64 bits: done by each workgroup
// of the step itself they took as long as its values.  Its time is that of
// fetching its instructions, which no cache holds: 1.6 us, with the compiler's
// division and square root 4.6.
__global__ void AdamWFactorsKernel(AdamWScalars s, Factors* out)
{
    const int32_t step = s.step[0] + 1;
    const double lr = s.lr_device != nullptr ? static_cast<double>(*s.lr_device) : s.lr;
    double power1 = 1.0, power2 = 1.0, base1 = s.beta1, base2 = s.beta2;
    for (int32_t n = step; n > 0; n >>= 1) {
        if (n & 1) {
            power1 *= base1;
            power2 *= base2;
        }
        base1 *= base1;
        base2 *= base2;
    }
    Factors f;
    f.beta1 = static_cast<float>(s.beta1);
    f.rest1 = static_cast<float>(1.0 - s.beta1);
    f.beta2 = static_cast<float>(s.beta2);
    f.rest2 = static_cast<float>(1.0 - s.beta2);
    f.decay = static_cast<float>(1.0 - lr * s.weight_decay);
    f.size = static_cast<float>(lr * Reciprocal(1.0 - power1));
    f.inverse_root = static_cast<float>(InverseRoot(1.0 - power2));
    f.eps = static_cast<float>(s.eps);
    f.scale = s.grad_scale != nullptr ? *s.grad_scale : 1.0f;
    f.key = Mix(Mix(s.seed, s.mix) + static_cast<uint32_t>(step), s.mix);
    f.mix = s.mix;
    *out = f;
    s.step[0] = step;
}

// V elements, of which `left` are the tensor's.
template <typename T, int V>
__device__ __forceinline__ void Load(const T* from, int64_t left, float (&v)[V])
{
    T t[V];
    if (left >= V) {
        __builtin_memcpy(t, from, sizeof(t));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = ToFloat(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < left ? ToFloat(from[i]) : 0.0f;
    }
}
template <bool kStream, typename T, int V>
__device__ __forceinline__ void Store(T* to, int64_t left, const float (&v)[V])
{
    T t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = FromFloat<T>(v[i]);
    if (left >= V) {
        StoreStreaming<sizeof(t), kStream>(to, t);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i < left) to[i] = t[i];
        }
    }
}

// Launches of more chunks store their results past the L2.  Small ones are soon read again, and storing them takes as long
// either way: a step and the next read of its bf16 parameters, past the L2 / by ordinary stores, 2^18 values with 8-bit
// moments 8.6 / 8.4 us, 2^19 9.1 / 8.9, 2^20 10.8 / 10.8, 2^22 (32 bits) 31.3 / 34.0; moments' values 2^12 4.3 / 4.0,
// 2^18 5.6 / 5.4, 2^20 10.6 / 10.8.
constexpr uint32_t kOrdinaryChunks = 256;

// V codes from one or two words
template <int kLeast, bool kSigned, int V>
__device__ __forceinline__ void Unpack(const uint8_t* codes, uint32_t e, float (&v)[V])
{
    uint32_t word[V / 4];
    __builtin_memcpy(word, __builtin_assume_aligned(codes, V), V);
    const float scale = Power(e);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        uint32_t bits;
        if constexpr (kSigned) {
            bits = static_cast<uint32_t>(static_cast<int32_t>(word[i / 4] << (24 - i % 4 * 8)) >> 4) & 0x87F00000U;
        } else {
            bits = (word[i / 4] >> (i % 4 * 8) & 0xFFU) << 20;
        }
        v[i] = Decode8<kLeast>(bits) * scale;
    }
}

// bits: those of the random numbers that are used, the 16 low ones or the high ones
template <int kLeast, bool kSigned>
__device__ __forceinline__ void Pack(const float (&v)[8], const uint32_t (&random)[8], uint8_t* codes, uint8_t* exponent)
{
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // v has no sign but NaN's, which the exponent's bits leave out
        const uint32_t bits = kSigned ? __float_as_uint(v[i]) & 0x7FFFFFFFU : __float_as_uint(v[i]);
        most = bits > most ? bits : most;
    }
    const uint32_t e = QuadMax(most) >> 23 & 0xFFU;
    // a block that holds infinity or NaN is NaN
    const float inverse = e >= 254 ? __uint_as_float(e == 254 ? 0x00400000U : 0) : __uint_as_float((254U - e) << 23);
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]) * inverse;
        const uint32_t draw = (kSigned ? random[i] << 4 : random[i] >> 12) & 0xFFFF0U;
        uint32_t code = Encode8<kLeast>(a, draw);
        if constexpr (kSigned) {
            code |= __float_as_uint(v[i]) >> 24 & 0x80U;
        } else {
            // a v of zero under an m that is none would make the step m / eps
            const uint32_t some = __float_as_uint(a) < 1U ? __float_as_uint(a) : 1U;
            code = code > some ? code : some;
        }
        word[i / 4] |= code << (i % 4 * 8);
    }
    if (e == 255) word[0] = word[1] = 0;
    __builtin_memcpy(__builtin_assume_aligned(codes, 8), word, 8);
    if ((threadIdx.x & 3) == 0) *exponent = static_cast<uint8_t>(e);
}

// A workgroup takes 2048 values: with 8-bit moments a thread eight neighbouring
// ones, so a quad a block, otherwise four in each half.  The chunks of all
// tensors are numbered in one row, and each wave finds a chunk's tensor by one
// comparison per lane.
template <typename TP, typename TG, int kBits, bool kMaster, bool kStream>
__global__ __launch_bounds__(kThreads) void AdamWKernel(AdamWTable table, const Factors* __restrict__ factors)
{
#pragma clang fp contract(off)
    constexpr int V = kBits == 8 ? 8 : 4, kUnits = 8 / V;
    const uint32_t first = table.first[threadIdx.x & 63], chunk = blockIdx.x;
    const int which = __popcll(__ballot(first <= chunk)) - 1;
    const AdamWTensor& t = table.tensor[which];
    const int64_t begin = static_cast<int64_t>(chunk - table.first[which]) * kAdamWChunk + threadIdx.x * V;
    const int64_t padded = (t.count + 31) / 32 * 32;
    float g[kUnits][V], p[kUnits][V], m[kUnits][V], v[kUnits][V];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = begin + u * kThreads * V, left = t.count - at;
        if (at >= padded) continue;  // whole quads
        Load(static_cast<const TG*>(t.grad) + at, left, g[u]);
        if constexpr (kMaster) {
            Load(t.master + at, left, p[u]);
        } else {
            Load(static_cast<const TP*>(t.param) + at, left, p[u]);
        }
        if constexpr (kBits == 8) {
            const uint8_t* codes = static_cast<const uint8_t*>(t.moments) + at;
            Unpack<kLeastM, true>(codes, t.exponents[at / 32], m[u]);
            Unpack<kLeastV, false>(codes + padded, t.exponents[(padded + at) / 32], v[u]);
        } else {
            const float* held = static_cast<const float*>(t.moments) + at;
            __builtin_memcpy(m[u], held, sizeof(m[u]));
            __builtin_memcpy(v[u], held + padded, sizeof(v[u]));
        }
    }
    const Factors f = *factors;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = begin + u * kThreads * V, left = t.count - at;
        if (at >= padded) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float grad = g[u][i] * f.scale;
            const float keptM = m[u][i] * f.beta1, newM = grad * f.rest1;
            m[u][i] = keptM + newM;
            const float keptV = v[u][i] * f.beta2, square = grad * grad, newV = square * f.rest2;
            v[u][i] = keptV + newV;
            const float kept = p[u][i] * f.decay, change = Change(f, m[u][i], v[u][i]);
            p[u][i] = kept - change;
        }
        if constexpr (kBits == 8) {
            if (left < V) {  // past the tensor's end the block holds zeros
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (i >= left) m[u][i] = v[u][i] = 0.0f;
                }
            }
            uint32_t random[V];
            const uint32_t seed = Mix(f.key + static_cast<uint32_t>(table.place[which]) +
                                          static_cast<uint32_t>(static_cast<uint64_t>(at) >> 32),
                                      f.mix);
#pragma unroll
            for (int i = 0; i < V; ++i) random[i] = Mix(static_cast<uint32_t>(at) + i + seed, f.mix);
            uint8_t* codes = static_cast<uint8_t*>(t.moments) + at;
            Pack<kLeastM, true>(m[u], random, codes, t.exponents + at / 32);
            Pack<kLeastV, false>(v[u], random, codes + padded, t.exponents + (padded + at) / 32);
        } else {
            float* held = static_cast<float*>(t.moments) + at;
            Store<kStream>(held, left, m[u]);
            Store<kStream>(held + padded, left, v[u]);
        }
        if constexpr (kMaster) Store<kStream>(t.master + at, left, p[u]);
        Store<kStream>(static_cast<TP*>(t.param) + at, left, p[u]);
    }
}

// Four codes per thread, so that neighbouring lanes write neighbouring places.
template <bool kStream>
__global__ __launch_bounds__(kThreads) void AdamWMomentsKernel(AdamWTable table)
{
    const uint32_t first = table.first[threadIdx.x & 63], chunk = blockIdx.x;
    const int which = __popcll(__ballot(first <= chunk)) - 1;
    const AdamWTensor& t = table.tensor[which];
    const int64_t padded = (t.count + 31) / 32 * 32;
    const uint8_t* codes = static_cast<const uint8_t*>(t.moments);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int64_t at = static_cast<int64_t>(chunk - table.first[which]) * kAdamWChunk + part * (kAdamWChunk / 2) +
                           threadIdx.x * 4;
        const int64_t left = t.count - at;
        if (left <= 0) break;
        float m[4], v[4];
        Unpack<kLeastM, true>(codes + at, t.exponents[at / 32], m);
        Unpack<kLeastV, false>(codes + padded + at, t.exponents[(padded + at) / 32], v);
        Store<kStream>(t.master + at, left, m);
        Store<kStream>(t.master + t.count + at, left, v);
    }
}

template <typename TP, typename TG>
void Launch(const AdamWTable& t, const Factors* s, int bits, bool master, hipStream_t stream)
{
    auto launch = [&](auto eight, auto kept) {
        constexpr int kBits = decltype(eight)::value ? 8 : 32;
        constexpr bool kMaster = decltype(kept)::value;
        if (t.chunks > kOrdinaryChunks) AdamWKernel<TP, TG, kBits, kMaster, true><<<t.chunks, kThreads, 0, stream>>>(t, s);
        else AdamWKernel<TP, TG, kBits, kMaster, false><<<t.chunks, kThreads, 0, stream>>>(t, s);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (bits == 8) {
        if (master) launch(yes, yes);
        else launch(yes, no);
    } else {
        if (master) launch(no, yes);
        else launch(no, no);
    }
}

template <typename TP>
void LaunchParam(const AdamWTable& t, const Factors* s, aclDataType grad, int bits, bool master, hipStream_t stream)
{
    if (grad == ACL_FLOAT) Launch<TP, float>(t, s, bits, master, stream);
    else if (grad == ACL_FLOAT16) Launch<TP, Half>(t, s, bits, master, stream);
    else Launch<TP, Bf16>(t, s, bits, master, stream);
}

}  // namespace

int LaunchAdamWFactors(const AdamWScalars& s, void* buffer, void* stream)
{
    AdamWFactorsKernel<<<1, 1, 0, static_cast<hipStream_t>(stream)>>>(s, static_cast<Factors*>(buffer));
    return 0;
}

int LaunchAdamW(const AdamWTable& t, const void* buffer, aclDataType param, aclDataType grad, int bits, bool master,
                void* stream)
{
    hipStream_t q = static_cast<hipStream_t>(stream);
    const auto* s = static_cast<const Factors*>(buffer);
    if (param == ACL_FLOAT) LaunchParam<float>(t, s, grad, bits, master, q);
    else if (param == ACL_FLOAT16) LaunchParam<Half>(t, s, grad, bits, master, q);
    else LaunchParam<Bf16>(t, s, grad, bits, master, q);
    return 0;
}

int LaunchAdamWMoments(const AdamWTable& t, void* stream)
{
    hipStream_t q = static_cast<hipStream_t>(stream);
    if (t.chunks > kOrdinaryChunks) AdamWMomentsKernel<true><<<t.chunks, kThreads, 0, q>>>(t);
    else AdamWMomentsKernel<false><<<t.chunks, kThreads, 0, q>>>(t);
    return 0;
}

}  // namespace aclsp
