// Ragged products grouped by expert: C_r = B_g A_index(r) for the rows r of
// each group g, their weight gradient W_g = sum_r gradC_r x X_index(r), and
// the 8-bit products with a scale for each row and column.
//
// Group boundaries stay on the device: the grid covers the most tiles that
// `rows` rows in `groups` groups can have, and every workgroup finds its tile
// by a scan of the offsets.  Sums are in fp32 (int32 for 8 bits, exact) and
// rounded once to the output's type.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "experts_device.h"
#include "experts_internal.h"

namespace aclsp {
namespace {

using Int4 = int __attribute__((ext_vector_type(4)));
using Float4 = float __attribute__((ext_vector_type(4)));
using Half8 = _Float16 __attribute__((ext_vector_type(8)));
using Bf168 = __bf16 __attribute__((ext_vector_type(8)));

// 16x16 matrix instructions on operands of 16 bytes per lane: lane l holds
// row l % 16 of its operand, contraction elements (l / 16) * (16 bytes) on.
// The result's lane l holds column l % 16 (row of the second operand) and
// rows 4 * (l / 16) + i (of the first).
template <typename T>
struct Mma;
template <>
struct Mma<Half> {
    using Acc = Float4;
    static __device__ __forceinline__ Acc Run(Int4 a, Int4 b, Acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Half8, a), __builtin_bit_cast(Half8, b), c, 0,
                                                      0, 0);
    }
};
template <>
struct Mma<Bf16> {
    using Acc = Float4;
    static __device__ __forceinline__ Acc Run(Int4 a, Int4 b, Acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf168, a), __builtin_bit_cast(Bf168, b), c,
                                                       0, 0, 0);
    }
};
template <>
struct Mma<int8_t> {
    using Acc = Int4;
    static __device__ __forceinline__ Acc Run(Int4 a, Int4 b, Acc c)
    {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    }
};

// ---------------------------------------------------------------------------
// Kernels for every size, stride and alignment: tiles of 64x64, loaded element
// by element through registers, zeros beyond the ends.
// ---------------------------------------------------------------------------
constexpr int kAnyTile = 64;
constexpr int kAnyRowBytes = 64;                 // of the contraction per turn
constexpr int kAnyLdsStride = kAnyRowBytes + 16;  // keeps the 16 rows of a read in different banks

template <typename T>
struct AnyTiles {
    static constexpr int kDepth = kAnyRowBytes / static_cast<int>(sizeof(T));
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements per thread and operand
    typename Mma<T>::Acc acc[2][2];

    // Adds the product of two 64-row tiles held in LDS as [row][contraction].
    __device__ __forceinline__ void Multiply(const char* a, const char* b)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        Int4 fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int ra = (wave & 1) * 32 + i * 16 + (lane & 15), rb = (wave >> 1) * 32 + i * 16 + (lane & 15);
            fa[i] = *reinterpret_cast<const Int4*>(a + ra * kAnyLdsStride + (lane >> 4) * 16);
            fb[i] = *reinterpret_cast<const Int4*>(b + rb * kAnyLdsStride + (lane >> 4) * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::Run(fb[j], fa[i], acc[i][j]);
        }
    }
};

// Rows of 64 bytes: thread t holds 16 bytes of row t / 4.
template <typename T>
__device__ __forceinline__ void AnyLoadRows(char* lds, const T* row, bool rowOk, int64_t depth, int64_t at)
{
    constexpr int kPer = AnyTiles<T>::kPer;
    const int chunk = threadIdx.x & 3;
    T v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t c = at + chunk * kPer + i;
        v[i] = rowOk && c < depth ? row[c] : static_cast<T>(0);
    }
    __builtin_memcpy(lds + (threadIdx.x >> 2) * kAnyLdsStride + chunk * 16, v, 16);
}

// The transposed tile: thread t holds 8 columns of contraction row t / 8.
template <typename T>
__device__ __forceinline__ void AnyLoadColumns(char* lds, const T* row, bool rowOk, int64_t width, int64_t at)
{
    const int kk = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const T v = rowOk && at + c0 + i < width ? row[at + c0 + i] : static_cast<T>(0);
        *reinterpret_cast<T*>(lds + (c0 + i) * kAnyLdsStride + kk * sizeof(T)) = v;
    }
}

__device__ __forceinline__ int64_t IndexedRow(const int32_t* index, int64_t r, int64_t count)
{
    if (index == nullptr) return r;
    const int32_t i = index[r];
    return i < 0 || i >= count ? 0 : i;  // stays within the operand whatever the index holds
}

template <typename T, typename TOut, bool kBTrans>
__global__ __launch_bounds__(256) void GroupedAnyKernel(GroupedLaunch p, int32_t tilesN)
{
    __shared__ __align__(16) char lds[2][kAnyTile * kAnyLdsStride];
    const RaggedTile tile = FindTile(p.offsets, p.rows, p.groups, kAnyTile, static_cast<int32_t>(blockIdx.x / tilesN));
    if (tile.group < 0) return;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x % tilesN) * kAnyTile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    AnyTiles<T> t{};
    if (tile.group < p.groups) {
        const T* b = static_cast<const T*>(p.b) + tile.group * p.stride_b;
        const int64_t r = tile.row + (threadIdx.x >> 2), nb = n0 + (threadIdx.x >> 2);
        const bool aOk = r < tile.end, bOk = nb < p.n;
        const T* aRow = static_cast<const T*>(p.a) + (aOk ? IndexedRow(p.row_index, r, p.rows_a) : 0) * p.lda;
        for (int64_t k0 = 0; k0 < p.k; k0 += AnyTiles<T>::kDepth) {
            AnyLoadRows<T>(lds[0], aRow, aOk, p.k, k0);
            if constexpr (kBTrans) {
                AnyLoadRows<T>(lds[1], b + nb * p.ldb, bOk, p.k, k0);
            } else {
                const int64_t kk = k0 + (threadIdx.x >> 3);
                AnyLoadColumns<T>(lds[1], b + kk * p.ldb, kk < p.k, p.n, n0);
            }
            __syncthreads();
            t.Multiply(lds[0], lds[1]);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t r = tile.row + (wave & 1) * 32 + i * 16 + (lane & 15);
        if (r >= tile.end) continue;
        float sa = 1.0f;
        if constexpr (sizeof(T) == 1) {
            if (tile.group < p.groups) sa = p.scale_a[IndexedRow(p.row_index, r, p.rows_a)];
        }
        TOut* c = static_cast<TOut*>(p.c) + r * p.ldc;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t n = n0 + (wave >> 1) * 32 + j * 16 + (lane >> 4) * 4 + x;
                if (n >= p.n) continue;
                float v = static_cast<float>(t.acc[i][j][x]);
                if constexpr (sizeof(T) == 1) {
                    if (tile.group < p.groups) v = v * (sa * p.scale_b[tile.group * p.n + n]);
                }
                c[n] = FromFloat<TOut>(v);
            }
        }
    }
}

template <typename T, typename TOut>
__global__ __launch_bounds__(256) void GroupedGradAnyKernel(GroupedGradLaunch p, int32_t tilesN, int32_t tilesK)
{
    __shared__ __align__(16) char lds[2][kAnyTile * kAnyLdsStride];
    uint32_t id = blockIdx.x;
    const int64_t k0 = static_cast<int64_t>(id % tilesK) * kAnyTile;
    id /= tilesK;
    const int64_t n0 = static_cast<int64_t>(id % tilesN) * kAnyTile;
    const int64_t g = id / tilesN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t begin, end;
    GroupRows(p.offsets, p.rows, static_cast<int>(g), begin, end);
    AnyTiles<T> t{};
    for (int64_t r0 = begin; r0 < end; r0 += AnyTiles<T>::kDepth) {
        const int64_t r = r0 + (threadIdx.x >> 3);
        const bool ok = r < end;
        AnyLoadColumns<T>(lds[0], static_cast<const T*>(p.grad) + r * p.ldg, ok, p.n, n0);
        AnyLoadColumns<T>(lds[1], static_cast<const T*>(p.x) + (ok ? IndexedRow(p.row_index, r, p.rows_x) : 0) * p.ldx,
                          ok, p.k, k0);
        __syncthreads();
        t.Multiply(lds[0], lds[1]);
        __syncthreads();
    }
    TOut* w = static_cast<TOut*>(p.w) + g * p.stride_w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t n = n0 + (wave & 1) * 32 + i * 16 + (lane & 15);
        if (n >= p.n) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t k = k0 + (wave >> 1) * 32 + j * 16 + (lane >> 4) * 4 + x;
                if (k < p.k) w[n * p.ldw + k] = FromFloat<TOut>(t.acc[i][j][x]);
            }
        }
    }
}

int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The most tiles of `height` rows: every group, and the tail, may end inside one.
int64_t MaxRowTiles(const int32_t* offsets, int64_t rows, int64_t groups, int64_t height)
{
    if (offsets == nullptr) return CeilDiv(rows, height);
    const int64_t most = rows / height + groups + 1;
    return most < rows ? most : rows;
}

template <typename T, typename TOut>
int GroupedTyped(const GroupedLaunch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, kAnyTile);
    const int64_t grid = MaxRowTiles(l.offsets, l.rows, l.groups, kAnyTile) * tilesN;
    if (grid > INT32_MAX) return kTooLarge;
    if constexpr (sizeof(T) == 2) {
        if (!l.b_trans) {
            GroupedAnyKernel<T, TOut, false><<<static_cast<uint32_t>(grid), 256, 0, s>>>(l, static_cast<int32_t>(tilesN));
            return 0;
        }
    }
    GroupedAnyKernel<T, TOut, true><<<static_cast<uint32_t>(grid), 256, 0, s>>>(l, static_cast<int32_t>(tilesN));
    return 0;
}

template <typename T, typename TOut>
int GroupedGradTyped(const GroupedGradLaunch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, kAnyTile), tilesK = CeilDiv(l.k, kAnyTile);
    if (tilesN * tilesK > INT32_MAX / l.groups) return kTooLarge;
    GroupedGradAnyKernel<T, TOut><<<static_cast<uint32_t>(tilesN * tilesK * l.groups), 256, 0, s>>>(
        l, static_cast<int32_t>(tilesN), static_cast<int32_t>(tilesK));
    return 0;
}

}  // namespace

int LaunchGroupedMM(const GroupedLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (l.ab_type) {
        case ACL_INT8:
            if (l.c_type == ACL_FLOAT) return GroupedTyped<int8_t, float>(l, s);
            if (l.c_type == ACL_FLOAT16) return GroupedTyped<int8_t, Half>(l, s);
            return GroupedTyped<int8_t, Bf16>(l, s);
        case ACL_FLOAT16:
            return l.c_type == ACL_FLOAT ? GroupedTyped<Half, float>(l, s) : GroupedTyped<Half, Half>(l, s);
        default:
            return l.c_type == ACL_FLOAT ? GroupedTyped<Bf16, float>(l, s) : GroupedTyped<Bf16, Bf16>(l, s);
    }
}

int LaunchGroupedMMGrad(const GroupedGradLaunch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.type == ACL_FLOAT16) {
        return l.w_type == ACL_FLOAT ? GroupedGradTyped<Half, float>(l, s) : GroupedGradTyped<Half, Half>(l, s);
    }
    return l.w_type == ACL_FLOAT ? GroupedGradTyped<Bf16, float>(l, s) : GroupedGradTyped<Bf16, Bf16>(l, s);
}

}  // namespace aclsp
