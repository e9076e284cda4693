// Device helpers of the experts' kernels: 16-bit types, sums and maxima over
// a 64-lane wave, and the search of a tile's group.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace aclsp {

using Half = _Float16;
using Bf16 = __bf16;

template <typename T>
__device__ __forceinline__ float ToFloat(T v)
{
    return static_cast<float>(v);
}
// Rounds to nearest even (one instruction for bfloat16 on gfx950).
template <typename T>
__device__ __forceinline__ T FromFloat(float v)
{
    return static_cast<T>(v);
}

// Moves within a wave by DPP: lanes that have no source keep `old`.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ uint32_t Dpp(uint32_t old, uint32_t v)
{
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(static_cast<int>(old), static_cast<int>(v), kCtrl, kRowMask, 0xF, false));
}
constexpr int kDppShr1 = 0x111, kDppShr2 = 0x112, kDppShr4 = 0x114, kDppShr8 = 0x118;
constexpr int kDppBcast15 = 0x142, kDppBcast31 = 0x143;

// Inclusive scan over the wave: within rows of 16 lanes, then row 15 -> next, then lane 31 -> upper half.
template <typename F>
__device__ __forceinline__ uint32_t WaveScan(uint32_t x, uint32_t identity, F op)
{
    x = op(x, Dpp<kDppShr1, 0xF>(identity, x));
    x = op(x, Dpp<kDppShr2, 0xF>(identity, x));
    x = op(x, Dpp<kDppShr4, 0xF>(identity, x));
    x = op(x, Dpp<kDppShr8, 0xF>(identity, x));
    x = op(x, Dpp<kDppBcast15, 0xA>(identity, x));
    x = op(x, Dpp<kDppBcast31, 0xC>(identity, x));
    return x;
}

__device__ __forceinline__ uint32_t LastLane(uint32_t x)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63));
}

__device__ __forceinline__ uint32_t WaveMaxU32(uint32_t x)
{
    return LastLane(WaveScan(x, 0U, [](uint32_t a, uint32_t b) { return a > b ? a : b; }));
}

// The same over each row of 16 lanes, in all of its lanes: rotations by 8, 4, 2 and 1.
constexpr int kDppRor8 = 0x128, kDppRor4 = 0x124, kDppRor2 = 0x122, kDppRor1 = 0x121;
template <typename F>
__device__ __forceinline__ uint32_t RowReduce(uint32_t x, F op)
{
    x = op(x, Dpp<kDppRor8, 0xF>(x, x));
    x = op(x, Dpp<kDppRor4, 0xF>(x, x));
    x = op(x, Dpp<kDppRor2, 0xF>(x, x));
    x = op(x, Dpp<kDppRor1, 0xF>(x, x));
    return x;
}

__device__ __forceinline__ uint32_t RowMaxU32(uint32_t x)
{
    return RowReduce(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ float RowSum(float x)
{
    return __uint_as_float(RowReduce(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

__device__ __forceinline__ int32_t WaveInclusiveSum(int32_t x)
{
    return static_cast<int32_t>(WaveScan(static_cast<uint32_t>(x), 0U, [](uint32_t a, uint32_t b) { return a + b; }));
}

__device__ __forceinline__ float WaveSum(float x)
{
    return __uint_as_float(LastLane(WaveScan(__float_as_uint(x), 0U, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    })));
}

__device__ __forceinline__ float WaveMax(float x)
{
    return __uint_as_float(LastLane(WaveScan(__float_as_uint(x), 0xFF800000U, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    })));
}

// Rows [begin, end) of a group, whatever the offsets hold: within [0, rows] and not negative in length.
__device__ __forceinline__ void GroupRows(const int32_t* offsets, int64_t rows, int group, int32_t& begin, int32_t& end)
{
    if (offsets == nullptr) {
        begin = 0;
        end = static_cast<int32_t>(rows);
        return;
    }
    const int32_t r = static_cast<int32_t>(rows);
    const int32_t b = offsets[group], e = offsets[group + 1];
    begin = b < 0 ? 0 : b > r ? r : b;
    end = e < begin ? begin : e > r ? r : e;
}

// Group g's tiles of `height` rows for lane g - g0; the tail's for the lane past the last group's.
__device__ __forceinline__ int32_t LaneTiles(const int32_t* offsets, int64_t rows, int32_t groups, int32_t height,
                                             int32_t g, int32_t& begin, int32_t& end)
{
    begin = end = 0;
    if (g < groups) {
        GroupRows(offsets, rows, g, begin, end);
    } else if (g == groups && offsets != nullptr) {
        int32_t unused;
        GroupRows(offsets, rows, g - 1, unused, begin);
        end = static_cast<int32_t>(rows);
    }
    return (end - begin + height - 1) / height;
}

// All tiles of `height` rows, through the groups and the tail.  Called by whole waves.
__device__ __forceinline__ int32_t CountTiles(const int32_t* offsets, int64_t rows, int64_t groups, int32_t height)
{
    int32_t total = 0, begin, end;
    for (int32_t g0 = 0; g0 <= static_cast<int32_t>(groups); g0 += 64) {
        const int32_t n = LaneTiles(offsets, rows, static_cast<int32_t>(groups), height, g0 + (threadIdx.x & 63),
                                    begin, end);
        total += __builtin_amdgcn_readlane(WaveInclusiveSum(n), 63);
    }
    return total;
}

// A tile of a ragged product: rows [row, end) of `group`; group == groups is
// the tail of rows that belong to no group, group < 0 no tile.
struct RaggedTile {
    int32_t group;
    int32_t row;
    int32_t end;
    int32_t begin;   // the group's first row,
    int32_t before;  // the tiles before it
    int32_t tiles;   // and its own
};

// The tile-th tile of `height` rows, counted through the groups and the tail.
// Called by whole waves with a uniform tile; 64 groups a turn.
__device__ __forceinline__ RaggedTile FindTile(const int32_t* offsets, int64_t rows, int64_t groups, int32_t height,
                                               int32_t tile)
{
    int32_t before = 0;
    for (int32_t g0 = 0; g0 <= static_cast<int32_t>(groups); g0 += 64) {
        int32_t begin, end;
        const int32_t n = LaneTiles(offsets, rows, static_cast<int32_t>(groups), height, g0 + (threadIdx.x & 63),
                                    begin, end);
        const int32_t incl = WaveInclusiveSum(n);
        const uint64_t hit = __ballot(before + incl > tile);
        if (hit != 0) {
            const int src = __builtin_ctzll(hit);
            const int32_t skipped = before + __builtin_amdgcn_readlane(incl - n, src);
            const int32_t first = __builtin_amdgcn_readlane(begin, src);
            return {g0 + src,  first + (tile - skipped) * height, __builtin_amdgcn_readlane(end, src), first, skipped,
                    __builtin_amdgcn_readlane(n, src)};
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return {-1, 0, 0, 0, 0, 0};
}

}  // namespace aclsp
