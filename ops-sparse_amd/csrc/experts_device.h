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

// Workgroups of 256 threads in two dimensions where one would not take them
// (fewer than 2^32 threads), and the number of each; those past the last do nothing.
inline dim3 GridOf(int64_t blocks)
{
    constexpr int64_t kRow = int64_t{1} << 23;
    return blocks <= kRow ? dim3(static_cast<uint32_t>(blocks))
                          : dim3(static_cast<uint32_t>(kRow), static_cast<uint32_t>((blocks + kRow - 1) / kRow));
}
__device__ __forceinline__ uint32_t BlockNumber() { return blockIdx.y * gridDim.x + blockIdx.x; }

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

// A tile of a ragged product: rows [row, end) of `group`; group == groups are
// the rows that belong to no group, group < 0 no tile.
struct RaggedTile {
    int32_t group;
    int32_t row;
    int32_t end;
    int32_t begin;   // the group's first row,
    int32_t before;  // the tiles before it
    int32_t tiles;   // and its own
};

// The tiles of `height` rows of all groups, of the rows past the last and of
// those before the first (offsets that are some of a longer list's), for whole
// waves: 64 groups at a time, one per lane.  The first 64 are read once for
// both the count and the search, which every workgroup waits for.
struct RaggedTiles {
    const int32_t* offsets;
    int32_t rows, groups, height;
    int32_t begin, end, tiles, upTo;  // this lane's group of the first 64; upTo: tiles through it
    int32_t head, tail;               // rows before the first group, and the first one past the last
    int32_t total;

    __device__ __forceinline__ int32_t Count(int32_t from, int32_t to) const
    {
        return (to - from + height - 1) / height;
    }

    __device__ __forceinline__ void Lane(int32_t g, int32_t& from, int32_t& to) const
    {
        from = to = 0;
        if (g < groups) GroupRows(offsets, rows, g, from, to);
    }

    __device__ __forceinline__ RaggedTiles(const int32_t* o, int64_t r, int64_t g, int32_t h)
        : offsets(o), rows(static_cast<int32_t>(r)), groups(static_cast<int32_t>(g)), height(h)
    {
        const int lane = threadIdx.x & 63;
        Lane(lane, begin, end);
        tiles = Count(begin, end);
        upTo = WaveInclusiveSum(tiles);
        total = __builtin_amdgcn_readlane(upTo, 63);
        int32_t last = end, lastLane = (groups < 64 ? groups : 64) - 1;
        for (int32_t g0 = 64; g0 < groups; g0 += 64) {
            int32_t from;
            Lane(g0 + lane, from, last);
            total += __builtin_amdgcn_readlane(WaveInclusiveSum(Count(from, last)), 63);
            lastLane = (groups - g0 < 64 ? groups - g0 : 64) - 1;
        }
        tail = offsets != nullptr ? __builtin_amdgcn_readlane(last, lastLane) : rows;
        head = offsets != nullptr ? __builtin_amdgcn_readlane(begin, 0) : 0;
        total += Count(tail, rows) + Count(0, head);
        if (total < 0) total = 0;  // the sum of offsets without meaning
    }

    // The tile-th tile; `tile` is uniform.
    __device__ __forceinline__ RaggedTile Find(int32_t tile) const
    {
        int32_t before = 0, from = begin, to = end, n = tiles, through = upTo;
        for (int32_t g0 = 0; g0 < groups; g0 += 64) {
            if (g0 > 0) {
                Lane(g0 + static_cast<int32_t>(threadIdx.x & 63), from, to);
                n = Count(from, to);
                through = WaveInclusiveSum(n);
            }
            const uint64_t hit = __ballot(before + through > tile);
            if (hit != 0) {
                const int src = __builtin_ctzll(hit);
                const int32_t skipped = before + __builtin_amdgcn_readlane(through - n, src);
                const int32_t first = __builtin_amdgcn_readlane(from, src);
                return {g0 + src, first + (tile - skipped) * height, __builtin_amdgcn_readlane(to, src), first, skipped,
                        __builtin_amdgcn_readlane(n, src)};
            }
            before += __builtin_amdgcn_readlane(through, 63);
        }
        const int32_t past = Count(tail, rows), ahead = Count(0, head);
        if (tile - before < past) return {groups, tail + (tile - before) * height, rows, tail, before, past};
        before += past;
        if (tile - before >= ahead) return {-1, 0, 0, 0, 0, 0};
        return {groups, (tile - before) * height, head, 0, before, ahead};
    }
};

// The `nth`-longest group (equal ones by number), by whole waves: work handed
// out in this order leaves no long group for the end.  Beyond 64 groups, where
// one weighs less, their own order.
__device__ __forceinline__ int32_t LongestGroup(const int32_t* offsets, int64_t rows, int32_t groups, int32_t nth)
{
    if (groups > 64 || offsets == nullptr) return nth;
    const int lane = threadIdx.x & 63;
    int32_t begin = 0, end = -1;
    if (lane < groups) GroupRows(offsets, rows, lane, begin, end);
    const int32_t length = end - begin;
    int32_t rank = 0;
    for (int i = 0; i < groups; ++i) {
        const int32_t other = __builtin_amdgcn_readlane(length, i);
        rank += other > length || (other == length && i < lane) ? 1 : 0;
    }
    return __builtin_ctzll(__ballot(lane < groups && rank == nth));
}

}  // namespace aclsp
