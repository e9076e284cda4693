// Parts of the grouped products' tiles: operands copied to LDS, sums of teams
// of waves, tiles stored by whole rows, and the order of the tiles.  For the
// files that hold the products' kernels; everything is local to each.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "experts_device.h"

namespace aclsp {
namespace {

using Int4 = int __attribute__((ext_vector_type(4)));
using Float4 = float __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int64_t IndexedRow(const int32_t* index, int64_t r, int64_t count)
{
    if (index == nullptr) return r;
    const int32_t i = index[r];
    return i < 0 || i >= count ? 0 : i;  // stays within the operand whatever the index holds
}

// ---------------------------------------------------------------------------
// Tiles through LDS.  A tile's contraction advances by 128 bytes per turn.
// While one turn's operands are multiplied the next ones' are copied to LDS,
// straight from memory where every row is aligned to 16 bytes, through
// registers by loads of any alignment where not.  Each wave keeps the operands
// of one matrix step ahead of the one it multiplies in registers.
// ---------------------------------------------------------------------------
constexpr int kTurnBytes = 128;
constexpr int kSteps = 2;  // matrix instructions take 64 bytes of each row

// What lanes copy that have nothing to copy: both operands read as zero past
// the contraction's end, so that no value beyond it, NaN among them, counts.
// (LoadPart may read up to 15 bytes before what it is given, which are zeros here too.)
__device__ const Int4 kZeroBytes[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
__device__ __forceinline__ const char* Zeros() { return reinterpret_cast<const char*>(&kZeroBytes[1]); }

// Copies 16 bytes per lane to 1024 bytes of LDS.  Written as assembly, without
// an output: the compiler would count the copy against every later LDS read
// that it cannot tell from the copy's target, and wait for it right there.
// Wait waits for the copies.  m0 is the copy's target and is set for each.  It
// is a reserved register, whose clobber the compiler does not heed, so a test
// looks that it has no other use in these kernels' code.  (Put back after each
// copy, the large products took 1% longer.)
__device__ __forceinline__ void CopyToLds(const char* from, char* to)
{
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(to)));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from));
}

// 16 bytes at any alignment.  The pointer is said to be global memory's: the
// compiler cannot tell where one that may be Zeros() points, and loads that
// might be LDS's make every read of LDS wait for them.
__device__ __forceinline__ Int4 LoadBytes(const char* from)
{
    using Bytes = int __attribute__((ext_vector_type(4), aligned(1)));
    return *(const __attribute__((address_space(1))) Bytes*)(from);
}

// The first `valid` bytes of a row's 16-byte chunk at `from`, zeros after them.  A chunk that the row's end cuts is
// read by the 16 bytes that end there and shifted, which a row of 16 bytes or more holds; `tiny`: it does not, and
// elements are read one at a time.  (With every cut chunk read so, a load and its wait after the other, 5418 rows
// in 6 groups x 1144 x 661 took 38 us, now 33; their weight gradient 92, now 59.)
template <typename T>
__device__ __forceinline__ Int4 LoadPart(const char* from, int valid, bool tiny)
{
    if (tiny) {
        constexpr int kCount = 16 / static_cast<int>(sizeof(T));
        const auto* elements = (const __attribute__((address_space(1))) T*)(from);
        T e[kCount];
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            e[i] = static_cast<T>(0);
            if (i * static_cast<int>(sizeof(T)) < valid) e[i] = elements[i];
        }
        Int4 v;
        __builtin_memcpy(&v, e, 16);
        return v;
    }
    const int cut = valid >= 16 || valid <= 0 ? 0 : 16 - valid;
    const Int4 v = LoadBytes(from - cut);
    uint64_t half[2];
    __builtin_memcpy(half, &v, 16);
    const int bits = cut * 8;
    const uint64_t down = bits >= 64 ? half[1] >> (bits & 63) : half[0] >> bits | half[1] << 1 << (63 - bits);
    half[1] = bits >= 64 ? 0 : half[1] >> bits;
    half[0] = down;
    Int4 out;
    __builtin_memcpy(&out, half, 16);
    return valid <= 0 ? Int4{0, 0, 0, 0} : out;
}

// All of a thread's chunks of a turn; whole ones without a branch between them.
template <typename T, int N>
__device__ __forceinline__ void LoadAll(const char* const (&ptr)[N], int valid, bool tiny, Int4 (&held)[N])
{
    if (__all(valid >= 16)) {
#pragma unroll
        for (int i = 0; i < N; ++i) held[i] = LoadBytes(ptr[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) held[i] = LoadPart<T>(ptr[i], valid, tiny);
    }
}

__device__ __forceinline__ int WaveNumber() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// This thread's and wave's number among the kThreads that work on one tile (a
// workgroup may hold several such teams).
template <int kThreads>
__device__ __forceinline__ int TeamThread()
{
    static_assert((kThreads & (kThreads - 1)) == 0, "");
    return static_cast<int>(threadIdx.x) & (kThreads - 1);
}
template <int kThreads>
__device__ __forceinline__ int TeamWave()
{
    return WaveNumber() & (kThreads / 64 - 1);
}

// An operand whose rows run along the contraction: R rows of 128 bytes per
// turn.  Its 16-byte chunk c of row r lies at slot c ^ (r / 2 & 7), so that the
// lanes that read one chunk of 16 rows touch each of the 64 banks once.
template <typename T, int R, int kThreads, bool kAligned>
struct RowOperand {
    static constexpr int kLoads = R * 8 / kThreads;
    static constexpr int kRowsPerLoad = kThreads / 8;
    static constexpr int kBytes = R * kTurnBytes;
    static constexpr bool kDirect = kAligned;
    const char* ptr[kLoads];
    Int4 held[kLoads];
    int valid = 16;     // bytes of this thread's chunks before the contraction's end
    bool tiny = false;  // whole rows have fewer than 16 bytes

    // This thread's rows are Row(i); its chunk of each is the same.
    static __device__ __forceinline__ int Row(int i) { return i * kRowsPerLoad + (TeamThread<kThreads>() >> 3); }
    static __device__ __forceinline__ int Chunk()
    {
        return (TeamThread<kThreads>() & 7) ^ ((TeamThread<kThreads>() >> 4) & 7);
    }

    __device__ __forceinline__ void Skip(int64_t turns)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) ptr[i] += turns * kTurnBytes;
    }
    // Before a turn's copies: `bytes` of the contraction are left (none, or less, for a turn of zeros).
    __device__ __forceinline__ void Prepare(int64_t bytes)
    {
        if (bytes >= kTurnBytes) return;
        const int here = static_cast<int>(bytes) - Chunk() * 16;
        if constexpr (!kAligned) valid = here < 0 ? 0 : here < 16 ? here : 16;
        if (here > 0) return;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) ptr[i] = Zeros();
    }
    __device__ __forceinline__ void Issue(char* lds, int i)
    {
        CopyToLds(ptr[i], lds + TeamWave<kThreads>() * 1024 + i * kThreads * 16);
        ptr[i] += kTurnBytes;
    }
    // The same through registers, for rows of any alignment.
    __device__ __forceinline__ void Load()
    {
        LoadAll<T>(ptr, valid, tiny, held);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) ptr[i] += kTurnBytes;
    }
    __device__ __forceinline__ void LookUp() {}
    __device__ __forceinline__ void Commit(char* lds)
    {
        if constexpr (!kAligned) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                *reinterpret_cast<Int4*>(lds + (i * kThreads + TeamThread<kThreads>()) * 16) = held[i];
            }
        }
    }

    // The operand of one matrix instruction: 16 rows from `row` on.
    static __device__ __forceinline__ Int4 Read(const char* lds, int row, int step)
    {
        const int lane = threadIdx.x & 63;
        const int chunk = (step * 4 + (lane >> 4)) ^ ((lane >> 1) & 7);
        return *reinterpret_cast<const Int4*>(lds + (row + (lane & 15)) * kTurnBytes + chunk * 16);
    }
};

// Waits for this wave's reads and its copies but the last kLeft of them, then for the other waves'.
template <int kLeft>
__device__ __forceinline__ void Wait()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Adds up what a workgroup's kTeams teams hold of one tile, in their order, in
// the first one; returns whether this team is that one.  `lds` holds the other
// teams' operands, which no wave uses any more; the first one's place is left
// to its store, which may begin before another of its waves has added up.
template <int kTeams, int kThreads, int kBytes, int MI, int NI, typename Acc>
__device__ __forceinline__ bool JoinTeams(char* lds, Acc (&acc)[MI][NI])
{
    if constexpr (kTeams == 1) return true;
    constexpr int kTeamBytes = kThreads * MI * NI * static_cast<int>(sizeof(Acc));
    static_assert(kTeams == 1 || (kTeams - 1) * kTeamBytes <= kBytes, "the sums must fit");
    const int team = WaveNumber() / (kThreads / 64);
    Acc* mine = reinterpret_cast<Acc*>(lds) + TeamThread<kThreads>();
    if (team > 0) {
#pragma unroll
        for (int i = 0; i < MI * NI; ++i) {
            mine[(team - 1) * (kTeamBytes / sizeof(Acc)) + i * kThreads] = acc[i / NI][i % NI];
        }
    }
    Wait<0>();
    if (team > 0) return false;
#pragma unroll
    for (int t = 0; t < kTeams - 1; ++t) {
#pragma unroll
        for (int i = 0; i < MI * NI; ++i) acc[i / NI][i % NI] += mine[t * (kTeamBytes / sizeof(Acc)) + i * kThreads];
    }
    return true;
}

// Writes a wave's MI*16 x NI*16 tile of the output, rows [0, rows) and columns
// [0, columns) of it, at c.  A result's lanes hold neighbouring rows: stored
// from there, each store would touch 16 rows by 32 bytes (a 256x256 tile then
// took 68 us).  The wave passes its tile through its own part of LDS instead
// and stores whole rows, 16 bytes per lane.  value(i, j, v) gives the four
// values of tile (i, j).  Chunk c of row r lies at slot c ^ r (c ^ r / 2 in
// rows of half the banks), which spreads the rows of a write over the banks.
// kStream: see StoreStreaming.
template <typename TOut, int MI, int NI, int kLdsBytes, bool kStream = false, typename Value>
__device__ __forceinline__ void StoreTile(char* lds, TOut* c, int64_t ldc, int64_t rows, int64_t columns, Value value)
{
    constexpr int kSize = static_cast<int>(sizeof(TOut));
    constexpr int kRowBytes = NI * 16 * kSize, kChunks = kRowBytes / 16, kPer = 16 / kSize;
    constexpr int kFit = kLdsBytes / (16 * kRowBytes), kTiles = kFit < MI ? kFit : MI;  // at a time
    constexpr int kRowsPerStore = 64 / kChunks;
    static_assert(kTiles > 0 && kChunks >= 8 && kChunks <= 64, "a row of tiles must fit the wave's LDS");
    const int lane = threadIdx.x & 63;
    auto slot = [](int r) { return kChunks == 8 ? (r >> 1) & 7 : r & (kChunks - 1); };
#pragma unroll
    for (int first = 0; first < MI; first += kTiles) {
        const int tiles = MI - first < kTiles ? MI - first : kTiles;
#pragma unroll
        for (int i = first; i < first + tiles; ++i) {
            const int r = (i - first) * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                float v[4];
                value(i, j, v);
                TOut o[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) o[x] = FromFloat<TOut>(v[x]);
                const int byte = (j * 16 + (lane >> 4) * 4) * kSize;
                char* to = lds + r * kRowBytes + (((byte >> 4) ^ slot(r)) << 4) + (byte & 8);
                __builtin_memcpy(__builtin_assume_aligned(to, sizeof(o)), o, sizeof(o));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
        for (int r = lane / kChunks; r < tiles * 16; r += kRowsPerStore) {
            const int chunk = (lane % kChunks) ^ slot(r);
            const int64_t row = first * 16 + r, left = columns - chunk * kPer;
            if (row >= rows || left <= 0) continue;
            const Int4 v = *reinterpret_cast<const Int4*>(lds + r * kRowBytes + (lane % kChunks) * 16);
            TOut* to = c + row * ldc + chunk * kPer;
            if (left >= kPer) {
                if constexpr (kStream) StoreStreaming<16>(to, &v);
                else __builtin_memcpy(to, &v, 16);  // whatever C's alignment
            } else {
                TOut o[kPer];
                __builtin_memcpy(o, &v, 16);
#pragma unroll
                for (int x = 0; x < kPer; ++x) {
                    if (x < left) to[x] = o[x];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// The id-th of m x n tiles in an order that keeps any 32 neighbours, about
// what one die works on at a time, near a square: bands of `width` columns
// of tiles, each walked row by row, so that they share the fewest operands
// (with rows of 32 tiles, 8192^3 in 16 bits took 1.30 ms).
struct TilePlace {
    int32_t m, n;
};
__device__ __forceinline__ TilePlace PlaceInBands(int64_t id, int32_t m, int32_t n)
{
    int32_t width = 32 / m;
    width = width < 4 ? 4 : width;
    const int32_t band = static_cast<int32_t>(id / (static_cast<int64_t>(width) * m));
    const int32_t first = band * width;
    const int32_t rest = static_cast<int32_t>(id - static_cast<int64_t>(first) * m);
    const int32_t w = n - first < width ? n - first : width;
    return {rest / w, first + rest % w};
}

// What a workgroup of GroupedTileKernel does: a tile of the list of 256x256
// tiles, or one of `parts` slices of its rows; tile < 0: nothing.
//
// Workgroups are dealt to the 8 dies in turn, so those of one remainder take
// one run of the list: neighbours then share an L2.  A die works on a tile per
// CU at a time; when the last round of its run would fill half or a quarter
// of the CUs, its tiles are cut into two or four slices.
struct TileShare {
    int64_t tile;
    int32_t part, parts;
};
__device__ __forceinline__ TileShare ShareOfWorkgroup(int64_t total, int32_t cus)
{
    const int32_t die = static_cast<int32_t>(blockIdx.x % 8);
    const int64_t per = (total + 7) / 8, at = blockIdx.x / 8;
    const int64_t first = die * per;
    const int64_t mine = total - first < per ? total - first : per;
    if (mine <= 0) return {-1, 0, 1};
    const int64_t whole = mine / cus * cus, rest = mine - whole;
    const int32_t parts = rest * 4 <= cus ? 4 : rest * 2 <= cus ? 2 : 1;
    if (at < whole) return {first + at, 0, 1};
    const int64_t tile = whole + (at - whole) / parts;
    return {tile < mine ? first + tile : -1, static_cast<int32_t>((at - whole) % parts), parts};
}

int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool Aligned16(const void* p, int64_t strideBytes) { return (reinterpret_cast<uintptr_t>(p) | strideBytes) % 16 == 0; }

// The most tiles of `height` rows: every group, and the rows on either side, may end inside one.
int64_t MaxRowTiles(const int32_t* offsets, int64_t rows, int64_t groups, int64_t height)
{
    if (offsets == nullptr) return CeilDiv(rows, height);
    const int64_t most = rows / height + groups + 2;
    return most < rows ? most : rows;
}

int CusPerDie()
{
    static const int cus = [] {
        int dev = 0, n = 0;
        const bool ok = hipGetDevice(&dev) == hipSuccess &&
                        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n >= 8;
        return ok ? n / 8 : 32;
    }();
    return cus;
}

}  // namespace
}  // namespace aclsp
