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
#include <type_traits>

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
// rows 4 * (l / 16) + i (of the first).  The 32x32 ones have the same rate, but
// draw more power on random operands: alone they sustain 1.82 PFLOP/s of
// bfloat16 where these do 2.05.
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
using Short4 = short __attribute__((ext_vector_type(4)));

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

// An operand of 16-bit elements whose rows run across the contraction: 64
// rows of C columns per turn, read through the transposing LDS load: of the
// 16 lanes that work together lane j supplies 4 columns (j % 4) of row j / 4,
// and lane i receives the 4 rows of column i.  32 lanes read 32 bytes each of
// rows r to r + 3 and r + 8 to r + 11: chunk c of row r lies at slot
// c ^ 2 h, h the row's number among those eight, so that they touch every bank
// once.  (Rows of 128 bytes lie in one half of the banks or the other by
// themselves: h counts the four of a half.)
template <typename T, int C, int kThreads, bool kIndexed, bool kAligned>
struct ColumnOperand {
    static constexpr int kChunks = C / 8;
    static constexpr int kRowsPerLoad = kThreads / kChunks;
    static constexpr int kLoads = 64 / kRowsPerLoad;
    static constexpr int kBytes = 64 * C * 2;
    static constexpr bool kDirect = kAligned;
    const char* ptr[kLoads];
    const char* base;  // this thread's chunk of row 0
    int64_t ld;        // bytes
    const int32_t* index;
    int64_t count;     // rows that an index may name
    int32_t row, end;  // of this thread's first load in the next turn, and of all
    static constexpr int kWaveRows = 64 / kChunks;  // rows of a wave's load
    int32_t next[kIndexed ? kLoads : 1][kWaveRows];
    Int4 held[kLoads];
    int valid;         // bytes of the chunk before the last column
    bool tiny;         // whole rows have fewer than 16 bytes

    static_assert(kLoads == 1 || kRowsPerLoad % 16 == 0, "a thread's chunk must not change with its rows");
    static __device__ __forceinline__ int Swizzle(int r)
    {
        return kChunks == 8 ? (r & 2) | ((r & 8) >> 1) : ((r & 3) << 1) | (r & 8);
    }
    static __device__ __forceinline__ int Row(int i) { return i * kRowsPerLoad + TeamThread<kThreads>() / kChunks; }
    static __device__ __forceinline__ int Chunk()
    {
        return (TeamThread<kThreads>() % kChunks) ^ Swizzle(TeamThread<kThreads>() / kChunks);
    }

    __device__ __forceinline__ void Init(const void* p, int64_t ldBytes, int64_t column, int64_t columns,
                                         const int32_t* rowIndex, int64_t rowCount, int32_t first, int32_t last)
    {
        const int64_t c = column + Chunk() * 8;
        const bool in = c < columns;
        valid = columns - c >= 8 ? 16 : static_cast<int>(columns - c) * 2;
        tiny = columns < 8;
        base = static_cast<const char*>(p) + c * 2;
        ld = ldBytes;
        index = rowIndex;
        count = rowCount;
        row = first + Row(0);
        end = last;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) ptr[i] = base + (row + i * kRowsPerLoad) * ld;
        LookUp();
        if (!in) {
            valid = 16;
            ld = 0;
            base = Zeros();
#pragma unroll
            for (int i = 0; i < kLoads; ++i) ptr[i] = base;
        }
    }

    // The next turn's rows; those past the end, which only the last turn has, read as zero.
    __device__ __forceinline__ void Prepare(int64_t bytes)
    {
        if constexpr (kIndexed) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                // by steps from one index to the next: a choice between them the compiler made one between addresses,
                // of an array in scratch memory
                uint32_t sum = static_cast<uint32_t>(next[i][0]);
#pragma unroll
                for (int j = 1; j < kWaveRows; ++j) {
                    const uint32_t step = static_cast<uint32_t>(next[i][j]) - static_cast<uint32_t>(next[i][j - 1]);
                    sum += (threadIdx.x & 63) / kChunks >= j ? step : 0;
                }
                const int32_t at = static_cast<int32_t>(sum);
                ptr[i] = base + (at < 0 || at >= count ? 0 : at) * ld;
            }
        }
        if (bytes < kTurnBytes) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                if (row + i * kRowsPerLoad >= end) ptr[i] = Zeros();
            }
        }
        row += 64;
    }
    __device__ __forceinline__ void Issue(char* lds, int i)
    {
        CopyToLds(ptr[i], lds + TeamWave<kThreads>() * 1024 + i * kThreads * 16);
        if constexpr (!kIndexed) ptr[i] += 64 * ld;
    }
    __device__ __forceinline__ void Load()
    {
        LoadAll<T>(ptr, valid, tiny, held);
        if constexpr (!kIndexed) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) ptr[i] += 64 * ld;
        }
    }
    __device__ __forceinline__ void Commit(char* lds)
    {
        if constexpr (!kAligned) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                *reinterpret_cast<Int4*>(lds + (i * kThreads + TeamThread<kThreads>()) * 16) = held[i];
            }
        }
    }
    // The next turn's indices, for Prepare after a wait for reads: each wave's rows are its own, so they come by
    // scalar loads, which that wait covers.  (As vector loads they were waited for behind all copies in flight:
    // the training case's gradient took 620 us where rows in order take 527.)
    __device__ __forceinline__ void LookUp()
    {
        if constexpr (kIndexed) {
            const auto* list = (const __attribute__((address_space(4))) int32_t*)(index);
            const int32_t first = __builtin_amdgcn_readfirstlane(row);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
#pragma unroll
                for (int j = 0; j < kWaveRows; ++j) {
                    const int32_t r = first + i * kRowsPerLoad + j;
                    next[i][j] = list[r < end ? r : end - 1];
                }
            }
        }
    }

    static __device__ __forceinline__ Int4 Read(const char* lds, int column, int step)
    {
        using LdsShort4 = __attribute__((address_space(3))) Short4;
        const int lane = threadIdx.x & 63, j = lane & 15;
        const int r = step * 32 + (lane >> 4) * 8 + (j >> 2);
        const int c = column + (j & 3) * 4;
        const char* p = lds + r * (C * 2) + ((((c >> 3) ^ Swizzle(r)) << 4) | ((c & 4) << 1));
        struct Pair {
            Short4 lo, hi;
        } v;
        v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)(p));
        v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4*)(p + 4 * (C * 2)));
        return __builtin_bit_cast(Int4, v);
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

// acc += the product over `bytes` of the contraction (of 16-bit elements when
// an operand's rows run across it) in `turns` turns, those past the bytes of
// zeros; MI x NI tiles of 16x16 per wave from rows
// (columns of the output) rowA and rowB on.
//
// A turn is two matrix steps of MI rows of products each.  After a row's
// products come the reads from LDS of the first operand D rows on, into the
// registers that the row has left, and of the second operand's next step.  One
// barrier per turn, before its last D rows, whose reads are the next turn's: by
// then every wave has read this turn's operands and the next turn's have
// arrived.  B has two places in LDS, A kPlacesA: the last D rows copy B of the
// turn after the next to where this turn's was; the rows before copy A of the
// turn kPlacesA - 1 ahead.  With three places the barrier need not wait for
// the A copied last, and the memory has two turns for it: the copies alone
// take most of a turn.
template <typename T, int MI, int NI, int kPlacesA, typename OperandA, typename OperandB>
__device__ __forceinline__ void MultiplyTile(OperandA& a, OperandB& b, char* lds, int64_t bytes, int64_t turns,
                                             int rowA, int rowB, typename Mma<T>::Acc (&acc)[MI][NI])
{
    constexpr bool kDirect = OperandA::kDirect;
    constexpr int kCopiesA = OperandA::kLoads, kCopiesB = OperandB::kLoads;
    constexpr int kAhead = kPlacesA - 1;
    constexpr int kLeft = kAhead == 2 ? kCopiesA : 0;  // copies that a barrier need not wait for
    constexpr int D = MI >= 4 ? MI / 2 : 2, kRows = kSteps * MI, kBefore = kRows - D;
    static_assert(kAhead == 1 || (kAhead == 2 && kDirect), "copies through registers are kept for one turn");
    char* const placesB = lds + kPlacesA * OperandA::kBytes;
    Int4 fa[D], fb[kSteps][NI];
    auto readA = [&](const char* from, int q) { fa[q % D] = OperandA::Read(from, rowA + q % MI * 16, q / MI); };
    auto readB = [&](const char* from, int s, int first, int last) {
#pragma unroll
        for (int j = first; j < last; ++j) fb[s][j] = OperandB::Read(from, rowB + j * 16, s);
    };
    // Rows [first, last) of a turn, in this order to the instruction; nextA: null, or where the next turn's operands
    // are.  `copies` calls of copy are spread over the rows, since a wave that issues copies faster than the memory
    // pipeline takes them (64 bytes per clock) waits with its products behind them.
    auto rows = [&](int first, int last, const char* fromA, const char* fromB, const char* nextA, const char* nextB,
                    int copies, auto copy) {
#pragma unroll
        for (int q = first; q < last; ++q) {
            const int s = q / MI, i = q % MI;
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = Mma<T>::Run(fb[s][j], fa[q % D], acc[i][j]);
            if (q < kBefore) {
                readA(fromA, q + D);
            } else if (nextA != nullptr) {
                readA(nextA, q - kBefore);
                readB(nextB, 0, (q - kBefore) * NI / D, (q - kBefore + 1) * NI / D);
            }
            if (q < MI / 2) readB(fromB, 1, q * NI / (MI / 2), (q + 1) * NI / (MI / 2));
            const int n = last - first;
#pragma unroll
            for (int c = (q - first) * copies / n; c < (q - first + 1) * copies / n; ++c) copy(c);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int64_t leftA = bytes, leftB = bytes;
    int toA = 0, toB = 0;  // places of the next copies, in bytes
    // straight to LDS one at a time, or through registers all at once (written by commit)
    auto copyA = [&](int i) { a.Issue(lds + toA, i); };
    auto copyB = [&](int i) { b.Issue(placesB + toB, i); };
    auto prepareA = [&] {
        a.Prepare(leftA);
        leftA -= kTurnBytes;
        if constexpr (!kDirect) a.Load();
    };
    auto prepareB = [&] {  // after b.LookUp() and a wait
        b.Prepare(leftB);
        leftB -= kTurnBytes;
        if constexpr (!kDirect) b.Load();
    };
    auto doneA = [&] { toA = toA == (kPlacesA - 1) * OperandA::kBytes ? 0 : toA + OperandA::kBytes; };
    auto doneB = [&] { toB ^= OperandB::kBytes; };
    auto copyAllA = [&] {
        prepareA();
        if constexpr (kDirect) {
#pragma unroll
            for (int i = 0; i < kCopiesA; ++i) copyA(i);
        } else {
            a.Commit(lds + toA);
        }
        doneA();
    };
    auto copyTurnB = [&] {
        prepareB();
        if constexpr (kDirect) {
#pragma unroll
            for (int i = 0; i < kCopiesB; ++i) copyB(i);
        }
    };
    copyAllA();
    copyTurnB();
    if constexpr (!kDirect) b.Commit(placesB);
    doneB();
    b.LookUp();
    if (kAhead == 2 && turns > 1) {
        copyAllA();
        Wait<kLeft>();
    } else {
        Wait<0>();
    }
    if (turns > 1) {
        if constexpr (!kDirect) prepareA();
        copyTurnB();
    }
    readB(placesB, 0, 0, NI);
#pragma unroll
    for (int q = 0; q < D; ++q) readA(lds, q);
    int nowA = 0, nowB = 0;
    // copiesA, copiesB: A of the turn kAhead on and B of the one after the next exist; more: the next one does
    auto turn = [&](auto copiesA, auto copiesB, auto more) {
        constexpr bool kA = decltype(copiesA)::value, kB = decltype(copiesB)::value, kMore = decltype(more)::value;
        const char* fromA = lds + nowA;
        const char* fromB = placesB + nowB;
        if constexpr (kA && kDirect) prepareA();
        rows(0, kBefore, fromA, fromB, nullptr, nullptr, kA && kDirect ? kCopiesA : 0, copyA);
        if constexpr (!kDirect && kMore) {
            a.Commit(lds + toA);
            b.Commit(placesB + toB);
        }
        if constexpr (kA) doneA();
        if constexpr (kMore) doneB();
        nowA = nowA == (kPlacesA - 1) * OperandA::kBytes ? 0 : nowA + OperandA::kBytes;
        nowB ^= OperandB::kBytes;
        if constexpr (kB) {
            b.LookUp();
            Wait<kLeft>();
            if constexpr (!kDirect) prepareA();  // in registers until the next turn's are multiplied
            prepareB();
        } else {
            Wait<0>();
        }
        rows(kBefore, kRows, fromA, fromB, kMore ? lds + nowA : nullptr, placesB + nowB,
             kB && kDirect ? kCopiesB : 0, copyB);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    for (int64_t t = 2; t < turns; ++t) turn(yes, yes, yes);
    if (turns > 1) turn(std::bool_constant<kAhead == 1>{}, no, yes);
    turn(no, no, no);
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
template <typename TOut, int MI, int NI, int kLdsBytes, typename Value>
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
                __builtin_memcpy(to, &v, 16);  // whatever C's alignment
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

constexpr int kTileRows = 256;  // of a whole tile

// One tile: MI*WM*16 rows by NI*WN*16 columns, of which each of a team's WM x
// WN waves takes MI x NI instructions' results.
template <typename T, typename TOut, bool kBTrans, bool kAligned, int kTeams, int kPlacesA, int MI, int NI, int WM,
          int WN>
__device__ __forceinline__ void GroupedTile(const GroupedLaunch& p, char* lds, int32_t group, int32_t firstRow,
                                            int32_t endRow, int64_t n0)
{
    constexpr int kThreads = WM * WN * 64, BM = MI * WM * 16, BN = NI * WN * 16;
    using OperandA = RowOperand<T, BM, kThreads, kAligned>;
    using OperandB = std::conditional_t<kBTrans, RowOperand<T, BN, kThreads, kAligned>,
                                        ColumnOperand<T, BN, kThreads, false, kAligned>>;
    constexpr int kLds = kPlacesA * OperandA::kBytes + 2 * OperandB::kBytes;
    const int lane = threadIdx.x & 63, wave = TeamWave<kThreads>();
    const int team = WaveNumber() / (kThreads / 64);
    const int rowA = (wave % WM) * MI * 16, rowB = (wave / WM) * NI * 16;
    typename Mma<T>::Acc acc[MI][NI] = {};
    const bool real = group < p.groups;
    if (real && p.k > 0) {
        const T* bg = static_cast<const T*>(p.b) + group * p.stride_b;
        OperandA a;
        OperandB b;
#pragma unroll
        for (int i = 0; i < OperandA::kLoads; ++i) {
            // rows past the tile's end repeat its first: they are computed and not stored
            const int32_t r = firstRow + OperandA::Row(i);
            const int64_t row = IndexedRow(p.row_index, r < endRow ? r : firstRow, p.rows_a);
            a.ptr[i] = reinterpret_cast<const char*>(static_cast<const T*>(p.a) + row * p.lda) + OperandA::Chunk() * 16;
        }
        // each team takes a run of turns
        const int64_t bytes = p.k * static_cast<int64_t>(sizeof(T));
        const int64_t per = ((bytes + kTurnBytes - 1) / kTurnBytes + kTeams - 1) / kTeams;
        a.tiny = bytes < 16;
        a.Skip(team * per);
        if constexpr (kBTrans) {
#pragma unroll
            for (int i = 0; i < OperandB::kLoads; ++i) {
                const int64_t n = n0 + OperandB::Row(i);
                b.ptr[i] = reinterpret_cast<const char*>(bg + (n < p.n ? n : n0) * p.ldb) + OperandB::Chunk() * 16;
            }
            b.tiny = bytes < 16;
            b.Skip(team * per);
        } else {
            b.Init(bg, p.ldb * 2, n0, p.n, nullptr, p.k, static_cast<int32_t>(team * per * 64),
                   static_cast<int32_t>(p.k));
        }
        MultiplyTile<T, MI, NI, kPlacesA>(a, b, lds + team * kLds, bytes - team * per * kTurnBytes, per, rowA, rowB,
                                          acc);
    }
    if (!JoinTeams<kTeams, kThreads, (kTeams - 1) * kLds>(lds + kLds, acc)) return;
    const int64_t n = n0 + rowB;
    TOut* c = static_cast<TOut*>(p.c) + (firstRow + rowA) * p.ldc + n;
    char* part = lds + wave * (kLds / (WM * WN));
    if constexpr (sizeof(T) == 1) {
        float sa[MI], sb[NI][4];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int32_t r = firstRow + rowA + i * 16 + (lane & 15);
            sa[i] = real && r < endRow ? p.scale_a[IndexedRow(p.row_index, r, p.rows_a)] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NI * 4; ++j) {
            const int64_t at = n + j / 4 * 16 + (lane >> 4) * 4 + j % 4;
            sb[j / 4][j % 4] = real && at < p.n ? p.scale_b[group * p.n + at] : 0.0f;
        }
        StoreTile<TOut, MI, NI, kLds / (WM * WN)>(
            part, c, p.ldc, endRow - firstRow - rowA, p.n - n, [&](int i, int j, float(&v)[4]) {
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = static_cast<float>(acc[i][j][x]) * (sa[i] * sb[j][x]);
            });
    } else {
        StoreTile<TOut, MI, NI, kLds / (WM * WN)>(
            part, c, p.ldc, endRow - firstRow - rowA, p.n - n, [&](int i, int j, float(&v)[4]) {
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = acc[i][j][x];
            });
    }
}

// Tiles of 256x256, or fewer rows where the group's end or a share leaves
// fewer: a tile of 64 or 128 rows costs about that part of a whole one.
//
// Bound by the matrix instructions, whose clock falls with the power that
// random operands draw: alone they sustain 2.05 PFLOP/s of bfloat16.  A tile of
// 256x256 reads each byte of LDS for the most instructions that the registers
// (128 of sums per lane) allow; the operands' five places of 32 KB fill a CU's
// LDS, three of them the first operand's, which is copied two turns ahead.
// 16384 rows in 8 groups, 4096x4096: 454 us, 1.21 PFLOP/s (int8, 32768 rows in
// 16 groups, 2048x4096: 259 us, 2.12); one group of 8192 rows, 8192x8192: 1.42
// and 2.67.  Outside its turns a round of tiles takes about 9.5 us: the search,
// the first copies and the stores.
template <typename T, typename TOut, bool kBTrans>
__global__ __launch_bounds__(512, 1) void GroupedTileKernel(GroupedLaunch p, int32_t tilesN, int32_t cus)
{
    __shared__ __align__(128) char lds[(3 * kTileRows + 2 * 256) * kTurnBytes];  // all of a CU's
    const RaggedTiles tiles(p.offsets, p.rows, p.groups, kTileRows);
    const TileShare share = ShareOfWorkgroup(static_cast<int64_t>(tiles.total) * tilesN, cus);
    if (share.tile < 0) return;
    const RaggedTile tile = tiles.Find(static_cast<int32_t>(share.tile / tilesN));
    if (tile.group < 0) return;
    const TilePlace place = PlaceInBands(share.tile - static_cast<int64_t>(tile.before) * tilesN, tile.tiles, tilesN);
    const int32_t height = kTileRows / share.parts;
    const int32_t row = tile.begin + place.m * kTileRows + share.part * height;
    if (row < tile.begin || row >= tile.end) return;  // also whatever offsets without meaning lead to
    const int32_t end = tile.end - row < height ? tile.end : row + height;
    const int64_t n0 = static_cast<int64_t>(place.n) * 256;
    if (end - row <= 64) {
        GroupedTile<T, TOut, kBTrans, true, 1, 3, 2, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    } else if (end - row <= 128) {
        GroupedTile<T, TOut, kBTrans, true, 1, 3, 4, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    } else {
        GroupedTile<T, TOut, kBTrans, true, 1, 3, 8, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    }
}

// Tiles of 64x128 for groups of few rows: three workgroups per CU, or, where
// there are not tiles enough for that, one whose three teams share a tile's
// contraction.  Bound by the latency of its copies, one turn ahead, and by the
// weights' bytes: 812 rows in 48 groups, 1001x1000, fp16, 22 us (98 MB, 4.4
// TB/s).  Registers are kept to what three workgroups leave each other (the
// input's gradient of 5418 rows in 6 groups x 1144 x 660, which would take a
// few more: 41 us, 51 with two workgroups).
constexpr int kSmallTileBytes = 2 * (64 + 128) * kTurnBytes;
template <typename T, typename TOut, bool kBTrans, bool kAligned, int kTeams>
__global__ __launch_bounds__(kTeams * 256, 3) void GroupedSmallTileKernel(GroupedLaunch p, int32_t tilesN)
{
    __shared__ __align__(128) char lds[kTeams * kSmallTileBytes];
    const RaggedTiles tiles(p.offsets, p.rows, p.groups, 64);
    const TileShare share = ShareOfWorkgroup(static_cast<int64_t>(tiles.total) * tilesN, 1);
    if (share.tile < 0) return;
    const RaggedTile tile = tiles.Find(static_cast<int32_t>(share.tile / tilesN));
    if (tile.group < 0) return;
    const TilePlace place = PlaceInBands(share.tile - static_cast<int64_t>(tile.before) * tilesN, tile.tiles, tilesN);
    const int32_t row = tile.begin + place.m * 64;
    if (row < tile.begin || row >= tile.end) return;
    GroupedTile<T, TOut, kBTrans, kAligned, kTeams, 2, 2, 4, 2, 2>(p, lds, tile.group, row,
                                                        tile.end - row < 64 ? tile.end : row + 64,
                                                        static_cast<int64_t>(place.n) * 128);
}

// Weight gradients, W_g[n, k] = sum over the group's rows of gradC[r, n] *
// X_index(r)[k]: both operands' rows run across the contraction, so both are
// read through the transposing LDS loads, and rows are copied by their index
// as they lie in memory.  Every tile has one workgroup that passes over all of
// its group's rows: no sums between workgroups.  Bound like
// GroupedTileKernel, and by uneven groups, the longest first: 65536 rows in 32
// groups, 2048x2048, bfloat16, 552 to 600 us, 0.92 to 1.0 PFLOP/s.
template <typename T, typename TOut, bool kIndexed, bool kAligned, int kTeams, int kPlacesA, int MI, int NI, int WM,
          int WN>
__global__ __launch_bounds__(kTeams * WM * WN * 64, 1) void GroupedGradTileKernel(GroupedGradLaunch p, int32_t tilesN,
                                                                                int32_t tilesK)
{
    constexpr int kThreads = WM * WN * 64, BM = MI * WM * 16, BN = NI * WN * 16;
    using OperandA = ColumnOperand<T, BM, kThreads, false, kAligned>;
    using OperandB = ColumnOperand<T, BN, kThreads, kIndexed, kAligned>;
    constexpr int kLds = kPlacesA * OperandA::kBytes + 2 * OperandB::kBytes;
    __shared__ __align__(128) char lds[kTeams * kLds];
    // Every die takes an eighth of each group's tiles, so that a long group is no die's alone; which
    // eighth turns with the group, so that the last, shorter ones go round too.
    const int32_t per = (tilesN * tilesK + 7) / 8, at = static_cast<int32_t>(blockIdx.x / 8);
    const int32_t nth = at / per;
    const int32_t id = static_cast<int32_t>((blockIdx.x + nth) % 8) * per + at % per;
    if (id >= tilesN * tilesK) return;
    const int32_t g = LongestGroup(p.offsets, p.rows, static_cast<int32_t>(p.groups), nth);
    const TilePlace place = PlaceInBands(id, tilesN, tilesK);
    const int64_t n0 = static_cast<int64_t>(place.m) * BM, k0 = static_cast<int64_t>(place.n) * BN;
    const int wave = TeamWave<kThreads>(), team = WaveNumber() / (kThreads / 64);
    const int rowA = (wave % WM) * MI * 16, rowB = (wave / WM) * NI * 16;
    int32_t begin, end;
    GroupRows(p.offsets, p.rows, g, begin, end);
    typename Mma<T>::Acc acc[MI][NI] = {};
    if (begin < end) {
        OperandA a;
        OperandB b;
        // each team takes a run of turns
        const int32_t per = ((end - begin + 63) / 64 + kTeams - 1) / kTeams, from = begin + team * per * 64;
        a.Init(p.grad, p.ldg * 2, n0, p.n, nullptr, p.rows, from, end);
        b.Init(p.x, p.ldx * 2, k0, p.k, p.row_index, p.rows_x, from, end);
        MultiplyTile<T, MI, NI, kPlacesA>(a, b, lds + team * kLds, static_cast<int64_t>(end - from) * 2, per, rowA,
                                          rowB, acc);
    }
    if (!JoinTeams<kTeams, kThreads, (kTeams - 1) * kLds>(lds + kLds, acc)) return;
    const int64_t n = n0 + rowA, k = k0 + rowB;
    StoreTile<TOut, MI, NI, kLds / (WM * WN)>(lds + wave * (kLds / (WM * WN)),
                                              static_cast<TOut*>(p.w) + g * p.stride_w + n * p.ldw + k, p.ldw, p.n - n,
                                              p.k - k, [&](int i, int j, float(&v)[4]) {
#pragma unroll
                                                  for (int x = 0; x < 4; ++x) v[x] = acc[i][j][x];
                                              });
}

// ---------------------------------------------------------------------------
// Few rows per group: the weights are read once and bound the time.  A
// workgroup multiplies MT*16 rows by NT*16 columns; its waves split the
// contraction, each lane loading its operands of 16x16 instructions straight
// from memory (16 rows of 64 bytes per load), and add their sums through LDS
// in the order of the waves.  4 groups of 4096x2048 with one row each,
// bfloat16, call after call: 67 MB in 14.7 us, 4.6 TB/s (17.0 with 8 waves).
// ---------------------------------------------------------------------------
template <typename T, typename TOut, bool kAligned, int MT, int NT, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void GroupedRowsKernel(GroupedLaunch p, int32_t tilesN)
{
    using Acc = typename Mma<T>::Acc;
    constexpr int kAhead = 16 / (MT + NT) > 4 ? 8 : 4;  // steps loaded before they are multiplied
    __shared__ Acc part[kWaves][MT * NT][64];
    const RaggedTile tile = RaggedTiles(p.offsets, p.rows, p.groups, MT * 16)
                                .Find(static_cast<int32_t>(blockIdx.x / static_cast<uint32_t>(tilesN)));
    const int32_t n0 = static_cast<int32_t>(blockIdx.x % static_cast<uint32_t>(tilesN)) * NT * 16;
    const int32_t width = static_cast<int32_t>(p.n);
    if (tile.group < 0 || n0 >= width || tile.row < tile.begin || tile.row >= tile.end) return;
    const int lane = threadIdx.x & 63, wave = WaveNumber();
    const bool real = tile.group < p.groups;
    Acc acc[MT][NT] = {};
    if (real) {
        const int32_t bytes = static_cast<int32_t>(p.k) * static_cast<int32_t>(sizeof(T));
        const char* b[NT];
        const char* a[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int32_t n = n0 + j * 16 + (lane & 15);
            b[j] = reinterpret_cast<const char*>(static_cast<const T*>(p.b) + tile.group * p.stride_b +
                                                 (n < width ? n : width - 1) * p.ldb);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int32_t r = tile.row + i * 16 + (lane & 15);
            a[i] = reinterpret_cast<const char*>(
                static_cast<const T*>(p.a) + IndexedRow(p.row_index, r < tile.end ? r : tile.row, p.rows_a) * p.lda);
        }
        // step s is 64 bytes; a wave takes two neighbouring ones, a memory line, at a time
        auto at = [&](int s) { return ((s >> 1) * kWaves + wave) * 128 + (s & 1) * 64 + (lane >> 4) * 16; };
        for (int s0 = 0; ((s0 >> 1) * kWaves + wave) * 128 < bytes; s0 += kAhead) {
            Int4 fb[kAhead][NT], fa[kAhead][MT];
            auto loadAll = [&](auto load) {
#pragma unroll
                for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) fb[s][j] = load(b[j], at(s0 + s));
                }
#pragma unroll
                for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) fa[s][i] = load(a[i], at(s0 + s));
                }
            };
            if (kAligned || (((s0 + kAhead - 1) >> 1) * kWaves + wave + 1) * 128 <= bytes) {
                loadAll([&](const char* row, int32_t byte) {
                    Int4 v;
                    if constexpr (kAligned) {
                        v = *reinterpret_cast<const Int4*>(row + (byte < bytes ? byte : 0));
                        if (byte >= bytes) v = Int4{0, 0, 0, 0};
                    } else {
                        v = LoadBytes(row + byte);
                    }
                    return v;
                });
            } else {
                loadAll([&](const char* row, int32_t byte) {
                    return LoadPart<T>(row + (byte < bytes ? byte : 0), bytes - byte, bytes < 16);
                });
            }
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = Mma<T>::Run(fb[s][j], fa[s][i], acc[i][j]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) part[wave][i][lane] = acc[i / NT][i % NT];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += kWaves) {
        Acc sum = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w][t][lane];
        const int32_t r = tile.row + t / NT * 16 + (lane & 15);
        const int32_t n = n0 + t % NT * 16 + (lane >> 4) * 4;
        if (r >= tile.end) continue;
        float sa = 1.0f;
        if constexpr (sizeof(T) == 1) {
            if (real) sa = p.scale_a[IndexedRow(p.row_index, r, p.rows_a)];
        }
        TOut* c = static_cast<TOut*>(p.c) + r * p.ldc;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (n + x >= width) continue;
            float v = static_cast<float>(sum[x]);
            if constexpr (sizeof(T) == 1) {
                if (real) v *= sa * p.scale_b[tile.group * p.n + n + x];
            }
            c[n + x] = FromFloat<TOut>(v);
        }
    }
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

template <typename T, typename TOut, bool kBTrans>
int LaunchTiles(const GroupedLaunch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, 256);
    // a die may cut the tiles of its last round into four
    const int64_t grid = CeilDiv(MaxRowTiles(l.offsets, l.rows, l.groups, kTileRows) * tilesN, 8) * 8 + 8 * CusPerDie();
    if (!GridFits(grid, 512)) return kTooLarge;
    GroupedTileKernel<T, TOut, kBTrans>
        <<<static_cast<uint32_t>(grid), 512, 0, s>>>(l, static_cast<int32_t>(tilesN), CusPerDie());
    return 0;
}

template <typename T, typename TOut, bool kBTrans, bool kAligned, int kTeams>
int LaunchSmallTiles(const GroupedLaunch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, 128);
    const int64_t grid = CeilDiv(MaxRowTiles(l.offsets, l.rows, l.groups, 64) * tilesN, 8) * 8;
    if (!GridFits(grid, kTeams * 256)) return kTooLarge;
    GroupedSmallTileKernel<T, TOut, kBTrans, kAligned, kTeams>
        <<<static_cast<uint32_t>(grid), kTeams * 256, 0, s>>>(l, static_cast<int32_t>(tilesN));
    return 0;
}

template <typename T, typename TOut, bool kAligned, int MT, int NT>
int LaunchRows(const GroupedLaunch& l, hipStream_t s)
{
    constexpr int kWaves = 4;
    // the row tiles of a group then read a column's weights on one die, whose L2 holds them
    const int64_t tilesN = CeilDiv(CeilDiv(l.n, NT * 16), 8) * 8;
    const int64_t grid = MaxRowTiles(l.offsets, l.rows, l.groups, MT * 16) * tilesN;
    if (!GridFits(grid, kWaves * 64)) return kTooLarge;
    GroupedRowsKernel<T, TOut, kAligned, MT, NT, kWaves>
        <<<static_cast<uint32_t>(grid), kWaves * 64, 0, s>>>(l, static_cast<int32_t>(tilesN));
    return 0;
}

template <typename T, typename TOut, bool kBTrans, bool kAligned>
int GroupedBySize(const GroupedLaunch& l, hipStream_t s)
{
    const int64_t cus = 8 * CusPerDie();
    const int64_t smallTiles = (CeilDiv(l.rows, 64) + (l.groups - 1) / 2) * CeilDiv(l.n, 128);
    if constexpr (kBTrans) {
        // Weights that no cache holds, bf16, us, here / by 64x128 tiles: 8 groups of 4096x4096 with 1 row each 51 /
        // 56, with 4 55 / 57, with 8 64 / 57; 32 of 2048x2048 with 1 53 / 60, with 8 64 / 60.  One group has too few
        // tiles: 4096x4096 with 1 row 10 / 38, with 32 19 / 39, with 64 21 (32 rows a time; 33 with 16) / 41.
        const bool few = l.rows <= 6 * l.groups || (l.rows <= 64 * l.groups && smallTiles <= cus / 4);
        if (few && l.k * static_cast<int64_t>(sizeof(T)) <= INT32_MAX / 2) {
            const int rc = l.rows <= 6 * l.groups || l.rows <= 32 ? LaunchRows<T, TOut, kAligned, 1, 1>(l, s)
                                                                  : LaunchRows<T, TOut, kAligned, 2, 2>(l, s);
            if (rc != kTooLarge) return rc;  // wider tiles may still fit
        }
    }
    // 256x256 tiles / 64x128 ones: 32 groups of 2048x2048 with 128 rows each 97 / 90 us, with 160 96 / 97, with 256
    // 104 / 134; 1 group of 4096x4096 with 1024 rows 51 / 49, with 2048 61 / 95.
    if constexpr (kAligned) {
        if (l.rows >= 160 * l.groups && smallTiles > 3 * cus) return LaunchTiles<T, TOut, kBTrans>(l, s);
    }
    // three teams a tile / one, us: 256 rows x 4096 x 4096 29 / 43; 1024 rows in 4 groups x 512 x 512 7.6 / 7.1; with
    // weights that no cache holds, 512 rows in 32 groups x 2048 x 2048 61 / 72, 816 in 48 x 1024 x 1024 32 / 27
    const int64_t turns = CeilDiv(l.k * static_cast<int64_t>(sizeof(T)), kTurnBytes);
    const bool teams = (smallTiles <= cus && turns >= 12) || (smallTiles <= cus + cus / 2 && turns >= 32);
    return teams ? LaunchSmallTiles<T, TOut, kBTrans, kAligned, 3>(l, s)
                 : LaunchSmallTiles<T, TOut, kBTrans, kAligned, 1>(l, s);
}

template <typename T, typename TOut>
int GroupedTyped(const GroupedLaunch& l, hipStream_t s)
{
    constexpr int64_t kSize = sizeof(T);
    const int64_t inner = l.b_trans ? l.k : l.n;  // what a row of B holds
    const bool aligned = Aligned16(l.a, l.lda * kSize) && Aligned16(l.b, l.ldb * kSize) &&
                         Aligned16(l.b, l.stride_b * kSize) && l.k * kSize % 16 == 0 && inner * kSize % 16 == 0;
    if constexpr (kSize == 2) {
        if (!l.b_trans) {
            return aligned ? GroupedBySize<T, TOut, false, true>(l, s) : GroupedBySize<T, TOut, false, false>(l, s);
        }
    }
    return aligned ? GroupedBySize<T, TOut, true, true>(l, s) : GroupedBySize<T, TOut, true, false>(l, s);
}

template <typename T, typename TOut, bool kAligned, int kTeams, int kPlacesA, int MI, int WN>
int LaunchGradTiles(const GroupedGradLaunch& l, hipStream_t s)
{
    constexpr int WM = 2, NI = 4, kThreads = kTeams * WM * WN * 64;
    const int64_t tilesN = CeilDiv(l.n, MI * WM * 16), tilesK = CeilDiv(l.k, NI * WN * 16);
    if (tilesN * tilesK + 7 > INT32_MAX / l.groups) return kTooLarge;
    const int64_t grid = CeilDiv(tilesN * tilesK, 8) * 8 * l.groups;
    if (!GridFits(grid, kThreads)) return kTooLarge;
    const auto kernel = l.row_index != nullptr
                            ? GroupedGradTileKernel<T, TOut, true, kAligned, kTeams, kPlacesA, MI, NI, WM, WN>
                            : GroupedGradTileKernel<T, TOut, false, kAligned, kTeams, kPlacesA, MI, NI, WM, WN>;
    kernel<<<static_cast<uint32_t>(grid), kThreads, 0, s>>>(l, static_cast<int32_t>(tilesN),
                                                            static_cast<int32_t>(tilesK));
    return 0;
}

template <typename T, typename TOut>
int GroupedGradTyped(const GroupedGradLaunch& l, hipStream_t s)
{
    const bool aligned =
        Aligned16(l.grad, l.ldg * 2) && Aligned16(l.x, l.ldx * 2) && l.n % 8 == 0 && l.k % 8 == 0;
    // 64x128 by three teams / 64x256 / 256x256, us: 4 groups of 4096 rows, 512x512 44 / 71 / 112; 8 of 4096, 1024x1024
    // 253 / 169 / 233; 32 of 256, 2048x2048 - / 261 / 131
    const bool fewest = CeilDiv(l.n, 64) * CeilDiv(l.k, 128) * l.groups <= 8 * CusPerDie();
    if (!aligned) {
        return fewest ? LaunchGradTiles<T, TOut, false, 3, 2, 2, 2>(l, s)
                      : LaunchGradTiles<T, TOut, false, 1, 2, 2, 4>(l, s);
    }
    if (fewest) return LaunchGradTiles<T, TOut, true, 3, 2, 2, 2>(l, s);
    const bool many = CeilDiv(l.n, 256) * CeilDiv(l.k, 256) * l.groups >= 6 * CusPerDie();
    return many ? LaunchGradTiles<T, TOut, true, 1, 3, 8, 4>(l, s) : LaunchGradTiles<T, TOut, true, 1, 3, 2, 4>(l, s);
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
