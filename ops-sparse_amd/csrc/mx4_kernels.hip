// Microscaled 4-bit floating point: rows of blocks of 32 values, each block
// with a power of two for a scale (the format of OCP's Microscaling
// specification with elements e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives), and the ragged products grouped by expert of two operands in it.
//
// gfx950 multiplies such operands itself: one instruction takes 128 values of
// each of 16 rows with the scales of their four blocks.  It takes as many bytes
// per clock as the 16-bit ones, for four times the products, so the tiles are
// those of the 16-bit products with the scales beside them.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "experts_device.h"
#include "experts_internal.h"
#include "grouped_tile.h"
#include "model_ops_internal.h"

namespace aclsp {
namespace {

using Int8x = int __attribute__((ext_vector_type(8)));
using Float2 = float __attribute__((ext_vector_type(2)));

constexpr int kDppQuadXor1 = 0xB1, kDppQuadXor2 = 0x4E;

// 2^(e - 127) for e in [0, 254], NaN for 255
__device__ __forceinline__ float ScaleValue(uint32_t e)
{
    return __uint_as_float(e == 0 ? 0x00400000U : e == 255 ? 0x7FC00000U : e << 23);
}

// ---------------------------------------------------------------------------
// To the format and back.  Four lanes share a block, eight values each: loads
// and stores of 16 and 4 bytes, the largest value by two exchanges in the quad.
// Bound by memory.  16381 rows of 4096 bf16 values there and back: 27.6 us (170
// MB, 6.2 TB/s of what the L2s partly hold) and 24.6 us (6.9 TB/s; most of it
// is written past the L2); one row 2.0 and 2.1 us, a round of latency.
// ---------------------------------------------------------------------------
// Values [c, c + 8) of a row of k, zeros past its end.
template <typename T>
__device__ __forceinline__ void LoadEight(const T* row, int64_t c, int64_t k, float (&v)[8])
{
    T t[8];
    if (c + 8 <= k) {
        __builtin_memcpy(t, row + c, sizeof(t));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ToFloat(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < k ? ToFloat(row[c + i]) : 0.0f;
    }
}

// The scale's exponent is that of the block's largest value less 2, e2m1's
// largest exponent; each value over the scale is rounded to the nearest of the
// format, ties to the even code, and at most 6.  A block with a value that is
// not finite has the scale NaN.  Dividing by the scale is exact, so the codes are
// those of the definition whatever the order of the steps.
template <typename T>
__global__ __launch_bounds__(256) void Mx4QuantizeKernel(Mx4Rows p, uint32_t chunks, uint32_t total)
{
    const uint32_t id = blockIdx.x * 256U + threadIdx.x;
    if (id >= total) return;  // whole quads: chunks are four to a block
    const uint32_t row = id / chunks, chunk = id - row * chunks;
    float v[8];
    LoadEight(static_cast<const T*>(p.x) + row * p.ldx, static_cast<int64_t>(chunk) * 8, p.k, v);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7FFFFFFFU;
        most = bits > most ? bits : most;
    }
    auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    most = larger(most, Dpp<kDppQuadXor1, 0xF>(most, most));
    most = larger(most, Dpp<kDppQuadXor2, 0xF>(most, most));
    const uint32_t field = most >> 23;
    const uint32_t e = field == 255 ? 255 : field < 2 ? 0 : field - 2;
    const float inverse = __uint_as_float((254U - e) << 23);  // of a scale up to 2^125: never subnormal
    uint32_t code = 0;
    if (e != 255) {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[0] * inverse, v[1] * inverse, 1.0f, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[2] * inverse, v[3] * inverse, 1.0f, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[4] * inverse, v[5] * inverse, 1.0f, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[6] * inverse, v[7] * inverse, 1.0f, 3);
    }
    __builtin_memcpy(p.codes + row * p.ld_codes + chunk * 4, &code, 4);
    if ((chunk & 3) == 0) p.scales[row * p.ld_scales + (chunk >> 2)] = static_cast<uint8_t>(e);
}

template <typename T>
__global__ __launch_bounds__(256) void Mx4DequantizeKernel(Mx4Rows p, uint32_t chunks, uint32_t total)
{
    const uint32_t id = blockIdx.x * 256U + threadIdx.x;
    if (id >= total) return;
    const uint32_t row = id / chunks, chunk = id - row * chunks;
    uint32_t code;
    __builtin_memcpy(&code, p.codes + row * p.ld_codes + chunk * 4, 4);
    const float scale = ScaleValue(p.scales[row * p.ld_scales + (chunk >> 2)]);
    // decoded for a scale of one and multiplied: whatever the instruction makes of the scales at the range's ends
    const Float2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0);
    const Float2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1);
    const Float2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2);
    const Float2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3);
    const float v[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = FromFloat<T>(v[i] * scale);
    const int64_t at = static_cast<int64_t>(chunk) * 8;
    T* to = static_cast<T*>(p.x) + row * p.ldx + at;
    if (at + 8 <= p.k) {
        StoreStreaming<sizeof(t)>(to, t);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (at + i < p.k) to[i] = t[i];
        }
    }
}

// ---------------------------------------------------------------------------
// Products.
// ---------------------------------------------------------------------------

// acc += a b^T for 16 rows of each operand and 128 of the contraction: lane l
// holds block l / 16 of row l % 16, in 16 bytes, and in byte kA (kB) of scaleA
// (scaleB) its scale.  The result's lane l holds column l % 16 (row of b) and
// rows 4 * (l / 16) + i (of a).
template <int kA, int kB>
__device__ __forceinline__ Float4 MmaMx4(Int4 a, Int4 b, Float4 c, uint32_t scaleA, uint32_t scaleB)
{
    constexpr int kFp4 = 4;
    const Int8x wideA = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    const Int8x wideB = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wideA, wideB, c, kFp4, kFp4, kA, static_cast<int>(scaleA),
                                                            kB, static_cast<int>(scaleB));
}

// The same with the sum kept where it is.  The builtin may put it elsewhere, and did: the loop over a 256x256 tile then
// moved all 128 registers of sums each turn and spilled others.  Assembly is outside the compiler's count of the wait
// that a matrix instruction needs behind an ordinary one that wrote an operand (two states, for which the s_nop stands;
// the instruction before it is still at work then), and of that behind the last one (SettleSums).
template <int kA, int kB>
__device__ __forceinline__ void AddMx4(Int4 a, Int4 b, Float4& c, uint32_t scaleA, uint32_t scaleB)
{
    asm volatile(
        "s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] "
        "cbsz:4 blgp:4"
        : "+v"(c)
        : "v"(a), "v"(b), "v"(scaleA), "v"(scaleB), "n"(kA & 1), "n"(kB & 1), "n"(kA >> 1), "n"(kB >> 1));
}

// Before other instructions read the sums: a matrix instruction's result takes up to 18 states.
template <int MI, int NI>
__device__ __forceinline__ void SettleSums(Float4 (&acc)[MI][NI])
{
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int i = 0; i < MI * NI; ++i) asm volatile("" : "+v"(acc[i / NI][i % NI]));
}

// The scales of a tile's operands, RA and RB rows in groups of GA and GB that
// one wave multiplies: sixteen bytes per row and two turns.  A load touches a
// memory line per row, however few bytes it takes of it, so few loads of many
// bytes are better (with eight bytes each turn, scales took a fifth of a
// turn).  They are loaded into registers, a thread's rows one after another over
// both operands, and put into LDS so that a lane reads those of all its
// instructions at once: within a group of G rows, the word of row 16 i + r and
// block b of each of the four steps lies at word (16 b + r) * G / 16 + i.
template <int RA, int GA, int RB, int GB, int kThreads>
struct ScaleRows {
    static constexpr int kBytes = (RA + RB) * 16;
    static constexpr int kLoads = (RA + RB + kThreads - 1) / kThreads;
    const uint8_t* ptr[kLoads];
    Int4 held[kLoads];

    // of both operands: below RA the first one's
    static __device__ __forceinline__ int Row(int i) { return i * kThreads + TeamThread<kThreads>(); }

    // The next two turns', of which `blocks` are left; zeros past the row's end.  A row's last bytes are read by the
    // sixteen that end there and shifted, without a branch (one in the loop costs registers, and time each turn).
    __device__ __forceinline__ void Load(int64_t blocks)
    {
        const int64_t over = blocks < 16 ? 16 - blocks : 0;
        const int bits = over < 16 ? static_cast<int>(over) * 8 : 0;
        const uint64_t mask = over < 16 ? ~uint64_t{0} : 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const Int4 v = LoadBytes(reinterpret_cast<const char*>(ptr[i] - over));
            uint64_t half[2];
            __builtin_memcpy(half, &v, 16);
            const uint64_t low = bits >= 64 ? half[1] >> (bits & 63) : half[0] >> bits | half[1] << 1 << (63 - bits);
            half[1] = bits >= 64 ? 0 : half[1] >> bits & mask;
            half[0] = low & mask;
            __builtin_memcpy(&held[i], half, 16);
            ptr[i] += 16;
        }
    }
    // The only turns of rows of fewer than sixteen.
    __device__ __forceinline__ void LoadShort(int64_t blocks)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            uint64_t half[2] = {0, 0};
            for (int64_t c = 0; c < blocks; ++c) {
                half[c / 8] |= static_cast<uint64_t>(((const __attribute__((address_space(1))) uint8_t*)(ptr[i]))[c])
                               << (8 * (c % 8));
            }
            __builtin_memcpy(&held[i], half, 16);
        }
    }
    template <int G>
    static __device__ __forceinline__ void Put(char* lds, int row, const Int4& v)
    {
        char* to = lds + row / G * (G * 16) + row % 16 * (G / 4) + row % G / 16 * 4;
        // a word of each block's bytes in the four steps: the transpose of 4 x 4 bytes
        const uint32_t w[4] = {static_cast<uint32_t>(v[0]), static_cast<uint32_t>(v[1]), static_cast<uint32_t>(v[2]),
                               static_cast<uint32_t>(v[3])};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            // bytes 0 to 3 of a selection are of the second operand, 4 to 7 of the first, 12 is zero
            const uint32_t pair = 0x0C0C0400U + static_cast<uint32_t>(b) * 0x0101U;
            const uint32_t low = __builtin_amdgcn_perm(w[1], w[0], pair), high = __builtin_amdgcn_perm(w[3], w[2], pair);
            *reinterpret_cast<uint32_t*>(to + b * (4 * G)) = low | high << 16;
        }
    }
    __device__ __forceinline__ void Commit(char* lds)
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row = Row(i);
            if (row < RA) {
                Put<GA>(lds, row, held[i]);
            } else if (kLoads * kThreads == RA + RB || row < RA + RB) {
                Put<GB>(lds + RA * 16, row - RA, held[i]);
            }
        }
    }
    template <int G>
    static __device__ __forceinline__ void Read(const char* lds, int group, uint32_t (&word)[G / 16])
    {
        __builtin_memcpy(word, __builtin_assume_aligned(lds + group * (G * 16) + (threadIdx.x & 63) * (G / 4), G / 4),
                         G / 4);
    }
};

template <int I, int N, typename F>
__device__ __forceinline__ void Unroll(F f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        Unroll<I + 1, N>(f);
    }
}

// acc += the product over `blocks` of the contraction in `turns` turns of eight, those past the blocks of zeros; MI x NI
// instructions' results per wave, from rows rowA and rowB on.
//
// Like the 16-bit products' turns: two matrix steps of MI rows of products each; after a row's products come the reads
// of the first operand D rows on and of the second operand's next step; one barrier per turn, before its last D rows.
// Both operands have two places in LDS.  Turns go in pairs, whose scales have one place: those of the next pair are put
// there behind the barrier of a pair's first turn, when all waves have read this pair's, and read at the end of its
// second; they were loaded a pair before that.
template <int MI, int NI, typename OperandA, typename OperandB, typename Scales>
__device__ __forceinline__ void MultiplyMx4(OperandA& a, OperandB& b, Scales& scales, char* lds, int64_t blocks,
                                            int64_t turns, bool tiny, int rowA, int rowB, Float4 (&acc)[MI][NI])
{
    constexpr int kCopiesA = OperandA::kLoads, kCopiesB = OperandB::kLoads;
    constexpr int D = MI >= 4 ? MI / 2 : 2, kRows = kSteps * MI, kBefore = kRows - D;
    char* const placesB = lds + 2 * OperandA::kBytes;
    char* const placeS = placesB + 2 * OperandB::kBytes;
    const int groupA = rowA / (MI * 16), groupB = rowB / (NI * 16);
    Int4 fa[D], fb[kSteps][NI];
    uint32_t scaleA[MI], scaleB[NI];
    auto readA = [&](const char* from, int q) { fa[q % D] = OperandA::Read(from, rowA + q % MI * 16, q / MI); };
    auto readB = [&](const char* from, int s, int first, int last) {
#pragma unroll
        for (int j = first; j < last; ++j) fb[s][j] = OperandB::Read(from, rowB + j * 16, s);
    };
    auto readScales = [&] {
        Scales::template Read<MI * 16>(placeS, groupA, scaleA);
        Scales::template Read<NI * 16>(placeS + OperandA::kBytes / kTurnBytes * 16, groupB, scaleB);
    };
    // Rows [first, last) of a pair's first or second turn, in this order to the instruction; nextA: null, or where the
    // next turn's operands are.
    auto rows = [&](auto second, auto first, auto last, const char* fromA, const char* fromB, const char* nextA,
                    const char* nextB, int copies, auto copy) {
        constexpr int kFirst = decltype(first)::value, kLast = decltype(last)::value;
        Unroll<kFirst, kLast>([&](auto at) {
            constexpr int q = decltype(at)::value, s = q / MI, i = q % MI, byte = decltype(second)::value * 2 + s;
            Unroll<0, NI>([&](auto column) {
                constexpr int j = decltype(column)::value;
                AddMx4<byte, byte>(fb[s][j], fa[q % D], acc[i][j], scaleB[j], scaleA[i]);
            });
            if (q < kBefore) {
                readA(fromA, q + D);
            } else if (nextA != nullptr) {
                readA(nextA, q - kBefore);
                readB(nextB, 0, (q - kBefore) * NI / D, (q - kBefore + 1) * NI / D);
            }
            if (q < MI / 2) readB(fromB, 1, q * NI / (MI / 2), (q + 1) * NI / (MI / 2));
            // close behind the barrier: what is copied last is waited for at the end of the turn
            constexpr int n = kFirst == 0 ? (kLast + 2) / 3 : kLast - kFirst;
#pragma unroll
            for (int c = (q - kFirst) * copies / n; c < (q - kFirst + 1) * copies / n && c < copies; ++c) copy(c);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    int64_t leftA = blocks * 16, leftB = blocks * 16, leftS = blocks;
    int toA = 0, toB = 0;  // places of the next copies, in bytes
    auto copyA = [&](int i) { a.Issue(lds + toA, i); };
    auto copyB = [&](int i) { b.Issue(placesB + toB, i); };
    auto prepareA = [&] {
        a.Prepare(leftA);
        leftA -= kTurnBytes;
    };
    auto prepareB = [&] {
        b.Prepare(leftB);
        leftB -= kTurnBytes;
    };
    auto loadScales = [&] {
        scales.Load(leftS);
        leftS -= 16;
    };
    // all loads at once, so that their latency is waited for once
    prepareA();
#pragma unroll
    for (int i = 0; i < kCopiesA; ++i) copyA(i);
    toA ^= OperandA::kBytes;
    prepareB();
#pragma unroll
    for (int i = 0; i < kCopiesB; ++i) copyB(i);
    toB ^= OperandB::kBytes;
    if (tiny) {
        scales.LoadShort(leftS);
        scales.Commit(placeS);
    } else {
        Scales first = scales;
        first.Load(leftS);
        scales = first;
        leftS -= 16;
        loadScales();
        first.Commit(placeS);
    }
    Wait<0>();
    int nowA = 0, nowB = 0;
    readScales();
    prepareB();
#pragma unroll
    for (int i = 0; i < kCopiesB; ++i) copyB(i);
    readB(placesB, 0, 0, NI);
#pragma unroll
    for (int q = 0; q < D; ++q) readA(lds, q);
    // second: of a pair; oneMore, twoMore: that many turns come after this one
    auto turn = [&](auto second, auto oneMore, auto twoMore) {
        constexpr bool kSecond = decltype(second)::value, kMore = decltype(oneMore)::value,
                       kTwo = decltype(twoMore)::value;
        const char* fromA = lds + nowA;
        const char* fromB = placesB + nowB;
        if constexpr (kMore) prepareA();
        rows(second, std::integral_constant<int, 0>{}, std::integral_constant<int, kBefore>{}, fromA, fromB, nullptr,
             nullptr, kMore ? kCopiesA : 0, copyA);
        toA ^= OperandA::kBytes;
        toB ^= OperandB::kBytes;
        nowA ^= OperandA::kBytes;
        nowB ^= OperandB::kBytes;
        Wait<0>();
        if constexpr (!kSecond && kTwo) {
            scales.Commit(placeS);
            loadScales();
        }
        if constexpr (kTwo) prepareB();
        rows(second, std::integral_constant<int, kBefore>{}, std::integral_constant<int, kRows>{}, fromA, fromB,
             kMore ? lds + nowA : nullptr, placesB + nowB, kTwo ? kCopiesB : 0, copyB);
        if constexpr (kSecond && kMore) readScales();
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    for (int64_t t = 2; t < turns; t += 2) {
        turn(first, yes, yes);
        turn(second, yes, yes);
    }
    turn(first, yes, no);
    turn(second, no, no);
    SettleSums(acc);
}

// 256x256 tiles by eight waves, one workgroup per CU, as the 16-bit products' but for the scales: the largest tile whose
// sums fit the registers, as each operand byte that comes into a CU then serves most products.  32768 rows by 8 groups of
// 4096 columns over 4096: 311 us, 3.5 PFLOP/s; the instructions alone reach 6.8 on random operands, for the clock that
// their power leaves.  One group of 8192 x 8192: a turn takes 1.8 us, of which the matrix instructions and the barrier
// alone 1.15, copies 0.3, scales 0.15, reads of LDS 0.1; a round of tiles takes 4.5 us of stores and 2 us of dispatch
// besides.  Slower: a ring of four half turns whose scales are copied by words (396 us for 339 at the time), four waves of
// 128x128 (378 for 348).
constexpr int kMx4TileRows = 256;

// One tile: MI*WM*16 rows by NI*WN*16 columns, of which each of a team's WM x
// WN waves takes MI x NI instructions' results.
// kStream: the output is large.
template <typename TOut, int kTeams, bool kStream, int MI, int NI, int WM, int WN>
__device__ __forceinline__ void Mx4Tile(const Mx4Launch& p, char* lds, int32_t group, int32_t firstRow, int32_t endRow,
                                        int64_t n0)
{
    constexpr int kThreads = WM * WN * 64, BM = MI * WM * 16, BN = NI * WN * 16;
    using OperandA = RowOperand<int8_t, BM, kThreads, true>;
    using OperandB = RowOperand<int8_t, BN, kThreads, true>;
    using Scales = ScaleRows<BM, MI * 16, BN, NI * 16, kThreads>;
    constexpr int kLds = 2 * (OperandA::kBytes + OperandB::kBytes) + Scales::kBytes;
    const int wave = TeamWave<kThreads>(), team = WaveNumber() / (kThreads / 64);
    const int rowA = (wave % WM) * MI * 16, rowB = (wave / WM) * NI * 16;
    Float4 acc[MI][NI] = {};
    if (group < p.groups && p.blocks > 0) {
        const uint8_t* codes = p.b.codes + group * p.b.stride;
        const uint8_t* scales = p.b.scales + group * p.b.stride_scales;
        OperandA a;
        OperandB b;
        Scales scale;
        auto rowOfA = [&](int at) {  // rows past the tile's end repeat its first: they are computed and not stored
            const int32_t r = firstRow + at;
            return IndexedRow(p.row_index, r < endRow ? r : firstRow, p.rows_a);
        };
        auto rowOfB = [&](int at) { return n0 + at < p.n ? n0 + at : n0; };
        // each team takes a run of turns
        const int64_t per = ((p.blocks + 15) / 16 + kTeams - 1) / kTeams * 2, skip = team * per * 8;
#pragma unroll
        for (int i = 0; i < OperandA::kLoads; ++i) {
            a.ptr[i] = reinterpret_cast<const char*>(p.a.codes) + rowOfA(OperandA::Row(i)) * p.a.ld +
                       OperandA::Chunk() * 16 + skip * 16;
        }
#pragma unroll
        for (int i = 0; i < OperandB::kLoads; ++i) {
            b.ptr[i] = reinterpret_cast<const char*>(codes) + rowOfB(OperandB::Row(i)) * p.b.ld +
                       OperandB::Chunk() * 16 + skip * 16;
        }
#pragma unroll
        for (int i = 0; i < Scales::kLoads; ++i) {
            const int row = Scales::Row(i), column = row - BM < BN ? row - BM : 0;
            scale.ptr[i] = skip + (row < BM ? p.a.scales + rowOfA(row) * p.a.ld_scales
                                            : scales + rowOfB(column) * p.b.ld_scales);
        }
        MultiplyMx4<MI, NI>(a, b, scale, lds + team * kLds, p.blocks - skip, per, p.blocks < 16, rowA, rowB,
                            acc);
    }
    if (!JoinTeams<kTeams, kThreads, (kTeams - 1) * kLds>(lds + kLds, acc)) return;
    const int64_t n = n0 + rowB;
    constexpr int kPart = kLds / (WM * WN) / 128 * 128;
    StoreTile<TOut, MI, NI, kPart, kStream>(lds + wave * kPart, static_cast<TOut*>(p.c) + (firstRow + rowA) * p.ldc + n, p.ldc,
                                   endRow - firstRow - rowA, p.n - n, [&](int i, int j, float(&v)[4]) {
#pragma unroll
                                       for (int x = 0; x < 4; ++x) v[x] = acc[i][j][x];
                                   });
}

template <typename TOut>
__global__ __launch_bounds__(512, 1) void Mx4TileKernel(Mx4Launch p, int32_t tilesN, int32_t cus)
{
    __shared__ __align__(128) char lds[(kMx4TileRows + 256) * (2 * kTurnBytes + 16)];
    const RaggedTiles tiles(p.offsets, p.rows, p.groups, kMx4TileRows);
    const TileShare share = ShareOfWorkgroup(static_cast<int64_t>(tiles.total) * tilesN, cus);
    if (share.tile < 0) return;
    const RaggedTile tile = tiles.Find(static_cast<int32_t>(share.tile / tilesN));
    if (tile.group < 0) return;
    const TilePlace place = PlaceInBands(share.tile - static_cast<int64_t>(tile.before) * tilesN, tile.tiles, tilesN);
    const int32_t height = kMx4TileRows / share.parts;
    const int32_t row = tile.begin + place.m * kMx4TileRows + share.part * height;
    if (row < tile.begin || row >= tile.end) return;  // also whatever offsets without meaning lead to
    const int32_t end = tile.end - row < height ? tile.end : row + height;
    const int64_t n0 = static_cast<int64_t>(place.n) * 256;
    if (end - row <= 64) {
        Mx4Tile<TOut, 1, true, 2, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    } else if (end - row <= 128) {
        Mx4Tile<TOut, 1, true, 4, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    } else {
        Mx4Tile<TOut, 1, true, 8, 4, 2, 4>(p, lds, tile.group, row, end, n0);
    }
}

// Tiles of 64x128 for groups of few rows: three workgroups per CU, or one whose
// three teams share a tile's contraction.  Bound by the latency of a turn's
// copies, 1 us, one turn ahead: 512 rows x 4096 x 4096 12.1 us, 812 rows of 48
// groups of 1001 x 1000 8.5 us (3.3 TB/s).
constexpr int kMx4SmallBytes = (64 + 128) * (2 * kTurnBytes + 16);
template <typename TOut, int kTeams>
__global__ __launch_bounds__(kTeams * 256, 3) void Mx4SmallTileKernel(Mx4Launch p, int32_t tilesN)
{
    __shared__ __align__(128) char lds[kTeams * kMx4SmallBytes];
    const RaggedTiles tiles(p.offsets, p.rows, p.groups, 64);
    const TileShare share = ShareOfWorkgroup(static_cast<int64_t>(tiles.total) * tilesN, 1);
    if (share.tile < 0) return;
    const RaggedTile tile = tiles.Find(static_cast<int32_t>(share.tile / tilesN));
    if (tile.group < 0) return;
    const TilePlace place = PlaceInBands(share.tile - static_cast<int64_t>(tile.before) * tilesN, tile.tiles, tilesN);
    const int32_t row = tile.begin + place.m * 64;
    if (row < tile.begin || row >= tile.end) return;
    Mx4Tile<TOut, kTeams, false, 2, 4, 2, 2>(p, lds, tile.group, row, tile.end - row < 64 ? tile.end : row + 64,
                                      static_cast<int64_t>(place.n) * 128);
}

// Few rows per group: the weights are read once and bound the time.  A
// workgroup multiplies MT*16 rows by NT*16 columns; its waves split the
// contraction, each lane loading its operands and their scales straight from
// memory, and add their sums through LDS in the order of the waves.  4 rows of 4
// groups of 4096 x 2048: 7.2 us for 18 MB from memory, a chain of two loads
// (offsets, then operands) and the sums behind a launch of 3.6.
template <typename TOut, int MT, int NT, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void Mx4RowsKernel(Mx4Launch p, int32_t tilesN)
{
    __shared__ Float4 part[kWaves][MT * NT][64];
    const RaggedTile tile = RaggedTiles(p.offsets, p.rows, p.groups, MT * 16)
                                .Find(static_cast<int32_t>(blockIdx.x / static_cast<uint32_t>(tilesN)));
    const int32_t n0 = static_cast<int32_t>(blockIdx.x % static_cast<uint32_t>(tilesN)) * NT * 16;
    const int32_t width = static_cast<int32_t>(p.n);
    if (tile.group < 0 || n0 >= width || tile.row < tile.begin || tile.row >= tile.end) return;
    const int lane = threadIdx.x & 63, wave = WaveNumber();
    Float4 acc[MT][NT] = {};
    if (tile.group < p.groups && p.blocks > 0) {
        const int32_t blocks = static_cast<int32_t>(p.blocks);
        // the rows' indices first and what needs them last: the weights' loads go out between
        int32_t index[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int32_t r = tile.row + i * 16 + (lane & 15);
            index[i] = r < tile.end ? r : tile.row;
            if (p.row_index != nullptr) index[i] = p.row_index[index[i]];
        }
        const uint8_t *b[NT], *sb[NT], *a[MT], *sa[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t n = n0 + j * 16 + (lane & 15) < width ? n0 + j * 16 + (lane & 15) : width - 1;
            b[j] = p.b.codes + tile.group * p.b.stride + n * p.b.ld;
            sb[j] = p.b.scales + tile.group * p.b.stride_scales + n * p.b.ld_scales;
        }
        // step s is four blocks; a wave takes two neighbouring ones, a memory line, at a time
        auto at = [&](int s) { return ((s >> 1) * kWaves + wave) * 8 + (s & 1) * 4 + (lane >> 4); };
        auto load = [&](const uint8_t* codes, const uint8_t* scales, int s, Int4& f, uint32_t& e) {
            const int block = at(s) < blocks ? at(s) : 0;
            f = *reinterpret_cast<const Int4*>(codes + block * static_cast<int64_t>(16));
            e = scales[block];
            if (at(s) >= blocks) {
                f = Int4{0, 0, 0, 0};
                e = 0;
            }
        };
        // kAhead steps from s0 on, all loaded before they are multiplied
        auto steps = [&](auto ahead, int s0, bool first) {
            constexpr int kAhead = decltype(ahead)::value;
            Int4 fb[kAhead][NT], fa[kAhead][MT];
            uint32_t eb[kAhead][NT], ea[kAhead][MT];
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                for (int j = 0; j < NT; ++j) load(b[j], sb[j], s0 + s, fb[s][j], eb[s][j]);
            }
            if (first) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    // stays within the operand whatever the index holds
                    const int64_t row = index[i] < 0 || index[i] >= p.rows_a ? 0 : index[i];
                    a[i] = p.a.codes + row * p.a.ld;
                    sa[i] = p.a.scales + row * p.a.ld_scales;
                }
            }
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                for (int i = 0; i < MT; ++i) load(a[i], sa[i], s0 + s, fa[s][i], ea[s][i]);
            }
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        acc[i][j] = MmaMx4<0, 0>(fb[s][j], fa[s][i], acc[i][j], eb[s][j], ea[s][i]);
                    }
                }
            }
        };
        constexpr int kMost = 16 / (MT + NT) > 4 ? 8 : 4;  // steps at once
        constexpr std::integral_constant<int, kMost> most{};
        if (blocks <= kWaves * kMost * 2) {
            // half as many cover the row: no loads past its end
            steps(std::integral_constant<int, kMost / 2>{}, 0, true);
        } else {
            steps(most, 0, true);
            for (int s0 = kMost; ((s0 >> 1) * kWaves + wave) * 8 < blocks; s0 += kMost) steps(most, s0, false);
        }
    }
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) part[wave][i][lane] = acc[i / NT][i % NT];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += kWaves) {
        Float4 sum = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += part[w][t][lane];
        const int32_t r = tile.row + t / NT * 16 + (lane & 15);
        const int32_t n = n0 + t % NT * 16 + (lane >> 4) * 4;
        if (r >= tile.end) continue;
        TOut* c = static_cast<TOut*>(p.c) + r * p.ldc;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (n + x < width) c[n + x] = FromFloat<TOut>(sum[x]);
        }
    }
}

template <typename TOut>
int LaunchMx4Tiles(const Mx4Launch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, 256);
    // a die may cut the tiles of its last round into four
    const int64_t grid =
        CeilDiv(MaxRowTiles(l.offsets, l.rows, l.groups, kMx4TileRows) * tilesN, 8) * 8 + 8 * CusPerDie();
    if (!GridFits(grid, 512)) return kTooLarge;
    Mx4TileKernel<TOut>
        <<<static_cast<uint32_t>(grid), 512, 0, s>>>(l, static_cast<int32_t>(tilesN), CusPerDie());
    return 0;
}

template <typename TOut, int kTeams>
int LaunchMx4SmallTiles(const Mx4Launch& l, hipStream_t s)
{
    const int64_t tilesN = CeilDiv(l.n, 128);
    const int64_t grid = CeilDiv(MaxRowTiles(l.offsets, l.rows, l.groups, 64) * tilesN, 8) * 8;
    if (!GridFits(grid, kTeams * 256)) return kTooLarge;
    Mx4SmallTileKernel<TOut, kTeams>
        <<<static_cast<uint32_t>(grid), kTeams * 256, 0, s>>>(l, static_cast<int32_t>(tilesN));
    return 0;
}

template <typename TOut, int MT, int NT>
int LaunchMx4Rows(const Mx4Launch& l, hipStream_t s)
{
    constexpr int kWaves = 4;
    // the row tiles of a group then read a column's weights on one die, whose L2 holds them
    const int64_t tilesN = CeilDiv(CeilDiv(l.n, NT * 16), 8) * 8;
    const int64_t grid = MaxRowTiles(l.offsets, l.rows, l.groups, MT * 16) * tilesN;
    if (!GridFits(grid, kWaves * 64)) return kTooLarge;
    Mx4RowsKernel<TOut, MT, NT, kWaves>
        <<<static_cast<uint32_t>(grid), kWaves * 64, 0, s>>>(l, static_cast<int32_t>(tilesN));
    return 0;
}

template <typename TOut>
int Mx4BySize(const Mx4Launch& l, hipStream_t s)
{
    switch (Mx4KernelOf(l.groups, l.rows, l.n, l.blocks, 8 * CusPerDie())) {
        case Mx4Kernel::kRows16: return LaunchMx4Rows<TOut, 1, 1>(l, s);
        case Mx4Kernel::kRows32: return LaunchMx4Rows<TOut, 2, 1>(l, s);
        case Mx4Kernel::kRows32x2: return LaunchMx4Rows<TOut, 2, 2>(l, s);
        case Mx4Kernel::kTiles: return LaunchMx4Tiles<TOut>(l, s);
        case Mx4Kernel::kSmallTiles: return LaunchMx4SmallTiles<TOut, 1>(l, s);
        case Mx4Kernel::kSmallTilesTeams: return LaunchMx4SmallTiles<TOut, 3>(l, s);
    }
    return kTooLarge;
}

// Launches of fewer than 2^31 threads each, so that a thread's number and its row's fit 32 bits.
template <typename F>
int ByRows(const Mx4Rows& l, int64_t elementBytes, F launch)
{
    const int64_t chunks = CeilDiv(l.k, kMx4Block) * 4;
    if (chunks > INT32_MAX) return kTooLarge;
    const int64_t most = INT32_MAX / chunks;
    for (int64_t first = 0; first < l.rows; first += most) {
        Mx4Rows part = l;
        part.rows = l.rows - first < most ? l.rows - first : most;
        part.x = static_cast<char*>(l.x) + first * l.ldx * elementBytes;
        part.codes = l.codes + first * l.ld_codes;
        part.scales = l.scales + first * l.ld_scales;
        const int64_t total = part.rows * chunks;
        launch(part, static_cast<uint32_t>(CeilDiv(total, 256)), static_cast<uint32_t>(chunks),
               static_cast<uint32_t>(total));
    }
    return 0;
}

}  // namespace

// The times beside the rules are microseconds with weights that no cache holds.
Mx4Kernel Mx4KernelOf(int64_t groups, int64_t rows, int64_t n, int64_t blocks, int64_t cus)
{
    auto tiles = [&](int64_t height, int64_t width) {  // about as many as there are
        const int64_t most = rows / height + groups;
        return (most < rows ? most : rows) * CeilDiv(n, width);
    };
    // Few rows, while the chip holds all workgroups at once, here / by 64x128 tiles: 4 groups of 4096x2048 with 1 row each
    // 9.0 / 12.0, with 6 9.2 / 12.0; 8 of 4096x4096 with 1 21 / 20; 48 of 1000x1024 with 4 21 / 11.  One group of
    // 4096x4096: 16 rows 9.1 (16 rows a time), 32 9.4 (32 a time; 11.1 with 16) / 17, 64 11.5 (32 by 32) / 17.
    if (blocks <= INT32_MAX / 32) {
        if (rows <= 16 * groups) {
            if (tiles(16, 16) <= 4 * cus) return Mx4Kernel::kRows16;
        } else if (rows <= 32 * groups) {
            if (tiles(32, 16) <= 2 * cus) return Mx4Kernel::kRows32;
        } else if (rows <= 64 * groups) {
            if (tiles(32, 32) <= 2 * cus) return Mx4Kernel::kRows32x2;
        }
    }
    // 256x256 tiles / 64x128 ones: 64 groups of 2048x2048 with 64 rows each 39 / 38, with 96 44 / 50; 32 with 128 25 / 32;
    // 1 group of 4096x4096 with 1024 rows 26 / 24, with 1536 29 / 29, with 2048 31 / 47
    const int64_t smallTiles = (CeilDiv(rows, 64) + (groups - 1) / 2) * CeilDiv(n, 128);
    if (rows >= 96 * groups && smallTiles > 3 * cus) return Mx4Kernel::kTiles;
    // three teams a tile / one: 512 rows x 4096 x 4096 18 / 21, x 2048 12 / 11; 768 rows x 4096 x 4096 29 / 23; 8 groups of
    // 4096x4096 with 4 rows 20 / 22
    return smallTiles <= cus && blocks >= 8 * 12 ? Mx4Kernel::kSmallTilesTeams : Mx4Kernel::kSmallTiles;
}

int LaunchMx4Quantize(const Mx4Rows& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    return ByRows(l, l.type == ACL_FLOAT ? 4 : 2, [&](const Mx4Rows& p, uint32_t grid, uint32_t chunks, uint32_t total) {
        if (l.type == ACL_FLOAT) Mx4QuantizeKernel<float><<<grid, 256, 0, s>>>(p, chunks, total);
        else if (l.type == ACL_FLOAT16) Mx4QuantizeKernel<Half><<<grid, 256, 0, s>>>(p, chunks, total);
        else Mx4QuantizeKernel<Bf16><<<grid, 256, 0, s>>>(p, chunks, total);
    });
}

int LaunchMx4Dequantize(const Mx4Rows& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    return ByRows(l, l.type == ACL_FLOAT ? 4 : 2, [&](const Mx4Rows& p, uint32_t grid, uint32_t chunks, uint32_t total) {
        if (l.type == ACL_FLOAT) Mx4DequantizeKernel<float><<<grid, 256, 0, s>>>(p, chunks, total);
        else if (l.type == ACL_FLOAT16) Mx4DequantizeKernel<Half><<<grid, 256, 0, s>>>(p, chunks, total);
        else Mx4DequantizeKernel<Bf16><<<grid, 256, 0, s>>>(p, chunks, total);
    });
}

int LaunchGroupedMMMx4(const Mx4Launch& l, void* stream)
{
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (l.c_type == ACL_FLOAT) return Mx4BySize<float>(l, s);
    return l.c_type == ACL_FLOAT16 ? Mx4BySize<Half>(l, s) : Mx4BySize<Bf16>(l, s);
}

}  // namespace aclsp
