// Launcher interface between the host checks of the operators of a model's
// training and serving (model_ops_host.cpp) and their gfx950 kernels: products
// in microscaled 4 bits, log probabilities, and the optimiser's step.  Nothing
// here is public.
#pragma once

#include <cstddef>
#include <cstdint>

#include "cann_ops_sparse.h"

namespace aclsp {

// ---- microscaled 4 bits: blocks of 32 values of 4 bits (16 bytes) and one scale byte each
constexpr int64_t kMx4Block = 32;

struct Mx4Rows {
    int64_t rows, k;    // k values a row, ceil(k / 32) blocks
    void* x;            // read by quantisation, written by its inverse
    int64_t ldx;        // elements
    aclDataType type;
    uint8_t* codes;
    int64_t ld_codes;   // bytes, as of scales
    uint8_t* scales;
    int64_t ld_scales;
};
int LaunchMx4Quantize(const Mx4Rows& l, void* stream);
int LaunchMx4Dequantize(const Mx4Rows& l, void* stream);

struct Mx4Operand {
    const uint8_t* codes;   // rows aligned to 16 bytes
    int64_t ld, stride;     // bytes from row to row, and from group to group
    const uint8_t* scales;  // any alignment
    int64_t ld_scales, stride_scales;
};
struct Mx4Launch {
    int64_t groups, rows, n, blocks;
    const int32_t* offsets;    // null: one group of all rows
    const int32_t* row_index;  // null: row r of C is row r of A
    int64_t rows_a;
    Mx4Operand a, b;
    void* c;
    int64_t ldc;
    aclDataType c_type;
};
int LaunchGroupedMMMx4(const Mx4Launch& l, void* stream);
// The kernel that multiplies operands of these sizes on a chip of so many CUs: few rows of each group, 16 or 32 at a time
// (and 16 columns, or 32), tiles of 256x256, or of 64x128 with one team of waves or three.
enum class Mx4Kernel : int { kRows16, kRows32, kRows32x2, kTiles, kSmallTiles, kSmallTilesTeams };
Mx4Kernel Mx4KernelOf(int64_t groups, int64_t rows, int64_t n, int64_t blocks, int64_t cus);

// ---- AdamW
// The tensors of one launch, passed by value: a kernel's arguments hold so many.
constexpr int kAdamWTensors = 64;

struct AdamWTensor {
    void* param;
    const void* grad;
    float* master;       // null: the parameter itself is the value that is kept
    void* moments;       // [2, count rounded up to 32] of fp32 or of 8-bit codes
    uint8_t* exponents;  // [2, blocks] of 8-bit codes, null for fp32
    int64_t count;
};
struct AdamWTable {
    AdamWTensor tensor[kAdamWTensors];
    uint32_t first[kAdamWTensors];  // chunk that each begins with; those past the last: UINT32_MAX
    int32_t place[kAdamWTensors];   // in the caller's list
    uint32_t chunks;                // of all
};
// Odd factors of the hash that 8-bit moments' random numbers come from.  The library's own are the first bits of the roots
// of 13 and 19 behind the point (made odd): numbers whose bits, and whose two halves, are independent.
struct AdamWMix {
    uint32_t first = 0x9B05688DU, second = 0x5BE0CD19U;
};
struct AdamWScalars {
    double lr, beta1, beta2, eps, weight_decay;
    const float* lr_device;   // null: lr
    const float* grad_scale;  // null: one
    int32_t* step;            // steps taken; this one is counted
    uint32_t seed;
    AdamWMix mix;
};
// Values of a workgroup; a launch has one for each chunk, and fewer than 2^32 threads.
constexpr int64_t kAdamWChunk = 2048, kAdamWMostChunks = (int64_t{1} << 24) - 1;
constexpr size_t kAdamWBufferBytes = 64;
int LaunchAdamWFactors(const AdamWScalars& s, void* buffer, void* stream);
// With the factors that LaunchAdamWFactors left in the buffer.
int LaunchAdamW(const AdamWTable& t, const void* buffer, aclDataType param, aclDataType grad, int bits, bool master,
                void* stream);
// Values of 8-bit moments, to the tables' masters, [2, count].
int LaunchAdamWMoments(const AdamWTable& t, void* stream);

// ---- log probabilities
constexpr int64_t kMaxTop = 64;

struct LogprobsLaunch {
    int64_t rows, vocab, top;
    const void* logits;
    int64_t ld;
    aclDataType type;
    const void* targets;  // int32 or int64; null: none asked for
    bool wide;            // targets are int64
    float* logprobs;      // null with targets
    float* entropy;       // null: not wanted
    float* stats;         // [rows, 2] for the gradient; null: not wanted
    float* top_logprobs;  // [rows, top]
    int32_t* top_ids;
    void* buffer;
};
size_t LogprobsBytes(int64_t rows, int64_t vocab, int64_t top);
int LaunchLogprobs(const LogprobsLaunch& l, void* stream);

struct LogprobsGradLaunch {
    int64_t rows, vocab, top;
    const void* logits;
    int64_t ld;
    aclDataType type;
    const void* targets;
    bool wide;
    const float* stats;
    const float* entropy;        // needed with grad_entropy
    const int32_t* top_ids;      // needed with grad_top
    const float* grad_logprobs;  // null: zero, as the others
    const float* grad_entropy;
    const float* grad_top;
    void* grad;
    int64_t ld_grad;
};
int LaunchLogprobsGrad(const LogprobsGradLaunch& l, void* stream);

}  // namespace aclsp
