// Entry points of the operators of a model's training and serving: rows in
// microscaled 4 bits and their grouped products, log probabilities of tokens,
// and the AdamW step.  The reference has no counterpart.
//
// Checks in this order, as in the other families: handle, counts and limits,
// types, pointers, leading dimensions.  Every call enqueues kernels on the
// handle's stream and returns; none allocates, copies or waits, so each may be
// captured in a HIP graph.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "aclsparse_internal.h"
#include "experts_internal.h"
#include "model_ops_internal.h"

namespace {

// sides of a product: positions past the end, in the last tile or the last step of a scan, fit int32 too
constexpr int64_t kMaxSide = INT32_MAX - 4096;
// logits of a row: places of the units behind its end, in a thread's last batch, fit int32 too
constexpr int64_t kMaxVocab = int64_t{1} << 30;

void* StreamOf(aclsparseHandle_t h)
{
    return (h->stream == nullptr || h->stream == ACL_SPARSE_HIP_NULL_STREAM) ? nullptr : h->stream;
}

aclsparseStatus_t CheckHandle(aclsparseHandle_t h)
{
    if (h == nullptr) return ACL_SPARSE_STATUS_HANDLE_IS_NULLPTR;
    if (h->signature != aclsp::kHandleSignature) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

bool IsFloat(int32_t t) { return t == ACL_FLOAT || t == ACL_FLOAT16 || t == ACL_BF16; }

aclsparseStatus_t Finish(int rc)
{
    if (rc == aclsp::kTooLarge) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    return rc != 0 || hipGetLastError() != hipSuccess ? ACL_SPARSE_STATUS_EXECUTION_FAILED
                                                      : ACL_SPARSE_STATUS_SUCCESS;
}

int64_t Blocks(int64_t k) { return (k + aclsp::kMx4Block - 1) / aclsp::kMx4Block; }

aclsparseStatus_t CheckMx4Rows(const aclsp::Mx4Rows& l)
{
    if (l.rows < 0 || l.k < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (l.k > kMaxSide) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (!IsFloat(l.type)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (l.rows == 0 || l.k == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (l.x == nullptr || l.codes == nullptr || l.scales == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const int64_t blocks = Blocks(l.k);
    if (l.ldx < l.k || l.ld_codes < blocks * 16 || l.ld_scales < blocks) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

bool Aligned(const void* p, int64_t strideBytes, int64_t to)
{
    return (reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(strideBytes)) % to == 0;
}

// The step's scalars, and bits of the moments
aclsparseStatus_t CheckAdamW(const aclsparseAdamWOptions_t& o)
{
    if (o.momentBits != 8 && o.momentBits != 32) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    const bool fine = o.beta1 >= 0 && o.beta1 < 1 && o.beta2 >= 0 && o.beta2 < 1 && o.eps >= 0 && std::isfinite(o.eps) &&
                      o.weightDecay >= 0 && std::isfinite(o.weightDecay) &&
                      (o.lrDevice != nullptr || (o.lr >= 0 && std::isfinite(o.lr)));
    return fine && o.step != nullptr && o.buffer != nullptr && Aligned(o.buffer, 0, 4) ? ACL_SPARSE_STATUS_SUCCESS : ACL_SPARSE_STATUS_INVALID_VALUE;
}

aclsparseStatus_t CheckAdamWTensor(const aclsparseAdamWTensor_t& t, int bits)
{
    if (t.count < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (t.count == 0 || t.grad == nullptr) return ACL_SPARSE_STATUS_SUCCESS;  // nothing to do
    if (!IsFloat(t.paramType) || !IsFloat(t.gradType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (t.param == nullptr || t.moments == nullptr || (bits == 8) != (t.exponents != nullptr)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return Aligned(t.moments, 0, bits == 8 ? 8 : 4) ? ACL_SPARSE_STATUS_SUCCESS : ACL_SPARSE_STATUS_INVALID_VALUE;
}

// Adds a tensor to a launch's table; false where it is full, or its chunks' numbers would not fit.
bool Add(aclsp::AdamWTable& table, int& used, const aclsp::AdamWTensor& t, int64_t place)
{
    const int64_t chunks = (t.count + aclsp::kAdamWChunk - 1) / aclsp::kAdamWChunk;
    if (used == aclsp::kAdamWTensors || table.chunks + chunks > aclsp::kAdamWMostChunks) return false;
    table.tensor[used] = t;
    table.first[used] = table.chunks;
    table.place[used] = static_cast<int32_t>(place);
    table.chunks += static_cast<uint32_t>(chunks);
    ++used;
    return true;
}

// Places that are not used come behind every chunk.
void Clear(aclsp::AdamWTable& table, int& used)
{
    for (uint32_t& first : table.first) first = UINT32_MAX;
    table.chunks = 0;
    used = 0;
}

aclsparseStatus_t CheckLogprobsShape(int64_t rows, int64_t vocab, int64_t top)
{
    if (rows < 0 || vocab < 1 || top < 0 || top > vocab) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rows > INT32_MAX || vocab > kMaxVocab || top > aclsp::kMaxTop) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    return ACL_SPARSE_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

aclsparseStatus_t aclsparseMx4Quantize(aclsparseHandle_t handle, int64_t rows, int64_t k, const void* X, int64_t ldx,
                                       aclDataType xType, uint8_t* codes, int64_t ldCodes, uint8_t* scales,
                                       int64_t ldScales)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const aclsp::Mx4Rows l{rows, k, const_cast<void*>(X), ldx, xType, codes, ldCodes, scales, ldScales};
    st = CheckMx4Rows(l);
    if (st != ACL_SPARSE_STATUS_SUCCESS || rows == 0 || k == 0) return st;
    (void)hipGetLastError();
    return Finish(aclsp::LaunchMx4Quantize(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseMx4Dequantize(aclsparseHandle_t handle, int64_t rows, int64_t k, const uint8_t* codes,
                                         int64_t ldCodes, const uint8_t* scales, int64_t ldScales, void* X, int64_t ldx,
                                         aclDataType xType)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    const aclsp::Mx4Rows l{rows, k, X, ldx, xType, const_cast<uint8_t*>(codes), ldCodes, const_cast<uint8_t*>(scales),
                           ldScales};
    st = CheckMx4Rows(l);
    if (st != ACL_SPARSE_STATUS_SUCCESS || rows == 0 || k == 0) return st;
    (void)hipGetLastError();
    return Finish(aclsp::LaunchMx4Dequantize(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseGroupedMMMx4(aclsparseHandle_t handle, int64_t groups, int64_t rows, int64_t n, int64_t k,
                                        const int32_t* offsets, const int32_t* rowIndex, int64_t rowsA,
                                        const uint8_t* A, int64_t lda, const uint8_t* scaleA, int64_t ldScaleA,
                                        const uint8_t* B, int64_t ldb, int64_t strideB, const uint8_t* scaleB,
                                        int64_t ldScaleB, int64_t strideScaleB, void* C, int64_t ldc, aclDataType cType)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (groups < 1 || rows < 0 || n < 0 || k < 0 || rowsA < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (groups > kMaxSide || rows > kMaxSide || n > kMaxSide || k > kMaxSide || rowsA > INT32_MAX) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (offsets == nullptr && groups != 1) return ACL_SPARSE_STATUS_INVALID_VALUE;
    // without an index, row r of the one is row r of the other
    if (rowIndex == nullptr ? rowsA < rows : (rows > 0 && rowsA == 0)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (!IsFloat(cType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    const int64_t blocks = Blocks(k);
    if (lda < blocks * 16 || ldb < blocks * 16 || ldScaleA < blocks || ldScaleB < blocks || ldc < n || strideB < 0 ||
        strideScaleB < 0) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (rows == 0 || n == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (C == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (k > 0) {
        if (A == nullptr || B == nullptr || scaleA == nullptr || scaleB == nullptr) {
            return ACL_SPARSE_STATUS_INVALID_VALUE;
        }
        if (!Aligned(A, lda, 16) || !Aligned(B, ldb | strideB, 16)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    const aclsp::Mx4Launch l{groups, rows, n, blocks, offsets, rowIndex, rowsA, {A, lda, 0, scaleA, ldScaleA, 0},
                             {B, ldb, strideB, scaleB, ldScaleB, strideScaleB}, C, ldc, cType};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchGroupedMMMx4(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseAdamW(aclsparseHandle_t handle, int64_t count, const aclsparseAdamWTensor_t* tensors,
                                 const aclsparseAdamWOptions_t* options)
{
    constexpr aclsp::AdamWMix own{};
    return aclsparseAdamWMixed(handle, count, tensors, options, own.first, own.second);
}

aclsparseStatus_t aclsparseAdamWMixed(aclsparseHandle_t handle, int64_t count, const aclsparseAdamWTensor_t* tensors,
                                      const aclsparseAdamWOptions_t* options, uint32_t factor1, uint32_t factor2)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (count < 0 || options == nullptr || (count > 0 && tensors == nullptr)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (count > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    st = factor1 % 2 != 0 && factor2 % 2 != 0 ? CheckAdamW(*options) : ACL_SPARSE_STATUS_INVALID_VALUE;
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    for (int64_t i = 0; i < count; ++i) {
        if (tensors[i].count > aclsp::kAdamWMostChunks * aclsp::kAdamWChunk) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
        st = CheckAdamWTensor(tensors[i], options->momentBits);
        if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    }
    const aclsp::AdamWScalars s{options->lr, options->beta1, options->beta2, options->eps, options->weightDecay,
                          options->lrDevice, options->gradScale, options->step, options->seed,
                                {factor1, factor2}};
    (void)hipGetLastError();
    void* stream = StreamOf(handle);
    int rc = aclsp::LaunchAdamWFactors(s, options->buffer, stream);
    // one launch for each 64 tensors of one kind
    constexpr aclDataType kTypes[] = {ACL_FLOAT, ACL_FLOAT16, ACL_BF16};
    aclsp::AdamWTable table{};
    int used = 0;
    aclDataType param = ACL_FLOAT, grad = ACL_FLOAT;
    bool master = false;
    auto flush = [&] {
        if (used == 0) return;
        if (rc == 0) rc = aclsp::LaunchAdamW(table, options->buffer, param, grad, options->momentBits, master, stream);
        Clear(table, used);
    };
    Clear(table, used);
    for (int kind = 0; kind < 18; ++kind) {
        param = kTypes[kind / 6];
        grad = kTypes[kind / 2 % 3];
        master = kind % 2 != 0;
        for (int64_t i = 0; i < count; ++i) {
            const aclsparseAdamWTensor_t& t = tensors[i];
            if (t.count == 0 || t.grad == nullptr || t.paramType != param || t.gradType != grad ||
                (t.master != nullptr) != master) {
                continue;
            }
            const aclsp::AdamWTensor one{t.param, t.grad, t.master, t.moments, t.exponents, t.count};
            if (Add(table, used, one, i)) continue;
            flush();
            Add(table, used, one, i);
        }
        flush();
    }
    return Finish(rc);
}

aclsparseStatus_t aclsparseAdamWMoments(aclsparseHandle_t handle, int64_t count, const aclsparseAdamWTensor_t* tensors)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (count < 0 || (count > 0 && tensors == nullptr)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (count > INT32_MAX) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    for (int64_t i = 0; i < count; ++i) {
        const aclsparseAdamWTensor_t& t = tensors[i];
        if (t.count < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
        if (t.count > aclsp::kAdamWMostChunks * aclsp::kAdamWChunk) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
        if (t.count > 0 && (t.master == nullptr || t.moments == nullptr || t.exponents == nullptr ||
                            !Aligned(t.moments, 0, 8))) {
            return ACL_SPARSE_STATUS_INVALID_VALUE;
        }
    }
    (void)hipGetLastError();
    aclsp::AdamWTable table{};
    int used = 0;
    Clear(table, used);
    for (int64_t i = 0; i < count; ++i) {
        const aclsparseAdamWTensor_t& t = tensors[i];
        if (t.count == 0) continue;
        const aclsp::AdamWTensor one{nullptr, nullptr, t.master, t.moments, t.exponents, t.count};
        if (Add(table, used, one, i)) continue;
        if (aclsp::LaunchAdamWMoments(table, StreamOf(handle)) != 0) return ACL_SPARSE_STATUS_EXECUTION_FAILED;
        Clear(table, used);
        Add(table, used, one, i);
    }
    return used == 0 ? ACL_SPARSE_STATUS_SUCCESS : Finish(aclsp::LaunchAdamWMoments(table, StreamOf(handle)));
}

aclsparseStatus_t aclsparseTokenLogprobs_bufferSize(aclsparseHandle_t handle, int64_t rows, int64_t vocab, int64_t top,
                                                    size_t* bufferSize)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckLogprobsShape(rows, vocab, top);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const size_t bytes = aclsp::LogprobsBytes(rows, vocab, top);
    *bufferSize = aclsp::AlignUp(bytes < aclsp::kWsAlign ? aclsp::kWsAlign : bytes);
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t aclsparseTokenLogprobs(aclsparseHandle_t handle, int64_t rows, int64_t vocab, const void* logits,
                                         int64_t ldLogits, aclDataType logitsType, const void* targets,
                                         aclDataType targetsType, float* logprobs, float* entropy, float* stats,
                                         int64_t top, float* topLogprobs, int32_t* topIds, void* buffer)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckLogprobsShape(rows, vocab, top);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (!IsFloat(logitsType) || (targetsType != ACL_INT32 && targetsType != ACL_INT64)) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (ldLogits < vocab) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rows == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (logits == nullptr || buffer == nullptr || (targets == nullptr) != (logprobs == nullptr) ||
        (top > 0 && (topLogprobs == nullptr || topIds == nullptr))) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    const aclsp::LogprobsLaunch l{rows, vocab, top, logits, ldLogits, logitsType, targets, targetsType == ACL_INT64,
                                  logprobs, entropy, stats, topLogprobs, topIds, buffer};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchLogprobs(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseTokenLogprobsGrad(aclsparseHandle_t handle, int64_t rows, int64_t vocab, const void* logits,
                                             int64_t ldLogits, aclDataType logitsType, const void* targets,
                                             aclDataType targetsType, const float* stats, const float* entropy,
                                             int64_t top, const int32_t* topIds, const float* gradLogprobs,
                                             const float* gradEntropy, const float* gradTop, void* gradLogits,
                                             int64_t ldGrad)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckLogprobsShape(rows, vocab, top);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (!IsFloat(logitsType) || (targetsType != ACL_INT32 && targetsType != ACL_INT64)) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (ldLogits < vocab || ldGrad < vocab) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rows == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (logits == nullptr || stats == nullptr || gradLogits == nullptr || (gradLogprobs != nullptr && targets == nullptr) ||
        (gradEntropy != nullptr && entropy == nullptr) || (gradTop != nullptr && (topIds == nullptr || top == 0))) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    // in the logits' place only row by row: other rows would be written over before they are read
    if (gradLogits == logits && rows > 1 && ldGrad != ldLogits) return ACL_SPARSE_STATUS_INVALID_VALUE;
    const aclsp::LogprobsGradLaunch l{rows, vocab, top, logits, ldLogits, logitsType, targets,
                                      targetsType == ACL_INT64, stats, entropy, topIds, gradLogprobs, gradEntropy,
                                      gradTop, gradLogits, ldGrad};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchLogprobsGrad(l, StreamOf(handle)));
}

}  // extern "C"
