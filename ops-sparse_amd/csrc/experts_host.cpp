// Entry points of the experts' operators: routing, ragged products grouped by
// expert with their gradients, 8-bit products with scales, and the weighted
// combination.  The reference has no counterpart.
//
// Checks in this order, as in the other families: handle, counts and limits,
// types, pointers, leading dimensions.  Every call enqueues kernels on the
// handle's stream and returns; none allocates, copies or waits, so each may be
// captured in a HIP graph.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "aclsparse_internal.h"
#include "experts_internal.h"

namespace {

constexpr int64_t kMaxCount = INT32_MAX;  // counts that index arrays of int32
// sides and groups of a product: positions past the end, in the last tile or the last step of a scan, fit int32 too
constexpr int64_t kMaxSide = INT32_MAX - 4096;

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

bool Is16Bit(aclDataType t) { return t == ACL_FLOAT16 || t == ACL_BF16; }

// tokens * k assignments, each of which an int32 numbers
aclsparseStatus_t CheckRouteShape(int64_t tokens, int64_t experts, int64_t k)
{
    if (tokens < 0 || experts < 1 || k < 1 || k > experts) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (experts > aclsp::kMaxRouteExperts || k > aclsp::kMaxRouteK || tokens > kMaxCount / k) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

size_t RouteBytes(int64_t tokens, int64_t experts)
{
    const size_t bytes = static_cast<size_t>(aclsp::RouteBlocks(tokens) * experts) * sizeof(int32_t);
    return aclsp::AlignUp(bytes < aclsp::kWsAlign ? aclsp::kWsAlign : bytes);
}

aclsparseStatus_t Finish(int rc)
{
    if (rc == aclsp::kTooLarge) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    return rc != 0 || hipGetLastError() != hipSuccess ? ACL_SPARSE_STATUS_EXECUTION_FAILED
                                                      : ACL_SPARSE_STATUS_SUCCESS;
}

// groups, rows, n and k of a grouped product
aclsparseStatus_t CheckGroupedShape(int64_t groups, int64_t rows, int64_t n, int64_t k, const int32_t* offsets,
                                    const int32_t* rowIndex, int64_t rowsA)
{
    if (groups < 1 || rows < 0 || n < 0 || k < 0 || rowsA < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (groups > kMaxSide || rows > kMaxSide || n > kMaxSide || k > kMaxSide || rowsA > kMaxCount) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (offsets == nullptr && groups != 1) return ACL_SPARSE_STATUS_INVALID_VALUE;
    // without an index, row r of the one is row r of the other
    if (rowIndex == nullptr ? rowsA < rows : (rows > 0 && rowsA == 0)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t CheckCombineShape(int64_t tokens, int64_t k, int64_t width, int64_t rows)
{
    if (tokens < 0 || k < 1 || width < 0 || rows < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (k > aclsp::kMaxRouteK || tokens > kMaxCount / k || rows > kMaxCount || width > kMaxCount) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

// What both gradients of a combination check, but the offsets and the buffer
aclsparseStatus_t CheckCombineGrad(const aclsp::CombineGradLaunch& l)
{
    const aclsparseStatus_t st = CheckCombineShape(l.tokens, l.k, l.width, l.rows);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (!Is16Bit(l.type)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (l.ldo < l.width || (l.grad_y != nullptr && l.ld_grad_y < l.width) ||
        (l.grad_weights != nullptr && l.ldy < l.width)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (l.tokens > 0 && (l.places == nullptr || (l.width > 0 && l.grad_out == nullptr))) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (l.grad_weights != nullptr && l.y == nullptr && l.rows > 0 && l.width > 0) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    return ACL_SPARSE_STATUS_SUCCESS;
}

// One int32 per row or assignment
size_t HeadBytes(int64_t count)
{
    const size_t bytes = static_cast<size_t>(count) * sizeof(int32_t);
    return aclsp::AlignUp(bytes < aclsp::kWsAlign ? aclsp::kWsAlign : bytes);
}

int32_t* NextOf(int32_t* head, int64_t rows) { return head + HeadBytes(rows) / sizeof(int32_t); }

aclsparseStatus_t Combine(aclsparseHandle_t handle, aclsp::CombineLaunch l, bool lists)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckCombineShape(l.tokens, l.k, l.width, l.rows);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    // rows of 32 bits (a gradient's partial sums) may be rounded to 16 here
    if (!Is16Bit(l.out_type) || (l.y_type != l.out_type && l.y_type != ACL_FLOAT)) {
        return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    }
    if (l.ldy < l.width || l.ldo < l.width) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (l.tokens == 0 || l.width == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (l.places == nullptr || l.out == nullptr || (l.rows > 0 && l.y == nullptr) || (lists && l.head == nullptr)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (lists) l.next = NextOf(l.head, l.rows);
    (void)hipGetLastError();
    return Finish(aclsp::LaunchCombine(l, StreamOf(handle)));
}

}  // namespace

extern "C" {

aclsparseStatus_t aclsparseRoute_bufferSize(aclsparseHandle_t handle, int64_t tokens, int64_t experts, int64_t k,
                                            size_t* bufferSize)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckRouteShape(tokens, experts, k);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    *bufferSize = RouteBytes(tokens, experts);
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t aclsparseRoute(aclsparseHandle_t handle, int64_t tokens, int64_t experts, int64_t k,
                                 const void* logits, int64_t ldLogits, aclDataType logitsType, int32_t normalize,
                                 float* weights, int32_t* ids, int32_t* offsets, int32_t* rowTokens, int32_t* places,
                                 void* buffer)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckRouteShape(tokens, experts, k);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (logitsType != ACL_FLOAT && !Is16Bit(logitsType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (offsets == nullptr || buffer == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (tokens > 0 && (logits == nullptr || weights == nullptr || ids == nullptr || rowTokens == nullptr ||
                       places == nullptr)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (ldLogits < experts) return ACL_SPARSE_STATUS_INVALID_VALUE;
    aclsp::RouteLaunch l{tokens, experts, k, logits, ldLogits, logitsType, normalize != 0 ? 1 : 0, weights, ids,
                         offsets, rowTokens, places, static_cast<int32_t*>(buffer)};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchRoute(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseExpertPlan(aclsparseHandle_t handle, int64_t tokens, int64_t experts, int64_t k,
                                      const int32_t* ids, int32_t* offsets, int32_t* rowTokens, int32_t* places,
                                      void* buffer)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckRouteShape(tokens, experts, k);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (offsets == nullptr || buffer == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (tokens > 0 && (ids == nullptr || rowTokens == nullptr || places == nullptr)) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    aclsp::RouteLaunch l{tokens, experts, k, nullptr, 0, ACL_FLOAT, 0, nullptr, const_cast<int32_t*>(ids),
                         offsets, rowTokens, places, static_cast<int32_t*>(buffer)};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchRoute(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseRouteGrad(aclsparseHandle_t handle, int64_t tokens, int64_t experts, int64_t k,
                                     const void* logits, int64_t ldLogits, aclDataType logitsType, int32_t normalize,
                                     const float* weights, const int32_t* ids, const float* gradWeights,
                                     void* gradLogits, int64_t ldGrad)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckRouteShape(tokens, experts, k);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (logitsType != ACL_FLOAT && !Is16Bit(logitsType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (tokens > 0 && (weights == nullptr || ids == nullptr || gradWeights == nullptr || gradLogits == nullptr ||
                       (normalize == 0 && logits == nullptr))) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (ldGrad < experts || (normalize == 0 && ldLogits < experts)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (tokens == 0) return ACL_SPARSE_STATUS_SUCCESS;
    aclsp::RouteGradLaunch l{tokens, experts, k, logits, ldLogits, logitsType, normalize != 0 ? 1 : 0, weights, ids,
                             gradWeights, gradLogits, ldGrad};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchRouteGrad(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseGroupedMM(aclsparseHandle_t handle, aclsparseOperation_t opB, int64_t groups, int64_t rows,
                                     int64_t n, int64_t k, const int32_t* offsets, const int32_t* rowIndex,
                                     int64_t rowsA, const void* A, int64_t lda, const void* B, int64_t ldb,
                                     int64_t strideB, aclDataType abType, void* C, int64_t ldc, aclDataType cType)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (opB != ACL_SPARSE_OP_NON_TRANSPOSE && opB != ACL_SPARSE_OP_TRANSPOSE) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    st = CheckGroupedShape(groups, rows, n, k, offsets, rowIndex, rowsA);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (!Is16Bit(abType) || (cType != abType && cType != ACL_FLOAT)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    const bool trans = opB == ACL_SPARSE_OP_TRANSPOSE;
    if (lda < k || ldc < n || ldb < (trans ? k : n) || strideB < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rows == 0 || n == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (C == nullptr || (k > 0 && (A == nullptr || B == nullptr))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    aclsp::GroupedLaunch l{groups, rows, n, k, offsets, rowIndex, rowsA, A, lda, B, ldb, strideB, trans ? 1 : 0,
                           abType, nullptr, nullptr, C, ldc, cType};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchGroupedMM(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseGroupedMMScaled(aclsparseHandle_t handle, int64_t groups, int64_t rows, int64_t n,
                                           int64_t k, const int32_t* offsets, const int32_t* rowIndex, int64_t rowsA,
                                           const int8_t* A, int64_t lda, const float* scaleA, const int8_t* B,
                                           int64_t ldb, int64_t strideB, const float* scaleB, void* C, int64_t ldc,
                                           aclDataType cType)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckGroupedShape(groups, rows, n, k, offsets, rowIndex, rowsA);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (k > aclsp::kMaxScaledK) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (cType != ACL_FLOAT && !Is16Bit(cType)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (lda < k || ldc < n || ldb < k || strideB < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (rows == 0 || n == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (C == nullptr || scaleA == nullptr || scaleB == nullptr || (k > 0 && (A == nullptr || B == nullptr))) {
        return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    aclsp::GroupedLaunch l{groups, rows, n, k, offsets, rowIndex, rowsA, A, lda, B, ldb, strideB, 1,
                           ACL_INT8, scaleA, scaleB, C, ldc, cType};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchGroupedMM(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseGroupedMMGrad(aclsparseHandle_t handle, int64_t groups, int64_t rows, int64_t n, int64_t k,
                                         const int32_t* offsets, const int32_t* rowIndex, int64_t rowsX,
                                         const void* gradC, int64_t ldg, const void* X, int64_t ldx, aclDataType type,
                                         void* W, int64_t ldw, int64_t strideW, aclDataType wType)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckGroupedShape(groups, rows, n, k, offsets, rowIndex, rowsX);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (!Is16Bit(type) || (wType != type && wType != ACL_FLOAT)) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    if (ldg < n || ldx < k || ldw < k || strideW < 0) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (n == 0 || k == 0) return ACL_SPARSE_STATUS_SUCCESS;
    if (groups > 1) {
        // matrices of W that overlap would race: one after another, or their rows in turn
        const __int128 apart = static_cast<__int128>(n - 1) * ldw + k;
        const __int128 inTurn = static_cast<__int128>(groups - 1) * strideW + k;
        if (strideW < apart && (strideW < k || ldw < inTurn)) return ACL_SPARSE_STATUS_INVALID_VALUE;
    }
    if (W == nullptr || (rows > 0 && (gradC == nullptr || X == nullptr))) return ACL_SPARSE_STATUS_INVALID_VALUE;
    aclsp::GroupedGradLaunch l{groups, rows, n, k, offsets, rowIndex, rowsX, gradC, ldg, X, ldx, type,
                               W, ldw, strideW, wType};
    (void)hipGetLastError();
    return Finish(aclsp::LaunchGroupedMMGrad(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseCombine(aclsparseHandle_t handle, int64_t tokens, int64_t k, int64_t width, int64_t rows,
                                   const int32_t* places, const float* weights, const void* Y, int64_t ldy,
                                   aclDataType yType, void* out, int64_t ldOut, aclDataType outType)
{
    return Combine(handle,
                   {tokens, k, width, rows, places, weights, Y, ldy, yType, out, ldOut, outType, nullptr, nullptr},
                   /*lists=*/false);
}

aclsparseStatus_t aclsparseCombineAndList(aclsparseHandle_t handle, int64_t tokens, int64_t k, int64_t width,
                                          int64_t rows, const int32_t* places, const float* weights, const void* Y,
                                          int64_t ldy, aclDataType yType, void* out, int64_t ldOut,
                                          aclDataType outType, void* buffer)
{
    auto* head = static_cast<int32_t*>(buffer);
    return Combine(handle, {tokens, k, width, rows, places, weights, Y, ldy, yType, out, ldOut, outType, head, nullptr},
                   /*lists=*/true);
}

aclsparseStatus_t aclsparseCombineGrad(aclsparseHandle_t handle, int64_t tokens, int64_t k, int64_t width,
                                       int64_t rows, int64_t groups, const int32_t* offsets, const int32_t* places,
                                       const float* weights, const void* Y, int64_t ldy, const void* gradOut,
                                       int64_t ldOut, aclDataType type, void* gradY, int64_t ldGradY,
                                       float* gradWeights)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (groups < 1) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (groups > kMaxCount) return ACL_SPARSE_STATUS_NOT_SUPPORTED;
    const aclsp::CombineGradLaunch l{tokens, k, width, rows, groups, offsets, places, weights, Y, ldy, gradOut, ldOut,
                                     type, gradY, ldGradY, gradWeights, nullptr, nullptr, false};
    st = CheckCombineGrad(l);
    if (st != ACL_SPARSE_STATUS_SUCCESS || (tokens == 0 && rows == 0)) return st;
    if (offsets == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    if (gradY == nullptr && gradWeights == nullptr) return ACL_SPARSE_STATUS_SUCCESS;
    (void)hipGetLastError();
    return Finish(aclsp::LaunchCombineGrad(l, StreamOf(handle)));
}

aclsparseStatus_t aclsparseCombineGradAny_bufferSize(aclsparseHandle_t handle, int64_t tokens, int64_t k,
                                                     int64_t rows, size_t* bufferSize)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    st = CheckCombineShape(tokens, k, 0, rows);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    if (bufferSize == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
    *bufferSize = HeadBytes(rows) + HeadBytes(tokens * k);
    return ACL_SPARSE_STATUS_SUCCESS;
}

aclsparseStatus_t aclsparseCombineGradAny(aclsparseHandle_t handle, int64_t tokens, int64_t k, int64_t width,
                                          int64_t rows, const int32_t* places, const float* weights, const void* Y,
                                          int64_t ldy, const void* gradOut, int64_t ldOut, aclDataType type,
                                          void* gradY, int64_t ldGradY, float* gradWeights, void* buffer,
                                          int32_t listed)
{
    aclsparseStatus_t st = CheckHandle(handle);
    if (st != ACL_SPARSE_STATUS_SUCCESS) return st;
    auto* head = static_cast<int32_t*>(buffer);
    aclsp::CombineGradLaunch l{tokens, k, width, rows, 0, nullptr, places, weights, Y, ldy, gradOut, ldOut,
                               type, gradY, ldGradY, gradWeights, head, nullptr, listed != 0};
    st = CheckCombineGrad(l);
    if (st != ACL_SPARSE_STATUS_SUCCESS || (tokens == 0 && rows == 0)) return st;
    if (gradY == nullptr && gradWeights == nullptr) return ACL_SPARSE_STATUS_SUCCESS;
    if (gradY != nullptr) {
        if (buffer == nullptr) return ACL_SPARSE_STATUS_INVALID_VALUE;
        l.next = NextOf(head, rows);
    }
    (void)hipGetLastError();
    return Finish(aclsp::LaunchCombineGrad(l, StreamOf(handle)));
}

}  // extern "C"
