// What the torch module's files share: the library's entry points, a call on a
// tensor's stream, argument checks, and what refuses a derivative.
#pragma once

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include "cann_ops_sparse.h"

namespace ops_sparse_torch {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxCount = INT32_MAX;

struct Library {
    decltype(&aclsparseCreate) create = nullptr;
    decltype(&aclsparseDestroy) destroy = nullptr;
    decltype(&aclsparseSetStream) setStream = nullptr;
    decltype(&aclsparseRoute_bufferSize) routeBufferSize = nullptr;
    decltype(&aclsparseRoute) route = nullptr;
    decltype(&aclsparseExpertPlan) expertPlan = nullptr;
    decltype(&aclsparseRouteGrad) routeGrad = nullptr;
    decltype(&aclsparseGroupedMM) groupedMM = nullptr;
    decltype(&aclsparseGroupedMMGrad) groupedMMGrad = nullptr;
    decltype(&aclsparseGroupedMMScaled) groupedMMScaled = nullptr;
    decltype(&aclsparseCombine) combine = nullptr;
    decltype(&aclsparseCombineAndList) combineAndList = nullptr;
    decltype(&aclsparseCombineGradAny_bufferSize) combineGradBufferSize = nullptr;
    decltype(&aclsparseCombineGradAny) combineGrad = nullptr;
    decltype(&aclsparseMx4Quantize) mx4Quantize = nullptr;
    decltype(&aclsparseMx4Dequantize) mx4Dequantize = nullptr;
    decltype(&aclsparseGroupedMMMx4) groupedMMMx4 = nullptr;
    decltype(&aclsparseAdamW) adamW = nullptr;
    decltype(&aclsparseAdamWMixed) adamWMixed = nullptr;
    decltype(&aclsparseAdamWMoments) adamWMoments = nullptr;
    decltype(&aclsparseTokenLogprobs_bufferSize) logprobsBufferSize = nullptr;
    decltype(&aclsparseTokenLogprobs) logprobs = nullptr;
    decltype(&aclsparseTokenLogprobsGrad) logprobsGrad = nullptr;
};
inline Library lib;

// A handle on the current stream of a tensor's device, with that device current.
class Call {
public:
    explicit Call(const Tensor& t) : guard_(t.device())
    {
        Ok(lib.create(&h_), "aclsparseCreate");
        void* stream = c10::hip::getCurrentHIPStream(t.get_device()).stream();
        Ok(lib.setStream(h_, stream != nullptr ? stream : ACL_SPARSE_HIP_NULL_STREAM), "aclsparseSetStream");
    }
    ~Call() { lib.destroy(h_); }
    Call(const Call&) = delete;
    Call& operator=(const Call&) = delete;
    operator aclsparseHandle_t() const { return h_; }

    static void Ok(aclsparseStatus_t st, const char* name)
    {
        TORCH_CHECK(st == ACL_SPARSE_STATUS_SUCCESS, name, " failed with status ", static_cast<int>(st));
    }

private:
    c10::DeviceGuard guard_;
    aclsparseHandle_t h_ = nullptr;
};

inline aclDataType TypeOf(at::ScalarType t)
{
    switch (t) {
        case at::kFloat: return ACL_FLOAT;
        case at::kHalf: return ACL_FLOAT16;
        case at::kBFloat16: return ACL_BF16;
        case at::kInt: return ACL_INT32;
        case at::kChar: return ACL_INT8;
        default: return ACL_DT_UNDEFINED;
    }
}

inline bool IsHalf(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
inline bool IsFloat(at::ScalarType t) { return t == at::kFloat || IsHalf(t); }

inline void OnGpu(const Tensor& t)
{
    TORCH_CHECK_VALUE(t.is_cuda(), "these operators need tensors on a ROCm device");
}

inline void SameDevice(const Tensor& first, const Tensor& t, const char* name)
{
    TORCH_CHECK_VALUE(!t.defined() || t.device() == first.device(), name, " must be on ", first.device(), ", got ",
                      t.device());
}

// t with its last dimension contiguous and rows that do not overlap: a copy only where it is not so
inline Tensor Rows(const Tensor& t)
{
    const int64_t d = t.dim(), width = t.size(d - 1);
    if ((width <= 1 || t.stride(d - 1) == 1) && (d < 2 || t.size(d - 2) <= 1 || t.stride(d - 2) >= width)) return t;
    return t.contiguous();
}

inline int64_t Ld(const Tensor& t)
{
    const int64_t d = t.dim(), width = std::max<int64_t>(t.size(d - 1), 1);
    return t.size(d - 2) > 1 ? std::max(t.stride(d - 2), width) : width;
}

inline Tensor Index(const Tensor& t, const char* name)
{
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
    return t.contiguous();
}

inline const int32_t* Ints(const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; }
inline float* Floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
inline void* Data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline Tensor Empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like)
{
    return at::empty(shape, like.options().dtype(type).requires_grad(false));
}

inline bool Tracked(const Tensor& a, const Tensor& b)
{
    return at::GradMode::is_enabled() && ((a.defined() && a.requires_grad()) || (b.defined() && b.requires_grad()));
}

// The kernels read a tensor's value alone: a tangent that it carries would pass for zero.
inline void NoTangent(const Tensor& t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "these operators have no forward-mode derivative");
}

// Results that autograd did not see being made of `inputs`: a derivative through them to any of those raises `message`,
// where a tensor without a node would pass for a constant.  (A node without edges to the inputs would not do: the
// engine skips it where a derivative with respect to given tensors is asked for.)
struct Results {
    variable_list tensors;
};
struct UndifferentiableNode : torch::autograd::Function<UndifferentiableNode> {
    using Input = optional<Tensor>;
    static variable_list forward(AutogradContext* ctx, const Input&, const Input&, const Input&, const Input&,
                                 const Results& results, const std::string& message)
    {
        ctx->saved_data["message"] = message;
        return results.tensors;
    }
    static variable_list backward(AutogradContext* ctx, variable_list)
    {
        TORCH_CHECK(false, ctx->saved_data["message"].toStringRef());
    }
};
inline variable_list Undifferentiable(const std::array<Tensor, 4>& inputs, variable_list results, const char* message)
{
    if (!at::GradMode::is_enabled()) return results;
    auto input = [&](int i) { return inputs[i].defined() ? optional<Tensor>(inputs[i]) : std::nullopt; };
    variable_list defined;
    for (const auto& t : results) {
        if (t.defined()) defined.push_back(t);
    }
    const variable_list made =
        UndifferentiableNode::apply(input(0), input(1), input(2), input(3), Results{defined}, std::string(message));
    size_t next = 0;
    for (auto& t : results) {
        if (t.defined()) t = made[next++];
    }
    return results;
}

// Gradients, of what comes in and of what the forward call kept.
inline variable_list Once(const std::array<Tensor, 4>& inputs, variable_list grads)
{
    return Undifferentiable(inputs, std::move(grads),
                            "these operators are differentiable once; their gradients are not");
}

inline void CheckPlan(const Tensor& a, const Tensor& offsets, const Tensor& tokens, int64_t groups)
{
    TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) >= 2,
                      "offsets must be one-dimensional, one more than the experts");
    SameDevice(a, offsets, "offsets");
    SameDevice(a, tokens, "tokens");
    TORCH_CHECK_VALUE(offsets.size(0) == groups + 1, "the plan has ", offsets.size(0) - 1, " experts, w ", groups);
}

// The rows of a that the plan reads: one per sorted row or, with gather, per token.  More are rows of no expert, or
// tokens that nothing names.
inline void CheckRows(const Tensor& a, const optional<Tensor>& tokens, const optional<Tensor>& places, bool gather)
{
    if (gather) {
        TORCH_CHECK_VALUE(!places.has_value() || places->dim() != 2 || a.size(0) >= places->size(0), "a has ",
                          a.size(0), " rows, the plan ", places->size(0), " tokens");
    } else {
        TORCH_CHECK_VALUE(!tokens.has_value() || a.size(0) >= tokens->numel(), "a has ", a.size(0),
                          " rows, the plan ", tokens->numel(), " (gather takes a in the order of the tokens)");
    }
}

// The operators of a model's training and serving (model_ops_torch.cpp).
void DefineModelOps(pybind11::module_& m);

}  // namespace ops_sparse_torch
