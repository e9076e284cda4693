// The experts' operators on torch tensors: argument checks, outputs, and the
// nodes that autograd walks back through.  A Python module of its own
// (lib/_ops_sparse_experts.so, built next to libaclsparse_hip.so), because a
// training step of a small layer spends its time between the kernels: the same
// nodes written in Python cost 50 to 80 us of a step.
//
// It calls the C entry points of include/cann_ops_sparse.h, which `bind` looks
// up in the library that the package has loaded; a handle lives as long as a
// call, since it holds nothing but the stream.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include "cann_ops_sparse.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxExperts = 1024, kMaxK = 64, kMaxScaledK = 131071, kMaxCount = INT32_MAX;

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
} lib;

void Bind(const std::string& path)
{
    void* so = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(so != nullptr, "cannot load ", path);
    auto look = [&](auto& fn, const char* name) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(so, name));
        TORCH_CHECK(fn != nullptr, path, " has no ", name);
    };
    look(lib.create, "aclsparseCreate");
    look(lib.destroy, "aclsparseDestroy");
    look(lib.setStream, "aclsparseSetStream");
    look(lib.routeBufferSize, "aclsparseRoute_bufferSize");
    look(lib.route, "aclsparseRoute");
    look(lib.expertPlan, "aclsparseExpertPlan");
    look(lib.routeGrad, "aclsparseRouteGrad");
    look(lib.groupedMM, "aclsparseGroupedMM");
    look(lib.groupedMMGrad, "aclsparseGroupedMMGrad");
    look(lib.groupedMMScaled, "aclsparseGroupedMMScaled");
    look(lib.combine, "aclsparseCombine");
    look(lib.combineAndList, "aclsparseCombineAndList");
    look(lib.combineGradBufferSize, "aclsparseCombineGradAny_bufferSize");
    look(lib.combineGrad, "aclsparseCombineGradAny");
}

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

aclDataType TypeOf(at::ScalarType t)
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

bool IsHalf(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
bool IsFloat(at::ScalarType t) { return t == at::kFloat || IsHalf(t); }

void OnGpu(const Tensor& t)
{
    TORCH_CHECK_VALUE(t.is_cuda(), "the experts' operators need tensors on a ROCm device");
}

void SameDevice(const Tensor& first, const Tensor& t, const char* name)
{
    TORCH_CHECK_VALUE(!t.defined() || t.device() == first.device(), name, " must be on ", first.device(), ", got ",
                      t.device());
}

// t with its last dimension contiguous and rows that do not overlap: a copy only where it is not so
Tensor Rows(const Tensor& t)
{
    const int64_t d = t.dim(), width = t.size(d - 1);
    if ((width <= 1 || t.stride(d - 1) == 1) && (d < 2 || t.size(d - 2) <= 1 || t.stride(d - 2) >= width)) return t;
    return t.contiguous();
}

int64_t Ld(const Tensor& t)
{
    const int64_t d = t.dim(), width = std::max<int64_t>(t.size(d - 1), 1);
    return t.size(d - 2) > 1 ? std::max(t.stride(d - 2), width) : width;
}

Tensor Index(const Tensor& t, const char* name)
{
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
    return t.contiguous();
}

const int32_t* Ints(const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; }
float* Floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
void* Data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor Empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like)
{
    return at::empty(shape, like.options().dtype(type).requires_grad(false));
}

bool Tracked(const Tensor& a, const Tensor& b)
{
    return at::GradMode::is_enabled() && ((a.defined() && a.requires_grad()) || (b.defined() && b.requires_grad()));
}

// The kernels read a tensor's value alone: a tangent that it carries would pass for zero.
void NoTangent(const Tensor& t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "the experts' operators have no forward-mode derivative");
}

// Results that autograd did not see being made of `inputs`: a derivative through them to any of those raises `message`,
// where a tensor without a node would pass for a constant.  (A node without edges to the inputs would not do: the
// engine skips it where a derivative with respect to given tensors is asked for.)
struct Results {
    variable_list tensors;
};
struct UndifferentiableNode : torch::autograd::Function<UndifferentiableNode> {
    using Input = optional<Tensor>;
    static variable_list forward(AutogradContext* ctx, const Input&, const Input&, const Input&, const Results& results,
                                 const std::string& message)
    {
        ctx->saved_data["message"] = message;
        return results.tensors;
    }
    static variable_list backward(AutogradContext* ctx, variable_list)
    {
        TORCH_CHECK(false, ctx->saved_data["message"].toStringRef());
    }
};
variable_list Undifferentiable(const std::array<Tensor, 3>& inputs, variable_list results, const char* message)
{
    if (!at::GradMode::is_enabled()) return results;
    auto input = [&](int i) { return inputs[i].defined() ? optional<Tensor>(inputs[i]) : std::nullopt; };
    variable_list defined;
    for (const auto& t : results) {
        if (t.defined()) defined.push_back(t);
    }
    const variable_list made =
        UndifferentiableNode::apply(input(0), input(1), input(2), Results{defined}, std::string(message));
    size_t next = 0;
    for (auto& t : results) {
        if (t.defined()) t = made[next++];
    }
    return results;
}

// Gradients, of what comes in and of what the forward call kept.
variable_list Once(const std::array<Tensor, 3>& inputs, variable_list grads)
{
    return Undifferentiable(inputs, std::move(grads),
                            "the experts' operators are differentiable once; their gradients are not");
}

// ------------------------------------------------------------------ routing

void CheckRoute(int64_t tokens, int64_t experts, int64_t k)
{
    TORCH_CHECK_VALUE(k >= 1 && k <= experts, "k must lie in [1, ", experts, "], got ", k);
    TORCH_CHECK_VALUE(experts <= kMaxExperts && k <= kMaxK, "at most ", kMaxExperts, " experts and k <= ", kMaxK,
                      ", got ", experts, " and ", k);
    TORCH_CHECK_VALUE(tokens <= kMaxCount / k, "tokens * k must fit int32");
}

struct Plan {
    Tensor offsets, tokens, places, buffer;
    Plan(const Call& call, int64_t t, int64_t experts, int64_t k, const Tensor& like)
        : offsets(Empty({experts + 1}, at::kInt, like)),
          tokens(Empty({t * k}, at::kInt, like)),
          places(Empty({t, k}, at::kInt, like))
    {
        size_t bytes = 0;
        Call::Ok(lib.routeBufferSize(call, t, experts, k, &bytes), "aclsparseRoute_bufferSize");
        buffer = Empty({static_cast<int64_t>(bytes)}, at::kByte, like);
    }
};

variable_list RunRoute(const Tensor& logits, int64_t k, bool normalize)
{
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    Call call(logits);
    Plan plan(call, tokens, experts, k, logits);
    Tensor weights = Empty({tokens, k}, at::kFloat, logits), ids = Empty({tokens, k}, at::kInt, logits);
    Call::Ok(lib.route(call, tokens, experts, k, Data(logits), Ld(logits), TypeOf(logits.scalar_type()), normalize,
                       Floats(weights), static_cast<int32_t*>(ids.data_ptr()),
                       static_cast<int32_t*>(plan.offsets.data_ptr()), static_cast<int32_t*>(plan.tokens.data_ptr()),
                       static_cast<int32_t*>(plan.places.data_ptr()), Data(plan.buffer)),
             "aclsparseRoute");
    return {weights, ids, plan.offsets, plan.tokens, plan.places};
}

struct RouteNode : torch::autograd::Function<RouteNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, bool normalize)
    {
        variable_list out = RunRoute(logits, k, normalize);
        ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({normalize ? Tensor() : logits, out[0], out[1]});
        ctx->saved_data["experts"] = logits.size(1);
        ctx->saved_data["type"] = static_cast<int64_t>(logits.scalar_type());
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        NoTangent(grads[0]);
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &weights = saved[1], &ids = saved[2];
        const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
        const int64_t tokens = ids.size(0), k = ids.size(1), experts = ctx->saved_data["experts"].toInt();
        const Tensor grad = grads[0].to(at::kFloat).contiguous();
        Tensor out = Empty({tokens, experts}, type, ids);
        Call call(ids);
        Call::Ok(lib.routeGrad(call, tokens, experts, k, Data(logits), logits.defined() ? Ld(logits) : 0, TypeOf(type),
                               !logits.defined(), Floats(weights), Ints(ids), Floats(grad), Data(out), experts),
                 "aclsparseRouteGrad");
        return Once({grads[0], logits, weights}, {out, Tensor(), Tensor()});
    }
};

variable_list Route(const Tensor& logits, int64_t k, bool normalize)
{
    NoTangent(logits);
    TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be two-dimensional");
    TORCH_CHECK_TYPE(IsFloat(logits.scalar_type()), "logits must be float32, float16 or bfloat16, got ",
                     logits.scalar_type());
    OnGpu(logits);
    CheckRoute(logits.size(0), logits.size(1), k);
    const Tensor rows = Rows(logits);
    return Tracked(logits, {}) ? RouteNode::apply(rows, k, normalize) : RunRoute(rows, k, normalize);
}

variable_list ExpertPlan(const Tensor& given, int64_t experts)
{
    TORCH_CHECK_VALUE(given.dim() == 2, "ids must be two-dimensional");
    OnGpu(given);
    const Tensor ids = Index(given, "ids");
    CheckRoute(ids.size(0), experts, ids.size(1));
    Call call(ids);
    Plan plan(call, ids.size(0), experts, ids.size(1), ids);
    Call::Ok(lib.expertPlan(call, ids.size(0), experts, ids.size(1), Ints(ids),
                            static_cast<int32_t*>(plan.offsets.data_ptr()),
                            static_cast<int32_t*>(plan.tokens.data_ptr()),
                            static_cast<int32_t*>(plan.places.data_ptr()), Data(plan.buffer)),
             "aclsparseExpertPlan");
    return {plan.offsets, plan.tokens, plan.places};
}

// ------------------------------------------------------------------ products

Tensor RunGrouped(aclsparseOperation_t op, const Tensor& a, const Tensor& b, const Tensor& offsets, const Tensor& index,
                  int64_t rows, int64_t n, int64_t k, at::ScalarType type)
{
    Tensor out = Empty({rows, n}, type, a);
    Call call(a);
    Call::Ok(lib.groupedMM(call, op, b.size(0), rows, n, k, Ints(offsets), Ints(index), a.size(0), Data(a), Ld(a),
                           Data(b), Ld(b), b.size(0) > 1 ? b.stride(0) : 0, TypeOf(a.scalar_type()), Data(out),
                           std::max<int64_t>(n, 1), TypeOf(type)),
             "aclsparseGroupedMM");
    return out;
}

// lists: where to put the buffer that lists each row's assignments, null for none
Tensor RunCombine(const Tensor& y, const Tensor& places, const Tensor& weights, at::ScalarType type,
                  Tensor* lists = nullptr)
{
    const int64_t tokens = places.size(0), k = places.size(1), width = y.size(1), rows = y.size(0);
    Tensor out = Empty({tokens, width}, type, y);
    Call call(y);
    if (lists == nullptr) {
        Call::Ok(lib.combine(call, tokens, k, width, rows, Ints(places), Floats(weights), Data(y), Ld(y),
                             TypeOf(y.scalar_type()), Data(out), std::max<int64_t>(width, 1), TypeOf(type)),
                 "aclsparseCombine");
        return out;
    }
    size_t bytes = 0;
    Call::Ok(lib.combineGradBufferSize(call, tokens, k, rows, &bytes), "aclsparseCombineGradAny_bufferSize");
    *lists = Empty({static_cast<int64_t>(bytes)}, at::kByte, y);
    Call::Ok(lib.combineAndList(call, tokens, k, width, rows, Ints(places), Floats(weights), Data(y), Ld(y),
                                TypeOf(y.scalar_type()), Data(out), std::max<int64_t>(width, 1), TypeOf(type),
                                Data(*lists)),
             "aclsparseCombineAndList");
    return out;
}

// A plan's tensors, of which some may be undefined: autograd sees only the operands.
struct Sorted {
    Tensor offsets, tokens, places;
};

struct GroupedNode : torch::autograd::Function<GroupedNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& w, const Sorted& plan)
    {
        const Tensor &offsets = plan.offsets, &tokens = plan.tokens;
        ctx->save_for_backward({a, w, offsets, tokens, plan.places});
        ctx->saved_data["a"] = a.requires_grad();
        ctx->saved_data["w"] = w.requires_grad();
        return RunGrouped(ACL_SPARSE_OP_TRANSPOSE, a, w, offsets, tokens, tokens.defined() ? tokens.size(0) : a.size(0),
                          w.size(1), w.size(2), a.scalar_type());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &a = saved[0], &w = saved[1], &offsets = saved[2], &tokens = saved[3], &places = saved[4];
        NoTangent(grads[0]);
        const Tensor grad = Rows(grads[0]);
        const int64_t rows = grad.size(0), groups = w.size(0), n = w.size(1), k = w.size(2);
        Tensor da, dw;
        if (ctx->saved_data["a"].toBool()) {
            if (tokens.defined()) {
                // a token's rows are summed in fp32 and rounded once
                const Tensor part =
                    RunGrouped(ACL_SPARSE_OP_NON_TRANSPOSE, grad, w, offsets, {}, rows, k, n, at::kFloat);
                da = RunCombine(part, places, {}, a.scalar_type());
            } else {
                da = RunGrouped(ACL_SPARSE_OP_NON_TRANSPOSE, grad, w, offsets, {}, rows, k, n, a.scalar_type());
            }
        }
        if (ctx->saved_data["w"].toBool()) {
            dw = Empty({groups, n, k}, w.scalar_type(), w);
            Call call(a);
            const aclDataType type = TypeOf(a.scalar_type());
            Call::Ok(lib.groupedMMGrad(call, groups, rows, n, k, Ints(offsets), Ints(tokens), a.size(0), Data(grad),
                                       Ld(grad), Data(a), Ld(a), type, Data(dw), std::max<int64_t>(k, 1), n * k, type),
                     "aclsparseGroupedMMGrad");
        }
        return Once({grads[0], a, w}, {da, dw, Tensor()});
    }
};

void CheckPlan(const Tensor& a, const Tensor& offsets, const Tensor& tokens, int64_t groups)
{
    TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) >= 2,
                      "offsets must be one-dimensional, one more than the experts");
    SameDevice(a, offsets, "offsets");
    SameDevice(a, tokens, "tokens");
    TORCH_CHECK_VALUE(offsets.size(0) == groups + 1, "the plan has ", offsets.size(0) - 1, " experts, w ", groups);
}

// The rows of a that the plan reads: one per sorted row or, with gather, per token.  More are rows of no expert, or
// tokens that nothing names.
void CheckRows(const Tensor& a, const optional<Tensor>& tokens, const optional<Tensor>& places, bool gather)
{
    if (gather) {
        TORCH_CHECK_VALUE(!places.has_value() || places->dim() != 2 || a.size(0) >= places->size(0), "a has ",
                          a.size(0), " rows, the plan ", places->size(0), " tokens");
    } else {
        TORCH_CHECK_VALUE(!tokens.has_value() || a.size(0) >= tokens->numel(), "a has ", a.size(0),
                          " rows, the plan ", tokens->numel(), " (gather takes a in the order of the tokens)");
    }
}

Tensor GroupedMM(const Tensor& a, const Tensor& w, const Tensor& planOffsets, const optional<Tensor>& planTokens,
                 const optional<Tensor>& planPlaces, bool gather)
{
    NoTangent(a);
    NoTangent(w);
    TORCH_CHECK_VALUE(a.dim() == 2 && w.dim() == 3 && a.size(1) == w.size(2),
                      "a must be [rows, K] and w [experts, N, K], got ", a.sizes(), " and ", w.sizes());
    TORCH_CHECK_TYPE(IsHalf(a.scalar_type()) && w.scalar_type() == a.scalar_type(),
                     "a and w must both be float16 or bfloat16, got ", a.scalar_type(), " and ", w.scalar_type());
    OnGpu(a);
    SameDevice(a, w, "w");
    TORCH_CHECK_VALUE(!gather || planTokens.has_value(), "gather needs the plan's tokens");
    const Tensor offsets = Index(planOffsets, "offsets");
    const Tensor tokens = gather ? Index(*planTokens, "tokens") : Tensor();
    CheckPlan(a, offsets, tokens, w.size(0));
    CheckRows(a, planTokens, planPlaces, gather);
    const Tensor ra = Rows(a), rw = Rows(w);
    if (!Tracked(a, w)) {
        return RunGrouped(ACL_SPARSE_OP_TRANSPOSE, ra, rw, offsets, tokens, gather ? tokens.size(0) : ra.size(0),
                          rw.size(1), rw.size(2), ra.scalar_type());
    }
    Tensor places;
    if (gather && a.requires_grad()) {
        TORCH_CHECK_VALUE(planPlaces.has_value() && planPlaces->dim() == 2 &&
                              planPlaces->numel() == tokens.numel() && planPlaces->size(0) == a.size(0),
                          "a gradient through gather needs the plan's places, [tokens, k]");
        places = Index(*planPlaces, "places");
        SameDevice(a, places, "places");
    }
    return GroupedNode::apply(ra, rw, Sorted{offsets, tokens, places});
}

Tensor GroupedMMScaled(const Tensor& a, const Tensor& aScale, const Tensor& wGiven, const Tensor& wScaleGiven,
                       const optional<Tensor>& planOffsets, const optional<Tensor>& planTokens,
                       const optional<Tensor>& planPlaces, bool gather, at::ScalarType type)
{
    NoTangent(aScale);
    NoTangent(wScaleGiven);
    Tensor w = wGiven, wScale = wScaleGiven, offsets, tokens;
    if (!planOffsets.has_value()) {
        TORCH_CHECK_VALUE(!gather, "gather needs a plan");
        TORCH_CHECK_VALUE(w.dim() == 2 && wScale.dim() == 1, "without a plan w is [N, K] and w_scale [N]");
        w = w.unsqueeze(0);
        wScale = wScale.unsqueeze(0);
    }
    TORCH_CHECK_VALUE(a.dim() == 2 && w.dim() == 3 && a.size(1) == w.size(2),
                      "a must be [rows, K] and w [experts, N, K], got ", a.sizes(), " and ", w.sizes());
    TORCH_CHECK_TYPE(a.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "a and w must be int8, got ",
                     a.scalar_type(), " and ", w.scalar_type());
    TORCH_CHECK_TYPE(aScale.scalar_type() == at::kFloat && wScale.scalar_type() == at::kFloat,
                     "the scales must be float32");
    TORCH_CHECK_VALUE(aScale.dim() == 1 && aScale.size(0) == a.size(0) && wScale.sizes() == w.sizes().slice(0, 2),
                      "a_scale must hold one scale per row of a, w_scale one per row of w");
    TORCH_CHECK_TYPE(IsFloat(type), "out_dtype must be float32, float16 or bfloat16, got ", type);
    TORCH_CHECK_VALUE(a.size(1) <= kMaxScaledK, "K must not exceed ", kMaxScaledK);
    OnGpu(a);
    SameDevice(a, aScale, "a_scale");
    SameDevice(a, w, "w");
    SameDevice(a, wScale, "w_scale");
    if (planOffsets.has_value()) {
        TORCH_CHECK_VALUE(!gather || planTokens.has_value(), "gather needs the plan's tokens");
        offsets = Index(*planOffsets, "offsets");
        if (gather) tokens = Index(*planTokens, "tokens");
        CheckPlan(a, offsets, tokens, w.size(0));
        CheckRows(a, planTokens, planPlaces, gather);
    }
    const Tensor ra = Rows(a), rw = Rows(w), sa = aScale.contiguous(), sw = wScale.contiguous();
    const int64_t rows = gather ? tokens.size(0) : ra.size(0), n = rw.size(1);
    Tensor out = Empty({rows, n}, type, a);
    Call call(a);
    Call::Ok(lib.groupedMMScaled(call, rw.size(0), rows, n, rw.size(2), Ints(offsets), Ints(tokens), ra.size(0),
                                 static_cast<const int8_t*>(Data(ra)), Ld(ra), Floats(sa),
                                 static_cast<const int8_t*>(Data(rw)), Ld(rw), rw.size(0) > 1 ? rw.stride(0) : 0,
                                 Floats(sw), Data(out), std::max<int64_t>(n, 1), TypeOf(type)),
             "aclsparseGroupedMMScaled");
    return Tracked(aScale, wScale) ? Undifferentiable({aScale, wScale}, {out}, "grouped_mm_scaled has no gradient")[0]
                                   : out;
}

// ------------------------------------------------------------------ combination

struct CombineNode : torch::autograd::Function<CombineNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const optional<Tensor>& given, const Sorted& plan)
    {
        const Tensor weights = given.value_or(Tensor()), &places = plan.places;
        Tensor lists;  // for y's gradient; kept only where one is asked for
        const Tensor out =
            RunCombine(y, places, weights, y.scalar_type(), y.requires_grad() ? &lists : nullptr);
        ctx->save_for_backward({y, weights, places, lists});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &y = saved[0], &weights = saved[1], &places = saved[2], &lists = saved[3];
        NoTangent(grads[0]);
        const Tensor grad = Rows(grads[0]);
        const int64_t tokens = places.size(0), k = places.size(1), rows = y.size(0), width = y.size(1);
        Call call(y);
        Tensor dy, dw;
        if (lists.defined()) dy = Empty({rows, width}, y.scalar_type(), y);
        if (weights.defined() && weights.requires_grad()) dw = Empty({tokens, k}, at::kFloat, y);
        Call::Ok(lib.combineGrad(call, tokens, k, width, rows, Ints(places), Floats(weights), Data(y), Ld(y),
                                 Data(grad), Ld(grad), TypeOf(y.scalar_type()), Data(dy), std::max<int64_t>(width, 1),
                                 Floats(dw), Data(lists), /*listed=*/1),
                 "aclsparseCombineGradAny");
        return Once({grads[0], y, weights}, {dy, dw, Tensor()});
    }
};

Tensor Combine(const Tensor& y, const Tensor& planOffsets, const optional<Tensor>& planPlaces,
               const optional<Tensor>& givenWeights)
{
    NoTangent(y);
    if (givenWeights.has_value()) NoTangent(*givenWeights);
    TORCH_CHECK_VALUE(planPlaces.has_value() && planPlaces->dim() == 2,
                      "combine needs the plan's places, [tokens, k]");
    TORCH_CHECK_VALUE(y.dim() == 2, "y must be [rows, width]");
    TORCH_CHECK_TYPE(IsHalf(y.scalar_type()), "y must be float16 or bfloat16, got ", y.scalar_type());
    TORCH_CHECK_VALUE(planPlaces->size(1) >= 1 && planPlaces->size(1) <= kMaxK, "k must lie in [1, ", kMaxK, "]");
    OnGpu(y);
    const Tensor places = Index(*planPlaces, "places"), offsets = Index(planOffsets, "offsets");
    SameDevice(y, places, "places");
    SameDevice(y, offsets, "offsets");
    Tensor weights;
    if (givenWeights.has_value()) {
        weights = *givenWeights;
        SameDevice(y, weights, "weights");
        TORCH_CHECK_TYPE(weights.scalar_type() == at::kFloat, "weights must be float32, got ", weights.scalar_type());
        TORCH_CHECK_VALUE(weights.sizes() == places.sizes(), "weights must be ", places.sizes(), ", got ",
                          weights.sizes());
        weights = weights.contiguous();
    }
    const Tensor rows = Rows(y);
    if (!Tracked(y, weights)) return RunCombine(rows, places, weights, y.scalar_type());
    return CombineNode::apply(rows, weights.defined() ? optional<Tensor>(weights) : std::nullopt,
                              Sorted{{}, {}, places});
}

}  // namespace

PYBIND11_MODULE(_ops_sparse_experts, m)
{
    m.attr("build_id") = ACLSPARSE_HIP_BUILD_ID;
    m.def("bind", &Bind);
    m.def("route", &Route);
    m.def("expert_plan", &ExpertPlan);
    m.def("grouped_mm", &GroupedMM);
    m.def("grouped_mm_scaled", &GroupedMMScaled);
    m.def("combine", &Combine);
}
