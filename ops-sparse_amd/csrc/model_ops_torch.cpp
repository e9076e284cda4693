// The operators of a model's training and serving on torch tensors: argument
// checks, outputs, and the node of the log probabilities.  Part of the module
// that experts_torch.cpp defines.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>

#include <algorithm>
#include <unordered_set>

#include "torch_common.h"

namespace ops_sparse_torch {
namespace {

constexpr int64_t kBlock = 32, kMaxTop = 64, kMaxVocab = int64_t{1} << 30;

uint8_t* Bytes(const Tensor& t) { return t.defined() ? static_cast<uint8_t*>(t.data_ptr()) : nullptr; }

// Rows of all but the last dimension
int64_t RowsOf(const Tensor& t)
{
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    return rows;
}

Tensor Flat(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({RowsOf(t), t.size(t.dim() - 1)}); }

std::vector<int64_t> WithLast(const Tensor& t, int64_t last)
{
    std::vector<int64_t> shape(t.sizes().begin(), t.sizes().end());
    shape.back() = last;
    return shape;
}

// ------------------------------------------------------------------ microscaled 4 bits

// codes [..., B * 16] and scales [..., B]
void CheckMx4(const Tensor& codes, const Tensor& scales, const char* name)
{
    TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, name,
                     "'s codes and scales must be uint8, got ", codes.scalar_type(), " and ", scales.scalar_type());
    TORCH_CHECK_VALUE(codes.dim() >= 1 && codes.dim() == scales.dim() &&
                          codes.sizes().slice(0, codes.dim() - 1) == scales.sizes().slice(0, codes.dim() - 1) &&
                          codes.size(-1) == scales.size(-1) * 16,
                      name, "'s codes must be [..., 16 * blocks] and its scales [..., blocks], got ", codes.sizes(),
                      " and ", scales.sizes());
}

// Rows of codes aligned to 16 bytes: a copy only where they are not
Tensor AlignedRows(const Tensor& t)
{
    const Tensor rows = Rows(t);
    bool aligned = reinterpret_cast<uintptr_t>(rows.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < rows.dim(); ++i) aligned = aligned && (rows.size(i) <= 1 || rows.stride(i) % 16 == 0);
    return aligned ? rows : rows.clone(at::MemoryFormat::Contiguous);
}

variable_list Mx4Quantize(const Tensor& x)
{
    NoTangent(x);
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have a dimension");
    TORCH_CHECK_TYPE(IsFloat(x.scalar_type()), "x must be float32, float16 or bfloat16, got ", x.scalar_type());
    OnGpu(x);
    const int64_t k = x.size(-1), blocks = (k + kBlock - 1) / kBlock;
    Tensor codes = Empty(WithLast(x, blocks * 16), at::kByte, x), scales = Empty(WithLast(x, blocks), at::kByte, x);
    if (x.numel() == 0) return {codes, scales};
    const Tensor rows = Rows(Flat(x.detach()));
    Call call(x);
    Call::Ok(lib.mx4Quantize(call, rows.size(0), k, Data(rows), Ld(rows), TypeOf(x.scalar_type()), Bytes(codes),
                             blocks * 16, Bytes(scales), blocks),
             "aclsparseMx4Quantize");
    return {codes, scales};
}

Tensor Mx4Dequantize(const Tensor& codes, const Tensor& scales, const optional<int64_t>& givenWidth,
                     at::ScalarType type)
{
    CheckMx4(codes, scales, "q");
    TORCH_CHECK_TYPE(IsFloat(type), "dtype must be float32, float16 or bfloat16, got ", type);
    const int64_t blocks = scales.size(-1), width = givenWidth.value_or(blocks * kBlock);
    const int64_t least = std::max<int64_t>((blocks - 1) * kBlock + 1, 0);
    TORCH_CHECK_VALUE(width >= least && width <= blocks * kBlock, "width must lie in [", least, ", ", blocks * kBlock,
                      "], got ", width);
    OnGpu(codes);
    SameDevice(codes, scales, "q's scales");
    Tensor out = Empty(WithLast(codes, width), type, codes);
    if (out.numel() == 0) return out;
    const Tensor c = Rows(Flat(codes)), s = Rows(Flat(scales));
    Call call(codes);
    Call::Ok(lib.mx4Dequantize(call, c.size(0), width, Bytes(c), Ld(c), Bytes(s), Ld(s), Data(out), width,
                               TypeOf(type)),
             "aclsparseMx4Dequantize");
    return out;
}

Tensor GroupedMMMx4(const Tensor& a, const Tensor& aScales, const Tensor& wGiven, const Tensor& wScalesGiven,
                    const optional<Tensor>& planOffsets, const optional<Tensor>& planTokens,
                    const optional<Tensor>& planPlaces, bool gather, at::ScalarType type)
{
    CheckMx4(a, aScales, "a");
    CheckMx4(wGiven, wScalesGiven, "w");
    Tensor w = wGiven, wScales = wScalesGiven, offsets, tokens;
    if (!planOffsets.has_value()) {
        TORCH_CHECK_VALUE(!gather, "gather needs a plan");
        TORCH_CHECK_VALUE(w.dim() == 2, "without a plan w is [N, K]");
        w = w.unsqueeze(0);
        wScales = wScales.unsqueeze(0);
    }
    TORCH_CHECK_VALUE(a.dim() == 2 && w.dim() == 3 && a.size(1) == w.size(2),
                      "a must be [rows, K] and w [experts, N, K], got codes of ", a.sizes(), " and ", w.sizes());
    TORCH_CHECK_TYPE(IsFloat(type), "out_dtype must be float32, float16 or bfloat16, got ", type);
    OnGpu(a);
    SameDevice(a, aScales, "a's scales");
    SameDevice(a, w, "w");
    SameDevice(a, wScales, "w's scales");
    if (planOffsets.has_value()) {
        TORCH_CHECK_VALUE(!gather || planTokens.has_value(), "gather needs the plan's tokens");
        offsets = Index(*planOffsets, "offsets");
        if (gather) tokens = Index(*planTokens, "tokens");
        CheckPlan(a, offsets, tokens, w.size(0));
        CheckRows(a, planTokens, planPlaces, gather);
    }
    const Tensor ra = AlignedRows(a), rw = AlignedRows(w), sa = Rows(aScales), sw = Rows(wScales);
    const int64_t rows = gather ? tokens.size(0) : ra.size(0), n = rw.size(1);
    Tensor out = Empty({rows, n}, type, a);
    const bool groups = rw.size(0) > 1;
    // a row of one dimension may have any stride
    auto ld = [](const Tensor& t) { return t.size(-2) > 1 ? Ld(t) : std::max<int64_t>(t.size(-1), 1); };
    Call call(a);
    Call::Ok(lib.groupedMMMx4(call, rw.size(0), rows, n, sa.size(1) * kBlock, Ints(offsets), Ints(tokens), ra.size(0),
                              Bytes(ra), ld(ra), Bytes(sa), ld(sa), Bytes(rw), ld(rw), groups ? rw.stride(0) : 0,
                              Bytes(sw), ld(sw), groups ? sw.stride(0) : 0, Data(out), std::max<int64_t>(n, 1),
                              TypeOf(type)),
             "aclsparseGroupedMMMx4");
    return out;
}

// ------------------------------------------------------------------ AdamW

using Tensors = std::vector<Tensor>;
using MaybeTensors = std::vector<optional<Tensor>>;

void OneFloat(const Tensor& first, const optional<Tensor>& t, const char* name)
{
    if (!t.has_value()) return;
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->numel() == 1, name, " must have one element");
    SameDevice(first, *t, name);
}

// A state's tensors for values of one shape
void CheckMoments(int64_t count, const Tensor& moments, const optional<Tensor>& exponents, const Tensor& like,
                  size_t place)
{
    const int64_t padded = (count + kBlock - 1) / kBlock * kBlock;
    const at::ScalarType type = exponents.has_value() ? at::kByte : at::kFloat;
    TORCH_CHECK_TYPE(moments.scalar_type() == type, "moments must be float32, or uint8 with exponents, got ",
                     moments.scalar_type(), " at ", place);
    TORCH_CHECK_VALUE(moments.dim() == 2 && moments.size(0) == 2 && moments.size(1) == padded &&
                          moments.is_contiguous(),
                      "moments must be contiguous, [2, ", padded, "] for ", count, " values, got ", moments.sizes(),
                      " at ", place);
    SameDevice(like, moments, "moments");
    if (!exponents.has_value()) return;
    TORCH_CHECK_TYPE(exponents->scalar_type() == at::kByte, "exponents must be uint8, got ", exponents->scalar_type());
    TORCH_CHECK_VALUE(exponents->dim() == 2 && exponents->size(0) == 2 && exponents->size(1) == padded / kBlock &&
                          exponents->is_contiguous(),
                      "exponents must be contiguous, [2, ", padded / kBlock, "] for ", count, " values, got ",
                      exponents->sizes(), " at ", place);
    SameDevice(like, *exponents, "exponents");
    TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(moments.data_ptr()) % 8 == 0, "moments must be aligned to 8 bytes");
}

// Memory that a step writes.  What two of a step's tensors share, they would write at once: the result would be any.
struct Written {
    uintptr_t begin, end;
    const char* name;
    size_t place;
};
void Add(std::vector<Written>& written, const Tensor& t, const char* name, size_t place)
{
    const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel() > 0) written.push_back({begin, begin + t.nbytes(), name, place});
}
void CheckApart(std::vector<Written>& written)
{
    std::sort(written.begin(), written.end(), [](const Written& a, const Written& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < written.size(); ++i) {
        const Written &a = written[i - 1], &b = written[i];
        TORCH_CHECK_VALUE(a.end <= b.begin, "the ", a.name, " at ", a.place, " and the ", b.name, " at ", b.place,
                          " share memory: no tensor may be there twice");
    }
}

void AdamWStep(const Tensors& params, const MaybeTensors& grads, const Tensors& moments,
               const optional<Tensors>& exponents, const optional<Tensors>& masters, const Tensor& step, int64_t seed,
               double lr, const optional<Tensor>& lrTensor, double beta1, double beta2, double eps, double weightDecay,
               const optional<Tensor>& gradScale, const optional<std::pair<int64_t, int64_t>>& factors)
{
    const size_t count = params.size();
    TORCH_CHECK_VALUE(grads.size() == count && moments.size() == count &&
                          (!exponents.has_value() || exponents->size() == count) &&
                          (!masters.has_value() || masters->size() == count),
                      "params, grads and the state's lists must have one entry per tensor");
    TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must lie in [0, 1)");
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps) && weightDecay >= 0 && std::isfinite(weightDecay) &&
                          (lrTensor.has_value() || (lr >= 0 && std::isfinite(lr))),
                      "lr, eps and weight_decay must be finite and not negative");
    TORCH_CHECK_VALUE(seed >= 0 && seed <= UINT32_MAX, "the seed must fit 32 bits without a sign");
    auto odd = [](int64_t f) { return f >= 0 && f <= UINT32_MAX && f % 2 != 0; };
    TORCH_CHECK_VALUE(!factors.has_value() || (odd(factors->first) && odd(factors->second)),
                      "the factors must be odd and fit 32 bits without a sign");
    TORCH_CHECK_TYPE(step.scalar_type() == at::kInt, "step must be int32, got ", step.scalar_type());
    TORCH_CHECK_VALUE(step.dim() == 1 && step.size(0) >= 1, "step must be one-dimensional and hold the steps taken");
    OnGpu(step);
    OneFloat(step, lrTensor, "lr");
    OneFloat(step, gradScale, "grad_scale");
    std::vector<aclsparseAdamWTensor_t> table(count);
    std::vector<Tensor> kept;  // gradients that had to be copied
    std::vector<Written> written;
    written.reserve(count * 4);
    for (size_t i = 0; i < count; ++i) {
        const Tensor& p = params[i];
        TORCH_CHECK_TYPE(IsFloat(p.scalar_type()), "params must be float32, float16 or bfloat16, got ",
                         p.scalar_type(), " at ", i);
        TORCH_CHECK_VALUE(p.is_contiguous(), "params must be contiguous, the one at ", i, " is not");
        OnGpu(p);
        SameDevice(step, p, "params");
        const int64_t n = p.numel();
        CheckMoments(n, moments[i], exponents.has_value() ? optional<Tensor>((*exponents)[i]) : std::nullopt, step, i);
        float* master = nullptr;
        if (masters.has_value()) {
            const Tensor& m = (*masters)[i];
            TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat, "masters must be float32, got ", m.scalar_type());
            TORCH_CHECK_VALUE(m.sizes() == p.sizes() && m.is_contiguous(),
                              "masters must be contiguous and of their params' shapes, the one at ", i, " is not");
            SameDevice(step, m, "masters");
            master = Floats(m);
            // a parameter in fp32 may be its own master
            if (p.scalar_type() != at::kFloat || master != Data(p)) Add(written, m, "master", i);
        }
        Add(written, p, "param", i);
        Add(written, moments[i], "moments", i);
        if (exponents.has_value()) Add(written, (*exponents)[i], "exponents", i);
        Tensor g;
        if (grads[i].has_value() && grads[i]->defined()) {
            TORCH_CHECK_TYPE(IsFloat(grads[i]->scalar_type()), "grads must be float32, float16 or bfloat16, got ",
                             grads[i]->scalar_type(), " at ", i);
            TORCH_CHECK_VALUE(grads[i]->layout() == at::kStrided && grads[i]->sizes() == p.sizes(),
                              "grads must be dense and of their params' shapes, the one at ", i, " is not");
            SameDevice(step, *grads[i], "grads");
            g = grads[i]->contiguous();
            kept.push_back(g);
        }
        table[i] = {Data(p), Data(g), master, Data(moments[i]),
                    exponents.has_value() ? Bytes((*exponents)[i]) : nullptr, n, TypeOf(p.scalar_type()),
                    g.defined() ? TypeOf(g.scalar_type()) : ACL_FLOAT};
    }
    CheckApart(written);
    aclsparseAdamWOptions_t o{};
    o.lr = lr;
    o.beta1 = beta1;
    o.beta2 = beta2;
    o.eps = eps;
    o.weightDecay = weightDecay;
    o.lrDevice = lrTensor.has_value() ? Floats(*lrTensor) : nullptr;
    o.gradScale = gradScale.has_value() ? Floats(*gradScale) : nullptr;
    o.step = static_cast<int32_t*>(step.data_ptr());
    const Tensor buffer = Empty({64}, at::kByte, step);
    o.buffer = Data(buffer);
    o.seed = static_cast<uint32_t>(seed);
    o.momentBits = exponents.has_value() ? 8 : 32;
    Call call(step);
    if (factors.has_value()) {
        Call::Ok(lib.adamWMixed(call, static_cast<int64_t>(count), table.data(), &o, static_cast<uint32_t>(factors->first),
                                static_cast<uint32_t>(factors->second)),
                 "aclsparseAdamWMixed");
    } else {
        Call::Ok(lib.adamW(call, static_cast<int64_t>(count), table.data(), &o), "aclsparseAdamW");
    }
    // a value that a backward pass still needs has changed: it raises, as after a torch operation in place
    for (size_t i = 0; i < count; ++i) {
        if (!params[i].is_inference() && grads[i].has_value()) torch::autograd::impl::bump_version(params[i]);
    }
}

Tensors AdamWMoments(const Tensors& moments, const Tensors& exponents)
{
    TORCH_CHECK_VALUE(moments.size() == exponents.size(), "there must be exponents for each of the moments");
    Tensors outs;
    std::vector<aclsparseAdamWTensor_t> table(moments.size());
    for (size_t i = 0; i < moments.size(); ++i) {
        OnGpu(moments[i]);
        TORCH_CHECK_VALUE(moments[i].dim() == 2, "moments must be two-dimensional");
        const int64_t count = moments[i].size(1);
        CheckMoments(count, moments[i], exponents[i], moments[0], i);
        outs.push_back(Empty({2, count}, at::kFloat, moments[i]));
        table[i] = {nullptr, nullptr, Floats(outs.back()), Data(moments[i]), Bytes(exponents[i]), count, ACL_FLOAT,
                    ACL_FLOAT};
    }
    if (moments.empty()) return outs;
    Call call(moments[0]);
    Call::Ok(lib.adamWMoments(call, static_cast<int64_t>(table.size()), table.data()), "aclsparseAdamWMoments");
    return outs;
}

// ------------------------------------------------------------------ log probabilities

// In a capture: raises where the gradient would go to a leaf that an autograd graph made on another stream still holds.
// torch's engine then orders that stream behind the captured one, which ends the process when the capture ends.
void CheckCapture(const Tensor& t)
{
    if (!t.requires_grad() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    // by id: autograd's streams are of another device type than HIP's own
    const c10::StreamId current = c10::hip::getCurrentHIPStream(t.get_device()).id();
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    std::unordered_set<torch::autograd::Node*> seen;
    auto add = [&](const std::shared_ptr<torch::autograd::Node>& node) {
        if (node != nullptr && seen.insert(node.get()).second) todo.push_back(node);
    };
    add(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        for (const auto& edge : node->next_edges()) add(edge.function);
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get()) == nullptr) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream.has_value() || stream->id() == current,
                    "token_logprobs is captured while an autograd graph of the same leaf, made on another stream, is "
                    "alive: delete what holds it (its results) before the capture");
    }
}

struct Logprobs {
    Tensor logprobs, entropy, topLogprobs, topIds, stats;
};

Logprobs RunLogprobs(const Tensor& logits, const Tensor& targets, int64_t top, bool entropy, bool stats)
{
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    Logprobs r;
    r.logprobs = Empty({rows}, at::kFloat, logits);
    if (entropy) r.entropy = Empty({rows}, at::kFloat, logits);
    if (stats) r.stats = Empty({rows, 2}, at::kFloat, logits);
    if (top > 0) {
        r.topLogprobs = Empty({rows, top}, at::kFloat, logits);
        r.topIds = Empty({rows, top}, at::kInt, logits);
    }
    Call call(logits);
    size_t bytes = 0;
    Call::Ok(lib.logprobsBufferSize(call, rows, vocab, top, &bytes), "aclsparseTokenLogprobs_bufferSize");
    const Tensor buffer = Empty({static_cast<int64_t>(bytes)}, at::kByte, logits);
    Call::Ok(lib.logprobs(call, rows, vocab, Data(logits), Ld(logits), TypeOf(logits.scalar_type()), Data(targets),
                          targets.scalar_type() == at::kLong ? ACL_INT64 : ACL_INT32, Floats(r.logprobs),
                          Floats(r.entropy), Floats(r.stats), top, Floats(r.topLogprobs),
                          static_cast<int32_t*>(Data(r.topIds)), Data(buffer)),
             "aclsparseTokenLogprobs");
    return r;
}

struct LogprobsNode : torch::autograd::Function<LogprobsNode> {
    // logprobs, then the entropy and the alternatives where they are asked for
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t top,
                                 bool entropy)
    {
        const Logprobs r = RunLogprobs(logits, targets, top, entropy, /*stats=*/true);
        variable_list out{r.logprobs};
        if (entropy) out.push_back(r.entropy);
        if (top > 0) {
            out.push_back(r.topLogprobs);
            out.push_back(r.topIds);
            ctx->mark_non_differentiable({r.topIds});
        }
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({logits, targets, r.stats, r.entropy, r.topIds});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &targets = saved[1], &stats = saved[2], &entropy = saved[3], &ids = saved[4];
        size_t next = 1;
        const Tensor gl = grads[0], ge = entropy.defined() ? grads[next++] : Tensor(),
                     gt = ids.defined() ? grads[next] : Tensor();
        if (!gl.defined() && !ge.defined() && !gt.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        for (const Tensor& g : {gl, ge, gt}) NoTangent(g);
        auto floats = [](const Tensor& g) { return g.defined() ? g.to(at::kFloat).contiguous() : Tensor(); };
        const Tensor fl = floats(gl), fe = floats(ge), ft = floats(gt);
        const int64_t rows = logits.size(0), vocab = logits.size(1);
        Tensor out = Empty({rows, vocab}, logits.scalar_type(), logits);
        Call call(logits);
        Call::Ok(lib.logprobsGrad(call, rows, vocab, Data(logits), Ld(logits), TypeOf(logits.scalar_type()),
                                  Data(targets), targets.scalar_type() == at::kLong ? ACL_INT64 : ACL_INT32,
                                  Floats(stats), Floats(entropy), ids.defined() ? ids.size(1) : 0, Ints(ids),
                                  Floats(fl), Floats(fe), Floats(ft), Data(out), vocab),
                 "aclsparseTokenLogprobsGrad");
        return Once({logits, gl, ge, gt}, {out, Tensor(), Tensor(), Tensor()});
    }
};

// (logprobs, entropy, top log probabilities, top ids), None where not asked for
std::vector<optional<Tensor>> TokenLogprobs(const Tensor& given, const Tensor& givenTargets, int64_t top, bool entropy)
{
    NoTangent(given);
    TORCH_CHECK_VALUE(given.dim() >= 1 && given.sizes().slice(0, given.dim() - 1) == givenTargets.sizes(),
                      "logits must be [..., vocabulary] and targets [...], got ", given.sizes(), " and ",
                      givenTargets.sizes());
    TORCH_CHECK_TYPE(IsFloat(given.scalar_type()), "logits must be float32, float16 or bfloat16, got ",
                     given.scalar_type());
    TORCH_CHECK_TYPE(givenTargets.scalar_type() == at::kInt || givenTargets.scalar_type() == at::kLong,
                     "targets must be int32 or int64, got ", givenTargets.scalar_type());
    const int64_t vocab = given.size(-1);
    TORCH_CHECK_VALUE(vocab >= 1 && vocab <= kMaxVocab, "the vocabulary must lie in [1, ", kMaxVocab, "], got ", vocab);
    TORCH_CHECK_VALUE(top >= 0 && top <= vocab && top <= kMaxTop, "top must lie in [0, ",
                      std::min(vocab, kMaxTop), "], got ", top);
    OnGpu(given);
    SameDevice(given, givenTargets, "targets");
    const Tensor logits = Rows(Flat(given)), targets = givenTargets.reshape({-1}).contiguous();
    variable_list out;
    if (Tracked(given, {})) {
        CheckCapture(given);
        out = LogprobsNode::apply(logits, targets, top, entropy);
    } else {
        const Logprobs r = RunLogprobs(logits, targets, top, entropy, /*stats=*/false);
        out.push_back(r.logprobs);
        if (entropy) out.push_back(r.entropy);
        if (top > 0) out.insert(out.end(), {r.topLogprobs, r.topIds});
    }
    std::vector<optional<Tensor>> all(4);
    const bool shaped = given.dim() != 2;
    auto rowsLike = [&](const Tensor& t) { return shaped ? t.reshape(givenTargets.sizes()) : t; };
    size_t next = 0;
    all[0] = rowsLike(out[next++]);
    if (entropy) all[1] = rowsLike(out[next++]);
    for (int i = 2; i < 4 && top > 0; ++i, ++next) all[i] = shaped ? out[next].reshape(WithLast(given, top)) : out[next];
    return all;
}

}  // namespace

void DefineModelOps(pybind11::module_& m)
{
    m.def("mx4_quantize", &Mx4Quantize);
    m.def("mx4_dequantize", &Mx4Dequantize);
    m.def("grouped_mm_mx4", &GroupedMMMx4);
    m.def("adamw_step", &AdamWStep);
    m.def("adamw_moments", &AdamWMoments);
    m.def("token_logprobs", &TokenLogprobs);
}

}  // namespace ops_sparse_torch
