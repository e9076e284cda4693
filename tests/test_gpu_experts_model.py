"""The example model: the experts' operators, log probabilities, the AdamW step and 4-bit serving together."""
import importlib.util
import os
import sys

import pytest
import torch

from ops_sparse import adamw_state, adamw_step, grouped_mm_mx4, mx4_dequantize, mx4_quantize, route

pytestmark = pytest.mark.gpu

_FOLDER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")
if _FOLDER not in sys.path:
    sys.path.append(_FOLDER)
_SPEC = importlib.util.spec_from_file_location("experts_model", os.path.join(_FOLDER, "experts_model.py"))
example = importlib.util.module_from_spec(_SPEC)
_SPEC.loader.exec_module(example)


def plain_loss(tokens, targets, parameters, ids, bonus):
    """The loss in float64 on the CPU for a given choice of experts; the roundings to 16 bits are not in it."""
    embedding, gate, w_in, w_out, head = parameters
    x = embedding[tokens]
    weights = torch.softmax(torch.gather(x @ gate.T, 1, ids), 1)
    out = []
    for t in range(len(x)):
        rows = [w_out[e] @ torch.nn.functional.silu(w_in[e] @ x[t]) for e in ids[t].tolist()]
        out.append(x[t] + sum(w * r for w, r in zip(weights[t], rows)))
    logs = torch.log_softmax(torch.stack(out) @ head.T, 1)
    named = targets >= 0
    entropy = -(logs.exp() * logs).sum(1)
    return -(logs[named].gather(1, targets[named][:, None]).sum() / named.sum() + bonus * entropy.mean())


def batch(tokens, vocabulary, seed):
    g = torch.Generator().manual_seed(seed)
    targets = torch.randint(0, vocabulary, (tokens,), generator=g)
    targets[::5] = -100
    return torch.randint(0, vocabulary, (tokens,), generator=g), targets


@pytest.mark.parametrize("tokens,vocabulary,experts,k,width,hidden", [(1, 64, 4, 2, 64, 96), (33, 1001, 5, 3, 40, 72)])
def test_the_models_gradients(tokens, vocabulary, experts, k, width, hidden):
    at, targets = batch(tokens, vocabulary, tokens)
    if tokens == 1:
        targets[0] = 3
    parameters = example.parameters_of(vocabulary, experts, width, hidden, 5, torch.float16)
    ids = route(parameters[0][at.cuda()].float() @ parameters[1].float().T, k)[1].cpu().long()
    given = [p.clone().requires_grad_() for p in parameters]
    loss = example.loss_of(at.cuda(), targets.cuda(), given, k, 0.01)
    grads = torch.autograd.grad(loss, given)
    exact = [p.cpu().double().requires_grad_() for p in parameters]
    want = plain_loss(at, targets, exact, ids, 0.01)
    wants = torch.autograd.grad(want, exact)
    # Each value passes at most ten roundings to fp16 on its way (hidden, activation, row, output, sum, logits, and back
    # the logits' gradient and three products), each 2^-11 of a value, and logits of a few units are off by 2^-11 of that
    # in the exponent: under 4 times 2^-11 of a probability.  Their sum stays under 14 * 2^-11 of the norm.  fp16 itself
    # ends at 2^-24: gradients of loss / T below that are lost, half a step of which each value may be off.
    for got, exact_grad in zip(grads, wants):
        error = (got.cpu().double() - exact_grad).norm()
        assert error <= 14 * 2**-11 * exact_grad.norm() + 2**-25 * got.numel() ** 0.5, error / exact_grad.norm()
    loss, want = loss.detach(), want.detach()
    assert abs(float(loss) - float(want)) <= 14 * 2**-11 * abs(float(want))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_moves_by_the_formula(bits):
    # the first step from moments of zero: m / sqrt(v) is the gradient's sign, so each value with a gradient far above eps
    # moves by the rate, decay apart
    at, targets = batch(64, 500, 3)
    parameters = [p.float().requires_grad_() if i == 1 else p.requires_grad_()
                  for i, p in enumerate(example.parameters_of(500, 4, 64, 64, 7))]
    grads = torch.autograd.grad(example.loss_of(at.cuda(), targets.cuda(), parameters, 2, 0.0), parameters)
    before = [p.detach().float().clone() for p in parameters]
    state = adamw_state(parameters, bits=bits)
    adamw_step(parameters, grads, state, 2.0**-8, weight_decay=0.0)
    for p, b, g, m in zip(parameters, before, grads, state.masters):
        big = g.float().abs() > 1e-4  # eps of 1e-8 is under 1e-4 of it
        moved = (b - m)[big]
        want = 2.0**-8 * g.float().sign()[big]
        # relative 1e-4 of eps and 12 roundings; the difference of fp32 values of a few units is off by 2^-22 or so
        assert bool(((moved - want).abs() <= 2.0**-8 * 1.1e-4 + 2.0**-23 * (b[big].abs() + 1)).all())
        assert torch.equal(p.detach(), m.to(p.dtype))
        assert torch.equal(m[g == 0], b[g == 0])


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_the_layer_in_4_bits(tokens):
    # against the products of the same codes in 64 bits, step by step
    embedding, gate, w_in, w_out, _ = example.parameters_of(512, 8, 192, 320, 9)
    x = embedding[torch.arange(tokens, device="cuda")]
    w4 = [mx4_quantize(w) for w in (w_in, w_out)]
    weights, ids, plan = route(x.float() @ gate.float().T, 2)
    rows = plan.tokens.long()

    def product(a, w, given):
        a, w = mx4_dequantize(a).double(), mx4_dequantize(w).double()
        expert = torch.searchsorted(plan.offsets.long()[1:].contiguous(), torch.arange(len(rows), device="cuda"), right=True)
        want = torch.stack([w[e] @ a[i] for e, i in zip(expert.tolist(), given.tolist())])
        size = torch.stack([w[e].abs() @ a[i].abs() for e, i in zip(expert.tolist(), given.tolist())])
        return want, size * a.shape[1] * 2.0**-23 + want.abs() * 2.0**-8 + 1e-30

    h = grouped_mm_mx4(mx4_quantize(x), w4[0], plan, gather=True)
    want, bound = product(mx4_quantize(x), w4[0], rows)
    assert bool(((h.double() - want).abs() <= bound).all())
    hidden = mx4_quantize(torch.nn.functional.silu(h))
    y = grouped_mm_mx4(hidden, w4[1], plan)
    want, bound = product(hidden, w4[1], torch.arange(len(rows), device="cuda"))
    assert bool(((y.double() - want).abs() <= bound).all())
    out = example.layer_4_bits(x, gate, *w4, 2)
    joined = (weights.double()[..., None] * y.double()[plan.places.long()]).sum(1)
    size = (weights.double()[..., None] * y.double()[plan.places.long()].abs()).sum(1)
    assert bool(((out.double() - joined).abs() <= joined.abs() * 2.0**-8 + size * 3 * 2.0**-24 + 1e-30).all())


def test_an_answer_and_its_alternatives():
    parameters = example.parameters_of(777, 4, 64, 96, 11)
    served = [mx4_quantize(w) for w in parameters[2:4]]
    tokens = torch.arange(20, device="cuda")
    r = example.answer(tokens, parameters, served, 2, 5)
    assert torch.equal(r.top_logprobs[:, 0], r.logprobs) and bool((r.top_logprobs.diff(dim=1) <= 0).all())
    one = example.answer(tokens[:1], parameters, served, 2, 5)
    assert one.top_ids.shape == (1, 5) and one.logprobs.shape == (1,)


def test_a_training_step_in_a_graph():
    # the embedding stays as it is: torch's gradient of a lookup adds in no order
    at, targets = (t.cuda() for t in batch(96, 700, 13))

    def start():
        return [p.requires_grad_(i > 0) for i, p in enumerate(example.parameters_of(700, 4, 64, 64, 15))]

    def step(parameters, state):
        grads = torch.autograd.grad(example.loss_of(at, targets, parameters, 2, 0.01), parameters[1:])
        adamw_step(parameters[1:], grads, state, 1e-2)

    eager, captured = start(), start()
    states = [adamw_state(p[1:], bits=8, seed=5) for p in (eager, captured)]
    side = torch.cuda.Stream()  # what the captured step sets up lazily
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = start()
        step(warm, adamw_state(warm[1:], bits=8))
        del warm
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, states[1])
    for seed in range(4):
        new = batch(96, 700, 20 + seed)
        at.copy_(new[0])
        targets.copy_(new[1])
        step(eager, states[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager[1:] + states[0].moments, captured[1:] + states[1].moments):
            assert torch.equal(a.detach(), b.detach()), seed
    assert states[0].step[0] == states[1].step[0] == 4


def test_command(capsys):
    example.main(["--tokens", "64", "--vocabulary", "300", "--experts", "4", "--width", "64", "--hidden", "64", "--steps",
                  "3"])
    out = capsys.readouterr().out
    assert "loss" in out and "in 4 bits" in out
