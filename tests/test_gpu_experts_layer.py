"""The example layer: every experts' operator together, forward, backward and in 8 bits."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "experts_layer.py")
_SPEC = importlib.util.spec_from_file_location("experts_layer", _PATH)
example = importlib.util.module_from_spec(_SPEC)
_SPEC.loader.exec_module(example)


def plain(x, gate, w_in, w_out, ids):
    """The layer in float64 on the CPU for a given choice; the roundings to 16 bits are not in it."""
    logits = x @ gate.T
    weights = torch.softmax(torch.gather(logits, 1, ids), 1)
    out = []
    for t in range(len(x)):
        rows = [w_out[e] @ torch.nn.functional.silu(w_in[e] @ x[t]) for e in ids[t].tolist()]
        out.append(sum(w * r for w, r in zip(weights[t], rows)))
    return torch.stack(out)


@pytest.mark.parametrize("tokens,experts,k,width,hidden", [(1, 4, 2, 64, 96), (37, 6, 3, 40, 72), (130, 3, 1, 128, 64)])
def test_layer_and_its_gradients(tokens, experts, k, width, hidden):
    dev = torch.device("cuda")
    x = torch.randn(tokens, width, generator=torch.Generator().manual_seed(tokens)).to(dev).half()
    gate, w_in, w_out = example.weights_of(experts, width, hidden, 3, torch.float16)
    ids = example.route(x.float() @ gate.T, k)[1].cpu().long()
    inputs = [t.clone().requires_grad_() for t in (x, gate, w_in, w_out)]
    out = example.layer(*inputs, k)
    seed = torch.randn(tokens, width, generator=torch.Generator().manual_seed(9)).to(dev).half()
    grads = torch.autograd.grad(out, inputs, seed)
    exact_inputs = [t.cpu().double().requires_grad_() for t in (x, gate, w_in, w_out)]
    exact = plain(*exact_inputs, ids)
    exact_grads = torch.autograd.grad(exact, exact_inputs, seed.cpu().double())
    # Each value passes at most six roundings to fp16 on its way (hidden, activation, row, output and the same
    # backwards), each 2^-11 of a value: their sum over independent terms stays under 6 * 2^-11 of the norm.
    for got, want in zip((out, *grads), (exact, *exact_grads)):
        error = (got.detach().cpu().double() - want.detach()).norm()
        assert error <= 6 * 2**-11 * want.detach().norm(), (error / want.detach().norm())


@pytest.mark.parametrize("tokens", [1, 64])
def test_layer_in_8_bits(tokens):
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(4)).cuda().bfloat16()
    gate, w_in, w_out = example.weights_of(8, 256, 512, 5)
    full = example.layer(x, gate, w_in, w_out, 2).float()
    eight = example.layer_8_bits(x, gate, example.to_8_bits(w_in), example.to_8_bits(w_out), 2).float()
    # A row of normal values has its largest at 3 to 4.5 deviations: a step is under 4.5 / 127 of a deviation and its
    # rounding adds step / sqrt(12) = 0.0103.  Four such factors (two products), and silu's skewed values, whose largest
    # may be twice as far out in deviations, stay under sqrt(3 * 0.0103^2 + (2 * 0.0103)^2) = 0.028; bf16 adds
    # sqrt(6) * 2^-9 = 0.005.
    assert (eight - full).norm() <= 0.034 * full.norm()


def test_training_lowers_the_loss():
    x = torch.randn(256, 64, generator=torch.Generator().manual_seed(6)).cuda().bfloat16()
    teacher = example.weights_of(4, 64, 128, 7)
    student = example.weights_of(4, 64, 128, 7)
    student = [student[0]] + [w * 1.5 for w in student[1:]]
    target = example.layer(x, *teacher, 2).float()
    losses = example.train(x, target, student, 2, 20, 20.0)
    assert losses[-1] < 0.5 * losses[0]


def test_command(capsys):
    example.main(["--tokens", "64", "--experts", "4", "--chosen", "2", "--width", "64", "--hidden", "64", "--steps",
                  "3", "--rate", "1"])
    out = capsys.readouterr().out
    assert "one token, 8 bits" in out and "of the norm" in out
