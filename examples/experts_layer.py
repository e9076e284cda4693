"""A layer of experts, trained and then served in 8 bits, by the experts' operators.

    python examples/experts_layer.py [--tokens 4096] [--experts 32] [--chosen 4] [--width 1024] [--hidden 2048]

Trains the layer for some steps to reproduce another layer of the same shape, lays its weights out in 8 bits once, and
compares what the two give for a batch and for a single token.
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ops-sparse_amd"))

import torch

from ops_sparse import combine, grouped_mm, grouped_mm_scaled, route


def layer(x, gate, w_in, w_out, k):
    """x [T, W] -> [T, W]: each token through the k experts that its router gives the largest logits."""
    weights, _, plan = route(x.float() @ gate.float().T, k)
    hidden = torch.nn.functional.silu(grouped_mm(x, w_in, plan, gather=True))
    return combine(grouped_mm(hidden, w_out, plan), plan, weights)


def to_8_bits(m):
    """Integers and the scale of each row (of each token, or of each expert's output channel)."""
    scale = (m.float().abs().amax(-1) / 127).clamp_min(1e-12)
    return (m.float() / scale.unsqueeze(-1)).round().to(torch.int8), scale


def layer_8_bits(x, gate, w_in, w_out, k):
    """:func:`layer` for serving; w_in and w_out as :func:`to_8_bits` gives them."""
    weights, _, plan = route(x.float() @ gate.float().T, k)
    hidden = grouped_mm_scaled(*to_8_bits(x), *w_in, plan, gather=True, out_dtype=x.dtype)
    hidden = torch.nn.functional.silu(hidden)
    return combine(grouped_mm_scaled(*to_8_bits(hidden), *w_out, plan, out_dtype=x.dtype), plan, weights)


def weights_of(experts, width, hidden, seed, dtype=torch.bfloat16, device="cuda"):
    """Random (gate, w_in, w_out) of a layer."""
    g = torch.Generator(device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device) * shape[-1] ** -0.5

    return normal(experts, width), normal(experts, hidden, width).to(dtype), normal(experts, width, hidden).to(dtype)


def train(x, target, parameters, k, steps, rate):
    """Plain gradient descent on the mean squared error; the losses of its steps."""
    parameters = [p.requires_grad_() for p in parameters]
    losses = []
    for _ in range(steps):
        loss = (layer(x, *parameters, k).float() - target).square().mean()
        grads = torch.autograd.grad(loss, parameters)
        with torch.no_grad():
            for p, g in zip(parameters, grads):
                p -= rate * g
        losses.append(loss.detach())
    for p in parameters:
        p.requires_grad_(False)
    return torch.stack(losses).tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 4096), ("experts", 32), ("chosen", 4), ("width", 1024), ("hidden", 2048),
                        ("steps", 30)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--rate", type=float, default=30.0)
    a = ap.parse_args(argv)
    x = torch.randn(a.tokens, a.width, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).bfloat16()
    teacher = weights_of(a.experts, a.width, a.hidden, 1)
    start = weights_of(a.experts, a.width, a.hidden, 1)
    start = [start[0]] + [w + 0.5 * v for w, v in zip(start[1:], weights_of(a.experts, a.width, a.hidden, 2)[1:])]
    target = layer(x, *teacher, a.chosen).float()
    losses = train(x, target, start, a.chosen, a.steps, a.rate)
    print(f"loss {losses[0]:.5f} -> {losses[-1]:.5f} in {a.steps} steps")
    gate, w_in, w_out = start
    w_in8, w_out8 = to_8_bits(w_in), to_8_bits(w_out)
    for name, batch in (("batch", x), ("one token", x[:1])):
        results = {}
        for bits, call in ((16, lambda: layer(batch, gate, w_in, w_out, a.chosen)),
                           (8, lambda: layer_8_bits(batch, gate, w_in8, w_out8, a.chosen))):
            for _ in range(3):
                call()
            torch.cuda.synchronize()
            begin = time.perf_counter()
            for _ in range(10):
                results[bits] = call()
            torch.cuda.synchronize()
            print(f"{name}, {bits} bits: {(time.perf_counter() - begin) * 1e5:.0f} us")
        error = (results[8].float() - results[16].float()).norm() / results[16].float().norm()
        print(f"{name}: 8 bits differ by {error:.4f} of the norm")


if __name__ == "__main__":
    main()
