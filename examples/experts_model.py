"""A small model of one layer of experts: trained on the log probabilities of tokens, then served in 4 bits.

    python examples/experts_model.py [--tokens 2048] [--vocabulary 8192] [--experts 16] [--chosen 2] [--width 512]

Each step asks for the log probability of every token's successor (with a small bonus on the entropy), takes the
gradient, and makes an AdamW step with 8-bit moments, clipped by the gradient's norm on the device.  The experts'
weights are then laid out in microscaled 4 bits once, and an answer's token is reported with its alternatives.
"""
import argparse
import os
import sys

sys.path[:0] = [os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ops-sparse_amd"),
                os.path.dirname(os.path.abspath(__file__))]

import torch

from experts_layer import layer, weights_of
from ops_sparse import (adamw_state, adamw_step, combine, grouped_mm_mx4, mx4_quantize, route, token_logprobs)


def parameters_of(vocabulary, experts, width, hidden, seed, dtype=torch.bfloat16, device="cuda"):
    """(embedding, gate, w_in, w_out, head), random."""
    g = torch.Generator(device).manual_seed(seed)
    embedding = torch.randn(vocabulary, width, generator=g, device=device).to(dtype)
    head = (torch.randn(vocabulary, width, generator=g, device=device) * width ** -0.5).to(dtype)
    return [embedding, *weights_of(experts, width, hidden, seed + 1, dtype, device), head]


def logits_of(tokens, parameters, k):
    """Logits [T, V] of what follows each token."""
    embedding, gate, w_in, w_out, head = parameters
    x = embedding[tokens]
    return (x + layer(x, gate, w_in, w_out, k)) @ head.T


def loss_of(tokens, targets, parameters, k, bonus):
    """Mean negative log probability of the targets (those outside the vocabulary left out), less the entropies'
    bonus."""
    logits = logits_of(tokens, parameters, k)
    r = token_logprobs(logits, targets, entropy=True)
    count = ((targets >= 0) & (targets < logits.shape[1])).sum()
    return -(r.logprobs.sum() / count + bonus * r.entropy.mean())


def train(tokens, targets, parameters, k, steps, rate, bonus=1e-3, bits=8, clip=1.0):
    """AdamW in place; the losses of its steps."""
    state = adamw_state(parameters, bits=bits, seed=1)
    losses = []
    for p in parameters:
        p.requires_grad_()
    for _ in range(steps):
        loss = loss_of(tokens, targets, parameters, k, bonus)
        grads = torch.autograd.grad(loss, parameters)
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
        adamw_step(parameters, grads, state, rate, grad_scale=(clip / (norm + 1e-6)).clamp(max=1.0))
        losses.append(loss.detach())
    for p in parameters:
        p.requires_grad_(False)
    return torch.stack(losses).tolist()


def layer_4_bits(x, gate, w_in, w_out, k):
    """The layer for serving; w_in and w_out as mx4_quantize gives them."""
    weights, _, plan = route(x.float() @ gate.float().T, k)
    hidden = torch.nn.functional.silu(grouped_mm_mx4(mx4_quantize(x), w_in, plan, gather=True, out_dtype=x.dtype))
    return combine(grouped_mm_mx4(mx4_quantize(hidden), w_out, plan, out_dtype=x.dtype), plan, weights)


def answer(tokens, parameters, served, k, top):
    """What follows each token in 4 bits: the likeliest, and the alternatives with their log probabilities."""
    embedding, gate, _, _, head = parameters
    x = embedding[tokens]
    logits = (x + layer_4_bits(x, gate, *served, k)) @ head.T
    return token_logprobs(logits, logits.argmax(1), top=top)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 2048), ("vocabulary", 8192), ("experts", 16), ("chosen", 2), ("width", 512),
                        ("hidden", 1024), ("steps", 20), ("top", 3)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--rate", type=float, default=1e-3)
    a = ap.parse_args(argv)
    g = torch.Generator("cuda").manual_seed(0)
    tokens = torch.randint(0, a.vocabulary, (a.tokens,), generator=g, device="cuda")
    targets = torch.randint(0, a.vocabulary, (a.vocabulary,), generator=g, device="cuda")[tokens]
    targets[::17] = -100  # the ends of sequences have no successor
    parameters = parameters_of(a.vocabulary, a.experts, a.width, a.hidden, 1)
    losses = train(tokens, targets, parameters, a.chosen, a.steps, a.rate)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    served = [mx4_quantize(w) for w in parameters[2:4]]
    r = answer(tokens[:1], parameters, served, a.chosen, a.top)
    print(f"in 4 bits, after token {int(tokens[0])}:",
          ", ".join(f"{i} ({p:.3f})" for i, p in zip(r.top_ids[0].tolist(), r.top_logprobs[0].tolist())))


if __name__ == "__main__":
    main()
