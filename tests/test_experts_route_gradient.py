"""The router's gradient entry by entry, within a bound of each entry's own size.

dl_e = p_e (g_e - sum_i w_i g_i), g_e = 0 off the chosen; p is the softmax over the row, or over the chosen with
`normalize`.  In fp32 p_e and the w_i are off by at most (experts + 30) roundings of themselves (exp of an argument
that is rounded, |argument| < 16; the sum; the division), the sum over i by k more of sum_i w_i |g_i|, and the
difference and the product by one each: together under 2 * (experts + 60) * 2^-24 of p_e (|g_e| + sum_i w_i |g_i|).
The result is rounded once to its type (2^-p of itself; float16 below its normal range by up to 2^-25).
"""
import pytest
import torch

from ops_sparse import route

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
SIZES = [(1, 1, 1), (3, 64, 8), (7, 60, 4), (65, 129, 2), (50, 1000, 64), (40, 257, 5), (300, 16, 2), (9, 1024, 1)]


def inputs(tokens, experts, k, dtype):
    """(logits, gradient of the weights, the choice) on the CPU."""
    g = torch.Generator().manual_seed(tokens + experts)
    logits = torch.randn(tokens, experts, generator=g).to(dtype)
    if tokens > 5 and experts > 8:
        logits[1, min(3, k):] = -float("inf")  # fewer than k experts left, unless k is small
        logits[2] = -float("inf")              # none left
    ids = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k]
    ids = torch.where(logits.float().gather(1, ids) == -float("inf"), -1, ids)
    return logits, torch.randn(tokens, k, generator=g), ids


def gradient(logits, grad, ids, normalize):
    """(p, g, dot, sum_i w_i |g_i|) in float64: the gradient is p * (g - dot)."""
    l, used = logits.double(), ids >= 0
    rows = torch.arange(len(l))[:, None].expand_as(ids)[used]
    g, chosen = torch.zeros_like(l), torch.zeros(l.shape, dtype=torch.bool)
    g[rows, ids[used]] = grad.double()[used]
    chosen[rows, ids[used]] = True
    if normalize:
        l = l.masked_fill(~chosen, -float("inf"))
    p = torch.softmax(l, 1).nan_to_num(0.0)  # rows without a finite logit have no weights
    return p, g, (p * g).sum(1, keepdim=True), (p * g.abs()).sum(1, keepdim=True)


def bound(p, g, dot, size, dtype):
    want = p * (g - dot)
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    return U[dtype] * want.abs() + 2 * (p.shape[1] + 60) * 2.0**-24 * p * (g.abs() + size) + tiny


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,experts,k", SIZES)
def test_the_bound_tells_wrong_gradients(tokens, experts, k, dtype, normalize):
    logits, grad, ids = inputs(tokens, experts, k, dtype)
    p, g, dot, size = gradient(logits, grad, ids, normalize)
    want, limit = p * (g - dot), bound(p, g, dot, size, dtype)
    for name, wrong in (("zero", torch.zeros_like(want)), ("no sum", p * g), ("sum's sign", p * (g + dot)),
                        ("zero off the chosen", torch.where(g == 0, 0.0, want))):
        off = (wrong - want).abs()
        differs = off > 1e-9 * p * (g.abs() + size)
        if differs.any():
            assert float((off > limit)[differs].double().mean()) > 0.8, name


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,experts,k", SIZES)
def test_route_gradient_by_entry(dev, tokens, experts, k, dtype, normalize):
    logits, grad, ids = inputs(tokens, experts, k, dtype)
    leaf = logits.to(dev).requires_grad_(True)
    weights, got_ids, _ = route(leaf, k, normalize=normalize)
    assert torch.equal(got_ids.cpu().long(), ids)
    got, = torch.autograd.grad(weights, leaf, grad.to(dev))
    p, g, dot, size = gradient(logits, grad, ids, normalize)
    err = (got.cpu().double() - p * (g - dot)).abs()
    limit = bound(p, g, dot, size, dtype)
    assert got.dtype == dtype and bool((err <= limit).all()), float((err / limit.clamp_min(1e-300)).max())
