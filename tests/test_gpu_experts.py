"""The experts' operators on the GPU against plain implementations in 64 bits.

Tolerances follow from the arithmetic: a sum of n products in fp32 is off by at most (n + 1) * 2^-24 times the sum of
the products' magnitudes, and the result is rounded once to a type of p significant bits (2^-p relative, 2^-11 for
float16 and 2^-8 for bfloat16; float16 results below its normal range by up to 2^-25).  Integers are exact.
"""
import numpy as np
import pytest
import torch

from ops_sparse import ExpertPlan, combine, expert_plan, grouped_mm, grouped_mm_scaled, route

pytestmark = pytest.mark.gpu

U32 = 2.0**-24
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: U32}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def close(got, want, magnitude, terms):
    """got against want (float64), a sum of `terms` products whose magnitudes sum to `magnitude`."""
    assert got.shape == want.shape
    bound = U[got.dtype] * want.abs() + (terms + 1) * U32 * magnitude * (1 + U[got.dtype]) + 2.0**-25
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst by {float((err / bound).max()):.3g} bounds"


def gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def lengths_to_plan(lens, tail=0, tokens=None, seed=0):
    """offsets of the given lengths, and `tail` rows past the last group; with tokens, a drawn gather index."""
    off = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    rows = int(off[-1]) + tail
    idx = None
    if tokens is not None:
        idx = torch.randint(0, tokens, (rows,), generator=gen(seed), device="cuda", dtype=torch.int32)
        if tail:
            idx[-tail:] = -1
    return ExpertPlan(off, idx, None), rows


def strided(shape, dtype, seed, pad, scale=1.0, offset=0):
    """Random values in rows longer than they need be, NaN (or -128) between them."""
    full = list(shape[:-1]) + [shape[-1] + pad]
    n = int(np.prod(full)) + offset
    if dtype == torch.int8:
        buf = torch.full((n,), -128, dtype=dtype, device="cuda")
        v = torch.randint(-127, 128, shape, generator=gen(seed), device="cuda", dtype=torch.int8)
    else:
        buf = torch.full((n,), float("nan"), dtype=dtype, device="cuda")
        v = (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)
    view = buf[offset:].view(full)[..., :shape[-1]]
    view.copy_(v)
    return view


# ------------------------------------------------------------------------------------------------------- routing


def plain_route(logits, k, normalize):
    """(weights, ids) of CPU logits in float64, one row at a time."""
    l = logits.double().cpu().numpy()
    t, e = l.shape
    w, ids = np.zeros((t, k)), np.full((t, k), -1, np.int64)
    for r in range(t):
        order = sorted((i for i in range(e) if l[r, i] != -np.inf), key=lambda i: (-l[r, i], i))[:k]
        if not order:
            continue
        top = l[r, order[0]]
        total = sum(np.exp(l[r, i] - top) for i in (order if normalize else range(e)))
        for j, i in enumerate(order):
            ids[r, j], w[r, j] = i, np.exp(l[r, i] - top) / total
    return w, ids


def plain_plan(ids, experts):
    flat = ids.reshape(-1)
    keep = (flat >= 0) & (flat < experts)
    order = np.argsort(np.where(keep, flat, experts), kind="stable")[:int(keep.sum())]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[keep], minlength=experts))])
    tokens = np.full(flat.size, -1, np.int64)
    tokens[:order.size] = order // ids.shape[1]
    places = np.full(flat.size, -1, np.int64)
    places[order] = np.arange(order.size)
    return offsets, tokens, places.reshape(ids.shape)


def check_plan(plan, ids, experts):
    offsets, tokens, places = plain_plan(ids, experts)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.places.cpu().numpy(), places)
    assert np.array_equal(plan.tokens.cpu().numpy(), tokens)


def check_weights(got, want, terms):
    # exp to 2 ulp of an argument rounded in 32 bits (|argument| * 2^-24), the sum, and the division
    err = (got.double().cpu() - torch.from_numpy(want)).abs()
    bound = torch.from_numpy(want) * (terms + 40) * 2 * U32 + 1e-38
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 64, 8), (2, 4, 4), (7, 60, 4), (33, 128, 8), (65, 129, 2),
                                              (200, 257, 6), (130, 1000, 64), (17, 64, 64), (2100, 16, 2),
                                              (9000, 96, 3)])
def test_route(dev, tokens, experts, k, dtype, normalize):
    logits = (torch.randn(tokens, experts, generator=gen(tokens + experts), device=dev) * 2).to(dtype)
    weights, ids, plan = route(logits, k, normalize=normalize)
    w, want = plain_route(logits, k, normalize)
    assert np.array_equal(ids.cpu().numpy(), want)
    check_weights(weights, w, experts)
    check_plan(plan, want, experts)


def test_route_ties_masks_and_strides(dev):
    inf = float("inf")
    lowest = float(torch.finfo(F32).min)
    rows = torch.tensor([[1.0, 1.0, 1.0, 1.0, 1.0], [-inf] * 5, [-inf, 2.0, -inf, -inf, 2.0],
                         [lowest] * 5, [lowest, 0.0, lowest, -inf, lowest], [0.0, -0.0, 0.0, -0.0, -1.0],
                         [3e38, -3e38, 3e38, 1.0, 2.0]], device=dev)
    for normalize in (True, False):
        buf = torch.full((7, 9), 1e30, device=dev)
        view = buf[:, 2:7]
        view.copy_(rows)
        weights, ids, plan = route(view, 3, normalize=normalize)
        w, want = plain_route(rows, 3, normalize)
        assert np.array_equal(ids.cpu().numpy(), want)
        assert np.array_equal(want[1], [-1, -1, -1]) and np.array_equal(want[2], [1, 4, -1])
        check_weights(weights, w, 5)
        assert weights[1].abs().max() == 0
        check_plan(plan, want, 5)


def test_route_nan_and_infinity_stay_in_their_row(dev):
    logits = torch.zeros(4, 6, device=dev)
    logits[1, 3] = float("nan")
    logits[2, 5] = float("inf")
    weights, ids, _ = route(logits, 2)
    assert ids.cpu().tolist() == [[0, 1], [3, 0], [5, 0], [0, 1]]
    assert weights[1].isnan().all() and weights[2, 0].isnan()
    assert weights[0].tolist() == [0.5, 0.5] and weights[3].tolist() == [0.5, 0.5]


def test_route_no_tokens(dev):
    weights, ids, plan = route(torch.empty(0, 8, device=dev), 2)
    assert weights.shape == (0, 2) and ids.shape == (0, 2) and plan.places.shape == (0, 2)
    assert plan.offsets.cpu().tolist() == [0] * 9


@pytest.mark.parametrize("tokens,experts,k", [(1, 3, 1), (5, 8, 3), (1000, 70, 4), (20000, 1024, 2), (300, 2, 2)])
def test_expert_plan_with_dropped_assignments(dev, tokens, experts, k):
    ids = torch.randint(-2, experts + 2, (tokens, k), generator=gen(k), device=dev, dtype=torch.int32)
    check_plan(expert_plan(ids, experts), ids.cpu().numpy().astype(np.int64), experts)


def test_expert_plan_of_one_expert(dev):
    ids = torch.full((3000, 2), 5, dtype=torch.int32, device=dev)
    check_plan(expert_plan(ids, 9), ids.cpu().numpy().astype(np.int64), 9)


def plain_route_grad(logits, ids, grad, normalize):
    """The softmax's gradient in float64 by autograd on the CPU, for the given choice."""
    l = logits.detach().double().cpu().requires_grad_(True)
    chosen = torch.zeros(l.shape, dtype=torch.bool)
    safe = torch.where(ids < 0, 0, ids).long()
    for r, row in enumerate(ids.tolist()):
        chosen[r, [i for i in row if i >= 0]] = True
    base = l.masked_fill(~chosen, -float("inf")) if normalize else l
    empty = (ids < 0).all(1, keepdim=True)
    p = torch.softmax(torch.where(empty, torch.zeros_like(base), base), 1)
    w = torch.where(ids < 0, torch.zeros_like(grad), p.gather(1, safe))
    (w * grad).sum().backward()
    return torch.where(empty, torch.zeros_like(l), l.grad)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (3, 64, 8), (7, 60, 4), (65, 129, 2), (50, 1000, 64)])
def test_route_gradient(dev, tokens, experts, k, dtype, normalize):
    logits = torch.randn(tokens, experts, generator=gen(1), device=dev).to(dtype)
    if tokens > 5 and experts > 8:
        logits[1, 3:] = -float("inf")   # fewer than k experts left
        logits[2] = -float("inf")       # none left
    logits.requires_grad_(True)
    weights, ids, _ = route(logits, k, normalize=normalize)
    grad = torch.randn(tokens, k, generator=gen(2), device=dev)
    got, = torch.autograd.grad(weights, logits, grad)
    want = plain_route_grad(logits, ids.cpu().long(), grad.double().cpu(), normalize)
    # p (g - sum): a few roundings of each factor, each relative to max |g| times p
    p = weights.detach().double().cpu().max() if normalize else 1.0
    bound = U[dtype] * want.abs() + (experts + 60) * 2 * U32 * float(grad.abs().max()) * k * float(p) + 2.0**-25
    assert got.dtype == dtype and bool(((got.double().cpu() - want).abs() <= bound).all())


def test_route_gradient_against_differences(dev):
    logits = torch.randn(4, 12, generator=gen(3), device=dev).requires_grad_(True)
    grad = torch.randn(4, 3, generator=gen(4), device=dev)
    for normalize in (True, False):
        weights, ids, _ = route(logits, 3, normalize=normalize)
        got, = torch.autograd.grad(weights, logits, grad)
        step = 2.0**-7
        for t, e in ((0, int(ids[0, 0])), (1, int(ids[1, 2])), (2, 5), (3, 0)):
            moved = []
            for s in (step, -step):
                l = logits.detach().clone()
                l[t, e] += s
                w, i, _ = route(l, 3, normalize=normalize)
                moved.append(float((w.double() * grad.double()).sum()) if torch.equal(i, ids) else None)
            if None in moved:
                continue  # the choice itself changed
            # third derivatives of a softmax are below 1; rounding 2^-22 over the step
            bound = step**2 * float(grad.abs().sum()) + 2.0**-20 / step * float(grad.abs().sum())
            assert abs((moved[0] - moved[1]) / (2 * step) - float(got[t, e])) <= bound


# ------------------------------------------------------------------------------------------------------- products


def plain_grouped(a, w, plan, rows):
    """(y, magnitudes) in float64."""
    off = plan.offsets.tolist()
    y = torch.zeros(rows, w.shape[1], dtype=torch.float64, device="cuda")
    m = torch.zeros_like(y)
    for e in range(w.shape[0]):
        lo, hi = off[e], off[e + 1]
        if lo < hi and a.shape[1]:
            r = a[plan.tokens[lo:hi].long()] if plan.tokens is not None else a[lo:hi]
            y[lo:hi] = r.double() @ w[e].double().t()
            m[lo:hi] = r.double().abs() @ w[e].double().abs().t()
    return y, m


GROUPS = {
    "one": [1], "one_of_many": [0, 0, 1, 0], "empty": [0, 0, 0], "single_rows": [1, 1, 0, 1, 1],
    "ragged": [5, 0, 17, 64, 1, 33], "tile_ends": [64, 128, 16, 256, 32, 0], "over": [65, 129, 17, 257],
    "many": [(i * 7) % 5 for i in range(130)], "long": [700, 3, 1100, 0, 260],
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (64, 64), (65, 33), (256, 264), (300, 40), (520, 1032), (40, 2048),
                                 (129, 1001)])
@pytest.mark.parametrize("groups", list(GROUPS))
def test_grouped_mm(dev, groups, n, k, dtype):
    lens = GROUPS[groups]
    gather = (n + k + len(lens)) % 2 == 0
    tokens = 97
    plan, rows = lengths_to_plan(lens, tail=3, tokens=tokens if gather else None)
    a = torch.randn(tokens if gather else rows, k, generator=gen(1), device=dev).to(dtype)
    w = torch.randn(len(lens), n, k, generator=gen(2), device=dev).to(dtype)
    y = grouped_mm(a, w, plan, gather=gather)
    want, magnitude = plain_grouped(a, w, plan, rows)
    close(y, want, magnitude, k)
    assert not y[rows - 3:].any()


@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (1, 0), (0, 1), (24, 8), (3, 5)])
@pytest.mark.parametrize("groups", ["ragged", "long", "single_rows"])
def test_grouped_mm_strides_and_alignment(dev, groups, pad, offset):
    lens = GROUPS[groups]
    plan, rows = lengths_to_plan(lens, tokens=50)
    a = strided((50, 136), BF16, 1, pad, offset=offset)
    w = strided((len(lens), 72, 136), BF16, 2, pad, offset=offset)
    want, magnitude = plain_grouped(a, w, plan, rows)
    close(grouped_mm(a, w, plan, gather=True), want, magnitude, 136)
    # every other expert of a larger tensor, and columns of it that are not contiguous
    big = strided((2 * len(lens), 72, 136), BF16, 3, pad, offset=offset)
    close(grouped_mm(a, big[::2], plan, gather=True), *plain_grouped(a, big[::2], plan, rows), 136)
    turned = strided((len(lens), 136, 72), BF16, 4, pad).transpose(1, 2)
    close(grouped_mm(a, turned, plan, gather=True), *plain_grouped(a, turned, plan, rows), 136)


def test_grouped_mm_no_rows_no_width(dev):
    plan, _ = lengths_to_plan([0, 0])
    w = torch.ones(2, 16, 8, dtype=F16, device=dev)
    assert grouped_mm(torch.empty(0, 8, dtype=F16, device=dev), w, plan).shape == (0, 16)
    plan, rows = lengths_to_plan([2, 1])
    y = grouped_mm(torch.empty(3, 0, dtype=F16, device=dev), w[:, :, :0], plan)
    assert y.shape == (3, 16) and not y.any()
    assert grouped_mm(torch.ones(3, 8, dtype=F16, device=dev), w[:, :0], plan).shape == (3, 0)


@pytest.mark.parametrize("k", [64, 72, 1000, 33])
def test_grouped_mm_non_finite_values_stay_in_their_rows(dev, k):
    lens = [20, 70, 3]
    plan, rows = lengths_to_plan(lens)
    a = torch.randn(rows, k, generator=gen(1), device=dev).to(BF16)
    w = torch.randn(3, 48, k, generator=gen(2), device=dev).to(BF16)
    clean = grouped_mm(a, w, plan)
    dirty = a.clone()
    dirty[19, k - 1] = float("nan")   # the last row of a group, next to another's first
    dirty[92, 0] = float("inf")
    wd = w.clone()
    wd[1, 7] = float("nan")
    y = grouped_mm(dirty, wd, plan)
    assert y[19].isnan().all() and not y[92].isfinite().any() and y[20:90, 7].isnan().all()
    keep = torch.ones(rows, 48, dtype=torch.bool, device=dev)
    keep[19] = keep[92] = False
    keep[20:90, 7] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("offsets", [[0, 40, 20, 60], [0, -5, 70, 1 << 30], [3, 3, 3, 3], [50, 40, 30, 20]])
def test_grouped_mm_offsets_without_meaning_stay_in_bounds(dev, offsets):
    off = torch.tensor(offsets, dtype=torch.int32, device=dev)
    tokens = torch.full((60,), 1 << 20, dtype=torch.int32, device=dev)
    a = torch.ones(60, 64, dtype=F16, device=dev, requires_grad=True)
    w = torch.ones(3, 64, 64, dtype=F16, device=dev, requires_grad=True)
    y = grouped_mm(a.detach(), w, ExpertPlan(off, tokens, None), gather=True)
    assert y.shape == (60, 64)
    dw, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert dw.shape == w.shape
    torch.cuda.synchronize()


def plain_grads(a, w, plan, grad):
    """(da, its magnitudes, dw, its magnitudes) in float64."""
    off = plan.offsets.tolist()
    index = plan.tokens.long() if plan.tokens is not None else torch.arange(a.shape[0], device="cuda")
    da, dw = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (a, w))
    ma, mw = torch.zeros_like(da), torch.zeros_like(dw)
    for e in range(w.shape[0]):
        s = slice(off[e], off[e + 1])
        if s.start < s.stop:
            g, x, b = grad[s].double(), a[index[s]].double(), w[e].double()
            da.index_add_(0, index[s], g @ b)
            ma.index_add_(0, index[s], g.abs() @ b.abs())
            dw[e], mw[e] = g.t() @ x, g.abs().t() @ x.abs()
    return da, ma, dw, mw


def routed(tokens, experts, k, seed, drop=0.0, taken=None):
    ids = torch.stack([torch.randperm(taken or experts, generator=gen(seed * 1000 + t, "cpu"))[:k]
                       for t in range(tokens)]).to(torch.int32)
    ids[torch.rand(tokens, k, generator=gen(seed, "cpu")) < drop] = -1
    return ids.cuda()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,experts,k,n,width,drop", [
    (1, 4, 2, 64, 64, 0.0), (9, 8, 3, 40, 72, 0.3), (70, 5, 2, 129, 33, 0.0), (300, 6, 2, 264, 520, 0.1),
    (513, 3, 3, 256, 256, 0.0), (40, 100, 4, 96, 128, 0.0), (700, 2, 1, 72, 1000, 0.5), (12, 3, 1, 64, 64, 1.0)])
def test_grouped_mm_gradients(dev, tokens, experts, k, n, width, drop, dtype):
    plan = expert_plan(routed(tokens, experts, k, 5, drop, taken=max(experts - 1, k)), experts)
    a = torch.randn(tokens, width, generator=gen(1), device=dev).to(dtype).requires_grad_(True)
    w = torch.randn(experts, n, width, generator=gen(2), device=dev).to(dtype).requires_grad_(True)
    y = grouped_mm(a, w, plan, gather=True)
    grad = torch.randn(y.shape, generator=gen(3), device=dev).to(dtype)
    da, dw = torch.autograd.grad(y, (a, w), grad)
    wa, ma, ww, mw = plain_grads(a.detach(), w.detach(), plan, grad)
    close(da, wa, ma, n + k)
    close(dw, ww, mw, tokens)
    assert not dw[experts - 1].any() or experts == k  # an expert that nobody chose


@pytest.mark.parametrize("n,width", [(64, 64), (129, 65), (256, 320)])
@pytest.mark.parametrize("groups", ["one_of_many", "ragged", "tile_ends", "over", "many", "long"])
def test_grouped_mm_gradients_without_gather(dev, groups, n, width):
    lens = GROUPS[groups]
    plan, rows = lengths_to_plan(lens)
    a = torch.randn(rows, width, generator=gen(1), device=dev).to(BF16).requires_grad_(True)
    w = torch.randn(len(lens), n, width, generator=gen(2), device=dev).to(BF16).requires_grad_(True)
    y = grouped_mm(a, w, plan)
    grad = torch.randn(y.shape, generator=gen(3), device=dev).to(BF16)
    da, dw = torch.autograd.grad(y, (a, w), grad)
    wa, ma, ww, mw = plain_grads(a.detach(), w.detach(), plan, grad)
    close(da, wa, ma, n)
    close(dw, ww, mw, max(lens))


def test_grouped_mm_gradients_of_strided_and_broadcast_inputs(dev):
    lens = [30, 0, 100]
    plan, rows = lengths_to_plan(lens)
    a = strided((rows, 72), BF16, 1, 9).requires_grad_(True)
    shared = torch.randn(1, 40, 72, generator=gen(2), device=dev).to(BF16).requires_grad_(True)
    y = grouped_mm(a, shared.expand(3, 40, 72), plan)
    grad = torch.randn(40, generator=gen(3), device=dev).to(BF16).expand(rows, 40)
    da, dw = torch.autograd.grad(y, (a, shared), grad)
    wa, ma, ww, mw = plain_grads(a.detach(), shared.detach().expand(3, 40, 72), plan, grad)
    close(da, wa, ma, 40)
    # each expert's part is rounded before torch adds them over the broadcast
    bound = BF16_SUM * ww.abs().sum(0) + (rows + 1) * U32 * mw.sum(0) * 2 + 2 * BF16_SUM * ww.sum(0).abs() + 2.0**-25
    assert bool(((dw[0].double() - ww.sum(0)).abs() <= bound).all())


BF16_SUM = 2.0**-8


def test_grouped_mm_gradient_against_differences(dev):
    plan = expert_plan(routed(12, 3, 2, 1), 3)
    a = torch.randn(12, 24, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    w = torch.randn(3, 16, 24, generator=gen(2), device=dev).to(F16).requires_grad_(True)
    c = torch.randn(24, 16, generator=gen(3), device=dev).to(F16)
    y = grouped_mm(a, w, plan, gather=True)
    da, dw = torch.autograd.grad(y, (a, w), c)
    # the product is linear in each input: differences are exact up to y's rounding
    for t, grad, at in ((a, da, (3, 5)), (a, da, (11, 23)), (w, dw, (0, 2, 7)), (w, dw, (2, 15, 0))):
        value, outs = float(t[at].detach()), []
        for v in (value + 1.0, value - 1.0):
            moved = t.detach().clone()
            moved[at] = v
            args = (moved, w.detach()) if t is a else (a.detach(), moved)
            outs.append((float(moved[at]), (grouped_mm(*args, plan, gather=True).double() * c.double()).sum()))
        slope = float(outs[0][1] - outs[1][1]) / (outs[0][0] - outs[1][0])
        rounding = 2.0**-11 * float((y.detach().double().abs() * c.double().abs()).sum() + 24 * 50)
        assert abs(slope - float(grad[at])) <= rounding


# Sizes that reach the 256x256 tiles: whole ones, ends of every height, a last round cut in slices, a tail.
LARGE = {
    "whole": [1024, 2048], "ends": [256 + 64, 512 + 1, 768 + 128, 1024 + 129, 255, 257], "one": [3333],
    "skewed": [2600, 0, 300, 64, 7], "few_rounds": [256 * 21],
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,k", [(2304, 64), (2312, 136), (2200, 200), (2560, 512), (4100, 72)])
@pytest.mark.parametrize("groups", list(LARGE))
def test_grouped_mm_large_tiles(dev, groups, n, k, dtype):
    lens = LARGE[groups]
    gather = k % 16 == 8
    plan, rows = lengths_to_plan(lens, tail=70, tokens=900 if gather else None)
    a = torch.randn(900 if gather else rows, k, generator=gen(1), device=dev).to(dtype)
    w = torch.randn(len(lens), n, k, generator=gen(2), device=dev).to(dtype)
    y = grouped_mm(a, w, plan, gather=gather)
    want, magnitude = plain_grouped(a, w, plan, rows)
    close(y, want, magnitude, k)
    assert not y[rows - 70:].any()


@pytest.mark.parametrize("n,k", [(2304, 128), (2312, 144), (2200, 400), (2560, 1024), (4100, 80)])
@pytest.mark.parametrize("groups", list(LARGE))
def test_grouped_mm_scaled_large_tiles(dev, groups, n, k):
    lens = LARGE[groups]
    plan, rows = lengths_to_plan(lens, tail=5, tokens=500)
    a, w = strided((500, k), torch.int8, 1, 16), strided((len(lens), n, k), torch.int8, 2, 0)
    sa = torch.rand(500, generator=gen(3), device=dev) * 1e-3
    sw = torch.rand(len(lens), n, generator=gen(4), device=dev) * 1e-2
    y = grouped_mm_scaled(a, sa, w, sw, plan, gather=True)
    scaled_close(y, plain_scaled(a, sa, w, sw, plan, rows))
    assert not y[rows - 5:].any()


@pytest.mark.parametrize("groups,n,k", [
    ("whole", 256, 2304), ("ends", 264, 2200), ("one", 200, 2304), ("skewed", 136, 2312),  # gradient of the input
    ("ends", 1536, 1544), ("skewed", 1544, 2056),                       # weight gradients of 256x256
    ("ends", 520, 776), ("skewed", 776, 1032), ("skewed", 777, 1033),   # of 64x256
    ("few_rounds", 128, 264), ("few_rounds", 129, 263)])                # of 64x128 by three teams
def test_grouped_mm_gradients_large(dev, groups, n, k):
    lens = LARGE[groups] * (4 if n >= 1536 else 2 if n >= 520 else 1)
    plan, rows = lengths_to_plan(lens)
    tokens = rows // 2 if k % 16 == 8 else rows
    index = torch.randint(0, tokens, (rows,), generator=gen(7), device=dev, dtype=torch.int32)
    a = torch.randn(tokens, k, generator=gen(1), device=dev).to(BF16).requires_grad_(True)
    w = (torch.randn(len(lens), n, k, generator=gen(2), device=dev)).to(BF16).requires_grad_(True)
    grad = torch.randn(rows, n, generator=gen(3), device=dev).to(BF16)
    if tokens == rows:
        y = grouped_mm(a, w, plan)
        da, dw = torch.autograd.grad(y, (a, w), grad)
        wa, ma, ww, mw = plain_grads(a.detach(), w.detach(), plan, grad)
        close(da, wa, ma, n)
    else:
        # an index without places serves the weight gradient alone
        plan = ExpertPlan(plan.offsets, index, None)
        y = grouped_mm(a.detach(), w, plan, gather=True)
        dw, = torch.autograd.grad(y, w, grad)
        _, _, ww, mw = plain_grads(a.detach(), w.detach(), plan, grad)
    close(dw, ww, mw, max(lens))


@pytest.mark.parametrize("rows,n,k,groups", [
    (1, 64, 4096, 1), (17, 100, 2056, 1), (40, 72, 1544, 1), (64, 520, 776, 1),   # few rows, two heights
    (200, 136, 4104, 3), (300, 256, 1000, 2), (513, 1000, 2048, 1),               # teams
    (100, 136, 1001, 2), (513, 1000, 2047, 1)])                                   # and unaligned
def test_grouped_mm_long_contractions(dev, rows, n, k, groups):
    lens = [rows // groups] * groups
    plan, total = lengths_to_plan(lens)
    a = torch.randn(total, k, generator=gen(1), device=dev).to(F16)
    w = torch.randn(groups, n, k, generator=gen(2), device=dev).to(F16)
    close(grouped_mm(a, w, plan), *plain_grouped(a, w, plan, total), k)


def test_results_are_differentiable_once(dev):
    logits = torch.randn(4, 8, generator=gen(1), device=dev).requires_grad_(True)
    weights, _, _ = route(logits, 2)
    grad, = torch.autograd.grad((weights ** 2).sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.sum().backward()


def test_second_derivatives_with_respect_to_given_tensors_raise(dev):
    # the engine runs the nodes on the way to these alone: the second derivative's has to be one of them
    plan = expert_plan(routed(6, 3, 2, 1), 3)
    x = torch.randn(6, 8, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    w = torch.randn(3, 8, 8, generator=gen(2), device=dev).to(F16).requires_grad_(True)
    y = torch.randn(12, 8, generator=gen(3), device=dev).to(F16).requires_grad_(True)
    weights = torch.rand(6, 2, generator=gen(4), device=dev).requires_grad_(True)
    logits = torch.randn(6, 3, generator=gen(5), device=dev).requires_grad_(True)
    for make, leaves in ((lambda: route(logits, 2)[0], (logits,)), (lambda: route(logits, 2, False)[0], (logits,)),
                         (lambda: grouped_mm(x, w, plan, gather=True), (x, w)),
                         (lambda: combine(y, plan, weights), (y, weights))):
        out = (make().float() ** 2).sum()
        grads = torch.autograd.grad(out, leaves, create_graph=True)
        for g in grads:
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad((g.float() ** 2).sum() + out, leaves, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            sum((g.float() ** 2).sum() for g in grads).backward(retain_graph=True)


def test_forward_mode_is_refused(dev):
    plan = expert_plan(routed(6, 3, 2, 1), 3)
    x, w = torch.ones(6, 8, dtype=F16, device=dev), torch.ones(3, 8, 8, dtype=F16, device=dev)
    y, weights = torch.ones(12, 8, dtype=F16, device=dev), torch.ones(6, 2, device=dev)
    logits = torch.randn(6, 3, generator=gen(1), device=dev)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: route(dual(logits), 2), lambda: grouped_mm(dual(x), w, plan, gather=True),
                     lambda: grouped_mm(x, dual(w), plan, gather=True), lambda: combine(dual(y), plan),
                     lambda: combine(y, plan, dual(weights))):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        # and of a gradient: the tangent of what comes in
        for out, leaf in ((combine(y.requires_grad_(True), plan), y),
                          (grouped_mm(x.requires_grad_(True), w, plan, gather=True), x),
                          (route(logits.requires_grad_(True), 2)[0], logits)):
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(out, leaf, dual(torch.ones_like(out)))


# ------------------------------------------------------------------------------------------------------- 8 bits


def plain_scaled(a, sa, w, sw, plan, rows):
    off = plan.offsets.tolist()
    y = torch.zeros(rows, w.shape[1], dtype=torch.float64, device="cuda")
    index = plan.tokens.long() if plan.tokens is not None else torch.arange(rows, device="cuda")
    for e in range(w.shape[0]):
        s = slice(off[e], off[e + 1])
        if s.start < s.stop:
            y[s] = (a[index[s]].double() @ w[e].double().t()) * sa[index[s]].double()[:, None] * sw[e].double()
    return y


def scaled_close(got, want):
    # the integer sum is exact; its conversion to fp32, the product of the scales and the product with it round
    bound = (U[got.dtype] + 4 * U32) * want.abs() + 2.0**-25
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 16), (64, 128), (65, 33), (256, 272), (300, 48), (129, 1001), (512, 1040)])
@pytest.mark.parametrize("groups", list(GROUPS))
def test_grouped_mm_scaled(dev, groups, n, k, out):
    lens = GROUPS[groups]
    gather = (n + len(lens)) % 2 == 0
    plan, rows = lengths_to_plan(lens, tail=2, tokens=97 if gather else None)
    rows_a = 97 if gather else rows
    a = strided((rows_a, k), torch.int8, 1, 0)
    w = strided((len(lens), n, k), torch.int8, 2, 0)
    sa = torch.rand(rows_a, generator=gen(3), device=dev) * 1e-3
    sw = torch.rand(len(lens), n, generator=gen(4), device=dev) * 1e-2
    y = grouped_mm_scaled(a, sa, w, sw, plan, gather=gather, out_dtype=out)
    scaled_close(y, plain_scaled(a, sa, w, sw, plan, rows))
    assert not y[rows - 2:].any()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 64, 100, 300, 1000])
@pytest.mark.parametrize("n,k,pad", [(64, 64, 0), (1000, 528, 16), (520, 77, 3), (256, 4096, 0)])
def test_scaled_dense(dev, rows, n, k, pad):
    a, w = strided((rows, k), torch.int8, 1, pad), strided((n, k), torch.int8, 2, pad)
    sa = torch.rand(rows, generator=gen(3), device=dev)
    sw = torch.rand(n, generator=gen(4), device=dev) * 1e-4
    y = grouped_mm_scaled(a, sa, w, sw, out_dtype=F32)
    want = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    scaled_close(y, want)


def test_scaled_extremes(dev):
    # the largest magnitudes in the longest contraction: -128 * -128 * 131071 is just within 32 bits
    a = torch.full((3, 131071), -128, dtype=torch.int8, device=dev)
    w = torch.full((5, 131071), -128, dtype=torch.int8, device=dev)
    one = torch.ones(5, device=dev)
    y = grouped_mm_scaled(a, one[:3], w, one, out_dtype=F32)
    assert bool((y.double() == float(np.float32(131071 * 16384))).all())
    with pytest.raises(ValueError):
        grouped_mm_scaled(torch.zeros(1, 131072, dtype=torch.int8, device=dev), one[:1],
                          torch.zeros(5, 131072, dtype=torch.int8, device=dev), one)


@pytest.mark.parametrize("of", ["a_scale", "w_scale", "both"])
def test_scales_that_ask_for_a_gradient_get_an_error(dev, of):
    a, w = strided((5, 32), torch.int8, 1, 0), strided((8, 32), torch.int8, 2, 0)
    sa, sw = torch.rand(5, generator=gen(3), device=dev), torch.rand(8, generator=gen(4), device=dev)
    want = grouped_mm_scaled(a, sa, w, sw)
    asked = [s.requires_grad_(True) for s, name in ((sa, "a_scale"), (sw, "w_scale")) if of in (name, "both")]
    with torch.no_grad():
        y = grouped_mm_scaled(a, sa, w, sw)
        assert not y.requires_grad and torch.equal(y, want)
    y = grouped_mm_scaled(a, sa, w, sw)
    assert torch.equal(y.detach(), want)
    # beside a part that has a gradient, without which torch itself would raise
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(y.float().sum() + sum(s.sum() for s in asked), asked)


# ------------------------------------------------------------------------------------------------------- combination


def plain_combine(y, weights, places):
    safe = torch.where(places < 0, 0, places).long()
    rows = y.double()[safe] * (places >= 0)[:, :, None]
    w = weights.double() if weights is not None else torch.ones(places.shape, dtype=torch.float64, device="cuda")
    return (rows * w[:, :, None]).sum(1), (rows.abs() * w.abs()[:, :, None]).sum(1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("tokens,experts,k,width,drop", [
    (1, 4, 1, 1, 0.0), (5, 8, 3, 33, 0.0), (64, 16, 8, 2048, 0.0), (100, 9, 4, 264, 0.4), (31, 40, 33, 72, 0.1),
    (7, 3, 2, 5000, 0.0), (6, 3, 2, 4104, 1.0)])
def test_combine_and_its_gradients(dev, tokens, experts, k, width, drop, weighted, dtype):
    plan = expert_plan(routed(tokens, experts, k, 3, drop), experts)
    y = torch.randn(tokens * k, width, generator=gen(1), device=dev).to(dtype).requires_grad_(True)
    weights = torch.randn(tokens, k, generator=gen(2), device=dev).requires_grad_(True) if weighted else None
    out = combine(y, plan, weights)
    want, magnitude = plain_combine(y.detach(), weights.detach() if weighted else None, plan.places)
    close(out, want, magnitude, k)
    grad = torch.randn(tokens, width, generator=gen(4), device=dev).to(dtype)
    grads = torch.autograd.grad(out, (y, weights) if weighted else (y,), grad)
    places = plan.places
    wy = torch.zeros(y.shape, dtype=torch.float64, device=dev)
    w = weights.detach().double() if weighted else torch.ones(tokens, k, dtype=torch.float64, device=dev)
    used = places >= 0
    wy[places[used].long()] = (w[:, :, None] * grad.double()[:, None, :])[used]
    close(grads[0], wy, wy.abs(), 1)
    if weighted:
        rows = y.detach().double()[torch.where(used, places, 0).long()] * used[:, :, None]
        prod = rows * grad.double()[:, None, :]
        close(grads[1], prod.sum(2), prod.abs().sum(2), width)


@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 3)])
def test_combine_strides(dev, pad, offset):
    plan = expert_plan(routed(20, 6, 2, 3), 6)
    y = strided((40, 520), F16, 1, pad, offset=offset).requires_grad_(True)
    weights = torch.rand(2, 20, generator=gen(2), device=dev).t().requires_grad_(True)
    out = combine(y, plan, weights)
    close(out, *plain_combine(y.detach(), weights.detach(), plan.places), 2)
    dy, dw = torch.autograd.grad(out, (y, weights), torch.ones(1, 1, dtype=F16, device=dev).expand(20, 520))
    wy = torch.zeros(40, 520, dtype=torch.float64, device=dev)
    wy[plan.places.long()] = weights.detach().double()[:, :, None]
    close(dy, wy, wy, 1)
    rows = y.detach().double()[plan.places.long()]
    close(dw, rows.sum(2), rows.abs().sum(2), 520)


def test_combine_gradient_against_differences(dev):
    plan = expert_plan(routed(5, 4, 2, 3), 4)
    y = torch.randn(10, 16, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    weights = torch.rand(5, 2, generator=gen(2), device=dev).requires_grad_(True)
    c = torch.randn(5, 16, generator=gen(3), device=dev).to(F16)
    out = combine(y, plan, weights)
    dy, dw = torch.autograd.grad(out, (y, weights), c)
    for t, grad, at in ((y, dy, (2, 3)), (y, dy, (9, 15)), (weights, dw, (4, 1)), (weights, dw, (0, 0))):
        outs = []
        for s in (1.0, -1.0):
            moved = t.detach().clone()
            moved[at] += s
            args = (moved, plan, weights.detach()) if t is y else (y.detach(), plan, moved)
            outs.append((float(moved[at]), float((combine(*args).double() * c.double()).sum())))
        slope = (outs[0][1] - outs[1][1]) / (outs[0][0] - outs[1][0])
        rounding = 2.0**-11 * float((out.detach().double().abs() * c.double().abs()).sum() + 16 * 30)
        assert abs(slope - float(grad[at])) <= rounding


def any_places(kind, tokens, k):
    """(places, rows of y) that are no plan's: rows that no place names, and rows that several do."""
    count = tokens * k
    plan = expert_plan(routed(tokens, max(k, 7), k, 11), max(k, 7)).places.cpu()
    g = gen(12, "cpu")
    if kind == "dropped":  # a capacity limit on a finished plan
        return plan.masked_fill(torch.rand(plan.shape, generator=g) < 0.4, -1), count
    if kind == "all dropped":
        return torch.full_like(plan, -1), count
    if kind == "more rows":
        return plan * 3 + 1, 3 * count + 5
    if kind == "outside":  # past y's rows and before them
        return torch.where(torch.rand(plan.shape, generator=g) < 0.5, plan - 3, plan + count // 2), count
    if kind == "drawn":  # most rows by none, one or two, some by more
        return torch.randint(0, count, plan.shape, generator=g, dtype=torch.int32), count
    if kind == "one row":
        return torch.full_like(plan, 3), 5
    # two rows by as many as fit a wave, and by one more; the rest each by one
    flat = plan.reshape(-1).clone()
    order = torch.randperm(count, generator=g)
    flat[order[:64]], flat[order[64:129]] = 0, 1
    return flat.view(tokens, k), count


@pytest.mark.parametrize("kind", ["dropped", "all dropped", "more rows", "outside", "drawn", "one row", "a wave"])
@pytest.mark.parametrize("tokens,k,width,dtype", [(100, 2, 1, F16), (70, 3, 33, BF16), (65, 4, 264, F16),
                                                  (300, 8, 2056, BF16)])
def test_combine_gradients_of_any_places(dev, kind, tokens, k, width, dtype):
    places, rows = any_places(kind, tokens, k)
    plan = ExpertPlan(torch.tensor([0, 2], dtype=torch.int32, device=dev), None, places.to(dev))
    y = torch.randn(rows, width, generator=gen(1), device=dev).to(dtype).requires_grad_(True)
    weights = torch.randn(tokens, k, generator=gen(2), device=dev).requires_grad_(True)
    grad = torch.randn(tokens, width, generator=gen(4), device=dev).to(dtype)
    used = ((places >= 0) & (places < rows)).to(dev)
    safe = torch.where(used, plan.places, 0).long()
    for w in (weights, None):
        factor = (torch.ones(tokens, k, dtype=torch.float64, device=dev) if w is None else w.detach().double()) * used
        part = (factor[:, :, None] * grad.double()[:, None, :]).reshape(-1, width)
        want, magnitude = (torch.zeros(rows, width, dtype=torch.float64, device=dev)
                           .index_add_(0, safe.reshape(-1), t) for t in (part, part.abs()))
        most = int(torch.bincount(safe[used], minlength=1).max()) if used.any() else 1
        first = None
        for turn in range(3):
            # what the allocator hands out next is not zeros: values, and numbers of assignments
            left = [torch.full((rows, width), float("nan"), dtype=dtype, device=dev),
                    torch.randint(0, tokens * k, (rows + 16,), device=dev, dtype=torch.int32),
                    torch.randint(0, tokens * k, (rows + tokens * k + 32,), device=dev, dtype=torch.int32)]
            del left
            out = combine(y, plan, w)
            grads = torch.autograd.grad(out, (y,) if w is None else (y, w), grad)
            close(grads[0], want, magnitude, most)
            named = torch.zeros(rows, dtype=torch.bool, device=dev)
            named[safe[used]] = True
            assert not grads[0][~named].any()
            if w is not None:
                prod = y.detach().double()[safe] * used[:, :, None] * grad.double()[:, None, :]
                close(grads[1], prod.sum(2), prod.abs().sum(2), width)
            assert first is None or all(torch.equal(a, b) for a, b in zip(first, grads))
            first = grads


@pytest.mark.parametrize("tokens", [5, 400])
def test_layer_gradients_after_assignments_are_dropped(dev, tokens):
    # a capacity of 3 rows an expert, set on the finished plan: what is dropped has no part in any gradient
    experts, k, n, width = 6, 2, 72, 136
    full = expert_plan(routed(tokens, experts, k, 2), experts)
    expert = (full.places[:, :, None] >= full.offsets[1:]).sum(2)
    place = torch.where(full.places - full.offsets[expert] < 3, full.places, -1)
    plan = full._replace(places=place)
    x = torch.randn(tokens, width, generator=gen(1), device=dev).to(BF16).requires_grad_(True)
    w = torch.randn(experts, n, width, generator=gen(2), device=dev).to(BF16).requires_grad_(True)
    weights = torch.rand(tokens, k, generator=gen(3), device=dev)
    grad = torch.randn(tokens, n, generator=gen(4), device=dev).to(BF16)
    out = combine(grouped_mm(x, w, plan, gather=True), plan, weights)
    dx, dw = torch.autograd.grad(out, (x, w), grad)
    kept = (place >= 0).double() * weights.double()
    rows = torch.zeros(tokens * k, n, dtype=torch.float64, device=dev)
    rows[full.places.long()] = kept[:, :, None] * grad.double()[:, None, :]
    wx, mx, ww, mw = plain_grads(x.detach(), w.detach(), full, rows)
    # the rows' gradients are rounded to bfloat16 between the two operators
    for got, want, magnitude in ((dx, wx, mx), (dw, ww, mw)):
        bound = 2 * U[BF16] * want.abs() + (2 * U[BF16] + (n + tokens) * U32) * magnitude + 2.0**-25
        assert bool(((got.double() - want).abs() <= bound).all())


# ------------------------------------------------------------------------------------------------------- as a whole


def test_results_do_not_change_from_run_to_run(dev):
    logits = torch.randn(700, 32, generator=gen(1), device=dev).requires_grad_(True)
    x = torch.randn(700, 264, generator=gen(2), device=dev).to(BF16).requires_grad_(True)
    w = (torch.randn(32, 264, 264, generator=gen(3), device=dev) / 16).to(BF16).requires_grad_(True)

    def step():
        weights, _, plan = route(logits, 4)
        out = combine(grouped_mm(x, w, plan, gather=True), plan, weights)
        return (out.detach(),) + torch.autograd.grad(out, (logits, x, w), torch.ones_like(out))

    first = step()
    for _ in range(3):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)


def test_another_stream(dev):
    x = torch.randn(256, 512, generator=gen(2), device=dev).to(BF16)
    w = (torch.randn(8, 512, 512, generator=gen(3), device=dev) / 16).to(BF16)
    logits = torch.randn(256, 8, generator=gen(1), device=dev)
    weights, _, plan = route(logits, 2)
    want = combine(grouped_mm(x, w, plan, gather=True), plan, weights)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late = torch.zeros_like(x)
        late.copy_(x)      # the operands exist only once this stream has got here
        lw, _, lp = route(logits.clone(), 2)
        got = combine(grouped_mm(late, w, lp, gather=True), lp, lw)
    stream.synchronize()
    assert torch.equal(got, want)


def test_hip_graph_capture_and_replay(dev):
    x = torch.randn(48, 256, generator=gen(2), device=dev).to(F16)
    w = (torch.randn(8, 256, 256, generator=gen(3), device=dev) / 16).to(F16)
    logits = torch.randn(48, 8, generator=gen(1), device=dev)

    def layer():
        weights, _, plan = route(logits, 2)
        return combine(grouped_mm(x, w, plan, gather=True), plan, weights)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for seed in range(4):
        logits.copy_(torch.randn(48, 8, generator=gen(10 + seed), device=dev))
        x.copy_(torch.randn(48, 256, generator=gen(20 + seed), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer())


def layer_step(logits, x, w, v, k):
    """A layer and its gradients, of leaves that ask for them."""
    weights, _, plan = route(logits, k)
    out = combine(grouped_mm(grouped_mm(x, w, plan, gather=True), v, plan), plan, weights)
    return (out.detach(),) + torch.autograd.grad(out, (logits, x, w, v), torch.ones_like(out))


def layer_leaves(tokens, experts, width, hidden, dtype, dev):
    shapes = ((tokens, experts), (tokens, width), (experts, hidden, width), (experts, width, hidden))
    leaves = [torch.randn(s, generator=gen(i), device=dev) for i, s in enumerate(shapes)]
    return [leaves[0]] + [(t / t.shape[-1] ** 0.5).to(dtype) for t in leaves[1:]]


@pytest.mark.parametrize("tokens,width,hidden", [(37, 64, 96), (600, 264, 129)])
def test_gradients_on_another_stream(dev, tokens, width, hidden):
    leaves = layer_leaves(tokens, 8, width, hidden, BF16, dev)
    want = layer_step(*[t.clone().requires_grad_(True) for t in leaves], 2)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late = [torch.zeros_like(t) for t in leaves]
        for t, value in zip(late, leaves):
            t.copy_(value)  # the operands exist only once this stream has got here
        got = layer_step(*[t.requires_grad_(True) for t in late], 2)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tokens,experts,width,hidden", [(48, 8, 64, 96), (300, 12, 264, 129), (1500, 70, 72, 256)])
def test_gradients_in_a_captured_graph(dev, tokens, experts, width, hidden):
    leaves = [t.requires_grad_(True) for t in layer_leaves(tokens, experts, width, hidden, F16, dev)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer_step(*leaves, 3)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer_step(*leaves, 3)
    for seed in range(4):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(torch.randn(t.shape, generator=gen(100 * seed + i), device=dev) / t.shape[-1] ** 0.5)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, layer_step(*leaves, 3)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("lens,n,k", [([20, 70, 3], 48, 72), ([64, 1, 63], 65, 33), ([130, 0, 64, 200], 264, 520),
                                      ([700, 800], 1536, 1544), ([5, 3], 1, 1)])
@pytest.mark.parametrize("gather", [True, False])
def test_non_finite_values_next_to_a_group_stay_out_of_its_weight_gradient(dev, lens, n, k, gather):
    # rows of the other groups, of no group, and of tokens that no row names
    plan, rows = lengths_to_plan(lens, tail=2)
    x = torch.randn(rows, k, generator=gen(1), device=dev).to(BF16)
    grad = torch.randn(rows, n, generator=gen(2), device=dev).to(BF16)
    w = torch.zeros(len(lens), n, k, dtype=BF16, device=dev, requires_grad=True)
    offsets = plan.offsets.tolist()
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if lo == hi:
            continue
        dirty, dirty_grad = (torch.full_like(t, float("nan")) for t in (x, grad))
        dirty[lo:hi], dirty_grad[lo:hi] = x[lo:hi], grad[lo:hi]
        p = plan
        if gather:  # the same rows, in another order of the tokens among others that are not finite
            order = torch.randperm(2 * rows, generator=gen(3), device=dev)[:rows]
            spread = torch.full((2 * rows, k), float("inf"), dtype=BF16, device=dev)
            spread[order] = dirty
            p, dirty = plan._replace(tokens=order.to(torch.int32)), spread
        dw, = torch.autograd.grad(grouped_mm(dirty, w, p, gather=gather), w, dirty_grad)
        g, a = grad[lo:hi].double(), x[lo:hi].double()
        close(dw[e], g.t() @ a, g.abs().t() @ a.abs(), hi - lo)


@pytest.mark.parametrize("tokens,experts,k,width,drop", [(9, 4, 2, 33, 0.0), (200, 7, 3, 264, 0.3)])
def test_combine_gradient_of_a_plan_in_c(dev, tokens, experts, k, width, drop):
    # the entry point for the places of a plan as they are, which takes no buffer
    import ctypes

    from ops_sparse import _lib

    plan = expert_plan(routed(tokens, experts, k, 3, drop), experts)
    y = torch.randn(tokens * k, width, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    weights = torch.randn(tokens, k, generator=gen(2), device=dev).requires_grad_(True)
    grad = torch.randn(tokens, width, generator=gen(3), device=dev).to(F16)
    want = torch.autograd.grad(combine(y, plan, weights), (y, weights), grad)
    dy = torch.full((tokens * k, width), float("nan"), dtype=F16, device=dev)
    dw = torch.full((tokens, k), float("nan"), device=dev)
    lib, handle = _lib.lib(), ctypes.c_void_p(0)
    assert lib.aclsparseCreate(ctypes.byref(handle)) == _lib.Status.SUCCESS
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: HIP's default stream
    assert lib.aclsparseSetStream(handle, ctypes.c_void_p(stream)) == _lib.Status.SUCCESS
    status = lib.aclsparseCombineGrad(
        handle, tokens, k, width, tokens * k, experts, plan.offsets.data_ptr(), plan.places.data_ptr(),
        weights.data_ptr(), y.data_ptr(), width, grad.data_ptr(), width, int(_lib.DataType.FLOAT16), dy.data_ptr(),
        width, dw.data_ptr())
    lib.aclsparseDestroy(handle)
    assert status == _lib.Status.SUCCESS
    assert torch.equal(dy, want[0]) and torch.equal(dw, want[1])


@pytest.mark.parametrize("kind", ["dropped", "more rows", "outside", "drawn", "one row", "a wave"])
def test_combine_gradient_of_any_places_in_c(dev, kind):
    # lists made by the gradient itself, and by the product
    import ctypes

    from ops_sparse import _lib

    tokens, k, width = 150, 3, 264
    places, rows = any_places(kind, tokens, k)
    places = places.to(dev)
    plan = ExpertPlan(torch.tensor([0, 2], dtype=torch.int32, device=dev), None, places)
    y = torch.randn(rows, width, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    weights = torch.randn(tokens, k, generator=gen(2), device=dev).requires_grad_(True)
    grad = torch.randn(tokens, width, generator=gen(3), device=dev).to(F16)
    product = combine(y, plan, weights)
    want = torch.autograd.grad(product, (y, weights), grad)
    lib, handle, size = _lib.lib(), ctypes.c_void_p(0), ctypes.c_size_t(0)
    assert lib.aclsparseCreate(ctypes.byref(handle)) == _lib.Status.SUCCESS
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: HIP's default stream
    assert lib.aclsparseSetStream(handle, ctypes.c_void_p(stream)) == _lib.Status.SUCCESS
    assert lib.aclsparseCombineGradAny_bufferSize(handle, tokens, k, rows, ctypes.byref(size)) == _lib.Status.SUCCESS
    f16 = int(_lib.DataType.FLOAT16)
    for listed in (0, 1):
        buffer = torch.randint(0, tokens * k, (size.value // 4,), device=dev, dtype=torch.int32)
        if listed:
            out = torch.empty(tokens, width, dtype=F16, device=dev)
            assert lib.aclsparseCombineAndList(
                handle, tokens, k, width, rows, places.data_ptr(), weights.data_ptr(), y.data_ptr(), width, f16,
                out.data_ptr(), width, f16, buffer.data_ptr()) == _lib.Status.SUCCESS
            assert torch.equal(out, product)
        for with_y, with_w in ((True, True), (True, False), (False, True)):
            dy = torch.full((rows, width), float("nan"), dtype=F16, device=dev) if with_y else None
            dw = torch.full((tokens, k), float("nan"), device=dev) if with_w else None
            assert lib.aclsparseCombineGradAny(
                handle, tokens, k, width, rows, places.data_ptr(), weights.data_ptr(), y.data_ptr(), width,
                grad.data_ptr(), width, f16, dy.data_ptr() if with_y else None, width,
                dw.data_ptr() if with_w else None, buffer.data_ptr() if with_y else None, listed) == _lib.Status.SUCCESS
            assert dy is None or torch.equal(dy, want[0])
            assert dw is None or torch.equal(dw, want[1])
    lib.aclsparseDestroy(handle)


def test_offsets_past_32_bits(dev):
    # an operand of more than 2^32 bytes, read at its far end
    width, tokens = 4096, 540_000
    x = torch.empty(tokens, width, dtype=F16, device=dev)
    x[-64:] = torch.randn(64, width, generator=gen(1), device=dev)
    x[:64] = 1.0
    idx = torch.cat([torch.arange(tokens - 64, tokens), torch.arange(64)]).to(torch.int32).to(dev)
    plan = ExpertPlan(torch.tensor([0, 100, 128], dtype=torch.int32, device=dev), idx, None)
    w = torch.randn(2, 64, width, generator=gen(2), device=dev).to(F16)
    y = grouped_mm(x, w, plan, gather=True)
    close(y, *plain_grouped(x, w, plan, 128), width)
    y8 = torch.empty(600_000, width, dtype=F16, device=dev)
    y8[-2:] = 1.0
    places = torch.tensor([[599_999, 599_998]], dtype=torch.int32, device=dev)
    out = combine(y8, ExpertPlan(plan.offsets, None, places))
    assert bool((out == 2.0).all())


@pytest.mark.parametrize("lens,first,last,n,k", [
    ([2, 1, 0, 3, 2, 1], 2, 5, 64, 72), ([30, 0, 200, 77, 5, 64], 1, 4, 40, 33), ([900, 0, 700, 1100, 90, 300], 2, 5, 2304, 64),
    ([5, 3, 4], 2, 3, 264, 136), ([(i * 7) % 5 for i in range(130)], 66, 130, 96, 128)])
def test_rows_before_the_first_expert_are_zero(dev, lens, first, last, n, k):
    # some of a plan's experts, as where they are spread over devices: the others' rows are no expert's
    full, rows = lengths_to_plan(lens, tail=3)
    offsets = full.offsets[first:last + 1]
    lo, hi = int(offsets[0]), int(offsets[-1])
    tokens = torch.randint(0, 50, (rows,), generator=gen(5), device=dev, dtype=torch.int32)
    w = torch.randn(last - first, n, k, generator=gen(2), device=dev).to(BF16).requires_grad_(True)
    w8 = torch.randint(-127, 128, w.shape, generator=gen(2), device=dev, dtype=torch.int8)
    for plan, count in ((ExpertPlan(offsets), rows), (ExpertPlan(offsets, tokens), 50)):
        gather = plan.tokens is not None
        a = torch.randn(count, k, generator=gen(1), device=dev).to(BF16)
        a.requires_grad_(not gather)
        left = [torch.full(s, float("nan"), dtype=BF16, device=dev) for s in ((rows, n), (rows, k))]
        del left  # what the allocator hands out next is not zeros
        y = grouped_mm(a, w, plan, gather=gather)
        close(y.detach(), *plain_grouped(a.detach(), w.detach(), plan, rows), k)
        assert not y[:lo].any() and not y[hi:].any()
        grad = torch.randn(rows, n, generator=gen(3), device=dev).to(BF16)
        grads = torch.autograd.grad(y, (w,) if gather else (w, a), grad)
        wa, ma, ww, mw = plain_grads(a.detach(), w.detach(), plan, grad)
        close(grads[0], ww, mw, max(lens))
        if not gather:
            close(grads[1], wa, ma, n)
        a8 = a.detach().mul(20).clamp(-127, 127).to(torch.int8)
        one, sw = torch.ones(count, device=dev), torch.ones(last - first, n, device=dev)
        left = torch.full((rows, n), float("nan"), device=dev)
        del left
        y8 = grouped_mm_scaled(a8, one, w8, sw, plan, gather=gather, out_dtype=F32)
        scaled_close(y8, plain_scaled(a8, one, w8, sw, plan, rows))


# Grids of more threads than one dimension takes (2^32): tokens or assignments by the million.


@pytest.mark.parametrize("tokens,width", [(2**24 + 9, 3), (2**20, 4097)])
def test_combine_of_many_tokens(dev, tokens, width):
    y = torch.randn(64, width, generator=gen(1), device=dev).to(F16)
    places = torch.randint(0, 64, (tokens, 1), generator=gen(2), device=dev, dtype=torch.int32)
    out = combine(y, ExpertPlan(torch.tensor([0, 64], dtype=torch.int32, device=dev), None, places))
    step = 2**17
    for first in range(0, tokens, step):
        assert torch.equal(out[first:first + step], y[places[first:first + step, 0].long()])


def test_combine_gradient_of_many_assignments(dev):
    tokens, k = 2**20 + 3, 64
    places = torch.arange(tokens * k - 1, -1, -1, dtype=torch.int32, device=dev).view(tokens, k)
    plan = ExpertPlan(torch.tensor([0, tokens * k], dtype=torch.int32, device=dev), None, places)
    y = torch.randn(tokens * k, 1, generator=gen(1), device=dev).to(F16).requires_grad_(True)
    weights = torch.randn(tokens, k, generator=gen(2), device=dev).requires_grad_(True)
    grad = torch.randn(tokens, 1, generator=gen(3), device=dev).to(F16)
    dy, dw = torch.autograd.grad(combine(y, plan, weights), (y, weights), grad)
    # one product each, of two fp16 numbers exact in fp32
    assert torch.equal(dw, y.detach().float().flip(0).view(tokens, k) * grad.float())
    want = (weights.detach().double() * grad.double()).view(-1, 1).flip(0)
    close(dy, want, want.abs(), 1)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_of_many_tokens(dev, normalize):
    tokens = 2**26 + 5
    logits = torch.randn(tokens, 2, generator=gen(1), device=dev).requires_grad_(True)
    weights, ids, _ = route(logits, 1 + normalize, normalize=normalize)
    grad = torch.zeros_like(weights)
    grad[:, 0] = 1.0
    got, = torch.autograd.grad(weights, logits, grad)
    step = 2**22
    for first in range(0, tokens, step):
        part = slice(first, first + step)
        p = torch.softmax(logits.detach()[part].double(), 1)
        top = p.argmax(1, keepdim=True)
        assert torch.equal(top, ids[part, :1].long())
        # p (1 - p) of the first choice, and its negative: each factor to a few roundings
        want = torch.full_like(p, -1.0).scatter_(1, top, 1.0) * p[:, :1] * p[:, 1:]
        assert bool(((got[part].double() - want).abs() <= 64 * U32 * p.gather(1, top)).all())


def test_scaled_of_many_columns(dev):
    n, k = 2**28 + 5, 16
    a = torch.randint(-127, 128, (1, k), generator=gen(1), device=dev, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=gen(2), device=dev, dtype=torch.int8)
    sw = torch.rand(n, generator=gen(3), device=dev)
    y = grouped_mm_scaled(a, torch.ones(1, device=dev), w, sw, out_dtype=F32)
    step = 2**24
    for first in range(0, n, step):
        part = slice(first, first + step)
        # integers below 2^24: exact in fp32, as is 1 * sw; one rounding
        assert torch.equal(y[0, part], (w[part].float() * a.float()).sum(1) * sw[part])


# ------------------------------------------------------------------------------------------------------- refusals


def test_refusals(dev):
    x = torch.zeros(4, 8, dtype=F16, device=dev)
    w = torch.zeros(2, 8, 8, dtype=F16, device=dev)
    plan = ExpertPlan(torch.tensor([0, 2, 4], dtype=torch.int32, device=dev),
                      torch.zeros(4, dtype=torch.int32, device=dev))
    for call, error in (
            (lambda: route(torch.zeros(4, 8, device=dev), 9), ValueError),
            (lambda: route(torch.zeros(4, 8, device=dev), 0), ValueError),
            (lambda: route(torch.zeros(4, 1025, device=dev), 2), ValueError),
            (lambda: route(torch.zeros(4, 200, device=dev), 65), ValueError),
            (lambda: route(torch.zeros(8, device=dev), 1), ValueError),
            (lambda: route(torch.zeros(4, 8, device=dev, dtype=torch.float64), 1), TypeError),
            (lambda: route(torch.zeros(4, 8), 1), ValueError),
            (lambda: expert_plan(torch.zeros(4, 2, dtype=torch.int64, device=dev), 4), TypeError),
            (lambda: expert_plan(torch.zeros(4, 2, dtype=torch.int32, device=dev), 1), ValueError),
            (lambda: grouped_mm(x.float(), w.float(), plan), TypeError),
            (lambda: grouped_mm(x, w.to(BF16), plan), TypeError),
            (lambda: grouped_mm(x, w[:, :, :4], plan), ValueError),
            (lambda: grouped_mm(x, w[0], plan), ValueError),
            (lambda: grouped_mm(x, w[:1], plan), ValueError),
            (lambda: grouped_mm(x.cpu(), w, plan), ValueError),
            (lambda: grouped_mm(x, w.cpu(), plan), ValueError),
            (lambda: grouped_mm(x, w, ExpertPlan(plan.offsets), gather=True), ValueError),
            (lambda: grouped_mm(x, w, ExpertPlan(plan.offsets.long(), plan.tokens)), TypeError),
            (lambda: grouped_mm(x, w, ExpertPlan(plan.offsets.cpu(), plan.tokens)), ValueError),
            (lambda: grouped_mm(x.requires_grad_(True), w, plan, gather=True), ValueError),
            (lambda: grouped_mm_scaled(x.detach(), torch.ones(4, device=dev), w, torch.ones(2, 8, device=dev), plan),
             TypeError),
            (lambda: grouped_mm_scaled(x.detach().to(torch.int8), torch.ones(3, device=dev), w.to(torch.int8),
                                       torch.ones(2, 8, device=dev), plan), ValueError),
            (lambda: grouped_mm_scaled(x.detach().to(torch.int8), torch.ones(4, device=dev), w.to(torch.int8),
                                       torch.ones(2, 8, device=dev), plan, out_dtype=torch.int32), TypeError),
            (lambda: grouped_mm_scaled(x.detach().to(torch.int8), torch.ones(4, device=dev), w.to(torch.int8),
                                       torch.ones(2, 8, device=dev)), ValueError),
            (lambda: combine(x.detach(), plan), ValueError),
            (lambda: combine(x.detach().float(), ExpertPlan(plan.offsets, None, plan.tokens.view(2, 2))), TypeError),
            (lambda: combine(x.detach(), ExpertPlan(plan.offsets, None, plan.tokens.view(2, 2)),
                             torch.ones(4, 1, device=dev)), ValueError)):
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()


def test_operands_of_fewer_rows_than_the_plan_are_refused(dev):
    tokens, experts, k = 20, 4, 2
    plan = expert_plan(routed(tokens, experts, k, 1), experts)
    x, w = torch.ones(tokens, 16, dtype=F16, device=dev), torch.ones(experts, 8, 16, dtype=F16, device=dev)
    x8, w8, one = x.to(torch.int8), w.to(torch.int8), torch.ones(tokens, device=dev)
    sw = torch.ones(experts, 8, device=dev)
    for call in (lambda: grouped_mm(x, w, plan),  # gather forgotten
                 lambda: grouped_mm(x.clone().requires_grad_(True), w, plan),
                 lambda: grouped_mm(x[:-1], w, plan, gather=True),
                 lambda: grouped_mm_scaled(x8, one, w8, sw, plan),
                 lambda: grouped_mm_scaled(x8[:-1], one[:-1], w8, sw, plan, gather=True)):
        with pytest.raises(ValueError, match="rows"):
            call()
    # more of them are none of the plan's: rows of no expert, which are zero, or tokens that nothing names
    more = torch.ones(tokens * k + 3, 16, dtype=F16, device=dev)
    y = grouped_mm(more, w, plan)
    assert y.shape[0] == tokens * k + 3 and bool((y[:-3] == 16).all()) and not y[-3:].any()
    assert bool((grouped_mm(more, w, plan, gather=True) == 16).all())
    y = grouped_mm_scaled(more.to(torch.int8), torch.ones(len(more), device=dev), w8, sw, plan)
    assert bool((y[:-3] == 16).all()) and not y[-3:].any()
