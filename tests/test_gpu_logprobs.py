"""Log probabilities of tokens on the GPU against the definition in 64 bits.

Tolerances: an exponential is off by a few units in the last place of its argument's rounding, (|d| + 4) * 2^-23 for a
logit d below the largest; the sum of V of them by V / 256 + 16 roundings of 2^-24 (each of 256 threads adds its own), and
the logarithm passes the sum's relative error on as an absolute one.
"""
import ctypes

import numpy as np
import pytest
import torch

from ops_sparse import _lib, token_logprobs
from ops_sparse._lib import DataType

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0**-24


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def plain(logits, targets):
    """(logprobs, entropy, log p) in float64 of two-dimensional logits; -inf has probability 0, a row of it entropy 0."""
    x = logits.double().cpu()
    logs = torch.log_softmax(x, 1)
    none = (x == -np.inf).all(1)
    logs[none] = -np.inf
    t = targets.cpu().long()
    named = (t >= 0) & (t < x.shape[1])
    lp = torch.where(named, logs.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], 0.0)
    p = logs.exp()
    terms = torch.where(logs == -np.inf, torch.zeros_like(p), p * logs)
    return lp, -terms.sum(1), logs


def error(logits):
    """Bound of a row's log S, absolute."""
    v = logits.shape[1]
    return (v / 256 + 16) * U + 40 * 2 * U  # terms that matter lie within 40 of the largest


def check(got, want, bound):
    got, want = got.detach().double().cpu(), want
    assert torch.equal(got.isnan(), want.isnan())
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = torch.isfinite(want)
    err = (got - want).abs()[fine]
    bound = (bound + 3 * U * want.abs())[fine]
    assert bool((err <= bound).all()), float((err / bound).max())


def check_top(r, logits, k):
    x, ids, values = logits.float().cpu().numpy(), r.top_ids.cpu().numpy(), r.top_logprobs.detach().cpu()
    _, _, logs = plain(logits, torch.zeros(len(x), dtype=torch.int64))
    for row in range(len(x)):
        order = sorted((i for i in range(x.shape[1]) if x[row, i] != -np.inf),
                       key=lambda i: (0 if np.isnan(x[row, i]) else 1, -x[row, i], i))[:k]
        order = np.array(order + [-1] * (k - len(order)))
        assert np.array_equal(ids[row], order), row
        want = torch.where(torch.from_numpy(order) >= 0, logs[row, torch.from_numpy(order)], -np.inf)
        check(values[row], want, error(logits))


def rows(t, v, dtype, seed=0, scale=2.5):
    return (torch.randn(t, v, generator=gen(seed + v), device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,v,k", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (1, 64, 64), (5, 65, 64), (2, 2049, 20),
                                   (1, 16384, 1), (1, 131072, 20), (9, 32003, 5), (700, 300, 3), (1100, 1030, 20),
                                   (1025, 4097, 64)])
def test_rows(dev, t, v, k, dtype):
    logits = rows(t, v, dtype)
    targets = torch.randint(0, v, (t,), generator=gen(1), device=dev)
    r = token_logprobs(logits, targets, top=k, entropy=True)
    lp, h, _ = plain(logits, targets)
    check(r.logprobs, lp, error(logits))
    check(r.entropy, h, error(logits) + 4 * error(logits) * h.abs())
    if t * v <= 1 << 19:
        check_top(r, logits, k)
    else:
        want = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_ids.long(), want)
    less = token_logprobs(logits, targets.int())
    assert less.entropy is None and less.top_ids is None and less.top_logprobs is None
    assert torch.equal(less.logprobs, r.logprobs)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,v", [(1, 9000), (30, 20000), (1200, 500)])
def test_masks(dev, t, v, dtype):
    low = torch.finfo(dtype).min
    logits = rows(t, v, dtype, 2)
    hide = torch.rand(t, v, generator=gen(3), device=dev)
    for value in (-float("inf"), low):
        x = logits.masked_fill(hide < 0.5, value)
        x[0, :] = value          # nothing is left
        if t > 4:
            x[1, 1:] = value     # one is
            x[2, :-1] = value
            x[3, :] = -float("inf")
            x[3, v // 2] = low   # the lowest value is a logit like others
        targets = torch.randint(0, v, (t,), generator=gen(4), device=dev)
        r = token_logprobs(x, targets, top=6, entropy=True)
        lp, h, _ = plain(x, targets)
        check(r.logprobs, lp, error(x))
        check(r.entropy, h, error(x) + 4 * error(x) * h.abs())
        part = slice(0, 5)
        check_top(type(r)(*(o[part] for o in r)), x[part], 6)


@pytest.mark.parametrize("t,v", [(1, 9000), (1200, 500)])
def test_infinity_and_nan(dev, t, v):
    x = rows(t, v, F32, 5)
    x[0, 7], x[-1, v - 1] = float("inf"), float("nan")
    targets = torch.zeros(t, dtype=torch.int64, device=dev)
    r = token_logprobs(x, targets, top=3, entropy=True)
    for row in {0, t - 1}:
        assert torch.isnan(r.logprobs[row]) and torch.isnan(r.entropy[row]) and torch.isnan(r.top_logprobs[row]).all()
        first = v - 1 if row == t - 1 else 7
        assert r.top_ids[row, 0] == first
    if t > 2:
        lp, h, _ = plain(x[1:-1], targets[1:-1])
        check(r.logprobs[1:-1], lp, error(x))


@pytest.mark.parametrize("t,v", [(1, 50000), (2, 5000), (1030, 3000)])
def test_alternatives_of_many_equal_logits(dev, t, v):
    x = torch.zeros(t, v, device=dev, dtype=BF16)
    x[:, v // 3::7] = 1.0
    r = token_logprobs(x, torch.zeros(t, dtype=torch.int64, device=dev), top=64)
    want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :64]
    assert torch.equal(r.top_ids.long(), want)
    x = torch.zeros(t, v, device=dev, dtype=BF16)
    r = token_logprobs(x, torch.zeros(t, dtype=torch.int64, device=dev), top=10)
    assert torch.equal(r.top_ids.long(), torch.arange(10, device=dev).expand(t, 10))


@pytest.mark.parametrize("t", [1, 1030])
def test_alternatives_in_one_threads_places(dev, t):
    # sorted both ways, and the largest all where one thread of a workgroup reads them
    v = 40000
    up = torch.arange(v, device=dev).float().expand(t, v) / 1000
    for x in (up.contiguous(), up.flip(1).contiguous()):
        r = token_logprobs(x, torch.zeros(t, dtype=torch.int64, device=dev), top=64)
        assert torch.equal(r.top_ids.long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :64])
    x = rows(t, v, F32, 6)
    for unit in range(0, v, 2048):
        x[:, unit:unit + 8] += 50.0
    r = token_logprobs(x, torch.zeros(t, dtype=torch.int64, device=dev), top=64)
    assert torch.equal(r.top_ids.long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :64])


@pytest.mark.parametrize("t,v", [(5, 1030), (3, 2047), (1, 2049), (2, 4096), (1, 4097), (512, 4100), (40, 8193),
                                 (513, 9000), (2, 32768), (3, 32769), (70, 32001), (1, 140000)])
@pytest.mark.parametrize("k", [0, 12, 13, 64])
def test_ways_of_cutting_rows(dev, t, v, k):
    # one workgroup or several a row, of 256 or 1024 threads; alternatives by a bound or one after another
    for dtype in (F32, BF16):
        logits = rows(t, v, dtype, 25)
        targets = torch.randint(-1, v + 1, (t,), generator=gen(26), device=dev)
        r = token_logprobs(logits, targets, top=k, entropy=True)
        lp, h, logs = plain(logits, targets)
        check(r.logprobs, lp, error(logits))
        check(r.entropy, h, error(logits) + 4 * error(logits) * h.abs())
        if k == 0:
            continue
        want = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_ids.long(), want)
        check(r.top_logprobs, logs.gather(1, want.cpu()), error(logits))


@pytest.mark.parametrize("t,v", [(1, 131072), (9, 60000), (6, 32000), (4, 2000)])
@pytest.mark.parametrize("k", [5, 64])
def test_alternatives_side_by_side(dev, t, v, k):
    # rising, falling, and all of what is not masked in one place: the largest are one segment's, or a few threads'
    up = torch.arange(v, device=dev, dtype=F32) * (40.0 / v)
    run = torch.full((v,), -float("inf"), device=dev)
    run[v // 2:v // 2 + 1900] = torch.randn(min(1900, v - v // 2), generator=gen(27), device=dev)
    for row in (up, up.flip(0), run):
        logits = row.repeat(t, 1)
        r = token_logprobs(logits, torch.zeros(t, dtype=torch.int64, device=dev), top=k)
        want = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(r.top_ids.long(), want)


def test_far_apart_logits(dev):
    x = torch.tensor([[0.0, 88.0, 200.0], [-200.0, -100.0, -150.0], [1e30, -1e30, 0.0], [3e38, -3e38, 3e38],
                      [100.0, 100.0, 100.0]], device=dev)
    for t in range(3):
        targets = torch.full((5,), t, device=dev)
        r = token_logprobs(x, targets, top=3, entropy=True)
        lp, h, _ = plain(x, targets)
        got = r.logprobs.double().cpu()
        lp = torch.where(lp < -3.4e38, torch.full_like(lp, -np.inf), lp)  # differences past fp32
        check(got, lp, error(x))
        check(r.entropy, h, error(x))


def test_padding_shapes_and_strides(dev):
    logits = rows(24, 501, BF16, 7)
    targets = torch.randint(0, 501, (24,), generator=gen(8), device=dev)
    targets[3], targets[5], targets[7] = -100, 501, 2**40
    want = token_logprobs(logits, targets, top=2, entropy=True)
    assert want.logprobs[[3, 5, 7]].tolist() == [0, 0, 0]
    lp, _, _ = plain(logits, targets)
    check(want.logprobs, lp, error(logits))
    wide = torch.full((24, 700), float("nan"), device=dev, dtype=BF16)
    wide[:, 99:600] = logits
    apart = torch.full((48, 501), float("nan"), device=dev, dtype=BF16)
    apart[::2] = logits
    for x in (wide[:, 99:600], apart[::2], logits.t().contiguous().t(), logits.view(24, 501)):
        for a, b in zip(token_logprobs(x, targets, top=2, entropy=True), want):
            assert torch.equal(a, b)
    r = token_logprobs(logits.view(2, 3, 4, 501), targets.view(2, 3, 4), top=2, entropy=True)
    assert r.logprobs.shape == r.entropy.shape == (2, 3, 4) and r.top_ids.shape == r.top_logprobs.shape == (2, 3, 4, 2)
    for a, b in zip(r, want):
        assert torch.equal(a.reshape(b.shape), b)
    one = token_logprobs(logits[0], targets[0], top=2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,) and torch.equal(one.top_ids, want.top_ids[0])
    none = token_logprobs(logits[:0], targets[:0], top=2, entropy=True)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 2)
    none = token_logprobs(logits.view(24, 501)[:0].requires_grad_(), targets[:0])
    assert none.logprobs.shape == (0,)


# ------------------------------------------------------------------------------------------------------ gradients


def exact_gradient(logits, targets, gl, ge, gt, ids):
    lp, h, logs = plain(logits, targets)
    v = logits.shape[1]
    t = targets.cpu().long()
    p = logs.exp()
    named = (t >= 0) & (t < v)
    d = torch.zeros_like(p)
    total = torch.zeros(len(p), dtype=torch.float64)
    alive = (logits.cpu() != -np.inf).any(1)
    if gl is not None:
        g = torch.where(named & alive, gl.double().cpu(), 0.0)
        d.scatter_add_(1, t.clamp(0, v - 1)[:, None], g[:, None])
        total += g
    if gt is not None:
        g = torch.where(ids.cpu() >= 0, gt.double().cpu(), 0.0)
        d.scatter_add_(1, ids.cpu().long().clamp(min=0), g)
        total += g.sum(1)
    d -= p * total[:, None]
    if ge is not None:
        d -= torch.where(p > 0, p * ge.double().cpu()[:, None] * (logs + h[:, None]), 0.0)
    return d, p


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,v,k", [(1, 1, 1), (1, 3, 2), (4, 70, 64), (2, 9001, 5), (33, 8192, 1), (1050, 333, 4)])
def test_gradient(dev, t, v, k, dtype):
    logits = rows(t, v, dtype, 9)
    if v > 50:
        logits[torch.rand(t, v, generator=gen(10), device=dev) < 0.2] = -float("inf")
        logits[0] = -float("inf")
    targets = torch.randint(0, v, (t,), generator=gen(11), device=dev)
    if t > 1:
        targets[1] = -1
    gl, ge = torch.randn(t, generator=gen(12), device=dev), torch.randn(t, generator=gen(13), device=dev)
    gt = torch.randn(t, k, generator=gen(14), device=dev)
    for use in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        x = logits.clone().requires_grad_()
        r = token_logprobs(x, targets, top=k, entropy=True)
        outs, given = zip(*[(o, g) for o, g, u in zip((r.logprobs, r.entropy, r.top_logprobs), (gl, ge, gt), use) if u])
        d = torch.autograd.grad(outs, x, given)[0]
        assert d.dtype == dtype
        args = [g if u else None for g, u in zip((gl, ge, gt), use)]
        want, p = exact_gradient(logits, targets, *args, r.top_ids)
        size = sum(g.abs().double().cpu().reshape(t, -1).sum(1) for g in given)[:, None]
        # p is off by the error of log p, d log p + h by two of them, at most log v + 40 in size
        e = 2 * error(logits) + 40 * U
        bound = p * size * e * (60 + np.log(v)) + want.abs() * (torch.finfo(dtype).eps / 2 + 8 * U) + (k + 4) * U * (
            want != 0) * size + (2.0**-25 if dtype == F16 else 1e-37)
        err = (d.double().cpu() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_large_gradient_of_the_entropy_beside_masked_logits(dev, dtype):
    t, v = 5, 300
    logits = rows(t, v, dtype, 21)
    logits[:, ::3] = -float("inf")
    logits[:, 1::3][:, :40] = torch.finfo(dtype).min
    ge = torch.tensor([1e30, -1e30, 3e12, -1e9, 1e8], device=dev)
    x = logits.clone().requires_grad_()
    d = torch.autograd.grad(token_logprobs(x, torch.zeros(t, dtype=torch.int64, device=dev), entropy=True).entropy, x,
                            ge)[0]
    want, p = exact_gradient(logits, torch.zeros(t, dtype=torch.int64), None, ge, None, None)
    size = ge.abs().double().cpu()[:, None]
    e = 2 * error(logits) + 40 * U  # as above
    bound = p * size * e * (60 + np.log(v)) + want.abs() * (torch.finfo(dtype).eps / 2 + 8 * U) + 4 * U * (
        want != 0) * size + 1e-37
    err = (d.double().cpu() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_gradient_against_differences(dev):
    # the fp64 definition agrees with the results to 1e-6, so a difference over 2^-5 shows the gradient to 1e-6 * 2^6 and
    # the third derivative's share, at most 2^-10 / 6 of weights below one
    x = rows(6, 40, F32, 15, 1.0)
    targets = torch.randint(0, 40, (6,), generator=gen(16), device=dev)
    weights = torch.rand(6, 40, generator=gen(17), device=dev)

    def f(z):
        r = token_logprobs(z, targets, top=3, entropy=True)
        return (r.logprobs * weights[:, 0] + r.entropy * weights[:, 1] + (r.top_logprobs * weights[:, 2:5]).sum(1)).double().sum()

    z = x.clone().requires_grad_()
    grad = torch.autograd.grad(f(z), z)[0]
    for _ in range(20):
        r, c = np.random.default_rng(_).integers(0, [6, 40])
        step = torch.zeros_like(x)
        step[r, c] = 2.0**-5
        change = (f(x + step) - f(x - step)) / 2.0**-4
        assert abs(float(change) - float(grad[r, c])) <= 2e-3


def test_gradients_once_and_through_shapes(dev):
    x = rows(12, 300, F32, 18).requires_grad_()
    targets = torch.randint(0, 300, (3, 4), generator=gen(19), device=dev)
    r = token_logprobs(x.view(3, 4, 300), targets, top=2)
    assert r.logprobs.requires_grad and r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    grad = torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)[0]
    p = torch.softmax(x.detach().double(), 1)
    want = torch.nn.functional.one_hot(targets.view(-1), 300) - p
    assert bool((grad.detach().double() - want).abs().max() <= 4 * error(x))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(grad.sum(), x)
    with torch.no_grad():
        assert not token_logprobs(x, targets.view(-1)).logprobs.requires_grad
    strided = rows(12, 600, F32, 18).requires_grad_()
    torch.autograd.grad(token_logprobs(strided[:, ::2], targets.view(-1)).logprobs.sum(), strided)


def test_a_training_step_in_a_graph(dev):
    x = rows(40, 5000, BF16, 20).requires_grad_()
    targets = torch.randint(0, 5000, (40,), generator=gen(21), device=dev)
    g = torch.full((40,), 0.5, device=dev)

    def step():
        r = token_logprobs(x, targets, top=4, entropy=True)
        return (*r, torch.autograd.grad((r.logprobs, r.entropy), x, (g, g))[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(rows(40, 5000, BF16, 30 + seed))
        targets.copy_(torch.randint(0, 5000, (40,), generator=gen(seed), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_answers_in_two_graphs(dev):
    # rows in segments that are joined, in one workgroup, and read again for alternatives; graphs with workspaces each
    sets = []
    for t, v, k in ((1, 131072, 20), (3, 40000, 5), (37, 9000, 50), (1100, 9000, 5)):
        x, targets = rows(t, v, BF16, 40), torch.zeros(t, dtype=torch.int64, device=dev)
        token_logprobs(x, targets, top=k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = token_logprobs(x, targets, top=k, entropy=True)
        sets.append((x, targets, k, graph, got))
    for seed in range(3):
        for x, targets, _, graph, _ in sets:
            x.copy_(rows(*x.shape, BF16, 50 + seed))
            targets.copy_(torch.randint(0, x.shape[1], targets.shape, generator=gen(seed), device=dev))
            graph.replay()
        torch.cuda.synchronize()
        for x, targets, k, _, got in sets:
            for one, other in zip(got, token_logprobs(x, targets, top=k, entropy=True)):
                assert torch.equal(one, other)


@pytest.mark.parametrize("leaf", [True, False])
def test_a_capture_beside_an_eager_graph_of_the_leaf_is_refused(dev, leaf):
    # torch's engine would make the eager graph's stream wait for the captured one and end the process
    x = rows(4, 100, F32, 23).requires_grad_()
    targets = torch.zeros(4, dtype=torch.int64, device=dev)

    def logits():
        return x if leaf else x * 2

    def refused():  # leaves nothing behind that would hold the leaf's graph
        try:
            token_logprobs(logits(), targets)
        except RuntimeError as e:
            return str(e)

    eager = token_logprobs(logits(), targets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        message = refused()
    assert "alive" in message
    assert eager.logprobs.shape == (4,)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = torch.autograd.grad(token_logprobs(logits(), targets).logprobs.sum(), x)[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, torch.autograd.grad(token_logprobs(logits(), targets).logprobs.sum(), x)[0])


def test_offsets_past_32_bits(dev):
    # rows of a matrix whose last lie past 2^31 elements; the others are read for a single one of them
    v, t = 70000, 31000
    x = torch.zeros(t, v, device=dev, dtype=BF16)
    x[-1] = rows(1, v, BF16, 22)[0]
    targets = torch.full((t,), 5, device=dev)
    targets[-1] = v - 2
    r = token_logprobs(x, targets, top=2, entropy=False)
    lp, _, _ = plain(x[-2:], targets[-2:])
    check(r.logprobs[-2:], lp, error(x))
    assert torch.equal(r.top_ids[-1].long(), torch.sort(x[-1].float(), descending=True, stable=True).indices[:2])
    assert r.top_ids[-2].tolist() == [0, 1]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t,v", [(1, 1), (1, 40), (3, 9000), (1, 70000), (2, 131072), (600, 9000), (1200, 500)])
def test_nan_in_the_first_places(dev, t, v, dtype):
    # NaN is the largest, the lowest id first: in the first column, in all, and at the ends of segments and threads' units
    k = min(v, 6)
    x = rows(t, v, dtype, 60)
    places = sorted({p for p in (0, 1, 7, 8, 2047, 2048, v // 2, v - 1) if p < v})
    targets = torch.zeros(t, dtype=torch.int64, device=dev)
    for named in ([0], places[-1:], places, slice(None)):
        y = x.clone()
        y[0, named] = float("nan")
        r = token_logprobs(y, targets, top=k, entropy=True)
        check_top(type(r)(*(o[:1] for o in r)), y[:1], k)
        assert torch.isnan(r.logprobs[0]) and torch.isnan(r.entropy[0]) and torch.isnan(r.top_logprobs[0]).all()
        if t > 1:
            check_top(type(r)(*(o[-1:] for o in r)), y[-1:], k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("t,v,k", [(1, 5, 3), (7, 20000, 20), (300, 8192, 64), (1200, 333, 0)])
def test_a_gradient_in_the_place_of_its_logits(dev, t, v, k, dtype):
    # the C entry point, whose caller may have no use for the logits any more; the torch one keeps them
    lib, types = _lib.lib(), {F32: DataType.FLOAT, F16: DataType.FLOAT16, BF16: DataType.BF16}
    logits, ld = rows(t, v + 3, dtype, 61), v + 3
    targets = torch.randint(-1, v, (t,), generator=gen(62), device=dev)
    x = logits[:, :v].clone().requires_grad_()
    r = token_logprobs(x, targets, top=k, entropy=True)
    gl, ge, gt = (torch.randn(*s, generator=gen(63 + i), device=dev) for i, s in enumerate(((t,), (t,), (t, max(k, 1)))))
    outs, given = [r.logprobs, r.entropy], [gl, ge]
    if k:
        outs, given = outs + [r.top_logprobs], given + [gt]
    want = torch.autograd.grad(outs, x, given)[0]
    m = x.detach().float().max(1).values
    stats = torch.stack([m, torch.log(torch.exp(x.detach().double() - m[:, None]).sum(1)).float()], 1).contiguous()
    h = ctypes.c_void_p(0)
    assert lib.aclsparseCreate(ctypes.byref(h)) == 0
    assert lib.aclsparseSetStream(h, ctypes.c_void_p(_lib.HIP_NULL_STREAM)) == 0
    entropy = r.entropy.detach().contiguous()
    apart = torch.zeros_like(logits)

    def run(out):
        torch.cuda.synchronize()
        assert lib.aclsparseTokenLogprobsGrad(
            h, t, v, logits.data_ptr(), ld, int(types[dtype]), targets.data_ptr(), int(DataType.INT64), stats.data_ptr(),
            entropy.data_ptr(), k, r.top_ids.data_ptr() if k else None, gl.data_ptr(), ge.data_ptr(),
            gt.data_ptr() if k else None, out.data_ptr(), ld) == 0
        torch.cuda.synchronize()

    run(apart)
    rest = logits[:, v:].clone()
    run(logits)
    lib.aclsparseDestroy(h)
    assert torch.equal(logits[:, :v], apart[:, :v]) and torch.equal(logits[:, v:], rest)
    # log S from 64 bits is the kernel's to its error, which p passes on
    size = 2 * error(x) * (sum(g.abs().reshape(t, -1).sum(1) for g in given)[:, None].double() * 60 + 1)
    assert bool(((apart[:, :v].double() - want.double()).abs() <= size + want.double().abs() * torch.finfo(dtype).eps).all())
