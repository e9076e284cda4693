"""The AdamW step on the GPU against the formulas.

The moments are each a fixed sequence of fp32 operations, which numpy repeats bit for bit, 8-bit codes included.  A
parameter is p (1 - lr wd) - change: with the change in 64 bits off by at most 12 roundings of 2^-24 (the moments' three
each, two of the square root and its division, the sum, the division and the product, and the two scalars), p's product
and scalar by two and their difference by one, and then half a step of its type.
"""
import numpy as np
import pytest
import torch

from ops_sparse import AdamWState, adamw_moments, adamw_state, adamw_step

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0**-24
HYPER = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------- the 8-bit format, from its definition


def decode(codes, exponents, second):
    """float64 values of numpy codes [P] and exponents [P / 32]."""
    least = -29 if second else -13
    c = codes.astype(np.int64)
    m = c if second else c & 127
    v = np.where(m < 8, np.ldexp(m / 8.0, least), np.ldexp(1 + (m & 7) / 8.0, (m >> 3) - 1 + least))
    if not second:
        v = np.where(c & 128, -v, v)
    e = np.repeat(exponents.astype(np.int64), 32)
    return np.where(e == 255, np.nan, np.ldexp(v, e - 127))


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9B05688D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x5BE0CD19) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(n, seed, step, place):
    key = (mix((int(mix(seed)) + step) & 0xFFFFFFFF) + place) & 0xFFFFFFFF
    return mix((np.arange(n, dtype=np.uint64) + np.uint64(mix(key))) & np.uint64(0xFFFFFFFF))


def encode(x, bits, second):
    """(codes, exponents) of float32 x [P], rounded by the 16 random bits."""
    least = -29 if second else -13
    blocks = x.reshape(-1, 32)
    e = (np.abs(blocks).view(np.uint32) >> 23).max(1)
    scale = np.ldexp(1.0, np.where(e == 255, 0, e).astype(np.int64) - 127)
    a = np.where(np.isfinite(blocks), np.abs(blocks).astype(np.float64), 0) / scale[:, None]  # exact
    a = a.reshape(-1).astype(np.float32)
    r = bits.astype(np.int64) * 16 + 8
    first = (least + 127) * 8
    normal = ((a.view(np.uint32).astype(np.int64) + r) >> 20) - first + 8
    lifted = (a + np.float32(2.0**least)).view(np.uint32).astype(np.int64)
    code = np.where(a < np.float32(2.0**least), ((lifted + r) >> 20) - first, normal)
    if second:
        code = np.where((a > 0) & (code == 0), 1, code)
    else:
        code = code + np.where(np.signbit(x), 128, 0)
    code = np.where(np.repeat(e, 32) == 255, 0, code)
    return code.astype(np.uint8), e.astype(np.uint8)


# ------------------------------------------------------------------------------------------------------- the step


class Plain:
    """One tensor, its moments in float32 step by step and its values in float64."""

    def __init__(self, p, state, i):
        self.n = p.numel()
        self.old = (state.masters[i] if state.masters is not None else p).double().cpu().numpy().reshape(-1)
        self.codes = state.moments[i].cpu().numpy().copy()
        self.exponents = state.exponents[i].cpu().numpy().copy() if state.exponents is not None else None
        self.seed, self.place = state.seed, i

    def step(self, grad, t, lr, betas, eps, weight_decay, scale=1.0):
        f = np.float32
        with np.errstate(over="ignore", invalid="ignore"):
            g = np.zeros(self.codes.shape[1], f)
            g[:self.n] = grad.float().cpu().numpy().reshape(-1) * f(scale)
            held = self.codes if self.exponents is None else np.stack(
                [decode(self.codes[j], self.exponents[j], j) for j in range(2)]).astype(f)
            m = held[0] * f(betas[0]) + g * f(1 - betas[0])
            v = held[1] * f(betas[1]) + (g * g) * f(1 - betas[1])
            m[self.n:], v[self.n:] = (0, 0) if self.exponents is not None else held[:, self.n:]
            change = lr / (1 - betas[0]**t) * m[:self.n].astype(np.float64) / (
                np.sqrt(v[:self.n].astype(np.float64)) / np.sqrt(1 - betas[1]**t) + eps)
        kept = self.old * (1 - lr * weight_decay)
        self.new = kept - change
        self.bound = 12 * U * np.abs(change) + 3 * U * (np.abs(kept) + np.abs(change)) + 1e-44
        if self.exponents is None:
            self.codes = np.stack([m, v])
        else:
            bits = random_bits(len(m), self.seed, t, self.place)
            both = [encode(m, bits & np.uint64(0xFFFF), 0), encode(v, bits >> np.uint64(16), 1)]
            self.codes, self.exponents = np.stack([b[0] for b in both]), np.stack([b[1] for b in both])

    def check(self, p, state, i):
        assert np.array_equal(state.moments[i].cpu().numpy(), self.codes, equal_nan=self.exponents is None)
        if self.exponents is not None:
            assert np.array_equal(state.exponents[i].cpu().numpy(), self.exponents)
        got = (state.masters[i] if state.masters is not None else p).double().cpu().numpy().reshape(-1)
        dtype = F32 if state.masters is not None else p.dtype
        half = torch.finfo(dtype).eps / 2
        bound = self.bound + (np.abs(self.new) + self.bound) * half + {F16: 2.0**-25}.get(dtype, 0)
        fine = np.isfinite(self.new)
        assert np.array_equal(np.isnan(got), np.isnan(self.new))
        assert (np.abs(got - self.new)[fine] <= bound[fine]).all()
        if state.masters is not None:
            assert torch.equal(p, state.masters[i].to(p.dtype))
        self.old = got


def tensors(shapes, dtype, grad_dtype=None, seed=0):
    g = gen(seed)
    params = [torch.randn(s, generator=g, device="cuda").to(dtype) for s in shapes]
    return params, lambda k: [(torch.randn(s, generator=gen(100 * k + i), device="cuda") *
                               torch.exp2(torch.randint(-12, 4, s, generator=gen(k), device="cuda").float())
                               ).to(grad_dtype or dtype) for i, s in enumerate(shapes)]


def steps(params, grads, state, count, scale=None, **hyper):
    hyper = {**HYPER, **hyper}
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    start = int(state.step[0])
    for k in range(count):
        g = grads(k)
        adamw_step(params, g, state, grad_scale=scale, **hyper)
        for i, one in enumerate(plain):
            one.step(g[i], start + k + 1, scale=1.0 if scale is None else float(scale), **hyper)
            one.check(params[i], state, i)
    assert state.step.tolist() == [start + count, 0]


SHAPES = [(1,), (31, 3), (32,), (7, 129), (2048,), (2049,), (64, 1000), (3, 5, 7)]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("dtype,grad_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16), (F16, BF16)])
def test_steps(dev, dtype, grad_dtype, masters, bits):
    params, grads = tensors(SHAPES, dtype, grad_dtype)
    state = adamw_state(params, bits=bits, masters=masters, seed=77)
    assert (state.masters is not None) == (masters and dtype != F32)
    steps(params, grads, state, 4)


@pytest.mark.parametrize("bits", [8, 32])
def test_scalars_on_the_device(dev, bits):
    params, grads = tensors(SHAPES, F32)
    state = adamw_state(params, bits=bits)
    rate, scale = torch.tensor(3e-4, device=dev), torch.tensor([0.37], device=dev)
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    g = grads(0)
    adamw_step(params, g, state, rate, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.0, grad_scale=scale)
    for i, one in enumerate(plain):
        one.step(g[i], 1, float(rate), (0.8, 0.95), 1e-6, 0.0, float(scale))
        one.check(params[i], state, i)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_of_many_steps_and_many_tensors(dev, bits):
    # more tensors than one launch takes, of several types, some empty, some without a gradient
    g = gen(5)
    dtypes = [F32, BF16, F16]
    params = [torch.randn(1 + 37 * i % 300, generator=g, device=dev).to(dtypes[i % 3]) for i in range(150)]
    params[10] = torch.empty(0, device=dev)
    grads = [None if i % 7 == 3 else torch.randn(p.shape, generator=g, device=dev).to(dtypes[i // 2 % 3])
             for i, p in enumerate(params)]
    state = adamw_state(params, bits=bits, masters=False, seed=2**32 - 1)
    state.step[0] = 123456
    before = [(p.clone(), m.clone()) for p, m in zip(params, state.moments)]
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    adamw_step(params, grads, state, **HYPER)
    for i, one in enumerate(plain):
        if grads[i] is None or params[i].numel() == 0:
            assert torch.equal(params[i], before[i][0]) and torch.equal(state.moments[i], before[i][1])
        else:
            one.step(grads[i], 123457, **HYPER)
            one.check(params[i], state, i)
    assert state.step.tolist() == [123457, 0]


def test_nothing_to_do_still_counts(dev):
    p = torch.randn(5, device=dev)
    state = adamw_state([p])
    adamw_step([p], [None], state, 1e-3)
    assert state.step.tolist() == [1, 0]


def test_gradients_of_any_strides_and_values_at_any_place(dev):
    base = torch.randn(3 * 40 * 50 + 1, generator=gen(6), device=dev)
    params = [base[1:2001].view(40, 50), base[2001:4001].view(40, 50)]  # not aligned to 16 bytes
    rest = base[4001:].clone(), base[0].clone()
    wide = torch.randn(50, 90, generator=gen(7), device=dev)
    grads = [wide[:, :40].t(), torch.tensor(0.25, device=dev).expand(40, 50)]
    state = adamw_state(params)
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    adamw_step(params, grads, state, **HYPER)
    for i, one in enumerate(plain):
        one.step(grads[i], 1, **HYPER)
        one.check(params[i], state, i)
    assert torch.equal(base[4001:], rest[0]) and torch.equal(base[0], rest[1])


@pytest.mark.parametrize("bits", [8, 32])
def test_values_that_are_not_finite(dev, bits):
    params, grads = tensors([(256,)], F32)
    state = adamw_state(params, bits=bits)
    g = grads(0)
    g[0][40], g[0][100], g[0][200] = float("nan"), float("inf"), 3e38  # the last one's square is infinite
    one = Plain(params[0], state, 0)
    adamw_step(params, g, state, **HYPER)
    one.step(g[0], 1, **HYPER)
    one.check(params[0], state, 0)
    if bits == 8:  # a block is NaN as a whole
        values = adamw_moments(state)[0]
        bad = torch.isnan(values).view(2, 8, 32).all(2)
        assert bad.tolist() == [[i in (1, 3) for i in range(8)], [i in (1, 3, 6) for i in range(8)]]


def test_moments_near_the_ends_of_the_range(dev):
    for power in (-140, -126, -64, -20, 0, 40):
        params = [torch.ones(512, device=dev)]
        state = adamw_state(params, bits=8)
        g = torch.randn(512, generator=gen(power + 200), device=dev) * 2.0**power
        one = Plain(params[0], state, 0)
        adamw_step(params, [g], state, **HYPER)
        one.step(g, 1, **HYPER)
        one.check(params[0], state, 0)


def test_moments_are_the_values_of_the_codes(dev):
    for second in (0, 1):
        codes = torch.zeros(2, 256 * 32, dtype=torch.uint8, device=dev)
        codes[second] = torch.arange(256, device=dev).repeat(32).to(torch.uint8)
        exponents = torch.zeros(2, 256, dtype=torch.uint8, device=dev)
        exponents[second] = torch.arange(256, device=dev).to(torch.uint8)
        state = AdamWState([codes], [exponents], None, torch.zeros(2, dtype=torch.int32, device=dev))
        got = adamw_moments(state)[0][second].cpu()
        want = torch.from_numpy(decode(codes[second].cpu().numpy(), exponents[second].cpu().numpy(), second))
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.float().nan_to_num(0.0))  # rounded once where subnormal


def test_slow_changes_add_up_in_8_bits(dev):
    # gradients of one size, below what v holds: beta2 moves v by a thousandth of the way each step, which rounding to the
    # nearest of 8 codes per power of two would never show.  Each of the n values takes up to 400 roundings at random, of
    # steps of at most v / 8 and each with a variance of at most a quarter step squared; the mean over n is then off by
    # under v / 16 * sqrt(400 / n), four deviations of which are allowed.
    n = 1 << 16
    p = [torch.zeros(n, device=dev)]
    state = adamw_state(p, bits=8)
    state.moments[0][1], state.exponents[0][1] = 231, 127  # (31 + 7 / 8) / 32 of 4: code (28 << 3) + 7, 2^-2 * 1.875
    start = float(adamw_moments(state)[0][1, 0])
    g = [torch.full((n,), 0.3, device=dev)]
    for _ in range(400):
        adamw_step(p, g, state, lr=0.0)
    want = start * 0.999**400 + 0.09 * (1 - 0.999**400)
    got = adamw_moments(state)[0][1].double().mean().item()
    assert abs(got - want) <= 4 * start / 16 * (400 / n)**0.5


def test_a_captured_step_counts_and_rounds_anew(dev):
    params, grads = tensors([(3000,), (17, 5)], BF16)
    state = adamw_state(params, bits=8, seed=3)
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    held = grads(0)
    rate = torch.tensor([1e-3], device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adamw_step(params, held, state, rate, **{k: v for k, v in HYPER.items() if k != "lr"})
    for k in range(4):
        for a, b in zip(held, grads(k)):
            a.copy_(b)
        rate.fill_(1e-3 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        for i, one in enumerate(plain):
            one.step(held[i], k + 1, **{**HYPER, "lr": float(rate)})
            one.check(params[i], state, i)


def test_two_runs_are_the_same(dev):
    def run():
        params, grads = tensors([(70000,), (33, 1000)], BF16)
        state = adamw_state(params, bits=8, seed=9)
        for k in range(3):
            adamw_step(params, grads(k), state, **HYPER)
        return params + state.moments + state.exponents

    for a, b in zip(run(), run()):
        assert torch.equal(a, b)


def test_another_stream(dev):
    params, grads = tensors([(5000,)], F32)
    state = adamw_state(params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps(params, grads, state, 2)


def test_a_value_that_a_backward_pass_needs_is_noticed(dev):
    p = torch.randn(4, device=dev, requires_grad=True)
    loss = (p * p).sum()
    adamw_step([p], [torch.ones_like(p)], adamw_state([p]), 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert p.requires_grad and p.is_leaf


@pytest.mark.parametrize("bits", [8, 32])
def test_a_large_tensor(dev, bits):
    # more chunks than workgroups, and a place past 2^24
    n = (1 << 25) + 77
    p = [torch.ones(n, device=dev, dtype=BF16)]
    g = [torch.full((n,), 1e-2, device=dev, dtype=BF16)]
    state = adamw_state(p, bits=bits, masters=False)
    adamw_step(p, g, state, lr=0.25, weight_decay=0.0)
    assert torch.equal(p[0], torch.full_like(p[0], 0.75))  # m / sqrt(v) is 1 to 2^-20, the change a quarter
    m = adamw_moments(state)[0]
    want = float(g[0][0].float()) * 0.1
    assert bool((m[0, :n] - want).abs().max() <= (want / 8 if bits == 8 else want * 2**-23))
    assert not m[:, n:].any()


def test_random_numbers_by_given_factors(dev, monkeypatch):
    first, second = 0x6A09E667, 0xBB67AE85  # the first bits of the roots of 2 and 3

    def other(x):
        x = x ^ (x >> 16)
        x = (x * first) & 0xFFFFFFFF
        x = x ^ (x >> 15)
        x = (x * second) & 0xFFFFFFFF
        return x ^ (x >> 16)

    params, grads = tensors(SHAPES, BF16)
    state = adamw_state(params, bits=8, seed=77)._replace(factors=(0x9B05688D, 0x5BE0CD19))
    steps(params, grads, state, 2)  # the library's own
    monkeypatch.setitem(globals(), "mix", other)
    steps(params, grads, state._replace(factors=(first, second)), 2)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_after_a_second_moment_that_is_not_finite(dev, bits):
    # one gradient's square is infinite: 8-bit moments make a NaN of v's whole block, under an m that stays finite, and
    # with it of the block's values from the next step on
    params, grads = tensors([(256,), (40,)], F32)
    state = adamw_state(params, bits=bits)
    plain = [Plain(p, state, i) for i, p in enumerate(params)]
    for k in range(3):
        g = grads(k)
        if k == 0:
            g[0][200] = 3e38
        adamw_step(params, g, state, **HYPER)
        for i, one in enumerate(plain):
            one.step(g[i], k + 1, **HYPER)
            one.check(params[i], state, i)
    bad = torch.isnan(params[0]).view(8, 32).all(1) if bits == 8 else torch.isnan(params[0])
    assert bad.nonzero().flatten().tolist() == ([6] if bits == 8 else []) and not torch.isnan(params[1]).any()


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_that_share_memory_are_refused(dev, bits):
    base = torch.randn(300, generator=gen(8), device=dev)
    params = [base[:100], base[100:200], base[200:].to(BF16)]
    grads = [torch.ones_like(p) for p in params]
    state = adamw_state(params, bits=bits)
    before = [t.clone() for t in params + state.moments + state.masters]

    def refused(p, s):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(p, grads, s, 1e-3)

    def twice(list_):
        return [list_[0], list_[0], list_[2]]

    refused([params[0], params[0], params[2]], state)
    refused([params[0], base[99:199], params[2]], state)
    refused(params, state._replace(moments=twice(state.moments)))
    refused(params, state._replace(masters=twice(state.masters)))
    refused(params, state._replace(masters=[state.masters[0], base[:100], state.masters[2]]))
    if bits == 8:
        refused(params, state._replace(exponents=twice(state.exponents)))
    assert all(torch.equal(a, b) for a, b in zip(before, params + state.moments + state.masters))
    assert state.step.tolist() == [0, 0]
    # a parameter in fp32 that is its own master, neighbours in one tensor, a shared gradient
    own = state._replace(masters=[params[0], params[1], state.masters[2]])
    shared = [grads[0], grads[0], grads[2]]
    plain = [Plain(p, own, i) for i, p in enumerate(params)]
    adamw_step(params, shared, own, **HYPER)
    for i, one in enumerate(plain):
        one.step(shared[i], 1, **HYPER)
        one.check(params[i], own, i)


def test_a_step_of_one_count(dev):
    params, grads = tensors([(100,)], F32)
    state = adamw_state(params)._replace(step=torch.zeros(1, dtype=torch.int32, device=dev))
    one = Plain(params[0], state, 0)
    for k in range(2):
        adamw_step(params, grads(k), state, **HYPER)
        one.step(grads(k)[0], k + 1, **HYPER)
        one.check(params[0], state, 0)
    assert state.step.tolist() == [2]
    with pytest.raises(ValueError, match="step"):
        adamw_step(params, grads(0), state._replace(step=state.step[:0]), 1e-3)


@pytest.mark.parametrize("second", [0, 1])
def test_roundings_are_to_a_neighbour_and_even_on_the_mean(dev, second):
    # Moments that are the gradients themselves (or their squares): betas of 0.  Each block has the same 32 values, a large
    # one beside ones down to under the format's least, of either sign; over many blocks each becomes one of the two codes'
    # values beside it, and on the mean itself.  n roundings by up to a step s have a deviation of at most s / 2 / sqrt(n);
    # five of them, and the 16 bits of a random number, are allowed.
    g = np.concatenate([[1.9], 2.0 ** (-0.6 * np.arange(31))]).astype(np.float32) * np.float32(37.0)
    g[1::3] *= -1
    assert g.size == 32
    n = 1 << 15  # blocks
    p = [torch.zeros(32 * n, device=dev)]
    state = adamw_state(p, bits=8, seed=11)
    adamw_step(p, [torch.from_numpy(g).to(dev).repeat(n)], state, lr=0.0, betas=(0.0, 0.0))
    got = adamw_moments(state)[0][second].double().view(n, 32).cpu().numpy()
    want = (g * g if second else g).astype(np.float64)
    # every value of the format under this block's exponent, from its definition
    exponent = np.uint8((np.abs(want).max().astype(np.float32).view(np.uint32) >> 23) & 255)
    codes = np.arange(256, dtype=np.uint8)
    values = np.unique(decode(codes, np.full(8, exponent), second))
    assert (state.exponents[0][second] == int(exponent)).all() and np.isin(got, values).all()
    for j, x in enumerate(want):
        below, above = values[values <= x].max(), values[values >= x].min()
        if second and below == 0:  # v that is not zero never becomes zero
            assert (got[:, j] == above).all()
            continue
        assert ((got[:, j] == below) | (got[:, j] == above)).all(), j
        step = above - below
        assert abs(got[:, j].mean() - x) <= step * (5 / 2 / n**0.5 + 2.0**-16), j
        if step > 0 and abs(x - below) / step > 0.05 and abs(above - x) / step > 0.05:
            assert (got[:, j] == below).any() and (got[:, j] == above).any()


def test_the_moments_of_a_value_are_rounded_apart(dev):
    # both moments half way between two codes: up or down independently, and so do neighbours
    n = 1 << 16
    p = [torch.zeros(n, device=dev)]
    state = adamw_state(p, bits=8, seed=12)
    grad = torch.full((n,), 1.0 + 1.0 / 16, device=dev)  # half way; its square, 1.12890625, is 0.03125 parts from it
    adamw_step(p, [grad], state, lr=0.0, betas=(0.0, 0.0))
    m, v = (x.cpu().numpy() for x in adamw_moments(state)[0])
    assert set(np.unique(m)) == {1.0, 1.125} and set(np.unique(v)) == {1.125, 1.25}
    up_m, up_v = (m == 1.125).astype(float), (v == 1.25).astype(float)
    chance_v = (1.12890625 - 1.125) / 0.125
    assert abs(up_m.mean() - 0.5) <= 5 * 0.5 / n**0.5
    assert abs(up_v.mean() - chance_v) <= 5 * (chance_v * (1 - chance_v) / n) ** 0.5
    # the covariance of independent ones has the deviation sqrt(var var / n)
    both = ((up_m - 0.5) * (up_v - chance_v)).mean()
    assert abs(both) <= 5 * 0.5 * (chance_v * (1 - chance_v)) ** 0.5 / n**0.5
    for d in (1, 32, 2048):
        assert abs(((up_m - 0.5) * (np.roll(up_m, d) - 0.5)).mean()) <= 5 * 0.25 / n**0.5
