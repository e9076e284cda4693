"""Microscaled 4 bits on the GPU: layout against the definition bit by bit, products against sums in 64 bits.

A product's tolerance follows from the arithmetic: a sum of n terms in fp32 is off by at most n * 2^-23 of the sum of their
sizes (each addition rounds by half a step, or cuts by one within a matrix instruction; the terms themselves, of two
bits each times powers of two, are exact), and its rounding to the output's type by half a step more.
"""
import numpy as np
import pytest
import torch

from ops_sparse import MX4, ExpertPlan, expert_plan, grouped_mm_mx4, mx4_dequantize, mx4_quantize

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def definition(x):
    """(codes, scales) of float64 rows [R, K] (numpy), value by value."""
    rows, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :k] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(2)
    most = np.abs(np.where(bad[..., None], 0, v)).max(2)
    e = np.where(most > 0, np.frexp(most)[1] - 3, -127)  # frexp's exponent is one above floor(log2)
    e = np.clip(e, -127, 125)
    a = np.abs(np.where(bad[..., None], 0, v)) / np.ldexp(1.0, e)[..., None]
    code = np.zeros(a.shape, np.int64)
    far = np.abs(a[..., None] - VALUES)
    best = far.min(-1)
    for i in (1, 3, 5, 7, 0, 2, 4, 6):  # of two equally near the even code, which is looked at last
        code = np.where(far[..., i] == best, i, code)
    code += np.where(np.signbit(v) & ~bad[..., None], 8, 0)
    code = code.reshape(rows, blocks * 32)
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    """The float64 values of numpy codes [..., 16 B] and scales [..., B]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = VALUES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, 32, -1)


def same(q, x):
    codes, scales = definition(x.reshape(-1, x.shape[-1]))
    blocks = scales.shape[-1]
    assert q.codes.shape == (*x.shape[:-1], blocks * 16) and q.scales.shape == (*x.shape[:-1], blocks)
    assert np.array_equal(q.scales.cpu().numpy().reshape(-1, blocks), scales)
    assert np.array_equal(q.codes.cpu().numpy().reshape(-1, blocks * 16), codes)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 31), (2, 32), (5, 33), (4, 8), (7, 520), (1, 4096), (3, 5, 100),
                                   (2000, 65), (257, 16384)])
def test_quantize(dev, shape, dtype):
    x = torch.randn(shape, generator=gen(shape[-1]), device=dev) * torch.exp2(
        torch.randint(-30 if dtype == F32 else -6, 10, shape, generator=gen(1), device=dev).float())
    x = x.to(dtype)
    q = mx4_quantize(x)
    same(q, x.double().cpu().numpy())
    back = mx4_dequantize(q, shape[-1], dtype)
    want = values(q.codes.cpu().numpy(), q.scales.cpu().numpy())[..., :shape[-1]]
    want = torch.from_numpy(want).to(dtype)  # exact in fp32 and bf16; fp16's subnormals are rounded once
    assert torch.equal(back.cpu(), want)


def test_quantize_ties_and_every_border(dev):
    # every half step of the format and its neighbours, under a largest value of 4 to 7.99 times the scale
    steps = np.arange(0, 8.25, 0.125)
    for top in (4.0, 5.0, 6.0, 7.0, 7.9375):
        for power in (-20, 0, 9):
            near = [steps, np.nextafter(np.float32(steps), np.float32(9)), np.nextafter(np.float32(steps), np.float32(0))]
            v = np.concatenate([s[s <= top] for s in near]).astype(np.float32)
            v = np.concatenate([v, -v])
            v = v[:v.size // 31 * 31].reshape(-1, 31)
            x = np.concatenate([v, np.full((len(v), 1), top, np.float32)], 1) * np.float32(2.0 ** power)
            same(mx4_quantize(torch.from_numpy(x).to(dev)), x.astype(np.float64))


def test_quantize_ends_of_the_range(dev):
    tiny, huge = 2.0**-149, float(np.finfo(np.float32).max)
    rows = [[0.0] * 32, [-0.0] * 32, [tiny] * 32, [2.0**-126] * 32, [2.0**-125] * 31 + [1e-45], [huge] * 32,
            [-huge] + [1.0] * 31, [2.0**127] + [2.0**125] * 31, [2.0**-127 * 3] * 32]
    x = torch.tensor(rows, dtype=F32, device=dev)
    same(mx4_quantize(x), x.double().cpu().numpy())
    q = mx4_quantize(x)
    want = torch.from_numpy(values(q.codes.cpu().numpy(), q.scales.cpu().numpy())).float()
    assert torch.equal(mx4_dequantize(q).cpu(), want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_quantize_values_that_are_not_finite(dev, dtype):
    x = torch.randn(4, 96, generator=gen(3), device=dev).to(dtype)
    x[0, 5], x[1, 40], x[2, 95] = float("nan"), float("inf"), -float("inf")
    q = mx4_quantize(x)
    same(q, x.double().cpu().numpy())
    back = mx4_dequantize(q, 96, dtype)
    bad = torch.zeros(4, 3, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(torch.isnan(back).cpu(), bad.repeat_interleave(32, 1))


def test_quantize_strides(dev):
    big = torch.randn(40, 300, generator=gen(4), device=dev)
    for x in (big[::2, 3:103], big[:, 1:], big.t(), big[5], big[:, 7:8], big.unflatten(0, (8, 5))[:, 1:4, :77]):
        same(mx4_quantize(x), x.double().cpu().numpy())
    for x in (big[:0], big[:, :0]):
        q = mx4_quantize(x)
        assert q.codes.numel() == 0 and mx4_dequantize(MX4(q.codes, q.scales)).numel() == 0
    q = mx4_quantize(big)
    part = MX4(q.codes[1::3, 16:64], q.scales[1::3, 1:4])
    assert torch.equal(mx4_dequantize(part), mx4_dequantize(q)[1::3, 32:128])


# ------------------------------------------------------------------------------------------------------ products


def rows_of(rows, k, seed, lead=()):
    """Random rows with scales over some powers of two, as codes and scales and in float64 on the GPU."""
    g = gen(seed)
    x = torch.randn(*lead, rows, k, generator=g, device="cuda") * torch.exp2(
        torch.randint(-4, 5, (*lead, rows, (k + 31) // 32), generator=g, device="cuda").float()
    ).repeat_interleave(32, -1)[..., :k]
    return mx4_quantize(x)


def exact_rows(q):
    return torch.from_numpy(values(q.codes.cpu().numpy(), q.scales.cpu().numpy())).cuda()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(y, a, w, offsets, index, dtype):
    """y against the sums in 64 bits over groups; a, w: MX4."""
    xa, xw = exact_rows(a), exact_rows(w)
    rows = y.shape[0]
    want, size = torch.zeros(rows, xw.shape[1], dtype=torch.float64, device="cuda"), None
    size = torch.zeros_like(want)
    for g in range(xw.shape[0]):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        if lo < hi:
            part = xa[index[lo:hi].long()] if index is not None else xa[lo:hi]
            want[lo:hi] = torch.mm(part, xw[g].t().contiguous())
            size[lo:hi] = torch.mm(part.abs(), xw[g].abs().t().contiguous())
    assert y.dtype == dtype
    bound = size * xa.shape[1] * 2.0**-23
    bound = bound + (want.abs() + bound) * half_step(dtype) + (2.0**-25 if dtype == F16 else 2.0**-149)
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


SHAPES = [  # groups' lengths, n, k: what reaches each kernel stands behind
    ([1], 16, 32), ([1], 1, 1), ([2], 17, 33), ([5, 0, 1], 33, 250),            # few rows
    ([1, 1, 0, 1], 4096, 2048), ([30], 100, 1000), ([33], 64, 96), ([64], 48, 4100),
    ([70, 0, 3], 129, 257), ([100, 64, 65], 200, 256), ([7, 500], 128, 224),    # 64x128 tiles
    ([256], 256, 3104), ([130, 20], 300, 2300),                                # with three teams
    ([2500], 2048, 288), ([2305], 1500, 512), ([700, 0, 900, 1300], 700, 520),  # 256x256 tiles and their parts
    ([3000, 65], 1100, 2000),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,n,k", SHAPES)
def test_product(dev, lens, n, k, dtype):
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)
    rows = int(offsets[-1])
    a, w = rows_of(rows, k, 1), rows_of(n, k, 2, (len(lens),))
    y = grouped_mm_mx4(a, w, ExpertPlan(offsets), out_dtype=dtype)
    check(y, a, w, offsets, None, dtype)
    if len(lens) == 1:
        assert torch.equal(grouped_mm_mx4(a, MX4(w.codes[0], w.scales[0]), out_dtype=dtype), y)


@pytest.mark.parametrize("tokens,experts,k,n,width", [(1, 8, 3, 40, 96), (37, 6, 2, 130, 640), (900, 4, 2, 520, 300),
                                                     (2000, 3, 2, 600, 256)])
def test_product_gathers(dev, tokens, experts, k, n, width):
    ids = torch.argsort(torch.rand(tokens, experts, generator=gen(5), device=dev), dim=1)[:, :k].to(torch.int32)
    plan = expert_plan(ids, experts)
    a, w = rows_of(tokens, width, 6), rows_of(n, width, 7, (experts,))
    check(grouped_mm_mx4(a, w, plan, gather=True), a, w, plan.offsets, plan.tokens, BF16)


@pytest.mark.parametrize("lens", [[3, 4], [90, 150], [1500, 1400]])
def test_product_rows_of_no_expert_are_zero(dev, lens):
    offsets = torch.tensor([5, 5 + lens[0], 5 + sum(lens)], dtype=torch.int32, device=dev)
    rows = int(offsets[-1]) + 9
    a, w = rows_of(rows, 320, 8), rows_of(600, 320, 9, (2,))
    torch.full((rows, 600), float("nan"), device=dev)  # what memory holds
    y = grouped_mm_mx4(a, w, ExpertPlan(offsets), out_dtype=F32)
    check(y, a, w, offsets, None, F32)
    assert not y[:5].any() and not y[-9:].any()


@pytest.mark.parametrize("rows,n,k", [(3, 40, 520), (100, 200, 520), (2500, 2048, 520)])
def test_product_strides(dev, rows, n, k):
    # blocks inside longer rows, groups apart, scales at odd places, codes that are not aligned
    a, w = rows_of(rows, k + 96, 10), rows_of(n + 3, k + 96, 11, (4,))
    blocks = (k + 31) // 32
    pa = MX4(a.codes[:, 16:16 + 16 * blocks], a.scales[:, 1:1 + blocks])
    pw = MX4(w.codes[1::2, 2:-1, 16:16 + 16 * blocks], w.scales[1::2, 2:-1, 1:1 + blocks])
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=dev)
    want = grouped_mm_mx4(MX4(*(t.contiguous() for t in pa)), MX4(*(t.contiguous() for t in pw)), ExpertPlan(offsets))
    check(want, pa, pw, offsets, None, BF16)
    assert torch.equal(grouped_mm_mx4(pa, pw, ExpertPlan(offsets)), want)
    shifted = torch.empty(pa.codes.numel() + 5, dtype=torch.uint8, device=dev)[5:].view(rows, -1)
    shifted.copy_(pa.codes)
    assert torch.equal(grouped_mm_mx4(MX4(shifted, pa.scales), pw, ExpertPlan(offsets)), want)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 520), (100, 200, 520), (2500, 2048, 520)])
def test_product_of_nan_and_range(dev, rows, n, k):
    a, w = rows_of(rows, k, 12), rows_of(n, k, 13, (1,))
    clean = grouped_mm_mx4(a, w, ExpertPlan(torch.tensor([0, rows], dtype=torch.int32, device=dev)), out_dtype=F32)
    a.scales[1, 2], w.scales[0, 7, 16] = 255, 255  # one block of a row of each, the last one cut by the width
    y = grouped_mm_mx4(a, MX4(w.codes[0], w.scales[0]), out_dtype=F32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[~bad])
    # scales at the ends: products of 2^127 * 2^-127, and zeros under the largest scale
    a.scales.fill_(254)
    w.scales.fill_(0)
    a.codes[0] = 0
    y = grouped_mm_mx4(a, MX4(w.codes[0], w.scales[0]), out_dtype=F32)
    offsets = torch.tensor([0, rows], dtype=torch.int32)
    check(y, a, w, offsets, None, F32)
    assert not y[0].any()


def test_product_of_nothing(dev):
    a, w = rows_of(4, 64, 14), rows_of(6, 64, 15, (2,))
    empty = MX4(a.codes[:, :0], a.scales[:, :0]), MX4(w.codes[..., :0], w.scales[..., :0])
    plan = ExpertPlan(torch.tensor([0, 1, 4], dtype=torch.int32, device=dev))
    assert not grouped_mm_mx4(*empty, plan).any()
    assert grouped_mm_mx4(MX4(a.codes[:0], a.scales[:0]), w, ExpertPlan(plan.offsets * 0)).shape == (0, 6)
    assert grouped_mm_mx4(a, MX4(w.codes[:, :0], w.scales[:, :0]), plan).shape == (4, 0)


def test_offsets_and_indices_without_meaning_stay_inside(dev):
    a, w = rows_of(700, 300, 16), rows_of(520, 300, 17, (3,))
    for offsets in ([0, -5, 9000, 3], [900, 1, 2, 2**31 - 1], [-2**31, 2**31 - 1, -1, 700], [700, 0, 700, 0]):
        index = torch.randint(-2**31, 2**31 - 1, (700,), generator=gen(18), device=dev).to(torch.int32)
        plan = ExpertPlan(torch.tensor(offsets, dtype=torch.int32, device=dev), index)
        assert grouped_mm_mx4(a, w, plan, gather=True).shape == (700, 520)
    torch.cuda.synchronize()


def test_serving_in_a_graph_on_another_stream(dev):
    x = torch.randn(33, 200, generator=gen(19), device=dev).bfloat16()
    w = rows_of(160, 200, 20, (4,))
    ids = torch.argsort(torch.rand(33, 4, generator=gen(21), device=dev), dim=1)[:, :2].to(torch.int32)

    def serve():
        plan = expert_plan(ids, 4)
        return mx4_dequantize(mx4_quantize(grouped_mm_mx4(mx4_quantize(x), w, plan, gather=True)))

    want = serve()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(serve(), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serve()
    for seed in range(3):
        x.copy_(torch.randn(33, 200, generator=gen(seed), device=dev))
        ids.copy_(torch.argsort(torch.rand(33, 4, generator=gen(seed), device=dev), dim=1)[:, :2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, serve())


# Shapes by the kernel that they reach on a chip of 256 CUs; test_model_ops_abi.py looks that they do.
KERNELS = ("16 rows", "32 rows", "32 rows by 32", "256x256", "64x128", "64x128 by teams")
REACHED = [  # kernel, groups' lengths, n, k
    ("16 rows", [5, 0, 1, 16], 70, 200), ("32 rows", [31, 20], 50, 1100), ("32 rows by 32", [64, 0, 70], 100, 500),
    ("64x128", [130, 20], 300, 2300), ("64x128", [70, 130, 65], 257, 500), ("64x128", [700, 900], 520, 96),
    ("64x128 by teams", [130, 20], 300, 3200), ("64x128 by teams", [200, 0, 100, 65], 520, 4001),
    ("64x128 by teams", [300], 130, 8200),
    # tiles' last rows of any number, halves of tiles in a die's last round
    ("256x256", [3300], 2048, 288), ("256x256", [2500, 0, 700, 1300], 2200, 520), ("256x256", [3000, 65], 2100, 2000),
    # whole tiles in the last round, and last tiles of 64, 128, 129, 1 and 130 rows; rows of fewer than 16 blocks
    ("256x256", [1088, 2176, 1153, 2049, 1154], 1100, 96), ("256x256", [5250], 2200, 512),
    # a die's last round in quarters
    ("256x256", [256 * 33], 2048, 64), ("256x256", [256 * 16, 256 * 17 - 40], 2041, 545),
]


def no_expert(lens, head, tail):
    """Offsets with `head` rows before the first group and `tail` behind the last, and the number of rows."""
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(lens)]) + head, dtype=torch.int32, device="cuda")
    return offsets, int(offsets[-1]) + tail


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kernel,lens,n,k", REACHED)
def test_products_of_each_kernel(dev, kernel, lens, n, k, dtype):
    offsets, rows = no_expert(lens, 0, 0)
    a, w = rows_of(rows, k, 30), rows_of(n, k, 31, (len(lens),))
    check(grouped_mm_mx4(a, w, ExpertPlan(offsets), out_dtype=dtype), a, w, offsets, None, dtype)


NO_EXPERT = [("256x256", [1500, 2000], 2100, 320), ("64x128 by teams", [130, 90], 520, 3300),
             ("64x128", [130, 90], 520, 330), ("32 rows by 32", [64, 0, 70], 100, 500)]


@pytest.mark.parametrize("kernel,lens,n,k", NO_EXPERT)
def test_rows_of_no_expert_in_each_kernel(dev, kernel, lens, n, k):
    offsets, rows = no_expert(lens, 5, 9)
    a, w = rows_of(rows, k, 32), rows_of(n, k, 33, (len(lens),))
    torch.full((rows, n), float("nan"), device=dev)  # what memory holds
    y = grouped_mm_mx4(a, w, ExpertPlan(offsets), out_dtype=F32)
    check(y, a, w, offsets, None, F32)
    assert not y[:5].any() and not y[-9:].any()


GATHERED = [("256x256", 4000, 4, 2, 1100, 300), ("64x128 by teams", 300, 4, 2, 300, 3300)]


@pytest.mark.parametrize("kernel,tokens,experts,chosen,n,k", GATHERED)
def test_gathered_products_of_tiles(dev, kernel, tokens, experts, chosen, n, k):
    ids = torch.argsort(torch.rand(tokens, experts, generator=gen(34), device=dev), dim=1)[:, :chosen].to(torch.int32)
    plan = expert_plan(ids, experts)
    a, w = rows_of(tokens, k, 35), rows_of(n, k, 36, (experts,))
    check(grouped_mm_mx4(a, w, plan, gather=True), a, w, plan.offsets, plan.tokens, BF16)


@pytest.mark.parametrize("k", [290, 520])
def test_strides_and_nan_in_large_tiles(dev, k):
    # blocks inside longer rows, groups apart, scales at odd places
    rows, n, blocks = 3300, 2048, (k + 31) // 32
    a, w = rows_of(rows, k + 96, 37), rows_of(n + 3, k + 96, 38, (4,))
    pa = MX4(a.codes[:, 16:16 + 16 * blocks], a.scales[:, 1:1 + blocks])
    pw = MX4(w.codes[1::2, 2:-1, 16:16 + 16 * blocks], w.scales[1::2, 2:-1, 1:1 + blocks])
    plan = ExpertPlan(torch.tensor([0, 1100, rows], dtype=torch.int32, device=dev))
    want = grouped_mm_mx4(MX4(*(t.contiguous() for t in pa)), MX4(*(t.contiguous() for t in pw)), plan, out_dtype=F32)
    check(want, pa, pw, plan.offsets, None, F32)
    assert torch.equal(grouped_mm_mx4(pa, pw, plan, out_dtype=F32), want)
    # one block of a row of each, the last one cut by the width; what lies beside the rows counts nothing
    a.scales.fill_(255)
    w.scales.fill_(255)
    pa.scales.copy_(MX4(*rows_of(rows, k, 39)).scales)
    pw.scales.copy_(MX4(*rows_of(n, k, 40, (2,))).scales)
    clean = grouped_mm_mx4(pa, pw, plan, out_dtype=F32)
    check(clean, pa, pw, plan.offsets, None, F32)
    pa.scales[1, 2], pw.scales[0, 7, blocks - 1] = 255, 255
    y = grouped_mm_mx4(pa, pw, plan, out_dtype=F32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1], bad[:1100, 7] = True, True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[~bad])


def test_offsets_and_indices_without_meaning_in_large_tiles(dev):
    rows = 3400
    a, w = rows_of(rows, 300, 41), rows_of(2048, 300, 42, (3,))
    for offsets in ([0, -5, 9000, 3], [900, 1, 2, 2**31 - 1], [-2**31, 2**31 - 1, -1, 700], [rows, 0, rows, 0]):
        index = torch.randint(-2**31, 2**31 - 1, (rows,), generator=gen(43), device=dev).to(torch.int32)
        plan = ExpertPlan(torch.tensor(offsets, dtype=torch.int32, device=dev), index)
        assert grouped_mm_mx4(a, w, plan, gather=True).shape == (rows, 2048)
    torch.cuda.synchronize()
