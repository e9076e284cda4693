"""The operators of learning, answering and 4-bit serving as they are measured: the cases, their inputs, one pass.

``listed()`` are the cases, ``draw(rng)`` one more of their ranges; ``prepare(case, seed)`` makes what a program has
in hand before the call, ``run(state)`` makes the call and returns its outputs, ``work(case)`` says what one pass
cannot do without, and ``exact(case, seed)`` gives the outputs in 64 bits.  With ``own`` false ``run`` computes the
operators in elementary torch operations in 32 bits; with ``own`` true it calls this library.

Four operators:
  quantize  rows in microscaled 4-bit floating point (blocks of 32 values that share a power of two), and back
  mx4       y_r = w_e x_i(r) for the rows r of each expert e, both operands in that format; E = 0 is one dense product
  adamw     one AdamW step over many tensors, moments in 32 bits or in microscaled 8-bit floating point
  logprobs  log probabilities of given tokens, with the entropy of each row and its largest alternatives; training:
            the gradient of both
"""
import math
import os
import sys

import torch

own = False

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _api():
    path = os.path.join(_REPO, "ops-sparse_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ops_sparse

    return ops_sparse


def _named(name, **c):
    return dict(c, name=name) if name else c


def _quantize(name, rows, width, dtype="bf16"):
    return _named(name, op="quantize", rows=rows, width=width, dtype=dtype)


def _mx4(name, tokens, experts, k, width, out, skew=0.5):
    return _named(name, op="mx4", tokens=tokens, experts=experts, k=k, width=width, out=out, skew=skew)


def _adamw(name, layers, width, hidden, dtype, bits, master=True, clip=False):
    """A model of `layers` times a matrix, a second one and a vector (the sizes of _shapes)."""
    return _named(name, op="adamw", layers=layers, width=width, hidden=hidden, dtype=dtype, bits=bits, master=master,
                  clip=clip)


def _logprobs(name, rows, vocab, dtype="bf16", top=0, entropy=True, train=False, masked=False):
    return _named(name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, entropy=entropy, train=train,
                  masked=masked)


def listed():
    return [
        # the activations of one decoding request, laid out for a product: latency alone counts
        _quantize("quantize_token", 1, 4096),
        # the rows of a prompt's hidden values, of an odd length, behind the first product of their experts
        _quantize("quantize_prompt", 16381, 4096),
        # one decoding step of one request: four experts' weights are read for one row each
        _mx4("mx4_token", 1, 32, 4, 2048, 4096),
        # a batch of decoding requests over many experts: a few ragged rows each, odd sizes
        _mx4("mx4_batch", 203, 48, 4, 1000, 1001, skew=1.0),
        # a batch through one dense layer around the experts
        _mx4("mx4_dense", 512, 0, 1, 4096, 4096),
        # the prompts of several requests through large experts: the largest
        _mx4("mx4_prompt", 16384, 8, 2, 4096, 4096),
        # fine-tuning a few small tensors: latency alone counts
        _adamw("adamw_small", 2, 520, 776, "f32", 32),
        # a step of a layer of experts in 16 bits with 32-bit master weights, clipped by a norm on the device
        _adamw("adamw_train", 6, 4096, 4096, "bf16", 32, clip=True),
        # the same memory held down: moments in 8 bits, no master weights, sizes that end inside a block
        _adamw("adamw_8bit", 4, 4095, 2049, "bf16", 8, master=False),
        # one decoded token with its alternatives, as an answer reports them
        _logprobs("logprobs_token", 1, 131072, top=20, entropy=False),
        # a batch of answers under a grammar that masks part of the vocabulary
        _logprobs("logprobs_batch", 37, 32003, "f32", top=5, masked=True),
        # a training step's loss on the log probabilities, with an entropy bonus and padded targets
        _logprobs("logprobs_train", 8192, 65536, train=True),
    ]


_MAX_MX4 = 2 * 32768 * 4096 * 4096   # mx4_prompt
_MAX_VALUES = 16381 * 4096           # quantize_prompt
_MAX_PARAMETERS = 100_000_000        # half of adamw_train's
_MAX_LOGITS = 8192 * 65536           # logprobs_train
_MAX_SORTED = 1 << 23                # where the plain form sorts whole rows


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A width: mostly a multiple of 8, as layers have, at times any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(("quantize", "mx4", "mx4", "mx4", "adamw", "adamw", "logprobs", "logprobs"))
    if op == "quantize":
        width = _dim(rng, 32, 16384)
        return _quantize(None, _log(rng, 1, min(65536, _MAX_VALUES // width)), width,
                         rng.choice(("bf16", "f16", "f32")))
    if op == "mx4":
        width, out = _dim(rng, 128, 8192), _dim(rng, 128, 8192)
        tokens = _log(rng, 1, 16384)
        experts = 0 if rng.random() < 0.3 else min(_log(rng, 4, 128), max(4, (1 << 28) // (width * out)))
        k = rng.randint(1, min(8, experts)) if experts else 1
        tokens = max(1, min(tokens, _MAX_MX4 // (2 * k * width * out)))
        return _mx4(None, tokens, experts, k, width, out, rng.choice((0.0, 0.5, 1.0)))
    if op == "adamw":
        layers, width, hidden = rng.randint(1, 6), _log(rng, 8, 4096), _log(rng, 8, 8192)
        layers = max(1, min(layers, _MAX_PARAMETERS // (2 * width * hidden)))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        return _adamw(None, layers, width, hidden, dtype, rng.choice((8, 32)),
                      dtype == "f32" or rng.random() < 0.5, rng.random() < 0.5)
    train = rng.random() < 0.4
    top = 0 if train else rng.choice((0, 1, 5, 20))
    vocab = _dim(rng, 1000, 200000)
    rows = _log(rng, 1, min(8192, (_MAX_SORTED if top else _MAX_LOGITS) // vocab))
    return _logprobs(None, rows, vocab, rng.choice(("bf16", "f16", "f32")), top, rng.random() < 0.7, train,
                     not train and rng.random() < 0.3)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(shape, g, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _rand(shape, g):
    return torch.rand(shape, generator=g, device="cuda")


# ------------------------------------------------------------- microscaled 4 bits: e2m1 values, e8m0 scales, blocks of 32

_VALUES4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^(e - 127) in 32 bits for e in [0, 254], NaN for 255."""
    f = torch.where(e == 0, torch.full_like(e, 0x00400000), e << 23).view(torch.float32)
    return torch.where(e == 255, torch.full_like(f, math.nan), f)


def _to_mx4(x):
    """(codes, scales) of float32 rows [..., K]: the scale's exponent is that of the block's largest value less 2, each
    value the nearest of the format (ties to the even code), at most 6; a block with a value that is not finite is NaN."""
    k = x.shape[-1]
    blocks = (k + 31) // 32
    x = torch.nn.functional.pad(x, (0, blocks * 32 - k)).unflatten(-1, (blocks, 32))
    field = (x.abs().amax(-1).view(torch.int32) >> 23).masked_fill(~torch.isfinite(x).all(-1), 257)
    e = (field - 2).clamp(0, 255)
    a = x * torch.where(e == 255, torch.zeros_like(x[..., 0]), _power((254 - e).clamp(0, 254)))[..., None]
    a = torch.where((e == 255)[..., None], torch.zeros_like(a), a)
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = (code + (torch.signbit(a) * 8)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, e.to(torch.uint8)


def _of_mx4(codes, scales, width, dtype=torch.float32):
    table = torch.tensor([*_VALUES4, *(-v for v in _VALUES4)], device=codes.device, dtype=dtype)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    v = v.unflatten(-1, (scales.shape[-1], 32)) * _power(scales.to(torch.int32)).to(dtype)[..., None]
    return v.flatten(-2)[..., :width]


# ------------------------------------------------------------------- microscaled 8 bits of the moments, blocks of 32

_EMIN = (-13, -29)  # least exponents: of a sign and 7 bits for the first moment, of 8 bits for the second
_MASK = 0xFFFFFFFF


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & _MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & _MASK
    return x ^ (x >> 16)


def _random_bits(n, seed, step, tensor):
    """32 random bits for each of n values: numbers that the seed, the step and the tensor's place in the list give."""
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    key = _mix(_mix(torch.tensor(seed, device="cuda") & _MASK) + (step & _MASK) & _MASK) + tensor & _MASK
    return _mix((i & _MASK) + _mix(key + (i >> 32) & _MASK) & _MASK)


def _to_8(x, bits, second):
    """(codes, exponents) of x [n]: values over 2^e, e the exponent of the block's largest, rounded to 3 bits behind
    the first by 16 random bits."""
    n, emin = x.numel(), _EMIN[second]
    x = torch.nn.functional.pad(x, (0, -n % 32))
    e = x.view(-1, 32).abs().amax(1).view(torch.int32) >> 23
    bad = torch.isnan(x.view(-1, 32)).any(1)
    e = torch.where(bad, torch.full_like(e, 255), e)
    inverse = torch.where(e == 255, torch.zeros_like(e).view(torch.float32), _power((254 - e).clamp(0, 254)))
    a = (x.abs().view(-1, 32) * inverse[:, None]).reshape(-1)
    least = 2.0 ** emin
    shifted = a + least
    first = (emin + 127) << 3
    r = (torch.nn.functional.pad(bits, (0, -n % 32)).to(torch.int32) << 4) + 8
    normal = ((a.view(torch.int32) + r) >> 20) - first + 8
    below = ((shifted.view(torch.int32) + r) >> 20) - first
    code = torch.where(a < least, below, normal)
    if second:
        code = torch.where((a > 0) & (code == 0), torch.ones_like(code), code)
    else:
        code = code + torch.signbit(x).to(torch.int32) * 128
    return torch.where((e == 255).repeat_interleave(32), torch.zeros_like(code), code).to(torch.uint8), e.to(torch.uint8)


def _of_8(codes, exponents, second):
    c = codes.to(torch.int32)
    magnitude = c if second else c & 127
    emin = _EMIN[second]
    normal = (((magnitude >> 3) + (emin + 126)) << 23 | (magnitude & 7) << 20).view(torch.float32)
    v = torch.where(magnitude < 8, magnitude.float() * 2.0 ** (emin - 3), normal)
    if not second:
        v = torch.where(c >= 128, -v, v)
    return (v.view(-1, 32) * _power(exponents.to(torch.int32))[:, None]).reshape(-1)


_HYPER = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _shapes(case):
    w, h = case["width"], case["hidden"]
    return [(h, w), (w, h), (w,)] * case["layers"]


# ------------------------------------------------------------------------------------------------------------ inputs


def _inputs(case, seed):
    g, op, s = _gen(seed), case["op"], {"case": case}
    if op == "quantize":
        # activations: a few channels are much larger than the others
        s["x"] = (_randn((case["rows"], case["width"]), g) * torch.exp(_randn((case["width"],), g, scale=0.7))).to(
            _DTYPE[case["dtype"]])
    elif op == "mx4":
        t, e, k, width, out = (case[n] for n in ("tokens", "experts", "k", "width", "out"))
        s["x"] = _to_mx4(_randn((t, width), g))
        s["w"] = _to_mx4(_randn(((e, out, width) if e else (out, width)), g, scale=1.0 / math.sqrt(width)))
        if e:
            liking = -case["skew"] * torch.log1p(torch.arange(e, device="cuda", dtype=torch.float32))
            liking = liking[torch.randperm(e, generator=g, device="cuda")]
            ids = torch.topk(_randn((t, e), g) + liking, k, dim=1).indices.reshape(-1)
            order = torch.argsort(ids, stable=True)
            offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
            offsets[1:] = torch.cumsum((ids[None, :] == torch.arange(e, device="cuda")[:, None]).sum(1), 0)
            places = torch.empty_like(order)
            places[order] = torch.arange(order.numel(), device="cuda")
            s["plan"] = (offsets, (order // k).to(torch.int32), places.to(torch.int32).reshape(-1, k))
    elif op == "adamw":
        dtype, shapes = _DTYPE[case["dtype"]], _shapes(case)
        s["params"] = [_randn(shape, g, dtype, shape[-1] ** -0.5) for shape in shapes]
        s["grads"] = [_randn(shape, g, dtype, 1e-3) for shape in shapes]
        s["masters"] = [p.float() + p.abs().float() * 1e-3 * (_rand(p.shape, g) - 0.5) for p in s["params"]] if (
            case["master"] and dtype != torch.float32) else None
        s["step"] = torch.tensor([100 + int(seed) % 1000, 0], dtype=torch.int32, device="cuda")
        s["seed"] = int(seed) & 0x7FFFFFFF
        s["clip"] = _rand((1,), g) * 0.5 + 0.5 if case["clip"] else None
        s["moments"], s["exponents"] = [], []
        for shape in shapes:
            n = math.prod(shape)
            padded = (n + 31) // 32 * 32
            m = torch.zeros(2, padded, device="cuda")
            m[0, :n] = _randn((n,), g, scale=3e-4)
            m[1, :n] = (_randn((n,), g, scale=0.7) - 13.8).exp_()  # about 1e-6, over a few orders of magnitude
            if case["bits"] == 8:
                packed = [_to_8(m[i], torch.full((padded,), 1 << 15, device="cuda"), i) for i in range(2)]
                s["moments"].append(torch.stack([c for c, _ in packed]))
                s["exponents"].append(torch.stack([e for _, e in packed]))
            else:
                s["moments"].append(m)
    else:
        rows, vocab = case["rows"], case["vocab"]
        # a model's logits: mostly far below the best few
        x = _randn((rows, vocab), g, scale=2.5)
        x[torch.arange(rows, device="cuda"), torch.randint(0, vocab, (rows,), generator=g, device="cuda")] += 12.0
        s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        if case["masked"]:
            hidden = _rand((rows, vocab), g) < 0.4
            hidden[torch.arange(rows, device="cuda"), s["targets"]] = False
            x = x.masked_fill_(hidden, -math.inf)
        if case["train"]:
            s["targets"] = s["targets"].masked_fill_(_rand((rows,), g) < 0.05, -100)  # the padded ends of sequences
            s["grad"] = _randn((rows,), g, scale=1.0 / rows)
            s["grad_entropy"] = _rand((rows,), g) * (0.01 / rows)
        s["logits"] = x.to(_DTYPE[case["dtype"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        api = _api()
        if case["op"] == "mx4":
            s["x"], s["w"] = api.MX4(*s["x"]), api.MX4(*s["w"])
            if case["experts"]:
                s["plan"] = api.ExpertPlan(*s["plan"])
        elif case["op"] == "adamw":
            s["state"] = api.AdamWState(s["moments"], s["exponents"] if case["bits"] == 8 else None, s["masters"],
                                        s["step"], s["seed"], (0x6A09E667, 0xBB67AE85))  # of _mix
        elif case["op"] == "logprobs" and case["train"]:
            s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------- passes


def _run_own(s):
    api, case = _api(), s["case"]
    if case["op"] == "quantize":
        q = api.mx4_quantize(s["x"])
        return (api.mx4_dequantize(q, case["width"], s["x"].dtype),)
    if case["op"] == "mx4":
        return (api.grouped_mm_mx4(s["x"], s["w"], s.get("plan"), gather=case["experts"] > 0),)
    if case["op"] == "adamw":
        api.adamw_step(s["params"], s["grads"], s["state"], grad_scale=s["clip"], **_HYPER)
        moments = s["moments"]
        if case["bits"] == 8:
            moments = [m[:, :p.numel()] for m, p in zip(api.adamw_moments(s["state"]), s["params"])]
        return {"params": s["params"], "masters": s["masters"], "moments": moments}
    r = api.token_logprobs(s["logits"], s["targets"], top=case["top"], entropy=case["entropy"])
    outs = [t.detach() for t in r if t is not None]
    if case["train"]:
        given = (r.logprobs, r.entropy) if case["entropy"] else (r.logprobs,)
        outs += torch.autograd.grad(given, s["logits"], (s["grad"], s["grad_entropy"])[:len(given)])
    return outs


def _plain_quantize(s):
    return (_of_mx4(*_to_mx4(s["x"].float()), s["case"]["width"]).to(s["x"].dtype),)


def _plain_mx4(s):
    case = s["case"]
    width = case["width"]
    x = _of_mx4(*s["x"], width)
    if not case["experts"]:
        return ((x @ _of_mx4(*s["w"], width).t()).to(torch.bfloat16),)
    offsets, tokens, _ = s["plan"]
    off = offsets.tolist()
    x = x[tokens]
    y = torch.empty(x.shape[0], case["out"], device="cuda", dtype=torch.bfloat16)
    for e in range(case["experts"]):
        if off[e] < off[e + 1]:
            y[off[e]:off[e + 1]] = x[off[e]:off[e + 1]] @ _of_mx4(s["w"][0][e], s["w"][1][e], width).t()
    return (y,)


def _plain_adamw(s):
    case, (b1, b2) = s["case"], _HYPER["betas"]
    lr, wd = _HYPER["lr"], _HYPER["weight_decay"]
    s["step"][0] += 1
    t = s["step"][:1].double()
    size, root = (lr / (1.0 - b1 ** t)).float(), (1.0 - b2 ** t).sqrt().float()
    moments = []
    for i, (p, grad) in enumerate(zip(s["params"], s["grads"])):
        n = p.numel()
        g = grad.reshape(-1).float()
        if s["clip"] is not None:
            g = g * s["clip"]
        held = s["moments"][i]
        old = [_of_8(held[j], s["exponents"][i][j], j)[:n] for j in range(2)] if case["bits"] == 8 else held[:, :n]
        m = old[0] * b1 + g * (1.0 - b1)
        v = old[1] * b2 + (g * g) * (1.0 - b2)
        value = (s["masters"][i] if s["masters"] is not None else p).reshape(-1)
        new = value.float() * (1.0 - lr * wd) - size * (m / (v.sqrt() / root + _HYPER["eps"]))
        if s["masters"] is not None:
            value.copy_(new)
        p.view(-1).copy_(new)
        if case["bits"] == 32:
            held[0, :n], held[1, :n] = m, v
            continue
        bits = _random_bits(n, s["seed"], s["step"][0].long(), i)
        for j, (x, r) in enumerate(((m, bits & 0xFFFF), (v, bits >> 16))):
            held[j], s["exponents"][i][j] = _to_8(x, r, j)
        moments.append(torch.stack([_of_8(held[j], s["exponents"][i][j], j)[:n] for j in range(2)]))
    return {"params": s["params"], "masters": s["masters"],
            "moments": s["moments"] if case["bits"] == 32 else moments}


def _plain_logprobs(s):
    case, x, targets = s["case"], s["logits"].float(), s["targets"]
    top = x.amax(1, keepdim=True)
    d = x - top
    p = torch.exp(d)
    total = p.sum(1, keepdim=True)
    d = d - torch.log(total)
    p = p / total
    named = (targets >= 0) & (targets < case["vocab"])
    at = targets.clamp(0, case["vocab"] - 1)[:, None]
    outs = [torch.where(named, d.gather(1, at)[:, 0], torch.zeros_like(total[:, 0]))]
    if case["entropy"]:
        entropy = -torch.where(p > 0, p * d, torch.zeros_like(p)).sum(1, keepdim=True)
        outs.append(entropy[:, 0])
    if case["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        outs += [d.gather(1, ids), ids.to(torch.int32)]
    if case["train"]:
        g = torch.where(named, s["grad"], torch.zeros_like(s["grad"]))[:, None]
        factor = g + s["grad_entropy"][:, None] * (d + entropy) if case["entropy"] else g
        outs.append((torch.zeros_like(x).scatter_(1, at, g) - p * factor).to(s["logits"].dtype))
    return outs


_PLAIN = {"quantize": _plain_quantize, "mx4": _plain_mx4, "adamw": _plain_adamw, "logprobs": _plain_logprobs}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


def _mx4_bytes(rows, width):
    blocks = (width + 31) // 32
    return rows * blocks * 17  # 16 bytes of codes and one of scale for each


def work(case):
    """Every input read once and every output written once, 8-bit moments also as the values that the pass returns; of
    the experts' weights those of as many as there can be chosen ones.  A multiplication and an addition are two."""
    op = case["op"]
    if op == "quantize":
        values = case["rows"] * case["width"]
        return {"bytes": values * 2 * _SIZE[case["dtype"]] + 2 * _mx4_bytes(case["rows"], case["width"]),
                "flops": 4 * values}
    if op == "mx4":
        rows, e = case["tokens"] * case["k"], case["experts"]
        used = min(e, rows) if e else 1
        return {"bytes": _mx4_bytes(case["tokens"], case["width"]) + used * _mx4_bytes(case["out"], case["width"])
                + rows * case["out"] * 2 + (4 * rows if e else 0), "flops": 2 * rows * case["out"] * case["width"]}
    if op == "adamw":
        n, size = sum(math.prod(shape) for shape in _shapes(case)), _SIZE[case["dtype"]]
        master = case["master"] and size == 2
        value = (8 + size) if master else 2 * size
        held = 16 if case["bits"] == 32 else 4 + 8 + 4 / 32
        return {"bytes": int(n * (size + value + held)), "flops": 14 * n}
    values, size = case["rows"] * case["vocab"], _SIZE[case["dtype"]]
    outs = case["rows"] * (12 + 4 * case["entropy"] + 8 * case["top"])
    if case["train"]:  # the gradient may only be asked for once the loss is known, and reads the logits again
        return {"bytes": 3 * values * size + outs + 8 * case["rows"], "flops": 12 * values}
    return {"bytes": values * size + outs, "flops": 5 * values}


# -------------------------------------------------------------------------------------------------------- 64 bits


def _values4_exact(x):
    """The values in the format of finite rows [rows, K], by the nearest of the 8 for each block's scale."""
    rows, k = x.shape
    values = torch.tensor(_VALUES4, dtype=torch.float64, device=x.device)
    out = torch.zeros_like(x)
    for begin in range(0, rows, 1024):
        part = torch.nn.functional.pad(x[begin:begin + 1024], (0, -k % 32))
        part = part.reshape(part.shape[0], -1, 32)
        exponent = torch.frexp(part.abs().max(2).values).exponent - 3  # of the largest, less 2: frexp's is one more
        scale = torch.ldexp(torch.ones_like(part[:, :, 0]), exponent.clamp(min=-127))[:, :, None]
        a = part.abs() / scale
        best, at = (a - values[0]).abs(), torch.zeros_like(a, dtype=torch.int64)
        for i in range(1, 8):
            far = (a - values[i]).abs()
            nearer = far <= best if i % 2 == 0 else far < best
            best, at = torch.where(nearer, far, best), torch.where(nearer, torch.full_like(at, i), at)
        back = torch.copysign(values[at] * scale, part)
        out[begin:begin + 1024] = back.reshape(part.shape[0], -1)[:, :k]
    return out


def _decoded(codes, scales, width):
    """Rows in 64 bits from the bits of their codes."""
    bits = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64)
    e, m = (bits >> 1) & 3, bits & 1
    v = torch.where(e > 0, torch.ldexp(1.0 + 0.5 * m.double(), e - 1), 0.5 * m.double())
    v = v * (1.0 - 2.0 * (bits >> 3).double())
    return (v * torch.ldexp(torch.ones_like(v[..., ::32]), scales.to(torch.int64) - 127).repeat_interleave(32, -1))[
        ..., :width]


def _moments_exact(state, i, n):
    if state["case"]["bits"] == 32:
        return state["moments"][i][:, :n].double()
    both = []
    for j in range(2):
        c = state["moments"][i][j].to(torch.int64)
        magnitude = c % 256 if j else c % 128
        e, f = magnitude // 8, (magnitude % 8).double() / 8
        v = torch.where(e > 0, torch.ldexp(1.0 + f, e - 1 + _EMIN[j]), torch.ldexp(f, torch.full_like(e, _EMIN[j])))
        v = torch.ldexp(v, state["exponents"][i][j].to(torch.int64).repeat_interleave(32) - 127)
        both.append(v if j else v * (1 - 2 * (c // 128)))
    return torch.stack(both)[:, :n]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quantize":
        return (_values4_exact(s["x"].double()),)
    if case["op"] == "mx4":
        width = case["width"]
        x = _decoded(*s["x"], width)
        if not case["experts"]:
            return (torch.mm(x, _decoded(*s["w"], width).t()),)
        off, tokens = s["plan"][0].cpu(), s["plan"][1].long()
        y = torch.zeros(tokens.numel(), case["out"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            part = slice(int(off[e]), int(off[e + 1]))
            if part.start < part.stop:
                y[part] = torch.mm(x[tokens[part]], _decoded(s["w"][0][e], s["w"][1][e], width).t())
        return (y,)
    if case["op"] == "adamw":
        t = int(s["step"][0]) + 1
        (b1, b2), lr = _HYPER["betas"], _HYPER["lr"]
        clip = 1.0 if s["clip"] is None else float(s["clip"])
        params, moments = [], []
        for i, p in enumerate(s["params"]):
            n = p.numel()
            old, g = _moments_exact(s, i, n), s["grads"][i].double().reshape(-1) * clip
            m, v = b1 * old[0] + (1 - b1) * g, b2 * old[1] + (1 - b2) * g.square()
            x = (s["masters"][i] if s["masters"] is not None else p).double().reshape(-1)
            x = x - lr * _HYPER["weight_decay"] * x
            x = x - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _HYPER["eps"])
            params.append(x.reshape(p.shape))
            # moments in 8 bits are rounded at random: they have no such value
            moments.append(torch.nn.functional.pad(torch.stack([m, v]), (0, -n % 32)) if case["bits"] == 32 else None)
        return {"params": params, "masters": params if s["masters"] is not None else None, "moments": moments}
    parts = []
    rows = max(1, (1 << 27) // case["vocab"])
    for begin in range(0, case["rows"], rows):
        x, targets = s["logits"][begin:begin + rows].double(), s["targets"][begin:begin + rows]
        logs = torch.log_softmax(x, 1)
        named = (targets >= 0) & (targets < case["vocab"])
        at = torch.where(named, targets, torch.zeros_like(targets))
        line = torch.arange(x.shape[0], device="cuda")
        outs = [torch.where(named, logs[line, at], torch.zeros((), dtype=torch.float64, device="cuda"))]
        p = logs.exp()
        entropy = -torch.nan_to_num(p * logs, nan=0.0).sum(1)
        if case["entropy"]:
            outs.append(entropy)
        if case["top"]:
            left, ids = x.clone(), []
            for _ in range(case["top"]):
                best = left.max(1, keepdim=True).values
                ids.append((left == best).to(torch.int32).argmax(1))
                left[line, ids[-1]] = -math.inf
            ids = torch.stack(ids, 1)
            outs += [logs[line[:, None], ids], ids.to(torch.int32)]
        if case["train"]:
            g = torch.where(named, s["grad"][begin:begin + rows].double(), 0.0)
            grad = -p * g[:, None]
            grad[line, at] += g
            if case["entropy"]:
                ge = s["grad_entropy"][begin:begin + rows].double()
                grad -= ge[:, None] * p * (torch.nan_to_num(logs, neginf=0.0) + entropy[:, None])
            outs.append(grad)
        parts.append(outs)
    return [torch.cat(column) for column in zip(*parts)]
