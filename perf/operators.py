"""The experts' operators as they are measured: what each case is, its inputs, and one pass through it.

``listed()`` are the cases, ``draw(rng)`` one more of their ranges; ``prepare(case, seed)`` makes what a program has
in hand before the call, ``run(state)`` makes the call and returns its outputs, ``work(case)`` says what one pass
cannot do without, and ``exact(case, seed)`` gives the outputs in 64 bits.  With ``own`` false ``run`` computes the
operators in elementary torch operations in 32 bits; with ``own`` true it calls this library.

Four operators, on T tokens that each choose k of E experts (R = T*k assignments):
  route    logits [T, E] -> the k largest of each row, their softmax weights, and the assignments sorted by expert
  grouped  y_r = w_e x_token(r) for the rows r of each expert e, w [E, N, K]; training: dx and dw too
  scaled   the same in 8-bit integers with a scale for each token and each output channel; E = 0 is one dense product
  combine  out_t = sum_j weight[t, j] * y[place(t, j)]; training: dy and dweights too
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


def _case(name, op, tokens, experts, k, width=0, out=0, dtype="bf16", train=False, skew=0.5, normalize=True):
    """width: K, the length of a token's row (H of combine); out: N, the channels of the product; skew: how unevenly
    the experts are liked (expert e's popularity falls as (e+1)^-skew, in an order of the seed's)."""
    c = dict(op=op, tokens=tokens, experts=experts, k=k, width=width, out=out, dtype=dtype, train=train, skew=skew,
             normalize=normalize)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the router of one decoding step of one request: latency alone counts
        _case("route_token", "route", 1, 64, 8, dtype="f32"),
        # the router of a batch of requests of odd length, weights not normalised over the chosen
        _case("route_batch", "route", 1021, 60, 4, normalize=False),
        # the router of a training step, with its gradient
        _case("route_train", "route", 16384, 128, 8, dtype="f32", train=True),
        # one decoding step of one request: four experts' weights are read for one row each
        _case("grouped_token", "grouped", 1, 32, 4, 2048, 4096),
        # a batch of decoding requests over many experts: a few ragged rows each, odd sizes
        _case("grouped_batch", "grouped", 203, 48, 4, 1000, 1001, dtype="f16", skew=1.0),
        # the prompt of several requests through a few large experts
        _case("grouped_prompt", "grouped", 8192, 8, 2, 4096, 4096),
        # fine-tuning a small layer: the product and both gradients, ragged sizes
        _case("grouped_tune", "grouped", 601, 12, 2, 520, 776, dtype="f16", train=True),
        # the largest: a training step of a layer of many experts, the product and both gradients
        _case("grouped_train", "grouped", 16384, 32, 4, 2048, 2048, train=True),
        # a decoding batch through one dense layer in 8 bits
        _case("scaled_tokens", "scaled", 16, 0, 1, 4096, 4096),
        # a prompt through experts in 8 bits
        _case("scaled_prompt", "scaled", 16384, 16, 2, 4096, 2048),
        # a decoding batch's experts joined to its tokens
        _case("combine_batch", "combine", 37, 32, 6, 2048),
        # a training step's experts joined to their tokens, with both gradients
        _case("combine_train", "combine", 16384, 64, 8, 2048, train=True),
    ]


_MAX_FLOPS = 6 * 65536 * 2048 * 2048  # grouped_train
_MAX_ROW_BYTES = 131072 * 2048 * 2    # combine_train's rows


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A width: mostly a multiple of 8, as layers have, at times any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(("route", "grouped", "grouped", "grouped", "scaled", "scaled", "combine"))
    tokens, experts = _log(rng, 1, 16384), _log(rng, 4, 128)
    k = rng.randint(1, min(8, experts))
    skew = rng.choice((0.0, 0.5, 1.0))
    train = rng.random() < 0.5
    if op == "route":
        return _case(None, op, tokens, experts, k, dtype=rng.choice(("f32", "bf16", "f16")), train=train, skew=skew,
                     normalize=rng.random() < 0.7)
    width, out = _dim(rng, 128, 4096), _dim(rng, 128, 4096)
    if op == "combine":
        tokens = min(tokens, _MAX_ROW_BYTES // (2 * width * k))
        return _case(None, op, tokens, experts, k, width, dtype=rng.choice(("bf16", "f16")), train=train, skew=skew)
    if op == "scaled":
        if rng.random() < 0.4:
            experts, k = 0, 1
        train = False
        dtype = "bf16"
    else:
        dtype = rng.choice(("bf16", "bf16", "f16"))
    experts = min(experts, max(4, (1 << 28) // (width * out))) if experts else 0  # half a GB of 16-bit weights
    k = min(k, max(1, experts))
    tokens = max(1, min(tokens, _MAX_FLOPS // ((6 if train else 2) * k * width * out)))
    return _case(None, op, tokens, experts, k, width, out, dtype, train, skew)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(shape, g, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _logits(case, g):
    t, e = case["tokens"], case["experts"]
    liking = -case["skew"] * torch.log1p(torch.arange(e, device="cuda", dtype=torch.float32))
    liking = liking[torch.randperm(e, generator=g, device="cuda")]
    return torch.randn(t, e, generator=g, device="cuda") + liking


def _assign(case, g):
    """(offsets, tokens, places): the assignments of drawn logits, sorted by expert."""
    logits, k, e = _logits(case, g), case["k"], case["experts"]
    ids = torch.topk(logits, k, dim=1).indices.reshape(-1)
    order = torch.argsort(ids, stable=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum((ids[None, :] == torch.arange(e, device="cuda")[:, None]).sum(1), 0)
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device="cuda")
    return offsets, (order // k).to(torch.int32), places.to(torch.int32).reshape(-1, k)


def _int8(shape, g):
    return torch.randn(shape, generator=g, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)


def _inputs(case, seed):
    g = _gen(seed)
    op, t, e, k = case["op"], case["tokens"], case["experts"], case["k"]
    width, out, dtype = case["width"], case["out"], _DTYPE[case["dtype"]]
    s = {}
    if op == "route":
        s["logits"] = _logits(case, g).to(dtype)
        if case["train"]:
            s["grad"] = torch.randn(t, k, generator=g, device="cuda")
        return s
    if e:
        s["plan"] = _assign(case, g)
    if op == "grouped":
        s["x"] = _randn((t, width), g, dtype)
        s["w"] = _randn((e, out, width), g, dtype, 1.0 / math.sqrt(width))
        if case["train"]:
            s["grad"] = _randn((t * k, out), g, dtype)
    elif op == "scaled":
        s["x"], s["xs"] = _int8((t, width), g), torch.rand(t, generator=g, device="cuda") * 0.02 + 0.01
        shape = (e, out) if e else (out,)
        s["w"] = _int8(shape + (width,), g)
        s["ws"] = (torch.rand(shape, generator=g, device="cuda") + 0.5) * (0.025 / math.sqrt(width))
    else:
        s["y"] = _randn((t * k, width), g, dtype)
        weights = torch.rand(t, k, generator=g, device="cuda") + 0.05
        s["weights"] = weights / weights.sum(1, keepdim=True)
        if case["train"]:
            s["grad"] = _randn((t, width), g, dtype)
    return s


_LEAVES = {"route": ("logits",), "grouped": ("x", "w"), "combine": ("y", "weights")}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        if "plan" in s:
            s["plan"] = _api().ExpertPlan(*s["plan"])
        if case["train"]:
            for name in _LEAVES[case["op"]]:
                s[name].requires_grad_(True)
    return s


def _run_own(s):
    api, case = _api(), s["case"]
    op, train = case["op"], case["train"]
    if op == "route":
        weights, ids, plan = api.route(s["logits"], case["k"], normalize=case["normalize"])
        outs = (weights.detach(), ids, plan.offsets, plan.tokens, plan.places)
        return outs + torch.autograd.grad(weights, s["logits"], s["grad"]) if train else outs
    if op == "grouped":
        y = api.grouped_mm(s["x"], s["w"], s["plan"], gather=True)
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"]), s["grad"]) if train else (y,)
    if op == "scaled":
        if case["experts"]:
            return (api.grouped_mm_scaled(s["x"], s["xs"], s["w"], s["ws"], s["plan"], gather=True,
                                          out_dtype=torch.bfloat16),)
        return (api.grouped_mm_scaled(s["x"], s["xs"], s["w"], s["ws"], out_dtype=torch.bfloat16),)
    out = api.combine(s["y"], s["plan"], s["weights"])
    return (out.detach(),) + torch.autograd.grad(out, (s["y"], s["weights"]), s["grad"]) if train else (out,)


def _plain_route(s):
    case, logits = s["case"], s["logits"].float()
    k, e = case["k"], case["experts"]
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = torch.gather(logits, 1, ids)
    top = chosen[:, :1]
    total = torch.exp((chosen if case["normalize"] else logits) - top).sum(1, keepdim=True)
    weights = torch.exp(chosen - top) / total
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=logits.device)
    offsets[1:] = torch.cumsum((flat[None, :] == torch.arange(e, device=logits.device)[:, None]).sum(1), 0)
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device=logits.device)
    outs = (weights, ids.to(torch.int32), offsets, (order // k).to(torch.int32), places.to(torch.int32).reshape(-1, k))
    if not case["train"]:
        return outs
    dot = (weights * s["grad"]).sum(1, keepdim=True)
    if case["normalize"]:
        grad = torch.zeros_like(logits).scatter_(1, ids, weights * (s["grad"] - dot))
    else:
        grad = torch.exp(logits - top) / total * (torch.zeros_like(logits).scatter_(1, ids, s["grad"]) - dot)
    return outs + (grad.to(s["logits"].dtype),)


def _plain_grouped(s):
    case = s["case"]
    offsets, tokens, places = s["plan"]
    off = offsets.tolist()
    dtype = s["x"].dtype
    rows = s["x"].float()[tokens]
    y = torch.empty(rows.shape[0], case["out"], device="cuda", dtype=dtype)
    spans = [(e, off[e], off[e + 1]) for e in range(case["experts"]) if off[e] < off[e + 1]]
    for e, lo, hi in spans:
        y[lo:hi] = rows[lo:hi] @ s["w"][e].float().t()
    if not case["train"]:
        return (y,)
    grad = s["grad"].float()
    dw, dr = torch.zeros_like(s["w"]), torch.empty_like(rows)
    for e, lo, hi in spans:
        dr[lo:hi] = grad[lo:hi] @ s["w"][e].float()
        dw[e] = grad[lo:hi].t() @ rows[lo:hi]
    return y, dr[places].sum(1).to(dtype), dw


def _plain_scaled(s):
    x = s["x"].float()
    if not s["case"]["experts"]:
        return ((x @ s["w"].float().t() * s["xs"][:, None] * s["ws"][None, :]).to(torch.bfloat16),)
    offsets, tokens, _ = s["plan"]
    off = offsets.tolist()
    rows, scale = x[tokens], s["xs"][tokens]
    y = torch.empty(rows.shape[0], s["case"]["out"], device="cuda", dtype=torch.bfloat16)
    for e in range(s["case"]["experts"]):
        lo, hi = off[e], off[e + 1]
        if lo < hi:
            y[lo:hi] = rows[lo:hi] @ s["w"][e].float().t() * scale[lo:hi, None] * s["ws"][e][None, :]
    return (y,)


def _plain_combine(s):
    places = s["plan"][2]
    weights = s["weights"]
    rows = s["y"].float()[places]
    out = (rows * weights[:, :, None]).sum(1).to(s["y"].dtype)
    if not s["case"]["train"]:
        return (out,)
    grad = s["grad"].float()
    dy = torch.empty_like(s["y"])
    dy[places.reshape(-1)] = (weights[:, :, None] * grad[:, None, :]).reshape(-1, grad.shape[1]).to(dy.dtype)
    return out, dy, (rows * grad[:, None, :]).sum(2)


_PLAIN = {"route": _plain_route, "grouped": _plain_grouped, "scaled": _plain_scaled, "combine": _plain_combine}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    """Every input read once and every output written once; of the weights, those of as many experts as there can be
    chosen ones.  A multiplication and an addition are two operations."""
    op, t, e, k = case["op"], case["tokens"], case["experts"], case["k"]
    width, out, b = case["width"], case["out"], _SIZE[case["dtype"]]
    rows = t * k
    if op == "route":
        size = t * e * b + rows * 16 + 4 * (e + 1)
        flops = t * e * 2 + rows * 4
        return {"bytes": size + rows * 4 + t * e * b, "flops": 2 * flops} if case["train"] else \
            {"bytes": size, "flops": flops}
    if op == "grouped":
        size = t * width * b + min(e, rows) * out * width * b + rows * out * b + rows * 4
        if case["train"]:
            return {"bytes": size + rows * out * b + t * width * b + e * out * width * b,
                    "flops": 6 * rows * out * width}
        return {"bytes": size, "flops": 2 * rows * out * width}
    if op == "scaled":
        used = min(e, rows) if e else 1
        return {"bytes": t * width + used * out * (width + 4) + 4 * t + rows * out * 2 + (4 * rows if e else 0),
                "flops": 2 * rows * out * width}
    size = rows * width * b + t * width * b + rows * 8
    if case["train"]:
        return {"bytes": size + t * width * b + rows * width * b + rows * 4, "flops": 5 * rows * width}
    return {"bytes": size, "flops": 2 * rows * width}


def exact(case, seed):
    s = _inputs(case, seed)
    op, k, e, train = case["op"], case["k"], case["experts"], case["train"]
    if op == "route":
        l = s["logits"].double()
        t = l.shape[0]
        # rank of every expert in its row: those above it, and equal ones of a lower index
        ids = torch.empty(t, k, dtype=torch.int64, device="cuda")
        left = l.clone()
        for j in range(k):
            best = left.max(1, keepdim=True).values
            ids[:, j] = (left == best).to(torch.int32).argmax(1)
            left[torch.arange(t, device="cuda"), ids[:, j]] = -math.inf
        mask = torch.zeros_like(l, dtype=torch.bool)
        mask[torch.arange(t, device="cuda")[:, None], ids] = True
        base = l.masked_fill(~mask, -math.inf) if case["normalize"] else l
        p = torch.softmax(base, 1)
        weights = p.gather(1, ids)
        key = ids.reshape(-1) * (t * k) + torch.arange(t * k, device="cuda")
        order = torch.sort(key).values % (t * k)
        counts = torch.bincount(ids.reshape(-1), minlength=e)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        places = torch.argsort(order).reshape(t, k).to(torch.int32)
        outs = (weights, ids.to(torch.int32), offsets, torch.div(order, k, rounding_mode="floor").to(torch.int32), places)
        if not train:
            return outs
        g = torch.zeros_like(l)
        g[torch.arange(t, device="cuda")[:, None], ids] = s["grad"].double()
        return outs + (p * (g - (p * g).sum(1, keepdim=True)),)
    if op == "scaled" and not e:
        return ((s["x"].double() * s["xs"].double()[:, None]) @ (s["w"].double() * s["ws"].double()[:, None]).t(),)
    off = s["plan"][0].cpu()
    tokens, places = s["plan"][1].long(), s["plan"][2].long()
    if op == "combine":
        t, width = case["tokens"], case["width"]
        out = torch.zeros(t, width, dtype=torch.float64, device="cuda")
        weights = s["weights"].double()
        dy = torch.zeros(t * k, width, dtype=torch.float64, device="cuda") if train else None
        dw = torch.zeros(t, k, dtype=torch.float64, device="cuda") if train else None
        for j in range(k):
            rows = s["y"][places[:, j]].double()
            out += weights[:, j:j + 1] * rows
            if train:
                g = s["grad"].double()
                dy[places[:, j]] = weights[:, j:j + 1] * g
                dw[:, j] = (rows * g).sum(1)
        return (out, dy, dw) if train else (out,)
    y = torch.zeros(case["tokens"] * k, case["out"], dtype=torch.float64, device="cuda")
    if train:
        dx = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda")
    for i in range(e):
        seg = slice(int(off[i]), int(off[i + 1]))
        if seg.start == seg.stop:
            continue
        a, w = s["x"][tokens[seg]].double(), s["w"][i].double()
        if op == "scaled":
            a, w = a * s["xs"][tokens[seg]].double()[:, None], w * s["ws"][i].double()[:, None]
        y[seg] = torch.mm(a, w.t())
        if train:
            g = s["grad"][seg].double()
            dx.index_add_(0, tokens[seg], torch.mm(g, w))
            dw[i] = torch.mm(g.t(), a)
    return (y, dx, dw) if train else (y,)
