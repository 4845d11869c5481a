"""The operators of sparse_amd.tokens on the shapes they are used at: each in a plain form (elementary torch operations in
32 bits, rounded once) and, where `own` is true, through the framework's own calls.

Three operators, each with its gradient.  All are products with a matrix that has one or a few entries in a row, given by
its column indices, which is how a language model meets sparse matrices:

  lookup    y = S E,           S [tokens x vocabulary], one entry per row (the token's id, times a scale)
  lookup gradient              dE = S^T dy
  route     xs = P x, y = C ys where P [slots x tokens] puts the tokens in the order of their experts and
                               C [tokens x slots] brings them back with the router's weights
  route gradient               dys = C^T dy, dw = <dy, ys> at C's entries, dx = P^T dxs
  experts   ys = blockdiag(W) xs, one dense block for each expert's slots
  experts gradient             dxs = blockdiag(W)^T dys, dW_e = dys_e^T xs_e
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ the cases
def _lookup(op, name, tokens, vocab, width, dtype, vals=False, skip=0.0):
    return {"name": name, "op": op, "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype, "vals": vals, "skip": skip}


def _route(op, name, tokens, chosen, experts, width, dtype, skew=0.0, skip=0.0):
    return {"name": name, "op": op, "tokens": tokens, "chosen": chosen, "experts": experts, "width": width, "dtype": dtype,
            "skew": skew, "skip": skip}


def _experts(op, name, tokens, chosen, experts, width, inner, dtype, skew=0.0, skip=0.0):
    return dict(_route(op, name, tokens, chosen, experts, width, dtype, skew, skip), inner=inner)


def listed():
    return [
        # one step of serving: the newest token of each of 32 sequences
        _lookup("lookup", "lookup, a serving step", 32, 32768, 2048, "bf16"),
        # a training step's input: 16384 tokens of a large vocabulary
        _lookup("lookup", "lookup, a training step", 16384, 131072, 4096, "bf16"),
        # a model of odd sizes in 32 bits, with a scale for each token (what a mono record holds as its values)
        _lookup("lookup", "lookup, odd sizes", 4099, 50021, 1001, "f32", vals=True),
        # fine-tuning a small model on a short batch
        _lookup("lookup gradient", "lookup gradient, small", 128, 4096, 512, "f32"),
        # the training step's gradient: nearly every row of the table is zero and still has to be written
        _lookup("lookup gradient", "lookup gradient, training", 16384, 131072, 2048, "bf16"),
        # byte-pair-like text in a small vocabulary: long runs of the commonest tokens, 30 % padding without a gradient
        _lookup("lookup gradient", "lookup gradient, skewed", 32768, 8192, 1024, "f16", vals=True, skip=0.3),
        # one step of serving through a router: 16 tokens to 4 of 64 experts and back
        _route("route", "route, a serving step", 16, 4, 64, 2048, "bf16"),
        # a training step's tokens to 8 of 128 experts and back
        _route("route", "route, a training step", 16384, 8, 128, 2048, "bf16"),
        # the way back through a router of few experts, an odd number of tokens, some of them dropped
        _route("route gradient", "route gradient", 8191, 2, 8, 4096, "f16", skew=1.0, skip=0.05),
        # the experts' products of one step of serving: bound by the weights' bytes
        _experts("experts", "experts, a serving step", 16, 4, 32, 2048, 4096, "bf16"),
        # the experts' products of a training step
        _experts("experts", "experts, a training step", 8192, 2, 8, 4096, 4096, "bf16", skew=0.5),
        # both gradients of a training step's products, more and smaller experts
        _experts("experts gradient", "experts gradient", 4096, 4, 16, 2048, 4096, "bf16", skew=0.5),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A row's length: a multiple of 64, of 8, or any number."""
    w, kind = _spread(rng, low, high), rng.random()
    return w // 64 * 64 if kind < 0.5 else w // 8 * 8 if kind < 0.8 else w


def draw(rng):
    op = rng.choice(["lookup", "lookup gradient", "route", "route gradient", "experts", "experts gradient"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    skip = rng.choice([0.0, 0.0, 0.1, 0.4])
    if op.startswith("lookup"):
        width = _width(rng, 64, 8192)
        vocab = _spread(rng, 500, min(131072, (1 << 29) // width))
        tokens = _spread(rng, 1, min(32768, (1 << 27) // width))
        return {k: v for k, v in _lookup(op, "", tokens, vocab, width, dtype, rng.random() < 0.3, skip).items() if k != "name"}
    experts = _spread(rng, 2, 256)
    chosen = min(experts, _spread(rng, 1, 8))
    skew = rng.choice([0.0, 0.5, 1.0])
    if op.startswith("route"):
        width = _width(rng, 64, 8192)
        tokens = _spread(rng, 1, min(16384, (1 << 28) // (width * chosen)))
        case = _route(op, "", tokens, chosen, experts, width, dtype, skew, skip)
    else:
        width, inner = _width(rng, 64, 4096), _width(rng, 64, 4096)
        experts = max(chosen, min(experts, (1 << 28) // (width * inner)))
        tokens = _spread(rng, 1, 8192)
        tokens = max(1, min(tokens, int(2.5e11 / (2.0 * width * inner * chosen))))
        case = _experts(op, "", tokens, chosen, experts, width, inner, "f16" if dtype == "f16" else "bf16", skew, skip)
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ the inputs
def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ids(case, g):
    """Token ids as text has them: the chance of an id falls as one over its place in the vocabulary; the places are dealt
    over the table, and a share `skip` are padding (-1)."""
    n, V = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    place = ((V + 1) ** u - 1).long().clamp_(0, V - 1)
    ids = torch.randperm(V, generator=g, device="cuda")[place]
    return torch.where(torch.rand(n, generator=g, device="cuda") < case["skip"], torch.full_like(ids, -1), ids)


def _choices(case, g):
    """Each token's experts, distinct and in the order of their scores, and the softmax of those scores; a share `skip` of
    the choices is dropped (-1), as a router with a capacity does."""
    n, k, X = case["tokens"], case["chosen"], case["experts"]
    score = torch.randn((n, X), generator=g, device="cuda") + case["skew"] * torch.randn((1, X), generator=g, device="cuda")
    top, chosen = score.topk(k, dim=1)
    weights = torch.exp(top - top[:, :1])
    weights = weights / weights.sum(1, keepdim=True)
    drop = torch.rand((n, k), generator=g, device="cuda") < case["skip"]
    return torch.where(drop, torch.full_like(chosen, -1), chosen), weights.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    s = {"case": case, "op": case["op"]}
    if case["op"].startswith("lookup"):
        n, V, D = case["tokens"], case["vocab"], case["width"]
        s["ids"] = _ids(case, g)
        s["vals"] = torch.rand(n, generator=g, device="cuda") + 0.5 if case["vals"] else None
        s["scale"] = math.sqrt(D)
        if case["op"] == "lookup":
            s["E"] = _normal(g, (V, D), t, 0.02)
        else:
            s["dy"] = _normal(g, (n, D), t)
            s["vocab"] = V
        return s
    s["chosen"], s["weights"] = _choices(case, g)
    slots, D = case["tokens"] * case["chosen"], case["width"]
    s["experts"] = case["experts"]
    if case["op"].startswith("route"):
        s["ys"] = _normal(g, (slots, D), t)
        if case["op"] == "route":
            s["x"] = _normal(g, (case["tokens"], D), t)
        else:
            s["dy"] = _normal(g, (case["tokens"], D), t)
            s["dxs"] = _normal(g, (slots, D), t)
        s["out"] = torch.zeros((slots, D), device="cuda", dtype=t)     # rows behind the last routed slot stay zero
        return s
    F = case["inner"]
    s["xs"] = _normal(g, (slots, D), t)
    s["W"] = _normal(g, (case["experts"], F, D), t, 1.0 / math.sqrt(D))
    # how many slots each expert has: the plain form's loop reads it on the host, the framework's calls do not need it
    s["counts"] = torch.bincount(s["chosen"].reshape(-1) + 1, minlength=case["experts"] + 1)[1:].tolist()
    if case["op"] == "experts":
        s["out"] = torch.zeros((slots, F), device="cuda", dtype=t)
    else:
        s["dys"] = _normal(g, (slots, F), t)
        s["out"] = torch.zeros((slots, D), device="cuda", dtype=t)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
_tk = {}


def _framework(dtype):
    if dtype not in _tk:
        from sparse_amd import mk_tokens
        _tk[dtype] = mk_tokens(dtype)
    return _tk[dtype]


def _run_own(s):
    op, tk = s["op"], _framework(s["case"]["dtype"])
    if op == "lookup":
        return tk.lookup(s["E"], s["ids"], vals=s["vals"], scale=s["scale"])
    if op == "lookup gradient":
        return tk.lookup_grad(s["dy"], s["ids"], s["vocab"], vals=s["vals"], scale=s["scale"])
    r = tk.route(s["chosen"], s["experts"])
    if op == "route":
        return r.pos, r.offsets, tk.dispatch(s["x"], r, out=s["out"]), tk.combine(s["ys"], r, s["weights"])
    if op == "route gradient":
        dys, dw = tk.combine_grad(s["dy"], s["ys"], r, s["weights"], out=s["out"])
        return dys, dw, tk.dispatch_grad(s["dxs"], r)
    if op == "experts":
        return tk.experts(s["xs"], s["W"], r, out=s["out"])
    return tk.experts_grad_x(s["dys"], s["W"], r, out=s["out"]), tk.experts_grad_w(s["dys"], s["xs"], r)


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_lookup(s):
    """y[i] = scale vals[i] E[ids[i]]; an id outside the table selects nothing."""
    ids, E = s["ids"], s["E"]
    f = torch.where(ids >= 0, s["scale"], 0.0).float()
    f = f * s["vals"] if s["vals"] is not None else f
    return (E[ids.clamp(min=0)].float() * f[:, None]).to(E.dtype)


def _plain_lookup_grad(s):
    """dE[v] = sum over i with ids[i] = v of scale vals[i] dy[i]."""
    ids, dy = s["ids"], s["dy"]
    f = torch.where(ids >= 0, s["scale"], 0.0).float()
    f = f * s["vals"] if s["vals"] is not None else f
    dE = torch.zeros((s["vocab"], dy.shape[1]), device="cuda", dtype=torch.float32)
    return dE.index_add_(0, ids.clamp(min=0), dy.float() * f[:, None]).to(dy.dtype)


def _plain_order(chosen, experts):
    """The slots in the order of their experts (a token's place in the batch within one): the place of every choice, -1
    where there is none, the choice at every place, and where each expert's slots begin."""
    n = chosen.numel()
    e = chosen.reshape(-1)
    e = torch.where(e >= 0, e, experts)
    order = e.argsort(stable=True)
    pos = torch.empty(n, device="cuda", dtype=torch.int64)
    pos[order] = torch.arange(n, device="cuda")
    pos = torch.where(e < experts, pos, -1)
    offsets = torch.searchsorted(e[order], torch.arange(experts + 1, device="cuda"))
    return pos.view(chosen.shape).int(), order, offsets.int()


def _plain_gather(x, order, offsets, per, factor=None):
    """Row p is x[order[p] / per], times its factor; zero behind the last routed slot."""
    y = x[order // per].float()
    y = y * factor.reshape(-1)[order][:, None] if factor is not None else y
    return torch.where((torch.arange(order.numel(), device="cuda") < offsets[-1])[:, None], y, 0.0).to(x.dtype)


def _plain_combine(ys, pos, weights=None):
    """y[t] = sum over j of w[t, j] ys[pos[t, j]] where there is such a place."""
    y = ys[pos.clamp(min=0).long()].float()
    y = y * weights[..., None] if weights is not None else y
    return torch.where((pos >= 0)[..., None], y, 0.0).sum(1).to(ys.dtype)


def _plain_dots(dy, ys, pos):
    """dw[t, j] = <dy[t], ys[pos[t, j]]>, 0 where there is no such place."""
    d = (ys[pos.clamp(min=0).long()].float() * dy.float()[:, None, :]).sum(2)
    return torch.where(pos >= 0, d, 0.0)


def _plain_experts(a, W, counts, out, transposed):
    """Every expert's slots times its matrix.  A loop over the experts is the quickest plain form of this: one padded
    batch would multiply many times the rows wherever the experts' shares differ."""
    out = torch.zeros_like(out)
    at = 0
    for e, n in enumerate(counts):
        if n:
            w = W[e].float()
            out[at:at + n] = (a[at:at + n].float() @ (w if transposed else w.t())).to(out.dtype)
        at += n
    return out


def _plain_experts_grad_w(dys, xs, counts):
    dW = torch.zeros((len(counts), dys.shape[1], xs.shape[1]), device="cuda", dtype=xs.dtype)
    at = 0
    for e, n in enumerate(counts):
        if n:
            dW[e] = (dys[at:at + n].float().t() @ xs[at:at + n].float()).to(xs.dtype)
        at += n
    return dW


def _run_plain(s):
    op = s["op"]
    if op == "lookup":
        return _plain_lookup(s)
    if op == "lookup gradient":
        return _plain_lookup_grad(s)
    if op == "experts":
        return _plain_experts(s["xs"], s["W"], s["counts"], s["out"], False)
    if op == "experts gradient":
        return _plain_experts(s["dys"], s["W"], s["counts"], s["out"], True), _plain_experts_grad_w(s["dys"], s["xs"], s["counts"])
    pos, order, offsets = _plain_order(s["chosen"], s["experts"])
    per = s["chosen"].shape[1]
    if op == "route":
        return pos, offsets, _plain_gather(s["x"], order, offsets, per), _plain_combine(s["ys"], pos, s["weights"])
    return (_plain_gather(s["dy"], order, offsets, per, s["weights"]), _plain_dots(s["dy"], s["ys"], pos),
            _plain_combine(s["dxs"], pos))


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------------------------------ the work of one pass
def _distinct(case):
    """How many rows of the table a batch is expected to name (ids as _ids() deals them)."""
    V, n = case["vocab"], case["tokens"] * (1 - case["skip"])
    v = np.arange(V, dtype=np.float64)
    p = np.log((v + 2) / (v + 1)) / math.log(V + 1)
    return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def work(case):
    b, op, n, D = SIZE[case["dtype"]], case["op"], case["tokens"], case["width"]
    if op.startswith("lookup"):
        small = n * 8 + (n * 4 if case["vals"] else 0)
        if op == "lookup":
            return {"bytes": (_distinct(case) + n) * D * b + small, "flops": n * D}
        return {"bytes": (n * (1 - case["skip"]) + case["vocab"]) * D * b + small, "flops": 2 * n * D}
    slots = n * case["chosen"]
    live = slots * (1 - case["skip"])
    small = slots * 8
    if op == "route":      # x in, xs out, ys in, y out, weights in, places and offsets out
        return {"bytes": 2 * (n + live) * D * b + small + slots * 8 + case["experts"] * 4, "flops": 2 * live * D}
    if op == "route gradient":     # dy, ys, dxs, weights in; dys, dw, dx out
        return {"bytes": (2 * n + 3 * live) * D * b + small + slots * 8, "flops": 4 * live * D}
    F = case["inner"]
    used = min(case["experts"], case["experts"] * -math.expm1(slots * math.log1p(-1.0 / case["experts"]))) if case["experts"] > 1 else 1
    if op == "experts":
        return {"bytes": live * (D + F) * b + used * D * F * b + small, "flops": 2 * live * D * F}
    return {"bytes": live * (2 * D + F) * b + (used + case["experts"]) * D * F * b + small, "flops": 4 * live * D * F}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64
    if op.startswith("lookup"):
        f = torch.full((case["tokens"],), s["scale"], device="cuda", dtype=d)
        if s["vals"] is not None:
            f = f * s["vals"].to(d)
        f = f * (s["ids"] >= 0)
        i = s["ids"].clamp(min=0)
        if op == "lookup":
            return torch.index_select(s["E"], 0, i).to(d).mul_(f.unsqueeze(1))
        dE = torch.zeros((case["vocab"], case["width"]), device="cuda", dtype=d)
        dE.index_put_((i,), s["dy"].to(d).mul_(f.unsqueeze(1)), accumulate=True)
        return dE
    # the places, expert by expert, from the definition: an expert's slots are its choices in the order of the batch
    flat = s["chosen"].reshape(-1)
    order = torch.cat([torch.nonzero(flat == e).reshape(-1) for e in range(case["experts"])])
    live, k = order.numel(), case["chosen"]
    if op in ("route", "route gradient"):
        token, w = order // k, s["weights"].reshape(-1)[order].to(d)
        slots, D = flat.numel(), case["width"]
        moved = torch.zeros((slots, D), device="cuda", dtype=d)
        back = torch.zeros((case["tokens"], D), device="cuda", dtype=d)
        if op == "route":
            moved[:live] = s["x"].to(d)[token]
            for j in range(k):         # a token's choices one by one: no row is added to twice at once
                at = torch.nonzero(order % k == j).reshape(-1)
                back[token[at]] += s["ys"].to(d)[at] * w[at].unsqueeze(1)
            return None, None, moved, back
        moved[:live] = s["dy"].to(d)[token] * w.unsqueeze(1)
        dw = torch.zeros(slots, device="cuda", dtype=d)
        dw[order] = (s["dy"].to(d)[token] * s["ys"].to(d)[:live]).sum(1)
        for j in range(k):
            at = torch.nonzero(order % k == j).reshape(-1)
            back[token[at]] += s["dxs"].to(d)[at]
        return moved, dw.view(-1, k), back
    begin = [0]
    for e in range(case["experts"]):
        begin.append(begin[-1] + int((flat == e).sum()))
    out = torch.zeros(s["out"].shape, device="cuda", dtype=d)
    dW = torch.zeros(s["W"].shape, device="cuda", dtype=d) if op != "experts" else None
    for e in range(case["experts"]):
        rows = slice(begin[e], begin[e + 1])
        if begin[e] == begin[e + 1]:
            continue
        if op == "experts":
            out[rows] = torch.mm(s["xs"][rows].to(d), s["W"][e].to(d).t().contiguous())
        else:
            out[rows] = torch.mm(s["dys"][rows].to(d), s["W"][e].to(d))
            dW[e] = torch.mm(s["dys"][rows].to(d).t().contiguous(), s["xs"][rows].to(d))
    return out if op == "experts" else (out, dW)
