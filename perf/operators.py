"""The mixture-of-experts operators and gradient clipping as measured work.

Three operators: the router (``route``), the experts' products (``expert_mlp``)
and the clipping of many gradient tensors by their global norm (``clip_grads``).
``run`` computes them in plain torch (``own`` false: elementary operations in
32 bits, rounded once at the end) or through this package's entry points
(``own`` true); ``exact`` restates each definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
TINY = 1e-20        # the renormalising sum is at least this
GELU = math.sqrt(2.0 / math.pi)


# ------------------------------------------------------------------- the cases
def _route(name, n, e, k, dtype, score="softmax", bias=False, groups=1, keep=1, top=1, renorm=True, scale=1.0,
           masked=0.0, train=True):
    c = {"op": "route", "n": n, "e": e, "k": k, "dtype": dtype, "score": score, "bias": bias, "groups": groups,
         "keep": keep, "top": top, "renorm": renorm, "scale": scale, "masked": masked, "train": train}
    return dict(c, name=name) if name else c


def _experts(name, n, c, h, e, k, bias=True, empty=0.0, train=True):
    d = {"op": "experts", "n": n, "c": c, "h": h, "e": e, "k": k, "bias": bias, "empty": empty, "train": train}
    return dict(d, name=name) if name else d


def _clip(name, dim, layers, vocab, ctx, experts, dtype, out):
    d = {"op": "clip", "dim": dim, "layers": layers, "vocab": vocab, "ctx": ctx, "experts": experts, "dtype": dtype,
         "out": out}
    return dict(d, name=name) if name else d


def listed():
    return [
        # one token of a generation: the router's latency
        _route("route 1 token", 1, 64, 6, "fp32", train=False),
        # the training batch of the GPT-2-small configuration (16 sequences of 1024), bf16 logits of the gate GEMM
        _route("route 16k x 16", 16384, 16, 4, "bf16"),
        # odd counts, plain softmax gates, masked experts and padding tokens (rows without any expert)
        _route("route 4099 x 60 masked", 4099, 60, 5, "fp32", groups=6, keep=3, renorm=False, masked=0.1),
        # many small experts, balanced by a bias, limited to groups: 32 sequences of 2048
        _route("route 64k x 256 groups", 65536, 256, 8, "fp32", score="sigmoid", bias=True, groups=8, keep=4, top=2,
               scale=2.5),
        # one token of a generation: the weights of two experts are read
        _experts("experts 1 token", 1, 768, 2048, 16, 2, train=False),
        # 48 sequences generating side by side: nearly every expert has a few rows
        _experts("experts 48 tokens", 48, 1024, 4096, 8, 2, train=False),
        # odd counts, padding tokens without an expert, no biases, forward and backward
        _experts("experts 1237 odd", 1237, 264, 712, 6, 3, bias=False, empty=0.1),
        # a training batch at dim 768: forward and backward
        _experts("experts 16k x 768", 16384, 768, 1536, 16, 4),
        # a training batch at the 1.3B configuration's dim 2048: forward and backward
        _experts("experts 8k x 2048", 8192, 2048, 2048, 32, 4),
        # the parameter list of a 2-layer test model: launch latency
        _clip("clip 2 layers d128", 128, 2, 512, 128, 0, "fp32", "fp32"),
        # a 12-layer model with 8 experts a layer, every expert a tensor: bf16 gradients into a flat fp32 buffer
        _clip("clip 12 layers 8 experts", 512, 12, 50304, 1024, 8, "bf16", "fp32"),
        # the GPT-2-medium parameter list in fp32
        _clip("clip 24 layers d1024", 1024, 24, 50304, 1024, 0, "fp32", "fp32"),
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    what = rng.choice(("route", "experts", "clip"))
    if what == "route":
        train = rng.random() < 0.75
        n = _log(rng, 64, 65536) if train else _log(rng, 1, 4096)
        k = rng.randint(1, 8)
        if rng.random() < 0.5:      # ungrouped, any number of experts
            return _route(None, n, rng.randint(max(k, 8), 256), k, rng.choice(("fp32", "bf16")), renorm=rng.random() < 0.7,
                          masked=rng.choice((0.0, 0.1)), train=train)
        groups = rng.choice((2, 4, 8))
        keep = rng.randint(1, groups)
        per = rng.randint(max(2, -(-k // keep)), 256 // groups)
        return _route(None, n, groups * per, k, "fp32", "sigmoid", rng.random() < 0.8, groups, keep, rng.choice((1, 2)),
                      True, rng.choice((1.0, 2.5)), rng.choice((0.0, 0.1)), train)
    if what == "experts":
        train = rng.random() < 0.6
        while True:
            n = _log(rng, 96, 16384) if train else _log(rng, 1, 512)
            c, h = _log(rng, 128, 2048, 8), _log(rng, 256, 4096, 8)
            e = _log(rng, 4, 64)
            k = rng.randint(1, min(4, e))
            if h != 3 * 1024 and e * c * h <= 2 ** 27 and n * k * c * h <= 2 ** 37:
                return _experts(None, n, c, h, e, k, rng.random() < 0.7, rng.choice((0.0, 0.1)), train)
    dim = _log(rng, 64, 1024, 8)
    return _clip(None, dim, rng.randint(1, 16), _log(rng, 256, 50304, 8), _log(rng, 64, 2048), rng.choice((0, 0, 4, 8)),
                 rng.choice(("fp32", "bf16")), "fp32")


def _clip_shapes(c):
    """The parameter shapes of a GPT (dense MLP, or ``experts`` MLPs a layer, each its own tensors)."""
    d, out = c["dim"], [(c["vocab"], c["dim"]), (c["ctx"], c["dim"])]
    for _ in range(c["layers"]):
        out += [(d,), (d,), (d, 3 * d), (3 * d,), (d, d), (d,), (d,), (d,)]
        if c["experts"]:
            out.append((d, c["experts"]))
        out += [(d, 4 * d), (4 * d,), (4 * d, d), (d,)] * max(1, c["experts"])
    return out + [(d,), (d,), (d, c["vocab"])]


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    s = {"case": case}
    if case["op"] == "route":
        n, e, k = case["n"], case["e"], case["k"]
        z = randn(n, e, std=1.2) + randn(e, std=0.6)     # some experts are more popular than others
        if case["masked"]:
            gone = torch.rand(n, e, generator=g, device=DEV) < case["masked"]
            gone |= torch.rand(n, 1, generator=g, device=DEV) < case["masked"] / 2   # padding tokens
            z = z.masked_fill(gone, -math.inf)
        s["logits"] = z.to(TYPES[case["dtype"]]).requires_grad_(case["train"])
        # the balancing bias moves in fixed steps
        s["bias"] = torch.randint(-60, 61, (e,), generator=g, device=DEV).float() * 1e-3 if case["bias"] else None
        s["dgates"] = randn(n, k, std=1e-2) if case["train"] else None
    elif case["op"] == "experts":
        n, c, h, e, k, t = case["n"], case["c"], case["h"], case["e"], case["k"], case["train"]
        bf = torch.bfloat16
        z = randn(n, e) + randn(e, std=0.4)
        top = torch.topk(z, k, dim=-1)
        idx = top.indices.to(torch.int32)
        if case["empty"]:
            idx[torch.rand(n, generator=g, device=DEV) < case["empty"]] = -1
        s["idx"] = idx
        s["gates"] = torch.softmax(top.values, -1).masked_fill(idx < 0, 0.0).to(bf).requires_grad_(t)
        s["x"] = randn(n, c, dtype=bf).requires_grad_(t)
        s["w1"] = randn(e, c, h, std=0.02, dtype=bf).requires_grad_(t)
        s["w2"] = randn(e, h, c, std=0.02, dtype=bf).requires_grad_(t)
        s["b1"] = randn(e, h, std=0.02, dtype=bf).requires_grad_(t) if case["bias"] else None
        s["b2"] = randn(e, c, std=0.02, dtype=bf).requires_grad_(t) if case["bias"] else None
        s["dy"] = randn(n, c, std=1e-2, dtype=bf) if t else None
    else:
        shapes = _clip_shapes(case)
        s["grads"] = [randn(*sh, std=1e-3, dtype=TYPES[case["dtype"]]) for sh in shapes]
        s["flat"] = torch.empty(sum(math.prod(sh) for sh in shapes), dtype=TYPES[case["out"]], device=DEV)
        s["views"], off = [], 0
        for sh in shapes:
            s["views"].append(s["flat"][off:off + math.prod(sh)].view(sh))
            off += math.prod(sh)
    return s


# -------------------------------------------------------------- the plain form
def _largest(c, k):
    """Values and places of the k largest of a row, ties to the lowest place."""
    v, i = torch.sort(c, dim=-1, descending=True, stable=True)
    return v[..., :k], i[..., :k]


def _plain_route(case, logits, bias, dgates):
    z = logits.detach().float()
    n, e = z.shape
    gone = z == -math.inf
    if case["score"] == "softmax":
        m = z.max(-1, keepdim=True).values
        p = torch.exp(z - m.masked_fill(m == -math.inf, 0.0))
        t = p.sum(-1, keepdim=True)
        s = p / t.masked_fill(t == 0, 1.0)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    if bias is None and case["top"] == 1:
        c = z
    else:
        c = (s if bias is None else s + bias).masked_fill(gone, -math.inf)
    if case["groups"] > 1:
        per = c.view(n, case["groups"], -1)
        best = _largest(per, case["top"])[0]
        score = best[..., 0] if case["top"] == 1 else best[..., 0] + best[..., 1].masked_fill(best[..., 1] == -math.inf, 0.0)
        keep = torch.zeros_like(score, dtype=torch.bool).scatter_(1, _largest(score, case["keep"])[1], True)
        c = per.masked_fill(~keep[..., None], -math.inf).view(n, e)
    v, idx = _largest(c, case["k"])
    none = v == -math.inf
    sj = s.gather(1, idx).masked_fill(none, 0.0)
    total = sj.sum(-1, keepdim=True)
    d = total.clamp(min=TINY) if case["renorm"] else torch.ones_like(total)
    gates = case["scale"] * sj / d
    load = torch.bincount(idx.masked_fill(none, e).view(-1), minlength=e + 1)[:e].to(torch.int32)
    out = {"gates": gates, "idx": idx.masked_fill(none, -1).to(torch.int32), "load": load}
    if dgates is not None:
        gj = dgates.masked_fill(none, 0.0)
        ds = gj
        if case["renorm"]:
            ds = gj - (gj * sj).sum(-1, keepdim=True) / d * (total > TINY)
        ds = case["scale"] * ds / d
        at = idx
        if case["score"] == "sigmoid":
            dz = torch.zeros_like(z).scatter_(1, at, (ds * sj * (1.0 - sj)).masked_fill(none, 0.0))
        else:
            dz = torch.zeros_like(z).scatter_(1, at, ds.masked_fill(none, 0.0))
            dz = s * (dz - (ds * sj).sum(-1, keepdim=True))
        out["dlogits"] = dz.to(logits.dtype)
    return out


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(GELU * (x + 0.044715 * x * x * x)))


def _gelu_slope(x):
    t = torch.tanh(GELU * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * GELU * (1.0 + 3 * 0.044715 * x * x)


def _plain_few(s):
    """Forward for fewer slots than experts: only the weights of the experts in use are read."""
    n, k = s["idx"].shape
    at = s["idx"].reshape(-1).long()
    some = (at >= 0)[:, None]
    at = at.clamp(min=0)
    x = s["x"].float().repeat_interleave(k, 0)
    h = torch.bmm(x[:, None], s["w1"][at].float())[:, 0]
    h = _gelu(h if s["b1"] is None else h + s["b1"][at].float())
    y = torch.bmm(h[:, None], s["w2"][at].float())[:, 0]
    y = (y if s["b2"] is None else y + s["b2"][at].float()).masked_fill(~some, 0.0)
    return {"y": (y.view(n, k, -1) * s["gates"].float()[..., None]).sum(1).to(s["x"].dtype)}


def _plain_experts(s):
    """Rows sorted by expert into a padded [experts, most rows, .] batch, products as batched matrix products."""
    x, gates, idx = s["x"].detach(), s["gates"].detach(), s["idx"]
    n, k = idx.shape
    e, c, h = s["w1"].shape
    if not s["case"]["train"] and n * k <= e:
        return _plain_few(s)
    bf = x.dtype
    w1, w2 = s["w1"].detach().float(), s["w2"].detach().float()
    b1 = None if s["b1"] is None else s["b1"].detach().float()
    b2 = None if s["b2"] is None else s["b2"].detach().float()
    flat = idx.reshape(-1).long()
    slots = torch.nonzero(flat >= 0)[:, 0]                      # slots that have an expert
    slots = slots[torch.sort(flat[slots], stable=True).indices]   # by expert
    at = flat[slots]
    count = torch.bincount(at, minlength=e)
    pos = torch.arange(at.numel(), device=x.device) - (torch.cumsum(count, 0) - count)[at]
    cap = int(count.max())
    tok = slots // k
    row = at * cap + pos
    xb = torch.zeros(e * cap, c, device=x.device).index_copy_(0, row, x[tok].float()).view(e, cap, c)
    pre = torch.bmm(xb, w1) if b1 is None else torch.baddbmm(b1[:, None], xb, w1)
    act = _gelu(pre)
    yb = torch.bmm(act, w2) if b2 is None else torch.baddbmm(b2[:, None], act, w2)
    ys = torch.zeros(n * k, c, device=x.device).index_copy_(0, slots, yb.view(e * cap, c)[row])
    gf = gates.float()
    out = {"y": (ys.view(n, k, c) * gf[..., None]).sum(1).to(bf)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        out["dgates"] = (ys.view(n, k, c) * dy[:, None]).sum(-1).to(gates.dtype)
        u = dy[tok] * gf.reshape(-1)[slots][:, None]
        ub = torch.zeros(e * cap, c, device=x.device).index_copy_(0, row, u).view(e, cap, c)
        dpre = torch.bmm(ub, w2.transpose(1, 2)) * _gelu_slope(pre)
        out["dw2"] = torch.bmm(act.transpose(1, 2), ub).to(bf)
        out["dw1"] = torch.bmm(xb.transpose(1, 2), dpre).to(bf)
        if b1 is not None:
            out["db1"] = dpre.sum(1).to(bf)
        if b2 is not None:
            out["db2"] = ub.sum(1).to(bf)
        dxb = torch.bmm(dpre, w1.transpose(1, 2)).view(e * cap, c)
        dxs = torch.zeros(n * k, c, device=x.device).index_copy_(0, slots, dxb[row])
        out["dx"] = dxs.view(n, k, c).sum(1).to(bf)
    return out


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    f = torch.where((norm <= 1.0) | (norm == 0), 1.0, 1.0 / (norm + 1e-6))
    flat = torch.cat([(g.float() * f).reshape(-1) for g in s["grads"]])
    return {"norm": norm, "flat": flat.to(s["flat"].dtype)}


# --------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            if case["op"] == "route":
                return _plain_route(case, state["logits"], state["bias"], state["dgates"])
            return _plain_experts(state) if case["op"] == "experts" else _plain_clip(state)
    if case["op"] == "clip":
        from dtrain_b200.optim import clip_grads

        norm = clip_grads(state["grads"], 1.0, out=state["views"])
        return {"norm": norm, "flat": state["flat"]}
    from dtrain_b200 import autograd as F

    if case["op"] == "route":
        gates, idx, load = F.route(state["logits"], case["k"], score=case["score"], bias=state["bias"],
                                   groups=case["groups"], keep_groups=case["keep"], group_top=case["top"],
                                   renorm=case["renorm"], scale=case["scale"])
        out = {"gates": gates, "idx": idx, "load": load}
        if case["train"]:
            out["dlogits"], = torch.autograd.grad(gates, state["logits"], state["dgates"])
        return out
    y = F.expert_mlp(state["x"], state["w1"], state["b1"], state["w2"], state["b2"], state["idx"], state["gates"])
    out = {"y": y}
    if case["train"]:
        names = [n for n in ("x", "gates", "w1", "b1", "w2", "b2") if state[n] is not None]
        grads = torch.autograd.grad(y, [state[n] for n in names], state["dy"])
        out.update(("d" + n, d) for n, d in zip(names, grads))
    return out


def work(case):
    if case["op"] == "route":
        n, e, k, b = case["n"], case["e"], case["k"], SIZE[case["dtype"]]
        size = n * e * b + 8 * n * k + 4 * e + (4 * e if case["bias"] else 0)
        if case["train"]:       # the gates' gradient read, the logits' written
            size += 4 * n * k + n * e * b
        return {"bytes": size, "flops": 8 * n * e}
    if case["op"] == "experts":
        n, c, h, e, k = case["n"], case["c"], case["h"], case["e"], case["k"]
        slots = n * k * (1 - case["empty"])
        used = e * (1 - (1 - k / e) ** n)                  # experts with a row, expected
        weights = 2 * used * (2 * c * h + (h + c if case["bias"] else 0))
        size = 4 * n * c + 6 * n * k + weights
        flops = 4 * slots * c * h
        if case["train"]:       # dy read, dx, the gates' and the weights' gradients written
            size += 4 * n * c + 2 * n * k + 2 * e * (2 * c * h + (h + c if case["bias"] else 0))
            flops *= 3
        return {"bytes": size, "flops": flops}
    n = sum(math.prod(sh) for sh in _clip_shapes(case))
    return {"bytes": n * (SIZE[case["dtype"]] + SIZE[case["out"]]), "flops": 3 * n}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "experts": _exact_experts, "clip": _exact_clip}[case["op"]](case, s)


def _exact_route(case, s):
    z = s["logits"].detach().double()
    n, e = z.shape
    k, valid = case["k"], torch.isfinite(z)
    if case["score"] == "softmax":
        score = torch.where(valid.any(-1, keepdim=True), torch.softmax(z, -1), 0.0)
    else:
        score = torch.sigmoid(z)
    c = score + (0.0 if s["bias"] is None else s["bias"].double())
    if s["bias"] is None and case["top"] == 1:
        c = z
    c = torch.where(valid, c, -math.inf)
    size = e // case["groups"]
    if case["groups"] > 1:
        rank = []
        for j in range(case["groups"]):
            b = torch.topk(c[:, j * size:(j + 1) * size], case["top"], -1).values
            rank.append(torch.where(torch.isfinite(b[:, 1:]), b[:, 1:], 0.0).sum(-1) + b[:, 0])
        order = torch.stack(rank, 1).argsort(dim=-1, descending=True, stable=True)
        for j in range(case["keep"], case["groups"]):
            out = order[:, j, None] == torch.arange(e, device=DEV) // size
            c = torch.where(out, -math.inf, c)
    idx = c.argsort(dim=-1, descending=True, stable=True)[:, :k]
    used = torch.isfinite(c.gather(1, idx))
    # gates = scale * score restricted to the chosen, over their sum; the gradient by the quotient's rule
    pick = torch.zeros_like(c).scatter_(1, idx, used.double())
    a = score * pick
    total = a.sum(-1, keepdim=True)
    den = total.clamp(min=TINY) if case["renorm"] else torch.ones_like(total)
    full = case["scale"] * a / den
    gates = full.gather(1, idx) * used
    dz = None
    if case["train"]:
        up = torch.zeros_like(c).scatter_(1, idx, s["dgates"].double()) * pick
        da = case["scale"] * up / den
        if case["renorm"]:
            da = da - pick * (up * full).sum(-1, keepdim=True) / den
        if case["score"] == "softmax":
            dz = score * (da - (da * score).sum(-1, keepdim=True))
        else:
            dz = da * score * (1 - score)
    out = {"gates": gates, "idx": None, "load": None}
    if dz is not None:
        out["dlogits"] = dz
    return out


def _exact_experts(case, s):
    if case["n"] * case["k"] * case["c"] * case["h"] > 2 ** 39:
        return None
    d = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    x, gates, idx = d["x"], d["gates"], d["idx"]
    y, dx, dg = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(gates)
    grads = {n: torch.zeros_like(d[n]) for n in ("w1", "b1", "w2", "b2") if d[n] is not None}
    for e in range(case["e"]):
        tok, j = torch.nonzero(idx == e, as_tuple=True)
        if not tok.numel():
            continue
        xe, ge = x[tok], gates[tok, j][:, None]
        pre = xe @ d["w1"][e] + (0.0 if d["b1"] is None else d["b1"][e])
        th = torch.tanh(GELU * (pre + 0.044715 * pre ** 3))
        act = 0.5 * pre * (1 + th)
        ye = act @ d["w2"][e] + (0.0 if d["b2"] is None else d["b2"][e])
        y.index_add_(0, tok, ge * ye)
        if not case["train"]:
            continue
        dye = d["dy"][tok]
        dg[tok, j] = (dye * ye).sum(-1)
        u = ge * dye
        slope = 0.5 * (1 + th) + 0.5 * pre * (1 - th ** 2) * GELU * (1 + 3 * 0.044715 * pre ** 2)
        dpre = (u @ d["w2"][e].T) * slope
        grads["w2"][e], grads["w1"][e] = act.T @ u, xe.T @ dpre
        if d["b1"] is not None:
            grads["b1"][e], grads["b2"][e] = dpre.sum(0), u.sum(0)
        dx.index_add_(0, tok, dpre @ d["w1"][e].T)
    out = {"y": y}
    if case["train"]:
        out.update({"dx": dx, "dgates": dg, **{"d" + n: v for n, v in grads.items()}})
    return out


def _exact_clip(case, s):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for g in s["grads"]:
        total += torch.linalg.vector_norm(g.double()) ** 2
    norm = total.sqrt()
    f = 1.0 if float(norm) <= 1.0 else 1.0 / (float(norm) + 1e-6)
    return {"norm": norm, "flat": torch.cat([g.double().view(-1) for g in s["grads"]]) * f}
