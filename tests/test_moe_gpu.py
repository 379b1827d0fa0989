"""The router, the experts' products and gradient clipping on the GPU against 64-bit definitions.

Tolerances.  Routing computes in fp32: a gate passes through an exponential (2 ulp, and
2^-24 |z - max| from its rounded argument, |z - max| <= 16 here), a sum in at most 21
steps, a division, and with renorm another sum (5 steps) and division: under 50 roundings
of 2^-24, 3e-6.  Its gradient has two more products and sums: 1e-5 of the largest.
A bf16 rounding is off by at most u = 2^-8 (8 significant bits), at random by about
0.43 u in the 2-norm.  The experts round the activations and each row's product to bf16
before they are joined and rounded, the gradients at five places at most: sqrt(5) * 0.43 u,
1.0 u, with the tanh approximation's 2^-11 beside it; 2 u is allowed.
The norm sums squares in fp32 eight at a time and then in fp64: 8 * 2^-24, and the fp32
result's own 2^-24; a scaled element adds two roundings of its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dtrain_b200 import autograd as F  # noqa: E402
from dtrain_b200.ops import kernels as K  # noqa: E402
from dtrain_b200.optim import clip_grads, clip_scale, global_norm  # noqa: E402

from moe_ref import experts64, gates64, route64  # noqa: E402
from test_moe import ROUTES, _case  # noqa: E402

U = 2.0 ** -8


@pytest.fixture(scope="module", autouse=True)
def _dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.manual_seed(0)
    yield
    assert K.device_status() == 0


# ----------------------------------------------------------------------- routing
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", ROUTES)
@pytest.mark.parametrize("n,e,k", [(1, 12, 1), (37, 12, 4), (70, 36, 6), (33, 60, 5), (65, 132, 8), (19, 252, 8),
                                   (9, 444, 32)])
def test_route(kw, n, e, k, dtype):
    z, kw, ref = _case(kw, n, e, seed=n + e)
    z = z.to(dtype)
    zg = z.cuda().requires_grad_()
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].cuda()
    gates, idx, load = F.route(zg, k, **kw)
    g, i, l = route64(z, k, **ref)
    assert gates.dtype == torch.float32 and idx.dtype == load.dtype == torch.int32
    assert torch.equal(idx.cpu().long(), i) and torch.equal(load.cpu().long(), l)
    torch.testing.assert_close(gates.detach().cpu().double(), g, rtol=3e-6, atol=1e-30)
    # gradient: autograd of the fp64 definition at the same choices
    G = torch.randn(n, k)
    dz, = torch.autograd.grad(gates, zg, G.cuda())
    z64 = z.double().requires_grad_()
    opts = {k_: ref[k_] for k_ in ("softmax", "renorm", "scale")}
    want, = torch.autograd.grad(gates64(z64, i, **opts), z64, G.double())
    want = torch.nan_to_num(want)  # a row without experts
    assert dz.dtype == dtype
    tol = 1e-5 * max(1e-30, float(want.abs().max()))
    if dtype == torch.bfloat16:
        assert torch.all((dz.cpu().double() - want).abs() <= tol + U * want.abs())
    else:
        assert float((dz.cpu().double() - want).abs().max()) <= tol
    # without a gradient: the same kernel, the same bits
    with torch.no_grad():
        g2, i2, l2 = F.route(zg, k, **kw)
    assert torch.equal(g2, gates) and torch.equal(i2, idx) and torch.equal(l2, load)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_against_differences(score, renorm):
    z = torch.randn(64, 16)
    d, G = torch.randn(64, 16), torch.randn(64, 4)
    zg = z.cuda().requires_grad_()
    gates, idx, _ = F.route(zg, 4, score=score, renorm=renorm)
    dz, = torch.autograd.grad(gates, zg, G.cuda())
    h = 1e-6
    at = [(gates64(z.double() + s * h * d.double(), idx.cpu().long(), softmax=score == "softmax", renorm=renorm)
           * G.double()).sum() for s in (1, -1)]
    num = float(at[0] - at[1]) / (2 * h)
    ana = float((dz.cpu().double() * d.double()).sum())
    # the difference's own error is about h^2 and 1e-16 / h times the sum's size
    assert abs(num - ana) <= 1e-5 * float((dz.cpu().double().abs() * d.double().abs()).sum())


def test_route_special_values():
    z = torch.zeros(6, 8)
    z[0, 3] = math.nan
    z[1] = -math.inf
    z[1, 5] = 0.0
    z[2, 2] = 3e38
    z[3] = -3e38
    z[4, 0] = -0.0
    z[5] = torch.arange(8) * 1e-38
    for score in ("softmax", "sigmoid"):
        gates, idx, load = F.route(z.cuda(), 2, score=score)
        assert idx[0, 0] == 3 and math.isnan(float(gates[0, 0]))       # a NaN shows
        assert idx[1].tolist() == [5, -1] and gates[1].tolist() == [1.0, 0.0]
        assert idx[2, 0] == 2 and math.isfinite(float(gates[2].sum()))
        assert idx[3].tolist() == [0, 1] and math.isfinite(float(gates[3].sum()))
        assert idx[4].tolist() == [0, 1]                                # -0 ties with 0
        assert idx[5].tolist() == [7, 6]                                # ordered by the logits themselves
        assert int(load.sum()) == 11
    # all experts masked by sigmoid scores and a bias
    gates, idx, load = F.route(torch.full((3, 8), -math.inf).cuda(), 2, score="sigmoid", bias=torch.ones(8).cuda())
    assert torch.all(idx == -1) and torch.all(gates == 0) and int(load.sum()) == 0


def test_route_shapes_streams_and_sizes():
    g, i, l = F.route(torch.empty(0, 8, device="cuda"), 2)
    assert g.shape == (0, 2) and i.shape == (0, 2) and int(l.sum()) == 0
    z = torch.randn(50000, 24, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = F.route(z[:, ::2], 3)                     # strided logits
    s.synchronize()
    b = F.route(z[:, ::2].contiguous().view(500, 100, 12), 3)
    assert torch.equal(a[0], b[0].view(-1, 3)) and torch.equal(a[1], b[1].view(-1, 3)) and torch.equal(a[2], b[2])
    assert int(a[2].sum()) == 150000
    # beyond the kernel's 512 experts: torch ops
    wide = torch.randn(5, 600, device="cuda")
    assert torch.equal(F.route(wide, 2)[1].long(), wide.topk(2).indices)


def test_route_refusals_gpu():
    z = torch.randn(4, 8, device="cuda")
    with pytest.raises(ValueError, match="bias"):
        F.route(z, 2, bias=torch.zeros(8))
    for bad in (dict(k=0), dict(k=9), dict(k=3, score="tanh"), dict(k=3, groups=3), dict(k=3, groups=4, keep_groups=5),
                dict(k=3, groups=4, keep_groups=1), dict(k=3, group_top=3), dict(k=3, bias=torch.zeros(7).cuda())):
        with pytest.raises(ValueError, match="route"):
            F.route(z, **bad)
    with pytest.raises(RuntimeError, match="route"):
        K.route_fwd(z, 9)
    with pytest.raises(RuntimeError, match="route"):
        K.route_fwd(z.half(), 2)
    with pytest.raises(RuntimeError, match="route"):
        K.route_fwd(z, 4, groups=4, keep=1)


# ----------------------------------------------------------------------- experts
def _rel(a, b):
    b = b.double()
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-30))


def _inputs(n, c, h, co, e, k, bias=True, skew=0.0, gate=torch.bfloat16, idx_type=torch.int32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    bf = torch.bfloat16
    z = r(n, e) - skew * torch.arange(e, device="cuda")
    idx = z.topk(k, -1).indices.to(idx_type)
    t = dict(x=r(n, c).to(bf), w1=(r(e, c, h) / math.sqrt(c)).to(bf), b1=(0.1 * r(e, h)).to(bf) if bias else None,
             w2=(r(e, h, co) / math.sqrt(h)).to(bf), b2=(0.1 * r(e, co)).to(bf) if bias else None, idx=idx,
             gates=torch.softmax(r(n, k), -1).to(gate))
    return t, r(n, co).to(bf)


@pytest.mark.parametrize("n,c,h,co,e,k,bias", [(1, 768, 200, 136, 5, 2, True), (4, 72, 1032, 264, 6, 2, False),
                                               (8, 200, 136, 72, 3, 1, True), (30, 264, 520, 200, 40, 3, True),
                                               (100, 136, 1544, 72, 4, 2, False), (300, 72, 136, 200, 64, 8, True)])
@pytest.mark.parametrize("gate,idx_type", [(torch.bfloat16, torch.int64), (torch.float32, torch.int32)])
def test_expert_mlp_without_gradient(n, c, h, co, e, k, bias, gate, idx_type):
    # the forms for a few slots and for few rows an expert
    t, _ = _inputs(n, c, h, co, e, k, bias, 0.0, gate, idx_type)
    if n > 1:
        t["idx"][n - 1] = -1
    y = F.expert_mlp(**t)
    ref = experts64(**{m: v.double() if v is not None and v.is_floating_point() else v for m, v in t.items()})
    assert _rel(y, ref) <= 2 * U
    assert n == 1 or torch.all(y[n - 1] == 0)
    assert torch.equal(y, F.expert_mlp(**t)), "fixed orders of summation"


EXPERTS = [  # n, c, h, co, e, k, bias, skew
    (1, 64, 128, 64, 4, 2, True, 0.0),
    (1, 8, 8, 8, 1, 1, False, 0.0),
    (3, 72, 136, 40, 5, 3, True, 0.0),
    (17, 128, 256, 128, 8, 2, False, 0.0),
    (64, 200, 328, 264, 7, 2, True, 3.0),       # most experts have no row
    (129, 256, 512, 256, 2, 1, True, 0.0),
    (257, 320, 640, 320, 3, 3, True, 0.0),
    (700, 136, 264, 520, 40, 6, False, 0.1),
    (2000, 512, 384, 512, 4, 2, True, 0.3),
    (200, 64, 72, 64, 512, 32, True, 0.0),      # the most experts and slots
    (5000, 64, 136, 64, 3, 1, True, 0.0),       # the plan of many slots, several row tiles an expert
]


@pytest.mark.parametrize("n,c,h,co,e,k,bias,skew", EXPERTS)
@pytest.mark.parametrize("gate,idx_type", [(torch.bfloat16, torch.int32), (torch.float32, torch.int64)])
def test_expert_mlp(n, c, h, co, e, k, bias, skew, gate, idx_type):
    t, dy = _inputs(n, c, h, co, e, k, bias, skew, gate, idx_type)
    if n > 2:
        t["idx"][n // 2] = -1                       # a token without an expert
        t["idx"][0, k - 1] = -1
    names = [m for m in ("x", "w1", "b1", "w2", "b2", "gates") if t[m] is not None]
    for m in names:
        t[m].requires_grad_()
    y = F.expert_mlp(**t)
    grads = torch.autograd.grad(y, [t[m] for m in names], dy)
    d = {m: v.detach().double().requires_grad_(m in names) if v is not None and v.is_floating_point() else v
         for m, v in t.items()}
    ref = experts64(**d)
    want = torch.autograd.grad(ref, [d[m] for m in names], dy.double())
    assert y.dtype == torch.bfloat16 and _rel(y, ref) <= 2 * U
    if n > 2:
        assert torch.all(y[n // 2] == 0)
    for m, a, b in zip(names, grads, want):
        assert a.dtype == t[m].dtype and a.shape == t[m].shape
        assert _rel(a, b) <= 2 * U, m
        if m[0] in "wb":                            # every expert by itself; unused ones exactly zero
            for q in range(e):
                if torch.any(t["idx"] == q):
                    assert _rel(a[q], b[q]) <= 2 * U, (m, q)
                else:
                    assert torch.all(a[q] == 0), (m, q)
    with torch.no_grad():
        y2 = F.expert_mlp(**t)
    assert _rel(y2, ref) <= 2 * U
    grads2 = torch.autograd.grad(F.expert_mlp(**t), [t[m] for m in names], dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads2)), "fixed orders of summation"


PAIR = dict.fromkeys(("up", "down", "dx", "dw1", "dw2"), "256x256 pair")
TILES = [  # the sizes of EXPERTS, and the tiles that they are to reach
    ((4096, 776, 1544, 520, 4, 2, True, 0.3), PAIR),
    ((6000, 520, 264, 520, 8, 2, True, 3.0), dict(PAIR, dw1="128x128", dw2="128x128")),     # experts without a row
    ((6001, 264, 520, 328, 8, 2, False, 0.2), dict(PAIR, dw1="128x128", dw2="128x128")),
    ((700, 264, 520, 328, 40, 6, True, 0.1), dict(PAIR, up="128x256", down="128x256", dx="128x256")),
    ((900, 104, 264, 264, 40, 2, True, 0.1), dict(up="128x256", down="128x256", dx="128x128", dw1="128x256",
                                                  dw2="256x256 pair")),
    ((900, 264, 120, 264, 40, 2, True, 0.0), dict(up="128x128", down="128x256", dx="128x256", dw1="128x128",
                                                  dw2="128x256")),
]


@pytest.mark.parametrize("sizes,tiles", TILES)
@pytest.mark.parametrize("gate,idx_type", [(torch.bfloat16, torch.int64), (torch.float32, torch.int32)])
def test_expert_mlp_on_every_tile(sizes, tiles, gate, idx_type):
    n, c, h, co, e, k = sizes[:6]
    assert K.experts_tiles(n, k, e, c, h, co) == tiles
    test_expert_mlp(*sizes, gate, idx_type)


def test_experts_bwd_fp32_weight_gradients_on_pairs():
    assert K.experts_tiles(4096, 2, 4, 776, 1544, 520) == PAIR
    t, dy = _inputs(4096, 776, 1544, 520, 4, 2)
    y, *saved = K.experts_fwd(**t, save=True)
    b = [torch.empty_like(t[m]) for m in ("w1", "b1", "w2", "b2")]
    f = [torch.empty_like(v, dtype=torch.float32) for v in b]
    a = K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, *b)
    c = K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, *f)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    assert all(torch.equal(p, q.to(torch.bfloat16)) for p, q in zip(b, f))


@pytest.mark.parametrize("n,c,h,co,e,k,train", [(2, 72, 136, 64, 4, 2, False), (40, 72, 136, 64, 4, 2, False),
                                                (600, 72, 136, 64, 4, 2, False), (300, 72, 136, 64, 4, 2, True),
                                                (4096, 776, 1544, 520, 4, 2, True)])
def test_route_and_experts_in_a_graph(n, c, h, co, e, k, train):
    names = ("x", "w1", "b1", "w2", "b2")

    def inputs(seed):
        t, dy = _inputs(n, c, h, co, e, k, seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        return [t[m] for m in names] + [torch.randn(n, e, generator=g, device="cuda"), dy]
    held = inputs(0)
    leaves = [v.requires_grad_(train) for v in held[:6]]

    def step():
        x, w1, b1, w2, b2, z, dy = held
        gates, idx, load = F.route(z, k, score="sigmoid")
        y = F.expert_mlp(x, w1, b1, w2, b2, idx, gates)
        return [gates, idx, load, y, *(torch.autograd.grad(y, leaves, dy) if train else ())]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        with torch.no_grad():
            for a, b in zip(held, inputs(seed)):
                a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_expert_mlp_gradient_against_differences():
    t, dy = _inputs(40, 64, 96, 64, 4, 2, gate=torch.float32)
    names = ("x", "w1", "b1", "w2", "b2", "gates")
    for m in names:
        t[m].requires_grad_()
    grads = torch.autograd.grad(F.expert_mlp(**t), [t[m] for m in names], dy)
    d = {m: v.detach().double() if v.is_floating_point() else v for m, v in t.items()}
    for m, a in zip(names, grads):
        step = torch.randn_like(d[m])
        h = 1e-5
        at = [(experts64(**{**d, m: d[m] + s * h * step}) * dy.double()).sum() for s in (1, -1)]
        num = float(at[0] - at[1]) / (2 * h)
        # the sum over entries of (gradient x step): errors of 2 u an entry, at random
        noise = 2 * U * float((a.double() * step).norm()) * 4
        assert abs(num - float((a.double() * step).sum())) <= noise, m


def test_expert_mlp_repeated_expert_and_bad_index():
    # the same expert twice for a token counts twice
    t, _ = _inputs(5, 64, 64, 64, 3, 2)
    t["idx"][:, 1] = t["idx"][:, 0]
    y = F.expert_mlp(**t)
    ref = experts64(**{m: v.double() if v.is_floating_point() else v for m, v in t.items()})
    assert _rel(y, ref) <= 2 * U
    # an index past the experts is skipped and reported
    t["idx"][2, 1] = 3
    K.device_status()
    y = F.expert_mlp(**t)
    assert K.device_status() != 0
    t["idx"][2, 1] = -1
    assert torch.equal(y, F.expert_mlp(**t)) and K.device_status() == 0


def test_expert_mlp_shapes_and_streams():
    t, _ = _inputs(24, 64, 128, 64, 4, 2)
    y = F.expert_mlp(**t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        v = dict(t, x=t["x"].view(2, 12, 64), idx=t["idx"].view(2, 12, 2), gates=t["gates"].view(2, 12, 2))
        y3 = F.expert_mlp(**v)
    s.synchronize()
    assert torch.equal(y3.view(24, 64), y)
    # strided inputs
    wide = torch.zeros(24, 128, device="cuda", dtype=torch.bfloat16)
    wide[:, ::2] = t["x"]
    assert torch.equal(F.expert_mlp(**dict(t, x=wide[:, ::2])), y)
    w1t = t["w1"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(F.expert_mlp(**dict(t, w1=w1t)), y)
    # no tokens
    e = F.expert_mlp(**dict(t, x=t["x"][:0].requires_grad_(), idx=t["idx"][:0], gates=t["gates"][:0]))
    assert e.shape == (0, 64)
    e.sum().backward()
    # widths that are not multiples of 8, and fp32: torch ops
    q, _ = _inputs(6, 12, 20, 12, 3, 2)
    assert _rel(F.expert_mlp(**q), experts64(**{m: v.double() if v.is_floating_point() else v for m, v in q.items()})) < 2 * U


def _off_by_one(t):
    """The same values one element past a 16-byte boundary."""
    v = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return v.copy_(t)


@pytest.mark.parametrize("n", [2, 40, 300])         # streaming, 64-row and 128-row tiles
@pytest.mark.parametrize("gate,idx_type", [(torch.bfloat16, torch.int32), (torch.float32, torch.int64)])
def test_expert_mlp_unaligned(n, gate, idx_type):
    t, dy = _inputs(n, 72, 136, 64, 4, 2, gate=gate, idx_type=idx_type)
    y = F.expert_mlp(**t)
    for m in t:
        assert torch.equal(y, F.expert_mlp(**dict(t, **{m: _off_by_one(t[m])}))), m
    names = ("x", "w1", "b1", "w2", "b2", "gates")
    a = {m: t[m].clone().requires_grad_(m in names) for m in t}
    b = {m: _off_by_one(t[m]).requires_grad_(m in names) for m in t}
    ga = torch.autograd.grad(F.expert_mlp(**a), [a[m] for m in names], dy)
    gb = torch.autograd.grad(F.expert_mlp(**b), [b[m] for m in names], _off_by_one(dy))
    assert all(torch.equal(p, q) for p, q in zip(ga, gb))
    # the output's gradient as a slice that starts at any element
    z = torch.cat([torch.zeros(1, device="cuda", dtype=torch.bfloat16), F.expert_mlp(**a).view(-1)])
    gc = torch.autograd.grad(z, [a[m] for m in names], torch.cat([z[:1].detach(), dy.view(-1)]))
    assert all(torch.equal(p, q) for p, q in zip(ga, gc))


def test_expert_mlp_all_slots_empty():
    for n in (2, 20, 600):
        t, dy = _inputs(n, 64, 136, 72, 4, 2)
        t["idx"].fill_(-1)
        with torch.no_grad():
            assert torch.all(F.expert_mlp(**t) == 0)
        for m in ("x", "w1", "b1", "w2", "b2", "gates"):
            t[m].requires_grad_()
        y = F.expert_mlp(**t)
        y.backward(dy)
        assert torch.all(y == 0) and all(torch.all(t[m].grad == 0) for m in ("x", "w1", "b1", "w2", "b2", "gates"))


def test_expert_mlp_inf_and_nan_stay_in_their_rows():
    t, _ = _inputs(40, 64, 64, 64, 4, 1)
    t["x"][7] = math.nan
    t["x"][9, 3] = math.inf
    y = F.expert_mlp(**t)
    assert torch.isnan(y[7]).all() and not torch.isfinite(y[9]).all()
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.isfinite(y[rest]).all()
    # in the gradients they reach their own experts' weights only
    t, dy = _inputs(300, 64, 64, 64, 4, 1)
    t["x"][7] = math.nan
    e = int(t["idx"][7, 0])
    for m in ("x", "w1", "w2", "gates"):
        t[m].requires_grad_()
    F.expert_mlp(**t).backward(dy)
    for q in range(4):
        assert torch.isfinite(t["w1"].grad[q]).all() == (q != e) and torch.isfinite(t["w2"].grad[q]).all() == (q != e)
    assert torch.isfinite(t["x"].grad[[i for i in range(300) if i != 7]]).all()
    # an expert that no token names may hold anything
    t, dy = _inputs(40, 64, 64, 64, 4, 1)
    t["idx"].clamp_(max=2)
    t["w1"][3] = math.nan
    t["w2"][3] = math.inf
    t["x"].requires_grad_()
    y = F.expert_mlp(**t)
    y.backward(dy)
    assert torch.isfinite(y).all() and torch.isfinite(t["x"].grad).all()


def test_experts_kernel_refusals():
    t, dy = _inputs(8, 64, 64, 64, 4, 2)
    ok = [t[m] for m in ("x", "w1", "b1", "w2", "b2", "idx", "gates")]
    for at, bad in ((0, t["x"].float()), (0, t["x"][:, :56]), (1, t["w1"].cpu()), (2, t["b1"][:2]), (3, t["w2"][:, :, :60]),
                    (5, t["idx"].short()), (5, t["idx"][:4]), (6, t["gates"].half())):
        args = list(ok)
        args[at] = bad
        with pytest.raises(RuntimeError, match="experts"):
            K.experts_fwd(*args)
    y, *saved = K.experts_fwd(*ok, save=True)
    g = [torch.empty_like(t[m]) for m in ("w1", "b1", "w2", "b2")]
    with pytest.raises(RuntimeError, match="experts_bwd"):
        K.experts_bwd(dy[:, :32].contiguous(), t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, *g)
    with pytest.raises(RuntimeError, match="experts_bwd"):
        K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, g[0].float(), *g[1:])
    with pytest.raises(RuntimeError, match="experts_bwd"):
        K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved[:1], *g)


def test_experts_bwd_fp32_weight_gradients():
    t, dy = _inputs(300, 136, 264, 72, 5, 2)
    y, *saved = K.experts_fwd(**t, save=True)
    b = [torch.empty_like(t[m]) for m in ("w1", "b1", "w2", "b2")]
    f = [torch.empty_like(v, dtype=torch.float32) for v in b]
    a = K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, *b)
    c = K.experts_bwd(dy, t["x"], t["w1"], t["w2"], t["b2"], t["gates"], saved, *f)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    assert all(torch.equal(p, q.to(torch.bfloat16)) for p, q in zip(b, f))


# ----------------------------------------------------------------------- derivatives of other kinds
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_forward_mode(score):
    import torch.autograd.forward_ad as fwd
    z, d = torch.randn(33, 12), torch.randn(33, 12)
    kw = dict(score=score, scale=1.5)
    with torch.no_grad(), fwd.dual_level():
        gates, idx, _ = F.route(fwd.make_dual(z.cuda(), d.cuda()), 3, **kw)
        got = fwd.unpack_dual(gates).tangent
    at = [gates64(z.double() + s * 1e-6 * d.double(), idx.cpu().long(), softmax=score == "softmax", scale=1.5) for s in (1, -1)]
    # the difference's own error is about h^2; fp32 tangents
    torch.testing.assert_close(got.cpu().double(), (at[0] - at[1]) / 2e-6, rtol=1e-5, atol=1e-6)
    zg = z.cuda().requires_grad_()
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="route"):
            g, _, _ = F.route(zg, 3, **kw)
            torch.autograd.grad(g, zg, fwd.make_dual(torch.ones_like(g), torch.ones_like(g)))


@pytest.mark.parametrize("name", ["x", "w1", "b1", "w2", "b2", "gates"])
def test_expert_mlp_forward_mode(name):
    import torch.autograd.forward_ad as fwd
    t, dy = _inputs(20, 64, 96, 64, 4, 2, gate=torch.float32)
    d = torch.randn_like(t[name])
    with torch.no_grad(), fwd.dual_level():
        y = F.expert_mlp(**dict(t, **{name: fwd.make_dual(t[name], d)}))
        got = fwd.unpack_dual(y).tangent
    t64 = {m: v.double() if v.is_floating_point() else v for m, v in t.items()}
    h = 1e-5
    at = [experts64(**dict(t64, **{name: t64[name] + s * h * d.double()})) for s in (1, -1)]
    assert got is not None and _rel(got, (at[0] - at[1]) / (2 * h)) <= 2 * U
    x = t["x"].requires_grad_()
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="expert_mlp"):
            torch.autograd.grad(F.expert_mlp(**t), x, fwd.make_dual(dy, dy))


def test_second_derivatives_raise():
    z = torch.randn(20, 8, device="cuda").requires_grad_()
    gates, _, _ = F.route(z, 2)
    w = torch.randn(20, 2, device="cuda")
    dz, = torch.autograd.grad((gates * w).sum() + (z ** 3).sum(), z, create_graph=True)
    plain, = torch.autograd.grad((F.route(z, 2)[0] * w).sum() + (z ** 3).sum(), z)
    assert torch.equal(dz, plain)                   # the first derivative is there
    with pytest.raises(RuntimeError, match="route.*not implemented"):
        (dz ** 2).sum().backward()
    for bias in (True, False):
        t, dy = _inputs(20, 64, 96, 64, 4, 2, bias)
        names = [m for m in ("x", "w1", "b1", "w2", "b2", "gates") if t[m] is not None]
        for m in names:
            t[m].requires_grad_()
        first = torch.autograd.grad(F.expert_mlp(**t), [t[m] for m in names], dy, create_graph=True)
        plain = torch.autograd.grad(F.expert_mlp(**t), [t[m] for m in names], dy)
        for m, a, b in zip(names, first, plain):
            assert torch.equal(a, b)
            with pytest.raises(RuntimeError, match="expert_mlp.*not implemented"):
                torch.autograd.grad(a.float().square().sum() + t[m].float().sum(), t[m], retain_graph=True)


# ----------------------------------------------------------------------- clipping
def _clip_check(grads, max_norm, outs=None):
    want = [g.double().clone() for g in grads]
    norm = math.sqrt(sum(float((w * w).sum()) for w in want))
    got = float(global_norm(grads))
    eps = 9 * 2.0 ** -24
    assert abs(got - norm) <= eps * norm
    ret = clip_grads(grads, max_norm, out=outs)
    assert ret.dtype == torch.float32 and ret.dim() == 0 and float(ret) == got
    f = clip_scale(norm ** 2, max_norm)
    for g, o, w in zip(grads, grads if outs is None else outs, want):
        ulp = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[o.dtype]
        tiny = {torch.float32: 1e-44, torch.bfloat16: 1e-38, torch.float16: 6e-8}[o.dtype]
        assert torch.all((o.double() - w * f).abs() <= (w * f).abs() * (ulp + 2 * eps) * 1.01 + tiny)
        if outs is not None:
            assert torch.equal(g.double(), w)


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_clip_sizes(dtype, max_norm):
    sizes = [(), (1,), (3,), (0,), (7, 9), (8192,), (8193,), (16391,), (257, 129), (64, 33, 5)]
    _clip_check([torch.randn(s, device="cuda").to(dtype) for s in sizes], max_norm)


@pytest.mark.parametrize("out_type", [torch.float32, torch.bfloat16, torch.float16])
def test_clip_into_other_types_and_unaligned_slices(out_type):
    grads, n = [], 0
    for i, dt in enumerate([torch.float32, torch.bfloat16, torch.float16] * 5):
        size = 1 + 613 * i
        grads.append(torch.randn(size + 7, device="cuda").to(dt)[i % 7:i % 7 + size])   # unaligned starts
        n += size
    flat = torch.empty(n + 1, device="cuda", dtype=out_type)
    outs, off = [], 1
    for g in grads:
        outs.append(flat[off:off + g.numel()])
        off += g.numel()
    _clip_check(grads, 2.0, outs)


def test_clip_layouts():
    a = torch.randn(40, 50, device="cuda")
    grads = [a[:, ::2], torch.randn(33, 21, device="cuda").t(), torch.randn(4, 6, 5, 7, device="cuda").permute(2, 0, 3, 1),
             torch.randn(3, 10, 12, device="cuda")[:, 2:9, 1::3], torch.randn(16, device="cuda")]
    rest = a[:, 1::2].clone()
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    _clip_check(grads, 1.0, outs)
    _clip_check(grads, 1.0)
    assert torch.equal(a[:, 1::2], rest)                                # what lies between is left alone
    assert abs(float(global_norm([torch.full((1,), 3.0, device="cuda").expand(16)])) - 12.0) < 1e-5


def test_clip_many_tensors_and_determinism():
    g = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(1 + (37 * i) % 301, device="cuda", generator=g) for i in range(2300)]
    first = [x.clone() for x in grads]
    second = [x.clone() for x in grads]
    _clip_check(grads, 1.0)
    n1, n2 = clip_grads(first, 1.0), clip_grads(second, 1.0)
    assert torch.equal(n1, n2) and all(torch.equal(p, q) for p, q in zip(first, second))


def test_clip_large_small_and_nonfinite():
    _clip_check([torch.full((5000,), 1e30, device="cuda"), torch.ones(3, device="cuda")], 1.0)
    _clip_check([torch.full((5000,), 1e-30, device="cuda")], 1.0)
    _clip_check([torch.full((5000,), 1e-30, device="cuda")], 1e-30)
    _clip_check([torch.zeros(100, device="cuda")], 1.0)
    x = [torch.ones(100, device="cuda"), torch.ones(9, device="cuda")]
    x[1][4] = math.nan
    assert math.isnan(float(clip_grads(x, 1.0))) and torch.isnan(x[0]).all()
    x = [torch.ones(100, device="cuda"), torch.ones(9, device="cuda")]
    x[1][4] = math.inf
    assert math.isinf(float(clip_grads(x, 1.0))) and torch.all(x[0] == 0) and torch.isnan(x[1][4])


def test_clip_graph_and_stream():
    grads = [torch.randn(1000, device="cuda"), torch.randn(77, device="cuda").bfloat16()]
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    clip_grads(grads, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grads(grads, 1.0, out=outs)
    for g in grads:
        g.mul_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(norm) - want) < 1e-6 * want
    torch.testing.assert_close(outs[0], grads[0] * clip_scale(want ** 2, 1.0), rtol=1e-6, atol=0)


def test_clip_refusals_gpu():
    a = torch.randn(100, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([a, a], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([a[:60], a[50:]], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([a[:50], torch.randn(50, device="cuda")], 1.0, out=[torch.empty(50, device="cuda"), a[20:70]])
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([torch.randn(1, device="cuda").expand(5)], 1.0)
    with pytest.raises(RuntimeError, match="overlays"):
        clip_grads([a], 1.0, out=[a.view(torch.bfloat16)[:100]])
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads([a], -1.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads([a], 1.0, out=[])
    with pytest.raises(ValueError, match="shape"):
        clip_grads([a], 1.0, out=[a[:50]])
    with pytest.raises(ValueError, match="shape"):
        clip_grads([a], 1.0, out=[None])
    with pytest.raises(RuntimeError, match="fp32"):
        clip_grads([a, a.double()], 1.0)
    with pytest.raises(RuntimeError, match="device"):
        clip_grads([a, torch.zeros(3)], 1.0)
    assert float(global_norm([None, torch.full((4,), 2.0, device="cuda"), None])) == 4.0


def test_clip_refuses_outputs_that_overlap_their_own_gradients():
    # each output overlaps the gradient that it is made from, at another address or in another type
    buf = torch.randn(20001, device="cuda")
    keep = buf.clone()
    narrow = buf.view(torch.bfloat16)
    for g, o in ((buf[:20000], buf[1:20001]), (buf[4:10004], buf[:10000]), (narrow[20000:30000], buf[5000:15000]),
                 (buf[:5000], narrow[9998:14998])):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads([torch.ones(3, device="cuda"), g], 1e-3, out=[torch.empty(3, device="cuda"), o])
    assert torch.equal(buf, keep)
    # side by side they are fine, and so is a gradient in its own place
    a, b = buf[:10000], buf[10000:20000]
    want = a.double()
    clip_grads([a], 1e9, out=[b])
    assert torch.equal(b.double(), want)
    clip_grads([a], 1e9, out=[a.view(100, 100).view(-1)])
    assert torch.equal(a.double(), want)


def test_clip_without_a_gradient_zeroes_its_output_gpu():
    flat = torch.full((12,), 7.0, device="cuda")
    g = [torch.ones(4, device="cuda"), None, torch.ones(4, device="cuda"), None]
    clip_grads(g, 1e9, out=[flat[:4], flat[4:8:2], flat[8:], None])
    assert flat.tolist() == [1.0] * 4 + [0.0, 7.0, 0.0, 7.0] + [1.0] * 4
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads(g[:2], 1.0, out=[flat[:4], flat[2:6]])


def _cells(shape, stride, at):
    cells = torch.tensor([at])
    for n, s in zip(shape, stride):
        cells = (cells[:, None] + s * torch.arange(n)).flatten()
    return cells.tolist()


def test_clip_refuses_overlapping_strided_outputs():
    a = torch.randn(60, 66, device="cuda")
    keep = a.clone()
    v = a[:, ::2]
    other = torch.randn(60, 33, device="cuda")
    for grads, out in (([v, v], None), ([v, a[:, 30:50]], None), ([a[:, 1::3], v], None), ([a[5:9], v], None),
                       ([other, other + 1], [v, v]), ([other, a[3]], [v, a[3]]),
                       ([v, other], [torch.empty_like(v), v]), ([v[1:]], [v[:-1]]),
                       ([a.as_strided((40, 50), (40, 1))], None), ([a.t(), v], None)):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads(grads, 1e-3, out=out)
    assert torch.equal(a, keep)
    # interleaved views, and the columns of one tensor, share nothing
    want = math.sqrt(float((a.double() ** 2).sum()))
    for parts in ([v, a[:, 1::2]], [a[:, 1::2], v], [a[:, :7], a[:, 7:20], a[:, 20:]], [a[::3], a[1::3], a[2::3]],
                  [a.t()[::2], a.t()[1::2]], [a[:30, ::2], a[30:, ::2], a[:, 1::2]]):
        a.copy_(keep)
        assert float(clip_grads(parts, want / 2)) == pytest.approx(want, rel=1e-6)
        torch.testing.assert_close(a, keep / 2, rtol=1e-6, atol=0)
    # gradients read from between the outputs' elements
    a.copy_(keep)
    clip_grads([a[:, 1::2]], 1e9, out=[v])
    assert torch.equal(v, keep[:, 1::2]) and torch.equal(a[:, 1::2], keep[:, 1::2])
    # gradients may overlap one another: each counts in the norm
    assert float(clip_grads([v, v], 1e9, out=[other, torch.empty_like(other)])) == pytest.approx(
        math.sqrt(2.0) * float(v.double().norm()), rel=1e-6)


def test_clip_overlap_of_any_views():
    g = torch.Generator().manual_seed(11)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    buf = torch.ones(4096, device="cuda")
    refused = 0
    for _ in range(600):
        views = []
        for _ in range(2):
            nd = pick(1, 3)
            views.append(([pick(1, 4) for _ in range(nd)], [pick(1, 14) for _ in range(nd)], pick(0, 20)))
        cells = sum((_cells(*v) for v in views), [])
        ts = [buf.as_strided(*v) for v in views]
        if len(set(cells)) < len(cells):
            refused += 1
            with pytest.raises(RuntimeError, match="overlap"):
                clip_grads(ts, 1.0)
        else:
            buf.fill_(1.0)
            clip_grads(ts, math.sqrt(len(cells)) / 2)
            assert int((buf < 0.75).sum()) == len(cells) and torch.all(buf[cells] < 0.75)
    assert 100 < refused < 500


# ----------------------------------------------------------------------- together
def test_example_learns_and_layer_matches_fp32():
    import numpy as np

    from dtrain_b200.models.moe import MoE
    from test_moe import _example
    losses = _example().main(["--device", "cuda", "--steps", "30", "--batch", "8", "--ctx", "64", "--vocab", "64",
                              "--layers", "1"])
    assert losses[0] == pytest.approx(math.log(64), abs=0.2) and losses[-1] < losses[0] - 0.5
    # the layer's output and gradients against its fp64 math at the same choices
    m = MoE(64, 128, 8, 2, np.random.default_rng(1), torch.bfloat16).cuda()
    with torch.no_grad():
        m.gate.mul_(20.0)
    x = torch.randn(40, 64, device="cuda").bfloat16()
    y = m(x)
    gates, idx, _ = F.route(F.linear(x, m.gate), 2, bias=m.bias, score="sigmoid")
    d = [t.detach().double() for t in (x, m.w1, m.b1, m.w2, m.b2)]
    ref = experts64(*d, idx, gates.detach().to(torch.bfloat16).double())
    assert _rel(y, ref) <= 2 * U
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    # generation's form: one token at a time gives what the batch gives, to the rounding of both
    with torch.no_grad():
        one = torch.cat([F.expert_mlp(x[i:i + 1], m.w1, m.b1, m.w2, m.b2, idx[i:i + 1], gates[i:i + 1].to(x.dtype))
                         for i in range(8)])
    assert _rel(one, ref[:8]) <= 2 * U
