"""Routing, the experts' products and gradient clipping on the CPU: the torch paths against
64-bit definitions and differences, and the refusals."""
import math

import pytest
import torch

from dtrain_b200 import autograd as F
from dtrain_b200.optim import clip_grads, clip_scale, global_norm

from moe_ref import experts64, gates64, route64

ROUTES = [dict(), dict(renorm=False), dict(scale=2.5), dict(score="sigmoid"), dict(score="sigmoid", bias=True),
          dict(score="softmax", bias=True), dict(groups=3, keep_groups=2), dict(groups=4, keep_groups=2, group_top=2),
          dict(score="sigmoid", bias=True, groups=4, keep_groups=2, group_top=2, scale=2.5)]


def _case(kw, n, e, seed=0):
    """Logits on a grid of 1/64 (so that there are ties) with masked experts and an empty row."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randint(-256, 257, (n, e), generator=g).float() / 64
    z[torch.rand(n, e, generator=g) < 0.15] = -math.inf
    z[n // 2] = -math.inf
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randint(-8, 9, (e,), generator=g).float() / 64
    ref = dict(softmax=kw.get("score", "softmax") == "softmax", bias=kw.get("bias"), groups=kw.get("groups", 1),
               keep=kw.get("keep_groups", 1), top=kw.get("group_top", 1), renorm=kw.get("renorm", True),
               scale=kw.get("scale", 1.0))
    return z, kw, ref


@pytest.mark.parametrize("kw", ROUTES)
def test_route_cpu(kw):
    z, kw, ref = _case(kw, 41, 12)
    gates, idx, load = F.route(z.double(), 3, **kw)
    g, i, l = route64(z, 3, **ref)
    assert torch.equal(idx.long(), i) and torch.equal(load.long(), l)
    torch.testing.assert_close(gates, g, rtol=1e-12, atol=1e-14)
    # shape in front of the experts is kept
    g3, i3, _ = F.route(z.double().view(41, 1, 12), 3, **kw)
    assert g3.shape == (41, 1, 3) and torch.equal(i3.view(41, 3), idx)


@pytest.mark.parametrize("kw", ROUTES)
def test_route_without_tokens(kw):
    z, kw, _ = _case(kw, 1, 12)
    for shape in ((0, 12), (3, 0, 12)):
        gates, idx, load = F.route(torch.empty(shape, requires_grad=True), 3, **kw)
        assert gates.shape == idx.shape == (*shape[:-1], 3) and load.tolist() == [0] * 12
        gates.sum().backward()


def test_route_gradient_cpu():
    z = torch.randn(5, 8, dtype=torch.float64, requires_grad=True)
    for kw in (dict(), dict(renorm=False), dict(score="sigmoid", scale=2.5)):
        assert torch.autograd.gradcheck(lambda q: F.route(q, 3, **kw)[0], (z,))


@pytest.mark.parametrize("bad", [dict(k=0), dict(k=9), dict(score="tanh"), dict(groups=3), dict(groups=4, keep_groups=5),
                                 dict(groups=4, keep_groups=1), dict(group_top=3), dict(groups=8, keep_groups=8, group_top=2),
                                 dict(bias=torch.zeros(7))])
def test_route_refusals(bad):
    kw = dict(k=3)
    kw.update(bad)
    with pytest.raises(ValueError, match="route"):
        F.route(torch.randn(4, 8), **kw)


def _experts(n, c, h, co, e, k, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    idx = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(n)])
    idx[n // 2] = -1
    return (r(n, c), r(e, c, h) * 0.3, r(e, h) if bias else None, r(e, h, co) * 0.3, r(e, co) if bias else None, idx,
            torch.rand(n, k, generator=g, dtype=torch.float64))


@pytest.mark.parametrize("bias", [True, False])
def test_expert_mlp_cpu(bias):
    x, w1, b1, w2, b2, idx, gates = _experts(9, 6, 10, 5, 4, 2, bias=bias)
    y = F.expert_mlp(x, w1, b1, w2, b2, idx, gates)
    torch.testing.assert_close(y, experts64(x, w1, b1, w2, b2, idx, gates), rtol=1e-12, atol=1e-12)
    assert torch.equal(y[4], torch.zeros(5, dtype=torch.float64))
    y3 = F.expert_mlp(x.view(3, 3, 6), w1, b1, w2, b2, idx.view(3, 3, 2), gates.view(3, 3, 2))
    assert torch.equal(y3.view(9, 5), y)


def test_expert_mlp_gradient_cpu():
    x, w1, b1, w2, b2, idx, gates = _experts(4, 3, 4, 3, 3, 2)
    leaves = [t.requires_grad_() for t in (x, w1, b1, w2, b2, gates)]
    assert torch.autograd.gradcheck(lambda x, w1, b1, w2, b2, g: F.expert_mlp(x, w1, b1, w2, b2, idx, g), leaves)


def test_expert_mlp_sums_of_bf16_rows():
    # 64 slots a token, outputs and input gradients of one sign: the sums over a token's slots are fp32.  Each
    # value passes four roundings to bf16 at most, 0.43 u each in the 2-norm; bf16 sums are off by 0.43 u sqrt(64 / 3).
    u = 2.0 ** -8
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    n, c, e = 40, 8, 64
    t = [r(n, c), r(e, c, 16), r(e, 16), r(e, 16, 6), r(e, 6)]
    idx = torch.stack([torch.randperm(e, generator=g) for _ in range(n)])
    t = [v.bfloat16().requires_grad_() for v in t]
    gates = (0.5 + r(n, e)).requires_grad_()
    dy = r(n, 6).bfloat16()
    y = F.expert_mlp(*t, idx, gates)
    d = [v.detach().double().requires_grad_() for v in (*t, gates)]
    ref = experts64(*d[:5], idx, d[5])
    rel = lambda a, b: float(((a.double() - b).norm() / b.norm()).detach())  # noqa: E731
    assert y.dtype == torch.bfloat16 and rel(y, ref) <= 1.0 * u
    dx, dg = torch.autograd.grad(y, (t[0], gates), dy)
    wx, wg = torch.autograd.grad(ref, (d[0], d[5]), dy.double())
    assert dg.dtype == torch.float32 and rel(dx, wx) <= 1.0 * u and rel(dg, wg) <= 1.0 * u


def test_expert_mlp_refusals():
    x, w1, b1, w2, b2, idx, gates = _experts(4, 3, 4, 3, 3, 2)
    for bad in ((x[:, :2], w1, b1, w2, b2, idx, gates), (x, w1, b1, w2[:2], b2, idx, gates),
                (x, w1, b1, w2, b2, idx[:3], gates), (x, w1, b1, w2, b2, idx, gates[:, :1]),
                (x, w1, b1, w2, b2, idx.float(), gates)):
        with pytest.raises(ValueError, match="expert_mlp"):
            F.expert_mlp(*bad)


@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip_cpu(max_norm):
    g = [torch.randn(7, 3, dtype=torch.float64), None, torch.randn(5, dtype=torch.float64), torch.zeros(0)]
    norm = math.sqrt(sum(float((t * t).sum()) for t in g if t is not None))
    f = clip_scale(norm ** 2, max_norm)
    want = [None if t is None else t * f for t in g]
    out = [None if t is None else torch.empty_like(t) for t in g]
    assert abs(float(global_norm(g)) - norm) < 1e-12 * norm
    assert abs(float(clip_grads(g, max_norm, out=out)) - norm) < 1e-12 * norm
    assert abs(float(clip_grads(g, max_norm)) - norm) < 1e-12 * norm
    for a, b, w in zip(g, out, want):
        if w is not None:
            torch.testing.assert_close(a, w, rtol=1e-12, atol=0)
            torch.testing.assert_close(b, w, rtol=1e-12, atol=0)


def test_clip_refusals():
    g = [torch.randn(3), torch.randn(4)]
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads(g, -1.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads(g, 1.0, out=g[:1])
    with pytest.raises(ValueError, match="shape"):
        clip_grads(g, 1.0, out=[torch.empty(3), torch.empty(3)])
    with pytest.raises(ValueError, match="shape"):
        clip_grads(g, 1.0, out=[torch.empty(3), None])
    with pytest.raises(TypeError, match="floating"):
        clip_grads([torch.zeros(3, dtype=torch.int64)], 1.0)
    assert float(global_norm([])) == 0.0 and float(clip_grads([None], 1.0)) == 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_clip_of_16_bits_into_fp32_keeps_fp32(dtype):
    g = torch.randn(1000).to(dtype)
    o = torch.empty(1000)
    f = clip_scale(float(g.double().square().sum()), 0.7)
    clip_grads([g], 0.7, out=[o])
    # the factor's rounding and the product's
    torch.testing.assert_close(o.double(), g.double() * f, rtol=3 * 2.0 ** -24, atol=0)


def test_clip_without_a_gradient_zeroes_its_output():
    flat = torch.full((12,), 7.0)
    g = [torch.ones(4), None, torch.ones(4)]
    assert float(clip_grads(g, 1e9, out=[flat[:4], flat[4:8], flat[8:]])) == pytest.approx(math.sqrt(8))
    assert flat.tolist() == [1.0] * 4 + [0.0] * 4 + [1.0] * 4
    clip_grads([None, None], 1.0, out=[flat[:6], None])
    assert flat.tolist() == [0.0] * 8 + [1.0] * 4
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grads([torch.ones(4), None], 1.0, out=[flat[:4], flat[2:6]])


def test_clip_refuses_overlapping_outputs():
    a = torch.randn(60, 66)
    keep, v, other = a.clone(), a[:, ::2], torch.randn(60, 33)
    for grads, out in (([a, a], None), ([a[:31], a[30:]], None), ([v, v], None), ([v, a[:, 30:50]], None), ([a[5:9], v], None),
                       ([other, a[3]], [v, a[3]]), ([v, other], [torch.empty_like(v), v]), ([v[1:]], [v[:-1]]),
                       ([a[:50]], [a[1:51]]), ([a.as_strided((40, 50), (40, 1))], None), ([torch.randn(1).expand(5)], None)):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads(grads, 1e-3, out=out)
    assert torch.equal(a, keep)
    for parts in ([v, a[:, 1::2]], [a[:, :7], a[:, 7:20], a[:, 20:]], [a.t()[::2], a.t()[1::2]], [a.t()]):
        a.copy_(keep)
        clip_grads(parts, float(keep.norm()) / 2)
        torch.testing.assert_close(a, keep / 2, rtol=1e-6, atol=0)
    a.copy_(keep)
    clip_grads([a[:, 1::2]], 1e9, out=[v])
    assert torch.equal(v, keep[:, 1::2])
    clip_grads([v, v], 1e9, out=[other, torch.empty_like(other)])


@pytest.mark.parametrize("stages", [3, 4, 5])
def test_ring_position_names_the_copies_in_flight(stages):
    # csrc/moe.cu finish_loads / finish_products: from the ring's next position, which phase of each barrier to wait for
    passed = lambda done, parity: done % 2 != parity    # a barrier with `done` phases complete  # noqa: E731
    for issued in range(4 * stages):
        stage, phase = issued % stages, issued // stages % 2
        done = [len(range(s, issued, stages)) for s in range(stages)]
        waits = [phase if s < stage else phase ^ 1 for s in range(stages)]
        assert all(passed(d, w) for d, w in zip(done, waits))       # all there: no wait
        for s in range(stages):                                     # one missing: it is waited for
            assert done[s] == 0 or not passed(done[s] - 1, waits[s])
        last = stage - 1 if stage else stages - 1
        assert issued == 0 or last == (issued - 1) % stages and waits[last] == (phase if stage else phase ^ 1)


def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_moe.py")
    spec = importlib.util.spec_from_file_location("train_moe", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_example_learns_cpu(score):
    losses = _example().main(["--device", "cpu", "--steps", "12", "--batch", "4", "--ctx", "32", "--vocab", "32", "--dim",
                              "32", "--experts", "4", "--layers", "1", "--lr", "5e-3", "--score", score])
    assert losses[0] == pytest.approx(math.log(32), abs=0.2) and losses[-1] < losses[0] - 0.3


def test_layer_hands_the_gates_on_as_they_are(monkeypatch):
    import numpy as np
    from dtrain_b200.models import moe
    seen = []
    real = F.expert_mlp
    monkeypatch.setattr(moe.F, "expert_mlp", lambda *a: (seen.append(a[-1]), real(*a))[1])
    m = moe.MoE(8, 16, 4, 2, np.random.default_rng(0), torch.bfloat16)
    x = torch.randn(12, 8).bfloat16()
    m(x)
    gates, _, _ = F.route(F.linear(x, m.gate), 2, score="sigmoid", bias=m.bias)
    assert seen[0].dtype == torch.float32 and torch.equal(seen[0], gates)


def test_balance_moves_the_bias_against_the_load():
    import numpy as np
    from dtrain_b200.models.moe import MoE
    m = MoE(8, 16, 4, 1, np.random.default_rng(0))
    with torch.no_grad():
        m.gate.zero_()
    m(torch.randn(12, 8))                                 # equal scores: every token goes to expert 0
    assert m.load.tolist() == [12, 0, 0, 0]
    m.balance(0.1)
    torch.testing.assert_close(m.bias, torch.tensor([-0.1, 0.1, 0.1, 0.1]))
    m(torch.randn(12, 8))
    assert m.load.tolist() == [0, 12, 0, 0]
