"""Functional ops with the reference's names and semantics (dtrain/autograd.py:199-266).

``embedding``, ``layer_norm``, ``causal_attention``, ``cross_entropy``, ``gelu``,
``relu``, ``linear``; and, beyond the reference, a mixture of experts' ``route`` and
``expert_mlp``.  Autograd is PyTorch's.  On CUDA bf16 tensors with
kernel-compatible shapes each op runs the sm_100a kernels through an autograd
Function (gradients in the inputs' dtypes); on every other input it runs the
reference math with torch ops - explicit causal softmax, population-variance
LayerNorm with eps 1e-5, tanh-approximated GELU, mean cross-entropy - which is
what the float64 oracle tests exercise.

``register_grad_ready_hook(t, fn)`` is the reference's grad-ready hook
(dtrain/autograd.py:63-65): ``fn(t)`` runs once per backward, after every use of
the leaf has been accumulated into ``t.grad`` (torch's post-accumulate-grad hook).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import kernels as K

no_grad = torch.no_grad
Tensor = torch.Tensor


def register_grad_ready_hook(t: torch.Tensor, fn):
    """Call ``fn(t)`` once per backward, when ``t.grad`` holds its final value."""
    return t.register_post_accumulate_grad_hook(fn)


def _fast(*ts) -> bool:
    return all(t.is_cuda and t.dtype == torch.bfloat16 for t in ts)


# ---------------------------------------------------------------- linear
class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        shp = x.shape
        x2 = x.reshape(-1, shp[-1]).contiguous()
        y = K.gemm(x2, w.contiguous(), bias=None if b is None else b.contiguous())
        ctx.save_for_backward(x2, w)
        ctx.has_b = b is not None
        ctx.shp = shp
        return y.view(*shp[:-1], w.shape[1])

    @staticmethod
    def backward(ctx, dy):
        x2, w = ctx.saved_tensors
        dy2 = dy.reshape(-1, w.shape[1]).contiguous()
        dx = K.gemm(dy2, w.contiguous(), b_trans=True).view(ctx.shp)
        dw = K.gemm(x2, dy2, a_trans=True)
        db = None
        if ctx.has_b:
            db32 = torch.empty(w.shape[1], dtype=torch.float32, device=dy.device)
            K.bias_grad(dy2, db32)
            db = db32.to(torch.bfloat16)
        return dx, dw, db


def linear(x, w, b=None):
    """x @ w + b with w stored (in, out) (dtrain/nn.py:60-65)."""
    ok = _fast(x, w) and (b is None or _fast(b))
    if ok and x.shape[-1] % 8 == 0 and w.shape[1] % 8 == 0 and x.numel() > 0:
        return _LinearFn.apply(x, w, b)
    y = x @ w
    return y + b if b is not None else y


# ------------------------------------------------------------- layer norm
class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        C = x.shape[-1]
        x2 = x.reshape(-1, C).contiguous()
        y, mu, rs = K.layernorm_fwd(x2, w.contiguous(), b.contiguous(), eps)
        ctx.save_for_backward(x2, w, mu, rs)
        ctx.shp = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, mu, rs = ctx.saved_tensors
        C = x2.shape[1]
        dw = torch.empty(C, dtype=torch.float32, device=dy.device)
        db = torch.empty(C, dtype=torch.float32, device=dy.device)
        dx = K.layernorm_bwd(dy.reshape(-1, C).contiguous(), x2, w.contiguous(), mu, rs, None, dw, db)
        return dx.view(ctx.shp), dw.to(w.dtype), db.to(w.dtype), None


def layer_norm(x, w, b, eps: float = 1e-5):
    C = x.shape[-1]
    if _fast(x, w, b) and C % 8 == 0 and C <= 2048 and x.numel() > 0:
        return _LayerNormFn.apply(x, w, b, eps)
    return F.layer_norm(x, (C,), w, b, eps)


# -------------------------------------------------------------- attention
class _AttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v):
        B, H, T, D = q.shape
        qkv = torch.stack([q, k, v], dim=2).permute(0, 3, 2, 1, 4).reshape(B * T, 3 * H * D).contiguous()
        out, lse = K.attn_fwd(qkv, B, T, H, D)
        ctx.save_for_backward(qkv, out, lse)
        ctx.dims = (B, H, T, D)
        return out.view(B, T, H, D).permute(0, 2, 1, 3)

    @staticmethod
    def backward(ctx, dout):
        qkv, out, lse = ctx.saved_tensors
        B, H, T, D = ctx.dims
        d = dout.permute(0, 2, 1, 3).reshape(B * T, H * D).contiguous()
        dqkv = K.attn_bwd(qkv, out, d, lse, B, T, H, D).view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
        return dqkv[0], dqkv[1], dqkv[2]


def causal_attention(q, k, v):
    """softmax(q k^T / sqrt(d) + causal mask) v for (B, H, T, D) inputs (dtrain/autograd.py:226-247)."""
    D = q.shape[-1]
    if _fast(q, k, v) and D in (64, 128) and q.numel() > 0:
        return _AttnFn.apply(q, k, v)
    T = q.shape[-2]
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    mask = torch.triu(torch.ones(T, T, dtype=torch.bool, device=q.device), 1)
    return torch.softmax(s.masked_fill(mask, float("-inf")), -1) @ v


# ---------------------------------------------------------- cross-entropy
class _XentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets):
        V = logits.shape[-1]
        z = logits.reshape(-1, V).contiguous()
        loss, lse = K.xent_fwd(z, targets.reshape(-1))
        ctx.save_for_backward(z, targets, lse)
        ctx.shp = logits.shape
        return loss

    @staticmethod
    def backward(ctx, g):
        z, targets, lse = ctx.saved_tensors
        dz = z.clone()
        K.xent_bwd(dz, targets, lse, g.reshape(1).float())
        return dz.view(ctx.shp), None


def cross_entropy(logits, targets):
    """Mean cross-entropy over all positions; logits (..., V), targets (...)."""
    if _fast(logits) and logits.numel() > 0:
        return _XentFn.apply(logits, targets)
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1))


# ----------------------------------------------------- mixture of experts
def _route_math(z, k, softmax, bias, groups, keep, top, renorm, scale):
    """``route`` with torch ops (any device, fp32 or fp64 arithmetic)."""
    z = z if z.dtype == torch.float64 else z.float()
    n, e = z.shape
    gone = z == -math.inf
    if softmax:
        s = torch.softmax(z.masked_fill(gone.all(-1, keepdim=True), 0.0), -1).masked_fill(gone, 0.0)
    else:
        s = torch.sigmoid(z)
    with torch.no_grad():
        if bias is None and top == 1:
            c = z
        else:
            c = (s if bias is None else s + bias.to(s.dtype)).masked_fill(gone, -math.inf)
        if groups > 1:
            per = c.view(n, groups, e // groups)
            best = torch.sort(per, dim=-1, descending=True).values[..., :top]
            score = best[..., 0] + best[..., 1:].masked_fill(best[..., 1:] == -math.inf, 0.0).sum(-1)
            order = torch.sort(score, dim=-1, descending=True, stable=True).indices
            kept = torch.zeros_like(score, dtype=torch.bool).scatter_(1, order[:, :keep], True)
            c = per.masked_fill(~kept[..., None], -math.inf).reshape(n, e)
        c, idx = torch.sort(c, dim=-1, descending=True, stable=True)
        idx, none = idx[:, :k], c[:, :k] == -math.inf
        load = torch.bincount(idx.masked_fill(none, e).reshape(-1), minlength=e + 1)[:e].to(torch.int32)
    sj = s.gather(1, idx).masked_fill(none, 0.0)
    if renorm:
        sj = sj / sj.sum(-1, keepdim=True).clamp(min=1e-20)
    gates = scale * sj
    return gates, idx.masked_fill(none, -1).to(torch.int32), load


def route(logits, k: int, *, score: str = "softmax", bias=None, groups: int = 1, keep_groups: int = 1,
          group_top: int = 1, renorm: bool = True, scale: float = 1.0):
    """Choose ``k`` of the experts for each token: ``(gates, idx, load)``.

    ``logits`` (..., experts) become scores s by ``score``: "softmax" over the experts,
    or "sigmoid" of each.  The choice goes by the logits, or by s + ``bias`` (fp32
    [experts]; it balances the load and takes no part in the gates) - with
    ``group_top`` 2 always by the scores.  With ``groups`` > 1 the experts form that
    many equal groups in a row, and only the ``keep_groups`` best ones stay: by their
    best expert (``group_top`` 1) or the sum of their two best (2).  Ties go to the
    lowest expert (group).  gates (..., k), fp32 and in falling order of the choice,
    are ``scale * s``, divided by the sum of the k scores (at least 1e-20) where
    ``renorm``.  A logit of -inf masks an expert; slots that no expert is left for have
    idx -1 and gate 0.  A NaN counts as the largest value and shows in the gates.

    idx (..., k) is int32, load int32 [experts] counts the slots of each expert.  The
    gates are differentiable in the logits (through the kernels once: a second derivative
    raises; forward mode runs torch ops).
    """
    if logits.is_cuda:
        out = K.route(logits, k, score, bias, groups, keep_groups, group_top, renorm, scale)
        if out is not None:
            return out
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"route: score must be 'softmax' or 'sigmoid', got {score!r}")
    e = logits.shape[-1]
    if not 1 <= k <= e:
        raise ValueError(f"route: k must be in [1, {e}], got {k}")
    if groups < 1 or e % groups or not 1 <= keep_groups <= groups or keep_groups * (e // groups) < k:
        raise ValueError(f"route: {e} experts in {groups} groups, {keep_groups} kept, do not give {k} experts a token")
    if group_top not in (1, 2) or group_top > e // groups:
        raise ValueError(f"route: group_top must be 1, or 2 with groups of at least 2, got {group_top}")
    if bias is not None and (bias.shape != (e,) or bias.device != logits.device):
        raise ValueError(f"route: bias must be [{e}] on the logits' device")
    gates, idx, load = _route_math(logits.reshape(-1, e), k, score == "softmax", bias, groups, keep_groups, group_top,
                                   renorm, scale)
    return gates.view(*logits.shape[:-1], k), idx.view(*logits.shape[:-1], k), load


def _experts_math(x, w1, b1, w2, b2, idx, gates):
    """``expert_mlp`` with torch ops, expert by expert.  The products are of the inputs' type; a token's sums over
    its slots (and those of its gradient) are fp32 at least."""
    wide = torch.promote_types(x.dtype, torch.float32)
    rows, y = x.to(wide), x.new_zeros(x.shape[0], w2.shape[2], dtype=wide)
    for e in range(w1.shape[0]):
        tok, slot = torch.nonzero(idx == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        h = rows[tok].to(x.dtype) @ w1[e]
        h = F.gelu(h if b1 is None else h + b1[e], approximate="tanh") @ w2[e]
        h = h if b2 is None else h + b2[e]
        y = y.index_add(0, tok, gates[tok, slot][:, None].to(wide) * h.to(wide))
    return y.to(x.dtype)


def expert_mlp(x, w1, b1, w2, b2, idx, gates):
    """Mixture of MLPs: ``y = sum_j gates_j (gelu(x @ w1[e] + b1[e]) @ w2[e] + b2[e])``, e = idx_j.

    x (..., c); w1 [experts, c, h], w2 [experts, h, co] (in, out) as in ``linear``; b1
    [experts, h], b2 [experts, co] or None; idx (..., k) int32 or int64, where -1 is a
    slot without an expert; gates (..., k).  y (..., co) has x's type; gradients reach
    x, the weights, the biases and the gates, each in its own type (through the kernels once:
    a second derivative raises; forward mode runs torch ops).  An expert that no slot names
    gets a gradient of zeros.  Any layout will do: what is not contiguous from a 16-byte
    boundary on is copied for the kernels first.
    """
    if x.is_cuda:
        y = K.experts(x, w1, b1, w2, b2, idx, gates)
        if y is not None:
            return y
    c = x.shape[-1]
    if w1.dim() != 3 or w2.dim() != 3 or w1.shape[1] != c or w2.shape[:2] != (w1.shape[0], w1.shape[2]):
        raise ValueError(f"expert_mlp: x {tuple(x.shape)}, w1 {tuple(w1.shape)} and w2 {tuple(w2.shape)} do not fit")
    if idx.shape != gates.shape or idx.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"expert_mlp: idx {tuple(idx.shape)} and gates {tuple(gates.shape)} must be x's rows by slots")
    if idx.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_mlp: idx must be int32 or int64, got {idx.dtype}")
    k = idx.shape[-1]
    y = _experts_math(x.reshape(-1, c), w1, b1, w2, b2, idx.reshape(-1, k), gates.reshape(-1, k))
    return y.view(*x.shape[:-1], w2.shape[2])


# ---------------------------------------------------------------- others
def embedding(weight, idx):
    """weight[idx]; the backward scatter-adds repeated indices (dtrain/autograd.py:199-204)."""
    return weight[idx]


def gelu(x):
    """tanh-approximated GELU (dtrain/autograd.py:133-144)."""
    return F.gelu(x, approximate="tanh")


def relu(x):
    return torch.relu(x)
