"""AdamW over flat tensors, and global-norm clipping.

API of dtrain/optim.py:7-52: ``AdamW(params, lr, betas, eps, weight_decay)`` with
``step(grads)``, ``state_dict()``, ``load_state_dict()``, ``state_bytes()``, and
``clip_scale(total_sq_norm, max_norm)``; beyond the reference, ``global_norm`` and
``clip_grads`` over a list of separate gradient tensors.  Parameters are updated in place, so
ZeRO can run the optimizer on a shard view of the flat master buffer.

Two code paths with the same formula and order of operations
(m = b1 m + (1-b1) g; v = b2 v + (1-b2) g^2; p -= lr*wd*p; p -= lr*(m/b1t)/(sqrt(v/b2t)+eps)):

* fp32 CUDA tensors -> the fused ``adamw_step`` kernel (one pass over p, g, m, v,
  also refreshing the bf16 working copy; the clip factor is computed on the device
  from a device-resident squared norm, so nothing waits on the host);
* anything else (CPU, float64) -> elementwise torch ops in exactly the reference's
  order, which makes float64 runs bit-identical to the NumPy reference.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def clip_scale(total_sq_norm: float, max_norm: float) -> float:
    """Factor that brings the global L2 norm down to ``max_norm`` (1.0 if already below)."""
    n = math.sqrt(float(total_sq_norm))
    return 1.0 if n <= max_norm or n == 0 else max_norm / (n + 1e-6)


def _on_gpu(grads) -> bool:
    """Whether the kernels take the list: its first tensor decides, the others must be like it."""
    g = next((g for g in grads if g is not None), None)
    return isinstance(g, torch.Tensor) and g.is_cuda and g.dtype in (torch.float32, torch.bfloat16, torch.float16)


def _floating(name, grads):
    ts = [g for g in grads if g is not None]
    for g in ts:
        if not isinstance(g, torch.Tensor) or not g.is_floating_point():
            raise TypeError(f"{name}: floating tensors expected, got {g.dtype if isinstance(g, torch.Tensor) else type(g)}")
    return ts


def _bytes(t, lo: int, hi: int) -> torch.Tensor:
    """Which of the addresses [lo, hi) belong to ``t``."""
    hit = torch.zeros(hi - lo, dtype=torch.bool)
    n = t.element_size()
    hit.as_strided((*t.shape, n), (*(s * n for s in t.stride()), 1), t.data_ptr() - lo).fill_(True)
    return hit


def _check_apart(grads, outs) -> None:
    """Outputs share no memory with one another nor with a gradient, their own in place apart (as csrc/clip.cu)."""
    ranges = []
    for i, (g, o) in enumerate(zip(grads, outs)):
        if g.numel() == 0 or g.layout != torch.strided or o.layout != torch.strided:
            continue
        place = lambda t: (t.data_ptr(), t.dtype, [s for n, s in zip(t.shape, t.stride()) if n > 1])  # noqa: E731
        for t, out in ((g, False), (o, True)) if place(g) != place(o) else ((o, True),):
            lo = t.data_ptr()
            hi = lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
            if out and hi - lo < t.numel() * t.element_size() or (
                    out and not t.is_contiguous() and int(_bytes(t, lo, hi).sum()) < t.numel() * t.element_size()):
                raise RuntimeError(f"clip_grads: output {i} overlaps itself")
            ranges.append((lo, hi, i, out, t))
    ranges.sort(key=lambda r: r[0])
    near = []                                       # ranges that reach past the start of the present one
    for r in ranges:
        near = [q for q in near if q[1] > r[0]]
        for q in near:
            if r[3] or q[3]:
                lo, hi = q[0], max(q[1], r[1])
                if torch.any(_bytes(q[4], lo, hi) & _bytes(r[4], lo, hi)):
                    raise RuntimeError(f"clip_grads: tensors {q[2]} and {r[2]} overlap in memory" if q[2] != r[2] else
                                       f"clip_grads: output {r[2]} overlaps its gradient in memory without being it")
        near.append(r)


def global_norm(grads) -> torch.Tensor:
    """L2 norm of all tensors together (a scalar tensor on their device; fp32 on a GPU).
    None stands for an absent gradient.  Nothing waits on the host."""
    grads = list(grads)
    if _on_gpu(grads):
        from . import kernels as K
        return K.clip_grads(grads, None, 0.0, scale=False)
    ts = _floating("global_norm", grads)
    if not ts:
        return torch.zeros(())
    return torch.stack([g.detach().double().square().sum() for g in ts]).sum().sqrt()


def clip_grads(grads, max_norm: float, out=None) -> torch.Tensor:
    """Scale the gradients so that their global norm is at most ``max_norm``; returns the norm before.

    The factor is ``clip_scale``'s, computed on the device, so nothing waits on the host.
    ``grads`` may differ in size, layout and type (fp32, bf16, fp16); None stands for an
    absent one.  They are scaled in place, or, with ``out`` (a list aligned with
    ``grads``), written there scaled - possibly in another type, such as bf16 gradients
    into the slices of a flat fp32 buffer - and left as they are; the output of an absent
    gradient becomes 0, so that nothing of an earlier step stays in the buffer.  Outputs
    that overlap one another or a gradient (other than in place) are refused.  A NaN or
    infinite norm shows in the result: the gradients become NaN or 0, as with any clipping
    that does not look at the norm on the host.
    """
    grads = list(grads)
    if _on_gpu(grads):
        from . import kernels as K
        return K.clip_grads(grads, out, float(max_norm))
    if not max_norm >= 0:
        raise ValueError(f"clip_grads: max_norm must not be negative, got {max_norm}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"clip_grads: {len(grads)} gradients but {len(out)} outputs")
    ts = _floating("clip_grads", grads)
    to = ts if out is None else _floating("clip_grads", [o for g, o in zip(grads, out) if g is not None])
    absent = [] if out is None else _floating("clip_grads", [o for g, o in zip(grads, out) if g is None])
    if len(to) != len(ts) or any(o.shape != g.shape for g, o in zip(ts, to)):
        raise ValueError("clip_grads: every gradient needs an output of its own shape")
    _check_apart(ts + absent, to + absent)
    norm = global_norm(ts)
    with torch.no_grad():
        f = torch.where((norm <= max_norm) | (norm == 0), 1.0, max_norm / (norm + 1e-6))
        for g, o in zip(ts, to):
            o.copy_((g if g.dtype == torch.float64 else g.float()) * f.to(g.device))  # rounded once, to o's type
        for o in absent:
            o.zero_()
    return norm


def _to_tensor(x):
    if isinstance(x, np.ndarray):
        return torch.from_numpy(x)
    return x


class AdamW:
    def __init__(self, params, lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1, work=None):
        self.params = [_to_tensor(p) for p in params]
        self.lr, self.b1, self.b2, self.eps, self.wd = lr, betas[0], betas[1], eps, weight_decay
        self.m = [torch.zeros_like(p) for p in self.params]
        self.v = [torch.zeros_like(p) for p in self.params]
        self.work = list(work) if work is not None else [None] * len(self.params)
        self.t = 0

    def _fused_ok(self, p, g) -> bool:
        return (p.is_cuda and p.dtype == torch.float32 and g is not None and g.dtype == torch.float32
                and p.is_contiguous() and g.is_contiguous())

    def step(self, grads, sq_norm: torch.Tensor | None = None, max_norm: float = 0.0):
        """One update.  ``grads`` is a list aligned with the params (None skips one).

        With ``sq_norm`` (a device fp64 scalar, sum of squared gradients) and
        ``max_norm`` > 0 the gradients are clipped on the device.
        """
        self.t += 1
        b1t = 1 - self.b1 ** self.t
        b2t = 1 - self.b2 ** self.t
        for i, (p, g) in enumerate(zip(self.params, grads)):
            if g is None:
                continue
            g = _to_tensor(g)
            m, v = self.m[i], self.v[i]
            if self._fused_ok(p, g):
                from . import kernels as K
                K.adamw_step(p, g, m, v, self.work[i], self.lr, self.b1, self.b2, self.eps, self.wd, self.t,
                             sq_norm, max_norm)
                continue
            if sq_norm is not None and max_norm:
                g = g * clip_scale(float(sq_norm.reshape(-1)[0]), max_norm)
            with torch.no_grad():
                m.mul_(self.b1)
                m.add_((1 - self.b1) * g)
                v.mul_(self.b2)
                v.add_((1 - self.b2) * (g * g))
                p.sub_(self.lr * (self.wd * p))
                p.sub_(self.lr * (m / b1t) / (torch.sqrt(v / b2t) + self.eps))
                if self.work[i] is not None:
                    self.work[i].copy_(p)

    def state_bytes(self) -> int:
        return sum(a.numel() * a.element_size() for a in self.m) + sum(a.numel() * a.element_size() for a in self.v)

    def state_dict(self):
        return {"t": self.t, "m": [a.clone() for a in self.m], "v": [a.clone() for a in self.v]}

    def load_state_dict(self, s):
        self.t = int(s["t"])
        with torch.no_grad():
            for dst, src in zip(self.m, s["m"]):
                dst.copy_(_to_tensor(np.asarray(src)) if isinstance(src, np.ndarray) else src)
            for dst, src in zip(self.v, s["v"]):
                dst.copy_(_to_tensor(np.asarray(src)) if isinstance(src, np.ndarray) else src)
