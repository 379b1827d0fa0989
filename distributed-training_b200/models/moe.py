"""Mixture-of-experts MLP layer and a GPT of such layers.

The layer takes the place of the dense MLP of dtrain/nn.py:90-101: a gate scores the
experts for each token, ``route`` chooses ``topk`` of them, ``expert_mlp`` computes
and joins their outputs (the same GELU MLP with biases, weights stored (in, out)).
With ``score="sigmoid"`` the load is balanced by a bias that takes part in the choice
only: after a step, ``balance`` moves it up for experts that got fewer tokens than
the mean and down for the others, by a fixed amount.

``MoEGPT`` is a GPT whose blocks use it.  Its parameters are separate tensors of one
type: bf16 on a GPU runs the kernels, fp32 and fp64 the torch math on any device.
Both serve one device: DDP, ZeroAdamW and Trainer need a model's flat buffers, which
``MoEGPT`` does not have, and ``balance`` goes by the load of its own process.
"""
from __future__ import annotations

import numpy as np
import torch
from torch import nn

from ..ops import functional as F


def _param(rng, shape, std, dtype) -> nn.Parameter:
    a = rng.standard_normal(shape).astype(np.float32) * std if std else np.zeros(shape, np.float32)
    return nn.Parameter(torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dtype))


class MoE(nn.Module):
    """y = sum over the chosen experts of gate * MLP_e(x), for x (..., dim)."""

    def __init__(self, dim, hidden, experts, topk, rng, dtype=torch.float32, *, score="sigmoid", groups=1,
                 keep_groups=1, group_top=1, scale=1.0, out_std=0.02):
        super().__init__()
        self.topk = topk
        self.how = dict(score=score, groups=groups, keep_groups=keep_groups, group_top=group_top, scale=scale)
        self.gate = _param(rng, (dim, experts), 0.02, dtype)
        self.w1 = _param(rng, (experts, dim, hidden), 0.02, dtype)
        self.b1 = _param(rng, (experts, hidden), 0.0, dtype)
        self.w2 = _param(rng, (experts, hidden, dim), out_std, dtype)
        self.b2 = _param(rng, (experts, dim), 0.0, dtype)
        self.register_buffer("bias", torch.zeros(experts) if score == "sigmoid" else None)
        self.register_buffer("load", torch.zeros(experts, dtype=torch.int32))

    def forward(self, x):
        gates, idx, load = F.route(F.linear(x, self.gate), self.topk, bias=self.bias, **self.how)
        if self.training:
            self.load += load
        return F.expert_mlp(x, self.w1, self.b1, self.w2, self.b2, idx, gates)

    @torch.no_grad()
    def balance(self, rate: float = 1e-3):
        """Move the balancing bias by the load seen since the last call."""
        if self.bias is not None:
            n = self.load.float()
            self.bias += rate * torch.sign(n.mean() - n)
        self.load.zero_()


class _Block(nn.Module):
    def __init__(self, dim, heads, hidden, experts, topk, layers, rng, dtype, **how):
        super().__init__()
        self.heads = heads
        one = lambda n: nn.Parameter(torch.ones(n, dtype=dtype))  # noqa: E731
        self.ln1_w, self.ln1_b = one(dim), _param(rng, dim, 0.0, dtype)
        self.qkv_w, self.qkv_b = _param(rng, (dim, 3 * dim), 0.02, dtype), _param(rng, 3 * dim, 0.0, dtype)
        deep = 0.02 / np.sqrt(2 * layers)
        self.proj_w, self.proj_b = _param(rng, (dim, dim), deep, dtype), _param(rng, dim, 0.0, dtype)
        self.ln2_w, self.ln2_b = one(dim), _param(rng, dim, 0.0, dtype)
        self.moe = MoE(dim, hidden, experts, topk, rng, dtype, out_std=deep, **how)

    def forward(self, x):
        B, T, C = x.shape
        qkv = F.linear(F.layer_norm(x, self.ln1_w, self.ln1_b), self.qkv_w, self.qkv_b)
        q, k, v = qkv.view(B, T, 3, self.heads, C // self.heads).permute(2, 0, 3, 1, 4)
        a = F.causal_attention(q, k, v).transpose(1, 2).reshape(B, T, C)
        x = x + F.linear(a, self.proj_w, self.proj_b)
        return x + self.moe(F.layer_norm(x, self.ln2_w, self.ln2_b))


class MoEGPT(nn.Module):
    """GPT with a mixture of experts in every block; ``forward`` as models/gpt.py:GPT's."""

    def __init__(self, vocab, ctx, dim, heads, layers, experts, topk=2, hidden=None, seed=0, dtype=torch.float32, **how):
        super().__init__()
        rng = np.random.default_rng(seed)
        self.tok, self.pos = _param(rng, (vocab, dim), 0.02, dtype), _param(rng, (ctx, dim), 0.01, dtype)
        self.blocks = nn.ModuleList(_Block(dim, heads, hidden or 4 * dim, experts, topk, layers, rng, dtype, **how)
                                    for _ in range(layers))
        self.ln_w, self.ln_b = nn.Parameter(torch.ones(dim, dtype=dtype)), _param(rng, dim, 0.0, dtype)
        self.head = _param(rng, (dim, vocab), 0.02, dtype)

    def forward(self, idx, targets=None):
        x = F.embedding(self.tok, idx) + self.pos[:idx.shape[1]]
        for b in self.blocks:
            x = b(x)
        logits = F.linear(F.layer_norm(x, self.ln_w, self.ln_b), self.head)
        if targets is None:
            return logits
        return logits, F.cross_entropy(logits, targets)

    def balance(self, rate: float = 1e-3):
        for b in self.blocks:
            b.moe.balance(rate)
