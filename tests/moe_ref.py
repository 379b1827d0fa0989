"""Plain 64-bit definitions of the mixture-of-experts operators, token by token, for the tests."""
import math

import torch


def route64(z, k, *, softmax=True, bias=None, groups=1, keep=1, top=1, renorm=True, scale=1.0):
    """Row by row in Python floats: (gates fp64 [n, k], idx [n, k], load [e])."""
    n, e = z.shape
    gates, idx = torch.zeros(n, k, dtype=torch.float64), torch.full((n, k), -1, dtype=torch.int64)
    load = torch.zeros(e, dtype=torch.int64)
    b = [0.0] * e if bias is None else bias.double().tolist()
    for t, row in enumerate(z.double().tolist()):
        live = [i for i in range(e) if row[i] != -math.inf]
        if softmax and live:
            m = max(row[i] for i in live)
            w = {i: math.exp(row[i] - m) for i in live}
            total = sum(w.values())
            s = {i: w[i] / total for i in live}
        else:
            s = {i: 1.0 / (1.0 + math.exp(-row[i])) for i in live}
        c = {i: row[i] if bias is None and top == 1 else s[i] + b[i] for i in live}
        if groups > 1:
            per = e // groups
            score = []
            for g in range(groups):
                best = sorted((c[i] for i in live if i // per == g), reverse=True)[:top]
                score.append(sum(best) if best else -math.inf)
            kept = set(sorted(range(groups), key=lambda g: (-score[g], g))[:keep])
            live = [i for i in live if i // per in kept]
        chosen = sorted(live, key=lambda i: (-c[i], i))[:k]
        d = max(sum(s[i] for i in chosen), 1e-20) if renorm else 1.0
        for j, i in enumerate(chosen):
            gates[t, j] = scale * s[i] / d
            idx[t, j] = i
            load[i] += 1
    return gates, idx, load


def gates64(z, idx, *, softmax=True, renorm=True, scale=1.0):
    """The gates of given choices as a differentiable fp64 function of the logits (idx -1: gate 0)."""
    none = idx < 0
    gone = z == -math.inf
    safe = z.masked_fill(gone, -1e30)
    if softmax:
        s = torch.softmax(safe, -1).masked_fill(gone, 0.0)
    else:
        s = torch.sigmoid(safe)
    sj = s.gather(1, idx.clamp(min=0).long()).masked_fill(none, 0.0)
    if renorm:
        sj = sj / sj.sum(-1, keepdim=True).clamp(min=1e-20)
    return scale * sj


def gelu64(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))


def experts64(x, w1, b1, w2, b2, idx, gates):
    """fp64 and differentiable: every expert on every token, the unused ones dropped."""
    y = 0.0
    for e in range(w1.shape[0]):
        h = x @ w1[e] + (0.0 if b1 is None else b1[e])
        o = gelu64(h) @ w2[e] + (0.0 if b2 is None else b2[e])
        g = (gates * (idx == e)).sum(-1, keepdim=True)
        y = y + g * o
    return y
