"""Train a small mixture-of-experts GPT on one device.

    python examples/train_moe.py                      # bf16 on a GPU, fp32 on the CPU
    python examples/train_moe.py --experts 16 --topk 4 --dim 512 --steps 200

The parameters are bf16 tensors (views of one work buffer) with an fp32 master copy.
After each backward ``clip_grads`` takes the separate bf16 gradients, computes their
global norm and writes them, scaled, into the flat fp32 buffer that the fused AdamW
reads; AdamW refreshes the bf16 parameters, and the experts' balancing bias moves by
the step's load.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from dtrain_b200.models.moe import MoEGPT  # noqa: E402
from dtrain_b200.optim import AdamW, clip_grads  # noqa: E402


def flatten(params):
    """fp32 master, work buffer in the parameters' type (the parameters become its views) and gradient views."""
    n = sum(p.numel() for p in params)
    master = torch.cat([p.detach().reshape(-1).float() for p in params])
    work = torch.empty(n, dtype=params[0].dtype, device=params[0].device)
    work.copy_(master)
    grad = torch.zeros_like(master)
    views, off = [], 0
    for p in params:
        p.data = work[off:off + p.numel()].view(p.shape)
        views.append(grad[off:off + p.numel()].view(p.shape))
        off += p.numel()
    return master, work, grad, views


def batch(gen, B, T, vocab, device):
    """Sequences that follow x -> 5 x + 3 (mod vocab) from a random start, one token in ten replaced."""
    x = torch.empty(B, T + 1, dtype=torch.int64)
    x[:, 0] = torch.randint(0, vocab, (B,), generator=gen)
    for t in range(T):
        x[:, t + 1] = (5 * x[:, t] + 3) % vocab
    noise = torch.rand(B, T + 1, generator=gen) < 0.1
    x[noise] = torch.randint(0, vocab, (int(noise.sum()),), generator=gen)
    return x[:, :-1].to(device), x[:, 1:].to(device)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, v in dict(steps=60, batch=16, ctx=128, vocab=256, dim=128, heads=2, layers=2, experts=8, topk=2, seed=0).items():
        ap.add_argument(f"--{name}", type=int, default=v)
    ap.add_argument("--lr", type=float, default=2e-3)
    ap.add_argument("--clip", type=float, default=1.0)
    ap.add_argument("--score", choices=("softmax", "sigmoid"), default="sigmoid")
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    a = ap.parse_args(argv)
    dtype = torch.bfloat16 if a.device.startswith("cuda") else torch.float32
    model = MoEGPT(a.vocab, a.ctx, a.dim, a.heads, a.layers, a.experts, a.topk, seed=a.seed, dtype=dtype,
                   score=a.score).to(a.device)
    params = list(model.parameters())
    master, work, grad, views = flatten(params)
    opt = AdamW([master], lr=a.lr, weight_decay=0.01, work=[work])
    gen = torch.Generator().manual_seed(a.seed)
    losses = []
    for step in range(a.steps):
        x, y = batch(gen, a.batch, a.ctx, a.vocab, a.device)
        _, loss = model(x, y)
        loss.backward()
        norm = clip_grads([p.grad for p in params], a.clip, out=views)
        opt.step([grad])
        load = model.blocks[0].moe.load.clone()
        model.balance()
        for p in params:
            p.grad = None
        losses.append(loss.detach())
        if step % 10 == 0 or step == a.steps - 1:
            print(f"step {step:4d}  loss {float(losses[-1]):.4f}  grad norm {float(norm):.3f}  "
                  f"load of block 0: {int(load.min())}..{int(load.max())}", flush=True)
    return [float(v) for v in losses]


if __name__ == "__main__":
    main()
