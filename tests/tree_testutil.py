"""Shared helpers of the tree tests: trees and inputs.

Bars.  The KDA calls compute in fp32 from the inputs as they are, so every type of
input keeps 1e-5, the package's bar for its exact mode (sums of 128 terms, products
and base-2 exponentials of a few units of 2^-24 each); a bf16 output adds its own
rounding, 2^-8.  The latent call's bars are its neighbours' (latent_testutil).
"""

from __future__ import annotations

import random

import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def tree(kind, N, seed=0):
    """Parents of N places."""
    rng = random.Random(seed)
    if kind == "chain":
        return [i - 1 for i in range(N)]
    if kind == "star":
        return [-1] * N
    if kind == "none":
        return [-2] * N
    if kind == "random":
        return [rng.randint(-1, i - 1) for i in range(N)]
    if kind == "deep":       # a chain with side branches of one
        return [-1 if i < 2 else i - 2 + (i % 2) if i % 3 else i - 2 for i in range(N)]
    assert kind == "broken"  # entries of every wrong kind; places below them hold no draft either
    wrong = [-2, -100, N, 2**31 - 1, -2**31, 5000]
    row = [rng.randint(-1, i - 1) for i in range(N)]
    for i in range(N):
        if rng.random() < 0.3:
            row[i] = rng.choice(wrong + [i, i + 1])
    return row


def trees(kinds, N, device, seed=0):
    return torch.tensor([tree(k, N, seed + 7 * b) for b, k in enumerate(kinds)], dtype=torch.int32, device=device)


def step_inputs(B, N, H, d, dtype, device, seed=0, decay=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, device=device, generator=gen)

    q, k = rnd(B, N, H, d), rnd(B, N, H, d)
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    g = -decay * torch.nn.functional.softplus(rnd(B, N, H, d))
    t = DT[dtype]
    return dict(q=q.to(t), k=k.to(t), v=rnd(B, N, H, d).to(t), g=g.to(t), beta=torch.sigmoid(rnd(B, N, H)).to(t),
                state=0.1 * rnd(B, H, d, d))
