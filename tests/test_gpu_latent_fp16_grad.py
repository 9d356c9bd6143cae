"""GPU: what the fp16 gradient of the expanded latent attention may lose, and what it may not."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs
from oracle import latent as O

pytestmark = pytest.mark.gpu


def _grads(q, kv, kr, do, **kw):
    q, kv, kr = (x.detach().requires_grad_(True) for x in (q, kv, kr))
    o = axiom_amd.latent_attn(q, kv, kr, **kw)
    return o.detach(), torch.autograd.grad(o, (q, kv, kr), do)


def _rounded(x):
    """fp16 of x times the column's power of two that brings its largest value into [2^10, 2^11)."""
    f = torch.exp2(10 - torch.floor(torch.log2(x.abs().amax(0, keepdim=True).clamp_min(1e-300))))
    return (x * f).half().double() / f


@pytest.mark.parametrize("dn,dr,T,H", [(128, 64, 1000, 4), (64, 32, 1000, 4), (128, 32, 513, 4)])
def test_only_the_operand_and_the_result_are_rounded(cuda, dn, dr, T, H):
    """dk's error is that of g as an fp16 operand and of the result: p enters g unrounded.

    The same roundings restated in float64, with D from the forward's rounded o in
    the rows past the first 128 as the kernels take it; everything else the
    kernels do is in fp32, 2^13 times finer.  A p rounded to fp16 on its way
    into g would add as much again as g's rounding: 1.2 times in all.  Some
    10^5 elements: the ratio of two such errors is known to better than 0.02.
    """
    q, kv, kr, do = attn_inputs(1, T, T, H, dn, dr, "fp16", cuda, seed=T + dn)
    o, (_, dkv, _) = _grads(q, kv, kr, do)
    _, _, _, ref, _ = O.attn(q, kv, kr, True, None, None, None, do)
    scale = (dn + dr) ** -0.5
    see = torch.tril(torch.ones(T, T, dtype=torch.bool))
    errs = []
    for h in range(H):
        Q, dO = q[0, :, h].cpu().double(), do[0, :, h].cpu().double()
        K, V = torch.cat([kv[0, :, h, :dn], kr[0]], 1).cpu().double(), kv[0, :, h, dn:].cpu().double()
        p = torch.softmax((scale * (Q @ K.T)).masked_fill(~see, float("-inf")), -1)
        dp = dO @ V.T
        D = torch.where(torch.arange(T) < 128, (p * dp).sum(1), (dO * o[0, :, h].cpu().double()).sum(1))
        g = _rounded(p * (dp - D[:, None]))
        restated = (scale * (g.T @ Q[:, :dn])).half().double()
        want, got = ref[0, :, h, :dn], dkv[0, :, h, :dn].cpu().double()
        errs.append(((got - want).norm() / (restated - want).norm()).item())
    print("  error over the roundings' own:", " ".join(f"{e:.3f}" for e in errs), flush=True)
    assert max(errs) <= 1.05
