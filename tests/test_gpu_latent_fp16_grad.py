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


# relative L2 of a part: p, g and the result are rounded (2^-11 each) and o in D, twice; below 2^-14
# the results themselves round to fp16's absolute step, 2^-25
def _close(name, got, ref):
    err = (got.cpu().double() - ref).square().mean().sqrt().item()
    rms = ref.square().mean().sqrt().item()
    print(f"  {name}: error {err:.2e} of {rms:.2e} ({err / rms:.2e})", flush=True)
    assert err <= 5 * 2.0 ** -11 * rms + 2.0 ** -25, f"{name}: {err:.3e} of {rms:.3e}"


@pytest.mark.parametrize("less", [10, 12, 14])
@pytest.mark.parametrize("dn,dr", [(64, 32), (128, 64)])
def test_packed_sequences_of_different_cotangents(cuda, dn, dr, less):
    """A sequence whose do is 2^-10 to 2^-14 of its neighbours' keeps its gradients' precision."""
    q, kv, kr, do = attn_inputs(1, 1100, 1100, 2, dn, dr, "fp16", cuda, seed=less)
    do = do.float() * 16
    do[:, 300:800] *= 2.0 ** -less
    do = do.half()
    cu = torch.tensor([0, 300, 800, 1100], dtype=torch.int32, device=cuda)
    _, _, *ref = O.attn(q, kv, kr, True, None, cu.tolist(), None, do)
    _, grads = _grads(q, kv, kr, do, cu_seqlens=cu)
    for name, got, r in zip(("dq", "dkv", "dk_rope"), grads, ref):
        for a, e in ((0, 300), (300, 800), (800, 1100)):
            _close(f"{name} {a}", got[:, a:e], r[:, a:e])


@pytest.mark.parametrize("less", [10, 14])
@pytest.mark.parametrize("T,late", [(40, 30), (130, 120), (1000, 500), (1000, 990), (3000, 1500)])
def test_late_queries_of_smaller_cotangents(cuda, T, late, less):
    """Keys that only queries of small do see; both the parts of a tile and whole blocks."""
    q, kv, kr, do = attn_inputs(1, T, T, 2, 64, 32, "fp16", cuda, seed=T + late)
    do = do.float() * 16
    do[:, late:] *= 2.0 ** -less
    do = do.half()
    _, _, *ref = O.attn(q, kv, kr, True, None, None, None, do)
    _, grads = _grads(q, kv, kr, do)
    for name, got, r in zip(("dq", "dkv", "dk_rope"), grads, ref):
        _close(f"{name} early", got[:, :late], r[:, :late])
        _close(f"{name} late", got[:, late:], r[:, late:])


@pytest.mark.parametrize("dn,dr", [(64, 32), (128, 64)])
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -9, 1.9])
def test_large_values(cuda, dn, dr, size):
    """do . v past fp16's largest value, the gradients inside its range: g is an operand, not a result."""
    q, kv, kr, do = attn_inputs(1, 150, 150, 2, dn, dr, "fp16", cuda, seed=dn)
    sign = torch.where(torch.arange(150, device=cuda) % 2 == 0, 1.0, -1.0)[None, :, None, None]
    kv = torch.cat([kv[..., :dn], (900 + 100 * torch.rand_like(kv[..., dn:].float())).half() * sign.half()], -1)
    q, kv, kr = q * 0.25, kv.contiguous(), kr.contiguous()
    kv[..., :dn] *= 0.0625
    kr *= 0.0625
    do = (size * (0.9 + 0.1 * torch.rand_like(do.float()))).half()
    _, _, *ref = O.attn(q, kv, kr, True, None, None, None, do)
    assert all(r.abs().max() < 60000 for r in ref)
    _, grads = _grads(q, kv, kr, do)
    for name, got, r in zip(("dq", "dkv", "dk_rope"), grads, ref):
        assert torch.isfinite(got).all(), name
        _close(name, got, r)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_packed_neighbour_not_finite(cuda, bad):
    """A sequence whose inputs and cotangents are not finite leaves its neighbours' gradients as they were."""
    q, kv, kr, do = attn_inputs(1, 700, 700, 2, 64, 32, "fp16", cuda, seed=12)
    do = do * 2.0 ** -10
    cu = torch.tensor([0, 70, 330, 700], dtype=torch.int32, device=cuda)
    _, grads = _grads(q, kv, kr, do, cu_seqlens=cu)
    spoiled = [x.clone() for x in (q, kv, kr, do)]
    for x in spoiled:
        x[:, 70:330] = bad
    _, grads2 = _grads(*spoiled, cu_seqlens=cu)
    for name, x, y in zip(("dq", "dkv", "dk_rope"), grads, grads2):
        for a, e in ((0, 70), (330, 700)):
            assert torch.equal(x[:, a:e], y[:, a:e]), name
