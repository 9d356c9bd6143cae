"""Shared helpers of the latent-attention tests: inputs and the bars.

The bars follow from the roundings.  With u the unit roundoff of the inputs'
type (bf16 2^-8, fp16 2^-11), o is rounded once and its probabilities once: 2 u.
A gradient's terms are p, g and o (in D, twice: against do and in the
difference) and the result's own rounding: 5 u.  fp32 keeps 1e-5, the package's
bar for its exact mode: its sums, products and base-2 exponentials each carry a
few units of 2^-24, the sums over up to thousands of terms.  Every (batch, head)
slice meets the bar in relative L2, and every element ten times the bar
against the larger of the slice's rms and its own magnitude.

A gradient through the softmax is a difference, do . v - D, that vanishes where
a query has one key: there its error is set against a tenth of the terms' own
size (``terms``), which is what the difference of a row of a hundred keys keeps.
"""

from __future__ import annotations

import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def bar(dtype, grad=False):
    return 1e-5 if dtype == "fp32" else (5 if grad else 2) * U[dtype]


def terms(q, kv, k_rope, do):
    """Size of one term of a gradient: scale |do . v| |k|, root mean squares."""
    r = [x.double().square().mean().sqrt().item() if x.numel() else 0.0 for x in (q, kv, k_rope, do)]
    return (q.shape[-1] ** -0.5) * (do.shape[-1] ** 0.5) * r[3] * r[1] * max(r[1], r[2])


def check(name, got, ref, tol, axes, floor=0.0):
    """Slices at one index of ``axes`` each within ``tol`` (relative L2; ten times it per
    element) of their size, or of ``floor`` where that is larger."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)} for {tuple(ref.shape)}"
    assert torch.isfinite(got).all(), f"{name}: not finite"
    red = [i for i in range(ref.dim()) if i not in axes]
    err = (got - ref).abs()
    rms = ref.square().mean(red, keepdim=True).sqrt().clamp_min(floor)
    rel = (err.square().mean(red, keepdim=True).sqrt() / rms.clamp_min(1e-30)).nan_to_num(0.0)
    zero = (rms == 0) & (err.amax(red, keepdim=True) == 0)
    rel = torch.where(zero, torch.zeros_like(rel), rel)
    worst = (err / torch.maximum(rms, ref.abs()).clamp_min(1e-30)).max().item() if err.numel() else 0.0
    top = rel.max().item() if rel.numel() else 0.0
    print(f"  {name}: rel {top:.2e} element {worst:.2e} (bar {tol:.2e})", flush=True)
    assert top <= tol and worst <= 10 * tol, f"{name}: rel {top:.3e}, element {worst:.3e}, bar {tol:.3e}"


def check_lse(name, got, ref):
    got = got.detach().cpu().double()
    none = torch.isinf(ref)
    assert torch.equal(torch.isneginf(got), none), f"{name}: rows without a key"
    err = (got - ref)[~none].abs()
    assert err.numel() == 0 or (err <= 1e-5 * (1 + ref[~none].abs())).all(), f"{name}: {err.max():.3e}"


def attn_inputs(B, Tq, Tk, H, dn, dr, dtype, device, seed=0, views=False):
    """q, kv, k_rope, do; ``views``: slices of wider projections (rows with strides of their own)."""
    g = torch.Generator(device=device).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, device=device, generator=g).to(DT[dtype])

    pad = 16 if views else 0
    q = rnd(B, Tq, H, dn + dr + pad)[..., :dn + dr] * 1.5
    if views:
        q = rnd(B, H, Tq, dn + dr + pad).transpose(1, 2)[..., pad:]
    kv = rnd(B, Tk + 3, H, 2 * dn)[:, 2:Tk + 2] if views else rnd(B, Tk, H, 2 * dn)
    kr = rnd(B, Tk, 4 * pad + dr)[..., 4 * pad:]
    return q, kv, kr, rnd(B, Tq, H, dn)
