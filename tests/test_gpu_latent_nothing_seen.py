"""GPU: a query that sees no key has o = 0, lse = -inf and dq = 0, whatever the keys it does not see hold."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import DT, attn_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("Tq,Tk,H", [(70, 50, 2), (900, 700, 3), (400, 300, 64)])
def test_expanded(cuda, Tq, Tk, H, bad, dtype):
    """Causal, more queries than keys; 900 x 700: the walks are shared out and joined."""
    q, kv, kr, do = attn_inputs(1, Tq, Tk, H, 64, 32, dtype, cuda, seed=Tq)
    kr = kr.contiguous()
    none = Tq - Tk
    kv[:, 0], kr[:, 0] = bad, bad                      # the first key, in a tile with the rows' wave
    kv[:, 20, :, 64:] = bad
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr)
    assert (o[:, :none] == 0).all() and torch.isneginf(lse[:, :, :none]).all()
    assert not torch.isfinite(o[:, none:]).any(-1).any()   # every other row sees the first key
    dq, _, _ = axiom_amd.latent_attn_bwd(q, kv, kr, o, lse, do)
    assert (dq[:, :none] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_packed(cuda, dtype):
    q, kv, kr, do = attn_inputs(1, 300, 170, 2, 128, 64, dtype, cuda, seed=3)
    kr = kr.contiguous()
    cu, cu_k = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 90, 100, 300], [0, 30, 30, 170]))
    kv[:], kr[:] = float("nan"), float("nan")
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, cu_seqlens=cu, cu_seqlens_k=cu_k)
    dq, _, _ = axiom_amd.latent_attn_bwd(q, kv, kr, o, lse, do, cu_seqlens=cu, cu_seqlens_k=cu_k)
    none = torch.zeros(300, dtype=torch.bool, device=cuda)
    none[:60] = none[90:100] = none[100:160] = True
    for x in (o, dq):
        assert (x[:, none] == 0).all() and torch.isnan(x[:, ~none]).all()
    assert torch.isneginf(lse[:, :, none]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H", [4, 24])
@pytest.mark.parametrize("per", [2, 20])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_decode(cuda, per, H, dtype, bad):
    """Sequences shorter than the tokens that are asked: the first tokens see nothing.  A table of 128
    tokens (a workgroup a sequence) and a longer one (runs and a join)."""
    Tq, R, dr, page = 4, 512, 64, 64
    lens = torch.tensor([3, 1, 200 if per == 20 else 100, 4, 0, 2], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(H)
    cache = torch.randn(6 * per, page, R + dr, device=cuda, generator=g).to(DT[dtype])
    table = torch.arange(6 * per, dtype=torch.int32, device=cuda).view(6, per)
    for b in (0, 1, 3, 5):
        cache[b * per] = bad
    q = torch.randn(6, Tq, H, R + dr, device=cuda, generator=g).to(DT[dtype])
    o, lse = axiom_amd.latent_decode(q, cache, table, lens, scale=0.05)
    for b, n in enumerate(lens.tolist()):
        none = min(Tq, max(0, Tq - n))
        assert (o[b, :none] == 0).all() and torch.isneginf(lse[b, :none]).all(), b
        if b in (0, 1, 3, 5):
            assert not torch.isfinite(o[b, none:]).any(), b
        elif n:
            assert torch.isfinite(o[b]).all() and torch.isfinite(lse[b]).all()
