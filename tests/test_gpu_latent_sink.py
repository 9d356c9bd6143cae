"""GPU: a key that outweighs each of very many others, which together still count.

The others' probabilities are 4e-8 of the leading one's, below fp16's smallest step
of 6e-8; 150 000 of them hold 6e-3 of the row.  o must meet the type's bar: the
probabilities' roundings are relative to what they add up to.
"""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import DT, bar, check, check_lse
from oracle import latent as O

pytestmark = pytest.mark.gpu

N, LEAD = 150000, 17.0     # keys, and the leading score above the others'


@pytest.mark.parametrize("H", [16, 40])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("where", [0, N // 2, N - 1])
def test_decode(cuda, H, dtype, where):
    R, dr, page = 256, 32, 64
    g = torch.Generator(device=cuda).manual_seed(H)
    pages = -(-N // page)
    cache = torch.zeros(pages, page, R + dr, device=cuda)
    rows = cache.view(-1, R + dr)
    rows[:, 1:R] = 1 + 0.25 * torch.randn(rows.shape[0], R - 1, device=cuda, generator=g)   # what the row adds up
    rows[where, 0] = LEAD                                                                   # the score's only part
    q = torch.zeros(1, 1, H, R + dr, device=cuda)
    q[..., 0] = 1
    cache, q = cache.to(DT[dtype]), q.to(DT[dtype])
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([N], dtype=torch.int32, device=cuda)
    rows = cache.view(-1, R + dr)
    rows[where, 1:R] = -1                                                                   # and the leading row the other way
    o_ref, lse_ref = O.decode(q, cache, table, lens, R, 1.0)
    o, lse = axiom_amd.latent_decode(q, cache, table, lens, scale=1.0)
    check("o", o[..., 1:], o_ref[..., 1:], bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded(cuda, causal, dtype):
    g = torch.Generator(device=cuda).manual_seed(1)
    dn, dr, H, Tq = 64, 32, 1, 40
    q, kv, kr = torch.zeros(1, Tq, H, dn + dr, device=cuda), torch.zeros(1, N, H, 2 * dn, device=cuda), torch.zeros(1, N, dr, device=cuda)
    q[..., 0] = 1
    kv[:, 1000, :, 0] = LEAD
    kv[..., dn:] = 1 + 0.25 * torch.randn(1, N, H, dn, device=cuda, generator=g)
    kv[:, 1000, :, dn:] = -1
    q, kv, kr = (x.to(DT[dtype]) for x in (q, kv, kr))
    o_ref, lse_ref = O.attn(q, kv, kr, causal, 1.0)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, causal=causal, scale=1.0)
    check("o", o, o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_expanded_in_one_walk(cuda, dtype):
    """So many queries that no block's keys are shared out: one running maximum over all of them."""
    g = torch.Generator(device=cuda).manual_seed(2)
    dn, dr, Tq = 64, 32, 258 * 128
    q, kv, kr = torch.zeros(1, Tq, 1, dn + dr, device=cuda), torch.zeros(1, N, 1, 2 * dn, device=cuda), torch.zeros(1, N, dr, device=cuda)
    q[..., 0] = 1
    kv[:, 1000, :, 0] = LEAD
    kv[..., dn:] = 1 + 0.25 * torch.randn(1, N, 1, dn, device=cuda, generator=g)
    kv[:, 1000, :, dn:] = -1
    q, kv, kr = (x.to(DT[dtype]) for x in (q, kv, kr))
    o_ref, lse_ref = O.attn(q[:, :1], kv, kr, False, 1.0)   # all queries are alike
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, causal=False, scale=1.0)
    assert (o == o[:, :1]).all() and (lse == lse[:, :, :1]).all()
    check("o", o[:, :1], o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse[:, :, :1], lse_ref)
