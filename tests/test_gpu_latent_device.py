"""GPU: calls on tensors of a device that is not the current one (two GPUs needed)."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")]


def test_tensors_of_another_device(cuda):
    other = torch.device("cuda:1")
    q, kv, kr, do = attn_inputs(1, 150, 150, 2, 64, 32, "bf16", cuda, seed=1)
    rows, cache = torch.randn(4, 288, device=cuda), torch.zeros(2, 16, 288, device=cuda)
    pos, cs = torch.arange(4, device=cuda), torch.randn(8, 32, device=cuda)
    qa, table = torch.randn(1, 1, 4, 288, device=cuda), torch.arange(2, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([4], dtype=torch.int32, device=cuda)

    def calls(to):
        a, b, c, d = (x.to(to).detach().requires_grad_(True) for x in (q, kv, kr, do))
        o = axiom_amd.latent_attn(a, b, c)
        page = cache.to(to).clone()
        axiom_amd.latent_append(rows.to(to), pos.to(to), pos.to(to), cs.to(to), page)
        return [o, *torch.autograd.grad(o, (a, b, c), d), page, *axiom_amd.latent_decode(qa.to(to), page, table.to(to), lens.to(to), 0.1)]

    want = calls(cuda)
    with torch.cuda.device(0):
        got = calls(other)
        assert torch.cuda.current_device() == 0
    for x, y in zip(got, want):
        assert x.device == other and torch.equal(x.cpu(), y.cpu())
