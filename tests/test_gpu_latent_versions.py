"""GPU: tensors that the latent operators write in place are known to autograd as written."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs

pytestmark = pytest.mark.gpu


def _append_args(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    rows = torch.randn(3, 288, device=cuda, generator=g)
    pos = torch.arange(3, device=cuda)
    return rows, pos, pos, torch.randn(8, 32, device=cuda, generator=g)


def test_append(cuda):
    cache, q, qa = torch.zeros(2, 16, 288, device=cuda), torch.randn(3, 2, 32, device=cuda), torch.zeros(3, 2, 288, device=cuda)
    before = cache._version, q._version, qa._version
    axiom_amd.latent_append(*_append_args(cuda), cache.view(2, 16, 288), q_rope=q, q_out=qa[..., 256:])
    assert cache._version > before[0] and qa._version > before[2] and q._version == before[1]
    axiom_amd.latent_append(*_append_args(cuda), cache, q_rope=q, q_out=q)
    assert q._version > before[1]


def test_a_saved_cache_is_noticed(cuda):
    cache = torch.ones(2, 16, 288, device=cuda)
    x = torch.ones(288, device=cuda, requires_grad=True)
    y = (x * cache).sum()                     # keeps the cache for its backward
    axiom_amd.latent_append(*_append_args(cuda), cache)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_given_outputs(cuda):
    q, kv, kr, _ = attn_inputs(1, 20, 20, 2, 64, 32, "fp32", cuda)
    out, lse = torch.empty(1, 20, 2, 64, device=cuda), torch.empty(1, 2, 20, device=cuda)
    axiom_amd.latent_attn_fwd(q, kv, kr, out=out, lse=lse)
    assert out._version == 1 and lse._version == 1
    qa, cache = torch.randn(1, 1, 2, 288, device=cuda), torch.randn(2, 16, 288, device=cuda)
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda), torch.tensor([20], dtype=torch.int32, device=cuda)
    out, lse = torch.empty(1, 1, 2, 256, device=cuda), torch.empty(1, 1, 2, device=cuda)
    axiom_amd.latent_decode(qa, cache, table, lens, 0.1, out=out, lse=lse)
    assert out._version == 1 and lse._version == 1 and cache._version == 0 and qa._version == 0


def test_inference_tensors(cuda):
    """A cache made under inference mode has no version; it is written all the same, inside the mode and outside."""
    args = _append_args(cuda)
    with torch.inference_mode():
        cache = torch.zeros(2, 16, 288, device=cuda)
        axiom_amd.latent_append(*args, cache)
    first = cache.clone()
    cache.data.zero_()
    axiom_amd.latent_append(*args, cache)
    assert torch.equal(cache, first) and (first != 0).any()
