"""GPU: the tree calls where an offset passes 32 bits: what the far end of a large call gets is
what a small call of the same rows gets, bit for bit."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from test_gpu_tree_cache import case
from test_gpu_tree_verify import case as verify_case
from tree_testutil import step_inputs, trees

pytestmark = pytest.mark.gpu


@pytest.fixture
def room(cuda):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of free GPU memory")
    yield
    torch.cuda.empty_cache()


def far(cache, table, pages):
    """The cache's pages at the end of one of `pages` pages, and their table."""
    big = torch.empty(*cache.shape[:-3], pages, *cache.shape[-2:], dtype=cache.dtype, device=cache.device)
    n = cache.shape[-3]
    big[..., pages - n:, :, :] = cache
    return big, torch.where(table >= 0, table + (pages - n), table)


@pytest.mark.parametrize("dtype,H", [("bf16", 4), ("bf16", 1), ("fp32", 2)])
def test_attention_over_a_cache_past_4_gb(cuda, room, dtype, H):
    q, cache, table, lens = case([900, 40, 333], 17, H, 512, 64, 32, dtype, cuda, seed=1)
    p = trees(["random", "broken", "chain"], 17, cuda)
    want = axiom_amd.latent_tree_decode(q, cache, table, lens, p, 0.07)
    big, at = far(cache, table, (5 << 30) // (32 * 576 * cache.element_size()))
    got = axiom_amd.latent_tree_decode(q, big, at, lens, p, 0.07)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_commit_to_caches_past_4_gb(cuda, room):
    _, cache, table, lens = case([900, 70, 333], 64, 1, 512, 64, 32, "bf16", cuda, seed=2, layers=3)
    p, last = trees(["random", "deep", "star"], 64, cuda), torch.tensor([60, 63, 9], dtype=torch.int32, device=cuda)
    big, at = far(cache, table, (5 << 30) // (32 * 576 * 2))
    want = axiom_amd.latent_tree_commit(cache, table, lens, p, last)
    assert torch.equal(axiom_amd.latent_tree_commit(big, at, lens, p, last), want)
    assert torch.equal(big[:, -cache.shape[1]:].nan_to_num(), cache.nan_to_num())


def test_rows_past_2_31_elements(cuda, room):
    B, N, V = 40, 60, 1 << 20
    small = verify_case(["random", "deep"], N, 1 << 15, "bf16", cuda, seed=3, noise=2.0)
    target = torch.zeros(B, N + 1, V, dtype=torch.bfloat16, device=cuda)
    draft = torch.zeros(B, N, V, dtype=torch.bfloat16, device=cuda)
    target[-2:, :, -(1 << 15):] = small[0]
    draft[-2:, :, -(1 << 15):] = small[4]
    tokens = torch.zeros(B, N, dtype=torch.int64, device=cuda)
    tokens[-2:] = small[1] + V - (1 << 15)
    p, u = small[2].repeat(B // 2, 1), small[3].repeat(B // 2, 1)
    for with_draft in (True, False):
        last, word, count = axiom_amd.tree_verify(target, tokens, p, u, draft if with_draft else None)
        want = axiom_amd.tree_verify(*small) if with_draft else axiom_amd.tree_verify(*small[:4])
        assert torch.equal(last[-2:], want[0]) and torch.equal(word[-2:], want[1] + V - (1 << 15)) and torch.equal(count[-2:], want[2])
        assert (last[:-2] == -1).all() and (word[:-2] == -1).all()
    last, word, _ = axiom_amd.tree_verify(target, tokens, p)
    want = axiom_amd.tree_verify(*small[:3])
    assert torch.equal(last[-2:], want[0]) and torch.equal(word[-2:], want[1] + V - (1 << 15)) and (word[:-2] == 0).all()


def test_states_past_2_32_elements(cuda, room):
    B, N, H, d = 4100, 64, 64, 128
    small = step_inputs(2, N, H, d, "bf16", cuda, seed=4)
    p2 = trees(["random", "chain"], N, cuda)
    o, u = axiom_amd.kda_tree_step(*(small[n] for n in ("q", "k", "v", "g", "beta")), p2, small["state"])
    x = {}
    for n, t in small.items():
        x[n] = torch.zeros(B, *t.shape[1:], dtype=t.dtype, device=cuda)
        x[n][-2:] = t
    p = torch.full((B, N), -2, dtype=torch.int32, device=cuda)
    p[-2:] = p2
    big_o, big_u = axiom_amd.kda_tree_step(*(x[n] for n in ("q", "k", "v", "g", "beta")), p, x["state"], out_dtype=torch.bfloat16)
    assert torch.equal(big_o[-2:], o.bfloat16()) and torch.equal(big_u[-2:], u)
    assert not big_u[1000].any()
    last2 = torch.tensor([50, 63], dtype=torch.int32, device=cuda)
    last = torch.full((B,), -1, dtype=torch.int32, device=cuda)
    last[-2:] = last2
    axiom_amd.kda_tree_commit(x["k"], x["g"], big_u, p, last, x["state"])
    want = axiom_amd.kda_tree_commit(small["k"], small["g"], u, p2, last2, small["state"])
    assert torch.equal(x["state"][-2:], want) and not x["state"][2000].any()
