"""GPU: verification of drafted trees against float64; whole numbers, so equal."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from oracle import tree as O
from tree_testutil import DT, trees

pytestmark = pytest.mark.gpu


def case(kinds, N, V, dtype, device, seed=0, noise=0.7):
    """target, draft rows (a parent's children share theirs), tokens drawn from them, uniforms."""
    g = torch.Generator(device=device).manual_seed(seed)
    B = len(kinds)
    p = trees(kinds, N, device, seed=seed)
    logits = 2 * torch.randn(B, N + 1, V, device=device, generator=g)
    target = torch.softmax(logits, -1).to(DT[dtype])
    near = torch.softmax(logits + noise * torch.randn(B, N + 1, V, device=device, generator=g), -1)
    at = (p.long() + 1).clamp(0, N)
    draft = near.gather(1, at[..., None].expand(B, N, V)).to(DT[dtype])
    tokens = torch.multinomial(draft.float().view(B * N, V), 1, generator=g).view(B, N)
    return target, tokens, p, torch.rand(B, N + 1, device=device, generator=g), draft


def same(got, want):
    for n, x, y in zip(("last", "next", "accepted"), got, want):
        assert x.tolist() == y, n
    assert [x.dtype for x in got] == [torch.int32, torch.int64, torch.int32]


KINDS = ["random", "chain", "star", "deep", "broken", "none", "random", "star"]


@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 65, 1000, 4099, 8200, 30011])
@pytest.mark.parametrize("N,dtype", [(1, "fp32"), (5, "bf16"), (12, "fp32"), (9, "fp16")])
def test_sampling(cuda, V, N, dtype):
    target, tokens, p, u, draft = case(KINDS, N, V, dtype, cuda, seed=V + N)
    same(axiom_amd.tree_verify(target, tokens, p, u, draft), O.verify(target, tokens, p, u, draft))
    same(axiom_amd.tree_verify(target, tokens, p, u), O.verify(target, tokens, p, u))
    same(axiom_amd.tree_verify(target, tokens, p), O.verify(target, tokens, p))


@pytest.mark.parametrize("B", [1, 3, 40, 300])
def test_batches(cuda, B):
    """From many slices a row to one, over rows that begin at odd places."""
    target, tokens, p, u, draft = case([KINDS[b % 8] for b in range(B)], 6, 20001, "bf16", cuda, seed=B, noise=2.0)
    same(axiom_amd.tree_verify(target, tokens, p, u, draft), O.verify(target, tokens, p, u, draft))
    same(axiom_amd.tree_verify(target, tokens, p), O.verify(target, tokens, p))


def test_all_places(cuda):
    target, tokens, p, u, draft = case(["chain", "star", "random", "deep"], 64, 501, "fp32", cuda, seed=1, noise=3.0)
    u[1, :64] = 0.999                       # the star's children are all asked
    same(axiom_amd.tree_verify(target, tokens, p, u, draft), O.verify(target, tokens, p, u, draft))
    same(axiom_amd.tree_verify(target, tokens, p, u), O.verify(target, tokens, p, u))


def test_uniforms_at_their_ends(cuda):
    target, tokens, p, u, draft = case(KINDS, 6, 3001, "fp32", cuda, seed=2)
    for x in (0.0, 1 - 2.0 ** -24):
        v = torch.full_like(u, x)
        same(axiom_amd.tree_verify(target, tokens, p, v, draft), O.verify(target, tokens, p, v, draft))
    v = torch.ones_like(u)                  # not below 1: the last entry that has a weight
    _, word, _ = axiom_amd.tree_verify(target, tokens, p, v)
    assert (word < 3001).all() and (word >= 0).all()


def test_the_same_distribution_is_always_accepted(cuda):
    """q = p: every first child is accepted; a point's remainder never gives the point."""
    target, tokens, p, u, _ = case(["chain"] * 32, 4, 900, "fp32", cuda, seed=3)
    draft = target[:, :4].contiguous()
    last, _, count = axiom_amd.tree_verify(target, tokens, p, u, draft)
    held = target[:, :4].gather(2, tokens[..., None])[..., 0] > 0
    assert ((last == 3) & (count == 4))[held.all(1)].all()
    v = torch.full_like(u, 0.9999)
    v[:, 4] = u[:, 4]
    last, word, _ = axiom_amd.tree_verify(target, tokens, p, v)
    assert (last == -1).all() and (word != tokens[:, 0]).all()


def test_distribution(cuda):
    """Accepted or not, the first token is distributed as the target's draws: chi-square of 40000 draws."""
    B, V = 40000, 12
    g = torch.Generator(device=cuda).manual_seed(4)
    prob = torch.softmax(1.5 * torch.randn(V, device=cuda, generator=g), 0)
    q = torch.softmax(1.5 * torch.randn(V, device=cuda, generator=g), 0)
    target = prob.expand(B, 4, V)
    for draft in (q.expand(B, 3, V), None):
        tokens = (torch.multinomial(q, B * 3, True, generator=g).view(B, 3) if draft is not None
                  else torch.tensor([3, 7, 1], device=cuda).expand(B, 3).contiguous())
        p = trees(["star"], 3, cuda).expand(B, 3).contiguous()
        u = torch.rand(B, 4, device=cuda, generator=g)
        last, word, _ = axiom_amd.tree_verify(target, tokens, p, u, draft)
        first = torch.where(last >= 0, tokens.gather(1, last.long().clamp(min=0)[:, None])[:, 0], word)
        seen = torch.bincount(first, minlength=V).double()
        expected = B * prob.double()
        chi = ((seen - expected) ** 2 / expected).sum().item()
        assert chi < 45, chi                # 11 degrees of freedom: 45 is passed once in 200000


def test_nothing_left_and_nothing_there(cuda):
    V = 700
    target = torch.zeros(3, 2, V, device=cuda)
    draft = torch.zeros(3, 1, V, device=cuda)
    target[0, 0, 5] = target[0, 0, 600] = 0.5            # p <= q everywhere: drawn from p itself
    draft[0, 0, 5], draft[0, 0, 600] = 0.75, 0.75
    target[2, 0, 9] = 1.0
    tokens, p = torch.tensor([[5], [3], [9]], device=cuda), torch.full((3, 1), -1, dtype=torch.int32, device=cuda)
    u = torch.tensor([[0.99, 0.7], [0.5, 0.5], [0.5, 0.5]], device=cuda)
    draft[2, 0, 9] = 1.0
    last, word, count = axiom_amd.tree_verify(target, tokens, p, u, draft)
    assert last.tolist() == [-1, -1, 0] and count.tolist() == [0, 0, 1] and word.tolist() == [600, -1, -1]


def test_tokens_outside_the_vocabulary(cuda):
    target, tokens, p, u, draft = case(["chain", "star", "random"], 5, 300, "fp32", cuda, seed=5)
    tokens[0, 1], tokens[1, 0], tokens[1, 2], tokens[2, 0] = 300, -1, 1 << 40, -(1 << 40)
    same(axiom_amd.tree_verify(target, tokens, p, u), O.verify(target, tokens, p, u))
    same(axiom_amd.tree_verify(target, tokens, p), O.verify(target, tokens, p))


@pytest.mark.parametrize("dtype", ["bf16", "fp32", "fp16"])
def test_greedy_ties_and_odd_values(cuda, dtype):
    V, inf, nan = 5000, float("inf"), float("nan")
    t = torch.full((7, 2, V), -3.0, device=cuda)
    t[0, 0, 4999] = t[0, 0, 77] = t[0, 0, 2048] = 1.0     # the lowest of several
    t[1, 0] = nan                                         # all NaN: 0
    t[2, 0] = -inf
    t[3, 0, :] = nan
    t[3, 0, 4321] = -inf                                  # the one that is a number
    t[4, 0, 3000], t[4, 0, 10] = 0.0, -0.0                # equal
    t[4, 0, 11] = nan
    t[5, 0, 4000] = t[5, 0, 4500] = inf
    t[6, 0] = -1.0
    t = t.to(DT[dtype])
    tokens, p = torch.full((7, 1), 77, device=cuda), torch.full((7, 1), -1, dtype=torch.int32, device=cuda)
    last, word, count = axiom_amd.tree_verify(t, tokens, p)
    assert last.tolist() == [0] + [-1] * 6 and count.tolist() == [1] + [0] * 6
    assert word.tolist() == [0, 0, 0, 4321, 10, 4000, 0]


def test_strides_and_shared_rows(cuda):
    target, tokens, p, u, draft = case(["random", "chain", "star"], 7, 1501, "bf16", cuda, seed=6)
    wide = torch.zeros(3, 10, 1600, dtype=torch.bfloat16, device=cuda)
    wide[:, 1:9, 3:1504] = target
    view = wide[:, 1:9, 3:1504]
    one = draft[:, :1].expand(3, 7, 1501)                 # every draft from one row
    same(axiom_amd.tree_verify(view, tokens, p, u, one), O.verify(target, tokens, p, u, one.contiguous()))
    same(axiom_amd.tree_verify(view, tokens, p), O.verify(target, tokens, p))


def test_rows_of_places_without_a_draft_are_not_read(cuda):
    target, tokens, p, u, draft = case(["random", "broken"], 9, 2000, "fp32", cuda, seed=7)
    p[0, 5:] = -2
    want = [axiom_amd.tree_verify(target, tokens, p, *a) for a in ((u, draft), (u,), ())]
    for b, row in enumerate(O.paths(p)):
        for i, path in enumerate(row):
            if not path:
                target[b, i + 1], draft[b, i], u[b, i], tokens[b, i] = float("nan"), float("nan"), float("nan"), -5
    for a, w in zip(((u, draft), (u,), ()), want):
        assert all(torch.equal(x, y) for x, y in zip(axiom_amd.tree_verify(target, tokens, p, *a), w))


def test_no_sequences(cuda):
    z = [torch.empty(0, 4, 10, device=cuda), torch.empty(0, 3, dtype=torch.int64, device=cuda), torch.empty(0, 3, dtype=torch.int32, device=cuda)]
    assert all(x.shape == (0,) for x in axiom_amd.tree_verify(*z))
