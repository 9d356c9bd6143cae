"""GPU: latent attention of a tree over the paged cache, and the cache after a path, against float64."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import DT, bar, check, check_lse
from oracle import tree as O
from tree_testutil import trees

pytestmark = pytest.mark.gpu


def case(lens, N, H, R, dr, page, dtype, device, seed=0, extra=0, layers=None):
    """Scattered pages; what no sequence holds (page tails, spare pages) is NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    B = len(lens)
    per = max(1, max(-(-n // page) for n in lens)) + extra
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    order = torch.randperm(pages, device=device, generator=g).int()
    table = torch.full((B, per), -7, dtype=torch.int32, device=device)
    cache = torch.full((layers or 1, pages, page, R + dr), float("nan"), dtype=DT[dtype], device=device)
    at = 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = order[at:at + used[b]]
        for i in range(used[b]):
            m = min(page, n - i * page)
            cache[:, int(order[at + i]), :m] = torch.randn(layers or 1, m, R + dr, device=device, generator=g).to(DT[dtype])
        at += used[b]
    q = (torch.randn(B, N, H, R + dr, device=device, generator=g) * 0.8).to(DT[dtype])
    return q, cache if layers else cache[0], table, torch.tensor(lens, dtype=torch.int32, device=device)


def rows_of(cache, table, lens):
    """Every sequence's rows in order."""
    page = cache.shape[-2]
    out = []
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n, device=cache.device)
        out.append(cache[..., table[b].long()[t // page], t % page, :])
    return out


def compare(c, p, R, dtype, scale=0.07):
    q, cache, table, lens = c
    o, lse = axiom_amd.latent_tree_decode(q, cache, table, lens, p, scale=scale)
    o_ref, lse_ref = O.decode(q, cache, table, lens, p, R, scale)
    check("o", o, o_ref, bar(dtype), (0, 1, 2))
    check_lse("lse", lse, lse_ref)
    return o, lse


@pytest.mark.parametrize("N,H", [(1, 4), (1, 16), (2, 8), (5, 3), (8, 16), (16, 4), (17, 7), (33, 2), (64, 1), (64, 4)])
@pytest.mark.parametrize("R,dr,dtype", [(512, 64, "bf16"), (256, 32, "fp32"), (512, 64, "fp16"), (256, 64, "bf16"), (512, 32, "fp32")])
def test_shapes(cuda, N, H, R, dr, dtype):
    kinds = ["random", "chain", "broken", "star", "deep"]
    lens = [N + 150, N, N + 1, N + 700, N + 31]
    p = trees(kinds, N, cuda, seed=N + H)
    compare(case(lens, N, H, R, dr, 16, dtype, cuda, seed=N), p, R, dtype)


@pytest.mark.parametrize("page", [1, 4, 8, 16, 32, 64, 256])
@pytest.mark.parametrize("H,dtype", [(2, "bf16"), (8, "bf16"), (2, "fp32")])
def test_pages(cuda, page, H, dtype):
    lens = [300, 7, 9, 64, 129]
    p = trees(["random", "chain", "broken", "deep", "star"], 7, cuda, seed=page)
    compare(case(lens, 7, H, 512, 64, page, dtype, cuda, seed=page, extra=1), p, 512, dtype)


@pytest.mark.parametrize("offset", range(0, 36, 5))
def test_places_across_tiles(cuda, offset):
    """The first place at every kind of position in a tile of 16 or 32 rows."""
    for H, dtype in ((1, "bf16"), (4, "bf16"), (2, "fp32")):
        p = trees(["random", "broken"], 14, cuda, seed=offset)
        compare(case([200 + offset + 14, offset + 14], 14, H, 256, 32, 16, dtype, cuda, seed=offset), p, 256, dtype)


def test_short_and_empty_sequences(cuda):
    """Fewer rows than places: those before the first row see nothing and are not seen."""
    for H, dtype in ((2, "bf16"), (8, "bf16"), (3, "fp32")):
        lens = [0, 1, 5, 9, 10, 11, 40]
        p = trees(["chain", "star", "random", "chain", "random", "deep", "none"], 10, cuda, seed=3)
        o, lse = compare(case(lens, 10, H, 512, 64, 16, dtype, cuda, seed=4), p, 512, dtype)
        assert (o[0] == 0).all() and torch.isneginf(lse[0]).all() and (o[6] == 0).all() and torch.isneginf(lse[6]).all()


def test_long_and_uneven(cuda):
    lens = [20000, 70, 3000, 12, 9000, 800]
    p = trees(["random", "deep", "chain", "broken", "random", "star"], 12, cuda, seed=5)
    for H, dtype in ((16, "bf16"), (1, "fp16"), (2, "fp32")):
        compare(case(lens, 12, H, 512, 64, 64, dtype, cuda, seed=6), p, 512, dtype)


@pytest.mark.parametrize("N,H", [(25, 16), (64, 16), (40, 48)])
def test_many_row_groups(cuda, N, H):
    """7, 16 and 30 groups of 64 rows, over long and short sequences."""
    p = trees(["random", "chain"], N, cuda, seed=N)
    compare(case([1500, N + 3], N, H, 512, 64, 32, "bf16", cuda, seed=N), p, 512, "bf16")


def test_a_chain_is_latent_decode(cuda):
    for N, H, dtype in ((3, 4, "bf16"), (6, 8, "fp16"), (5, 3, "fp32")):
        q, cache, table, lens = case([400, 33, N, 2000], N, H, 512, 64, 32, dtype, cuda, seed=7)
        o, lse = axiom_amd.latent_tree_decode(q, cache, table, lens, trees(["chain"] * 4, N, cuda), scale=0.05)
        o2, lse2 = axiom_amd.latent_decode(q, cache, table, lens, scale=0.05)
        # both sides round their probabilities, and the result, on their own
        check("o", o, o2.cpu().double(), 2 * bar(dtype), (0, 1, 2))
        check_lse("lse", lse, lse2.cpu().double())


def test_places_without_a_draft_reach_nothing(cuda):
    for H, dtype in ((1, "bf16"), (8, "bf16"), (2, "fp32")):
        N = 13
        q, cache, table, lens = case([500, 60, N, N, 200], N, H, 512, 64, 16, dtype, cuda, seed=8)
        p = trees(["broken", "random", "broken", "none", "none"], N, cuda, seed=9)
        p[1, 9:] = -2
        p[2, 0] = -2
        o, lse = axiom_amd.latent_tree_decode(q, cache, table, lens, p, scale=0.07)
        for b, row in enumerate(O.paths(p)):
            for i, path in enumerate(row):
                if not path:
                    q[b, i] = float("nan")
                    t = int(lens[b]) - N + i
                    cache[int(table[b, t // 16]), t % 16] = float("inf")
        o2, lse2 = axiom_amd.latent_tree_decode(q, cache, table, lens, p, scale=0.07)
        assert torch.equal(o, o2) and torch.equal(lse, lse2) and torch.isfinite(o).all()


def test_lengths_and_pages_out_of_range_are_clamped(cuda):
    q, cache, table, lens = case([40, 40], 4, 2, 512, 64, 16, "bf16", cuda, seed=10)
    cache.nan_to_num_(0.0)
    p = trees(["random", "chain"], 4, cuda)
    lens[0], table[1, 1] = 10 ** 6, 10 ** 6
    compare((q, cache, table, lens), p, 512, "bf16")
    lens[:] = -3
    o, lse = axiom_amd.latent_tree_decode(q, cache, table, lens, p, scale=0.1)
    assert (o == 0).all() and torch.isneginf(lse).all()


def test_given_outputs_and_workspace(cuda):
    q, cache, table, lens = case([300, 77], 6, 8, 512, 64, 32, "bf16", cuda, seed=11)
    p = trees(["random", "deep"], 6, cuda)
    want = axiom_amd.latent_tree_decode(q, cache, table, lens, p, 0.1)
    from axiom_amd.tree import latent_tree_decode_workspace_bytes
    ws = torch.full((latent_tree_decode_workspace_bytes(2, 6, 8, 512, 64, 32, table.shape[1]),), 255, dtype=torch.uint8, device=cuda)
    out, lse = torch.full_like(want[0], float("nan")), torch.full_like(want[1], float("nan"))
    got = axiom_amd.latent_tree_decode(q, cache, table, lens, p, 0.1, out=out, lse=lse, workspace=ws)
    assert got[0].data_ptr() == out.data_ptr() and torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("N", [1, 2, 9, 33, 64])
@pytest.mark.parametrize("R,dr,dtype", [(512, 64, "bf16"), (256, 32, "fp32"), (512, 64, "fp32"), (256, 32, "fp16")])
@pytest.mark.parametrize("layers", [None, 3])
def test_commit(cuda, N, R, dr, dtype, layers):
    kinds = ["random", "chain", "star", "deep", "broken", "chain", "random", "deep"]
    lens = [N + 100, N, N + 7, N + 300, N + 15, N + 1, N + 64, N - 1]
    p = trees(kinds, N, cuda, seed=N)
    last = torch.tensor([N - 1, N // 2, N - 1, N - 1, N - 1, -1, N + 5, N - 1], dtype=torch.int32, device=cuda)
    _, cache, table, lens = case(lens, N, 1, R, dr, 16, dtype, cuda, seed=N, layers=layers)
    before, old = cache.clone(), rows_of(cache, table, lens)
    version = cache._version
    new = axiom_amd.latent_tree_commit(cache, table, lens, p, last)
    assert cache._version > version and new.dtype == torch.int32
    want = before.clone()
    for b, i in enumerate(last.tolist()):
        n = int(lens[b])
        path = O.paths(p)[b][i] if 0 <= i < N and n >= N else []
        assert int(new[b]) == (n - N + len(path) if n >= N else n)
        for to, j in enumerate(path):
            t = n - N + to
            want[..., int(table[b, t // 16]), t % 16, :] = old[b][..., n - N + j, :]
    assert torch.equal(cache.nan_to_num(7.0), want.nan_to_num(7.0))


def test_commit_out_and_clamps(cuda):
    _, cache, table, lens = case([50, 60], 8, 1, 512, 64, 16, "bf16", cuda, seed=13)
    p, last = trees(["deep", "random"], 8, cuda), torch.tensor([7, 6], dtype=torch.int32, device=cuda)
    other = cache.clone()
    want = axiom_amd.latent_tree_commit(other, table, lens, p, last)
    out = torch.zeros(2, dtype=torch.int32, device=cuda)
    got = axiom_amd.latent_tree_commit(cache, table, lens, p, last, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and torch.equal(cache.nan_to_num(), other.nan_to_num())
    lens[:] = 10 ** 6                       # past the table: taken as full
    table[:] = 10 ** 6
    axiom_amd.latent_tree_commit(cache, table, lens, p, last)
