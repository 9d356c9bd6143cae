"""GPU: the KDA step over a tree where its decays are strong: row by row against float64.

Inputs are coherent (keys and queries near one direction, every channel of a head with the
same decay), so that no error of a decay averages out over the channels and no row is small
by cancellation.  Bar, per row.  A pair's share q_i (gamma_i / gamma_j) k_j errs by two
exponentials (2^-23 each), four roundings (2^-24 each), the parts that the products leave out
(2^-22 at most) and the logarithms between the two places, 64 roundings of 2^-25 ln 2 at most,
1e-7 rms: 4e-7 where every channel errs alike.  Its sum has some 24 roundings of 2^-24 in the
matrix unit, 3e-7 rms.  2^-19 = 1.9e-6 is four times the two together.
"""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from oracle import tree as O
from tree_testutil import DT, trees

pytestmark = pytest.mark.gpu
ROW = 2.0 ** -19
KINDS = ["chain", "deep", "random", "chain"]


def coherent(B, N, H, d, dtype, first, rest, seed):
    """Log-decays: ``first`` at the first place of each path, ``rest`` over the N others together."""
    gen = torch.Generator().manual_seed(seed)

    def near_one(*s):
        x = 1 + 0.3 * torch.randn(*s, generator=gen)
        return x / x.norm(dim=-1, keepdim=True)

    share = torch.rand(B, N, H, 1, generator=gen)
    share[:, 0] = 0
    g = -rest * share / share.sum(1, keepdim=True).clamp_min(1e-3)
    g[:, 0] -= first
    x = dict(q=near_one(B, N, H, d), k=near_one(B, N, H, d), v=torch.randn(B, N, H, d, generator=gen),
             g=g.expand(B, N, H, d).contiguous(), beta=0.02 + 0.1 * torch.rand(B, N, H, generator=gen))
    x = {n: t.to(DT[dtype]).cuda() for n, t in x.items()}
    x["state"] = 0.1 * torch.randn(B, H, d, d, generator=gen).cuda()
    return x


def term_sizes(x, parents, u):
    """What a row of o and of u sums: the read-out of the state and every ancestor's share."""
    q, k, v, g, beta, S = (x[n].cpu().double() for n in ("q", "k", "v", "g", "beta", "state"))
    o_size, u_size = torch.zeros(q.shape[:3]), torch.zeros(q.shape[:3])
    for b, row in enumerate(O.paths(parents)):
        for i, path in enumerate(row):
            if not path:
                continue
            logs = g[b, path].flip(0).cumsum(0).flip(0)                        # from each place on, itself included
            for left, size in ((q, o_size), (k, u_size)):
                size[b, i] = torch.einsum("hk,hkv->hv", logs[0].exp() * left[b, i], S[b]).norm(dim=-1)
                for n, j in enumerate(path):
                    decay = (logs[n] - g[b, j]).exp()
                    if j != i or left is q:
                        size[b, i] += (left[b, i] * decay * k[b, j]).sum(-1).abs() * u[b, j].norm(dim=-1)
            u_size[b, i] = beta[b, i] * (u_size[b, i] + v[b, i].norm(dim=-1))
    return o_size.double(), u_size.double()


def rows_right(x, parents, bar=ROW, of_terms=False):
    o, u = axiom_amd.kda_tree_step(*(x[n] for n in ("q", "k", "v", "g", "beta")), parents, x["state"])
    o_ref, u_ref, _ = O.step(*(x[n] for n in ("q", "k", "v", "g", "beta")), parents, x["state"])
    sizes = term_sizes(x, parents, u_ref) if of_terms else (o_ref.norm(dim=-1), u_ref.norm(dim=-1))
    for name, got, ref, size in (("o", o, o_ref, sizes[0]), ("u", u, u_ref, sizes[1])):
        err = (got.cpu().double() - ref).norm(dim=-1)
        worst = torch.where(size > 0, err / size.clamp_min(1e-300), err)
        assert torch.isfinite(worst).all()
        assert worst.max() <= bar, f"{name}: a row is off by {worst.max():.2e}, {bar:.2e} allowed"


def one_root(kind_rows):
    """Every path begins at place 0."""
    p = kind_rows.clone()
    p[:, 1:] = p[:, 1:].clamp_min(0)
    return p


@pytest.mark.parametrize("first,rest", [(50.0, 0.05), (45.0, 4.0), (30.0, 8.0), (0.0, 54.0), (20.0, 20.0)])
@pytest.mark.parametrize("N,d", [(8, 128), (9, 128), (16, 64), (17, 128), (32, 128), (33, 64), (64, 128)])
def test_a_row_errs_by_its_own_decay(cuda, N, d, first, rest):
    """However far a path has decayed before, a pair's decay is the one between its two places."""
    rows_right(coherent(len(KINDS), N, 2, d, "fp32", first, rest, seed=N), one_root(trees(KINDS, N, cuda, seed=N)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N", [12, 40])
def test_of_16_bit_inputs(cuda, N, dtype):
    rows_right(coherent(len(KINDS), N, 2, 128, dtype, 48.0, 3.0, seed=N), one_root(trees(KINDS, N, cuda, seed=N)))


@pytest.mark.parametrize("N", [12, 33, 64])
@pytest.mark.parametrize("down,up", [(20.0, 40.0), (40.0, 80.0), (60.0, 80.0)])
def test_growing_and_decaying_gates(cuda, N, down, up):
    """A later place grows by more than the first has decayed.  Past 2^80, which exp(80) = 2^115 is by itself,
    the pairs' decays are products of exp2(g log2 e), whose argument is off by 2^-18 there: 2.6e-6 more.

    The rows below the place that grows are small beside what they sum: the state there is far larger than
    any v, so o_i is q_i^T (I - beta k k^T) ... (I - beta k k^T) S, with k's and q near one direction, betas of
    0.07 on average and 31 of them in the longest chain: exp(-31 * 0.07 * 0.92) = 0.14 of S, out of terms
    of S and of the u_j, 1 + 31 * 0.07 = 3.2 times S together.  Their rounding is 2^-19 of the terms, and up to
    3.2 / 0.14 = 23 times that of the row: the terms are the measure."""
    x = coherent(len(KINDS), N, 2, 128, "fp32", down, 0.5, seed=N)
    x["g"][:, N // 2] += up
    rows_right(x, one_root(trees(KINDS, N, cuda, seed=N)), ROW if up <= 40 else ROW + 2.0 ** -18 * 0.6932, of_terms=True)


@pytest.mark.parametrize("strong", [2, 4, 5, 8])
def test_sums_that_pass_the_range_several_times(cuda, strong):
    """Gates of 2^-64: the whole numbers that a path's logarithms are held in wrap to 0 at every fourth."""
    x = coherent(len(KINDS), 24, 2, 128, "fp32", 0.0, 0.5, seed=strong)
    x["g"][:, 3:3 + strong] -= 64 * 0.6931471805599453
    rows_right(x, one_root(trees(KINDS, 24, cuda, seed=strong)))


SIZED = [(9, 128), (16, 64), (17, 128), (40, 64), (64, 128)]


@pytest.mark.parametrize("N,d", SIZED)
def test_large_keys_far_down_a_path(cuda, N, d):
    """A key of 2^58 where the path has decayed to 2^-78: k / gamma has no float, the pair's share has."""
    x = coherent(2, N, 2, d, "fp32", 54.0, 0.5, seed=N)
    p = one_root(trees(["chain", "star"], N, cuda))
    x["k"][0, -1] *= 2.0 ** 58                      # places that nothing continues
    x["k"][1, N // 2:] *= 2.0 ** 58
    rows_right(x, p)


@pytest.mark.parametrize("N,d", SIZED)
def test_small_queries_far_down_a_path(cuda, N, d):
    """gamma q below the least float: the read-out of what the path itself wrote is as exact as ever."""
    x = coherent(2, N, 2, d, "fp32", 50.0, 0.5, seed=N)
    x["q"][0] *= 2.0 ** -60
    x["q"][1, N // 2] *= 2.0 ** -70
    rows_right(x, one_root(trees(["chain", "deep"], N, cuda)))


@pytest.mark.parametrize("N,d", SIZED)
def test_small_keys_behind_growing_gates(cuda, N, d):
    """k / gamma below the least float, over a state of nothing."""
    x = coherent(2, N, 2, d, "fp32", -50.0, 0.5, seed=N)
    x["k"][0] *= 2.0 ** -60
    x["k"][1, N // 2:] *= 2.0 ** -70
    x["state"].zero_()
    rows_right(x, one_root(trees(["chain", "star"], N, cuda)))


def test_a_small_scale(cuda):
    x = coherent(2, 33, 2, 128, "fp32", 50.0, 0.5, seed=1)
    p = one_root(trees(["chain", "random"], 33, cuda))
    ins = [x[n] for n in ("q", "k", "v", "g", "beta")]
    o, u = axiom_amd.kda_tree_step(*ins, p, x["state"])
    small, same = axiom_amd.kda_tree_step(*ins, p, x["state"], scale=2.0 ** -60)
    want = O.step(*ins, p, x["state"])[0]
    err = (small.cpu().double() * 2.0 ** 60 - want).norm(dim=-1) / want.norm(dim=-1)
    assert err.max() <= ROW and ((u - same).norm(dim=-1) <= ROW * u.norm(dim=-1)).all()


@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -118])
@pytest.mark.parametrize("N,d", [(6, 128), (7, 64), (14, 128), (30, 64), (50, 128)])
def test_a_state_near_the_least_float(cuda, N, d, size):
    """Nothing but such a state is read out: no v."""
    x = coherent(4, N, 2, d, "fp32", 0.0, 0.5, seed=N)
    x["v"].zero_()
    x["state"] *= size
    rows_right(x, one_root(trees(KINDS, N, cuda, seed=N)), of_terms=True)
