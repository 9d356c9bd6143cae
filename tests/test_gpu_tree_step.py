"""GPU: the delta rule over a tree and the state after a path, against float64."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import check
from oracle import tree as O
from tree_testutil import step_inputs, trees

pytestmark = pytest.mark.gpu
BAR = 1e-5
NAMES = ("q", "k", "v", "g", "beta")


def run(d, parents, **kw):
    before = d["state"].clone()
    o, u = axiom_amd.kda_tree_step(*(d[n] for n in NAMES), parents, d["state"], **kw)
    assert torch.equal(d["state"], before)
    return o, u


def compare(d, parents, scale=1.0):
    o, u = run(d, parents, scale=scale)
    o_ref, u_ref, states = O.step(*(d[n] for n in NAMES), parents, d["state"], scale)
    check("o", o, o_ref, BAR, (0, 2))
    check("u", u, u_ref, BAR, (0, 2))
    return o, u, states


@pytest.mark.parametrize("N", [1, 2, 7, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64])
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp32"), (128, "fp32"), (64, "fp16")])
def test_sizes(cuda, N, d, dtype):
    kinds = ["random", "chain", "star", "deep", "broken", "none"]
    p = trees(kinds, N, cuda, seed=N)
    compare(step_inputs(len(kinds), N, 2, d, dtype, cuda, seed=N, decay=0.2), p, scale=0.5)


@pytest.mark.parametrize("N", [8, 9, 12])
@pytest.mark.parametrize("d,dtype", [(128, "fp32"), (64, "bf16")])
def test_sizes_where_products_replace_the_walk(cuda, N, d, dtype):
    p = trees(["random", "chain", "star", "broken"], N, cuda, seed=N)
    compare(step_inputs(4, N, 3, d, dtype, cuda, seed=N, decay=0.2), p, scale=2.0)


@pytest.mark.parametrize("N", [5, 14, 30, 50])
def test_states_of_any_size(cuda, N):
    """fp32 factors are split for the products: no size of a state's entry costs them precision."""
    x = step_inputs(3, N, 2, 128, "fp32", cuda, seed=N, decay=0.1)
    gen = torch.Generator(device=cuda).manual_seed(N)
    x["state"][0] *= 1e-20
    x["state"][1] *= 1e20
    x["state"][2] *= 10.0 ** (30 * torch.rand(2, 128, 1, device=cuda, generator=gen) - 15)
    compare(x, trees(["random", "chain", "deep"], N, cuda, seed=N))


@pytest.mark.parametrize("decay", [0.0, 1.0, 30.0, 150.0])
def test_decays(cuda, decay):
    """No decay at all, and decays under which a product of a few underflows."""
    p = trees(["chain", "random", "deep"], 40, cuda)
    compare(step_inputs(3, 40, 3, 128, "fp32", cuda, seed=3, decay=decay), p)


@pytest.mark.parametrize("decay", [60.0, 300.0, float("inf")])
@pytest.mark.parametrize("kind", ["star", "chain"])
@pytest.mark.parametrize("N,d", [(17, 128), (33, 64), (64, 128), (64, 64)])
def test_one_place_of_strong_decay(cuda, N, d, kind, decay):
    """A sequence a place: whichever wave holds it, no quotient overflows.  exp(60) = 2^87 is still
    carried by two factors: twice six additions of logarithms, each off by 2^-18 / sqrt(3) rms,
    are sqrt(12) 2^-18 / sqrt(3) ln 2 = 5.3e-6 of a pair's share, and the bar holds the rest."""
    x = step_inputs(N, N, 1, d, "fp32", cuda, seed=N, decay=0.02)
    for b in range(N):
        x["g"][b, b, :, 1::2] -= decay
    compare(x, trees([kind] * N, N, cuda))


def test_growing_gates(cuda):
    d = step_inputs(2, 12, 2, 64, "fp32", cuda, seed=4, decay=-0.1)     # g > 0
    compare(d, trees(["random", "chain"], 12, cuda))


def test_a_chain_is_the_recurrent_step(cuda):
    B, N, H, dim = 3, 20, 4, 128
    d = step_inputs(B, N, H, dim, "bf16", cuda, seed=5)
    p = trees(["chain"] * B, N, cuda)
    o, u = run(d, p, scale=0.7)
    S = d["state"].clone()
    for i in range(N):
        oi = axiom_amd.kda_recurrent_step(*(d[n][:, i].contiguous() for n in NAMES), S, scale=0.7)
        check(f"o{i}", o[:, i], oi.cpu().double(), BAR, (0,))
    got = axiom_amd.kda_tree_commit(d["k"], d["g"], u, p, torch.full((B,), N - 1, dtype=torch.int32, device=cuda), d["state"])
    assert got.data_ptr() == d["state"].data_ptr()
    check("state", got, S.cpu().double(), BAR, (0, 1))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_bf16_output(cuda, dtype):
    d = step_inputs(2, 19, 3, 128, dtype, cuda, seed=6)
    p = trees(["random", "chain"], 19, cuda)
    o, u = run(d, p)
    ob, ub = run(d, p, out_dtype=torch.bfloat16)
    assert torch.equal(ob, o.bfloat16()) and torch.equal(ub, u)


def test_given_outputs(cuda):
    d = step_inputs(2, 9, 2, 64, "bf16", cuda, seed=7)
    p = trees(["random", "deep"], 9, cuda)
    o, u = run(d, p)
    out, uu = torch.full_like(o, float("nan")), torch.full_like(u, float("nan"))
    versions = out._version, uu._version
    a, b = run(d, p, out=out, u=uu)
    assert a.data_ptr() == out.data_ptr() and b.data_ptr() == uu.data_ptr() and torch.equal(out, o) and torch.equal(uu, u)
    assert out._version > versions[0] and uu._version > versions[1]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_places_without_a_draft_reach_nothing(cuda, dtype):
    B, N = 3, 37
    d = step_inputs(B, N, 2, 128, dtype, cuda, seed=8)
    p = trees(["broken", "random", "none"], N, cuda, seed=2)
    p[1, 30:] = -2
    o, u = run(d, p)
    dead = torch.tensor([[not x for x in row] for row in O.paths(p)], device=cuda)
    for n in NAMES:
        d[n][dead] = float("nan") if n != "g" else float("inf")
    o2, u2 = run(d, p)
    assert torch.equal(o, o2) and torch.equal(u, u2)
    assert (o[dead] == 0).all() and (u[dead] == 0).all()


def test_the_same_bits_again_and_in_another_batch(cuda):
    d = step_inputs(5, 33, 4, 128, "bf16", cuda, seed=9)
    p = trees(["random", "chain", "deep", "star", "broken"], 33, cuda)
    o, u = run(d, p)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(run(d, p), (o, u)))
    one = {n: x[3:4].contiguous() for n, x in d.items()}
    a, b = run(one, p[3:4].contiguous())
    assert torch.equal(a, o[3:4]) and torch.equal(b, u[3:4])


def test_no_sequences(cuda):
    d = step_inputs(0, 4, 2, 64, "bf16", cuda)
    o, u = run(d, torch.empty(0, 4, dtype=torch.int32, device=cuda))
    assert o.shape == u.shape == (0, 4, 2, 64)


@pytest.mark.parametrize("N", [1, 5, 16, 17, 40, 64])
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp32"), (128, "fp16"), (64, "bf16")])
def test_commit(cuda, N, d, dtype):
    kinds = ["random", "chain", "star", "deep", "broken", "chain", "random"]
    x = step_inputs(len(kinds), N, 3, d, dtype, cuda, seed=N, decay=0.3)
    p = trees(kinds, N, cuda, seed=N)
    _, u, states = compare(x, p)
    last = torch.tensor([N - 1, N - 1, N // 2, N - 1, N - 1, -1, N], dtype=torch.int32, device=cuda)
    before = x["state"].clone()
    version = x["state"]._version
    axiom_amd.kda_tree_commit(x["k"], x["g"], u, p, last, x["state"])
    assert x["state"]._version > version
    ref = before.cpu().double()
    for b, i in enumerate(last.tolist()):
        if 0 <= i < N and i in states[b]:
            ref[b] = states[b][i]
        else:
            assert torch.equal(x["state"][b], before[b])
    check("state", x["state"], ref, BAR, (0, 1))


def test_commit_reads_the_path_alone(cuda):
    B, N = 2, 30
    x = step_inputs(B, N, 2, 128, "bf16", cuda, seed=11)
    p = trees(["random", "deep"], N, cuda)
    _, u = run(x, p)
    last = torch.tensor([N - 1, N - 2], dtype=torch.int32, device=cuda)
    want = axiom_amd.kda_tree_commit(x["k"], x["g"], u, p, last, x["state"].clone())
    off = torch.ones(B, N, dtype=torch.bool)
    for b, row in enumerate(O.paths(p)):
        off[b, row[int(last[b])]] = False
    for t in (x["k"], x["g"], u):
        t[off.to(cuda)] = float("nan")
    assert torch.equal(axiom_amd.kda_tree_commit(x["k"], x["g"], u, p, last, x["state"]), want)
