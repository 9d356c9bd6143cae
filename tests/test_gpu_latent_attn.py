"""GPU: the expanded latent attention and its gradient against float64."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs, bar, check, check_lse, terms
from oracle import latent as O

pytestmark = pytest.mark.gpu

# lengths around the tiles (32, 64), the blocks (128) and one token
SHAPES = [(1, 1, 1), (1, 1, 200), (2, 63, 63), (1, 64, 64), (1, 65, 190), (1, 127, 129), (2, 200, 200), (1, 300, 77)]


def _run(q, kv, kr, do, **kw):
    q, kv, kr = (x.detach().requires_grad_(True) for x in (q, kv, kr))
    o = axiom_amd.latent_attn(q, kv, kr, **kw)
    grads = torch.autograd.grad(o, (q, kv, kr), do)
    return o, grads


def _compare(q, kv, kr, do, dtype, causal=True, scale=None, cu=None, cu_k=None):
    cu_h = None if cu is None else cu.tolist()
    cuk_h = None if cu_k is None else cu_k.tolist()
    o_ref, lse_ref, *g_ref = O.attn(q, kv, kr, causal, scale, cu_h, cuk_h, do)
    kw = dict(cu_seqlens=cu, cu_seqlens_k=cu_k, causal=causal, scale=scale)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, **kw)
    check("o", o, o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)
    o2, grads = _run(q, kv, kr, do, **kw)
    assert torch.equal(o, o2)
    for name, got, ref, axes in zip(("dq", "dkv", "dk_rope"), grads, g_ref, ((0, 2), (0, 2), (0,))):
        assert got.dtype == q.dtype
        check(name, got, ref, bar(dtype, True), axes, 0.1 * terms(q, kv, kr, do))


@pytest.mark.parametrize("B,Tq,Tk", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(cuda, B, Tq, Tk, dtype, causal):
    _compare(*attn_inputs(B, Tq, Tk, 2, 128, 64, dtype, cuda, seed=Tq), dtype, causal)


@pytest.mark.parametrize("dn,dr", [(64, 32), (64, 64), (128, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_head_dims(cuda, dn, dr, dtype):
    _compare(*attn_inputs(2, 150, 170, 3, dn, dr, dtype, cuda, seed=dn + dr), dtype)


@pytest.mark.parametrize("H", [1, 5, 8, 16])
def test_heads_over_the_dies(cuda, H):
    """Head counts that do and do not divide over the eight dies; several blocks of queries."""
    _compare(*attn_inputs(1, 400, 400, H, 64, 32, "bf16", cuda, seed=H), "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_inputs(cuda, dtype):
    q, kv, kr, do = attn_inputs(2, 130, 140, 3, 128, 64, dtype, cuda, seed=9, views=True)
    assert not q.is_contiguous() and not kv.is_contiguous() and not kr.is_contiguous()
    _compare(q, kv, kr, do, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Tq,Tk,H", [(700, 1100, 2), (900, 500, 3), (1000, 1000, 8), (8400, 8400, 1)])
def test_uneven_causal_walks(cuda, dtype, Tq, Tk, H):
    """Few blocks with walks of different lengths, shared out in equal pieces; 8400 rows: more blocks than lanes."""
    _compare(*attn_inputs(1, Tq, Tk, H, 64, 32, dtype, cuda, seed=Tq + H), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_queries_without_keys(cuda, dtype):
    """Causal with more queries than keys: the first rows see none."""
    q, kv, kr, do = attn_inputs(1, 200, 30, 2, 128, 64, dtype, cuda, seed=4)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr)
    assert (o[:, :170] == 0).all() and torch.isneginf(lse[:, :, :170]).all()
    _compare(q, kv, kr, do, dtype)


def test_no_keys_and_no_queries(cuda):
    q, kv, kr, do = attn_inputs(1, 5, 0, 2, 64, 32, "bf16", cuda)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr)
    assert (o == 0).all() and torch.isneginf(lse).all()
    _, (dq, dkv, dkr) = _run(q, kv, kr, do)
    assert (dq == 0).all() and dkv.shape == kv.shape and dkr.shape == kr.shape
    q, kv, kr, do = attn_inputs(1, 0, 7, 2, 64, 32, "bf16", cuda)
    _, (dq, dkv, dkr) = _run(q, kv, kr, do)
    assert dq.shape == q.shape and (dkv == 0).all() and (dkr == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(cuda, dtype, causal):
    """Packed sequences of zero, one and many tokens equal the float64 runs of each."""
    cu = torch.tensor([0, 1, 1, 64, 193, 200, 330], dtype=torch.int32, device=cuda)
    _compare(*attn_inputs(1, 330, 330, 2, 128, 64, dtype, cuda, seed=6), dtype, causal, cu=cu)


def test_packed_other_key_lengths(cuda):
    cu = torch.tensor([0, 5, 5, 140, 150], dtype=torch.int32, device=cuda)
    cu_k = torch.tensor([0, 300, 310, 400, 403], dtype=torch.int32, device=cuda)
    _compare(*attn_inputs(1, 150, 403, 2, 64, 64, "bf16", cuda, seed=7), "bf16", True, cu=cu, cu_k=cu_k)


def test_packed_many_sequences(cuda):
    """More sequences than a wave looks at in one step."""
    lens = [(7 * i) % 11 for i in range(150)]
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    T = sum(lens)
    _compare(*attn_inputs(1, T, T, 1, 64, 32, "bf16", cuda, seed=8), "bf16", True, cu=cu)


def test_packed_equals_separate_bit_for_bit(cuda):
    q, kv, kr, do = attn_inputs(1, 300, 300, 2, 128, 64, "bf16", cuda, seed=11)
    cu = torch.tensor([0, 130, 300], dtype=torch.int32, device=cuda)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, cu_seqlens=cu)
    for a, e in ((0, 130), (130, 300)):
        o1, l1 = axiom_amd.latent_attn_fwd(q[:, a:e], kv[:, a:e], kr[:, a:e])
        assert torch.equal(o[:, a:e], o1) and torch.equal(lse[:, :, a:e], l1)


def test_packed_neighbour_not_finite(cuda):
    """A sequence of infinities and NaN leaves its neighbours' results as they were."""
    q, kv, kr, do = attn_inputs(1, 220, 220, 2, 128, 64, "bf16", cuda, seed=12)
    cu = torch.tensor([0, 70, 150, 220], dtype=torch.int32, device=cuda)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, cu_seqlens=cu)
    _, grads = _run(q, kv, kr, do, cu_seqlens=cu)
    q2, kv2, kr2, do2 = (x.clone() for x in (q, kv, kr, do))
    q2[:, 70:150], kv2[:, 70:150], kr2[:, 70:150], do2[:, 70:150] = float("nan"), float("inf"), float("nan"), float("nan")
    o2, lse2 = axiom_amd.latent_attn_fwd(q2, kv2, kr2, cu_seqlens=cu)
    _, grads2 = _run(q2, kv2, kr2, do2, cu_seqlens=cu)
    for a, e in ((0, 70), (150, 220)):
        assert torch.equal(o[:, a:e], o2[:, a:e]) and torch.equal(lse[:, :, a:e], lse2[:, :, a:e])
        for x, y in zip(grads, grads2):
            assert torch.equal(x[:, a:e], y[:, a:e])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_large_scores(cuda, dtype):
    """Scores of several hundred: the running maximum rises many times, softmax picks single keys."""
    q, kv, kr, do = attn_inputs(1, 140, 260, 2, 128, 64, dtype, cuda, seed=13)
    ramp = torch.linspace(0.1, 6.0, 260, device=cuda).to(kv.dtype)
    kv = torch.cat([kv[..., :128] * ramp[None, :, None, None], kv[..., 128:]], -1).contiguous()
    o_ref, lse_ref = O.attn(q * 4, kv, kr, False)
    o, lse = axiom_amd.latent_attn_fwd((q * 4).contiguous(), kv, kr, causal=False)
    # an exponent of magnitude 2^8 carries 2^8 units of the fp32 score: 2^8 2^-23 on top of the type's bar
    check("o", o, o_ref, bar(dtype) + 2.0 ** -13, (0, 2))
    err = (lse.cpu().double() - lse_ref).abs()
    assert (err <= 1e-5 * (1 + lse_ref.abs())).all(), err.max()


def test_small_gradients_in_fp16(cuda):
    """Cotangents near fp16's smallest values over long rows: p times them must not vanish."""
    q, kv, kr, do = attn_inputs(1, 1000, 1000, 1, 64, 32, "fp16", cuda, seed=14)
    do = (do.float() * 2.0 ** -9).half()
    _, _, *ref = O.attn(q, kv, kr, True, None, None, None, do)
    _, grads = _run(q, kv, kr, do)
    for name, got, r in zip(("dq", "dkv", "dk_rope"), grads, ref):
        # the results themselves round to fp16's absolute step of 2^-25 below 2^-14
        err = (got.cpu().double() - r).abs()
        assert (err.square().mean().sqrt() <= bar("fp16", True) * r.square().mean().sqrt() + 2.0 ** -25), name


def test_gradient_against_differences(cuda):
    """Directional derivatives of the float64 forward by central differences."""
    q, kv, kr, do = attn_inputs(1, 40, 50, 2, 64, 32, "fp32", cuda, seed=15)
    _, grads = _run(q, kv, kr, do)
    gen = torch.Generator().manual_seed(3)
    xs = [x.cpu().double() for x in (q, kv, kr)]
    for i, g in enumerate(grads):
        d = torch.randn(xs[i].shape, generator=gen, dtype=torch.float64)
        side = []
        for e in (1e-5, -1e-5):
            ys = list(xs)
            ys[i] = xs[i] + e * d
            side.append((O.attn(*ys)[0] * do.cpu().double()).sum().item())
        want = (side[0] - side[1]) / 2e-5
        got = (g.cpu().double() * d).sum().item()
        size = g.cpu().double().norm().item()   # the sum's own size: cancellation between its terms is not an error
        assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_same_bits_every_run(cuda):
    q, kv, kr, do = attn_inputs(2, 500, 500, 8, 128, 64, "bf16", cuda, seed=16)
    first = _run(q, kv, kr, do)
    for _ in range(3):
        again = _run(q, kv, kr, do)
        assert torch.equal(first[0], again[0]) and all(torch.equal(x, y) for x, y in zip(first[1], again[1]))


def test_other_stream_and_outputs_given(cuda):
    q, kv, kr, _ = attn_inputs(1, 100, 100, 2, 128, 64, "bf16", cuda, seed=17)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr)
    out, l2 = torch.full_like(o, 7.0), torch.full_like(lse, 7.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r = axiom_amd.latent_attn_fwd(q, kv, kr, out=out, lse=l2)
    torch.cuda.current_stream().wait_stream(s)
    assert r[0] is out and r[1] is l2 and torch.equal(out, o) and torch.equal(l2, lse)


def test_graph_replays(cuda):
    """Forward and backward captured once, replayed over new inputs."""
    q, kv, kr, do = attn_inputs(1, 190, 190, 2, 64, 32, "bf16", cuda, seed=18)
    ws = torch.empty(1 << 22, dtype=torch.uint8, device=cuda)

    def both():
        o, lse = axiom_amd.latent_attn_fwd(q, kv, kr)
        return o, *axiom_amd.latent_attn_bwd(q, kv, kr, o, lse, do, workspace=ws)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = both()
    for seed in (1, 2, 3):
        for x, y in zip((q, kv, kr, do), attn_inputs(1, 190, 190, 2, 64, 32, "bf16", cuda, seed=seed)):
            x.copy_(y)
        graph.replay()
        got = [x.clone() for x in res]
        torch.cuda.synchronize()
        for x, y in zip(got, both()):
            assert torch.equal(x, y)
