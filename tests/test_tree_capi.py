"""CPU: the tree calls' C ABI and refusals; the oracle against itself in another form.

Nothing here launches a kernel: every call only computes sizes or fails the
host's validation before anything is enqueued.
"""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from axiom_amd import _lib
from axiom_amd import tree as T
from oracle import kda_oracle, latent as OL, tree as O
from tree_testutil import step_inputs, trees

OK = 0x10000   # a non-null aligned address; no call here gets far enough to use it


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        from axiom_amd import build
        build.build()
    return _lib.lib()


def test_header_declares_the_binding():
    assert set(_lib.header_symbols(_lib.TREE_HEADER)) == set(_lib._TREE)


def _step(L, q=OK, k=OK, v=OK, g=OK, beta=OK, par=OK, S=OK, o=OK, u=OK, B=1, N=4, H=2, dk=128, dv=128, scale=1.0, dt=1, out=0):
    return L.kda_tree_step(None, q, k, v, g, beta, par, S, o, u, B, N, H, dk, dv, scale, dt, out)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -1) for n in ("q", "k", "v", "g", "beta", "par", "S", "o", "u")],
    *[({n: OK + 8}, -1) for n in ("q", "k", "v", "g", "S", "o", "u")],
    (dict(B=-1), -1), (dict(N=0), -1), (dict(N=-3), -1), (dict(H=0), -1), (dict(N=65), -2), (dict(dk=96, dv=96), -2),
    (dict(dk=64), -2), (dict(dk=256, dv=256), -2), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(dt=3), -1), (dict(dt=-1), -1), (dict(out=2), -1), (dict(B=1 << 20, H=1 << 10), -2)])
def test_step_refuses(L, kw, code):
    assert _step(L, **kw) == code
    assert _lib.last_error()


def _commit(L, k=OK, g=OK, u=OK, par=OK, last=OK, S=OK, B=1, N=4, H=2, dk=128, dv=128, dt=1):
    return L.kda_tree_commit(None, k, g, u, par, last, S, B, N, H, dk, dv, dt)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -1) for n in ("k", "g", "u", "par", "last", "S")], *[({n: OK + 8}, -1) for n in ("k", "g", "u", "S")],
    (dict(B=-1), -1), (dict(N=0), -1), (dict(H=0), -1), (dict(N=65), -2), (dict(dk=32, dv=32), -2), (dict(dv=64), -2), (dict(dt=3), -1)])
def test_commit_refuses(L, kw, code):
    assert _commit(L, **kw) == code
    assert _lib.last_error()


def _decode(L, q=OK, cache=OK, table=OK, lens=OK, par=OK, o=OK, lse=OK, B=1, N=4, H=2, R=512, dr=64, pages=9, page=16, per=4,
            scale=0.1, dt=1, ws=OK, bytes=1 << 40):
    return L.kda_latent_tree_decode(None, q, cache, table, lens, par, o, lse, B, N, H, R, dr, pages, page, per, scale, dt, ws, bytes)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -1) for n in ("q", "cache", "table", "lens", "par", "o", "lse")],
    *[({n: OK + 8}, -1) for n in ("q", "cache", "o", "ws")], (dict(ws=None), -3), (dict(bytes=64), -3),
    (dict(B=-1), -1), (dict(N=0), -1), (dict(N=65), -2), (dict(H=0), -1), (dict(R=384), -2), (dict(dr=16), -2), (dict(page=24), -1),
    (dict(page=0), -1), (dict(per=-1), -1), (dict(pages=-1), -1), (dict(pages=1 << 28), -2), (dict(B=70000), -2), (dict(scale=0.0), -1),
    (dict(scale=float("nan")), -1), (dict(dt=3), -1), (dict(H=1 << 20), -2)])
def test_decode_refuses(L, kw, code):
    assert _decode(L, **kw) == code
    assert _lib.last_error()


def _keep(L, cache=OK, table=OK, lens=OK, par=OK, last=OK, new=2 * OK, layers=1, B=1, N=4, R=512, dr=64, pages=9, page=16, per=4, dt=1):
    return L.kda_latent_tree_commit(None, cache, table, lens, par, last, new, layers, B, N, R, dr, pages, page, per, dt)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -1) for n in ("cache", "table", "lens", "par", "last", "new")], (dict(cache=OK + 8), -1), (dict(new=OK), -1),
    (dict(B=-1), -1), (dict(N=0), -1), (dict(N=65), -2), (dict(layers=0), -1), (dict(layers=70000), -2), (dict(R=100), -2),
    (dict(dr=8), -2), (dict(page=3), -1), (dict(per=-1), -1), (dict(pages=-1), -1), (dict(pages=1 << 28), -2), (dict(per=1 << 28), -2),
    (dict(dt=3), -1)])
def test_cache_commit_refuses(L, kw, code):
    assert _keep(L, **kw) == code
    assert _lib.last_error()


def _verify(L, t=OK, tb=500, tr=100, tok=OK, par=OK, u=OK, d=None, db=0, dr=0, last=OK, nxt=OK, acc=OK, B=1, N=4, V=100, dt=0, ws=OK,
            bytes=1 << 40):
    return L.kda_tree_verify(None, t, tb, tr, tok, par, u, d, db, dr, last, nxt, acc, B, N, V, dt, ws, bytes)


@pytest.mark.parametrize("kw,code", [
    *[({n: None}, -1) for n in ("t", "tok", "par", "last", "nxt", "acc")], (dict(u=None, d=OK), -1), (dict(tb=-1), -1), (dict(tr=-1), -1),
    (dict(db=-1), -1), (dict(dr=-4), -1), (dict(B=-1), -1), (dict(N=0), -1), (dict(N=65), -2), (dict(V=0), -1), (dict(V=2 ** 31 - 1), -2),
    (dict(B=1 << 21), -2), (dict(dt=3), -1), (dict(ws=None), -3), (dict(bytes=100), -3), (dict(ws=OK + 8), -1)])
def test_verify_refuses(L, kw, code):
    assert _verify(L, **kw) == code
    assert _lib.last_error()


@pytest.mark.parametrize("call,kw", [
    ("step", dict(o="q")), ("step", dict(u="q")), ("step", dict(u="S")), ("step", dict(o="u")), ("step", dict(o="beta")), ("step", dict(u="par")),
    ("commit", dict(S="u")), ("commit", dict(S="last")), ("commit", dict(S="k")), ("decode", dict(o="q")), ("decode", dict(lse="lens")),
    ("decode", dict(ws="cache")), ("decode", dict(ws="o")), ("decode", dict(o="par")), ("keep", dict(new="lens")), ("keep", dict(new="last")),
    ("keep", dict(new="par")), ("keep", dict(new="table")), ("keep", dict(new="cache")), ("verify", dict(nxt="tok")), ("verify", dict(last="par")),
    ("verify", dict(acc="last")), ("verify", dict(ws="t")), ("verify", dict(nxt="u")), ("verify", dict(acc="ws"))])
def test_overlaps_are_refused(L, call, kw):
    """What a call writes in the last bytes of another argument; every other one far from the rest."""
    names, sizes, f = {
        "step": (("q", "k", "v", "g", "beta", "par", "S", "o", "u"), dict(q=2048, beta=16, par=16, S=131072, u=4096), _step),
        "commit": (("k", "g", "u", "par", "last", "S"), dict(u=4096, last=4, k=2048), _commit),
        "decode": (("q", "cache", "table", "lens", "par", "o", "lse", "ws"), dict(q=9216, lens=4, cache=165888, o=8192, par=16), _decode),
        "keep": (("cache", "table", "lens", "par", "last", "new"), dict(lens=4, last=4, par=16, table=16, cache=165888), _keep),
        "verify": (("t", "tok", "par", "u", "last", "nxt", "acc", "ws"), dict(tok=32, par=16, last=4, t=2000, u=20, ws=784), _verify)}[call]
    at = {n: OK + (i << 24) for i, n in enumerate(names)}
    (n, other), = kw.items()
    big = n in ("o", "u", "S", "ws") and call != "verify"
    step = 16 if big or n == "ws" else 8 if n == "nxt" else 4
    for p in {at[other], at[other] + (sizes[other] - 1) // step * step}:
        assert f(L, **{**at, n: p}) == -1, hex(p)
        assert "overlap" in _lib.last_error()


def test_empty_calls_do_nothing(L):
    z = dict(B=0)
    assert _step(L, q=None, **z) == 0 and _commit(L, k=None, **z) == 0 and _decode(L, q=None, **z) == 0
    assert _keep(L, cache=None, **z) == 0 and _verify(L, t=None, ws=None, **z) == 0


@pytest.mark.parametrize("args", [(-1, 4, 8, 512, 64, 16, 4, 1), (1, 0, 8, 512, 64, 16, 4, 1), (1, 65, 8, 512, 64, 16, 4, 1),
                                  (1, 4, 0, 512, 64, 16, 4, 1), (1, 4, 8, 500, 64, 16, 4, 1), (1, 4, 8, 512, 60, 16, 4, 1),
                                  (1, 4, 8, 512, 64, 17, 4, 1), (1, 4, 8, 512, 64, 16, -4, 1), (1, 4, 8, 512, 64, 16, 4, 7)])
def test_decode_workspace_of_bad_sizes(L, args):
    assert L.kda_latent_tree_decode_workspace(*args) == 0


def _up(x):
    return -(-x // 256) * 256


@pytest.mark.parametrize("B,N,H,R,page,per,code", [(1, 8, 16, 512, 64, 8, 1), (32, 16, 16, 512, 64, 128, 1), (4, 25, 64, 512, 32, 1024, 2),
                                                   (3, 5, 8, 256, 16, 90, 0), (1, 64, 128, 512, 64, 400, 1), (2, 2, 4, 512, 64, 100, 1),
                                                   (2, 3, 5, 512, 16, 8, 2), (1, 64, 512, 512, 64, 400, 1)])
def test_decode_workspace(L, B, N, H, R, page, per, code):
    """Starts of the sequences on the line, and two parts a workgroup of every run where there are runs."""
    m = 16 if N * H <= 16 or code == 0 else 64
    groups = -(-N * H // m)
    kt, pad, cap = (16, 8, page * per) if m == 16 else (32, 4 if groups == 1 else 8, page * per)
    least = 2 if groups == 1 else 4
    runs = ((-(-cap // kt) + pad) * B + least - 1) // least
    if cap <= 128:
        slots = 0
    elif groups == 1:
        slots = 2 * min(256, runs) * m
    else:
        slots = 2 * min(max(256 // groups, 1), runs) * groups * m
    assert L.kda_latent_tree_decode_workspace(B, N, H, R, 64, page, per, code) == _up(4 * (B + 1)) + _up(slots * 8) + _up(slots * R * 4)
    assert T.latent_tree_decode_workspace_bytes(B, N, H, R, 64, page, per, {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}[code]) \
        == L.kda_latent_tree_decode_workspace(B, N, H, R, 64, page, per, code)


def test_verify_workspace(L):
    assert [L.kda_tree_verify_workspace(*a) for a in ((-1, 4, 9), (1, 0, 9), (1, 65, 9), (1, 4, 0))] == [0] * 4
    for B, N, V in ((1, 1, 1), (1, 64, 10 ** 6), (64, 16, 128000), (300, 3, 50021), (0, 4, 100)):
        draw, rows = max(1, min(64, 256 // max(B, 1), V // 4096)), B * (N + 1)
        greedy = max(1, min(64, 1024 // max(rows, 1), V // 2048))
        assert L.kda_tree_verify_workspace(B, N, V) == max(B * (528 + 256 * draw), 8 * rows * greedy, 16)


# ---------------------------------------------------------------------------------------------- the Python calls

def _args(B=2, N=5, H=2, d=64):
    x = step_inputs(B, N, H, d, "bf16", "cpu")
    return [x[n] for n in ("q", "k", "v", "g", "beta")] + [trees(["chain", "star"][:B], N, "cpu"), x["state"]]


def bad(args, i, t):
    return args[:i] + [t] + args[i + 1:]


@pytest.mark.parametrize("i,change", [(0, lambda t: t[0]), (1, lambda t: t[:, 1:]), (2, lambda t: t[:, :, :1]), (3, lambda t: t[..., 1:]),
                                      (4, lambda t: t[..., None]), (0, lambda t: t.half()), (1, lambda t: t.double()), (4, lambda t: t.float()),
                                      (5, lambda t: t.long()), (5, lambda t: t[:, 1:]), (5, lambda t: t[:1]), (6, lambda t: t.bfloat16()),
                                      (6, lambda t: t[:1]), (6, lambda t: t.transpose(2, 3)), (0, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)),
                                      (5, lambda t: t.t().contiguous().t())])
def test_step_checks(i, change):
    a = _args()
    with pytest.raises(ValueError):
        axiom_amd.kda_tree_step(*bad(a, i, change(a[i])))


def test_cpu_tensors_and_types():
    a = _args()
    with pytest.raises(RuntimeError, match="only on the GPU"):
        axiom_amd.kda_tree_step(*a)
    with pytest.raises(ValueError, match="out_dtype"):
        axiom_amd.kda_tree_step(*a, out_dtype=torch.float16)
    big = [t.repeat_interleave(13, 1) if t.dim() > 2 and t is not a[6] else t for t in a]
    with pytest.raises(ValueError, match="64 places"):
        axiom_amd.kda_tree_step(*big[:5], torch.zeros(2, 65, dtype=torch.int32), a[6])


def test_commit_checks():
    q, k, v, g, beta, p, S = _args()
    u, last = torch.zeros(2, 5, 2, 64), torch.zeros(2, dtype=torch.int32)
    good = [k, g, u, p, last, S]
    with pytest.raises(RuntimeError, match="only on the GPU"):
        axiom_amd.kda_tree_commit(*good)
    for i, t in ((0, k[0]), (1, g.half()), (1, g[:, 1:]), (2, u.bfloat16()), (2, u[:, :4]), (3, p.long()), (4, last.long()), (4, last[:1]),
                 (5, S.half()), (5, S[:, :1])):
        with pytest.raises(ValueError):
            axiom_amd.kda_tree_commit(*bad(good, i, t))


def test_cache_checks():
    B, N, H, W = 2, 5, 4, 576
    q, cache = torch.zeros(B, N, H, W), torch.zeros(7, 16, W)
    table, lens, p = torch.zeros(B, 3, dtype=torch.int32), torch.full((B,), 20, dtype=torch.int32), trees(["chain", "star"], N, "cpu")
    last = torch.zeros(B, dtype=torch.int32)
    good = [q, cache, table, lens, p]
    with pytest.raises(RuntimeError, match="only on the GPU"):
        axiom_amd.latent_tree_decode(*good, 0.1)
    for i, t in ((0, q[0]), (0, q.half()), (0, q[..., 1:]), (1, cache[0]), (1, cache[None]), (1, cache[:, ::2]), (2, table.long()),
                 (2, table[:1]), (3, lens.long()), (3, lens[:1]), (4, p.long()), (4, p[:, :3])):
        with pytest.raises(ValueError):
            axiom_amd.latent_tree_decode(*bad(good, i, t), 0.1)
    good = [cache, table, lens, p, last]
    with pytest.raises(RuntimeError, match="only on the GPU"):
        axiom_amd.latent_tree_commit(*good)
    for i, t in ((0, cache[0]), (0, cache[None, None]), (0, cache.double()), (0, cache[None][:0]), (1, table[0]), (2, lens.long()), (3, p[0]),
                 (4, last.long())):
        with pytest.raises(ValueError):
            axiom_amd.latent_tree_commit(*bad(good, i, t))


def test_verify_checks():
    B, N, V = 2, 3, 50
    t, d = torch.zeros(B, N + 1, V), torch.zeros(B, N, V)
    tok, p, u = torch.zeros(B, N, dtype=torch.int64), trees(["chain", "star"], N, "cpu"), torch.zeros(B, N + 1)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        axiom_amd.tree_verify(t, tok, p, u, d)
    for a in ((t[0], tok, p, u, d), (t.double(), tok, p, u, d), (t[:, :1], tok, p, u, d), (t[..., :0], tok, p, u, d), (t[..., ::2], tok, p, u, None),
              (t, tok.int(), p, u, d), (t, tok[:, :2], p, u, d), (t, tok, p.long(), u, d), (t, tok, p, u[:, :3], d), (t, tok, p, u.double(), d),
              (t, tok, p, None, d), (t, tok, p, u, d.half()), (t, tok, p, u, d[:, :2]), (t, tok, p, u, d[..., :49])):
        with pytest.raises(ValueError):
            axiom_amd.tree_verify(*a)


# ---------------------------------------------------------------------------------------------- the oracle

def test_oracle_chain_is_the_recurrent_step():
    x = step_inputs(2, 6, 3, 64, "fp32", "cpu", seed=1)
    o, u, states = O.step(*(x[n] for n in ("q", "k", "v", "g", "beta")), trees(["chain", "chain"], 6, "cpu"), x["state"])
    S = x["state"].double().numpy()
    for i in range(6):
        ref, S = kda_oracle.decode_step(*(x[n][:, i].double().numpy() for n in ("q", "k", "v", "g", "beta")), S)
        assert abs(o[:, i].numpy() - ref).max() < 1e-12
    assert max(abs(states[b][5].numpy() - S[b]).max() for b in range(2)) < 1e-12


def test_oracle_chain_is_latent_decode():
    g = torch.Generator().manual_seed(2)
    q, cache = torch.randn(2, 4, 3, 288, generator=g), torch.randn(9, 8, 288, generator=g)
    table, lens = torch.randperm(8, generator=g).view(2, 4).int(), torch.tensor([30, 3])
    o, lse = O.decode(q, cache, table, lens, trees(["chain", "chain"], 4, "cpu"), 256, 0.1)
    o2, lse2 = OL.decode(q, cache, table, lens, 256, 0.1)
    assert torch.allclose(o, o2, atol=1e-12) and torch.equal(torch.isneginf(lse), torch.isneginf(lse2))
    assert torch.allclose(lse.nan_to_num(neginf=0), lse2.nan_to_num(neginf=0), atol=1e-12)


def test_oracle_paths():
    assert O.paths([[-1, 0, -2, 2, 1, 5, -1, 7, 2**31 - 1]]) == [[[0], [0, 1], [], [], [0, 1, 4], [], [6], [], []]]
