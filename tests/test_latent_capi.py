"""CPU: the latent attention's C ABI and refusals; the oracle against plain softmax.

Nothing here launches a kernel: every call only computes sizes or fails the
host's validation before anything is enqueued.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

import axiom_amd
from axiom_amd import _lib
from axiom_amd import latent as lat
from oracle import latent as O

OK = 0x10000   # a non-null aligned address; no call here gets far enough to use it


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        from axiom_amd import build
        build.build()
    return _lib.lib()


def test_header_declares_the_binding():
    assert set(_lib.header_symbols(_lib.LATENT_HEADER)) == set(_lib._LATENT)


def _st(*s):
    return (ctypes.c_int64 * 8)(*s)


DENSE = (192 * 100 * 2, 192 * 2, 192, 256 * 100 * 2, 256 * 2, 256, 6400, 64)


def _fwd(L, q=OK, kv=OK, kr=OK, st=DENSE, cu_q=None, cu_k=None, n=0, o=OK, lse=OK, B=1, Tq=100, Tk=100, H=2, dn=128, dr=64,
         causal=1, scale=0.1, dtype=1, ws=None, bytes=0):
    return L.kda_latent_attn_fwd(None, q, kv, kr, None if st is None else _st(*st), cu_q, cu_k, n, o, lse, B, Tq, Tk, H, dn,
                                 dr, causal, scale, dtype, ws, bytes)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(kv=None), -1), (dict(kr=None), -1), (dict(o=None), -1), (dict(lse=None), -1), (dict(st=None), -1),
    (dict(q=OK + 8), -1), (dict(kv=OK + 2), -1), (dict(kr=OK + 4), -1), (dict(o=OK + 8), -1),
    (dict(B=-1), -1), (dict(Tq=-1), -1), (dict(Tk=-5), -1), (dict(H=0), -1), (dict(dn=96), -2), (dict(dr=16), -2), (dict(dr=0), -2),
    (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(cu_q=OK), -1), (dict(cu_q=OK, cu_k=OK, n=0), -1),
    (dict(cu_q=OK, cu_k=OK, n=2, B=2), -1), (dict(st=DENSE[:1] + (193,) + DENSE[2:]), -1), (dict(st=DENSE[:7] + (-64,)), -1),
    (dict(st=DENSE[:4] + (1 << 24,) + DENSE[5:]), -2), (dict(B=70000, H=1), -2), (dict(Tq=1 << 30, H=128), -2),
    (dict(Tk=1000), -3), (dict(Tk=1000, ws=OK, bytes=64), -3), (dict(Tk=1000, ws=OK + 4, bytes=1 << 40), -1)])
def test_forward_refuses(L, kw, code):
    assert _fwd(L, **kw) == code
    assert _lib.last_error()


def test_empty_calls_do_nothing(L):
    assert _fwd(L, B=0) == 0 and _fwd(L, Tq=0) == 0
    assert L.kda_latent_append(None, None, 0, None, None, None, 0, None, 0.0, None, 0, None, 0, 0, None, 0, 0, 0, 0, 512, 64, 0, 1) == 0
    assert L.kda_latent_decode(None, None, None, None, None, None, None, 0, 1, 1, 512, 64, 1, 16, 1, 0.1, 1, None, 0) == 0


def _up(x):
    return -(-x // 256) * 256


def _splits(T, other, B, H, n, slots):
    """Workgroups of a block of 128 rows along the other axis: until `slots` workgroups, 16 at most, 128 rows each at least."""
    blocks = (T // 128 + n if n else -(-T // 128)) * B * H
    return max(1, min(slots // blocks, -(-other // 128), 16)) if blocks else 1


@pytest.mark.parametrize("B,Tq,Tk,H,dn,dr,n", [(2, 300, 400, 3, 128, 64, 0), (1, 1, 5000, 16, 128, 64, 0), (4, 4096, 4096, 16, 128, 64, 0),
                                               (1, 700, 700, 2, 64, 32, 9), (1, 0, 50, 2, 64, 32, 0), (1, 50, 0, 2, 64, 32, 0)])
@pytest.mark.parametrize("code", [0, 1, 2])
def test_attention_workspaces(L, B, Tq, Tk, H, dn, dr, n, code):
    s = _splits(Tq, Tk, B, H, n, 256)
    rows = s * B * H * Tq if s > 1 else 0
    assert L.kda_latent_attn_fwd_workspace(B, Tq, Tk, H, dn, dr, n, code) == _up(rows * dn * 4) + _up(rows * 8)
    # D, the blocks' largest |do|, each head's (and part's) share of the rotary key's gradient, the parts of dq and of dkv
    k = _splits(Tk, Tq, B, H, n, 256)
    want = _up(B * H * Tq * 4) + _up(B * H * (Tq // 128 + n if n else -(-Tq // 128)) * 4) + _up(k * B * H * Tk * dr * 4)
    want += _up(rows * (dn + dr) * 4) + _up(k * B * H * Tk * 2 * dn * 4 if k > 1 else 0) + 256
    assert L.kda_latent_attn_bwd_workspace(B, Tq, Tk, H, dn, dr, n, code) == want


@pytest.mark.parametrize("bad", [(-1, 1, 1, 1, 64, 64, 0, 1), (1, -1, 1, 1, 64, 64, 0, 1), (1, 1, 1, 0, 64, 64, 0, 1),
                                 (1, 1, 1, 1, 96, 64, 0, 1), (1, 1, 1, 1, 64, 48, 0, 1), (1, 1, 1, 1, 64, 64, -1, 1), (1, 1, 1, 1, 64, 64, 0, 3)])
def test_attention_workspaces_refuse(L, bad):
    assert L.kda_latent_attn_fwd_workspace(*bad) == 0 and L.kda_latent_attn_bwd_workspace(*bad) == 0


def test_backward_refuses(L):
    def bwd(ws=OK, n=None, o=OK, do=OK, dq=OK, dkv=OK, dkr=OK):
        need = L.kda_latent_attn_bwd_workspace(1, 100, 100, 2, 128, 64, 0, 1)
        return L.kda_latent_attn_bwd(None, OK, OK, OK, _st(*DENSE), None, None, 0, o, OK, do, dq, dkv, dkr, 1, 100, 100, 2, 128,
                                     64, 1, 0.1, 1, ws, need - 1 if n is None else n)
    assert bwd() == -3 and bwd(ws=None, n=1 << 30) == -3
    for kw in (dict(o=None), dict(do=None), dict(dq=None), dict(dkv=None), dict(dkr=None), dict(do=OK + 2), dict(dkv=OK + 8)):
        assert bwd(n=1 << 30, **kw) == -1, kw
    assert bwd(ws=OK + 4, n=1 << 30) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(rows=None), -1), (dict(pos=None), -1), (dict(slots=None), -1), (dict(cs=None), -1), (dict(P=0), -1), (dict(cache=None), -1),
    (dict(q=None), -1), (dict(qo=None), -1), (dict(rows=OK + 8), -1), (dict(cache=OK + 2), -1), (dict(cs=OK + 4), -1),
    (dict(rs=577), -1), (dict(q=OK + 2), -1), (dict(qh=66), -1), (dict(N=-1), -1), (dict(H=0), -1), (dict(R=384), -2), (dict(dr=48), -2),
    (dict(dtype=3), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1)])
def test_append_refuses(L, kw, code):
    d = dict(rows=OK, rs=576, pos=OK, slots=OK, cs=OK, P=10, w=OK, eps=1e-6, cache=OK, n=64, q=OK, qt=256, qh=64, qo=OK, N=3, H=4,
             R=512, dr=64, dtype=1)
    d.update(kw)
    rc = L.kda_latent_append(None, d["rows"], d["rs"], d["pos"], d["slots"], d["cs"], d["P"], d["w"], d["eps"], d["cache"], d["n"],
                             d["q"], d["qt"], d["qh"], d["qo"], d["qt"], d["qh"], d["N"], d["H"], d["R"], d["dr"], 0, d["dtype"])
    assert rc == code and _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(cache=None), -1), (dict(table=None), -1), (dict(lens=None), -1), (dict(o=None), -1), (dict(lse=None), -1),
    (dict(q=OK + 8), -1), (dict(cache=OK + 4), -1), (dict(o=OK + 2), -1), (dict(ws=OK + 8), -1), (dict(ws=None), -3), (dict(bytes=100), -3),
    (dict(B=-1), -1), (dict(B=70000), -2), (dict(Tq=0), -1), (dict(H=0), -1), (dict(R=128), -2), (dict(dr=128), -2), (dict(page=48), -1),
    (dict(page=0), -1), (dict(pages=1 << 27), -2), (dict(per=-1), -1), (dict(per=1 << 27), -2), (dict(scale=0.0), -1), (dict(dtype=3), -1)])
def test_decode_refuses(L, kw, code):
    d = dict(q=OK, cache=OK, table=OK, lens=OK, o=OK, lse=OK, B=2, Tq=1, H=16, R=512, dr=64, pages=100, page=16, per=20, scale=0.1,
             dtype=1, ws=OK, bytes=1 << 40)
    d.update(kw)
    rc = L.kda_latent_decode(None, d["q"], d["cache"], d["table"], d["lens"], d["o"], d["lse"], d["B"], d["Tq"], d["H"], d["R"], d["dr"],
                             d["pages"], d["page"], d["per"], d["scale"], d["dtype"], d["ws"], d["bytes"])
    assert rc == code and _lib.last_error()


def test_decode_workspace(L):
    assert L.kda_latent_decode_workspace(4, 1, 16, 512, 64, 64, 100, 1) > 0
    for bad in ((-1, 1, 16, 512, 64, 64, 100, 1), (4, 0, 16, 512, 64, 64, 100, 1), (4, 1, 16, 384, 64, 64, 100, 1),
                (4, 1, 16, 512, 48, 64, 100, 1), (4, 1, 16, 512, 64, 48, 100, 1), (4, 1, 16, 512, 64, 64, 100, 3)):
        assert L.kda_latent_decode_workspace(*bad) == 0


def _cpu(*s, dt=torch.bfloat16):
    return torch.zeros(*s, dtype=dt)


def test_python_refuses():
    q, kv, kr = _cpu(1, 8, 2, 192), _cpu(1, 8, 2, 256), _cpu(1, 8, 64)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    bad = [(q[0], kv, kr, {}), (q, kv[..., :255], kr, {}), (q[..., :190], kv, kr, {}), (q.float(), kv, kr, {}), (q, kv, kr[:, :7], {}),
           (q.to(torch.float64), kv.to(torch.float64), kr.to(torch.float64), {}), (q.transpose(2, 3).contiguous().transpose(2, 3), kv, kr, {}),
           (q, kv, kr, dict(cu_seqlens=cu.long())), (q, kv, kr, dict(cu_seqlens_k=cu)), (q, kv, kr, dict(cu_seqlens=cu[:1])),
           (q[:, :4], kv, kr, dict(cu_seqlens=cu)), (q, kv, kr, dict(cu_seqlens=cu, cu_seqlens_k=torch.tensor([0, 4, 8], dtype=torch.int32)))]
    for a, b, c, kw in bad:
        with pytest.raises(ValueError):
            axiom_amd.latent_attn_fwd(a, b, c, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        axiom_amd.latent_attn_fwd(q, kv, kr)
    with pytest.raises(RuntimeError):
        axiom_amd.latent_attn(q, kv, kr)
    o, lse = _cpu(1, 8, 2, 128), _cpu(1, 2, 8, dt=torch.float32)
    for args in ((o[..., :64], lse, o), (o, lse[:, :1], o), (o, lse.half(), o), (o, lse, o.float()), (o, lse, o.expand(1, 8, 2, 128)[:, :, :1])):
        with pytest.raises(ValueError):
            axiom_amd.latent_attn_bwd(q, kv, kr, *args)
    rows, cache, cs = _cpu(4, 576), _cpu(3, 16, 576), _cpu(10, 64, dt=torch.float32)
    pos = torch.zeros(4, dtype=torch.int64)
    good = dict(rows=rows, positions=pos, slots=pos, cos_sin=cs, cache=cache)
    for kw in (dict(rows=rows[0]), dict(cache=cache[..., :512]), dict(cos_sin=cs.half()), dict(cos_sin=cs[:0]), dict(positions=pos.int()),
               dict(slots=pos[:3]), dict(norm_weight=_cpu(512)), dict(norm_weight=_cpu(256, dt=torch.float32)), dict(q_out=_cpu(4, 2, 64)),
               dict(q_rope=_cpu(4, 2, 32)), dict(q_rope=_cpu(4, 2, 64), q_out=_cpu(4, 3, 64)), dict(cache=cache.float()),
               dict(cache=_cpu(16, 3, 576).transpose(0, 1)), dict(q_rope=_cpu(4, 0, 64))):
        with pytest.raises(ValueError):
            axiom_amd.latent_append(**{**good, **kw})
    with pytest.raises(RuntimeError):
        axiom_amd.latent_append(**good)
    qa, table, lens = _cpu(2, 1, 4, 576), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args in ((qa[0], cache, table, lens), (qa[..., :512], cache, table, lens), (qa, cache.float(), table, lens), (qa, cache, table.long(), lens),
                 (qa, cache, table[:1], lens), (qa, cache, table, lens.long()), (qa, cache, table, lens[:1])):
        with pytest.raises(ValueError):
            axiom_amd.latent_decode(*args, scale=0.1)
    with pytest.raises(RuntimeError):
        axiom_amd.latent_decode(qa, cache, table, lens, scale=0.1)
    assert lat.latent_decode_workspace_bytes(2, 1, 4, 512, 64, 16, 3) > 0


def test_oracle_against_autograd():
    """The oracle's gradient against autograd through torch's softmax in float64; empty rows apart."""
    g = torch.Generator().manual_seed(0)
    q, kv, kr, do = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 5, 3, 12), (2, 7, 3, 16), (2, 7, 4), (2, 5, 3, 8)))
    o, lse, dq, dkv, dkr = O.attn(q, kv, kr, True, 0.3, do=do)
    x = [t.clone().requires_grad_(True) for t in (q, kv, kr)]
    k = torch.cat([x[1][..., :8], x[2][:, :, None].expand(2, 7, 3, 4)], -1)
    s = 0.3 * torch.einsum("bihd,bjhd->bhij", x[0], k)
    s = s.masked_fill(torch.arange(7)[None] > torch.arange(5)[:, None] + 2, float("-inf"))
    want = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), x[1][..., 8:])
    grads = torch.autograd.grad(want, x, do)
    assert torch.allclose(o, want) and torch.allclose(lse, torch.logsumexp(s, -1))
    for a, b in zip((dq, dkv, dkr), grads):
        assert torch.allclose(a, b)
