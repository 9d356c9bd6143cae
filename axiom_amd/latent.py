"""Latent attention: the softmax layers that stand between KDA layers.

A latent-attention layer keeps, per token, one normed latent vector of R
elements and one rotated key part of dr elements that all heads share.

* :func:`latent_attn` -- the expanded form, differentiable: attention on the
  up-projected keys and values (prompts, training); :func:`latent_attn_fwd` /
  :func:`latent_attn_bwd` are its two directions.
* :func:`latent_append` -- norm and rotation of new tokens' rows, stored in a
  paged cache, the queries' rotary parts rotated in the same launch.
* :func:`latent_decode` -- the absorbed form: one to a few query tokens of every
  sequence over the paged cache.

With ``W_uk [H, dn, R]`` and ``W_uv [H, dn, R]`` the up-projection's halves, the
two forms agree: ``kv = (c W_uk^T | c W_uv^T)`` per head in the expanded one;
``q = (q_n W_uk | q_r)`` and ``o_latent W_uv^T`` around the absorbed one.

Every function calls the HIP library through its C ABI on torch's current
stream; nothing here computes on the CPU.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kda import _IN_CODES, _contig, _ptr, _require_gpu, _stream, _ws_bytes

_Strides = ctypes.c_int64 * 8


def _attn_check(what, q, kv, k_rope, cu_seqlens, cu_seqlens_k, scale):
    """Sizes, strides and packed offsets of an expanded-form call."""
    if q.dim() != 4 or kv.dim() != 4 or k_rope.dim() != 3:
        raise ValueError(f"{what}: q must be [B,Tq,H,dn+dr], kv [B,Tk,H,2 dn], k_rope [B,Tk,dr]")
    B, Tq, H, dqk = q.shape
    Tk, dn, dr = kv.shape[1], kv.shape[3] // 2, k_rope.shape[2]
    if kv.shape != (B, Tk, H, 2 * dn) or k_rope.shape != (B, Tk, dr) or dqk != dn + dr:
        raise ValueError(f"{what}: q {tuple(q.shape)}, kv {tuple(kv.shape)} and k_rope {tuple(k_rope.shape)} do not fit "
                         "q [B,Tq,H,dn+dr], kv [B,Tk,H,2 dn], k_rope [B,Tk,dr]")
    if q.dtype not in _IN_CODES or kv.dtype != q.dtype or k_rope.dtype != q.dtype:
        raise ValueError(f"{what}: q, kv, k_rope must share a dtype in bf16/fp16/fp32")
    st = q.stride()[:3] + kv.stride()[:3] + k_rope.stride()[:2]
    if (dqk > 0 and q.stride(3) != 1) or kv.stride(3) != 1 or k_rope.stride(2) != 1:
        raise ValueError(f"{what}: the last axis of q, kv and k_rope must be contiguous")
    n_seqs = 0
    if cu_seqlens is not None:
        if cu_seqlens_k is None:
            if Tq != Tk:
                raise ValueError(f"{what}: cu_seqlens alone needs Tq == Tk, got {Tq} and {Tk}")
            cu_seqlens_k = cu_seqlens
        for name, cu in (("cu_seqlens", cu_seqlens), ("cu_seqlens_k", cu_seqlens_k)):
            if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 2:
                raise ValueError(f"{what}: {name} must be a 1-D int32 tensor of N+1 >= 2 offsets")
            _contig(name, cu)
        if cu_seqlens_k.numel() != cu_seqlens.numel():
            raise ValueError(f"{what}: cu_seqlens and cu_seqlens_k must have the same length")
        if B != 1:
            raise ValueError(f"{what}: cu_seqlens requires B == 1, got B={B}")
        n_seqs = cu_seqlens.numel() - 1
    elif cu_seqlens_k is not None:
        raise ValueError(f"{what}: cu_seqlens_k requires cu_seqlens")
    scale = (dn + dr) ** -0.5 if scale is None else float(scale)
    return B, Tq, Tk, H, dn, dr, _Strides(*st), cu_seqlens, cu_seqlens_k, n_seqs, scale


def _output(name, what, t, shape, dtype, dev):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if t.shape != shape or t.dtype != dtype or t.device != dev:
        raise ValueError(f"{what}: {name} must be {dtype} {list(shape)} on {dev}")
    _contig(name, t)
    return t


def latent_attn_fwd(q, kv, k_rope, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None, out=None, lse=None,
                    workspace=None):
    """Latent attention, expanded form; returns ``(o, lse)``.

    ``q [B,Tq,H,dn+dr]`` (nope part, then the rotated part), ``kv [B,Tk,H,2 dn]``
    (nope key, then value: the up-projection's output as it is), ``k_rope
    [B,Tk,dr]`` the rotated key of all heads; one dtype (bf16, fp16 or fp32),
    last axis contiguous, other strides free (multiples of 16 bytes).  ``o
    [B,Tq,H,dn]`` in that dtype; ``lse [B,H,Tq]`` fp32, natural logarithm.
    ``causal``: query i sees keys ``j <= i + Tk - Tq``.  A query that sees no key
    gets zeros and ``-inf``.  ``cu_seqlens`` (int32 ``[N+1]`` on the device, B ==
    1) packs N sequences; ``cu_seqlens_k`` its key offsets where they differ.
    ``scale``: default ``(dn + dr) ** -0.5``.  dn in {64, 128}, dr in {32, 64}.
    ``out`` / ``lse``: optional preallocated outputs; ``workspace``: an optional
    uint8 device buffer (a call of few blocks needs one; a smaller one than
    needed is replaced by a new one).
    """
    what = "latent_attn_fwd"
    B, Tq, Tk, H, dn, dr, st, cu_q, cu_k, n_seqs, scale = _attn_check(what, q, kv, k_rope, cu_seqlens, cu_seqlens_k, scale)
    dev = _require_gpu([q, kv, k_rope, cu_q, cu_k], what)
    o = _output("out", what, out, (B, Tq, H, dn), q.dtype, dev)
    lse = _output("lse", what, lse, (B, H, Tq), torch.float32, dev)
    code = _IN_CODES[q.dtype]
    ws_bytes = _ws_bytes("kda_latent_attn_fwd_workspace", B, Tq, Tk, H, dn, dr, n_seqs, code)
    if ws_bytes and (workspace is None or workspace.numel() * workspace.element_size() < ws_bytes):
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    rc = _lib.lib().kda_latent_attn_fwd(_stream(dev), _ptr(q), _ptr(kv), _ptr(k_rope), st, _ptr(cu_q), _ptr(cu_k), n_seqs,
                                        _ptr(o), _ptr(lse), B, Tq, Tk, H, dn, dr, 1 if causal else 0, scale, code,
                                        _ptr(workspace), ws_bytes)
    _lib.check(rc, what)
    return o, lse


def latent_attn_bwd(q, kv, k_rope, o, lse, do, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None,
                    workspace=None):
    """Gradients ``(dq, dkv, dk_rope)`` of :func:`latent_attn_fwd`'s ``o``, contiguous, in the inputs' dtype.

    ``o``, ``lse`` as the forward returned them, ``do`` the cotangent of ``o``
    (contiguous, the inputs' dtype).  ``dk_rope`` is summed over the heads.  The
    same bits in every run (no atomics).  ``workspace``: an optional uint8
    device buffer; a smaller one than needed is replaced by a new one.
    """
    what = "latent_attn_bwd"
    B, Tq, Tk, H, dn, dr, st, cu_q, cu_k, n_seqs, scale = _attn_check(what, q, kv, k_rope, cu_seqlens, cu_seqlens_k, scale)
    for name, t in (("o", o), ("do", do)):
        if t.shape != (B, Tq, H, dn) or t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} must be {q.dtype} [{B},{Tq},{H},{dn}]")
        _contig(name, t)
    if lse.shape != (B, H, Tq) or lse.dtype != torch.float32:
        raise ValueError(f"{what}: lse must be fp32 [{B},{H},{Tq}]")
    _contig("lse", lse)
    dev = _require_gpu([q, kv, k_rope, o, lse, do, cu_q, cu_k], what)
    ws_bytes = _ws_bytes("kda_latent_attn_bwd_workspace", B, Tq, Tk, H, dn, dr, n_seqs, _IN_CODES[q.dtype])
    if workspace is None or workspace.numel() * workspace.element_size() < ws_bytes:
        workspace = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    dq = torch.empty((B, Tq, H, dn + dr), dtype=q.dtype, device=dev)
    dkv = torch.empty((B, Tk, H, 2 * dn), dtype=q.dtype, device=dev)
    dkr = torch.empty((B, Tk, dr), dtype=q.dtype, device=dev)
    rc = _lib.lib().kda_latent_attn_bwd(_stream(dev), _ptr(q), _ptr(kv), _ptr(k_rope), st, _ptr(cu_q), _ptr(cu_k), n_seqs,
                                        _ptr(o), _ptr(lse), _ptr(do), _ptr(dq), _ptr(dkv), _ptr(dkr), B, Tq, Tk, H, dn, dr,
                                        1 if causal else 0, scale, _IN_CODES[q.dtype], _ptr(workspace), ws_bytes)
    _lib.check(rc, what)
    return dq, dkv, dkr


class _LatentAttn(torch.autograd.Function):
    """``o`` of the expanded form with the HIP backward as its VJP."""

    @staticmethod
    def forward(ctx, q, kv, k_rope, cu_q, cu_k, causal, scale):
        o, lse = latent_attn_fwd(q, kv, k_rope, cu_q, cu_k, causal, scale)
        ctx.save_for_backward(q, kv, k_rope, o, lse, cu_q, cu_k)
        ctx.args = causal, scale
        return o

    @staticmethod
    def backward(ctx, do):
        q, kv, k_rope, o, lse, cu_q, cu_k = ctx.saved_tensors
        return (*latent_attn_bwd(q, kv, k_rope, o, lse, do.contiguous(), cu_q, cu_k, *ctx.args), None, None, None, None)


def latent_attn(q, kv, k_rope, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None):
    """Differentiable latent attention, expanded form: ``o`` of :func:`latent_attn_fwd` with the HIP backward.

    Gradients flow to ``q``, ``kv`` and ``k_rope`` (the heads' sum), in their dtype.
    """
    return _LatentAttn.apply(q, kv, k_rope, cu_seqlens, cu_seqlens_k, causal, scale)


def latent_append(rows, positions, slots, cos_sin, cache, norm_weight=None, eps: float = 1e-6, q_rope=None, q_out=None,
                  interleaved: bool = False):
    """Norm, rotate and store new tokens in the paged latent cache; returns ``q_out``.

    ``rows [N, R+dr]`` the down-projection's output (row stride free); the first
    R elements are RMS-normed with ``norm_weight`` (fp32 ``[R]``; None: taken as
    they are), the last dr rotated at ``positions`` (int64 ``[N]``) with
    ``cos_sin`` (fp32 ``[P, dr]``: cosines of the dr/2 angles, then sines), and
    the row is stored in place at ``slots`` (int64 ``[N]``: page * page_size +
    offset) of ``cache [n_pages, page_size, R+dr]``.  A slot outside the cache
    (-1) is not stored; a position outside the table takes its nearest row.
    ``q_rope [N,H,dr]`` (strided views allowed) is rotated in the same launch
    into ``q_out`` (same shape, may be a slice of the absorbed query or
    ``q_rope`` itself; None: a new tensor).  ``interleaved``: pairs (2i, 2i+1)
    instead of (i, i + dr/2).  Slots of one call must differ.
    """
    what = "latent_append"
    if rows.dim() != 2 or cache.dim() != 3 or cache.shape[2] != rows.shape[1]:
        raise ValueError(f"{what}: rows must be [N, R+dr] and cache [n_pages, page_size, R+dr]")
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or cos_sin.shape[0] < 1:
        raise ValueError(f"{what}: cos_sin must be fp32 [P, dr]")
    N, dr = rows.shape[0], cos_sin.shape[1]
    R = rows.shape[1] - dr
    if rows.dtype not in _IN_CODES or cache.dtype != rows.dtype:
        raise ValueError(f"{what}: rows and cache must share a dtype in bf16/fp16/fp32")
    for name, t in (("positions", positions), ("slots", slots)):
        if t.dtype != torch.int64 or t.shape != (N,):
            raise ValueError(f"{what}: {name} must be int64 [{N}]")
        _contig(name, t)
    if norm_weight is not None:
        if norm_weight.dtype != torch.float32 or norm_weight.shape != (R,):
            raise ValueError(f"{what}: norm_weight must be fp32 [{R}]")
        _contig("norm_weight", norm_weight)
    _contig("cos_sin", cos_sin)
    _contig("cache", cache)
    if rows.stride(1) != 1:
        raise ValueError(f"{what}: the last axis of rows must be contiguous")
    H, qs, os_ = 0, (0, 0), (0, 0)
    if q_rope is not None:
        if q_rope.dim() != 3 or q_rope.shape[0] != N or q_rope.shape[2] != dr or q_rope.dtype != rows.dtype:
            raise ValueError(f"{what}: q_rope must be {rows.dtype} [{N}, H, {dr}]")
        if q_out is None:
            q_out = torch.empty(q_rope.shape, dtype=q_rope.dtype, device=q_rope.device)
        if q_out.shape != q_rope.shape or q_out.dtype != q_rope.dtype:
            raise ValueError(f"{what}: q_out must match q_rope")
        if q_rope.stride(2) != 1 or q_out.stride(2) != 1:
            raise ValueError(f"{what}: the last axis of q_rope and q_out must be contiguous")
        H, qs, os_ = q_rope.shape[1], q_rope.stride(), q_out.stride()
        if H == 0:
            raise ValueError(f"{what}: q_rope has no heads")
    elif q_out is not None:
        raise ValueError(f"{what}: q_out requires q_rope")
    dev = _require_gpu([rows, positions, slots, cos_sin, cache, norm_weight, q_rope, q_out], what)
    rc = _lib.lib().kda_latent_append(_stream(dev), _ptr(rows), rows.stride(0), _ptr(positions), _ptr(slots), _ptr(cos_sin),
                                      cos_sin.shape[0], _ptr(norm_weight), float(eps), _ptr(cache),
                                      cache.shape[0] * cache.shape[1], _ptr(q_rope), qs[0], qs[1], _ptr(q_out), os_[0],
                                      os_[1], N, H, R, dr, 1 if interleaved else 0, _IN_CODES[rows.dtype])
    _lib.check(rc, what)
    return q_out


def latent_decode_workspace_bytes(B, Tq, H, R, dr, page_size, max_pages, dtype=torch.bfloat16) -> int:
    """Workspace bytes of :func:`latent_decode` (``kda_latent_decode_workspace``)."""
    return int(_lib.lib().kda_latent_decode_workspace(B, Tq, H, R, dr, page_size, max_pages, _IN_CODES[dtype]))


def latent_decode(q, cache, block_table, seq_lens, scale: float, out=None, lse=None, workspace=None):
    """Latent attention over the paged cache (absorbed form); returns ``(o, lse)``.

    ``q [B,Tq,H,R+dr]`` (the nope query times the key up-projection, then the
    rotated part), ``cache [n_pages, page_size, R+dr]``, ``block_table`` int32
    ``[B, max_pages]``, ``seq_lens`` int32 ``[B]`` (tokens in the cache, the Tq
    new ones among them).  ``o [B,Tq,H,R]`` in q's dtype (bf16, fp16 or fp32),
    ``lse [B,Tq,H]`` fp32.  Token t sees the first ``seq_len - (Tq-1-t)`` rows;
    with none it gets zeros and ``-inf``.  ``scale`` is that of the expanded
    head, ``(dn + dr) ** -0.5``.  R in {256, 512}, dr in {32, 64} (taken from the
    row's width), ``page_size`` a power of two.  ``workspace``: an optional uint8
    device buffer; a smaller one than needed is replaced by a new one.
    """
    what = "latent_decode"
    if q.dim() != 4 or cache.dim() != 3 or q.shape[3] != cache.shape[2]:
        raise ValueError(f"{what}: q must be [B,Tq,H,R+dr] and cache [n_pages, page_size, R+dr]")
    B, Tq, H, W = q.shape
    R = 512 if W > 512 else 256
    dr = W - R
    if q.dtype not in _IN_CODES or cache.dtype != q.dtype:
        raise ValueError(f"{what}: q and cache must share a dtype in bf16/fp16/fp32")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype != torch.int32:
        raise ValueError(f"{what}: block_table must be int32 [{B}, max_pages]")
    if seq_lens.shape != (B,) or seq_lens.dtype != torch.int32:
        raise ValueError(f"{what}: seq_lens must be int32 [{B}]")
    for name, t in (("q", q), ("cache", cache), ("block_table", block_table), ("seq_lens", seq_lens)):
        _contig(name, t)
    dev = _require_gpu([q, cache, block_table, seq_lens], what)
    code = _IN_CODES[q.dtype]
    n_pages, page, per = cache.shape[0], cache.shape[1], block_table.shape[1]
    ws_bytes = _ws_bytes("kda_latent_decode_workspace", B, Tq, H, R, dr, page, per, code)
    if workspace is None or workspace.numel() * workspace.element_size() < ws_bytes:
        workspace = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    o = _output("out", what, out, (B, Tq, H, R), q.dtype, dev)
    lse = _output("lse", what, lse, (B, Tq, H), torch.float32, dev)
    rc = _lib.lib().kda_latent_decode(_stream(dev), _ptr(q), _ptr(cache), _ptr(block_table), _ptr(seq_lens), _ptr(o),
                                      _ptr(lse), B, Tq, H, R, dr, n_pages, page, per, float(scale), code, _ptr(workspace),
                                      ws_bytes)
    _lib.check(rc, what)
    return o, lse
