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

Every function calls the HIP library through its C ABI (``include/latent_mi355x.h``)
on torch's current stream, by the C++ binding ``_latent_torch`` that also checks
the arguments; nothing here computes on the CPU.
"""

from __future__ import annotations

import torch

from . import _lib
from .kda import _IN_CODES

_binding = None


def _ext():
    """The C++ binding; raises RuntimeError when it has not been built."""
    global _binding
    if _binding is None:
        _lib.lib()   # the library itself: its own message where it is missing
        try:
            from . import _latent_torch
        except ImportError as e:
            raise RuntimeError("axiom_amd: _latent_torch.so is not built (run `python -m axiom_amd.build`); "
                               "the latent attention has no fallback implementation") from e
        _binding = _latent_torch
    return _binding


def latent_attn_fwd(q, kv, k_rope, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None, out=None, lse=None,
                    workspace=None):
    """Latent attention, expanded form; returns ``(o, lse)``.

    ``q [B,Tq,H,dn+dr]`` (nope part, then the rotated part), ``kv [B,Tk,H,2 dn]``
    (nope key, then value: the up-projection's output as it is), ``k_rope
    [B,Tk,dr]`` the rotated key of all heads; one dtype (bf16, fp16 or fp32),
    last axis contiguous, other strides free (multiples of 16 bytes).  ``o
    [B,Tq,H,dn]`` in that dtype; ``lse [B,H,Tq]`` fp32, natural logarithm.
    ``causal``: query i sees keys ``j <= i + Tk - Tq``.  A query that sees no key
    gets zeros and ``-inf``, whatever the keys hold; else values that are not finite
    may reach rows of the same sequence that do not see them.  ``cu_seqlens`` (int32 ``[N+1]`` on the device, B ==
    1) packs N sequences; ``cu_seqlens_k`` its key offsets where they differ.
    ``scale``: default ``(dn + dr) ** -0.5``.  dn in {64, 128}, dr in {32, 64}.
    ``out`` / ``lse``: optional preallocated outputs; ``workspace``: an optional
    uint8 device buffer (a call of few blocks needs one; a smaller one than
    needed is replaced by a new one).
    """
    return _ext().attn_fwd(q, kv, k_rope, cu_seqlens, cu_seqlens_k, causal, scale, out, lse, workspace)


def latent_attn_bwd(q, kv, k_rope, o, lse, do, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None,
                    workspace=None):
    """Gradients ``(dq, dkv, dk_rope)`` of :func:`latent_attn_fwd`'s ``o``, contiguous, in the inputs' dtype.

    ``o``, ``lse`` as the forward returned them, ``do`` the cotangent of ``o``
    (contiguous, the inputs' dtype).  ``dk_rope`` is summed over the heads.  The
    same bits in every run (no atomics).  ``workspace``: an optional uint8
    device buffer; a smaller one than needed is replaced by a new one.
    """
    return _ext().attn_bwd(q, kv, k_rope, o, lse, do, cu_seqlens, cu_seqlens_k, causal, scale, workspace)


def latent_attn(q, kv, k_rope, cu_seqlens=None, cu_seqlens_k=None, causal: bool = True, scale=None):
    """Differentiable latent attention, expanded form: ``o`` of :func:`latent_attn_fwd` with the HIP backward.

    Gradients flow to ``q``, ``kv`` and ``k_rope`` (the heads' sum), in their dtype.
    Differentiable once: differentiating the gradients themselves raises RuntimeError.
    """
    return _ext().attn(q, kv, k_rope, cu_seqlens, cu_seqlens_k, causal, scale)


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
    return _ext().append(rows, positions, slots, cos_sin, cache, norm_weight, eps, q_rope, q_out, interleaved)


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
    return _ext().decode(q, cache, block_table, seq_lens, scale, out, lse, workspace)
