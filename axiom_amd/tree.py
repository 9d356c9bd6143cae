"""Trees of drafted tokens: decoded in one step, verified, and the accepted path kept.

A program that drafts several tokens ahead (a multi-token head, a small model)
gives every sequence N places, 1 to 64.  ``parents`` int32 ``[B,N]`` says what
place i continues: a place in ``[0, i)``, or -1, the sequence itself; any other
entry marks a place without a draft (and those below it hold none either).  A
chain has ``parents[i] = i - 1``.  The path of a place: its ancestors and itself.

* :func:`kda_tree_step` -- the KDA layers: :func:`~axiom_amd.kda_recurrent_step` for
  every place, from the state that its path leads to; the state stays as it is.
* :func:`latent_tree_decode` -- the latent layers: :func:`~axiom_amd.latent_decode`
  where a place sees the cache and its own path.
* :func:`tree_verify` -- the path that the target's distributions accept, from given
  random numbers or greedily, and the token that follows.
* :func:`kda_tree_commit`, :func:`latent_tree_commit` -- states and caches after it.

All of them read trees, lengths and accepted places on the device and never wait
for the host, so a step of a serving loop can be captured into a HIP graph.  A
place without a draft gets zeros, and what its inputs hold reaches nothing; a
draft whose own values are not finite may reach the other drafts of its sequence.

What a call writes must not overlap its other arguments.

Every function calls the HIP library through its C ABI (``include/tree_mi355x.h``)
on torch's current stream, by the C++ binding that also checks the arguments;
nothing here computes on the CPU.  None is differentiable.
"""

from __future__ import annotations

import torch

from . import _lib
from .kda import _IN_CODES
from .latent import _ext


def kda_tree_step(q, k, v, g, beta, parents, state, scale: float = 1.0, out_dtype=torch.float32, out=None, u=None):
    """The delta rule over a tree; returns ``(o, u)``, ``state`` is read only.

    ``q, k, g [B,N,H,dk]``, ``v [B,N,H,dv]``, ``beta [B,N,H]`` (one dtype: bf16,
    fp16 or fp32), ``state [B,H,dk,dv]`` fp32, dk == dv in {64, 128}.  With S
    the state after the parent of place i (``state`` for -1): ``S~ = diag(exp g_i)
    S``, ``u_i = beta_i (v_i - S~^T k_i)``, ``S_i = S~ + k_i u_i^T`` and ``o_i =
    scale S_i^T q_i``.  ``o [B,N,H,dv]`` in ``out_dtype`` (fp32 or bf16), ``u
    [B,N,H,dv]`` fp32 for :func:`kda_tree_commit`.  ``out`` / ``u``: optional
    preallocated outputs.  A decay between two places is as exact as those of the places
    between them, however far the path has decayed before.
    """
    return _ext().tree_step(q, k, v, g, beta, parents, state, scale, out_dtype, out, u)


def kda_tree_commit(k, g, u, parents, last, state):
    """``state`` after the path of place ``last[b]`` (int32 ``[B]``), in place; returns it.

    ``k``, ``g``, ``parents`` as given to :func:`kda_tree_step` and its ``u``.  A
    ``last[b]`` outside ``[0, N)``, or a place without a draft, leaves the state of
    its sequence as it is.
    """
    return _ext().tree_commit(k, g, u, parents, last, state)


def latent_tree_decode_workspace_bytes(B, N, H, R, dr, page_size, max_pages, dtype=torch.bfloat16) -> int:
    """Workspace bytes of :func:`latent_tree_decode` (``kda_latent_tree_decode_workspace``)."""
    return int(_lib.lib().kda_latent_tree_decode_workspace(B, N, H, R, dr, page_size, max_pages, _IN_CODES[dtype]))


def latent_tree_decode(q, cache, block_table, seq_lens, parents, scale: float, out=None, lse=None, workspace=None):
    """Latent attention of a tree of drafts over the paged cache; returns ``(o, lse)``.

    ``q [B,N,H,R+dr]`` and the other arguments as :func:`~axiom_amd.latent_decode`'s; the N
    newest rows of a sequence are its places', place i in row ``seq_lens[b] - N + i``
    (:func:`~axiom_amd.latent_append` puts them there; their rotary positions follow
    their depth).  Place i sees every row before the places' and those of its path.
    A place without a draft needs a row too, which is not read.  ``o [B,N,H,R]`` in
    q's dtype, ``lse [B,N,H]`` fp32; zeros and ``-inf`` for places without a draft and
    for those before the sequence's first row.
    """
    return _ext().tree_decode(q, cache, block_table, seq_lens, parents, scale, out, lse, workspace)


def latent_tree_commit(cache, block_table, seq_lens, parents, last, out=None):
    """The accepted path's rows moved to the front of the places', in place; returns the new lengths.

    ``cache [n_pages, page_size, R+dr]`` or, for several layers that share the block
    table, ``[layers, n_pages, page_size, R+dr]``.  Row ``seq_len - N + path[i]``
    goes to row ``seq_len - N + i``; the new length is ``seq_len - N`` and the path's
    (int32 ``[B]``; ``out``: an optional preallocated one, not ``seq_lens``, which
    later layers' calls still read).  ``last[b]`` outside ``[0, N)``, or a place
    without a draft: the path is empty, all places are dropped.  A sequence of fewer
    than N rows is left as it is.
    """
    return _ext().tree_cache_commit(cache, block_table, seq_lens, parents, last, out)


def tree_verify(target, tokens, parents, uniforms=None, draft=None, workspace=None):
    """The accepted path of a tree and the token after it; returns ``(last, next_token, accepted)``.

    ``target [B,N+1,V]`` (bf16, fp16 or fp32; V contiguous, other strides free): row 0
    belongs to the sequence's end, row i + 1 to place i; ``tokens`` int64 ``[B,N]``.
    ``last`` int32 ``[B]``: the last accepted place, -1 for none; ``next_token``
    int64 ``[B]``; ``accepted`` int32 ``[B]``: the path's length.

    ``uniforms`` None: greedy.  ``target`` holds scores of any kind; the walk goes
    on to the first child whose token is the row's largest (the lowest index where
    several are; NaN is never the largest).

    ``uniforms`` fp32 ``[B,N+1]`` in [0, 1): ``target`` holds probabilities.  Children
    are asked in the order of their indices; child i of token x is accepted if
    ``uniforms[i] q_i(x) Z < R(x)``, with R the row and Z = 1 at first; a refusal makes
    R ``max(R - Z q_i, 0)`` and Z its sum.  ``q_i``: ``draft[b, i]`` (``[B,N,V]`` in
    target's dtype), the distribution that the token was drawn from, or, without
    ``draft``, 1 at the token.  Where no child is left the next token is drawn from R
    with ``uniforms[N]``.  Accepted tokens and the next are then distributed as draws
    from the target.  Sums and comparisons are in 64 bits.  With ``draft`` the k-th refusal at
    a row reads k + 1 rows of V again: many refused children of one place are slow.  A row without any positive
    entry gives -1; a token outside [0, V) is never accepted.
    """
    return _ext().tree_verify(target, tokens, parents, uniforms, draft, workspace)
