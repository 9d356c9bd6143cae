"""Latent attention in float64 on the CPU: both forms, the gradient and the cache's append.

Plain restatements of the formulas, one head of one sequence at a time:

* expanded: ``s = scale (q_n k_n^T + q_r k_r^T)``, ``o = softmax(s) v``,
  ``lse = log sum exp s``; a row without a visible key has ``o = 0``, ``lse = -inf``;
* its gradient: ``D = sum do o``, ``p = exp(s - lse)``, ``g = scale p (do v^T - D)``,
  ``dq = g k``, ``dk = g^T q``, ``dv = p^T do``, the rotary key's summed over heads;
* absorbed: ``s = scale q row^T``, ``o = softmax(s) row[:, :R]``;
* append: ``x / sqrt(mean x^2 + eps) w`` and the rotation of pairs.
"""

from __future__ import annotations

import torch


def _softmax(s, ok):
    s = torch.where(ok, s, torch.full_like(s, float("-inf")))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    return torch.where(ok, p, torch.zeros_like(p)), lse


def attn(q, kv, k_rope, causal=True, scale=None, cu_q=None, cu_k=None, do=None):
    """``(o, lse)`` in float64, or ``(o, lse, dq, dkv, dk_rope)`` given the cotangent ``do``."""
    q, kv, kr = (x.detach().cpu().double() for x in (q, kv, k_rope))
    do = None if do is None else do.detach().cpu().double()
    B, Tq, H, _ = q.shape
    Tk, dn = kv.shape[1], kv.shape[3] // 2
    scale = q.shape[3] ** -0.5 if scale is None else scale
    o = torch.zeros(B, Tq, H, dn, dtype=torch.float64)
    lse = torch.full((B, H, Tq), float("-inf"), dtype=torch.float64)
    dq, dkv, dkr = torch.zeros_like(q), torch.zeros_like(kv), torch.zeros_like(kr)
    cu_q = [0, Tq] if cu_q is None else [int(x) for x in cu_q]
    cu_k = ([0, Tk] if len(cu_q) == 2 and cu_q[1] == Tq else cu_q) if cu_k is None else [int(x) for x in cu_k]
    for b in range(B):
        for i in range(len(cu_q) - 1):
            qs, ks = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
            nq, nk = cu_q[i + 1] - cu_q[i], cu_k[i + 1] - cu_k[i]
            if nq == 0 or nk == 0:
                continue
            ok = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                ok = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)
            for h in range(H):
                K = torch.cat([kv[b, ks, h, :dn], kr[b, ks]], 1)
                V, Q = kv[b, ks, h, dn:], q[b, qs, h]
                p, z = _softmax(scale * (Q @ K.T), ok)
                O = p @ V
                o[b, qs, h], lse[b, h, qs] = O, z
                if do is not None:
                    dO = do[b, qs, h]
                    g = scale * p * (dO @ V.T - (dO * O).sum(1, keepdim=True))
                    dK = g.T @ Q
                    dq[b, qs, h] = g @ K
                    dkv[b, ks, h] = torch.cat([dK[:, :dn], p.T @ dO], 1)
                    dkr[b, ks] += dK[:, dn:]
    return (o, lse) if do is None else (o, lse, dq, dkv, dkr)


def decode(q, cache, table, lens, R, scale):
    """``(o [B,Tq,H,R], lse [B,Tq,H])`` of the absorbed form in float64."""
    q = q.detach().cpu().double()
    B, Tq, H, W = q.shape
    page = cache.shape[1]
    o = torch.zeros(B, Tq, H, R, dtype=torch.float64)
    lse = torch.full((B, Tq, H), float("-inf"), dtype=torch.float64)
    table = table.cpu()
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        pages = table[b, :-(-n // page)].long().to(cache.device)
        rows = cache[pages].reshape(-1, W)[:n].cpu().double()
        for t in range(Tq):
            m = n - (Tq - 1 - t)
            if m > 0:
                p, lse[b, t] = _softmax(scale * (q[b, t] @ rows[:m].T), torch.ones(H, m, dtype=torch.bool))
                o[b, t] = p @ rows[:m, :R]
    return o, lse


def rotate(x, cos, sin, interleaved):
    """Pairs (a, b) of the last axis to (a cos - b sin, b cos + a sin)."""
    y = torch.empty_like(x)
    h = x.shape[-1] // 2
    ia = slice(0, None, 2) if interleaved else slice(0, h)
    ib = slice(1, None, 2) if interleaved else slice(h, None)
    y[..., ia] = x[..., ia] * cos - x[..., ib] * sin
    y[..., ib] = x[..., ib] * cos + x[..., ia] * sin
    return y


def append(rows, positions, slots, cos_sin, cache, w=None, eps=1e-6, q=None, interleaved=False):
    """``(cache, q_out)`` after the append, in float64; a slot outside the cache is not stored."""
    rows, cs = rows.detach().cpu().double(), cos_sin.cpu().double()
    dr = cs.shape[1]
    R = rows.shape[1] - dr
    flat = cache.detach().cpu().double().reshape(-1, R + dr).clone()
    pos = positions.cpu().clamp(0, cs.shape[0] - 1)
    cos, sin = cs[pos, :dr // 2], cs[pos, dr // 2:]
    c = rows[:, :R]
    if w is not None:
        c = c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * w.cpu().double()
    new = torch.cat([c, rotate(rows[:, R:], cos, sin, interleaved)], 1)
    for i, s in enumerate(slots.cpu().tolist()):
        if 0 <= s < flat.shape[0]:
            flat[s] = new[i]
    qo = None if q is None else rotate(q.detach().cpu().double(), cos[:, None], sin[:, None], interleaved)
    return flat.reshape(cache.shape), qo
