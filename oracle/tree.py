"""Trees of drafted tokens in float64 on the CPU, place by place from the definitions.

``parents[b][i]``: the place in ``[0, i)`` that place i continues, -1 the sequence, anything
else (or a place below such a one) no draft.
"""

from __future__ import annotations

import torch


def paths(parents):
    """``[b][i]``: the places on the way to place i, itself last; empty where it holds no draft."""
    out = []
    for row in (parents.tolist() if hasattr(parents, "tolist") else parents):
        got = []
        for i, p in enumerate(row):
            above = [] if p == -1 else got[p] if 0 <= p < i else None
            got.append([] if above is None or (p >= 0 and not above) else above + [i])
        out.append(got)
    return out


def step(q, k, v, g, beta, parents, state, scale=1.0):
    """``(o, u, states)``: the delta rule, one place after the other; states[b][i] after place i."""
    q, k, v, g, beta, state = (x.detach().cpu().double() for x in (q, k, v, g, beta, state))
    B, N, H, _ = q.shape
    o, u = torch.zeros_like(v), torch.zeros_like(v)
    states = []
    for b, row in enumerate(paths(parents)):
        after = {}
        for i, path in enumerate(row):
            if not path:
                continue
            S = after[path[-2]] if len(path) > 1 else state[b]
            S = torch.exp(g[b, i])[..., None] * S
            u[b, i] = beta[b, i, :, None] * (v[b, i] - torch.einsum("hkv,hk->hv", S, k[b, i]))
            S = S + k[b, i][..., None] * u[b, i][:, None]
            o[b, i] = scale * torch.einsum("hkv,hk->hv", S, q[b, i])
            after[i] = S
        states.append(after)
    return o, u, states


def decode(q, cache, table, lens, parents, R, scale):
    """``(o, lse)``: place i over the rows before the places' and those of its path that exist."""
    q, cache = q.detach().cpu().double(), cache.detach().cpu().double()
    B, N, H, W = q.shape
    page, cap = cache.shape[1], table.shape[1] * cache.shape[1]
    o = torch.zeros(B, N, H, R, dtype=torch.float64)
    lse = torch.full((B, N, H), float("-inf"), dtype=torch.float64)
    for b, row in enumerate(paths(parents)):
        n = min(max(int(lens[b]), 0), cap)
        for i, path in enumerate(row):
            toks = list(range(max(n - N, 0))) + [n - N + j for j in path if n - N + j >= 0]
            if not path or n - N + i < 0:
                continue
            t = torch.tensor(toks)
            k = cache[table[b].cpu().long()[t // page].clamp(0, cache.shape[0] - 1), t % page]
            s = scale * (q[b, i] @ k.T)
            lse[b, i] = torch.logsumexp(s, -1)
            o[b, i] = torch.softmax(s, -1) @ k[:, :R]
    return o, lse


def verify(target, tokens, parents, uniforms=None, draft=None):
    """``(last, next, accepted)`` as lists."""
    target = target.detach().cpu().double()
    draft = None if draft is None else draft.detach().cpu().double()
    u = None if uniforms is None else uniforms.detach().cpu().double()
    tokens, rows = tokens.tolist(), parents.tolist()
    B, N1, V = target.shape
    out = []
    for b, row in enumerate(paths(parents)):
        def best(r):
            x = torch.where(torch.isnan(target[b, r]), torch.tensor(float("-inf"), dtype=torch.float64), target[b, r])
            hit = torch.nonzero((target[b, r] == x.max()))
            return int(hit[0]) if len(hit) else 0

        cur, count = -1, 0
        R, Z = target[b, 0].clone(), 1.0
        for i in range(N1 - 1):
            if not row[i] or rows[b][i] != cur:
                continue
            x = tokens[b][i]
            inside = 0 <= x < V
            if u is None:
                ok = x == best(cur + 1)
            else:
                share = 1.0 if draft is None else float(draft[b, i, x]) if inside else 0.0
                ok = inside and float(u[b, i]) * share * Z < float(R[x])
            if ok:
                cur, count = i, count + 1
                R, Z = target[b, i + 1].clone(), 1.0
            elif u is not None and draft is not None:
                R = (R - Z * draft[b, i]).clamp_min(0)
                Z = float(R.sum())
            elif u is not None and inside:
                Z = max(Z - float(R[x]), 0.0)
                R[x] = 0.0
        if u is None:
            word = best(cur + 1)
        else:
            R = R.clamp_min(0)
            if not float(R.sum()) > 0:
                R = target[b, cur + 1].clamp_min(0)
            over = torch.nonzero(torch.cumsum(R, 0) > float(u[b, N1 - 1]) * float(R.sum()))
            some = torch.nonzero(R > 0)
            word = int(over[0]) if len(over) else int(some[-1]) if len(some) else -1
        out.append((cur, word, count))
    return [list(x) for x in zip(*out)] if out else [[], [], []]
