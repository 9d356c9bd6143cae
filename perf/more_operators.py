"""Trees of drafted tokens over KDA states and the latent cache: the calls of a serving program.

A program that drafts several tokens ahead lets the model look at all of them in one step and
keeps those that the model's own distribution allows. The drafts form a tree: node i continues
node ``parents[i] < i``, or the sequence itself (-1); any other entry marks a place that holds no
draft. Five operators of the package serve a step of such a program, and every case here is one
call of one of them:

* ``latent_tree_decode``: the latent layers, every node attending to the cache and its ancestors;
* ``kda_tree_step``: the KDA layers, every node's read-out of the state that its path leads to;
* ``tree_verify``: which path the target's distributions accept, from given random numbers;
* ``kda_tree_commit`` / ``latent_tree_commit``: states and caches after the accepted path.

``listed`` names the workloads, ``draw`` gives further ones of the same ranges, ``prepare``
makes a case's inputs on the GPU from a seed, ``run`` is one pass (in plain torch, or, where
``own`` is set, through the package), ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one request, eight drafts, early in its answer: latency
        dict(name="attn_b1_n8_t512", kind="attn", B=1, N=8, shape="tree", H=16, R=512, dr=64, page=64, lo=512, hi=512,
             lseed=0, dtype="bf16"),
        # a serving batch of requests of very different lengths, 16 places a request, not all of them used
        dict(name="attn_b32_n16_t8192", kind="attn", B=32, N=16, shape="tree", H=16, R=512, dr=64, page=64, lo=40, hi=8192,
             lseed=5, dtype="bf16"),
        # a few long contexts, many heads, an odd number of drafts
        dict(name="attn_b4_n25_h64_t32768", kind="attn", B=4, N=25, shape="tree", H=64, R=512, dr=64, page=32, lo=20000,
             hi=32768, lseed=7, dtype="fp16"),
        # a KDA layer of small heads in full precision: latency and the fp32 path
        dict(name="step_fp32_b2_n7", kind="step", B=2, N=7, shape="tree", H=4, d=64, lseed=1, dtype="fp32"),
        # the heads of the package's benchmark, one chain of drafts (a multi-token head's)
        dict(name="step_b8_n6_chain", kind="step", B=8, N=6, shape="chain", H=16, d=128, lseed=2, dtype="bf16"),
        # ... a serving batch with a tree a request
        dict(name="step_b64_n32", kind="step", B=64, N=32, shape="tree", H=16, d=128, lseed=3, dtype="bf16"),
        # the state after the accepted path: one request ...
        dict(name="state_b1_n8", kind="state", B=1, N=8, shape="tree", H=16, d=128, lseed=0, dtype="bf16"),
        # ... a serving batch
        dict(name="state_b64_n32", kind="state", B=64, N=32, shape="tree", H=16, d=128, lseed=3, dtype="bf16"),
        # the accepted rows of the cache move up: one layer of one request ...
        dict(name="cache_b1_n8", kind="cache", L=1, B=1, N=8, shape="tree", R=512, dr=64, page=64, lo=512, hi=512, lseed=0,
             dtype="bf16"),
        # ... eight layers of a large batch at once
        dict(name="cache_l8_b256_n64", kind="cache", L=8, B=256, N=64, shape="tree", R=512, dr=64, page=16, lo=64, hi=2000,
             lseed=4, dtype="bf16"),
        # greedy decoding: a chain against the logits, an odd vocabulary
        dict(name="greedy_b16_n8_v50021", kind="verify", B=16, N=8, shape="chain", V=50021, mode="greedy", lseed=2,
             dtype="bf16"),
        # sampling: trees against probabilities and the drafts' own
        dict(name="sample_b64_n16_v128000", kind="verify", B=64, N=16, shape="tree", V=128000, mode="drafts", lseed=6,
             dtype="fp32"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "step", "step", "state", "cache", "verify", "verify"])
    c = dict(kind=kind, N=_spread(rng, 1, 64), shape=rng.choice(["tree", "tree", "chain", "star"]), lseed=rng.randrange(1000),
             dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "attn":
        B, hi, H = _spread(rng, 1, 64), _spread(rng, 65, 32768), rng.choice([4, 8, 16, 16, 32, 64])
        hi = max(65, min(hi, (1 << 17) // B))
        c.update(R=rng.choice([512, 512, 256]), dr=rng.choice([64, 64, 32]), page=rng.choice([16, 32, 64, 128]))
        most = 1 << (25 if c["dtype"] == "fp32" else 27)          # rows times keys
        while B * hi * c["N"] * H > most:
            if H > 4:
                H //= 2
            elif B > 1:
                B //= 2
            else:
                hi = hi * 3 // 4
        hi = max(hi, c["N"])
        return dict(c, B=B, H=H, lo=max(c["N"], hi // rng.choice([1, 2, 50])), hi=hi)
    if kind in ("step", "state"):
        B, H = _spread(rng, 1, 64), rng.choice([2, 4, 8, 12, 16])
        while B * H * c["N"] > 1 << 15:
            B = B // 2
        return dict(c, B=max(1, B), H=H, d=rng.choice([64, 128, 128]))
    if kind == "cache":
        L, B = rng.choice([1, 2, 6]), _spread(rng, 1, 128)
        hi = max(65, min(_spread(rng, 65, 4000), (1 << 18) // (L * B)))
        return dict(c, L=L, B=B, R=rng.choice([512, 512, 256]), dr=rng.choice([64, 64, 32]),
                    page=rng.choice([16, 32, 64, 128]), lo=max(c["N"], hi // rng.choice([1, 2, 50])), hi=hi)
    B, V, N = _spread(rng, 1, 64), _spread(rng, 200, 160000), min(c["N"], 24)
    while B * (N + 1) * V > 1 << 27:
        B = B // 2
    return dict(c, N=N, B=max(1, B), V=V, mode=rng.choice(["greedy", "points", "drafts", "drafts"]))


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(n, lo, hi, lseed):
    """n lengths in [lo, hi], spread over their logarithm; they belong to the case, not to the seed."""
    u = torch.rand(n, generator=torch.Generator().manual_seed(1000 + int(lseed)))
    x = torch.exp(math.log(lo) + u * (math.log(hi + 1) - math.log(lo))).long().clamp(lo, hi)
    if n > 1:
        x[0] = hi
    return x


def _trees(c):
    """Parents of every sequence's places and the node that is accepted (-1: none), as lists.

    "chain": every node continues the one before; "star": all continue the sequence; "tree": a node
    continues one of the three before it or the sequence. In a batch some sequences use fewer places.
    """
    rng, N = random.Random(77 + c["lseed"]), c["N"]
    parents, last = [], []
    for b in range(c["B"]):
        n = N if b == 0 or N == 1 else rng.randint((N + 1) // 2, N)
        row = []
        for i in range(N):
            if i >= n:
                row.append(-2)
            elif c["shape"] == "chain":
                row.append(i - 1)
            elif c["shape"] == "star":
                row.append(-1)
            else:
                row.append(max(-1, i - rng.choice([1, 1, 2, 3])) if i > 2 else rng.choice([-1, i - 1]))
        parents.append(row)
        last.append(rng.randint(0, n - 1) if b == 0 else rng.randint(-1, n - 1))
    return parents, last


def _path(row, i):
    """The places on the way from the sequence to place i."""
    path = []
    while i >= 0:
        path.append(i)
        i = row[i]
    return path[::-1]


def _cache(c, gen, lens, layers=None):
    """A paged cache with its pages dealt out at random, and the block table."""
    R, dr, page, dt = c["R"], c["dr"], c["page"], DTYPES[c["dtype"]]
    per = -(-int(lens.max()) // page)
    used = (lens + page - 1) // page
    pages = int(used.sum()) + 1
    flat = torch.empty((layers or 1) * pages, page, R + dr, dtype=dt, device="cuda")
    for i in range(0, flat.shape[0], 4096):   # in pieces: the fp32 draw of a large cache is not kept
        part = flat[i:i + 4096]
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen))
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    col = torch.arange(per, device="cuda")[None]
    used = used.cuda()
    first = torch.cumsum(used, 0) - used
    at = (first[:, None] + col).clamp(max=pages - 1)
    table = torch.where(col < used[:, None], order[at], torch.zeros_like(order[at]))
    return (flat.view(layers, pages, page, R + dr) if layers else flat), table


def prepare(case, seed):
    c, gen, dt = case, _gen(seed), DTYPES[case["dtype"]]
    B, N = c["B"], c["N"]
    parents, last = _trees(c)
    s = dict(kind=c["kind"], parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if c["kind"] == "attn":
        lens = _lengths(B, c["lo"], c["hi"], c["lseed"])
        s["cache"], s["table"] = _cache(c, gen, lens)
        s["q"] = (randn(B, N, c["H"], c["R"] + c["dr"]) * 0.8).to(dt)
        s["lens"], s["R"], s["scale"] = lens.int().cuda(), c["R"], (128 + c["dr"]) ** -0.5
        return s
    if c["kind"] == "cache":
        lens = _lengths(B, c["lo"], c["hi"], c["lseed"])
        s["cache"], s["table"] = _cache(c, gen, lens, c["L"])
        s["lens"], s["last"] = lens.int().cuda(), torch.tensor(last, dtype=torch.int32, device="cuda")
        return s
    if c["kind"] in ("step", "state"):
        H, d = c["H"], c["d"]
        q, k = randn(B, N, H, d), randn(B, N, H, d)
        s["q"], s["k"] = (q / q.norm(dim=-1, keepdim=True)).to(dt), (k / k.norm(dim=-1, keepdim=True)).to(dt)
        # log-decays: a rate a head, from slow to several hundredths a token
        rate = torch.exp(-2 * torch.rand(H, device="cuda", generator=gen))[:, None]
        s["g"] = (-torch.nn.functional.softplus(randn(B, N, H, d)) * rate).to(dt)
        s["state"] = 0.1 * randn(B, H, d, d)
        if c["kind"] == "step":
            s["v"], s["beta"] = randn(B, N, H, d).to(dt), torch.sigmoid(randn(B, N, H)).to(dt)
        else:
            s["u"], s["last"] = randn(B, N, H, d), torch.tensor(last, dtype=torch.int32, device="cuda")
        return s

    # verify: the drafting model's logits are the target's with an error
    V, mode = c["V"], c["mode"]
    at = (s["parents"].long() + 1).clamp(min=0)                         # the row a node's token was drawn at
    s["mode"] = mode
    logits = randn(B, N + 1, V) * 2.5
    if mode == "greedy":
        s["target"] = logits.to(dt)
        best = s["target"].float().argmax(-1).gather(1, at)
        off = torch.rand(B, N, device="cuda", generator=gen) < 0.2
        s["tokens"] = torch.where(off, torch.randint(0, V, (B, N), device="cuda", generator=gen), best)
        s["draft"] = s["uniforms"] = None
        return s
    s["target"] = torch.softmax(logits, -1).to(dt)
    logits += 0.5 * randn(B, N + 1, V)
    proposed = torch.softmax(logits, -1)
    s["tokens"] = torch.empty(B, N, dtype=torch.int64, device="cuda")
    for i in range(N):                                                  # Gumbel's maximum draws from the proposed row
        noise = -torch.log(-torch.log(torch.rand(B, V, device="cuda", generator=gen).clamp(1e-20, 1 - 1e-7)))
        rows = logits.gather(1, at[:, i, None, None].expand(B, 1, V))[:, 0]
        s["tokens"][:, i] = (rows + noise).argmax(-1)
    s["draft"] = None
    if mode == "drafts":
        s["draft"] = proposed.gather(1, at[:, :, None].expand(B, N, V)).to(dt)
    s["uniforms"] = torch.rand(B, N + 1, device="cuda", generator=gen)
    return s


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _ancestors(parents):
    """[B,N,N] truth values: j is i or one of its ancestors; nothing for a place that holds no draft."""
    B, N = parents.shape
    seen = torch.zeros(B, N, N, dtype=torch.bool, device=parents.device)
    eye = torch.eye(N, dtype=torch.bool, device=parents.device)
    p = parents.long()
    b = torch.arange(B, device=parents.device)
    for i in range(N):
        root, inner = p[:, i] == -1, (p[:, i] >= 0) & (p[:, i] < i)
        up = seen[b, p[:, i].clamp(0, N - 1)]
        live = root | (inner & up.any(-1))
        seen[:, i] = live[:, None] & ((up & inner[:, None]) | eye[i])
    return seen


def _plain_attn(s):
    B, N, H, W = s["q"].shape
    page, per, R = s["cache"].shape[1], s["table"].shape[1], s["R"]
    k = s["cache"][s["table"].long()].view(B, per * page, W).float()
    sc = torch.matmul(s["q"].float().view(B, N * H, W), k.transpose(-1, -2).contiguous()) * s["scale"]
    base = (s["lens"] - N).long()
    j = torch.arange(per * page, device="cuda")[None] - base[:, None]    # which place a row holds
    seen = _ancestors(s["parents"])
    live = seen.any(-1)
    inner = seen.gather(2, j.clamp(0, N - 1)[:, None].expand(B, N, -1)) & ((j >= 0) & (j < N))[:, None]
    ok = (live[..., None] & (j < 0)[:, None]) | inner
    sc = sc.view(B, N, H, -1).masked_fill_(~ok[:, :, None], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(sc.sub_(m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, N * H, -1), k[..., :R].contiguous()).view(B, N, H, -1) / l.clamp_min(1e-38)
    return o.to(s["q"].dtype), (m + torch.log(l))[..., 0]


def _plain_step(s):
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "g", "beta"))
    B, N, H, d = q.shape
    par, b = s["parents"].long(), torch.arange(B, device="cuda")
    live = _ancestors(s["parents"]).any(-1)
    states = torch.empty(N + 1, B, *s["state"].shape[1:], device="cuda")     # before all nodes, after each
    states[0] = s["state"]
    o, u = torch.zeros_like(v), torch.zeros_like(v)
    for i in range(N):
        S = states[(par[:, i] + 1).clamp(0, i), b] * torch.exp(g[:, i])[..., None]
        new = beta[:, i, :, None] * (v[:, i] - (S * k[:, i, ..., None]).sum(-2))
        S = S + k[:, i, ..., None] * new[..., None, :]
        states[i + 1] = S
        on = live[:, i, None, None]
        u[:, i] = torch.where(on, new, u[:, i])
        o[:, i] = torch.where(on, (S * q[:, i, ..., None]).sum(-2), o[:, i])
    return o, u


def _plain_state(s):
    k, g = s["k"].float(), s["g"].float()
    B, N, H, d = k.shape
    seen = _ancestors(s["parents"])
    on = seen[torch.arange(B, device="cuda"), s["last"].long().clamp(0)] & (s["last"] >= 0)[:, None]   # [B,N]: on the path
    S = s["state"]
    for i in range(N):
        step = on[:, i, None, None, None]
        S = torch.where(step, S * torch.exp(g[:, i])[..., None] + k[:, i, ..., None] * s["u"][:, i, :, None], S)
    s["state"].copy_(S)
    return s["state"]


def _plain_cache(s):
    B, N = s["parents"].shape
    L, pages, page, W = s["cache"].shape
    seen = _ancestors(s["parents"])
    on = seen[torch.arange(B, device="cuda"), s["last"].long().clamp(0)] & (s["last"] >= 0)[:, None]
    base = (s["lens"] - N).long()
    place = torch.arange(N, device="cuda")[None].expand(B, N)
    to = torch.where(on, torch.cumsum(on, 1) - 1, place)                   # where a place's row goes

    def slot(x):
        tok = base[:, None] + x
        return (s["table"].long().gather(1, tok // page) * page + tok % page)[on]

    flat = s["cache"].view(L, pages * page, W)
    flat[:, slot(to)] = flat[:, slot(place)]
    return s["cache"], (base + on.sum(1)).int()


def _lowest_best(rows):
    """Index of the largest value of every row, the lowest where several are."""
    at = torch.arange(rows.shape[-1], device=rows.device)
    return torch.where(rows == rows.amax(-1, keepdim=True), at, rows.shape[-1]).amin(-1)


def _plain_verify(s):
    target, tokens, par = s["target"], s["tokens"], s["parents"].long()
    B, N1, V = target.shape
    N, b = N1 - 1, torch.arange(B, device="cuda")
    cur = torch.full((B,), -1, dtype=torch.int64, device="cuda")
    count = torch.zeros_like(cur)
    if s["uniforms"] is None:
        best = _lowest_best(target)
        for i in range(N):
            ok = (par[:, i] == cur) & (tokens[:, i] == best[b, cur + 1])
            cur, count = torch.where(ok, i, cur), count + ok
        return cur.int(), best[b, cur + 1], count.int()
    # weights, their sum and products in 64 bits: a decision next to its border is the same in any order of sums
    uni = s["uniforms"].double()
    R, Z = target[:, 0].double(), torch.ones(B, dtype=torch.float64, device="cuda")
    for i in range(N):
        asked = par[:, i] == cur
        r = R[b, tokens[:, i]]
        q = s["draft"][:, i].double() if s["draft"] is not None else None
        qx = q[b, tokens[:, i]] if q is not None else 1.0
        ok = asked & (uni[:, i] * qx * Z < r)
        no = asked & ~ok
        if q is not None:
            R2 = (R - Z[:, None] * q).clamp_min(0)
            Z2 = R2.sum(-1)
        else:
            R2 = R.clone()
            R2[b, tokens[:, i]] = 0
            Z2 = (Z - r).clamp_min(0)
        R, Z = torch.where(no[:, None], R2, R), torch.where(no, Z2, Z)
        cur, count = torch.where(ok, i, cur), count + ok
        R, Z = torch.where(ok[:, None], target[:, i + 1].double(), R), torch.where(ok, 1.0, Z)
    W = R.sum(-1, keepdim=True)
    R = torch.where(W > 0, R, target[b, cur + 1].double())
    total = torch.cumsum(R, -1)
    over = total > uni[:, N, None] * R.sum(-1, keepdim=True)
    at = torch.arange(V, device="cuda")
    first = torch.where(over, at, V).amin(-1)
    final = torch.where(R > 0, at, -1).amax(-1)
    return cur.int(), torch.where(first < V, first, final), count.int()


_plain = dict(attn=_plain_attn, step=_plain_step, state=_plain_state, cache=_plain_cache, verify=_plain_verify)


def _own_attn(s):
    import axiom_amd
    return axiom_amd.latent_tree_decode(s["q"], s["cache"], s["table"], s["lens"], s["parents"], scale=s["scale"])


def _own_step(s):
    import axiom_amd
    return axiom_amd.kda_tree_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["parents"], s["state"])


def _own_state(s):
    import axiom_amd
    return axiom_amd.kda_tree_commit(s["k"], s["g"], s["u"], s["parents"], s["last"], s["state"])


def _own_cache(s):
    import axiom_amd
    return s["cache"], axiom_amd.latent_tree_commit(s["cache"], s["table"], s["lens"], s["parents"], s["last"])


def _own_verify(s):
    import axiom_amd
    return axiom_amd.tree_verify(s["target"], s["tokens"], s["parents"], uniforms=s["uniforms"], draft=s["draft"])


_own = dict(attn=_own_attn, step=_own_step, state=_own_state, cache=_own_cache, verify=_own_verify)


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    parents, last = _trees(case)
    paths = [[_path(row, i) if row[i] >= -1 else [] for i in range(len(row))] for row in parents]
    return dict(attn=_exact_attn, step=_exact_step, state=_exact_state, cache=_exact_cache,
                verify=_exact_verify)[case["kind"]](s, paths, last)


def _exact_attn(s, paths, last):
    q, R = s["q"].double(), s["R"]
    B, N, H, W = q.shape
    page = s["cache"].shape[1]
    o = torch.zeros(B, N, H, R, dtype=torch.float64, device="cuda")
    lse = torch.full((B, N, H), float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        k = s["cache"][s["table"][b, :-(-n // page)].long()].reshape(-1, W)[:n].double()
        old = s["scale"] * (q[b].reshape(N * H, W) @ k[:n - N].T).view(N, H, n - N)
        for i, path in enumerate(paths[b]):
            if path:
                rows = k[n - N:][path]
                sc = torch.cat([old[i], s["scale"] * (q[b, i] @ rows.T)], 1)
                lse[b, i] = torch.logsumexp(sc, -1)
                p = torch.softmax(sc, -1)
                o[b, i] = p[:, :n - N] @ k[:n - N, :R] + p[:, n - N:] @ rows[:, :R]
    return o, lse


def _exact_step(s, paths, last):
    """By the triangular system: u = beta (v - decayed reads of the state - sum over ancestors)."""
    B, N, H, d = s["q"].shape
    o = torch.zeros(B, N, H, d, dtype=torch.float64, device="cuda")
    u = torch.zeros_like(o)
    for b in range(B):
        up = torch.zeros(N, N, dtype=torch.float64)
        for i, path in enumerate(paths[b]):
            up[i, path] = 1
        up = up.cuda()
        q, k, v, g, beta = (s[n][b].double().transpose(0, 1) for n in ("q", "k", "v", "g", "beta"))   # [H,N,...]
        G = torch.matmul(up, g)                                                        # decay along the path
        fade = torch.exp((G[:, :, None] - G[:, None]).clamp(max=0)) * k[:, None]       # [H,i,j,d]
        A = torch.matmul(fade, q[..., None])[..., 0] * up
        K = torch.matmul(fade, k[..., None])[..., 0] * (up - torch.diag(torch.diag(up)))
        S = s["state"][b].double()
        on = torch.diag(up)[None, :, None]
        rhs = beta[..., None] * (v - torch.matmul(torch.exp(G) * k, S)) * on
        x = torch.linalg.solve_triangular(torch.eye(N, device="cuda", dtype=torch.float64) + beta[..., None] * K, rhs, upper=False,
                                          unitriangular=True)
        u[b] = x.transpose(0, 1)
        o[b] = (torch.matmul(torch.exp(G) * q, S) * on + torch.matmul(A, x)).transpose(0, 1)
    return o, u


def _exact_state(s, paths, last):
    S = s["state"].double()
    for b, i in enumerate(last):
        if i >= 0:
            path = paths[b][i]
            g, k, u = (s[n][b, path].double() for n in ("g", "k", "u"))          # [m,H,d]
            after = g.flip(0).cumsum(0).flip(0) - g                              # decay behind each token
            S[b] = torch.exp(g.sum(0))[..., None] * S[b] + torch.einsum("mhk,mhv->hkv", torch.exp(after) * k, u)
    return S


def _exact_cache(s, paths, last):
    cache, lens, page = s["cache"].double(), s["lens"].tolist(), s["cache"].shape[2]
    N = s["parents"].shape[1]
    old, table = cache.clone(), s["table"].tolist()
    new = []
    for b, i in enumerate(last):
        path = paths[b][i] if i >= 0 else []
        for to, at in enumerate(path):
            x, y = lens[b] - N + to, lens[b] - N + at
            cache[:, table[b][x // page], x % page] = old[:, table[b][y // page], y % page]
        new.append(lens[b] - N + len(path))
    return cache, torch.tensor(new, dtype=torch.int32, device="cuda")


def _exact_verify(s, paths, last):
    target, tokens, uni, draft = s["target"], s["tokens"].tolist(), s["uniforms"], s["draft"]
    parents = s["parents"].tolist()
    B, N = len(tokens), len(tokens[0])
    out = []
    for b in range(B):
        cur, count, i = -1, 0, 0
        if uni is None:
            word = int(_lowest_best(target[b, 0].double()))
        else:
            weight, total = target[b, 0].double(), 1.0
        for i in range(N):
            if parents[b][i] != cur:
                continue
            x = tokens[b][i]
            if uni is None:
                ok = x == word
            else:
                share = float(draft[b, i, x]) if draft is not None else 1.0
                ok = float(uni[b, i]) * share * total < float(weight[x])
            if ok:
                cur, count = i, count + 1
                if uni is None:
                    word = int(_lowest_best(target[b, i + 1].double()))
                else:
                    weight, total = target[b, i + 1].double(), 1.0
            elif uni is not None and draft is not None:
                weight = torch.relu(weight - total * draft[b, i].double())
                total = float(weight.sum())
            elif uni is not None:
                total = max(0.0, total - float(weight[x]))
                weight = weight.clone()
                weight[x] = 0
        if uni is not None:
            if not float(weight.sum()) > 0:
                weight = target[b, cur + 1].double()
            over = torch.nonzero(weight.cumsum(0) > float(uni[b, N]) * weight.sum())
            word = int(over[0]) if len(over) else int(torch.nonzero(weight > 0)[-1])
        out.append((cur, word, count))
    a = torch.tensor(out, dtype=torch.int64, device="cuda")
    return a[:, 0].int(), a[:, 1], a[:, 2].int()


# ---------------------------------------------------------------------------------------------- cost

def work(case):
    c, es = case, 4 if case["dtype"] == "fp32" else 2
    B, N = c["B"], c["N"]
    parents, last = _trees(c)
    pairs = sum(len(_path(row, i)) for row in parents for i in range(N) if row[i] >= -1)
    moved = sum(len(_path(row, i)) for row, i in zip(parents, last))
    if c["kind"] == "attn":
        R, dr, H = c["R"], c["dr"], c["H"]
        lens = _lengths(B, c["lo"], c["hi"], c["lseed"]).tolist()
        nodes = sum((n - N) * sum(p >= -1 for p in row) for n, row in zip(lens, parents)) + pairs
        return {"bytes": es * (sum(lens) * (R + dr) + B * N * H * (2 * R + dr)) + 4 * B * N * H, "flops": 2 * nodes * H * (2 * R + dr)}
    if c["kind"] == "step":   # state in; q, k, v, g, beta in; o and u out
        H, d = c["H"], c["d"]
        return {"bytes": B * H * (4 * d * d + N * (es * (4 * d + 1) + 8 * d)), "flops": H * (4 * B * N * d * d + 8 * pairs * d)}
    if c["kind"] == "state":   # state in and out; the path's k, g, u
        H, d = c["H"], c["d"]
        return {"bytes": H * (8 * B * d * d + moved * d * (2 * es + 4)), "flops": H * d * d * (B + 2 * moved)}
    if c["kind"] == "cache":
        return {"bytes": 2 * es * c["L"] * moved * (c["R"] + c["dr"]) + 8 * B, "flops": moved}
    rows = 2 if c["mode"] == "drafts" else 1   # the row of the last token's own draw, and the draft's it left
    return {"bytes": B * c["V"] * es * rows + B * N * 20, "flops": 3 * B * c["V"] * rows}
