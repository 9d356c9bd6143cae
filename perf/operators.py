"""Latent attention and its cache: the calls of a serving or training program, at the sizes it makes them.

A latent-attention layer keeps one latent vector and one rotated key part a token. Three
operators of the package serve it, and every case here is one call of one of them:

* ``latent_attn`` / ``latent_attn_fwd``: the expanded form (prompts, training), on the
  up-projected keys and values and the rotary key that all heads share;
* ``latent_append``: norm and rotation of new tokens' latents, stored in a paged cache,
  with the rotation of the queries;
* ``latent_decode``: the absorbed form, one to a few query tokens over the paged cache.

``listed`` names the workloads, ``draw`` gives further ones of the same ranges, ``prepare``
makes a case's inputs on the GPU from a seed, ``run`` is one pass (in plain torch in 32 bits,
or, where ``own`` is set, through the package), ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # a short prompt in full precision with small heads: latency and the fp32 path
        dict(name="prefill_fp32_t512", kind="prefill", B=1, Tq=512, Tk=512, H=4, dn=64, dr=32, dtype="fp32", causal=True),
        # the next piece of a prompt over what was read before it, a ragged length
        dict(name="prefill_t333_after_1000", kind="prefill", B=1, Tq=333, Tk=1333, H=16, dn=128, dr=64, dtype="bf16",
             causal=True),
        # one long document
        dict(name="prefill_t16384", kind="prefill", B=1, Tq=16384, Tk=16384, H=16, dn=128, dr=64, dtype="bf16", causal=True),
        # packed prompts of very different lengths
        dict(name="packed_24", kind="packed", N=24, lo=17, hi=1024, lseed=3, H=8, dn=128, dr=64, dtype="fp16"),
        # training steps: a small ragged batch with small heads ...
        dict(name="train_d64_t1000", kind="train", B=2, T=1000, H=8, dn=64, dr=32, dtype="bf16", causal=True),
        # ... in full precision (gradient checks, fp32 training)
        dict(name="train_fp32_t1024", kind="train", B=1, T=1024, H=8, dn=128, dr=64, dtype="fp32", causal=True),
        # ... the batch, length and heads of the package's benchmark
        dict(name="train_b4_t4096", kind="train", B=4, T=4096, H=16, dn=128, dr=64, dtype="bf16", causal=True),
        # one generated token of one request: the latency of the smallest call
        dict(name="append_b1", kind="append", N=1, H=16, R=512, dr=64, page=64, dtype="bf16", interleaved=False),
        # a batch of prompts going into the cache, padding rows among them
        dict(name="append_n16384", kind="append", N=16384, H=16, R=512, dr=64, page=64, dtype="bf16", interleaved=True),
        # one request early in its answer
        dict(name="decode_b1_t512", kind="decode", B=1, Tq=1, H=16, R=512, dr=64, page=64, lo=512, hi=512, lseed=0, dtype="bf16"),
        # a serving batch of requests of very different lengths
        dict(name="decode_b64_t8192", kind="decode", B=64, Tq=1, H=16, R=512, dr=64, page=64, lo=1, hi=8192, lseed=5,
             dtype="bf16"),
        # a few long contexts, many heads, two tokens to verify at a time
        dict(name="decode_b8_h64_t32768", kind="decode", B=8, Tq=2, H=64, R=512, dr=64, page=32, lo=20000, hi=32768, lseed=7,
             dtype="fp16"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "packed", "train", "train", "append", "decode", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dn, dr = rng.choice([(64, 32), (128, 64), (128, 64), (128, 32), (64, 64)])
    H = rng.choice([2, 4, 8, 12, 16, 24])
    if kind == "prefill":
        B = _spread(rng, 1, 8)
        Tq = _spread(rng, 1, 8192)
        Tk = Tq + rng.choice([0, 0, _spread(rng, 1, 4096)])
        while B * H * Tq * Tk > 1 << 30:
            B, H, Tq, Tk = max(1, B // 2), max(2, H // 2), Tq - Tq // 5, Tk - Tk // 5
        return dict(kind=kind, B=B, Tq=Tq, Tk=max(Tq, Tk), H=H, dn=dn, dr=dr, dtype=dtype, causal=rng.random() < 0.8)
    if kind == "packed":
        lo = _spread(rng, 1, 200)
        return dict(kind=kind, N=_spread(rng, 2, 32), lo=lo, hi=lo + _spread(rng, 8, 300), lseed=rng.randrange(1000),
                    H=rng.choice([2, 4, 8]), dn=dn, dr=dr, dtype=dtype)
    if kind == "train":
        B, T = _spread(rng, 1, 4), _spread(rng, 17, 4096)
        while B * H * T * T > 1 << (28 if dtype == "fp32" else 29):
            B, T = max(1, B // 2), T - T // 5
        return dict(kind=kind, B=B, T=T, H=H, dn=dn, dr=dr, dtype=dtype, causal=rng.random() < 0.8)
    R, dr, page = rng.choice([512, 512, 256]), rng.choice([64, 64, 32]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        return dict(kind=kind, N=_spread(rng, 1, 12000), H=rng.choice([4, 8, 12, 16]), R=R, dr=dr, page=page, dtype=dtype,
                    interleaved=rng.random() < 0.5)
    B, hi = _spread(rng, 1, 256), _spread(rng, 1, 32768)
    hi = max(1, min(hi, (1 << 18) // B))
    H, Tq = rng.choice([4, 8, 16, 16, 32, 64, 128]), rng.choice([1, 1, 1, 2, 3, 4])
    while H * Tq > 128:
        H //= 2
    return dict(kind=kind, B=B, Tq=Tq, H=H, R=R, dr=dr, page=page, lo=max(1, hi // rng.choice([1, 2, 50])), hi=hi,
                lseed=rng.randrange(1000), dtype=dtype)


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


def _offsets(c):
    lens = _lengths(c["N"], c["lo"], c["hi"], c["lseed"])
    return [0] + torch.cumsum(lens, 0).tolist()


def prepare(case, seed):
    c, gen, dt = case, _gen(seed), DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if c["kind"] in ("prefill", "packed", "train"):
        if c["kind"] == "packed":
            offs = _offsets(c)
            B, Tq, Tk = 1, offs[-1], offs[-1]
        else:
            B, Tq, Tk = c["B"], c.get("Tq", c.get("T")), c.get("Tk", c.get("T"))
        H, dn, dr = c["H"], c["dn"], c["dr"]
        s = dict(kind=c["kind"], causal=c.get("causal", True), scale=(dn + dr) ** -0.5, dn=dn, dr=dr, cu=None)
        # queries somewhat larger than unit normal: softmax rows between flat and a few leading keys
        s["q"] = (randn(B, Tq, H, dn + dr) * 1.5).to(dt)
        s["kv"] = randn(B, Tk, H, 2 * dn).to(dt)
        # the rotary key is the tail of the down-projection's row, as the layer has it
        s["kr"] = randn(B, Tk, 4 * dn + dr).to(dt)[..., 4 * dn:]
        if c["kind"] == "packed":
            s["cu"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
        if c["kind"] == "train":
            s["kr"] = s["kr"].contiguous()
            s["do"] = randn(B, Tq, H, dn).to(dt)
            for n in ("q", "kv", "kr"):
                s[n].requires_grad_(True)
        return s

    R, dr, page, H = c["R"], c["dr"], c["page"], c["H"]
    if c["kind"] == "append":
        N = c["N"]
        pages = 2 * -(-N // page) + 1
        s = dict(kind="append", R=R, dr=dr, interleaved=c["interleaved"])
        s["cache"] = randn(pages, page, R + dr).to(dt)
        s["rows"] = randn(N, R + dr).to(dt) * 0.7
        s["weight"] = 1 + 0.1 * randn(R)
        s["q"] = randn(N, H, 128 + dr).to(dt)
        s["q_abs"] = torch.zeros(N, H, R + dr, dtype=dt, device="cuda")
        s["positions"] = torch.randint(0, 32768, (N,), device="cuda", generator=gen)
        s["slots"] = torch.randperm(pages * page, device="cuda", generator=gen)[:N]
        # some rows of a batch are padding; the program knows which
        pad = torch.arange(N, device="cuda") % 37 == 36
        s["slots"][pad] = -1
        s["real"] = torch.nonzero(~pad)[:, 0]
        f = 10000.0 ** (-torch.arange(0, dr, 2, device="cuda", dtype=torch.float64) / dr)
        a = torch.arange(32768, device="cuda", dtype=torch.float64)[:, None] * f[None]
        s["cos_sin"] = torch.cat([a.cos(), a.sin()], 1).float()
        return s

    B, Tq = c["B"], c["Tq"]
    lens = _lengths(B, c["lo"], c["hi"], c["lseed"])
    per = -(-int(lens.max()) // page)
    used = (lens + page - 1) // page
    pages = int(used.sum()) + 1
    s = dict(kind="decode", R=R, scale=(128 + dr) ** -0.5)
    s["cache"] = torch.empty(pages, page, R + dr, dtype=dt, device="cuda")
    for i in range(0, pages, 4096):   # in pieces: the fp32 draw of a large cache is not kept
        s["cache"][i:i + 4096] = randn(min(4096, pages - i), page, R + dr)
    s["q"] = (randn(B, Tq, H, R + dr) * 0.8).to(dt)
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    table = torch.zeros(B, per, dtype=torch.int32, device="cuda")
    col = torch.arange(per, device="cuda")[None]
    used = used.cuda()
    first = torch.cumsum(used, 0) - used
    at = (first[:, None] + col).clamp(max=pages - 1)
    table[:] = torch.where(col < used[:, None], order[at], table)
    s["table"] = table
    s["lens"] = lens.int().cuda()
    return s


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _allowed(s, Tq, Tk):
    """[Tq, Tk] truth values: the pairs that a query sees."""
    i = torch.arange(Tq, device="cuda")[:, None]
    j = torch.arange(Tk, device="cuda")[None]
    ok = (j <= i + (Tk - Tq)) if s["causal"] else torch.ones(Tq, Tk, dtype=torch.bool, device="cuda")
    if s["cu"] is not None:
        inner = s["cu"][1:-1].long()
        ok = ok & ((i >= inner[:, None, None]).sum(0) == (j >= inner[:, None, None]).sum(0))
    return ok


def _plain_parts(s):
    """fp32 q_nope, q_rope, k_nope, v [B,H,T,d] and k_rope [B,1,T,dr]."""
    dn = s["dn"]
    q, kv = s["q"].detach().float().transpose(1, 2), s["kv"].detach().float().transpose(1, 2)
    return q[..., :dn], q[..., dn:], kv[..., :dn], kv[..., dn:], s["kr"].detach().float()[:, None]


def _plain_scores(s, qn, qr, kn, kr):
    sc = torch.matmul(qn, kn.transpose(-1, -2))
    sc += torch.matmul(qr, kr.transpose(-1, -2))
    sc *= s["scale"]
    sc.masked_fill_(~_allowed(s, qn.shape[2], kn.shape[2]), float("-inf"))
    return sc


def _plain_prefill(s):
    qn, qr, kn, v, kr = _plain_parts(s)
    sc = _plain_scores(s, qn, qr, kn, kr)
    m = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(sc.sub_(m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / l.clamp_min(1e-38)
    return o.transpose(1, 2).to(s["q"].dtype).contiguous(), (m + torch.log(l))[..., 0]


def _plain_train(s):
    qn, qr, kn, v, kr = _plain_parts(s)
    p = _plain_scores(s, qn, qr, kn, kr)
    p = torch.exp(p.sub_(p.amax(-1, keepdim=True).clamp_min(-3e38)))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(p, v)
    do = s["do"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (do * o).sum(-1, keepdim=True)
    ds *= p
    ds *= s["scale"]
    dq = torch.cat([torch.matmul(ds, kn), torch.matmul(ds, kr)], -1)
    dsT = ds.transpose(-1, -2)
    dkv = torch.cat([torch.matmul(dsT, qn), dv], -1)
    dkr = torch.matmul(dsT, qr).sum(1)
    dt = s["q"].dtype
    return [o.transpose(1, 2).to(dt).contiguous(), dq.transpose(1, 2).to(dt).contiguous(),
            dkv.transpose(1, 2).to(dt).contiguous(), dkr.to(dt)]


def _plain_rotate(x, cs, interleaved):
    h = x.shape[-1] // 2
    cos, sin = cs[..., :h], cs[..., h:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :h], x[..., h:])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)


def _plain_append(s):
    R, dt = s["R"], s["cache"].dtype
    x, cs = s["rows"].float(), s["cos_sin"][s["positions"]]
    c = x[:, :R]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s["weight"]
    row = torch.cat([c, _plain_rotate(x[:, R:], cs, s["interleaved"])], -1).to(dt)
    s["cache"].view(-1, row.shape[1])[s["slots"][s["real"]]] = row[s["real"]]
    s["q_abs"][..., R:] = _plain_rotate(s["q"][..., 128:].float(), cs[:, None], s["interleaved"]).to(dt)
    return [s["cache"], s["q_abs"][..., R:]]


def _plain_decode(s):
    B, Tq, H, W = s["q"].shape
    page, per = s["cache"].shape[1], s["table"].shape[1]
    k = s["cache"][s["table"].long()].view(B, per * page, W).float()
    sc = torch.matmul(s["q"].float().view(B, Tq * H, W), k.transpose(-1, -2)) * s["scale"]
    t = torch.arange(Tq, device="cuda")
    seen = s["lens"][:, None] - (Tq - 1 - t)[None]
    ok = torch.arange(per * page, device="cuda")[None, None] < seen[..., None]
    sc = sc.view(B, Tq, H, -1).masked_fill_(~ok[:, :, None], float("-inf"))
    m = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(sc.sub_(m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Tq * H, -1), k[..., :s["R"]]).view(B, Tq, H, -1) / l.clamp_min(1e-38)
    return o.to(s["q"].dtype), (m + torch.log(l))[..., 0]


_plain = dict(prefill=_plain_prefill, packed=_plain_prefill, train=_plain_train, append=_plain_append, decode=_plain_decode)


def _own_prefill(s):
    import axiom_amd
    return axiom_amd.latent_attn_fwd(s["q"], s["kv"], s["kr"], cu_seqlens=s["cu"], causal=s["causal"], scale=s["scale"])


def _own_train(s):
    import axiom_amd
    o = axiom_amd.latent_attn(s["q"], s["kv"], s["kr"], causal=s["causal"], scale=s["scale"])
    return [o.detach(), *torch.autograd.grad(o, (s["q"], s["kv"], s["kr"]), s["do"])]


def _own_append(s):
    import axiom_amd
    q_out = s["q_abs"][..., s["R"]:]
    axiom_amd.latent_append(s["rows"], s["positions"], s["slots"], s["cos_sin"], s["cache"], norm_weight=s["weight"], eps=EPS,
                            q_rope=s["q"][..., 128:], q_out=q_out, interleaved=s["interleaved"])
    return [s["cache"], q_out]


def _own_decode(s):
    import axiom_amd
    return axiom_amd.latent_decode(s["q"], s["cache"], s["table"], s["lens"], scale=s["scale"])


_own = dict(prefill=_own_prefill, packed=_own_prefill, train=_own_train, append=_own_append, decode=_own_decode)


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["kind"] == "append":
            return _exact_append(s)
        if s["kind"] == "decode":
            return _exact_decode(s)
        return _exact_attn(s)


def _softmax64(sc, ok):
    """Probabilities and log-sum-exp of the allowed scores; a row with none: zeros and -inf."""
    sc = torch.where(ok, sc, torch.full_like(sc, float("-inf")))
    lse = torch.logsumexp(sc, -1)
    return torch.where(ok, torch.exp(sc - torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))[..., None]),
                       torch.zeros_like(sc)), lse


def _exact_attn(s):
    q, kv, kr, dn = s["q"].double(), s["kv"].double(), s["kr"].double(), s["dn"]
    B, Tq, H, _ = q.shape
    Tk = kv.shape[1]
    o = torch.zeros(B, Tq, H, dn, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, Tq), float("-inf"), dtype=torch.float64, device="cuda")
    train = s["kind"] == "train"
    dq, dkv, dkr = torch.zeros_like(q), torch.zeros_like(kv), torch.zeros_like(kr)
    offs = [0, Tq] if s["cu"] is None else s["cu"].tolist()
    for b in range(B):
        for a, e in zip(offs[:-1], offs[1:]):
            ka, ke = (a, e) if s["cu"] is not None else (0, Tk)
            i = torch.arange(e - a, device="cuda")[:, None]
            j = torch.arange(ke - ka, device="cuda")[None]
            ok = j - i <= (ke - ka) - (e - a) if s["causal"] else (j >= 0) & (i >= 0)
            for h in range(H):
                Q = q[b, a:e, h]
                K = torch.cat([kv[b, ka:ke, h, :dn], kr[b, ka:ke]], -1)
                V = kv[b, ka:ke, h, dn:]
                p, z = _softmax64(s["scale"] * (Q @ K.T), ok)
                O = p @ V
                o[b, a:e, h], lse[b, h, a:e] = O, z
                if train:
                    dO = s["do"][b, a:e, h].double()
                    g = p * (dO @ V.T - (dO * O).sum(-1, keepdim=True)) * s["scale"]
                    dK = g.T @ Q
                    dq[b, a:e, h] = g @ K
                    dkv[b, ka:ke, h, :dn], dkv[b, ka:ke, h, dn:] = dK[:, :dn], p.T @ dO
                    dkr[b, ka:ke] += dK[:, dn:]
    return [o, dq, dkv, dkr] if train else (o, lse)


def _exact_append(s):
    R, dr, dt = s["R"], s["dr"], s["cache"].dtype
    cache = s["cache"].double().view(-1, R + dr)
    table = s["cos_sin"].double()[s["positions"]]
    x = s["rows"].double()

    def rotate(v, z):
        # a complex product: the pair (a, b) is a + ib, the table's row cos + i sin
        if s["interleaved"]:
            w = torch.view_as_complex(v.reshape(*v.shape[:-1], dr // 2, 2).contiguous()) * z
            return torch.view_as_real(w).reshape(v.shape)
        w = torch.complex(v[..., :dr // 2].contiguous(), v[..., dr // 2:].contiguous()) * z
        return torch.cat([w.real, w.imag], -1)

    z = torch.complex(table[:, :dr // 2].contiguous(), table[:, dr // 2:].contiguous())
    norm = (x[:, :R].square().mean(1) + EPS).sqrt()
    new = torch.cat([x[:, :R] / norm[:, None] * s["weight"].double(), rotate(x[:, R:], z)], 1)
    cache.index_copy_(0, s["slots"][s["real"]], new[s["real"]])
    return [cache.view(s["cache"].shape), rotate(s["q"][..., 128:].double(), z[:, None])]


def _exact_decode(s):
    q, R = s["q"].double(), s["R"]
    B, Tq, H, W = q.shape
    page = s["cache"].shape[1]
    o = torch.zeros(B, Tq, H, R, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Tq, H), float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        k = s["cache"][s["table"][b, :-(-n // page)].long()].reshape(-1, W)[:n].double()
        for t in range(Tq):
            m = n - (Tq - 1 - t)
            if m > 0:
                sc = s["scale"] * (q[b, t] @ k[:m].T)
                lse[b, t] = torch.logsumexp(sc, -1)
                o[b, t] = torch.softmax(sc, -1) @ k[:m, :R]
    return o, lse


# ---------------------------------------------------------------------------------------------- cost

def work(case):
    c, es = case, 4 if case["dtype"] == "fp32" else 2
    if c["kind"] in ("prefill", "packed", "train"):
        H, dn, dr = c["H"], c["dn"], c["dr"]
        if c["kind"] == "packed":
            offs = _offsets(c)
            B, Tq, Tk = 1, offs[-1], offs[-1]
            pairs = sum((e - a) * (e - a + 1) / 2 for a, e in zip(offs[:-1], offs[1:]))
        else:
            B, Tq, Tk = c["B"], c.get("Tq", c.get("T")), c.get("Tk", c.get("T"))
            pairs = B * (Tq * (Tk - Tq) + Tq * (Tq + 1) / 2 if c["causal"] else Tq * Tk)
        rows = B * Tq * H * (2 * dn + dr) + B * Tk * (H * 2 * dn + dr)   # q, o, kv, k_rope
        flops = 2 * pairs * H * (2 * dn + dr)
        if c["kind"] == "train":   # do in, dq, dkv, dk_rope out; the gradient's five products
            rows += B * Tq * H * (2 * dn + dr) + B * Tk * (H * 2 * dn + dr)
            flops += 2 * pairs * H * (5 * dn + 3 * dr)
            return {"bytes": es * rows, "flops": flops}
        return {"bytes": es * rows + 4 * B * Tq * H, "flops": flops}
    R, dr, H = c["R"], c["dr"], c["H"]
    if c["kind"] == "append":
        N = c["N"]
        return {"bytes": 2 * es * N * (R + dr + H * dr) + 4 * R + N * (16 + 4 * dr), "flops": N * (4 * R + 3 * dr * (H + 1))}
    lens = _lengths(c["B"], c["lo"], c["hi"], c["lseed"])
    tokens, rows = int(lens.sum()), c["B"] * c["Tq"] * H
    return {"bytes": es * (tokens * (R + dr) + rows * (2 * R + dr)) + 4 * rows, "flops": 2 * tokens * c["Tq"] * H * (2 * R + dr)}
