"""GPU: the latent cache's append and the absorbed attention over it against float64."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import DT, U, bar, check, check_lse
from oracle import latent as O

pytestmark = pytest.mark.gpu


def _table(P, dr, device):
    f = 10000.0 ** (-torch.arange(0, dr, 2, dtype=torch.float64) / dr)
    a = torch.arange(P, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().to(device)


def _append_case(N, H, R, dr, page, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, device=device, generator=g).to(DT[dtype])

    pages = 2 * -(-max(N, 1) // page) + 1
    d = dict(rows=rnd(N, R + dr + 32)[:, 32:], cache=rnd(pages, page, R + dr), q=rnd(N, H, 128 + dr)[..., 128:])
    d["positions"] = torch.randint(0, 500, (N,), device=device, generator=g)
    d["slots"] = torch.randperm(pages * page, device=device, generator=g)[:N].contiguous()
    d["w"] = 1 + 0.2 * torch.randn(R, device=device, generator=g)
    return d


# one rounding of each result; the rotation's two fp32 products and the norm's sum stay below 1e-6
def _append_bar(dtype):
    return 1e-6 if dtype == "fp32" else U[dtype]


@pytest.mark.parametrize("N", [0, 1, 3, 70, 1024, 1500])
@pytest.mark.parametrize("R,dr,dtype,inter", [(512, 64, "bf16", False), (512, 64, "fp32", True), (256, 32, "fp16", True),
                                              (512, 32, "bf16", True), (256, 64, "fp32", False)])
def test_append(cuda, N, R, dr, dtype, inter):
    d = _append_case(N, 3, R, dr, 16, dtype, cuda, seed=N)
    cs = _table(500, dr, cuda)
    if N > 2:
        d["slots"][1] = -1                                  # padding
        d["slots"][2] = d["cache"].shape[0] * 16            # past the cache
    ref, q_ref = O.append(d["rows"], d["positions"], d["slots"], cs, d["cache"], d["w"], 1e-5, d["q"], inter)
    before = d["cache"].clone()
    q_out = axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"], norm_weight=d["w"], eps=1e-5,
                                    q_rope=d["q"], interleaved=inter)
    if N:
        check("cache", d["cache"], ref, _append_bar(dtype), ())
        check("q", q_out, q_ref, _append_bar(dtype), ())
    kept = torch.ones(before.shape[0] * 16, dtype=torch.bool, device=cuda)
    good = d["slots"][(d["slots"] >= 0) & (d["slots"] < kept.numel())]
    kept[good] = False
    same = (d["cache"] == before).view(kept.numel(), -1).all(1)
    assert same[kept].all() and not same[good].any()


def test_append_without_norm_and_queries(cuda):
    d = _append_case(40, 2, 512, 64, 32, "bf16", cuda, seed=5)
    cs = _table(500, 64, cuda)
    ref, _ = O.append(d["rows"], d["positions"], d["slots"], cs, d["cache"])
    assert axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"]) is None
    check("cache", d["cache"], ref, U["bf16"], ())
    flat = d["cache"].view(-1, 576)[d["slots"]]
    assert torch.equal(flat[:, :512], d["rows"][:, :512])   # taken as they are


def test_append_into_absorbed_query_and_in_place(cuda):
    d = _append_case(50, 4, 512, 64, 32, "bf16", cuda, seed=6)
    cs = _table(500, 64, cuda)
    q_abs = torch.zeros(50, 4, 576, dtype=torch.bfloat16, device=cuda)
    r = axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"], q_rope=d["q"], q_out=q_abs[..., 512:])
    assert r.data_ptr() == q_abs[..., 512:].data_ptr() and (q_abs[..., :512] == 0).all()
    axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"], q_rope=d["q"], q_out=d["q"])
    assert torch.equal(d["q"], q_abs[..., 512:])


def test_append_positions_outside_the_table(cuda):
    d = _append_case(4, 1, 256, 32, 16, "fp32", cuda, seed=7)
    cs = _table(10, 32, cuda)
    d["positions"] = torch.tensor([-5, 0, 9, 1 << 40], device=cuda)
    ref, q_ref = O.append(d["rows"], d["positions"], d["slots"], cs, d["cache"], d["w"], 1e-6, d["q"])
    q = axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"], norm_weight=d["w"], q_rope=d["q"])
    check("cache", d["cache"], ref, 1e-6, ())
    check("q", q, q_ref, 1e-6, ())


def _decode_case(lens, Tq, H, R, dr, page, dtype, device, seed=0, extra=0):
    """Scattered pages; what no sequence holds (page tails, spare pages) is NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    B = len(lens)
    per = max(1, max(-(-n // page) for n in lens)) + extra
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    order = torch.randperm(pages, device=device, generator=g).int()
    table = torch.full((B, per), -7, dtype=torch.int32, device=device)
    cache = torch.full((pages, page, R + dr), float("nan"), dtype=DT[dtype], device=device)
    at = 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = order[at:at + used[b]]
        for i in range(used[b]):
            k = min(page, n - i * page)
            cache[int(order[at + i]), :k] = torch.randn(k, R + dr, device=device, generator=g).to(DT[dtype])
        at += used[b]
    q = (torch.randn(B, Tq, H, R + dr, device=device, generator=g) * 0.8).to(DT[dtype])
    return q, cache, table, torch.tensor(lens, dtype=torch.int32, device=device)


def _decode_compare(case, R, dtype, scale=0.07):
    q, cache, table, lens = case
    o_ref, lse_ref = O.decode(q, cache, table, lens, R, scale)
    o, lse = axiom_amd.latent_decode(q, cache, table, lens, scale=scale)
    check("o", o, o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)
    return o, lse


LENS = [[1], [0], [31, 32, 33, 0, 64, 65], [1, 2, 3, 500, 7], [129, 1000, 0, 0, 64]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Tq", [1, 3])
def test_decode_lengths(cuda, lens, dtype, Tq):
    _decode_compare(_decode_case(lens, Tq, 5, 512, 64, 16, dtype, cuda, seed=len(lens)), 512, dtype)


@pytest.mark.parametrize("Tq,H", [(1, 1), (1, 16), (1, 17), (2, 16), (1, 33), (1, 64), (1, 65), (1, 128), (4, 40)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_decode_rows(cuda, Tq, H, dtype):
    """Row counts around the 16-row blocks, the groups of blocks and more than one group."""
    _decode_compare(_decode_case([200, 3, 90], Tq, H, 512, 64, 32, dtype, cuda, seed=H), 512, dtype)


@pytest.mark.parametrize("R,dr", [(512, 32), (256, 64), (256, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H", [8, 24, 48])
def test_decode_dims(cuda, R, dr, dtype, H):
    _decode_compare(_decode_case([70, 333], 1, H, R, dr, 64, dtype, cuda, seed=R + dr), R, dtype)


@pytest.mark.parametrize("page", [1, 2, 16, 128, 1024])
def test_decode_pages(cuda, page):
    _decode_compare(_decode_case([1, 100, 257], 1, 16, 512, 64, page, "bf16", cuda, seed=page, extra=3), 512, "bf16")


def test_decode_many_sequences(cuda):
    """More sequences than a wave looks at in one step, and than there are workgroups."""
    lens = [(13 * i) % 90 for i in range(300)]
    _decode_compare(_decode_case(lens, 1, 16, 256, 32, 16, "bf16", cuda, seed=2), 256, "bf16")


def test_decode_long(cuda):
    """One long sequence split over the whole chip, and beside it short ones."""
    _decode_compare(_decode_case([40000, 5, 300], 1, 16, 512, 64, 64, "bf16", cuda, seed=3), 512, "bf16")
    _decode_compare(_decode_case([20001], 2, 64, 512, 64, 64, "fp16", cuda, seed=4), 512, "fp16")


def test_decode_past_32_bits(cuda):
    """A cache of more than 4 GiB: rows on both sides of the 32-bit byte offset."""
    pages, page, W = 62000, 64, 576          # 4.57 GB
    cache = torch.empty(pages, page, W, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    table = torch.tensor([[0, 61999, 58253, 58254, 31000]], dtype=torch.int32, device=cuda)
    for p in table[0].tolist():
        cache[p] = torch.randn(page, W, device=cuda, generator=g).to(torch.bfloat16)
    q = torch.randn(1, 1, 16, W, device=cuda, generator=g).to(torch.bfloat16)
    lens = torch.tensor([300], dtype=torch.int32, device=cuda)
    _decode_compare((q, cache, table, lens), 512, "bf16")
    rows = torch.randn(2, W, device=cuda, generator=g).to(torch.bfloat16)
    slots = torch.tensor([61999 * 64 + 63, 58254 * 64], device=cuda)
    cs = _table(8, 64, cuda)
    axiom_amd.latent_append(rows, torch.zeros(2, dtype=torch.int64, device=cuda), slots, cs, cache)
    assert torch.equal(cache.view(-1, W)[slots], rows)


def test_decode_bad_tables_stay_inside(cuda):
    """Page numbers and lengths out of range are clamped: other sequences keep their results."""
    q, cache, table, lens = _decode_case([70, 200, 64], 1, 16, 512, 64, 32, "bf16", cuda, seed=8)
    cache = torch.nan_to_num(cache)
    o, lse = axiom_amd.latent_decode(q, cache, table, lens, scale=0.07)
    t2, l2 = table.clone(), lens.clone()
    t2[1] = torch.tensor([1 << 30, -1, -(1 << 31), 5, 9, 2, 3], dtype=torch.int32, device=cuda)[:t2.shape[1]]
    l2[1] = 1 << 30
    o2, lse2 = axiom_amd.latent_decode(q, cache, t2, l2, scale=0.07)
    for b in (0, 2):
        # the split over workgroups differs with the lengths: equal up to the join's fp32 order and o's rounding
        check("o", o2[b], o[b].cpu().double(), bar("bf16"), ())
    l2[1] = -3
    o3, lse3 = axiom_amd.latent_decode(q, cache, table, l2, scale=0.07)
    assert (o3[1] == 0).all() and torch.isneginf(lse3[1]).all()


def test_decode_given_workspace_and_outputs(cuda):
    from axiom_amd.latent import latent_decode_workspace_bytes
    q, cache, table, lens = _decode_case([700, 20], 1, 16, 512, 64, 32, "bf16", cuda, seed=9)
    o, lse = axiom_amd.latent_decode(q, cache, table, lens, scale=0.07)
    ws = torch.full((latent_decode_workspace_bytes(2, 1, 16, 512, 64, 32, table.shape[1]),), 255, dtype=torch.uint8, device=cuda)
    out, l2 = torch.empty_like(o), torch.empty_like(lse)
    r = axiom_amd.latent_decode(q, cache, table, lens, scale=0.07, out=out, lse=l2, workspace=ws)
    assert r[0] is out and torch.equal(out, o) and torch.equal(l2, lse)


def test_decode_same_bits_every_run(cuda):
    case = _decode_case([3000, 17, 900], 1, 64, 512, 64, 64, "bf16", cuda, seed=10)
    first = axiom_amd.latent_decode(*case, scale=0.07)
    for _ in range(3):
        again = axiom_amd.latent_decode(*case, scale=0.07)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_decode_loop_in_a_graph(cuda):
    """Append and attention of one token captured once; lengths, slots and rows change between replays."""
    q, cache, table, lens = _decode_case([100, 37], 1, 16, 512, 64, 64, "bf16", cuda, seed=11, extra=1)
    cache = torch.nan_to_num(cache)
    table.clamp_(min=0)
    cs = _table(400, 64, cuda)
    rows = torch.randn(2, 576, device=cuda).to(torch.bfloat16)
    pos = (lens - 1).long()
    slots = (table[torch.arange(2, device=cuda), pos // 64].long() * 64 + pos % 64).contiguous()
    from axiom_amd.latent import latent_decode_workspace_bytes
    ws = torch.empty(latent_decode_workspace_bytes(2, 1, 16, 512, 64, 64, table.shape[1]), dtype=torch.uint8, device=cuda)

    def token():
        axiom_amd.latent_append(rows, pos, slots, cs, cache)
        return axiom_amd.latent_decode(q, cache, table, lens, scale=0.07, workspace=ws)

    token()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = token()
    for step in range(4):
        rows.copy_(torch.randn(2, 576, device=cuda))
        lens += 1
        pos.copy_((lens - 1).long())
        slots.copy_(table[torch.arange(2, device=cuda), pos // 64].long() * 64 + pos % 64)
        graph.replay()
        got = o.clone(), lse.clone()
        torch.cuda.synchronize()
        want = token()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_absorbed_equals_expanded(cuda):
    """The two forms of one layer: prompt through the expanded one, its last token through the cache."""
    B, T, H, dn, R, dr = 2, 150, 8, 128, 512, 64
    g = torch.Generator(device=cuda).manual_seed(12)

    def rnd(*s):
        return torch.randn(*s, device=cuda, generator=g)

    down, w_uk, w_uv = rnd(B * T, R + dr), rnd(H, dn, R) * R ** -0.5, rnd(H, dn, R) * R ** -0.5
    q = rnd(B, T, H, dn + dr)
    cs, pos = _table(T, dr, cuda), torch.arange(T, device=cuda).repeat(B)
    page, per = 16, -(-T // 16)
    cache = torch.zeros(B * per, page, R + dr, device=cuda)
    table = torch.randperm(B * per, device=cuda, generator=g).int().view(B, per)
    slots = (table.long()[torch.arange(B, device=cuda).repeat_interleave(T), pos // page] * page + pos % page).contiguous()
    qf = q.view(B * T, H, dn + dr)
    axiom_amd.latent_append(down, pos, slots, cs, cache, norm_weight=torch.ones(R, device=cuda), q_rope=qf[..., dn:],
                            q_out=qf[..., dn:])
    lat = cache.view(-1, R + dr)[slots].view(B, T, R + dr)
    kv = torch.cat([torch.einsum("btr,hdr->bthd", lat[..., :R], w_uk), torch.einsum("btr,hdr->bthd", lat[..., :R], w_uv)], -1)
    o, lse = axiom_amd.latent_attn_fwd(q, kv.contiguous(), lat[..., R:])
    q_abs = torch.cat([torch.einsum("bhd,hdr->bhr", q[:, -1, :, :dn], w_uk), q[:, -1, :, dn:]], -1)[:, None].contiguous()
    lens = torch.full((B,), T, dtype=torch.int32, device=cuda)
    o_lat, lse1 = axiom_amd.latent_decode(q_abs, cache, table, lens, scale=(dn + dr) ** -0.5)
    o1 = torch.einsum("bhr,hdr->bhd", o_lat[:, 0], w_uv)
    # fp32 throughout; the two forms' scores differ by the fp32 products of the projections (R terms): 1e-4
    assert (o1 - o[:, -1]).norm() <= 1e-4 * o[:, -1].norm()
    assert (lse1[:, 0] - lse[:, :, -1]).abs().max() <= 1e-4
