"""GPU: branches of the latent kernels that sizes lead to: groups of heads in the order of blocks, both sides
of the shares' rule, and the 64-row decode with empty sequences, rows that see nothing, small tables and pages."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs, bar, check, check_lse, terms
from oracle import latent as O
from test_gpu_latent_cache import _append_bar, _append_case, _decode_case, _decode_compare, _table

pytestmark = pytest.mark.gpu


def _all(q, kv, kr, do, causal=True):
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, causal=causal)
    return o, lse, *axiom_amd.latent_attn_bwd(q, kv, kr, o, lse, do, causal=causal)


def _against_oracle(B, T, H, dtype, causal=True):
    q, kv, kr, do = attn_inputs(B, T, T, H, 64, 32, dtype, torch.device("cuda:0"), seed=T + H)
    o_ref, lse_ref, *g_ref = O.attn(q, kv, kr, causal, do=do)
    o, lse, *grads = _all(q, kv, kr, do, causal)
    check("o", o, o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)
    for name, got, ref, axes in zip(("dq", "dkv", "dk_rope"), grads, g_ref, ((0, 2), (0, 2), (0,))):
        check(name, got, ref, bar(dtype, True), axes, 0.1 * terms(q, kv, kr, do))


# heads over the eight dies: 5, 6 and 7 a die, taken four at a time, so that the last group is a partial one
@pytest.mark.parametrize("B,H,T", [(1, 40, 900), (3, 16, 800), (2, 28, 700)])
@pytest.mark.parametrize("causal", [True, False])
def test_partial_groups_of_heads(cuda, B, H, T, causal):
    _against_oracle(B, T, H, "bf16", causal)


@pytest.mark.parametrize("T,H", [(1500, 24), (11100, 24), (16500, 24), (33000, 16)])
def test_heads_by_themselves(cuda, T, H):
    """A call's heads equal the calls of eight of them bit for bit: 12, 87, 129 and 258 blocks a head, so groups
    of four, two and one head a die (no call here shares its walks out)."""
    q, kv, kr, do = attn_inputs(1, T, T, H, 64, 32, "bf16", cuda, seed=T)
    kr = kr.contiguous()
    # eight heads of 12 blocks would be shared out: calls of 24 heads that differ in the others instead
    n = 8 if 8 * -(-T // 128) > 256 else H
    whole = _all(q, kv, kr, do)
    for h in range(0, H, n) if n == 8 else (0, 8, 16):
        if n == 8:
            part = _all(*(x[:, :, h:h + 8].contiguous() for x in (q, kv)), kr, do[:, :, h:h + 8].contiguous())
        else:
            roll = [x.roll(-h, 2).contiguous() for x in (q, kv, do)]
            part = _all(roll[0], roll[1], kr, roll[2])
            part = [x[:, :8] if i == 1 else x[:, :, :8] for i, x in enumerate(part[:4])]
        for name, a, b in zip(("o", "lse", "dq", "dkv"), whole, part):
            a = a[:, h:h + 8] if name == "lse" else a[:, :, h:h + 8]
            assert torch.equal(a, b), (name, h)


# 248, 256 and 264 blocks: below, at and past the most that are shared out
@pytest.mark.parametrize("H", [31, 32, 33])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_around_the_shares_rule(cuda, H, dtype):
    _against_oracle(1, 1024, H, dtype)


ROWS = [(1, 24), (3, 24), (1, 128), (4, 7)]   # 24, 72, 128 and 28 rows: partial groups of 64, two groups


@pytest.mark.parametrize("Tq,H", ROWS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [[1], [0], [31, 32, 33, 0, 64, 65], [129, 1000, 0, 0, 64], [1, 2, 3, 500, 7], [0, 0, 2000, 0, 1, 0]], ids=str)
def test_64_row_decode_lengths(cuda, Tq, H, dtype, lens):
    """Tables of at most 128 tokens (a workgroup a sequence) and longer ones (runs); sequences of no token,
    of fewer than the queries, around the tiles of 32 keys."""
    _decode_compare(_decode_case(lens, Tq, H, 512, 64, 16, dtype, cuda, seed=len(lens) + Tq), 512, dtype)


@pytest.mark.parametrize("Tq,H", ROWS)
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64])
@pytest.mark.parametrize("lens", [[100, 1, 37], [300, 0, 5, 1111]], ids=str)
def test_64_row_decode_pages(cuda, Tq, H, page, lens):
    """Pages smaller than a tile, as long and longer."""
    _decode_compare(_decode_case(lens, Tq, H, 512, 64, page, "bf16", cuda, seed=page + H, extra=1), 512, "bf16")


@pytest.mark.parametrize("R,dr", [(256, 64), (256, 32), (512, 32)])
@pytest.mark.parametrize("Tq,H", [(2, 24), (1, 100)])
def test_64_row_decode_dims(cuda, R, dr, Tq, H):
    _decode_compare(_decode_case([0, 1, 90, 700, 33], Tq, H, R, dr, 32, "fp16", cuda, seed=R + dr + H), R, "fp16")


def test_64_row_decode_many_sequences(cuda):
    """More sequences than lanes and than runs, a third of them empty."""
    lens = [(13 * i) % 200 if i % 3 else 0 for i in range(300)]
    _decode_compare(_decode_case(lens, 1, 40, 256, 32, 16, "bf16", cuda, seed=2), 256, "bf16")


@pytest.mark.parametrize("H", [16, 40])
def test_decode_in_small_pages_and_tables(cuda, H):
    """A workgroup a sequence with pages of one token."""
    _decode_compare(_decode_case([17, 0, 1, 60], 2, H // 2, 512, 64, 1, "bf16", cuda, seed=H), 512, "bf16")


@pytest.mark.parametrize("N", [2047, 2048, 2049, 2051, 5000])
@pytest.mark.parametrize("R,dr,dtype,inter", [(512, 64, "bf16", False), (512, 64, "fp32", True), (256, 32, "fp16", True)])
def test_append_of_many_tokens(cuda, N, R, dr, dtype, inter):
    """Both ways to split tokens over waves, a last workgroup of one to four tokens among them."""
    d, cs = _append_case(N, 3, R, dr, 16, dtype, cuda, seed=N), _table(500, dr, cuda)
    d["slots"][1] = -1
    ref, q_ref = O.append(d["rows"], d["positions"], d["slots"], cs, d["cache"], d["w"], 1e-5, d["q"], inter)
    q_out = axiom_amd.latent_append(d["rows"], d["positions"], d["slots"], cs, d["cache"], norm_weight=d["w"], eps=1e-5,
                                    q_rope=d["q"], interleaved=inter)
    check("cache", d["cache"], ref, _append_bar(dtype), ())
    check("q", q_out, q_ref, _append_bar(dtype), ())
