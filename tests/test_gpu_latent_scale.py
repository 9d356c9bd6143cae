"""GPU: scales far from one over a square root, with inputs that make up for them."""

from __future__ import annotations

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs, bar, check, check_lse, terms
from oracle import latent as O
from test_gpu_latent_cache import _decode_case

pytestmark = pytest.mark.gpu

SCALES = [1e-30, 1e-9, 1.0, 1e9, 1e30]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("Tq,Tk,H", [(150, 150, 2), (90, 40, 2), (900, 700, 1)])
def test_expanded(cuda, Tq, Tk, H, dtype, scale):
    """Causal, with rows that see nothing and with shares in which a row sees nothing."""
    q, kv, kr, do = attn_inputs(1, Tq, Tk, H, 64, 32, dtype, cuda, seed=Tq)
    q = (q.float() * (0.1 / scale)).to(q.dtype)
    o_ref, lse_ref, *g_ref = O.attn(q, kv, kr, True, scale, do=do)
    o, lse = axiom_amd.latent_attn_fwd(q, kv, kr, scale=scale)
    check("o", o, o_ref, bar(dtype), (0, 2))
    check_lse("lse", lse, lse_ref)
    grads = axiom_amd.latent_attn_bwd(q, kv, kr, o, lse, do, scale=scale)
    size = terms(q, kv, kr, do) * 96 ** 0.5 * scale   # of a gradient's term; dk's has q in place of the key
    for name, got, ref, part in (("dq", grads[0], g_ref[0], 1.0), ("dk", grads[1][..., :64], g_ref[1][..., :64], 0.15 / scale),
                                 ("dv", grads[1][..., 64:], g_ref[1][..., 64:], 0.0), ("dk_rope", grads[2], g_ref[2], 0.15 / scale)):
        check(name, got, ref, bar(dtype, True), (0,), 0.1 * size * part)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("H", [5, 24])
@pytest.mark.parametrize("lens", [[3, 100], [3, 700, 1, 0]], ids=str)
def test_decode(cuda, lens, H, scale):
    q, cache, table, n = _decode_case(lens, 4, H, 256, 32, 32, "bf16", cuda, seed=H)
    q = (q.float() * (0.07 / scale)).to(q.dtype)
    o_ref, lse_ref = O.decode(q, cache, table, n, 256, scale)
    o, lse = axiom_amd.latent_decode(q, cache, table, n, scale=scale)
    check("o", o, o_ref, bar("bf16"), (0, 2))
    check_lse("lse", lse, lse_ref)
