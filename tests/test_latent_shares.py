"""CPU: the plan of a call's shares, restated, against the workspace sizes that follow from it.

A walk is what a block of 128 rows does along the other axis, in tiles (64 rows,
fp32 32).  A call of at most 256 (block, head) pairs may cut its walks into shares of
one length, the shortest with which all shares (an empty walk is one too) are at
most 256 over the heads; at least 128 rows, at most 16 shares of the longest
walk, and not at all where the longest share would be more than 3/4 of the longest
walk.  The workspace holds the parts of the larger plan of causal and not.
"""

from __future__ import annotations

import random

import pytest

from axiom_amd import _lib


@pytest.fixture(scope="module")
def L():
    if not _lib.LIB_PATH.exists():
        from axiom_amd import build
        build.build()
    return _lib.lib()


def _cdiv(a, b):
    return -(-a // b)


def _walks(Tq, Tk, tile, causal, queries):
    """Tiles that each block walks, counted row by row."""
    out = []
    for r0 in range(0, Tq if queries else Tk, 128):
        r1 = min(r0 + 128, Tq if queries else Tk) - 1
        if queries:
            last = min(Tk - 1, r1 + Tk - Tq) if causal else Tk - 1      # the last key that any of its queries sees
            out.append(0 if last < 0 else last // tile + 1)
        else:
            first = max(0, r0 + Tq - Tk) if causal else 0                # the first query that sees any of its keys
            out.append(max(0, _cdiv(Tq, tile) - first // tile))
    return out


def _parts(Tq, Tk, heads, causal, code, queries):
    walks = _walks(Tq, Tk, 32 if code == 0 else 64, causal, queries)
    other = Tk if queries else Tq
    longest = max(walks, default=0)
    most = min(16, _cdiv(other, 128))
    if not walks or len(walks) * heads > 256 or most <= 1:
        return 1
    for length in range(1, longest + 1):
        if length < (4 if code == 0 else 2) or _cdiv(longest, length) > most:
            continue
        if heads * sum(max(1, _cdiv(w, length)) for w in walks) <= 256:
            return _cdiv(longest, length) if 4 * length <= 3 * longest else 1
    return 1


def _up(x):
    return _cdiv(x, 256) * 256


def _check(L, B, Tq, Tk, H, dn, dr, code):
    q = max(_parts(Tq, Tk, B * H, c, code, True) for c in (False, True))
    rows = q * B * H * Tq if q > 1 else 0
    assert L.kda_latent_attn_fwd_workspace(B, Tq, Tk, H, dn, dr, 0, code) == _up(rows * dn * 4) + _up(rows * 8), (B, Tq, Tk, H, code)
    sizes = []
    for c in (False, True):
        q, k = (_parts(Tq, Tk, B * H, c, code, side) for side in (True, False))
        want = _up(B * H * Tq * 4) + _up(B * H * _cdiv(Tq, 128) * 4) + _up(k * B * H * Tk * dr * 4)
        want += _up(q * B * H * Tq * (dn + dr) * 4 if q > 1 else 0) + _up(k * B * H * Tk * 2 * dn * 4 if k > 1 else 0) + 256
        sizes.append(want)
    assert L.kda_latent_attn_bwd_workspace(B, Tq, Tk, H, dn, dr, 0, code) == max(sizes), (B, Tq, Tk, H, code)


@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("B,Tq,Tk,H", [(1, 1000, 1000, 8), (1, 8400, 8400, 1), (1, 1024, 1024, 8), (2, 1000, 1000, 8), (1, 512, 512, 4),
                                       (1, 333, 1333, 16), (1, 900, 500, 3), (1, 700, 1100, 2), (1, 1024, 1024, 31), (1, 1024, 1024, 32),
                                       (1, 1024, 1024, 33), (1, 1, 5000, 16), (1, 4096, 4096, 8), (1, 100, 20000, 1)])
def test_listed(L, B, Tq, Tk, H, code):
    _check(L, B, Tq, Tk, H, 128, 64, code)


def test_equal_lengths_are_not_equal_numbers(L):
    """Causal walks of 1000 rows and 8 heads: 6 shares of the longest in 16 bits and 7 in fp32; 256 // 64 blocks would be 4."""
    assert _parts(1000, 1000, 8, True, 1, True) == 6 and _parts(1000, 1000, 8, True, 0, True) == 7


def test_drawn(L):
    rng = random.Random(7)
    for _ in range(400):
        B, H = rng.choice([1, 1, 1, 2, 3]), rng.choice([1, 2, 3, 4, 8, 12, 16, 24])
        Tq, Tk = int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 13))
        if rng.random() < 0.5:
            Tk = Tq
        _check(L, B, Tq, Tk, H, rng.choice([64, 128]), rng.choice([32, 64]), rng.choice([0, 1, 2]))
