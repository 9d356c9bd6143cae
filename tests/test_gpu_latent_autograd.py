"""GPU: the differentiable latent attention as autograd uses it."""

from __future__ import annotations

import itertools

import pytest
import torch

import axiom_amd
from latent_testutil import attn_inputs

pytestmark = pytest.mark.gpu


def _inputs(cuda):
    q, kv, kr, do = attn_inputs(1, 90, 90, 2, 64, 32, "fp32", cuda, seed=5)
    return [x.contiguous().requires_grad_(True) for x in (q, kv, kr)], do


@pytest.mark.parametrize("what", ["penalty", "plain cotangent", "cotangent alone"])
def test_second_derivative_raises(cuda, what):
    """With create_graph the first gradient is there, and differentiating it raises: no term is left out silently."""
    xs, do = _inputs(cuda)
    if what == "cotangent alone":
        do.requires_grad_(True)
    o = axiom_amd.latent_attn(*xs)
    want = torch.autograd.grad(o, xs, do.detach(), retain_graph=True)
    grads = torch.autograd.grad(o, xs, do, create_graph=True)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
    # beside a path that has a second derivative of its own
    loss = sum(g.square().sum() for g in grads) + (xs[0] ** 3).sum()
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        if what == "penalty":
            loss.backward()
        else:
            torch.autograd.grad(loss, do if what == "cotangent alone" else xs[0])


@pytest.mark.parametrize("need", [n for r in (1, 2, 3) for n in itertools.combinations(range(3), r)])
def test_a_subset_of_gradients(cuda, need):
    xs, do = _inputs(cuda)
    want = torch.autograd.grad(axiom_amd.latent_attn(*xs), xs, do)
    for i, x in enumerate(xs):
        x.requires_grad_(i in need)
    o = axiom_amd.latent_attn(*xs)
    o.backward(do)
    for i, x in enumerate(xs):
        assert (x.grad is not None) == (i in need) and (x.grad is None or torch.equal(x.grad, want[i]))


def test_no_gradient_wanted(cuda):
    xs, _ = _inputs(cuda)
    with torch.no_grad():
        assert axiom_amd.latent_attn(*xs).grad_fn is None
    assert axiom_amd.latent_attn(*(x.detach() for x in xs)).grad_fn is None


def test_expanded_cotangent(cuda):
    """The cotangent of a plain sum has stride 0."""
    xs, do = _inputs(cuda)
    got = torch.autograd.grad(axiom_amd.latent_attn(*xs).sum(), xs)
    want = torch.autograd.grad(axiom_amd.latent_attn(*xs), xs, torch.ones_like(do))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
