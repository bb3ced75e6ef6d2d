"""Forward-mode derivatives of the block operators: there are none, and an input with a tangent is refused instead of losing it."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import gcpnet_amd as G
from gcpnet_amd import block_ops


def test_a_tangent_is_noticed():
    x = torch.ones(2, 3)
    assert not block_ops._wants_grad((x, None)) and block_ops._wants_grad((x, x.clone().requires_grad_()))
    with forward_ad.dual_level():
        assert not block_ops._wants_grad((x, None))  # (a level alone is no tangent)
        dual = forward_ad.make_dual(x, x)
        for context in (torch.enable_grad(), torch.no_grad()):  # (no_grad does not end forward mode)
            with context, pytest.raises(NotImplementedError, match="forward-mode"):
                block_ops._wants_grad((None, dual))
    assert not block_ops._wants_grad((x,))


@pytest.mark.gpu
def test_tangents_are_refused():
    x, w = torch.randn(5, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    for call in (lambda v: G.linear_act(v, w, act="silu"), lambda v: G.linear_act(x, w, residual=v), lambda v: G.residual_norm(v, pre="rms")[1],
                 lambda v: G.residual_norm(x, v, pre="layer")[0]):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        call(x)


@pytest.mark.gpu
def test_a_tangent_of_the_gradient_is_refused():
    x, w = torch.randn(5, 8, device="cuda", requires_grad=True), torch.randn(8, 8, device="cuda")
    for y in (G.linear_act(x, w, act="silu"), G.residual_norm(x, pre="rms")[1]):
        up = torch.ones_like(y)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(up, up), retain_graph=True)
        torch.autograd.grad(y, x, up)
