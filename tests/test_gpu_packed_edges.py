"""Smallest and largest calls of the packed operators."""
import pytest
import torch

from test_gpu_packed import P, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("lead,n_in,n_out", [((5,), 8, 0), ((5,), 0, 3), ((0,), 8, 3), ((), 8, 3), ((2, 0), 0, 0)])
def test_linear8_with_nothing_on_an_axis(act, lead, n_in, n_out):
    g = gen(130)
    x, W = normal(g, *lead, n_in).requires_grad_(), normal(g, n_out, n_in).requires_grad_()
    b = normal(g, n_out).requires_grad_()
    out = P().linear8(x, W, b, act=act)
    grads = torch.autograd.grad(out, (x, W, b), torch.ones_like(out))
    assert out.shape == (*lead, n_out)
    for a, leaf in zip(grads, (x, W, b)):
        assert a.shape == leaf.shape and torch.isfinite(a).all()
    if not lead:
        assert torch.equal(grads[2], torch.ones_like(b))
    elif 0 in (n_in, n_out, *lead):
        rows = 1
        for m in lead:
            rows *= m
        assert not grads[1].any() and not grads[0].any() and (grads[2] == rows).all()
