"""linear8 inside an autocast region keeps its tensors' own type, forward and backward, as every operator beside it."""
import pytest
import torch

from test_gpu_packed import P, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inside", ["forward", "both", "backward"])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
def test_linear8_under_autocast(t, act, inside):
    g = gen(120)
    x, W, b = normal(g, 9, 64, dtype=t), normal(g, 40, 64, dtype=t), normal(g, 40, dtype=t)
    do = normal(g, 9, 40, dtype=t)
    leaves = [v.requires_grad_() for v in (x, W, b)]
    want = P().linear8(*leaves, act=act)
    grads = torch.autograd.grad(want, leaves, do)
    with torch.autocast("cuda", dtype=torch.float16, enabled=inside != "backward"):
        got = P().linear8(*leaves, act=act)
        with torch.no_grad():
            plain = P().linear8(*leaves, act=act)
    assert got.dtype == t and torch.equal(got, want) and torch.equal(plain, want)
    with torch.autocast("cuda", dtype=torch.float16, enabled=inside != "forward"):
        again = torch.autograd.grad(got, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
