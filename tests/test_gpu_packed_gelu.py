"""GELU and its slope with their error relative to the result, far into the negative tail.

The tail is erfc(|x| / sqrt 2) / 2 = exp(-x^2 / 2) R(|x|).  16-bit types: R is off by 9e-6 of itself, the
exponential's argument (up to 2^7) is rounded in fp32 (2^7 2^-24 ln 2 = 5e-6), and a few fp32 roundings follow: 1.6e-5
together, then the rounding to the type.  fp32: R with its roundings 6 of 2^-24, an exponential with its argument in two
parts and three products: 16 of 2^-24.  Below 2^-126 the exponential's hardware instruction gives 0."""
import pytest
import torch

from test_gpu_packed import F, TYPES, P, eight_bits, gen, half_step, normal, smallest

pytestmark = pytest.mark.gpu


def cdf64(x):
    return torch.erfc(-x / 2 ** 0.5) / 2               # (torch's ndtr is 0 on the device below -8)


def density64(x):
    return torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5


def off(t):
    return 16 * F if t == torch.float32 else 1.6e-5


def values(t):
    """Every value of a 16-bit type from -13 to 13 (fp32: spread over it)."""
    if t == torch.float32:
        return torch.cat([torch.linspace(-13, 13, 1 << 20, device="cuda"), -torch.rand(1 << 16, device="cuda", generator=gen(1))])
    x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32, device="cuda").to(torch.int16).view(t)
    return x[x.abs() <= 13]


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gelu_is_relatively_exact(t):
    x = values(t)
    y = P().gelu8(x).double()
    want = x.double() * cdf64(x.double())
    bad = (y - want).abs() - ((half_step(t) + off(t)) * want.abs() + max(smallest(t), 2.0 ** -122))
    assert bad.max() <= 0, x[bad.argmax()]
    assert torch.equal(P().gelu8(x.detach().requires_grad_()).detach().double(), y)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gelu_gradient_is_relatively_exact(t):
    """Its two terms, Phi and x phi, have opposite signs below 0: the error is relative to their sizes."""
    x = values(t).sort()[0]
    x = x[:x.numel() // 32 * 32].reshape(-1, 32).requires_grad_()    # neighbours share a power of two
    dy = normal(gen(2), *x.shape, dtype=t)
    d, = torch.autograd.grad(P().gelu8(x), x, dy)
    kept = eight_bits(x)[0].reshape(x.shape)
    size = dy.double().abs() * (cdf64(kept) + (kept * density64(kept)).abs())
    want = dy.double() * (cdf64(kept) + kept * density64(kept))
    assert ((d.double() - want).abs() <= half_step(t) * want.abs() + off(t) * size + max(smallest(t), 2.0 ** -122)).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gelu_at_the_ends(t):
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, -40.0, 40.0, torch.finfo(t).max, torch.finfo(t).min],
                     device="cuda").to(t)
    y = P().gelu8(x).tolist()
    assert y[0] == float("inf") and y[1] == 0 and y[2] != y[2] and y[3:6] == [0, 0, 0] and y[6] == 40
    assert y[7] == torch.finfo(t).max and y[8] == 0
    keep = x.masked_fill(~torch.isfinite(x), 1.0).requires_grad_()
    d, = torch.autograd.grad(P().gelu8(keep), keep, torch.ones_like(keep))
    assert torch.isfinite(d).all()
