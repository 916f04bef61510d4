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


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_queries_without_any_keys(t, causal):
    L, g = P(), gen(131)
    buckets = L.RelativeBuckets(8, 6)
    q = normal(g, 7, 2, 16, dtype=t).requires_grad_()
    k, v = (torch.empty(0, 2, 16, dtype=t, device="cuda", requires_grad=True) for _ in range(2))
    table = normal(g, 8, 2, dtype=t).requires_grad_()
    seqs = L.PackedSequences([3, 4], [0, 0])
    for more, leaves in (({}, [q, k, v]), ({"bias": table, "buckets": buckets}, [q, k, v, table])):
        o = L.packed_attention(q, k, v, seqs, causal=causal, **more)
        grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
        assert not o.any() and all(not d.any() and d.shape == x.shape for d, x in zip(grads, leaves))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_one_tensor_for_everything_and_two_backward_passes(t):
    L, g = P(), gen(132)
    n = [40, 1, 90]
    x, do = normal(g, sum(n), 3, 32, dtype=t).requires_grad_(), normal(g, sum(n), 3, 32, dtype=t)
    table = normal(g, 8, 3, dtype=t).requires_grad_()
    seqs, buckets = L.PackedSequences(n), L.RelativeBuckets(8, 6)
    o = L.packed_attention(x, x, x, seqs, bias=table, buckets=buckets)
    first = torch.autograd.grad(o, [x, table], do, retain_graph=True)
    again = torch.autograd.grad(o, [x, table], do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    apart = torch.autograd.grad(L.packed_attention(*parts, seqs, bias=table, buckets=buckets), [*parts, table], do)
    assert torch.equal(first[1], apart[3])
    # autograd adds the three in the tensors' type: two more roundings
    total = sum(p.double() for p in apart[:3])
    size = sum(p.double().abs() for p in apart[:3])
    assert ((first[0].double() - total).abs() <= 2 * torch.finfo(t).eps * size).all()


def test_a_join_of_a_tensor_with_itself():
    L, g = P(), gen(133)
    x, w = normal(g, 9, 40).requires_grad_(), normal(g, 40, mean=1.0)
    y, n = L.gated_norm(x, x, w, w, gate=x)
    d, = torch.autograd.grad([y, n], x, [torch.ones_like(y), torch.ones_like(n)])
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    y2, n2 = L.gated_norm(parts[0], parts[1], w, w, gate=parts[2])
    ds = torch.autograd.grad([y2, n2], parts, [torch.ones_like(y), torch.ones_like(n)])
    assert torch.equal(y, y2) and torch.equal(n, n2)
    assert (d - sum(ds)).abs().max() <= 4 * torch.finfo(torch.float32).eps * sum(v.abs() for v in ds).max()
