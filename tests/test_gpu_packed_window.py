"""A window made by the bias: one bucket far below the others masks its keys.  Whole tiles of masked keys come before
the first that counts, and the scores after them must keep their digits.

Errors are norms against the formula in 64 bits with the masked keys left out (their weight is below e^-290), in units of
one rounding of the exact result, as in test_gpu_packed_f16.  P is rounded once and, in bf16, dS once: 1.6 and
1.8.  fp32: scores of 24 products and a bias, and sums over 50 keys, all in fp32: 2^-24 times 60, in norm."""
import math

import pytest
import torch

from test_gpu_packed import F, TYPES, P, gen, normal, run_attention

pytestmark = pytest.mark.gpu


def window64(q, k, v, do, table, buckets, masked, causal):
    n, D = q.shape[0], q.shape[2]
    q, k, v, do = (x.double().transpose(0, 1).contiguous() for x in (q, k, v, do))
    rel = torch.arange(n, device="cuda")[None] - torch.arange(n, device="cuda")[:, None]
    R = buckets.max_distance
    bucket = buckets.lut.cuda().long()[rel.clamp(-R, R) + R]
    S = q @ k.transpose(1, 2).contiguous() * D ** -0.5 + table.double()[bucket].permute(2, 0, 1)
    gone = torch.isin(bucket, torch.tensor(masked, device="cuda")) | ((rel > 0) if causal else torch.zeros_like(rel, dtype=torch.bool))
    W = torch.softmax(S.masked_fill(gone, -math.inf), 2)
    o = W @ v
    dS = W * (do @ v.transpose(1, 2).contiguous() - (do * o).sum(2, keepdim=True))
    dtable = torch.zeros(table.shape, dtype=torch.float64, device="cuda").index_add_(0, bucket.reshape(-1), dS.permute(1, 2, 0).reshape(-1, q.shape[0]))
    out = dict(o=o, dq=dS @ k * D ** -0.5, dk=dS.transpose(1, 2).contiguous() @ q * D ** -0.5, dv=W.transpose(1, 2).contiguous() @ do)
    return {**{name: x.transpose(0, 1) for name, x in out.items()}, "dtable": dtable}


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [24, 128])
@pytest.mark.parametrize("low", [-300.0, -3000.0, -1e4, -3e4, "lowest", -1e9, -math.inf])
def test_a_window_by_a_low_bias(t, causal, D, low):
    if low == -1e9 and t == torch.float16:
        pytest.skip("past the type")
    low = torch.finfo(t).min if low == "lowest" else low
    g = gen(140)
    n = 500
    buckets = P().RelativeBuckets(16, 25, bidirectional=not causal)
    q, k, v, do = (normal(g, n, 3, D, dtype=t) for _ in range(4))
    table = normal(g, 16, 3, dtype=t)
    far = sorted({int(buckets.lut[0]), int(buckets.lut[-1])} - ({int(buckets.lut[-1])} if causal else set()))
    table[far] = low
    got = run_attention(q, k, v, P().PackedSequences([n]), do, table, buckets, causal)
    want = window64(q, k, v, do, table.float().masked_fill(torch.isinf(table), 0.0), buckets, far, causal)
    for name in want:
        assert torch.isfinite(got[name]).all(), name
        off = (got[name].double() - want[name]).norm()
        if t == torch.float32:
            assert off <= 60 * F * want[name].norm(), (name, (off / want[name].norm() / F).item())
        else:
            once = (want[name].to(t).double() - want[name]).norm()
            most = 1.8 if t == torch.bfloat16 and name in ("dq", "dk") else 1.6 if name != "dtable" else 2.2
            assert off <= most * once, (name, (off / once).item())
    assert not got["dtable"][far].any()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_a_bias_that_masks_every_key_gives_zeros(t):
    """Below -11356 (-2^14 in powers of two) a bias masks, whatever the type holds: a query that has nothing else gives
    zeros and no gradient, its neighbours what they give without it."""
    g = gen(141)
    n, D = 90, 32
    buckets = P().RelativeBuckets(4, 2)                     # own position | one behind | before | far behind, far before
    q, k, v, do = (normal(g, n, 2, D, dtype=t) for _ in range(4))
    table = torch.full((4, 2), torch.finfo(t).min, dtype=t, device="cuda")
    table[:, 1] = 0.5
    seqs = P().PackedSequences([n])
    got = run_attention(q, k, v, seqs, do, table, buckets)
    for name in ("o", "dq", "dk", "dv"):
        assert not got[name][:, 0].any(), name
    plain = run_attention(q[:, 1:], k[:, 1:], v[:, 1:], seqs, do[:, 1:])
    once = 2.0 ** -24 * 200 if t == torch.float32 else torch.finfo(t).eps * 2
    for name in ("o", "dq", "dk", "dv"):
        a, b = got[name][:, 1].double(), plain[name][:, 0].double()
        assert (a - b).norm() <= once * b.norm(), name


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [30.0, 1000.0])
def test_keys_that_score_far_below_come_first(t, D, size):
    """The same without a bias: the first 100 keys point away from every query."""
    g = gen(142)
    n = 300
    q, k, v, do = (normal(g, n, 2, D, dtype=torch.float32) for _ in range(4))
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:100, :, 0] = -size * D ** 0.5
    q, k, v, do = (x.to(t) for x in (q, k, v, do))
    got = run_attention(q, k, v, P().PackedSequences([n]), do)
    buckets = P().RelativeBuckets(2, 2, bidirectional=False)
    want = window64(q, k, v, do, torch.zeros(2, 2, device="cuda"), buckets, [], False)
    for name in ("o", "dq", "dk", "dv"):
        rows = slice(100, n) if name in ("dk", "dv") else slice(0, n)      # (nothing reaches the first keys)
        a, b = got[name][rows].double(), want[name][rows]
        cols = slice(1, D) if name == "dq" else slice(0, D)                # (dq's first column is a sum of large terms)
        a, b = a[..., cols], b[..., cols]
        off = (a - b).norm()
        if t == torch.float32:
            assert off <= 60 * F * b.norm(), (name, (off / b.norm() / F).item())
        else:
            assert off <= (1.8 if t == torch.bfloat16 and name in ("dq", "dk") else 1.6) * (b.to(t).double() - b).norm(), name
