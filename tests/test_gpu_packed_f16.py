"""fp16's small exponent range in packed attention: gradients of very different size in one batch, long keys,
large values.

Errors are measured as norms against the formula in 64 bits, in units of the error that rounding the exact
result to the type makes.  What is allowed besides that one rounding, each part far below it in these cases:
dS enters its products in two fp16 parts (2^-22 of each term, and 2^-37 of the largest dS of its row or
column); rowsum(dO O) takes O rounded (2^-11, averaged over a row's keys); fp32 sums.  So dq and dk stay within 1.2
roundings.  P enters dV in one part: a second rounding of the same size, independent between terms, so dv
stays within sqrt(2), and 1.6 allows for a mantissa distribution that favours it.  bf16's dS enters in one part: 1.8.
"""
import math

import pytest
import torch

from test_gpu_packed import TYPES, P, gen, normal, run_attention

pytestmark = pytest.mark.gpu

ROUNDINGS = {"o": 1.6, "dq": 1.2, "dk": 1.2, "dv": 1.6}


def formula(q, k, v, do, scale, causal=False):
    """One sequence, heads as many as key heads, in 64 bits."""
    q, k, v, do = (x.double().transpose(0, 1).contiguous() for x in (q, k, v, do))
    S = q @ k.transpose(1, 2).contiguous() * scale
    if causal:
        m, n = S.shape[1:]
        S = S.masked_fill(torch.ones(m, n, device="cuda", dtype=torch.bool).triu(n - m + 1), -math.inf)
    W = torch.softmax(S, 2)
    o = W @ v
    dS = W * (do @ v.transpose(1, 2).contiguous() - (do * o).sum(2, keepdim=True))
    out = dict(o=o, dq=dS @ k * scale, dk=dS.transpose(1, 2).contiguous() @ q * scale, dv=W.transpose(1, 2).contiguous() @ do)
    return {name: x.transpose(0, 1) for name, x in out.items()}


def roundings(got, want):
    """The error's norm over the norm of one rounding's error."""
    assert torch.isfinite(got).all()
    once = (want.to(got.dtype).double() - want).norm()
    return ((got.double() - want).norm() / once).item()


@pytest.mark.parametrize("apart", [0, 6, 10, 14])
@pytest.mark.parametrize("causal", [False, True])
def test_a_sequence_with_large_gradients_takes_nothing_from_its_neighbours(apart, causal):
    g = gen(100)
    n, D = [700, 1500], 64
    T = sum(n)
    q, k, v = (normal(g, T, 2, D, dtype=torch.float16) for _ in range(3))
    do = normal(g, T, 2, D, scale=2.0 ** -4)
    do[:n[0]] *= 2.0 ** apart
    do = do.half()
    seqs = P().PackedSequences(n)
    got = run_attention(q, k, v, seqs, do, causal=causal)
    for rows in (slice(0, n[0]), slice(n[0], T)):
        want = formula(q[rows], k[rows], v[rows], do[rows], D ** -0.5, causal)
        for name in want:
            r = roundings(got[name][rows], want[name])
            assert r <= ROUNDINGS[name], (name, rows, r)
    # and not a bit of the second depends on the first's
    do[:n[0]] = 0
    again = run_attention(q, k, v, seqs, do, causal=causal)
    assert all(torch.equal(got[name][n[0]:], again[name][n[0]:]) for name in got)


def test_rows_of_very_different_gradients_in_one_sequence():
    """Under a causal mask keys behind the large rows get small gradients only."""
    g = gen(101)
    n, D, cut = 1024, 64, 500
    q, k, v = (normal(g, n, 1, D, dtype=torch.float16) for _ in range(3))
    do = normal(g, n, 1, D, scale=2.0 ** -4)
    do[:cut] *= 2.0 ** 12
    do = do.half()
    got = run_attention(q, k, v, P().PackedSequences([n]), do, causal=True)
    want = formula(q, k, v, do, D ** -0.5, True)
    for name in ("dq", "dk", "dv"):
        for rows in (slice(0, cut), slice(cut, n)):
            assert roundings(got[name][rows], want[name][rows]) <= ROUNDINGS[name], (name, rows)


@pytest.mark.parametrize("keys,D", [(2047, 64), (8192, 64), (16384, 128), (65536, 128), (65536, 64), (200000, 64)])
def test_gradients_over_long_keys(keys, D):
    """A few queries; dO large enough that the results themselves are normal numbers."""
    g = gen(102)
    m = 40
    q, do = normal(g, m, 1, D, dtype=torch.float16), normal(g, m, 1, D, dtype=torch.float16, scale=64.0)
    k, v = normal(g, keys, 1, D, dtype=torch.float16), normal(g, keys, 1, D, dtype=torch.float16)
    got = run_attention(q, k, v, P().PackedSequences([m], [keys]), do)
    want = formula(q, k, v, do, D ** -0.5)
    for name in ("dq", "dk"):
        r = roundings(got[name], want[name])
        assert r <= ROUNDINGS[name], (name, r)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_other_sequences_are_out_of_reach_in_every_type(t, causal):
    g = gen(103)
    n = [40, 70, 33]
    q, k, v, do = (normal(g, sum(n), 4, 64, dtype=t) for _ in range(4))
    seqs = P().PackedSequences(n)
    clean = run_attention(q, k, v, seqs, do, causal=causal)
    for bad in (float("nan"), float("inf"), torch.finfo(t).min, torch.finfo(t).smallest_normal):
        for which in range(4):
            ins = [x.clone() for x in (q, k, v, do)]
            ins[which][40:110] = bad
            got = run_attention(*ins[:3], seqs, ins[3], causal=causal)
            for name in clean:
                for rows in (slice(0, 40), slice(110, 143)):
                    assert torch.equal(got[name][rows], clean[name][rows]), (name, bad, which)


@pytest.mark.parametrize("D", [64, 128])
def test_large_values_leave_the_gradients_finite(D):
    """Values of +-30000: dP reaches 128 x 30000, far past fp16's range; the gradients do not."""
    g = gen(104)
    n = 120                                               # 60 sequences of two keys: P is near a half
    q = normal(g, n, 2, D, dtype=torch.float16, scale=0.1)
    k = normal(g, n, 2, D, dtype=torch.float16, scale=2.0 ** -9)
    v = torch.where(torch.rand(n, 2, 1, generator=g, device="cuda") < 0.5, -3e4, 3e4).expand(-1, -1, D).contiguous().half()
    do = normal(g, n, 2, D, dtype=torch.float16, scale=0.01, mean=0.5)
    got = run_attention(q, k, v, P().PackedSequences([2] * 60), do)
    parts = [formula(*(x[i:i + 2] for x in (q, k, v, do)), D ** -0.5) for i in range(0, n, 2)]
    want = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    for name in ("dq", "dk"):
        r = roundings(got[name], want[name])
        assert r <= 2 * ROUNDINGS[name], (name, r)


@pytest.mark.parametrize("keys,D", [(2047, 64), (8192, 64), (65536, 128), (200000, 64)])
def test_value_gradients_over_long_keys(keys, D):
    """P is about 1 / keys: below fp16's normal range from 16384 keys on."""
    g = gen(105)
    m = 40
    q, do = normal(g, m, 1, D, dtype=torch.float16), normal(g, m, 1, D, dtype=torch.float16, scale=64.0)
    k, v = normal(g, keys, 1, D, dtype=torch.float16), normal(g, keys, 1, D, dtype=torch.float16)
    got = run_attention(q, k, v, P().PackedSequences([m], [keys]), do)
    want = formula(q, k, v, do, D ** -0.5)
    r = roundings(got["dv"], want["dv"])
    assert r <= ROUNDINGS["dv"], r


@pytest.mark.parametrize("keys,sink", [(16384, 14.0625), (65536, 17.0625), (131072, 17.0625)])
def test_many_keys_far_below_the_largest_score(keys, sink):
    """The first key's score (in powers of two) lies `sink` above all others', which together still hold
    a good part of the sum.  Their P are equal, so its rounding does not average out: one rounding (2^-11) of their
    share at most.  The mean over all results leaves little of the rounding of o itself (rms 2^-11 / 2 over 64 values of
    each row): 2^-13.  (So many rows that the parts' workspace keeps the keys in one walk.)"""
    D, rows = 64, 1 << 17
    q = torch.zeros(rows, 8, D, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    k = torch.zeros(keys, 1, D, dtype=torch.float16, device="cuda")
    k[0, :, 0] = sink
    v = normal(gen(106), keys, 1, D, dtype=torch.float16, mean=2.0, scale=0.1)
    scale = math.log(2.0)
    got = P().packed_attention(q, k, v, P().PackedSequences([rows], [keys]), scale=scale)[:2, :1]
    want = formula(q[:2, :1], k, v, torch.zeros_like(q[:2, :1]), scale)["o"]
    off = (got.double() / want - 1).mean().abs().item() * 2.0 ** 11
    assert off <= 1.25, off
