"""The bias table's gradient where one bucket holds nearly every key.

A row's dS sum to zero, so what such a bucket gets is the small rest of large terms: an error of the row's mean (rowsum(dO O)
from a rounded O and rounded P) stays whole in it.  In bf16 the mean is summed from P and dP themselves, and
dS enters the table in fp32: the error is the output's own rounding, at most half a step u of each value, and a tenth for
the rest (fp32 sums of up to 10^6 terms of both signs).  In fp16 the mean is rowsum(dO O).  Its error, beside the spread of
a row's dP, is that of two roundings, sqrt(2) u at most, and the bucket of share M keeps M of it where the terms
themselves leave sqrt(M (1 - M)) of that spread: sqrt(2) u sqrt(M / (1 - M)) of the result, twice over for
the few values of a table."""
import pytest
import torch

from test_gpu_packed import P, gen, half_step, normal, run_attention

pytestmark = pytest.mark.gpu


def most(t, table_and_share):
    share = table_and_share[1]
    return 1.1 if t == torch.bfloat16 else 1.1 + 2 * (2 * share / (1 - share)) ** 0.5


def dtable64(q, k, do, v, nq, nk, causal, table, buckets):
    """(the table's gradient, the largest bucket's mean share of a row)"""
    mass, rows = torch.zeros(table.shape[0], device="cuda"), 0
    out, a, b, R, D = torch.zeros(table.shape, dtype=torch.float64, device="cuda"), 0, 0, buckets.max_distance, q.shape[2]
    for m, n in zip(nq, nk):
        rel = torch.arange(n, device="cuda")[None] - (torch.arange(m, device="cuda")[:, None] + n - m)
        bucket = buckets.lut.cuda().long()[rel.clamp(-R, R) + R]
        for h in range(q.shape[1]):
            Q, K, V, G = q[a:a + m, h].double(), k[b:b + n, h].double(), v[b:b + n, h].double(), do[a:a + m, h].double()
            S = Q @ K.T * D ** -0.5 + table.double()[bucket, h]
            W = torch.softmax(S.masked_fill(rel > 0, float("-inf")) if causal else S, 1)
            dP = G @ V.T
            dS = W * (dP - (W * dP).sum(1, keepdim=True))
            for i in range(table.shape[0]):
                out[i, h] += dS[bucket == i].sum()
                mass[i] += W[bucket == i].sum()
            rows += m
        a, b = a + m, b + n
    return out, (mass / rows).max().item()


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lengths,D,heads,count,distance,causal", [
    ([815, 1105, 1103], 16, 6, 8, 512, True),
    ([2473, 309], 24, 4, 32, 64, False),
    ([3001], 64, 4, 8, 100, True),
    ([900, 1, 33], 128, 2, 4, 16, False),
    ([5000], 64, 1, 16, 20, False),
    ([64, 65, 31], 32, 3, 8, 6, True)])
def test_a_bucket_of_nearly_all_keys(t, lengths, D, heads, count, distance, causal):
    g = gen(150)
    T = sum(lengths)
    buckets = P().RelativeBuckets(count, distance, bidirectional=not causal)
    q, k, v = (normal(g, T, heads, D, dtype=t) for _ in range(3))
    do, table = normal(g, T, heads, D, dtype=t, scale=0.05), normal(g, count, heads, dtype=t, scale=0.5)
    got = run_attention(q, k, v, P().PackedSequences(lengths), do, table, buckets, causal)
    want = dtable64(q, k, do, v, lengths, lengths, causal, table, buckets)
    off = (got["dtable"].double() - want[0]).norm() / want[0].norm() / half_step(t)
    assert off <= most(t, want), (off.item(), want[1])


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
def test_the_same_with_few_queries_over_long_keys(t):
    """The keys of a row are split over workgroups."""
    g = gen(151)
    m, n, D = 5, 9001, 64
    buckets = P().RelativeBuckets(16, 200, bidirectional=False)
    q, do = normal(g, m, 2, D, dtype=t), normal(g, m, 2, D, dtype=t)
    k, v = normal(g, n, 2, D, dtype=t), normal(g, n, 2, D, dtype=t)
    table = normal(g, 16, 2, dtype=t, scale=0.5)
    got = run_attention(q, k, v, P().PackedSequences([m], [n]), do, table, buckets, True)
    want = dtable64(q, k, do, v, [m], [n], True, table, buckets)
    off = (got["dtable"].double() - want[0]).norm() / want[0].norm() / half_step(t)
    assert off <= most(t, want), (off.item(), want[1])
