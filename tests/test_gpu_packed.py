"""Packed-sequence operators on the GPU against plain 64-bit forms.

Tolerances are bounds, computed from the same 64-bit quantities: u is half a step of the tensors'
type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), f = 2^-24 that of fp32.
Attention.  A score sums D products in fp32 (error <= D f sum|q||k| scale, and a few roundings of the
score itself), so P carries twice that; P enters its product rounded to the type (u), fp32 sums of at
most n terms add n f (the worst case, never met).  dS = P (dP - D): dP likewise, D is the sum of dO O with
O rounded to the type (u sum|dO||O|).  fp16's dS is scaled to half its range's size; below its normal
range it is off by half of 2^-24, in units of 8 max|dO|.
Small values.  An output in a type's subnormal range is off by half its smallest step (fp16: 2^-25), and the
hardware's exp2 returns 0 for a P below 2^-126; no sum here has 2^20 such terms of size 1, so 2^-100 covers them.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
F = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half a step in the subnormal range (fp16), or what flushed probabilities leave."""
    return max(torch.finfo(t).smallest_normal * half_step(t), 2.0 ** -100)


def P():
    from VAESNe import PackedLayers
    return PackedLayers


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)


# ------------------------------------------------------------------------------------------------
# attention: formulas and bounds in 64 bits, a sequence and head at a time
# ------------------------------------------------------------------------------------------------
def oracle(q, k, v, nq, nk, causal, scale, do=None, table=None, lut=None):
    """{name: (value, bound)}"""
    t = q.dtype
    u, D = half_step(t), q.shape[2]
    up = u if t != torch.float32 else 0.0              # rounding of P and dS before their products
    q, k, v = q.double(), k.double(), v.double()
    G = q.shape[1] // k.shape[1]
    z = torch.zeros_like
    out = {"o": [z(q), z(q)]}
    if do is not None:
        do = do.double()
        out.update(dq=[z(q), z(q)], dk=[z(k), z(k)], dv=[z(k), z(k)])
        if table is not None:
            out["dtable"] = [torch.zeros(table.shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    a = b = 0
    for m, n in zip(nq, nk):
        rel = torch.arange(n, device="cuda")[None] - (torch.arange(m, device="cuda")[:, None] + n - m)
        for h in range(q.shape[1]):
            if m == 0 or n == 0:
                continue
            Q, K, V = q[a:a + m, h], k[b:b + n, h // G], v[b:b + n, h // G]
            S = Q @ K.T * scale
            mag = (Q.abs() @ K.T.abs()) * scale
            if table is not None:
                R = (len(lut) - 1) // 2
                bucket = lut.long()[rel.clamp(-R, R) + R]
                S = S + table.double()[bucket, h]
                mag = mag + table.double()[bucket, h].abs()
            if causal:
                S = S.masked_fill(rel > 0, float("-inf"))
            W = torch.softmax(S, 1).nan_to_num(0.0)
            # the score, its exponent's product and sum, exp2 (a few f each); the normalising sum likewise
            es = ((D + 8) * F * mag).amax(1, keepdim=True) * 2 + 8 * F
            acc = (n + 16) * F
            O = W @ V
            out["o"][0][a:a + m, h] = O
            eo = (es + up + acc) * (W @ V.abs())
            out["o"][1][a:a + m, h] = eo + u * O.abs()
            if do is None:
                continue
            g = do[a:a + m, h]
            dP = g @ V.T
            D0 = (g * O).sum(1, keepdim=True)
            ed = (D + 8) * F * (g.abs() @ V.abs().T) + (g.abs() * (eo + u * O.abs() + D * F * O.abs())).sum(1, keepdim=True)
            dS = W * (dP - D0)
            E = W * (es * (dP - D0).abs() + ed) + 4 * F * dS.abs()
            tiny = 2.0 ** -25 * 16 * do.abs().max() if t == torch.float16 else 0.0
            Er = E + up * dS.abs() + tiny * (W > 0)
            racc = (m * G + 16) * F
            for name, val, err in (("dq", dS @ K * scale, (Er + acc * dS.abs()) @ K.abs() * scale),
                                   ("dk", dS.T @ Q * scale, (Er + racc * dS.abs()).T @ Q.abs() * scale),
                                   ("dv", W.T @ g, ((es + up + racc) * W + (2.0 ** -25 if t == torch.float16 else 0.0)).T @ g.abs())):
                at = (slice(a, a + m), h) if name == "dq" else (slice(b, b + n), h // G)
                out[name][0][at] += val
                out[name][1][at] += err
            if table is not None:
                idx = bucket.reshape(-1)
                out["dtable"][0][:, h].index_add_(0, idx, dS.reshape(-1))
                out["dtable"][1][:, h].index_add_(0, idx, (E + (m + n + 64) * F * dS.abs()).reshape(-1))
        a, b = a + m, b + n
    for name in out:
        out[name][1] += smallest(t)
        if name != "o":
            out[name][1] += u * out[name][0].abs() * (1 + G)
    return out


def check(got, want, what=""):
    val, bound = want
    assert got.shape == val.shape
    over = (got.double() - val).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 0, f"{what}: {worst:.3g} past the bound"


def run_attention(q, k, v, seqs, do=None, table=None, buckets=None, causal=False, scale=None):
    leaves = [x.detach().requires_grad_(do is not None) for x in (q, k, v)]
    tab = None if table is None else table.detach().requires_grad_(do is not None)
    o = P().packed_attention(*leaves, seqs, causal=causal, scale=scale, bias=tab, buckets=buckets)
    out = {"o": o.detach()}
    if do is not None:
        grads = torch.autograd.grad(o, leaves + ([] if tab is None else [tab]), do)
        out.update(zip(("dq", "dk", "dv", "dtable"), grads))
    return out


def compare_attention(nq, nk, Hq, Hkv, D, t, causal, seed=0, buckets=None, scale=None, g_scale=0.3, amp=1.0):
    g = gen(seed)
    q = normal(g, sum(nq), Hq, D, dtype=t, scale=amp)
    k, v = normal(g, sum(nk), Hkv, D, dtype=t, scale=amp), normal(g, sum(nk), Hkv, D, dtype=t)
    do = normal(g, sum(nq), Hq, D, dtype=t, scale=g_scale)
    table = None if buckets is None else normal(g, buckets.num_buckets, Hq, dtype=t, scale=0.7)
    seqs = P().PackedSequences(nq, nk)
    got = run_attention(q, k, v, seqs, do, table, buckets, causal, scale)
    want = oracle(q, k, v, nq, nk, causal, scale or D ** -0.5, do, table, None if buckets is None else buckets.lut.cuda())
    for name in want:
        check(got[name], want[name], name)
    return got


LENGTHS = {
    "one": ([1], [1]),
    "ragged": ([1, 31, 33, 64, 65, 127, 130], [1, 31, 33, 64, 65, 127, 130]),
    "empty": ([0, 5, 0, 3, 0], [0, 5, 7, 3, 0]),
    "few_long": ([1, 8, 3], [700, 1000, 3]),
    "more_queries": ([40, 70, 5], [3, 64, 0]),
}


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 8), (4, 2, 64), (6, 2, 24), (8, 1, 128)])
def test_attention_matches_formula(t, causal, lengths, Hq, Hkv, D):
    nq, nk = LENGTHS[lengths]
    got = compare_attention(nq, nk, Hq, Hkv, D, t, causal, seed=1)
    if lengths == "more_queries" and causal:          # queries that see nothing: zeros, no gradient
        assert not got["o"][:37].any() and not got["dq"][:37].any()
        assert not got["o"][-5:].any() and not got["dq"][-5:].any()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [16, 32, 40, 48, 80, 96, 112])
def test_attention_head_dims(t, D):
    compare_attention([70, 33], [70, 90], 4, 2, D, t, True, seed=2)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("G", [3, 5, 7, 12, 32, 48])
def test_attention_group_sizes(t, G):
    compare_attention([1, 37], [150, 37], G * 2, 2, 32, t, True, seed=3)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_long(t, causal):
    # several tiles of every kind, splits in every kernel
    compare_attention([1500], [1500], 2, 1, 64, t, causal, seed=4)
    compare_attention([1, 2], [3001, 40], 4, 1, 128, t, causal, seed=5)
    compare_attention([2000, 1], [9, 1], 2, 2, 128, t, False, seed=6)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("amp,g", [(6.0, 1.0), (0.01, 1e-3), (1.0, 30.0)])
def test_attention_magnitudes(t, amp, g):
    # sharp and flat softmax, small and large gradients (fp16: scaled dS)
    compare_attention([150], [150], 2, 2, 64, t, True, seed=7, amp=amp, g_scale=g)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("count,distance", [(32, 128), (8, 5), (64, 512), (4, 3)])
@pytest.mark.parametrize("lengths", [([1, 33, 200, 64], [1, 33, 200, 64]), ([5, 0, 40], [300, 3, 20]), ([700], [700])])
def test_bias_matches_formula(t, causal, count, distance, lengths):
    b = P().RelativeBuckets(count, distance, bidirectional=not causal)
    compare_attention(*lengths, 4, 2, 32, t, causal, seed=8, buckets=b)


@pytest.mark.parametrize("D", [8, 64, 128])
def test_bias_both_ways_under_a_causal_mask(D):
    b = P().RelativeBuckets(16, 40, bidirectional=True)
    compare_attention([130, 257], [130, 257], 3, 3, D, torch.bfloat16, True, seed=9, buckets=b)


def test_bias_spans_many_tiles():
    b = P().RelativeBuckets(32, 128, bidirectional=True)
    compare_attention([1300], [1300], 1, 1, 16, torch.float32, False, seed=10, buckets=b)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_reads_strided_tensors(t):
    g = gen(11)
    n = [50, 77]
    T = sum(n)
    qkv = normal(g, T, 8 + 2 * 2, 32, dtype=t)
    q, k, v = qkv.split([8, 2, 2], 1)
    headmajor = normal(g, 8, T, 32, dtype=t).transpose(0, 1)
    seqs = P().PackedSequences(n)
    do = normal(g, T, 8, 32, dtype=t)
    for qq, dd in ((q, do), (headmajor, do), (q[..., :24], do[..., :24]), (q, headmajor),
                   (q, torch.ones((), dtype=t, device="cuda").expand(T, 8, 32))):
        D = qq.shape[2]
        kk, vv = k[..., :D], v[..., :D]
        got = run_attention(qq, kk, vv, seqs, dd, causal=True)
        want = oracle(qq, kk, vv, n, n, True, D ** -0.5, dd)
        for name in want:
            check(got[name], want[name], name)
    odd = normal(g, T * 8 * 32 + 3, dtype=t)[3:].view(T, 8, 32)       # rows off the 16-byte grid: copied
    check(run_attention(odd, k, v, seqs)["o"], oracle(odd, k, v, n, n, False, 32 ** -0.5)["o"])


def test_attention_broadcast_key_heads():
    g = gen(12)
    n = [65, 20]
    kv = normal(g, sum(n), 1, 64, dtype=torch.bfloat16)
    q = normal(g, sum(n), 4, 64, dtype=torch.bfloat16)
    do = normal(g, sum(n), 4, 64, dtype=torch.bfloat16)
    seqs = P().PackedSequences(n)
    leaf = kv.detach().requires_grad_()
    o = P().packed_attention(q, leaf.expand(-1, 4, -1), leaf.expand(-1, 4, -1), seqs)
    d, = torch.autograd.grad(o, leaf, do)
    want = oracle(q, kv, kv, n, n, False, 1 / 8, do)
    check(o.detach(), want["o"])
    val = want["dk"][0] + want["dv"][0]
    # autograd sums the four heads' rounded gradients and the two tensors' in bf16: seven more roundings
    per_head = oracle(q, kv.expand(-1, 4, -1), kv.expand(-1, 4, -1), n, n, False, 1 / 8, do)
    size = (per_head["dk"][0].abs() + per_head["dv"][0].abs()).sum(1, keepdim=True)
    check(d, (val, want["dk"][1] + want["dv"][1] + 8 * half_step(torch.bfloat16) * size))


def test_other_sequences_and_rows_behind_are_out_of_reach():
    g = gen(13)
    n = [40, 70, 33]
    q, k, v, do = (normal(g, sum(n), 2, 64, dtype=torch.bfloat16) for _ in range(4))
    seqs = P().PackedSequences(n)
    clean = run_attention(q, k, v, seqs, do, causal=True)
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        q2, k2, v2, do2 = (x.clone() for x in (q, k, v, do))
        for x in (q2, k2, v2, do2):
            x[40:110] = bad
        got = run_attention(q2, k2, v2, seqs, do2, causal=True)
        for name in clean:
            for rows in (slice(0, 40), slice(110, 143)):
                assert torch.equal(got[name][rows], clean[name][rows]), (name, bad)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_is_bitwise_reproducible_and_the_same_without_gradients(t):
    g = gen(14)
    n, b = [300, 1, 77], P().RelativeBuckets(32, 64)
    q, k, v, do = (normal(g, sum(n), 4, 64, dtype=t) for _ in range(4))
    table = normal(g, 32, 4, dtype=t)
    seqs = P().PackedSequences(n)
    first = run_attention(q, k, v, seqs, do, table, b)
    for _ in range(3):
        again = run_attention(q, k, v, seqs, do, table, b)
        assert all(torch.equal(first[x], again[x]) for x in first)
    assert torch.equal(run_attention(q, k, v, seqs, None, table, b)["o"], first["o"])


def test_gradients_against_differences():
    """Along a direction d, (f(x + e d) - f(x - e d)) / 2e: its own error is e^2 / 6 of the third
    derivative (below 1e-4 here, as the 64-bit differences of the formula confirm) and 2^-24 |f| / e of
    rounding."""
    g = gen(15)
    n, D = [20, 9], 16
    b = P().RelativeBuckets(8, 6)
    seqs = P().PackedSequences(n)
    x = [normal(g, sum(n), 2, D) for _ in range(3)] + [normal(g, 8, 2)]
    do = normal(g, sum(n), 2, D)
    got = run_attention(x[0], x[1], x[2], seqs, do, x[3], b)

    def f(xs):
        o = run_attention(xs[0], xs[1], xs[2], seqs, None, xs[3], b)["o"]
        return (o.double() * do.double()).sum().item()

    def exact(xs):
        w = oracle(xs[0], xs[1], xs[2], n, n, False, D ** -0.5, None, xs[3], b.lut.cuda())["o"][0]
        return (w * do.double()).sum().item()
    e = 1e-2
    for i, name in enumerate(("dq", "dk", "dv", "dtable")):
        d = normal(g, *x[i].shape)
        moved = [[y + s * e * d if i == j else y for j, y in enumerate(x)] for s in (1, -1)]
        slope = (got[name].double() * d.double()).sum().item()
        size = (do.abs().sum() * 4).item()
        assert abs((exact(moved[0]) - exact(moved[1])) / (2 * e) - slope) <= 2e-3 * max(1.0, abs(slope)) + 1e-3
        assert abs((f(moved[0]) - f(moved[1])) / (2 * e) - slope) <= 2e-3 * max(1.0, abs(slope)) + 1e-3 + size * 2.0 ** -22 / e


def test_attention_refuses():
    g = gen(16)
    L = P()
    seqs = L.PackedSequences([5, 6])
    q, k = normal(g, 11, 4, 16), normal(g, 11, 2, 16)
    b = L.RelativeBuckets(8, 6)
    for err, call in (
            (ValueError, lambda: L.packed_attention(q[:10], k, k, seqs)),
            (ValueError, lambda: L.packed_attention(q, k[:10], k[:10], seqs)),
            (ValueError, lambda: L.packed_attention(q, k, k[:, :1], seqs)),
            (ValueError, lambda: L.packed_attention(q[:, :3], k, k, seqs)),
            (ValueError, lambda: L.packed_attention(q[..., :12], k[..., :12], k[..., :12], seqs)),
            (ValueError, lambda: L.packed_attention(normal(g, 11, 4, 136), normal(g, 11, 2, 136), normal(g, 11, 2, 136), seqs)),
            (ValueError, lambda: L.packed_attention(q, k, k, seqs, scale=0.0)),
            (ValueError, lambda: L.packed_attention(q, k, k, seqs, scale=float("inf"))),
            (ValueError, lambda: L.packed_attention(q, k, k, seqs, buckets=b)),
            (ValueError, lambda: L.packed_attention(q, k, k, seqs, bias=normal(g, 8, 3), buckets=b)),
            (TypeError, lambda: L.packed_attention(q, k, k.half(), seqs)),
            (TypeError, lambda: L.packed_attention(q, k, k, seqs, bias=normal(g, 8, 4).half(), buckets=b)),
            (TypeError, lambda: L.packed_attention(q.double(), k.double(), k.double(), seqs)),
            (TypeError, lambda: L.packed_attention(q, k, k, [5, 6])),
            (RuntimeError, lambda: L.packed_attention(q.cpu(), k, k, seqs)),
            (RuntimeError, lambda: seqs.pack(q))):
        with pytest.raises(err):
            call()
    o = L.packed_attention(q.requires_grad_(), k, k, seqs)
    d, = torch.autograd.grad(o.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):                      # no second derivatives
        d.sum().backward()


def test_nothing_at_all():
    L = P()
    seqs = L.PackedSequences([])
    q = torch.empty(0, 2, 16, device="cuda", requires_grad=True)
    o = L.packed_attention(q, q, q, seqs)
    assert o.shape == (0, 2, 16) and torch.autograd.grad(o.sum(), q)[0].shape == (0, 2, 16)
    b = L.RelativeBuckets(8, 6)
    table = torch.ones(8, 2, device="cuda", requires_grad=True)
    o = L.packed_attention(q, q, q, seqs, bias=table, buckets=b)
    assert not torch.autograd.grad(o.sum(), table)[0].any()
    # keys without queries: their gradients are zeros
    seqs = L.PackedSequences([0, 0], [3, 70])
    k = torch.randn(73, 2, 16, device="cuda", requires_grad=True)
    o = L.packed_attention(q, k, k, seqs, bias=table, buckets=b)
    dk, dt = torch.autograd.grad(o.sum(), (k, table))
    assert not dk.any() and not dt.any()


def test_pack_and_unpack_a_padded_batch():
    g = gen(17)
    L = P()
    mask = torch.ones(4, 9, dtype=torch.bool, device="cuda")
    for i, n in enumerate((9, 1, 0, 5)):
        mask[i, :n] = False
    mask[3, 2] = True                                      # an observation left out in the middle
    seqs = L.PackedSequences.from_mask(mask)
    assert seqs.lengths == [9, 1, 0, 4]
    x = normal(g, 4, 9, 3).requires_grad_()
    p = seqs.pack(x)
    assert torch.equal(p, x[~mask])
    back = seqs.unpack(p)
    assert torch.equal(back, x * ~mask[..., None])
    d, = torch.autograd.grad(back.sum(), x)
    assert torch.equal(d, (~mask[..., None]).float().expand_as(x))
    with pytest.raises(ValueError):
        seqs.pack(x[:, :8])
    with pytest.raises(ValueError):
        seqs.unpack(p[:-1])


# ------------------------------------------------------------------------------------------------
# gated norm
# ------------------------------------------------------------------------------------------------
def norm64(x, kind, eps=1e-5):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def join64(x, f, w2, w1, b2, b1, gate, c, kind):
    u = norm64(f, kind) * w1 + (0 if b1 is None else b1)
    y = c * x + (u if gate is None else gate * u)
    return y, norm64(y, kind) * w2 + (0 if b2 is None else b2)


def join_case(rows, C, t, kind, gate, c, seed, lead=None):
    g = gen(seed)
    shape = (rows, C) if lead is None else (*lead, C)
    ts = dict(x=normal(g, *shape, dtype=t), branch=normal(g, *shape, dtype=t, scale=0.5, mean=0.2),
              pre_weight=normal(g, C, dtype=t, scale=0.2, mean=1.0), post_weight=normal(g, C, dtype=t, scale=0.2, mean=1.0),
              pre_bias=None, post_bias=None, gate=None)
    if kind == "layer":
        ts["pre_bias"], ts["post_bias"] = normal(g, C, dtype=t), normal(g, C, dtype=t)
    if gate != "none":
        ts["gate"] = normal(g, *((C,) if gate == "channel" else shape), dtype=t, scale=0.5, mean=0.3)
    return ts, normal(g, *shape, dtype=t), normal(g, *shape, dtype=t)


def join_compare(ts, dy, dn, c, kind, use=("y", "n")):
    leaves = {k: v.detach().requires_grad_() for k, v in ts.items() if v is not None}
    args = {k: leaves.get(k) for k in ts}
    y, n = P().gated_norm(**args, residual_scale=c, kind=kind)
    outs, gs = zip(*[(o, d) for k, o, d in (("y", y, dy), ("n", n, dn)) if k in use])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs)))
    ref = {k: v.detach().double().requires_grad_() for k, v in leaves.items()}
    ra = {k: ref.get(k) for k in ts}
    ry, rn = join64(ra["x"], ra["branch"], ra["pre_weight"], ra["post_weight"], ra["pre_bias"], ra["post_bias"], ra["gate"], c, kind)
    router, rgs = zip(*[(o, d.double()) for k, o, d in (("y", ry, dy), ("n", rn, dn)) if k in use])
    # (dy alone leaves the second norm's parameters out: zeros)
    rg = torch.autograd.grad(router, list(ref.values()), rgs, allow_unused=True)
    rgrads = {k: torch.zeros_like(v) if d is None else d for (k, v), d in zip(ref.items(), rg)}
    C = ts["x"].shape[-1]
    rows = max(1, ts["x"].numel() // C)
    u = half_step(ts["x"].dtype)
    # fp32 arithmetic: sums over a row pass 8 to 16 serial and 8 tree additions; means, squares, root and
    # quotient a few more: 64 f of the row's largest magnitude covers them, twice over for the second norm,
    # and the backward's two projections again.  A column sum adds rows / 512 + 16 + 16 terms serially.
    big = lambda r: r.abs().amax(-1, keepdim=True) if r.dim() > 1 or r.shape == ts["x"].shape else r.abs().max()   # noqa: E731
    for name, got, want in (("y", y, ry), ("n", n, rn)):
        spread = 1 + big(want) if name == "y" else 1 + big(want) * (1 + big(ry.detach()))
        assert ((got.double() - want).abs() <= u * want.abs() + 256 * F * spread).all(), name
    stats = (1 + ts["pre_weight"].double().abs().max()) * (1 + (0 if ts["gate"] is None else ts["gate"].double().abs().max()))
    scale = (1 + dy.double().abs().max() + dn.double().abs().max()) * stats * (1 + rgrads["branch"].abs().max())
    for name in leaves:
        want = rgrads[name]
        tol = 512 * F * scale * (1 + (rows / 512 + 32 if want.dim() == 1 and ts["x"].dim() > 1 else 0) * 4)
        assert torch.isfinite(grads[name]).all()
        assert ((grads[name].double() - want).abs() <= u * want.abs() + tol).all(), (name, (grads[name].double() - want).abs().max().item(), tol)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("rows,C", [(1, 8), (33, 32), (70, 33), (5, 1), (129, 64), (17, 520), (9, 1024), (6, 2048)])
def test_join_matches_formula(t, kind, gate, rows, C):
    ts, dy, dn = join_case(rows, C, t, kind, gate, 0.5, seed=20)
    join_compare(ts, dy, dn, 0.5, kind)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("C", [256, 257, 1000, 2047, 2056, 2049, 4096, 4104, 8191, 8192])
def test_join_widths(t, C):
    for kind, gate in (("rms", "token"), ("layer", "channel")):
        ts, dy, dn = join_case(3, C, t, kind, gate, 1.0, seed=21)
        join_compare(ts, dy, dn, 1.0, kind)


def test_join_many_rows_and_leading_axes():
    ts, dy, dn = join_case(0, 32, torch.float32, "layer", "channel", 1.0, 22, lead=(7, 3, 211))
    join_compare(ts, dy, dn, 1.0, "layer")
    ts, dy, dn = join_case(5000, 48, torch.bfloat16, "rms", "token", 1.0, 23)
    join_compare(ts, dy, dn, 1.0, "rms")


@pytest.mark.parametrize("use", ["y", "n"])
@pytest.mark.parametrize("C", [32, 600, 2304])
def test_join_with_one_output_used(use, C):
    ts, dy, dn = join_case(40, C, torch.float32, "layer", "token", 0.7, 24)
    join_compare(ts, dy, dn, 0.7, "layer", use=(use,))


def test_join_strided_rows_and_expanded_gradients():
    g = gen(25)
    wide = normal(g, 50, 128, dtype=torch.bfloat16)
    ts, dy, dn = join_case(50, 64, torch.bfloat16, "rms", "token", 1.0, 25)
    ts["x"], ts["gate"] = wide[:, :64], wide[:, 64:]
    join_compare(ts, dy, dn, 1.0, "rms")
    join_compare(ts, dy[:1].expand(50, 64), dn, 1.0, "rms")
    ts["x"] = wide[:, 3:67]                               # rows off the 16-byte grid: one element at a time
    join_compare(ts, dy, dn, 1.0, "rms")


@pytest.mark.parametrize("C", [32, 300, 2304])
def test_pre_norm(C):
    g = gen(26)
    for kind in ("rms", "layer"):
        x, w = normal(g, 37, C).requires_grad_(), normal(g, C, mean=1.0).requires_grad_()
        b = normal(g, C).requires_grad_() if kind == "layer" else None
        d = normal(g, 37, C)
        n = P().pre_norm(x, w, b, kind=kind)
        leaves = [x, w] + ([b] if b is not None else [])
        grads = torch.autograd.grad(n, leaves, d)
        ref = [v.detach().double().requires_grad_() for v in leaves]
        rn = norm64(ref[0], kind) * ref[1] + (ref[2] if b is not None else 0)
        rg = torch.autograd.grad(rn, ref, d.double())
        assert (n - rn).abs().max() <= 256 * F * (1 + rn.abs().max())
        for a, r in zip(grads, rg):
            assert (a - r).abs().max() <= 2048 * F * (1 + r.abs().max())


def test_join_rows_do_not_mix_and_repeat_bitwise():
    ts, dy, dn = join_case(64, 32, torch.bfloat16, "layer", "token", 1.0, 27)
    with torch.no_grad():
        y, n = P().gated_norm(**ts, kind="layer")
        bad = {**ts, "x": ts["x"].clone()}
        bad["x"][7] = float("nan")
        y2, n2 = P().gated_norm(**bad, kind="layer")
    keep = torch.arange(64, device="cuda") != 7
    assert torch.equal(y[keep], y2[keep]) and torch.equal(n[keep], n2[keep]) and n2[7].isnan().all()

    def grads():
        leaves = [ts[k].detach().requires_grad_() for k in ts]
        o = P().gated_norm(*leaves[:4], pre_bias=leaves[4], post_bias=leaves[5], gate=leaves[6], kind="layer")
        return torch.autograd.grad(o, leaves, [dy, dn])
    first = grads()
    assert all(torch.equal(a, b) for a, b in zip(first, grads()))


def test_join_refuses():
    L = P()
    x, w = torch.randn(4, 16, device="cuda"), torch.ones(16, device="cuda")
    for err, call in ((ValueError, lambda: L.gated_norm(x, x[:2], w, w)), (ValueError, lambda: L.gated_norm(x, x, w[:8], w)),
                      (ValueError, lambda: L.gated_norm(x, x, w, w, gate=x[:2])),
                      (ValueError, lambda: L.gated_norm(x, x, w, w, kind="group")),
                      (ValueError, lambda: L.gated_norm(x, x, w, w, pre_bias=w)),
                      (ValueError, lambda: L.gated_norm(x, x, w, w, eps=0.0)),
                      (ValueError, lambda: L.gated_norm(x, x, w, w, residual_scale=float("nan"))),
                      (ValueError, lambda: L.pre_norm(torch.randn(2, 8193, device="cuda"), torch.ones(8193, device="cuda"))),
                      (TypeError, lambda: L.gated_norm(x, x.half(), w, w)), (TypeError, lambda: L.pre_norm(x.double(), w.double())),
                      (RuntimeError, lambda: L.gated_norm(x, x, w.cpu(), w))):
        with pytest.raises(err):
            call()
    e = torch.empty(0, 16, device="cuda", requires_grad=True)
    y, n = L.gated_norm(e, e, w.requires_grad_(), w)
    dw, = torch.autograd.grad(n.sum() + y.sum(), w)
    assert y.shape == (0, 16) and not dw.any()


# ------------------------------------------------------------------------------------------------
# activations in 8 bits
# ------------------------------------------------------------------------------------------------
def eight_bits(x):
    """(values, codes) of x's 8-bit form, in 64 bits."""
    flat = x.detach().double().reshape(-1)
    b = torch.nn.functional.pad(flat, (0, -flat.numel() % 32)).reshape(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    step = torch.exp2((torch.frexp(top)[1].double() - 1).clamp(min=-126) - 6)
    codes = (b / step).round().clamp(-127, 127)
    codes = torch.where(torch.isfinite(b).all(1, keepdim=True), codes, float("nan"))
    return (codes * step).reshape(-1)[:flat.numel()].reshape(x.shape), codes.reshape(-1)[:flat.numel()]


SPECIAL = [0.0, -0.0, 1e-45, -1e-40, 2.0 ** -126, 1.0, -1.0, 127.5, 126.5, 0.5, 1.9999999, 3e38, -3e38]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 7, 8, 31, 32, 33, 64, 1000, 2048, 2049, 70001])
def test_pack8_is_exact(t, n):
    g = gen(30)
    x = normal(g, n, dtype=torch.float32) * torch.exp2(normal(g, n) * 8).clamp(2.0 ** -20, 2.0 ** 12)
    x[::5] = 0
    k = min(n, len(SPECIAL))
    x[:k] = torch.tensor(SPECIAL[:k], device="cuda")
    x = x.clamp(-torch.finfo(t).max, torch.finfo(t).max).to(t)
    for y in (x, x.flip(0), torch.zeros_like(x)):
        p = P().pack8(y)
        want, codes = eight_bits(y)
        assert torch.equal(p.codes.double(), codes)
        assert p.codes.shape == (n,) and p.exponents.shape == ((n + 31) // 32,)
        back = P().unpack8(p)
        assert back.dtype == t and torch.equal(back, want.to(t))
        assert ((back.double() - y.double()).abs() <= want.abs() * 0 + torch.exp2(p.exponents.double().repeat_interleave(32)[:n] - 133)).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_pack8_marks_blocks_with_infinities_and_nan(t):
    x = torch.ones(200, dtype=t, device="cuda")
    x[40], x[100], x[199] = float("inf"), float("nan"), float("-inf")
    back = P().unpack8(P().pack8(x))
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    for a in (32, 96, 192):
        bad[a:a + 32] = True
    assert torch.equal(back.isnan(), bad) and (back[~bad] == 1).all()


def test_pack8_shapes_and_unaligned_tensors():
    g = gen(31)
    x = normal(g, 7, 5, 33)
    for y in (x, x.transpose(0, 2), x[1:, 1:, 1:], x.reshape(-1)[1:], x[:0]):
        want, _ = eight_bits(y.contiguous())
        back = P().unpack8(P().pack8(y))
        assert back.shape == y.shape and torch.equal(back, want.float())


def gelu64(x):
    return x * torch.special.ndtr(x)


def slope64(x):
    return torch.special.ndtr(x) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1,), (3, 33), (64, 96), (1000, 7)])
def test_gelu8(t, shape):
    """The distribution function is within 1.5e-7 / 2 of exact for 16-bit types (Abramowitz & Stegun
    7.1.26) and a few f for fp32; its products and exponential add a few f of x."""
    g = gen(32)
    x = (normal(g, *shape) * 3).to(t).requires_grad_()
    dy = normal(g, *shape, dtype=t)
    y = P().gelu8(x)
    d, = torch.autograd.grad(y, x, dy)
    u = half_step(t)
    want = gelu64(x.double())
    assert ((y.double() - want).abs() <= u * want.abs() + (1e-7 + 16 * F) * (1 + x.double().abs()) + smallest(t)).all()
    kept, _ = eight_bits(x)
    slope = slope64(kept)
    want = dy.double() * slope
    assert ((d.double() - want).abs() <= u * want.abs() + (1e-7 + 16 * F) * dy.double().abs() * (1 + kept.abs()) + smallest(t)).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_act8_without_gradients_is_the_same(t):
    g = gen(34)
    x, W, b = normal(g, 9, 50, dtype=t), normal(g, 20, 50, dtype=t), normal(g, 20, dtype=t)
    leaf = x.detach().requires_grad_()
    assert torch.equal(P().gelu8(x), P().gelu8(leaf))
    for act in (None, "gelu"):
        assert torch.equal(P().linear8(x, W, b, act=act), P().linear8(leaf, W, b, act=act))
    assert torch.equal(P().gelu8(x.t()), P().gelu8(x).t())


def test_gelu8_far_out():
    x = torch.tensor([float("-inf"), -30.0, -6.0, 0.0, 6.0, 30.0, float("inf"), float("nan")], device="cuda")
    for t in TYPES:
        y = P().gelu8(x.to(t)).double()
        assert y[0] == 0 and abs(y[1]) < 1e-6 and abs(y[2]) < 1e-6 and y[3] == 0 and y[5] == 30 and y[6] == float("inf")
        assert y[7].isnan()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear8(t, act):
    """The products are the library's (fp32 sums of K terms: K f, rounded to the type); their operands
    are the 8-bit form's values, rounded to the type once more by GELU."""
    g = gen(33)
    x = normal(g, 2, 30, 72, dtype=t).requires_grad_()
    W = normal(g, 40, 72, dtype=t, scale=0.2).requires_grad_()
    b = normal(g, 40, dtype=t).requires_grad_()
    do = normal(g, 2, 30, 40, dtype=t)
    out = P().linear8(x, W, b, act=act)
    dx, dW, db = torch.autograd.grad(out, (x, W, b), do)
    u = half_step(t)
    up = u if t != torch.float32 else 0.0
    X, K, Wd, G = x.double(), eight_bits(x)[0], W.double(), do.double()
    y, ky = (gelu64(X), gelu64(K)) if act else (X, K)
    slack = lambda a, b, n: (n + 32) * F * (a.abs() @ b.abs()) + (up + 1e-6) * (a.abs() @ b.abs())    # noqa: E731
    want = y @ Wd.T + b.double()
    assert ((out.double() - want).abs() <= u * want.abs() + slack(y, Wd.T, 72) + (72 * 1e-6 if act else 0)).all()
    g2, k2 = G.reshape(60, 40), ky.reshape(60, 72)
    want = g2.T @ k2
    assert ((dW.double() - want).abs() <= u * want.abs() + slack(g2.T, k2, 60) + (1e-5 if act else 0)).all()
    want = g2.sum(0)
    assert ((db.double() - want).abs() <= u * want.abs() + 100 * F * g2.abs().sum(0)).all()
    dy = G @ Wd
    want = dy * slope64(K) if act else dy
    assert ((dx.double() - want).abs() <= 3 * u * want.abs() + 2 * slack(G, Wd, 40) + 1e-6).all()


def test_act8_refuses():
    L = P()
    x = torch.randn(4, 8, device="cuda")
    for err, call in ((TypeError, lambda: L.gelu8(x.double())), (TypeError, lambda: L.pack8(x.int())),
                      (TypeError, lambda: L.linear8(x, x.half())), (ValueError, lambda: L.linear8(x, x[:, :4])),
                      (ValueError, lambda: L.linear8(x, x, act="relu")), (ValueError, lambda: L.linear8(x, x, x[0]))):
        with pytest.raises(err):
            call()


# ------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------
class Keep8(torch.autograd.Function):
    """act(x) forward, act'(8-bit x) backward, in 64 bits; `kept` in place of x for what follows backward."""

    @staticmethod
    def forward(ctx, x, W, b, act):
        ctx.save_for_backward(eight_bits(x.float())[0], W)
        ctx.act = act
        return (gelu64(x) if act else x) @ W.T + b

    @staticmethod
    def backward(ctx, g):
        k, W = ctx.saved_tensors
        y = gelu64(k) if ctx.act else k
        dx = g @ W
        return (dx * slope64(k) if ctx.act else dx), g.T @ y, g.sum(0), None


def block64(block, p, x, nq, causal, lut):
    kind = block.kind
    H, Hk, D = block.num_heads, block.num_kv_heads, block.head_dim

    def attend(q, k, v):
        outs, a = [], 0
        for m in nq:
            rel = torch.arange(m, device="cuda")[None] - torch.arange(m, device="cuda")[:, None]
            R = (len(lut) - 1) // 2
            bias = p["relative.weight"][lut.long()[rel.clamp(-R, R) + R]].permute(2, 0, 1)
            qq = q[a:a + m].transpose(0, 1)
            kk = k[a:a + m].transpose(0, 1).repeat_interleave(H // Hk, 0)
            vv = v[a:a + m].transpose(0, 1).repeat_interleave(H // Hk, 0)
            s = qq @ kk.transpose(1, 2).contiguous() * D ** -0.5 + bias
            if causal:
                s = s.masked_fill(rel > 0, float("-inf"))
            outs.append((torch.softmax(s, -1) @ vv).transpose(0, 1).reshape(m, H * D))
            a += m
        return torch.cat(outs)

    def join(name, x, f):
        g = lambda n: p.get(f"{name}.{n}")       # noqa: E731
        return join64(x, f, g("pre_weight"), g("post_weight"), g("pre_bias"), g("post_bias"), g("gate"), 1.0, kind)
    n = norm64(x, kind) * p["enter_weight"]
    for _ in range(2):
        q, k, v = (n @ p["qkv.weight"].T + p["qkv.bias"]).view(-1, H + 2 * Hk, D).split([H, Hk, Hk], 1)
        x, n = join("join1", x, attend(q, k, v) @ p["out.weight"].T + p["out.bias"])
        h = Keep8.apply(n, p["up.weight"], p["up.bias"], False)
        x, n = join("join2", x, Keep8.apply(h, p["down.weight"], p["down.bias"], True))
    return x, n


def make_block(kind, causal, t):
    L = P()
    torch.manual_seed(3)
    block = L.PackedTransformerBlock(64, 8, 96, num_kv_heads=2, causal=causal, kind=kind, gate=0.7,
                                     buckets=L.RelativeBuckets(16, 20, bidirectional=not causal)).cuda()
    with torch.no_grad():
        block.relative.weight.normal_(0, 0.3)
    return block.to(t)


@pytest.mark.parametrize("kind,causal", [("rms", True), ("layer", False)])
def test_a_block_run_twice_matches_the_formulas(kind, causal):
    """Forward: fp32 through six products of up to 96 terms and eight norms, 1e-5 of the largest value.
    Backward: where fp32 and 64 bits round an activation to different codes (a few in 10^5 values lie
    that near a border) one term of a sum differs by a step, 2^-6 of its block's largest value; the
    gradients, sums of 162 and more such terms, stay within 1e-3 of their norm."""
    block = make_block(kind, causal, torch.float32)
    n = [37, 60, 1, 64]
    g = gen(40)
    x = normal(g, sum(n), 64).requires_grad_()
    seqs = P().PackedSequences(n)
    dx, dn = normal(g, sum(n), 64), normal(g, sum(n), 64)
    y, m = x, block.enter(x)
    for _ in range(2):
        y, m = block(y, m, seqs)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad([y, m], [x, *params.values()], [dx, dn])
    ref = {k: v.detach().double().requires_grad_() for k, v in params.items()}
    X = x.detach().double().requires_grad_()
    ry, rm = block64(block, ref, X, n, causal, block.relative.buckets.lut.cuda())
    rg = torch.autograd.grad([ry, rm], [X, *ref.values()], [dx.double(), dn.double()])
    assert (y - ry).abs().max() <= 1e-5 * ry.abs().max() and (m - rm).abs().max() <= 1e-5 * rm.abs().max()
    for name, a, r in zip(["x", *params], grads, rg):
        assert (a - r).norm() <= 1e-3 * r.norm(), (name, ((a - r).norm() / r.norm()).item())


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_a_captured_training_pass_replays(t):
    """Forward and backward of a block in one graph, replayed on new inputs with eager passes of the same
    leaves between the replays: bit for bit the eager results."""
    block = make_block("layer", True, t)
    params = list(block.parameters())
    seqs = P().PackedSequences([40, 3, 70])
    static = [torch.zeros(113, 64, dtype=t, device="cuda") for _ in range(3)]

    def step(x, gy, gn):
        leaf = x.detach().requires_grad_()
        y, m = block(leaf, block.enter(leaf), seqs)
        return [y.detach(), m.detach(), *torch.autograd.grad([y, m], [leaf, *params], [gy, gn])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for seed in range(4):
        g = gen(50 + seed)
        ins = [normal(g, 113, 64, dtype=t) for _ in range(3)]
        for s, i in zip(static, ins):
            s.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = step(*ins)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_a_capture_without_tables_is_refused():
    L = P()
    seqs, b = L.PackedSequences([8, 9]), L.RelativeBuckets(8, 6)
    q = torch.randn(17, 2, 16, device="cuda")
    table = torch.randn(8, 2, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            L.packed_attention(q, q, q, seqs)
        with pytest.raises(RuntimeError, match="capture"):
            L.packed_attention(q, q, q, seqs, bias=table, buckets=b)
        q.add(1)                                          # (a graph with something in it)
    want = L.packed_attention(q, q, q, seqs)
    check(want, oracle(q, q, q, [8, 9], [8, 9], False, 0.25)["o"])


def test_on_another_stream():
    g = gen(60)
    L = P()
    n = [100, 333]
    q, k, v, do = (normal(g, sum(n), 4, 64, dtype=torch.bfloat16) for _ in range(4))
    seqs = L.PackedSequences(n)
    want = run_attention(q, k, v, seqs, do, causal=True)
    packed = L.unpack8(L.pack8(q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_attention(q, k, v, seqs, do, causal=True)
        again = L.unpack8(L.pack8(q))
        fresh = L.PackedSequences(n)
        other = run_attention(q, k, v, fresh, do, causal=True)
        del fresh
    torch.cuda.current_stream().wait_stream(side)
    for name in want:
        assert torch.equal(want[name], got[name]) and torch.equal(want[name], other[name])
    assert torch.equal(packed, again)


def test_two_calls_at_once_keep_apart():
    """Two streams, the same plan: every call has its own workspace."""
    g = gen(61)
    L = P()
    n = [1, 1]
    seqs = L.PackedSequences(n, [5000, 40])
    sets = [[normal(g, 2, 8, 128, dtype=torch.bfloat16), normal(g, 5040, 2, 128, dtype=torch.bfloat16),
             normal(g, 5040, 2, 128, dtype=torch.bfloat16)] for _ in range(2)]
    want = [run_attention(*s, seqs)["o"] for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run_attention(*sets[i], seqs)["o"])
    torch.cuda.synchronize()
    assert all(torch.equal(want[i], o) for i in range(2) for o in got[i])


# ------------------------------------------------------------------------------------------------
# what surrounds the calls: copies, hooks, streams, hand-made arguments
# ------------------------------------------------------------------------------------------------
def test_copied_and_pickled_sequences_work_by_themselves():
    import copy
    import pickle
    L, g = P(), gen(70)
    n = [5, 70, 0, 31]
    q, k, v, do = (normal(g, sum(n), 4, 32, dtype=torch.bfloat16) for _ in range(4))
    seqs = L.PackedSequences(n)
    want = run_attention(q, k, v, seqs, do, causal=True)
    twins = [copy.deepcopy(seqs), pickle.loads(pickle.dumps(seqs))]
    del seqs
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for twin in twins:
        got = run_attention(q, k, v, twin, do, causal=True)
        assert all(torch.equal(want[name], got[name]) for name in want)


def test_saved_tensors_that_come_back_with_other_strides():
    """Hooks that keep saved tensors elsewhere return them contiguous."""
    L, g = P(), gen(71)
    wide = normal(g, 50, 3, 64)
    x, f, gate = (wide[:, i].detach().requires_grad_() for i in range(3))
    w1, w2 = (normal(g, 64, mean=1.0, scale=0.1).requires_grad_() for _ in range(2))
    dy, dn = normal(g, 50, 64), normal(g, 50, 64)
    n = [20, 30]
    qkv = normal(g, 50, 12, 16)
    q, k, v = (qkv[:, 4 * i:4 * i + 4].detach().requires_grad_() for i in range(3))
    do = normal(g, 50, 4, 16)
    h, W = normal(g, 50, 64).requires_grad_(), normal(g, 33, 64).requires_grad_()
    seqs = L.PackedSequences(n)

    def grads():
        y, m = L.gated_norm(x, f, w1, w2, gate=gate)
        a = L.packed_attention(q, k, v, seqs)
        z = L.linear8(h, W, act="gelu")
        u = L.gelu8(h)
        return torch.autograd.grad([y, m, a, z, u], [x, f, gate, w1, w2, q, k, v, h, W],
                                   [dy, dn, do, torch.ones_like(z), dy])
    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_tables_made_on_one_stream_and_read_on_another():
    L, g = P(), gen(72)
    n = [40, 90]
    q, k, v = (normal(g, 130, 4, 32) for _ in range(3))
    want = L.packed_attention(q, k, v, L.PackedSequences(n))
    seqs = L.PackedSequences(n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = L.packed_attention(q, k, v, seqs)
    assert all(s == side.cuda_stream for call in seqs._calls.values() for _, s in call[2])
    second = L.packed_attention(q, k, v, seqs)
    del seqs
    with torch.cuda.stream(side):
        spoiled = torch.full((4096,), -1, dtype=torch.int32, device="cuda")     # (where the tables were, if free)
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want) and int(spoiled[0]) == -1


@pytest.mark.parametrize("change", [dict(codes=lambda p: p.codes[:-1]), dict(exponents=lambda p: p.exponents[:-1]),
                                    dict(codes=lambda p: p.codes.to(torch.int16)), dict(shape=lambda p: torch.Size([41])),
                                    dict(codes=lambda p: p.codes.repeat(2)[::2]), dict(dtype=lambda p: torch.float64)])
def test_unpack8_checks_what_it_is_given(change):
    L = P()
    p = L.pack8(torch.randn(40, device="cuda"))
    for name, new in change.items():
        setattr(p, name, new(p))
    with pytest.raises(ValueError, match="unpack8"):
        L.unpack8(p)


def test_buckets_must_be_relative_buckets():
    L = P()
    seqs = L.PackedSequences([8])
    q = torch.randn(8, 2, 16, device="cuda")
    with pytest.raises(TypeError, match="RelativeBuckets"):
        L.packed_attention(q, q, q, seqs, bias=torch.zeros(8, 2, device="cuda"), buckets=[0] * 8)


def test_norm_of_more_rows_than_an_axis_of_a_grid():
    """A wave a row: 2^26 rows are 2^32 threads.  Rows are independent: the last ones alone give the same."""
    L, g = P(), gen(73)
    rows = (1 << 26) + 5
    x = torch.empty(rows, 2, dtype=torch.float16, device="cuda")
    x.copy_(torch.arange(rows, device="cuda")[:, None] % 61 - 30)
    f, w = normal(g, rows, 2, dtype=torch.float16), normal(g, 2, dtype=torch.float16)
    with torch.no_grad():
        y, n = L.gated_norm(x, f, w, w)
        for part in (slice(0, 4099), slice(rows - 4099, rows)):
            py, pn = L.gated_norm(x[part], f[part], w, w)
            assert torch.equal(y[part], py) and torch.equal(n[part], pn)
