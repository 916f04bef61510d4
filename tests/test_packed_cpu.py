"""Host side of the packed-sequence operators: bucket tables, tile tables, refusals.  Nothing here
launches a kernel: every bad argument is turned down before one could run."""
import copy
import ctypes as C
import math

import numpy as np
import pytest
import torch

from VAESNe import PackedLayers as P
from VAESNe import _lib, _packed_ops

BAD = 1          # hipErrorInvalidValue


# ---- buckets -------------------------------------------------------------------------------------
@pytest.mark.parametrize("count,distance,both", [(32, 128, True), (32, 128, False), (8, 64, True), (64, 512, True),
                                                 (64, 100, False), (2, 2, False), (4, 2, True), (16, 9, False)])
def test_buckets_are_monotone_and_complete(count, distance, both):
    lut = P.RelativeBuckets(count, distance, both).lut.tolist()
    assert len(lut) == 2 * distance + 1
    m = count // 2 if both else count
    back = lut[distance::-1]                       # distances 0, 1, 2, ... towards earlier keys
    assert back[:m // 2] == list(range(m // 2)) and back[-1] == m - 1
    assert all(0 <= b - a <= m for a, b in zip(back, back[1:])) and max(back) == m - 1
    ahead = lut[distance + 1:]
    assert ahead == ([b + m for b in back[1:]] if both else [0] * distance)


def test_buckets_on_exact_borders():
    # near 8, far buckets 8 * 2^(k/2): 16, 32 and 64 lie on borders and belong to the bucket above
    lut = P.RelativeBuckets(32, 128, True).lut
    of = lambda n: int(lut[128 - n])      # noqa: E731
    assert [of(n) for n in (15, 16, 31, 32, 63, 64, 90, 91, 128)] == [9, 10, 11, 12, 13, 14, 14, 15, 15]


@pytest.mark.parametrize("args", [(0, 128), (3, 128, True), (2, 128, True), (1, 8, False), (32, 8, True), (32, 513),
                                  (2048, 512, False)])
def test_buckets_refuse(args):
    with pytest.raises(ValueError):
        P.RelativeBuckets(*args)


# ---- tiles ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("side", ["q", "k"])
@pytest.mark.parametrize("tile", [1, 32, 128])
def test_tile_table_covers_every_position_once_longest_first(side, tile, causal):
    nq = np.array([0, 1, 31, 32, 33, 500, 7], dtype=np.int64)
    nk = np.array([9, 0, 40, 32, 20, 500, 4000], dtype=np.int64)
    t = _packed_ops.tile_table(nq, nk, side, tile, causal)
    n = nq if side == "q" else nk
    q0, k0 = np.cumsum(nq) - nq, np.cumsum(nk) - nk
    want = sorted((q0[s], k0[s], nq[s], nk[s], p, 0, 0, 0) for s in range(len(n)) for p in range(0, int(n[s]), tile))
    assert sorted(map(tuple, t.tolist())) == want and t.dtype == np.int32
    which = [[s for s in range(len(n)) if (q0[s], k0[s], nq[s], nk[s]) == tuple(r[:4])][0] for r in t.tolist()]

    def work(s, p):
        if side == "q":
            return sum(1 for j in range(nk[s]) if j <= min(p + tile, nq[s]) - 1 + nk[s] - nq[s]) if causal else nk[s]
        return sum(1 for i in range(nq[s]) if p <= i + nk[s] - nq[s]) if causal else nq[s]
    got = [work(s, r[4]) for s, r in zip(which, t.tolist())]
    # (a last, short tile is ranked as a whole one)
    assert all(b <= a + tile for a, b in zip(got, got[1:]))
    assert _packed_ops.tile_table(nq[:0], nk[:0], side, tile, causal).shape == (0, 8)


# ---- refusals of the Python entry points ------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: P.gated_norm(x, x, w, w), lambda: P.pre_norm(x, w), lambda: P.gelu8(x), lambda: P.pack8(x),
                 lambda: P.linear8(x, torch.ones(3, 8)),
                 lambda: P.packed_attention(x[:, None], x[:, None], x[:, None], None),
                 lambda: P.PackedSequences([4], device="cpu"),
                 lambda: P.PackedSequences.from_mask(torch.zeros(1, 4, dtype=torch.bool))):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()


@pytest.mark.parametrize("lengths", [[-1], [2.5], torch.tensor([1.0]), torch.zeros(2, 2, dtype=torch.long),
                                     [1 << 30, 1 << 30]])
def test_bad_lengths_are_refused(lengths):
    with pytest.raises(ValueError):
        P.PackedSequences(lengths, device="cpu")


def test_lengths_must_pair():
    with pytest.raises(ValueError):
        P.PackedSequences([1, 2], [3], device="cpu")


def test_unpack8_takes_only_its_own():
    with pytest.raises(TypeError):
        P.unpack8(torch.zeros(3))


# ---- refusals at the C entry points -------------------------------------------------------------------
def attn_args(backward=0, **kw):
    a = _packed_ops._AttnArgs(type=1, Hq=8, Hkv=2, D=64, causal=1, nseq=1, scale=0.125, max_q=100, max_k=100,
                              total_q=100, total_k=100, q_tiles=64, k_tiles=64, q=64, k=64, v=64,
                              q_ts=512, q_hs=64, k_ts=128, k_hs=64, v_ts=128, v_hs=64, o=64, lse=64, dout=64, do_ts=512,
                              do_hs=64, dq=64, dk=64, dv=64, workspace=64, n_q_tiles=4, n_k_tiles=1)
    qt, kt = C.c_int(), C.c_int()
    assert _lib.load().vaesne_packed_attn_tiles(C.addressof(a), backward, C.byref(qt), C.byref(kt)) == 0
    a.q_tile, a.k_tile = qt.value, kt.value
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [
    dict(type=3), dict(type=-1), dict(Hq=0), dict(Hkv=3), dict(Hkv=0), dict(D=0), dict(D=12), dict(D=136),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(q_tile=31), dict(k_tile=64), dict(max_q=1 << 26),
    dict(max_k=1 << 26), dict(total_q=-1), dict(q=None), dict(k=None), dict(o=None), dict(lse=None),
    dict(q_tiles=None), dict(n_q_tiles=0), dict(n_q_tiles=-1), dict(n_q_tiles=1 << 22), dict(n_k_tiles=1 << 24), dict(q=72), dict(k=66), dict(q_ts=516), dict(v_hs=4), dict(k_ts=1 << 23),
    dict(q_hs=-64), dict(table=64, max_distance=0, num_buckets=4), dict(table=64, max_distance=513, num_buckets=4),
    dict(table=64, max_distance=8, num_buckets=0), dict(table=64, max_distance=8, num_buckets=4, lut=None)])
def test_attention_entry_refuses(change):
    lib = _lib.load()
    if "k_tile" not in change:
        assert lib.vaesne_packed_attn_fwd(C.addressof(attn_args(0, **change)), None) == BAD
    assert lib.vaesne_packed_attn_bwd(C.addressof(attn_args(1, **change)), None) == BAD


@pytest.mark.parametrize("change", [dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(workspace=None),
                                    dict(workspace=68), dict(k_tiles=None), dict(n_k_tiles=0), dict(do_hs=2)])
def test_attention_backward_entry_refuses(change):
    a = attn_args(1, **change)
    assert _lib.load().vaesne_packed_attn_bwd(C.addressof(a), None) == BAD


def test_attention_workspace_counts():
    lib = _lib.load()
    a = attn_args(type=0)
    delta = 4 * 100 * 8
    assert lib.vaesne_packed_attn_workspace(C.addressof(a), 1) >= delta
    few = attn_args(type=1, max_q=1, total_q=1, max_k=100000, total_k=100000)      # split over the keys
    assert lib.vaesne_packed_attn_workspace(C.addressof(few), 0) >= 2 * 8 * (64 + 1) * 4
    assert lib.vaesne_packed_attn_workspace(C.addressof(attn_args(D=7)), 0) < 0


def norm_args(**kw):
    a = _packed_ops._NormArgs(type=1, kind=0, gate_kind=0, C=64, rows=4, residual_scale=1.0, eps=1e-5, x=64, branch=64,
                              pre_w=64, post_w=64, ldx=64, ldbranch=64, y=64, n=64, stats=64, dy=64, dn=64, lddy=64,
                              lddn=64, dx=64, dbranch=64, dpre_w=64, dpost_w=64, workspace=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [dict(type=5), dict(kind=2), dict(gate_kind=3), dict(C=0), dict(C=8193), dict(rows=-1),
                                    dict(rows=1 << 31), dict(x=None), dict(pre_w=None), dict(post_w=None),
                                    dict(gate_kind=1), dict(stats=72)])
def test_norm_entry_refuses(change):
    lib = _lib.load()
    a = norm_args(**change)
    assert lib.vaesne_gated_norm_fwd(C.addressof(a), None) == BAD
    assert lib.vaesne_gated_norm_bwd(C.addressof(a), None) == BAD


@pytest.mark.parametrize("change", [dict(n=None), dict(y=None)])
def test_norm_forward_entry_refuses(change):
    a = norm_args(**change)
    assert _lib.load().vaesne_gated_norm_fwd(C.addressof(a), None) == BAD


@pytest.mark.parametrize("change", [dict(workspace=None), dict(dx=None), dict(stats=None), dict(dbranch=None)])
def test_norm_backward_entry_refuses(change):
    a = norm_args(**change)
    assert _lib.load().vaesne_gated_norm_bwd(C.addressof(a), None) == BAD


def test_act8_entries_refuse():
    lib = _lib.load()
    for bad in ((3, 64, 32, 64, 64), (0, None, 32, 64, 64), (0, 64, -1, 64, 64), (0, 64, 32, 68, 64), (0, 64, 32, 64, None)):
        t, x, n, codes, exps = bad
        assert lib.vaesne_pack8(t, x, n, codes, exps, None) == BAD
        assert lib.vaesne_unpack8(t, codes, exps, n, x, None) == BAD
        assert lib.vaesne_gelu8_fwd(t, x, n, 64, codes, exps, None) == BAD
        assert lib.vaesne_gelu8_bwd(t, codes, exps, 64, n, x, None, None) == BAD
    assert lib.vaesne_gelu8_fwd(0, 64, 32, None, 64, 64, None) == BAD
    assert lib.vaesne_gelu8_fwd(0, 64, 32, 64, None, 64, None) == BAD
    assert lib.vaesne_gelu8_bwd(0, 64, 64, None, 32, 64, None, None) == BAD
    for fn, args in (("pack8", (0, None, 0, None, None)), ("unpack8", (0, None, None, 0, None)),
                     ("gelu8_fwd", (0, None, 0, None, None, None)), ("gelu8_bwd", (0, None, None, None, 0, None, None))):
        assert getattr(lib, "vaesne_" + fn)(*args, None) == 0                      # nothing to do


@pytest.mark.parametrize("change", [dict(total_q=1 << 30), dict(total_k=1 << 30),
                                    dict(n_q_tiles=(1 << 21) - 1, n_k_tiles=(1 << 23) - 1)])
def test_launches_past_a_grid_are_refused(change):
    """An axis of a grid has fewer than 2^32 threads."""
    a = attn_args(1, **change)
    assert _lib.load().vaesne_packed_attn_bwd(C.addressof(a), None) == BAD
    lib = _lib.load()
    n = 1 << 35
    assert lib.vaesne_pack8(1, 64, n, 64, 64, None) == BAD
    assert lib.vaesne_unpack8(1, 64, 64, n, 64, None) == BAD
    assert lib.vaesne_gelu8_fwd(1, 64, n, 64, 64, 64, None) == BAD
    assert lib.vaesne_gelu8_bwd(1, 64, 64, 64, n, 64, None, None) == BAD


@pytest.mark.parametrize("total", [[1 << 30], [1 << 29, 1 << 29]])
def test_sequences_of_too_many_tokens_are_refused(total):
    with pytest.raises(ValueError, match="2\\^30"):
        P.PackedSequences(total, device="cpu")


def test_unpack8_refuses_codes_on_the_host():
    kept = P.Packed8(torch.zeros(40, dtype=torch.int8), torch.zeros(2, dtype=torch.uint8), torch.Size([40]), torch.float32)
    with pytest.raises(RuntimeError, match="ROCm"):
        P.unpack8(kept)


def test_a_copy_of_sequences_makes_its_own_tables():
    seqs = object.__new__(P.PackedSequences)
    seqs.__dict__.update(lengths=[3], _tables={"a": 1}, _calls={"b": 2}, _index=None)
    twin = copy.deepcopy(seqs)
    assert twin.lengths == [3] and twin._tables == {} and twin._calls == {}
    assert seqs._tables == {"a": 1} and seqs._calls == {"b": 2}
