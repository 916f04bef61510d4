"""Tile tables that say what they should not (a plan that was dropped while a graph still replays, memory written over):
the kernels stay inside the tensors and end."""
import ctypes as C

import pytest
import torch

from test_gpu_packed import P, gen, normal

pytestmark = pytest.mark.gpu
EDGE = 4096          # elements on either side of every output that must keep their value


def framed(n, dtype):
    t = torch.full((n + 2 * EDGE,), 7.0, dtype=dtype, device="cuda")
    return t, t[EDGE:EDGE + n]


def spoil(table, how, g):
    rows = table.view(-1, 8)
    if how == "lengths":                                   # tokens and lengths run past the end
        rows[::2, 2:4] += 1000
        rows[1::2, :2] += 30
    elif how == "positions":
        rows[::3, 4] += 64
        rows[1::3, 4] = -5
    elif how == "random":
        rows.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, rows.shape, generator=g, device="cuda", dtype=torch.int64).int())
    else:
        rows.fill_(how)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("how", ["lengths", "positions", "random", -1, 0, 2 ** 31 - 1])
@pytest.mark.parametrize("bias", [False, True])
def test_spoiled_tables_stay_inside_the_tensors(t, how, bias):
    from VAESNe import _packed_ops as ops
    L, g = P(), gen(110)
    nq, nk, H, Hk, D = [40, 1, 130, 9], [40, 300, 130, 0], 4, 2, 32
    seqs, buckets = L.PackedSequences(nq, nk), L.RelativeBuckets(8, 20)
    q, do = normal(g, sum(nq), H, D, dtype=t), normal(g, sum(nq), H, D, dtype=t)
    k, v = normal(g, sum(nk), Hk, D, dtype=t), normal(g, sum(nk), Hk, D, dtype=t)
    table = normal(g, 8, H, dtype=t)
    b = buckets if bias else None
    calls = [seqs._call(ops.TYPES[t], H, Hk, D, True, b, back) for back in (False, True)]
    for got, _, _ in seqs._tables.values():
        spoil(got, how, g)
    frames = {n: framed(x.numel(), x.dtype) for n, x in dict(o=q, dq=q, dk=k, dv=v, dtable=table).items()}
    frames["lse"] = framed(sum(nq) * H, torch.float32)
    for back, call in enumerate(calls):
        frames[f"ws{back}"] = framed((call[1] + 15) // 4, torch.float32)
        a = seqs._args(call)
        a.scale = D ** -0.5
        a.q, a.k, a.v, a.dout = (x.data_ptr() for x in (q, k, v, do))
        a.q_ts, a.q_hs, _ = q.stride()
        a.k_ts, a.k_hs, _ = k.stride()
        a.v_ts, a.v_hs, _ = v.stride()
        a.do_ts, a.do_hs, _ = do.stride()
        a.o, a.lse, a.dq, a.dk, a.dv = (frames[n][1].data_ptr() for n in ("o", "lse", "dq", "dk", "dv"))
        a.workspace = frames[f"ws{back}"][1].data_ptr()
        if bias:
            a.table, a.lut = table.data_ptr(), buckets.on(q.device).data_ptr()
            a.dtable = frames["dtable"][1].data_ptr() if back else None
        ops._lib_call("packed_attn_bwd" if back else "packed_attn_fwd", q.device, C.addressof(a))
        torch.cuda.synchronize()
    for name, (whole, inside) in frames.items():
        assert (whole[:EDGE] == 7).all() and (whole[EDGE + inside.numel():] == 7).all(), name
