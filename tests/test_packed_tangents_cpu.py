"""The packed-sequence operators have no forward-mode derivatives: a call with a dual tensor raises before anything
else, it does not drop the tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from VAESNe import PackedLayers as P

NORM = ["x", "branch", "pre_weight", "post_weight", "pre_bias", "post_bias", "gate"]


def attention(**ts):
    seqs, buckets = P.PackedSequences([4], device="cuda:0"), P.RelativeBuckets(8, 6)
    return P.packed_attention(ts["q"], ts["k"], ts["v"], seqs, bias=ts["bias"], buckets=buckets)


CALLS = {
    "packed_attention": (attention, dict(q=(4, 2, 8), k=(4, 2, 8), v=(4, 2, 8), bias=(8, 2))),
    "gated_norm": (lambda **ts: P.gated_norm(**ts, kind="layer"),
                   {n: (5, 8) if n in ("x", "branch", "gate") else (8,) for n in NORM}),
    "pre_norm": (lambda x, weight, bias: P.pre_norm(x, weight, bias, kind="layer"), dict(x=(5, 8), weight=(8,), bias=(8,))),
    "gelu8": (lambda x: P.gelu8(x), dict(x=(5, 8))),
    "linear8": (lambda x, weight, bias: P.linear8(x, weight, bias, act="gelu"), dict(x=(5, 8), weight=(3, 8), bias=(3,))),
    "pack8": (lambda x: P.pack8(x), dict(x=(5, 8))),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_dual_tensors_are_refused(name, grad):
    call, shapes = CALLS[name]
    plain = {n: torch.randn(s) for n, s in shapes.items()}
    for which in plain:
        with fwd.dual_level():
            ts = dict(plain)
            ts[which] = fwd.make_dual(plain[which].clone().requires_grad_(grad), torch.ones_like(plain[which]))
            with pytest.raises(NotImplementedError, match=f"{name}: .*forward-mode"):
                call(**ts)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(**ts)
            with pytest.raises(RuntimeError, match="ROCm"):           # no tangent: the usual checks
                call(**plain)
