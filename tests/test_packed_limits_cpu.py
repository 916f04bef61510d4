"""The largest sizes that the packed operators accept, at the C entries and in Python: past them every call is refused
before a launch."""
import ctypes as C

import pytest

from VAESNe import PackedLayers as P
from VAESNe import _lib
from test_packed_cpu import BAD, attn_args

MOST = (1 << 30) - 64       # tokens: a launch of 4 threads a token, in whole workgroups, is below 2^32


@pytest.mark.parametrize("change", [dict(total_q=MOST + 1), dict(total_q=(1 << 30) - 1), dict(total_k=MOST + 1)])
def test_tokens_past_a_launch_are_refused(change):
    lib = _lib.load()
    assert lib.vaesne_packed_attn_fwd(C.addressof(attn_args(0, **change)), None) == BAD
    assert lib.vaesne_packed_attn_bwd(C.addressof(attn_args(1, **change)), None) == BAD
    assert lib.vaesne_packed_attn_workspace(C.addressof(attn_args(1, **change)), 1) < 0


def test_as_many_tokens_as_a_launch_holds_are_not():
    lib = _lib.load()
    assert lib.vaesne_packed_attn_workspace(C.addressof(attn_args(1, total_q=MOST, total_k=MOST)), 1) > 0
    assert P.PackedSequences([MOST - 5, 5], device="cuda:0").total == MOST
    with pytest.raises(ValueError, match="2\\^30"):
        P.PackedSequences([MOST - 5, 6], device="cuda:0")
