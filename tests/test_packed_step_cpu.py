"""Packed sequences and training_step's captured steps, on the CPU: where the sequences of a batch lie is
no part of a captured step's inputs, so a step that uses a PackedSequences runs eagerly."""
import types

import pytest
import torch
from torch import nn

from VAESNe import PackedLayers as P
from VAESNe import _capture, _packed_ops
from VAESNe import _stepgraph as SG

GLOBAL_SEQS = None


def plan(*lengths):
    return P.PackedSequences(list(lengths), device="cuda:0")


def with_cell(seqs):
    return lambda m, x: (m, x, seqs)


def with_default(value):
    def fn(m, x, *, seqs=value):
        return m, x, seqs
    return fn


def with_global(m, x):
    return m, x, GLOBAL_SEQS


def signature(net, fn):
    return SG._signature(net, fn, [torch.zeros(100, 3)], False, list(net.parameters()))


def on_module(seqs):
    net = nn.Sequential(nn.Linear(3, 4), nn.Linear(4, 2))
    net[1].seqs = seqs
    return net, lambda m, x: (m, x)


PLACES = {
    "module": on_module,
    "module list": lambda s: on_module([s]),
    "closure": lambda s: (nn.Linear(3, 4), with_cell(s)),
    "closure dict": lambda s: (nn.Linear(3, 4), with_cell({"seqs": s})),
    "closure list in a dict": lambda s: (nn.Linear(3, 4), with_cell({"seqs": [s, 3]})),
    "default": lambda s: (nn.Linear(3, 4), with_default(s)),
}


@pytest.mark.parametrize("place", PLACES)
def test_another_plan_is_another_signature_and_runs_eagerly(place):
    a, b = plan(40, 60), plan(10, 90)
    net, fn = PLACES[place](a)
    first = signature(net, fn)
    assert signature(net, fn) == first
    assert SG._uses_plan(net, fn)
    if "module" in place:
        held = net[1].seqs
        net[1].seqs = [b] if isinstance(held, list) else b
        assert signature(net, fn) != first
        net[1].seqs = held
        assert signature(net, fn) == first
    else:
        assert signature(net, PLACES[place](b)[1]) != first


def test_a_plan_that_changes_inside_a_closure_dict():
    state = {"seqs": plan(40, 60)}
    net, fn = nn.Linear(3, 4), with_cell(state)
    first = signature(net, fn)
    state["seqs"] = plan(10, 90)
    assert signature(net, fn) != first and SG._uses_plan(net, fn)


def test_a_plan_in_a_global():
    global GLOBAL_SEQS
    net = nn.Linear(3, 4)
    try:
        GLOBAL_SEQS = plan(40, 60)
        first = signature(net, with_global)
        assert SG._uses_plan(net, with_global)
        GLOBAL_SEQS = plan(10, 90)
        assert signature(net, with_global) != first
    finally:
        GLOBAL_SEQS = None
    assert not SG._uses_plan(net, with_global)


def test_a_plan_set_later_is_seen():
    """The walk over the modules is kept from batch to batch while nothing changes."""
    net, fn = nn.Linear(3, 4), lambda m, x: (m, x)
    net.seqs = None
    signature(net, fn)
    assert not SG._uses_plan(net, fn)
    net.seqs = plan(40, 60)
    assert SG._uses_plan(net, fn)
    net.seqs = None
    assert not SG._uses_plan(net, fn)


def test_ranks_agree_on_a_loss_function_whatever_its_plan():
    """The data-parallel exchange keys its gradient pattern by the loss function and meets the other ranks when
    the key is new: a plan for each batch is no new key."""
    assert SG._fn_key(with_cell(plan(40, 60))) == SG._fn_key(with_cell(plan(10, 90)))


def test_step_does_not_count_batches_with_a_plan(monkeypatch):
    x = types.SimpleNamespace(is_cuda=True, shape=(100, 3), dtype=torch.float32)
    net, fn = on_module(plan(40, 60))
    for _ in range(5):
        assert SG.step(net, fn, (x,), False) is None
    assert not SG._CACHE.get(net)


@pytest.mark.parametrize("use", ["attention forward or backward", "pack", "unpack"])
def test_a_hidden_plan_is_refused_inside_a_captured_step(use, monkeypatch):
    """Found nowhere (a global dict, a helper function's closure): the call raises, so the step stays eager."""
    seqs = plan(40, 60)
    seqs._index = (torch.arange(100), (2, 60))
    call = {"attention forward or backward": lambda: seqs._args((bytes(_packed_ops._AttnArgs()), 0, [])),
                                  "pack": lambda: seqs.pack(torch.zeros(2, 60, 3)),
                                  "unpack": lambda: seqs.unpack(torch.zeros(100, 3))}[use]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with _capture.whole_step(), pytest.raises(RuntimeError, match="training_step"):
        call()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with _capture.whole_step():                       # another thread's or stream's eager work
        with pytest.raises(Exception) as e:           # (no ROCm device here: it gets past the check only)
            call()
        assert "training_step" not in str(e.value)
