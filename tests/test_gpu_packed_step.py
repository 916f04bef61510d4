"""training_step over packed batches of the same token count and different boundaries, against the eager loop."""
import types

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

LENGTHS = [[40, 60], [10, 90], [100], [33, 33, 34], [1, 99]]


class Net(nn.Module):
    def __init__(self):
        super().__init__()
        from VAESNe import PackedLayers as P
        self.block = P.PackedTransformerBlock(32, 4, 48, causal=True, kind="layer", gate=0.5,
                                              buckets=P.RelativeBuckets(8, 20, bidirectional=False))
        self.seqs = None

    def forward(self, x, seqs):
        y, n = self.block(x, self.block.enter(x), seqs)
        return y.square().mean() + n.mean()


class Loader:
    """Batches of 100 tokens; before each is handed out `place` gets its plan."""

    def __init__(self, data, plans, place):
        self.data, self.plans, self.place = data, plans, place

    def __iter__(self):
        for x, plan in zip(self.data, self.plans):
            self.place(plan)
            yield (x,)


def train(graph, how, monkeypatch):
    from VAESNe import PackedLayers as P
    from VAESNe import _config, _stepgraph, rng
    from VAESNe.training_util import training_step
    monkeypatch.setattr(_config, "step_graph", graph)
    torch.manual_seed(0)
    net = Net().cuda()
    rng.manual_seed(5)
    opt = torch.optim.AdamW(net.parameters(), lr=1e-2)
    plans = [P.PackedSequences(n) for n in LENGTHS for _ in range(4)]
    data = [torch.randn(100, 32, generator=torch.Generator().manual_seed(i)) for i in range(len(plans))]
    state, hidden = {"seqs": None}, types.SimpleNamespace(seqs=None)
    place, fn = {
        "module": (lambda s: setattr(net, "seqs", s), lambda m, x: -m(x[0], m.seqs)),
        "closure dict": (lambda s: state.update(seqs=s), lambda m, x: -m(x[0], state["seqs"])),
        "object": (lambda s: setattr(hidden, "seqs", s), lambda m, x: -m(x[0], hidden.seqs)),
    }[how]
    losses = [training_step(net, opt, Loader(data, plans, place), loss_fn=fn) for _ in range(2)]
    torch.cuda.synchronize()
    captured = sum(e.graph is not None for e in _stepgraph._CACHE.get(net, {}).values())
    _stepgraph.clear()
    return losses, [p.detach().clone() for p in net.parameters()], captured


@pytest.mark.parametrize("how", ["module", "closure dict", "object"])
def test_every_batch_keeps_its_own_boundaries(how, monkeypatch):
    eager = train(False, how, monkeypatch)
    got = train(True, how, monkeypatch)
    assert got[0] == eager[0] and got[2] == 0
    assert all(torch.equal(a, b) for a, b in zip(eager[1], got[1]))


def test_a_packed_step_without_plans_is_still_captured(monkeypatch):
    """gated_norm, gelu8 and linear8 read their inputs only."""
    from VAESNe import PackedLayers as P
    from VAESNe import _config, _stepgraph, rng
    from VAESNe.training_util import training_step
    runs = []
    for graph in (False, True):
        monkeypatch.setattr(_config, "step_graph", graph)
        torch.manual_seed(0)
        net = nn.ModuleDict({"up": nn.Linear(32, 48), "down": nn.Linear(48, 32), "join": P.GatedNorm(32)}).cuda()
        rng.manual_seed(5)
        opt = torch.optim.AdamW(net.parameters(), lr=1e-2)
        data = [(torch.randn(100, 32, generator=torch.Generator().manual_seed(i)),) for i in range(8)]

        def fn(m, x):
            h = P.linear8(x[0], m["up"].weight, m["up"].bias)
            y, n = m["join"](x[0], P.linear8(h, m["down"].weight, m["down"].bias, act="gelu"))
            return -(y.square().mean() + n.mean())
        losses = training_step(net, opt, data, loss_fn=fn)
        torch.cuda.synchronize()
        captured = sum(e.graph is not None for e in _stepgraph._CACHE.get(net, {}).values())
        runs.append((losses, [p.detach().clone() for p in net.parameters()], captured))
        _stepgraph.clear()
    assert runs[0][0] == runs[1][0] and runs[1][2] == 1
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))
