"""The capture of a training step, on the host: torch.cuda's streams and graphs are replaced by stand-ins that run everything eagerly, and the
module looks, in each of its passes, at which of its parameters' gradient accumulators some autograd graph holds."""
import contextlib

import pytest
import torch

from deepinteraction_amd import graphed
from deepinteraction_amd.graphed import GraphedTrainingModule, accumulators_alive


@contextlib.contextmanager
def nothing(*a, **k):
    yield


class Stream:
    def __init__(self, *a, **k):
        pass

    def wait_stream(self, other):
        pass

    __enter__ = __exit__ = lambda self, *a: None


class Graph:
    """A graph whose replay does nothing: the buffers keep what the capture left in them."""

    def __init__(self, keep_graph=False):
        assert keep_graph
        self.replays = 0

    def replay(self):
        self.replays += 1


@pytest.fixture
def eager_cuda(monkeypatch):
    for name, value in dict(Stream=Stream, stream=nothing, current_stream=Stream, synchronize=lambda *a: None, CUDAGraph=Graph, graph=nothing,
                            graph_pool_handle=lambda: (0, 0)).items():
        monkeypatch.setattr(torch.cuda, name, value)
    monkeypatch.setattr(graphed, '_without_memsets', lambda graph: graph)


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.a, self.b = torch.nn.Linear(3, 4), torch.nn.Linear(4, 2)
        self.held = []

    def forward(self, x):
        self.held.append(len(accumulators_alive(list(self.parameters()))))
        y = self.a(x)
        return self.b(y).sum(-1), y.detach(), y


def test_accumulators_are_alive_as_long_as_a_graph_is():
    m = torch.nn.Linear(3, 2)
    params = list(m.parameters())
    assert accumulators_alive(params) == []
    y = m(torch.ones(1, 3)).sum()
    assert len(accumulators_alive(params)) == 2 and len(accumulators_alive(params)) == 2
    y.backward()                                                     # frees what it saved, not its nodes
    assert len(accumulators_alive(params)) == 2
    del y
    assert accumulators_alive(params) == [] and m.weight.grad is not None
    m.bias.requires_grad_(False)
    y = m(torch.ones(1, 3))
    assert [p is m.weight for p in accumulators_alive(params)] == [True]


def test_nothing_is_alive_when_the_step_is_captured(eager_cuda):
    m = Layer()
    GraphedTrainingModule(m, (torch.randn(5, 3),), warmup=3)
    assert m.held == [0, 0, 0, 0]                                    # three passes ahead of the capture, and the capture


def test_a_graph_that_the_caller_holds_is_refused(eager_cuda):
    m = Layer()
    loss = m(torch.randn(5, 3))[0].sum()
    with pytest.raises(RuntimeError, match='4 of the 4 parameters'):
        GraphedTrainingModule(m, (torch.randn(5, 3),))
    del loss
    m.held.clear()
    GraphedTrainingModule(m, (torch.randn(5, 3),), warmup=1)
    assert m.held == [0, 0]


def test_the_collector_runs_again_afterwards(eager_cuda):
    import gc

    class Fails(Layer):
        def forward(self, x):
            if self.held:
                raise ValueError('in the capture')
            return super().forward(x)
    assert gc.isenabled()
    with pytest.raises(ValueError):
        GraphedTrainingModule(Fails(), (torch.randn(5, 3),), warmup=1)
    assert gc.isenabled()


def test_a_replay_s_outputs_and_gradients(eager_cuda):
    """Outputs and gradients are the buffers of the captures, every replay runs its graph once, nothing is held afterwards, and an output without
    a gradient stays without."""
    m, x = Layer(), torch.randn(5, 3, requires_grad=True)
    g = GraphedTrainingModule(m, (x,))
    params = list(m.parameters())
    assert accumulators_alive(params) == [] and accumulators_alive([x]) == []
    for n in range(3):
        outs = g(x)
        want = m(x)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert [o.requires_grad for o in outs] == [True, False, True]
        seeds = (torch.ones_like(want[0]), torch.full_like(want[2], 0.5))
        for static, s in zip(g.grad_outs, seeds):                    # the stand-in's replay leaves the capture's gradients: of zeros
            assert not static.any() or n > 0
        got = torch.autograd.grad((outs[0], outs[2]), [x] + params, seeds)
        assert all(torch.equal(a, b) for a, b in zip(g.grad_outs, seeds))
        assert all(a.shape == b.shape and not a.any() for a, b in zip(got, [x] + params))
        assert (g.forward_graph.replays, g.backward_graph.replays) == (n + 1, n + 1)
    with torch.no_grad():
        assert not g(torch.zeros(5, 3))[0].requires_grad
    assert not g.args[0].any()                                        # another input is copied into the captured one


def test_inputs_of_other_shapes_are_refused(eager_cuda):
    g = GraphedTrainingModule(Layer(), (torch.randn(5, 3),))
    for bad in ((), (torch.randn(1, 3),), (torch.randn(5, 3), torch.randn(5, 3))):
        with pytest.raises(ValueError):
            g(*bad)
