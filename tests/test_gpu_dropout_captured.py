"""Dropout layers in captured graphs: every replay drops other values, its backward those of its forward."""

import copy
import gc
import pickle

import pytest
import torch
import torch.utils.checkpoint

import memfast_amd as memfast
from memfast_amd.nn import Dropout, GatedRecurrence, gated

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_garbage_within_captures():
    """Graphed callables and tracebacks hold their graphs in cycles. A graph that the collector destroys waits for
    the device, which ends the process while another is being captured: they go between tests alone, and
    none is left to other files' captures."""
    gc.collect()
    gc.disable()
    yield
    gc.enable()
    gc.collect()


def captured(call):
    """The graph of ``call`` after a pass of it on a side stream, and what it returns."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.manual_seed(6)
    with torch.cuda.graph(graph):
        results = call()
    return graph, results


def test_every_replay_has_a_mask_of_its_own(hip_device):
    layer = Dropout(0.5)
    x = torch.randn(3000, device=hip_device, requires_grad=True)

    def call():
        y = layer(x)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    graph, (y, dx) = captured(call)
    torch.manual_seed(6)
    seed, seen, start = int(torch.randint(1 << 62, ())), [], int(gated._counters[0])
    for turn in range(start, start + 4):
        graph.replay()
        layer(x)                                            # eager work between replays
        torch.cuda.synchronize()
        assert torch.equal(y, memfast.dropout(x.detach(), 0.5, seed=seed, event=turn))
        assert torch.equal(dx, memfast.dropout(torch.ones_like(y), 0.5, seed=seed, event=turn))
        seen.append(y != 0)
    assert not any(torch.equal(a, b) for n, a in enumerate(seen) for b in seen[:n])
    # Another graph of the same layer goes on counting, with a seed of its own.
    again, (z, dz) = captured(call)
    for graph_, out, grad in ((again, z, dz), (graph, y, dx), (again, z, dz)):
        graph_.replay()
        torch.cuda.synchronize()
        assert torch.equal(out != 0, grad != 0) and not any(torch.equal(out != 0, a) for a in seen)
        seen.append((out != 0).clone())


def test_a_stacked_layer_trains_on_new_masks(hip_device):
    torch.manual_seed(1)
    layer = GatedRecurrence(16, 24, 3, dropout=0.5).to(hip_device)
    x = torch.randn(20, 4, 16, device=hip_device)
    weights = list(layer.parameters())

    def call():
        y, _ = layer(x)
        return y.detach(), *torch.autograd.grad(y.square().sum(), weights)

    graph, (y, *grads) = captured(call)
    torch.manual_seed(6)
    seeds, rows, start = [int(torch.randint(1 << 62, ())) for _ in range(2)], [], int(gated._counters[0])
    for turn in range(3):
        graph.replay()
        h = x
        for n, projection in enumerate(layer.projections):
            h, _ = memfast.gated_recurrence(projection(h))
            if n < 2:
                h = memfast.dropout(h, 0.5, seed=seeds[n], event=start + 2 * turn + n)
        expected = torch.autograd.grad(h.square().sum(), weights)
        torch.cuda.synchronize()
        # The same kernels on the same values but for the library's products, whose order of sums may differ.
        assert torch.allclose(y, h, rtol=1e-5, atol=1e-6)
        for a, b in zip(grads, expected):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
        rows.append(y.clone())
    assert not any(torch.allclose(a, b, rtol=1e-2, atol=1e-2) for n, a in enumerate(rows) for b in rows[:n])


def test_graphed_callables(hip_device):
    """Forward and backward as two graphs."""
    layer = Dropout(0.5)
    x = torch.ones(2000, device=hip_device, requires_grad=True)
    graphed = torch.cuda.make_graphed_callables(layer, (torch.ones_like(x).requires_grad_(True),))
    seen = []
    for _ in range(3):
        y = graphed(x)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx != 0, y != 0)
        seen.append((y != 0).clone())
    assert not any(torch.equal(a, b) for n, a in enumerate(seen) for b in seen[:n])


def test_a_capture_without_a_counter_is_refused(hip_device, monkeypatch):
    """No layer has run on the device: one mask for all replays is not taken silently."""
    monkeypatch.setattr(gated, "_counters", {})
    layer, x = Dropout(0.5), torch.ones(100, device=hip_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="before one is captured"):
            layer(x)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((y == 2).all())
    for quiet in (layer.eval(), Dropout(0.0)):              # nothing is dropped: nothing to refuse
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = quiet(x) + 1
        graph.replay()
        torch.cuda.synchronize()
        assert bool((y == 2).all())


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_layer_is_captured(hip_device, reentrant):
    """The forward that the backward takes again drops what the first one dropped, in every replay."""
    layer = Dropout(0.5)
    x = torch.ones(3000, device=hip_device, requires_grad=True)

    def checkpointed(v):
        return torch.utils.checkpoint.checkpoint(lambda u: layer(layer(u * u)), v, use_reentrant=reentrant)

    def call():
        y = checkpointed(x)
        if not reentrant:
            return y.detach(), torch.autograd.grad(y.sum(), x)[0]
        inner = x.detach().requires_grad_(True)
        y = checkpointed(inner)
        y.sum().backward()
        return y.detach(), inner.grad

    graph, (y, dx) = captured(call)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx != 0, y != 0)
        seen.append((y != 0).clone())
        for eager in call(), call():                        # eager passes stay whole beside it
            assert torch.equal(eager[0] != 0, eager[1] != 0)
    assert not any(torch.equal(a, b) for n, a in enumerate(seen) for b in seen[:n])


def test_checkpointed_graphed_callables(hip_device):
    """The backward is a graph, and a capture, of its own."""

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.drop = Dropout(0.5)

        def forward(self, v):
            return torch.utils.checkpoint.checkpoint(lambda u: self.drop(u * u), v, use_reentrant=False)

    x = torch.ones(2000, device=hip_device, requires_grad=True)
    graphed = torch.cuda.make_graphed_callables(Block(), (torch.ones_like(x).requires_grad_(True),))
    seen = []
    for _ in range(3):
        y = graphed(x)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx != 0, y != 0)
        seen.append((y != 0).clone())
    assert not any(torch.equal(a, b) for n, a in enumerate(seen) for b in seen[:n])


def test_a_captured_forward_is_not_taken_again_after_an_eager_one(hip_device):
    """Its event is gone then, and another mask would be wrong."""
    layer = Dropout(0.5)
    x = torch.ones(300, device=hip_device, requires_grad=True)
    graph, y = captured(lambda: torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=False))
    graph.replay()
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    assert torch.equal(dx != 0, y != 0)                     # an eager backward of a captured forward
    layer(x)
    with pytest.raises(RuntimeError, match="after an eager one"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_the_same_seed_is_the_same_mask_within_a_capture(hip_device):
    """As it is in eager passes; another capture with it counts on."""
    layer, x = Dropout(0.5), torch.ones(700, device=hip_device)

    def call():
        torch.manual_seed(6)
        a = layer(x)
        torch.manual_seed(6)
        return a, layer(x)

    eager = call()
    assert torch.equal(*eager)
    graph, pair = captured(call)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):                          # no eager pass between the captures
        other = call()
    graph.replay()
    torch.cuda.synchronize()
    first = pair[0].clone()
    assert torch.equal(*pair) and not torch.equal(first, eager[0])
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(*other) and not torch.equal(other[0], first)


def test_graphs_outlive_their_layers(hip_device):
    """What a graph counts up is not the layer's: nothing of it is freed, copied or saved."""
    x = torch.ones(500, device=hip_device)
    layer = Dropout(0.5)
    assert not layer.state_dict() and not list(layer.buffers())
    graphs = [captured(lambda: layer(x)), captured(lambda twin=copy.deepcopy(layer): twin(x))]
    del layer
    others = [torch.full((1,), -1, device=hip_device) for _ in range(100)]
    seen = []
    for _ in range(3):
        for graph, y in graphs:
            graph.replay()
            seen.append((y != 0).clone())
    torch.cuda.synchronize()
    assert all(bool((o == -1).all()) for o in others)
    assert not any(torch.equal(a, b) for n, a in enumerate(seen) for b in seen[:n])


def test_copies_and_pickles_have_captured_nothing(hip_device):
    """The events of a capture are its layer's own; a layer that was pickled without a place for them has one."""
    x = torch.ones(100, device=hip_device)
    layer = Dropout(0.5)
    captured(lambda: layer(x))
    assert len(layer._captured) == 1
    older = Dropout(0.5)
    older.__setstate__({k: v for k, v in layer.__dict__.items() if k != "_captured"})
    for other in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer)), older):
        assert other._captured == {} and other.p == 0.5
        torch.manual_seed(3)
        y = other(x)
        torch.manual_seed(3)
        assert torch.equal(y, memfast.dropout(x, 0.5, seed=int(torch.randint(1 << 62, ()))))
