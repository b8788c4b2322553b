"""The guard that keeps a capture from autograd graphs of another stream: the condition as the calls meet it, on the CPU with a stand-in for the GPU's
streams."""
import pytest
import torch


class Leaf(torch.Tensor):
    is_cuda = True


class Twice(torch.autograd.Function):
    calls = 0

    @staticmethod
    def forward(ctx, x):
        Twice.calls += 1
        return x.as_subclass(torch.Tensor) * 2

    @staticmethod
    def backward(ctx, g):
        return g * 2


@pytest.fixture
def gpu(monkeypatch):
    from univtg_amd import attention, ops

    class State:
        stream, capturing = 0, False

        def call(self, x, stream=0, capturing=False):
            self.stream, self.capturing = stream, capturing
            return attention._apply(Twice, (x,), x)
    state = State()
    monkeypatch.setattr(ops, "_stream_of", lambda t: state.stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    return state


def leaf():
    return torch.zeros(3).as_subclass(Leaf).requires_grad_(True)


def test_capture_is_refused_before_anything_runs(gpu):
    x = leaf()
    alive = gpu.call(x)
    before = Twice.calls
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        gpu.call(x, stream=7, capturing=True)
    assert Twice.calls == before
    gpu.call(leaf(), stream=7, capturing=True)               # leaves of its own
    gpu.call(x, stream=7)                                    # no capture
    del alive
    gpu.call(x, stream=7, capturing=True)


def test_capture_is_let_through_on_the_stream_of_the_living_graph(gpu):
    x = leaf()
    alive = gpu.call(x, stream=7)
    first = gpu.call(x, stream=7, capturing=True)            # (the same leaf twice in one capture)
    gpu.call(x, stream=7, capturing=True)
    assert alive is not None and first is not None


def test_an_accumulator_keeps_the_stream_that_it_was_made_on(gpu):
    """As long as some graph of the leaf lives it is the first one's accumulator that all of them share, on the first one's stream."""
    x = leaf()
    first = gpu.call(x, stream=0)
    second = gpu.call(x, stream=7)
    assert first.grad_fn.next_functions[0][0] is second.grad_fn.next_functions[0][0]
    del first
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        gpu.call(x, stream=7, capturing=True)
    third = gpu.call(x, stream=7)
    del second
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        gpu.call(x, stream=7, capturing=True)
    del third
    gpu.call(x, stream=7, capturing=True)
