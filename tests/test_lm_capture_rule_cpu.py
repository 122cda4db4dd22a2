"""The rule by which nsparse_amd.lm refuses a capture, without a GPU: which leaves an autograd graph reaches, and threads beside a capture."""
import sys
import threading
import time

import pytest

torch = pytest.importorskip("torch")


class Node(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        from nsparse_amd import lm
        lm._may_capture(ctx, *inputs)
        return sum(x.sum() for x in inputs)

    @staticmethod
    def backward(ctx, g):
        return g


@pytest.fixture
def streams(monkeypatch):
    """Whether this thread is capturing, and its stream's handle."""
    from nsparse_amd import lm
    here = threading.local()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: getattr(here, "capturing", False))
    monkeypatch.setattr(lm, "_raw_stream", lambda dev: getattr(here, "stream", 0))
    return here


def test_leaves_of_a_graph():
    from nsparse_amd import lm
    w, b, x = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True), torch.ones(3)
    y = (x * w + b).exp()
    assert lm._leaves_behind(y) == {id(w), id(b)} and lm._leaves_behind(w) == {id(w)} and lm._leaves_behind(x) == set()
    assert lm._leaves_behind(y.grad_fn, w) == {id(w), id(b)}
    deep = w
    for _ in range(5000):
        deep = deep + b
    assert lm._leaves_behind(deep) == {id(w), id(b)}


def test_graphs_that_keep_a_capture_from_its_leaves(streams):
    w, v = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)

    def captured(*inputs):
        streams.capturing, before = True, getattr(streams, "stream", 0)
        streams.stream = 5
        try:
            return Node.apply(*inputs)
        finally:
            streams.capturing, streams.stream = False, before

    alive = Node.apply(w * 2)
    captured(v), captured(v * 2)  # other leaves
    for inputs in ((w,), (w * 3,), (v, (w + v).exp())):
        with pytest.raises(RuntimeError, match="alive"):
            captured(*inputs)
    del alive
    captured(w), captured(w * 3)
    streams.stream = 7  # a stream that can join a capture: only the call's own leaves are refused
    alive = Node.apply(w * 2), Node.apply(v)
    captured(w * 3)
    with pytest.raises(RuntimeError, match="alive"):
        captured(v)
    del alive
    captured(v)


def test_threads_beside_a_capture(streams):
    stop, errors = time.time() + 1.0, []
    many = torch.ones(1, requires_grad=True)
    crowd = [Node.apply(many) for _ in range(2000)]
    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)

    def work():
        w = torch.ones(1, requires_grad=True)
        kept = []
        while time.time() < stop:
            kept = [Node.apply(w) for _ in range(20)]
        del kept

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    streams.capturing, streams.stream = True, 5
    x = torch.ones(1, requires_grad=True)
    while time.time() < stop:
        try:
            Node.apply(x, x * 2)
        except RuntimeError as e:
            errors.append(str(e))
    for t in threads:
        t.join()
    sys.setswitchinterval(before)
    assert crowd and not errors, errors[0]
