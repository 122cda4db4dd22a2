"""The rule by which nsparse_amd.lm refuses a capture, without a GPU: threads beside a capture."""
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
    """Whether this thread is capturing."""
    here = threading.local()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: getattr(here, "capturing", False))
    return here


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
    streams.capturing = True
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
