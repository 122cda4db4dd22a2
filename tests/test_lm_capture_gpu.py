"""Forward and backward through autograd, captured into a graph."""
import pytest

torch = pytest.importorskip("torch")
from test_lm_gpu import DEV, lm, rand, random_pattern  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def on_a_side_stream(f):
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        f()
    torch.cuda.current_stream().wait_stream(st)


@pytest.mark.parametrize("rows", [70, 600])
def test_attention_and_its_gradient_in_a_graph(lm, rows):
    gen = torch.Generator().manual_seed(rows)
    H, G, D, B, W = 8, 4, 64, 16, 3
    leaves = [rand(gen, rows, h, D, dtype=torch.bfloat16).to(DEV).requires_grad_() for h in (H, G, G)]
    idx = random_pattern(gen, rows, G, W, -(-rows // B)).to(DEV)
    dout = rand(gen, rows, H, D, dtype=torch.bfloat16).to(DEV)

    def step():
        out = lm.block_attention(*leaves, idx, block=B)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    alive = lm.block_attention(*leaves, idx, block=B)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(g):
            step()
    alive.backward(dout)  # the eager graph is as it was
    assert all(x.grad is not None for x in leaves)
    del alive
    for x in leaves:
        x.grad = None
    on_a_side_stream(step)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for x in (*leaves, dout):
                x.copy_(rand(gen, *x.shape, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            out, lse = lm.block_attention(*leaves, idx, block=B, return_lse=True)
            want = (out, *lm.block_attention_backward(dout, *leaves, idx, out, lse, block=B))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_routing_and_its_gradient_in_a_graph(lm):
    gen = torch.Generator().manual_seed(7)
    T, K, E, C = 90, 2, 5, 48
    x, w = rand(gen, T, C).to(DEV).requires_grad_(), torch.rand(T, K, generator=gen).to(DEV).requires_grad_()
    ids = torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32).to(DEV)
    dout = rand(gen, T, C).to(DEV)

    def step():
        plan = lm.route(ids, E)
        out = lm.combine_tokens(lm.gather_tokens(x, plan), plan, w)
        return (out.detach(), *torch.autograd.grad(out, (x, w), dout))

    plan = lm.route(ids, E)
    for alive in (lm.gather_tokens(x, plan), lm.combine_tokens(lm.gather_tokens(x.detach(), plan), plan, w)):
        with pytest.raises(RuntimeError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
    del alive
    on_a_side_stream(step)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (x, w, dout):
                t.copy_(torch.rand(t.shape, generator=gen))
            ids.copy_(torch.randint(-1, E, (T, K), generator=gen, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want


def test_weights_have_to_be_given(lm):
    plan = lm.route(torch.zeros(3, 2, dtype=torch.int32, device=DEV), 4)
    with pytest.raises(ValueError):
        lm.combine_tokens(torch.zeros(6, 8, device=DEV), plan, None)
