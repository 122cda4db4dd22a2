"""What autograd hands to the operators of nsparse_amd.lm, and what they hand back."""
import math

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, TYPES, i32, lm, rand, random_pattern, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def small(seed, dtype, n=50, H=4, G=2, D=64, B=16, W=3):
    """Leaves q, k, v, a pattern and a gradient of the output."""
    gen = torch.Generator().manual_seed(seed)
    leaves = [rand(gen, n, h, D, dtype=dtype).to(DEV).requires_grad_() for h in (H, G, G)]
    return leaves, random_pattern(gen, n, G, W, -(-n // B)).to(DEV), rand(gen, n, H, D, dtype=dtype).to(DEV), B


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("before", [1, 3, 8])
def test_a_gradient_that_begins_anywhere(lm, dtype, before):
    """The output joined behind a few other numbers: its gradient is a piece of the whole's that begins off 16 bytes."""
    leaves, idx, dout, B = small(81, dtype)
    out = lm.block_attention(*leaves, idx, block=B)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    whole = torch.cat([torch.zeros(before, dtype=dtype, device=DEV), out.flatten()])
    got = torch.autograd.grad(whole, leaves, torch.cat([torch.ones(before, dtype=dtype, device=DEV), dout.flatten()]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_is_refused(lm):
    """A tensor with a tangent, in any place of any differentiable call: the derivative must not be lost silently."""
    import torch.autograd.forward_ad as fw
    leaves, idx, dout, B = small(82, torch.float32)
    q, k, v = (x.detach() for x in leaves)
    out, lse = lm.block_attention(q, k, v, idx, block=B, return_lse=True)
    gen = torch.Generator().manual_seed(82)
    T, K, E, Ch = 20, 2, 4, 8
    plan = lm.route(torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32).to(DEV), E)
    x, w, y = rand(gen, T, Ch).to(DEV), torch.rand(T, K, generator=gen).to(DEV), rand(gen, T * K, Ch).to(DEV)
    calls = [(lambda *a: lm.block_attention(*a, idx, block=B), (q, k, v)),
             (lambda *a: lm.block_attention(*a, idx, block=B, out=torch.empty_like(q)), (q, k, v)),
             (lambda d, a, b, c, o, s: lm.block_attention_backward(d, a, b, c, idx, o, s, block=B), (dout, q, k, v, out, lse)),
             (lambda a: lm.gather_tokens(a, plan), (x,)), (lambda a: lm.gather_tokens_backward(a, plan), (y,)),
             (lambda a, b: lm.combine_tokens(a, plan, b), (y, w)),
             (lambda a, b, c: lm.combine_tokens_backward(a, b, plan, c), (x, y, w))]
    with fw.dual_level():
        for f, args in calls:
            f(*args)
            for i in range(len(args)):
                with pytest.raises(NotImplementedError):
                    f(*[fw.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)])
        # through a backward pass: a gradient with a tangent
        o = lm.block_attention(*leaves, idx, block=B)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(o, leaves, fw.make_dual(dout, torch.ones_like(dout)))
