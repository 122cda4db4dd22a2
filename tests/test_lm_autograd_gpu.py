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
