"""Calls at the edges of what their documentation allows."""
import math

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, TYPES, check_attention, i32, lm, rand, random_pattern  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("last", [1, 15, 16, 17, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("packed", [False, True])
def test_means_of_the_last_keys_of_any_number(lm, last, packed):
    gen = torch.Generator().manual_seed(95)
    n, each, G, D, B = 16, 40, 2, 64, 16
    k = rand(gen, n * each, G, D, dtype=torch.bfloat16).to(DEV)
    seqs = lm.Seqs(n, cu_k=i32([each * s for s in range(n + 1)]).to(DEV)) if packed else lm.Seqs(n)
    whole = lm.block_means(k, block=B, seqs=seqs)
    out = torch.full_like(whole, 7.0)
    lm.block_means(k, block=B, seqs=seqs, last=last, out=out)
    for s in range(n):
        base = each * s // B + s if packed else 3 * s
        for b in range(3):
            if 16 * b + 16 > each - last:
                assert torch.equal(out[base + b], whole[base + b])
            else:
                assert (out[base + b] == 7).all()
