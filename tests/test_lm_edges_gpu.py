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


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_conversations_without_a_page(lm, dtype, n):
    """A table of no columns: no keys, so no blocks, outputs of zeros."""
    gen = torch.Generator().manual_seed(96)
    G, D, B = 2, 64, 16
    k, v = (rand(gen, 4, 32, G, D, dtype=dtype).to(DEV) for _ in range(2))
    q = rand(gen, n, 4, D, dtype=dtype).to(DEV)
    seqs = lm.Seqs(n, k_len=i32([7] * n).to(DEV), page_table=torch.empty(n, 0, dtype=torch.int32, device=DEV))
    means = torch.full((8, G, D), 7.0, dtype=dtype, device=DEV)
    for last in (0, 1):
        lm.block_means(k, block=B, seqs=seqs, last=last, out=means)
    assert (means == 7).all()
    idx = lm.select_blocks(q, means, block=B, width=4, k_rows=4, seqs=seqs)
    assert (idx == -1).all()
    for listed in (idx, torch.zeros_like(idx)):
        out, lse = lm.block_attention(q, k, v, listed, block=B, seqs=seqs, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
