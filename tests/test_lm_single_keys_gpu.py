"""Queries that see one key: their softmax is constant, so nothing goes back to q and k, exactly."""
import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, TYPES, i32, lm, rand, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, G, D, B", [(4, 2, 64, 16), (6, 1, 96, 64), (32, 1, 128, 32), (2, 2, 256, 16)])
def test_first_tokens_and_lone_sequences(lm, dtype, H, G, D, B):
    gen = torch.Generator().manual_seed(D + B)
    lens = [1, 1, 70, 1, 0, 40, 2 * B + 1]
    n = sum(lens)
    q, dout = (rand(gen, n, H, D, dtype=dtype) for _ in range(2))
    k, v = (rand(gen, n, G, D, dtype=dtype) for _ in range(2))
    idx = i32([0, 1, 2]).expand(n, G, 3).contiguous()
    last = n - 1
    idx[last] = i32([2, -1, -1])  # lists the block of which it is the only key
    cu = i32([sum(lens[:i]) for i in range(len(lens) + 1)]).to(DEV)
    seqs, lay, scale = lm.Seqs(len(lens), cu_q=cu, cu_k=cu), lo.packed(lens, lens), D ** -0.5
    a = [x.to(DEV) for x in (q, k, v, idx)]
    out, lse = lm.block_attention(*a, block=B, seqs=seqs, return_lse=True)
    dq, dk, dv = lm.block_attention_backward(dout.to(DEV), *a, out, lse, block=B, seqs=seqs)
    starts = [sum(lens[:i]) for i in range(len(lens)) if lens[i]]
    assert (dq[starts] == 0).all() and (dq[last] == 0).all()
    lone = [s for s in starts if lens[sum(x <= s for x in [sum(lens[:i + 1]) for i in range(len(lens))])] == 1] + [last]
    assert len(lone) == 4 and (dk[lone] == 0).all()
    want = lo.attention(q, k, v, idx, lay, B, scale, True, dout)
    every = torch.ones(n, dtype=torch.bool)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        within(x, want[name], want["tol_" + name], every, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_queries_over_one_key(lm, dtype):
    """Not causal, a last block of one key: rows that list it alone stand among rows that list more."""
    gen = torch.Generator().manual_seed(98)
    n, H, G, D, B = 75, 4, 1, 64, 64
    q, dout = (rand(gen, n, H, D, dtype=dtype) for _ in range(2))
    k, v = (rand(gen, 65, G, D, dtype=dtype) for _ in range(2))
    idx = i32([0, 1]).expand(n, G, 2).contiguous()
    alone = torch.arange(n) % 3 == 1
    idx[alone] = i32([1, -1])
    a = [x.to(DEV) for x in (q, k, v, idx)]
    out, lse = lm.block_attention(*a, block=B, causal=False, return_lse=True)
    dq, dk, dv = lm.block_attention_backward(dout.to(DEV), *a, out, lse, block=B, causal=False)
    assert (dq[alone.to(DEV)] == 0).all()
    want = lo.attention(q, k, v, idx, lo.uniform(1, n, 65), B, D ** -0.5, False, dout)
    every = torch.ones(n, dtype=torch.bool)
    for name, x, rows in (("dq", dq, every), ("dk", dk, every[:65]), ("dv", dv, every[:65])):
        within(x, want[name], want["tol_" + name], rows, name)
    # the last key's gradient without the rows that have no part in it
    rest = [x[~alone].contiguous().to(DEV) for x in (q, idx, dout)]
    o, s = lm.block_attention(rest[0], a[1], a[2], rest[1], block=B, causal=False, return_lse=True)
    _, ek, _ = lm.block_attention_backward(rest[2], rest[0], a[1], a[2], rest[1], o, s, block=B, causal=False)
    lw = lo.attention(q[~alone], k, v, idx[~alone], lo.uniform(1, int((~alone).sum()), 65), B, D ** -0.5, False, dout[~alone])
    within(dk, lw["dk"], want["tol_dk"], every[:65], "dk")
    within(ek, lw["dk"], lw["tol_dk"], every[:65], "dk")


def test_numbers_that_are_none_stay_none(lm):
    """A single key whose query has a gradient that is no number: its own gradients are none, as the formula's."""
    gen = torch.Generator().manual_seed(97)
    q, k, v = (rand(gen, 1, 2, 64).to(DEV) for _ in range(3))
    idx = torch.zeros(1, 2, 1, dtype=torch.int32, device=DEV)
    out, lse = lm.block_attention(q, k, v, idx, block=16, return_lse=True)
    dout = torch.full_like(q, float("nan"))
    assert all(x.isnan().all() for x in lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=16))
