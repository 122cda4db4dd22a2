"""Prompts and batches large enough for the forms that share keys between neighbouring rows, share a block's rows out, or select over very
many blocks, against the plain 64-bit forms and with the bounds of tests/lm_oracle.py."""
import math

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, TYPES, check_attention, i32, lm, rand, random_pattern, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def starts(lens):
    return i32([sum(lens[:i]) for i in range(len(lens) + 1)]).to(DEV)


# ---- prompts -------------------------------------------------------------------------------------------------------------------
# rows x key heads (x slices of 16 query heads) reaches 2048 in each, so that neighbouring rows walk their blocks together
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads, kv, dim, block, width, ql, kl", [
    (8, 4, 64, 16, 5, [130, 1, 0, 300, 89], [130, 1, 7, 300, 89]),      # several sequences in a workgroup
    (12, 4, 96, 32, 20, [513], [513]),                                   # rows wider than 16, columns without a row
    (40, 2, 128, 64, 3, [500, 20], [700, 5]),                            # 20 query heads a key head; more and fewer keys than queries
    (4, 4, 128, 64, 70, [520], [4600]),                                  # one query head a key head, rows wider than 64
    (5, 5, 200, 128, 2, [417], [417]),
    (3, 3, 256, 256, 3, [700], [1000])])
def test_prompts(lm, dtype, heads, kv, dim, block, width, ql, kl):
    gen = torch.Generator().manual_seed(heads * 100 + dim + block)
    Tq, Tk = sum(ql) + 3, sum(kl) + 5
    q, dout = rand(gen, Tq, heads, dim, dtype=dtype), rand(gen, Tq, heads, dim, dtype=dtype)
    k, v = rand(gen, Tk, kv, dim, dtype=dtype), rand(gen, Tk, kv, dim, dtype=dtype)
    idx = random_pattern(gen, Tq, kv, width, -(-max(kl) // block))
    idx[::3] = random_pattern(gen, len(range(0, Tq, 3)), kv, width, -(-max(kl) // block), wild=True)
    seqs = lm.Seqs(len(ql), cu_q=starts(ql), cu_k=starts(kl))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.packed(ql, kl), seqs, block, None, True, dout)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("dim", [64, 120, 128])
def test_prompts_with_two_sets_of_columns(lm, dtype, dim):
    """16 query heads a key head: a wavefront has two rows of 16 columns."""
    gen = torch.Generator().manual_seed(dim)
    heads, kv, block, width, ql = 64, 4, 64, 3, [600, 3, 441]
    T = sum(ql)
    q, k, v = (rand(gen, T, h, dim, dtype=dtype) for h in (heads, kv, kv))
    idx = random_pattern(gen, T, kv, width, 10)
    idx[::4] = random_pattern(gen, len(range(0, T, 4)), kv, width, 10, wild=True)
    seqs = lm.Seqs(len(ql), cu_q=starts(ql), cu_k=starts(ql))
    lay = lo.packed(ql, ql)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lay, seqs, block, None, True, None, kv_flat=(k, v))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale, causal", [(-0.2, True), (0.0, True), (0.11, False)])
def test_prompts_of_any_scale(lm, dtype, scale, causal):
    gen = torch.Generator().manual_seed(41)
    n, heads, kv, dim, block, width = 520, 8, 4, 64, 64, 3
    q, dout = rand(gen, n, heads, dim, dtype=dtype), rand(gen, n, heads, dim, dtype=dtype)
    k, v = rand(gen, n, kv, dim, dtype=dtype), rand(gen, n, kv, dim, dtype=dtype)
    idx = random_pattern(gen, n, kv, width, 9)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.uniform(1, n, n), None, block, scale, causal, dout)
    few = 30
    check_attention(lm, q[:few].to(DEV), k.to(DEV), v.to(DEV), idx[:few].contiguous(), lo.uniform(1, few, n), None, block, scale, causal, dout[:few])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("block", [16, 32, 64])
def test_neighbours_do_not_see_each_others_blocks(lm, dtype, block):
    """Blocks that hold NaN or infinities are listed by every seventh row only: the other rows' outputs and gradients are as ever."""
    gen = torch.Generator().manual_seed(42)
    n, heads, kv, dim, width = 600, 8, 4, 64, 4
    q, dout = rand(gen, n, heads, dim, dtype=dtype), rand(gen, n, heads, dim, dtype=dtype)
    k, v = rand(gen, n, kv, dim, dtype=dtype), rand(gen, n, kv, dim, dtype=dtype)
    blocks = -(-n // block)
    idx = random_pattern(gen, n, kv, width, blocks)
    k[block:2 * block], v[3 * block:4 * block], v[5 * block + 3] = math.nan, math.inf, math.nan
    clean = torch.ones(n, dtype=torch.bool)
    clean[::7] = False
    bad = (idx == 1) | (idx == 3) | (idx == 5)
    idx[clean.view(-1, 1, 1) & bad] = -1  # entries that do not count
    want = lo.attention(q, torch.nan_to_num(k.float(), 0, 0, 0).to(dtype), torch.nan_to_num(v.float(), 0, 0, 0).to(dtype), idx, lo.uniform(1, n, n), block,
                        0.125, True, dout)
    dev = [x.to(DEV) for x in (q, k, v, idx)]
    out, lse = lm.block_attention(*dev, block=block, scale=0.125, return_lse=True)
    within(out, want["out"], want["tol_out"], clean, "out")
    within(lse, want["lse"], want["tol_lse"], clean, "lse")
    dq, _, _ = lm.block_attention_backward(dout.to(DEV), *dev, out, lse, block=block, scale=0.125)
    within(dq, want["dq"], want["tol_dq"], clean, "dq")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_prompts_over_very_many_blocks(lm, dtype):
    """More blocks than one range of the walk, both in the forward and in the gradients."""
    gen = torch.Generator().manual_seed(43)
    rows, heads, kv, dim, block, width = 300, 8, 8, 64, 16, 6
    n = 2500 * block + 5
    q, dout = rand(gen, rows, heads, dim, dtype=dtype), rand(gen, rows, heads, dim, dtype=dtype)
    k, v = rand(gen, n, kv, dim, dtype=dtype), rand(gen, n, kv, dim, dtype=dtype)
    idx = random_pattern(gen, rows, kv, width, 2501)
    idx[::2, :, :2] = i32([1023, 1024])  # around the border of the ranges
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.uniform(1, rows, n), None, block, None, True, dout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("block, page", [(16, 48), (64, 64), (32, 128)])
def test_pieces_of_prompts_over_a_paged_cache(lm, dtype, block, page):
    """40 new tokens of each of 14 conversations; some pages of the table are none, and such keys are hidden."""
    gen = torch.Generator().manual_seed(44)
    n, each, heads, kv, dim, width = 14, 40, 16, 4, 64, 5
    per = -(-600 // page)
    pages = n * per
    lens = [40 + int(x) for x in torch.randint(0, 560, (n,), generator=gen)]
    table = torch.randperm(pages, generator=gen).view(n, per)
    table[3, 1] = table[5, 0] = -1
    table[7, 0] = pages
    k, v = (rand(gen, pages, page, kv, dim, dtype=dtype) for _ in range(2))
    q = rand(gen, n * each, heads, dim, dtype=dtype)
    idx = random_pattern(gen, n * each, kv, width, -(-600 // block))
    seqs = lm.Seqs(n, k_len=i32(lens).to(DEV), page_table=table.int().to(DEV))
    lay = lo.paged(lens, table.tolist(), page, pages, q_each=each)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lay, seqs, block, None, True, None, kv_flat=(k.view(-1, kv, dim), v.view(-1, kv, dim)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 100 // 8 * 8, 128, 256])
def test_single_tokens_of_very_many_conversations(lm, dtype, dim):
    gen = torch.Generator().manual_seed(45)
    n, heads, kv, block, page, width = 1030, 4, 2, 16, 32, 4
    pages = 2 * n
    lens = [int(x) for x in torch.randint(0, 65, (n,), generator=gen)]
    table = torch.randperm(pages, generator=gen).view(n, 2)
    k, v = (rand(gen, pages, page, kv, dim, dtype=dtype) for _ in range(2))
    q = rand(gen, n, heads, dim, dtype=dtype)
    idx = random_pattern(gen, n, kv, width, 4)
    seqs = lm.Seqs(n, k_len=i32(lens).to(DEV), page_table=table.int().to(DEV))
    lay = lo.paged(lens, table.tolist(), page, pages)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lay, seqs, block, None, True, None, kv_flat=(k.view(-1, kv, dim), v.view(-1, kv, dim)))


def test_gradients_of_shared_out_blocks_do_not_depend_on_timing(lm):
    """Every row lists the first block: its rows are many items' work, their sums are joined in order."""
    gen = torch.Generator().manual_seed(46)
    n, heads, kv, dim, block = 3000, 8, 2, 64, 64
    q, k, v, dout = (rand(gen, n, h, dim, dtype=torch.bfloat16).to(DEV) for h in (heads, kv, kv, heads))
    idx = random_pattern(gen, n, kv, 30, 47)
    idx[:, :, 0] = 0
    idx = torch.sort(idx, dim=2).values.to(DEV)
    out, lse = lm.block_attention(q, k, v, idx, block=block, return_lse=True)
    first = lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=block)
    for _ in range(3):
        again = lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=block)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- selection -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("nb, dim, width", [(200, 64, 16), (255, 200, 5), (700, 128, 16), (700, 256, 200), (1900, 64, 33), (1900, 256, 8)])
def test_selection_of_prompts(lm, dtype, nb, dim, width):
    gen = torch.Generator().manual_seed(nb + dim)
    B, rows, H, G = 16, 37, 6, 2
    n = nb * B - 3
    q = rand(gen, rows, H, dim, dtype=dtype)
    means = rand(gen, nb, G, dim, dtype=dtype)
    means[5] = means[9]  # ties
    held = {(0, b): means[b] for b in range(nb)}
    lay = lo.uniform(1, rows, n)
    seqs = lm.Seqs(1, q_len=i32([rows]).to(DEV), k_len=i32([n]).to(DEV))
    for first, local, causal in ((1, 2, True), (0, 0, False)):
        got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=width, first=first, local=local, causal=causal, k_rows=n, seqs=seqs)
        assert torch.equal(got.cpu(), lo.select(q, held, lay, B, width, first, local, causal))


def test_selection_over_more_blocks_than_scores_are_held_for(lm):
    gen = torch.Generator().manual_seed(51)
    nb, B, D = 33001, 16, 8
    q = rand(gen, 2, 2, D)
    means = rand(gen, nb, 1, D)
    for width, first in ((16, 1), (256, 0)):
        got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=width, first=first, local=2, k_rows=nb * B)
        want = lo.select(q, {(0, b): means[b] for b in range(nb)}, lo.uniform(1, 2, nb * B), B, width, first, 2, True)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("each", [1, 20])
def test_selection_where_pages_are_none(lm, each):
    """Blocks of pages that are none score lowest, whatever their number."""
    gen = torch.Generator().manual_seed(52)
    n, per, page, B, H, G, D, W = 6, 12, 64, 32, 4, 2, 64, 9
    pages = n * per
    lens = [each, 30, 64, 333, 700, 768]
    table = torch.randperm(pages, generator=gen).view(n, per)
    table[3, 2:4] = -1
    table[4, 1:] = -1
    table[5, ::2] = pages + 3
    means = rand(gen, pages * page // B, G, D, dtype=torch.bfloat16)
    q = rand(gen, n * each, H, D, dtype=torch.bfloat16)
    held = {}
    for s in range(n):
        for b in range(-(-lens[s] // B)):
            p = int(table[s, b * B // page])
            if 0 <= p < pages:
                held[s, b] = means[p * (page // B) + b % (page // B)]
    seqs = lm.Seqs(n, k_len=i32(lens).to(DEV), page_table=table.int().to(DEV))
    got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=W, first=1, local=1, k_rows=pages, seqs=seqs)
    want = lo.select(q, held, lo.paged(lens, table.tolist(), page, pages, q_each=each), B, W, 1, 1, True)
    assert torch.equal(got.cpu(), want)
