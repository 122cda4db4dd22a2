"""Launches of more workgroups than one grid dimension holds threads for, page tables cut out of wider ones, numbers that do not fit."""
import math

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, check_attention, i32, lm, rand, random_pattern, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def test_more_tokens_than_one_grid_dimension_holds(lm):
    tokens, channels, experts = 2 ** 24 + 5, 520, 3
    gen = torch.Generator(device=DEV).manual_seed(61)
    ids = torch.randint(-1, experts, (tokens, 1), generator=gen, dtype=torch.int32, device=DEV)
    plan = lm.route(ids, experts)
    x = torch.empty(tokens, channels, dtype=torch.bfloat16, device=DEV)
    x.view(torch.int16).random_(0, 16000, generator=gen)  # the bits of numbers from 0 to 0.25
    xs = lm.gather_tokens(x, plan)
    pick = torch.cat([torch.randint(0, tokens, (2000,), generator=gen, device=DEV), torch.arange(tokens - 300, tokens, device=DEV)])
    there = plan.place[pick, 0] >= 0
    assert torch.equal(xs[plan.place[pick, 0].clamp(min=0).long()][there], x[pick][there])
    out = lm.combine_tokens(xs, plan, torch.full((tokens, 1), 2.0, device=DEV))
    assert torch.equal(out[pick], torch.where(there[:, None], 2 * x[pick], 0))
    del out
    w = torch.full((tokens, 1), 0.5, device=DEV)
    dy, dw = lm.combine_tokens_backward(x, xs, plan, w)
    assert torch.equal(dy[plan.place[pick, 0].clamp(min=0).long()][there], (x[pick].float() * 0.5).bfloat16()[there])
    square = (x[pick].double() ** 2).sum(1)
    # a sum of 520 products in 32 bits
    assert ((dw[pick, 0].double() - torch.where(there, square, 0)).abs() <= 522 * lo.U32 * square).all()


def test_more_rows_than_one_grid_dimension_holds(lm):
    gen = torch.Generator().manual_seed(62)
    rows, nb, B, D, W = 2 ** 22 + 7, 2050, 16, 8, 4
    q = torch.randn(rows, 1, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(62)).bfloat16()
    means = rand(gen, nb, 1, D, dtype=torch.bfloat16)
    seqs = lm.Seqs(1, k_len=i32([nb * B]).to(DEV))
    got = lm.select_blocks(q, means.to(DEV), block=B, width=W, first=0, local=0, causal=False, k_rows=nb * B, seqs=seqs)
    pick = [0, 1, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, 3000000, 2 ** 22 - 1, 2 ** 22, rows - 2, rows - 1]
    want = lo.select(q[pick].cpu(), {(0, b): means[b] for b in range(nb)}, lo.uniform(1, len(pick), nb * B), B, W, 0, 0, False)
    assert torch.equal(got[pick].cpu(), want)


def test_more_conversations_than_one_grid_dimension_holds(lm):
    gen = torch.Generator(device=DEV).manual_seed(63)
    n, D, B, pages = 2 ** 23 + 9, 8, 16, 64
    k, v = (torch.randn(pages, B, 1, D, device=DEV, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(n, 1, D, device=DEV, generator=gen).bfloat16()
    lens = torch.randint(0, B + 1, (n,), generator=gen, dtype=torch.int32, device=DEV)
    table = torch.randint(0, pages, (n, 1), generator=gen, dtype=torch.int32, device=DEV)
    idx = torch.zeros(n, 1, 1, dtype=torch.int32, device=DEV)
    out, lse = lm.block_attention(q, k, v, idx, block=B, seqs=lm.Seqs(n, k_len=lens, page_table=table), return_lse=True)
    pick = torch.cat([torch.randint(0, n, (300,), generator=gen, device=DEV), torch.arange(n - 40, n, device=DEV)])
    lay = lo.paged(lens[pick].tolist(), table[pick].tolist(), B, pages)
    want = lo.attention(q[pick].cpu(), k.cpu().view(-1, 1, D), v.cpu().view(-1, 1, D), idx[pick].cpu(), lay, B, 1 / math.sqrt(D), True)
    every = torch.ones(len(pick), dtype=torch.bool)
    within(out[pick], want["out"], want["tol_out"], every, "out")
    within(lse[pick], want["lse"], want["tol_lse"], every, "lse")


def test_page_table_cut_out_of_a_wider_one(lm):
    gen = torch.Generator().manual_seed(64)
    n, per, page, G, D, B = 5, 4, 32, 2, 64, 16
    pages = n * per
    deal = torch.randperm(pages, generator=gen).view(n, per)
    wide = torch.full((n, 9), -1, dtype=torch.int32)
    wide[:, 2:6] = deal.int()
    lens = [1, 128, 77, 0, 100]
    k, v = (rand(gen, pages, page, G, D, dtype=torch.bfloat16) for _ in range(2))
    q = rand(gen, n, 4, D, dtype=torch.bfloat16)
    idx = random_pattern(gen, n, G, 5, 8)
    # a cut from the table's middle keeps the last row's end only if something stands behind the table
    room = torch.cat([wide.flatten(), torch.full((9,), -1, dtype=torch.int32)]).to(DEV)[:n * 9 + 2].view(-1)
    table = torch.as_strided(room, (n, per), (9, 1), 2)
    seqs = lm.Seqs(n, k_len=i32(lens).to(DEV), page_table=table)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.paged(lens, deal.tolist(), page, pages), seqs, B, None, True, None,
                    kv_flat=(k.view(-1, G, D), v.view(-1, G, D)))


def test_numbers_that_do_not_fit(lm):
    x = torch.zeros(4, 2, 64, device=DEV)
    idx = torch.zeros(4, 2, 1, dtype=torch.int32, device=DEV)
    for change in (dict(block=2 ** 40), dict(scale=1e39), dict(block=16, scale=math.nan)):
        with pytest.raises(ValueError):
            lm.block_attention(x, x, x, idx, **{"block": 16, **change})
    with pytest.raises(ValueError):
        lm.select_blocks(x, x[:1], block=16, width=2 ** 33, k_rows=4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("channels", [1, 7, 8, 37, 1029])
def test_rows_of_tokens_that_begin_anywhere(lm, dtype, channels):
    """Tensors whose first element stands behind any multiple of 16 bytes: as tensors that begin at one, and nothing beside them is written."""
    gen = torch.Generator().manual_seed(channels)
    T, K, E = 41, 3, 5
    ids = torch.randint(-1, E, (T, K), generator=gen, dtype=torch.int32).to(DEV)
    plan = lm.route(ids, E)
    live = int(plan.offsets[-1])
    w = torch.rand(T, K, generator=gen).to(DEV)

    def off(t, by):
        room = torch.full((t.numel() + 32,), 9.0, dtype=t.dtype, device=DEV)
        room[by:by + t.numel()] = t.flatten()
        return room[by:by + t.numel()].view(t.shape)

    x, dout = rand(gen, T, channels, dtype=dtype).to(DEV), rand(gen, T, channels, dtype=dtype).to(DEV)
    xs = lm.gather_tokens(x, plan)
    y = lm.combine_tokens(xs, plan, w)
    dy, dw = lm.combine_tokens_backward(dout, xs, plan, w)
    from nsparse_amd.capi import load_lm
    for by in (1, 3, 5):
        assert torch.equal(lm.gather_tokens(off(x, by), plan)[:live], xs[:live])
        assert torch.equal(lm.combine_tokens(off(xs, by), plan, w), y)
        a, b = lm.combine_tokens_backward(off(dout, by), off(xs, by), plan, w)
        assert torch.equal(a[:live], dy[:live]) and torch.equal(b, dw)
        # an output in the middle of other numbers
        room = torch.full((T * channels + 32,), 9.0, dtype=dtype, device=DEV)
        code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
        assert load_lm().nsparse_lm_combine_tokens(code, xs.data_ptr(), plan.place.data_ptr(), w.data_ptr(), T, K, channels,
                                                   room[by:].data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(room[by:by + T * channels].view(T, channels), y)
        assert (room[:by] == 9).all() and (room[by + T * channels:] == 9).all()
