"""The operators of include/nsparse_lm.h on the GPU against plain 64-bit forms (tests/lm_oracle.py, bounds derived there)."""
import math

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def lm():
    from nsparse_amd import lm as module
    return module


def rand(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def random_pattern(gen, rows, groups, width, blocks, wild=False):
    """Ascending rows with -1 behind; wild: any order, repeats, entries outside the sequence, empty rows."""
    if wild:
        x = torch.randint(-2, blocks + 2, (rows, groups, width), generator=gen, dtype=torch.int32)
        x[::5] = -1
        return x
    out = torch.full((rows, groups, width), -1, dtype=torch.int32)
    for t in range(rows):
        for g in range(groups):
            n = min(blocks, int(torch.randint(0, width + 1, (1,), generator=gen)))
            out[t, g, :n] = torch.sort(torch.randperm(blocks, generator=gen)[:n]).values.int()
    return out


def within(got, want, tol, rows, what):
    d = (got.cpu().double() - want).abs()[rows]
    t = tol[rows]
    both = torch.isinf(want[rows]) & (got.cpu().double()[rows] == want[rows])
    bad = ~((d <= t) | both)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / t)[bad].max()):.3g} of the bound"


def check_attention(lm, q, k, v, idx, layout, seqs, block, scale, causal, dout, kv_flat=None):
    """Forward and (not paged) backward; k, v as the call takes them (any strides), kv_flat their rows for the oracle."""
    kf, vf = kv_flat if kv_flat is not None else (k.cpu(), v.cpu())
    want = lo.attention(q.cpu(), kf, vf, idx, layout, block, scale if scale is not None else 1 / math.sqrt(q.shape[2]), causal,
                        dout if kv_flat is None else None)
    rows = want["covered"]
    ix = idx.to(DEV)
    n, H, D = q.shape
    out = torch.full((n, H, D), 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full((n, H), 7.0, device=DEV)
    with torch.no_grad():
        lm.block_attention(q, k, v, ix, block=block, scale=scale, causal=causal, seqs=seqs, out=out, lse=lse)
    within(out, want["out"], want["tol_out"], rows, "out")
    within(lse, want["lse"], want["tol_lse"], rows, "lse")
    assert (out.cpu()[~rows] == 7).all() and (lse.cpu()[~rows] == 7).all(), "rows of no sequence were written"
    if kv_flat is not None:
        return
    got = lm.block_attention_backward(dout.to(DEV), q, k, v, ix, out, lse, block=block, scale=scale, causal=causal, seqs=seqs)
    every = torch.ones(k.shape[0], dtype=torch.bool)
    for name, x in zip(("dq", "dk", "dv"), got):
        w = want[name]
        within(x, w, want["tol_" + name], rows if name == "dq" else every, name)


# ---- attention: types, heads, sizes -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads, kv, dim, block, width", [
    (8, 2, 64, 16, 4), (4, 4, 128, 64, 3), (6, 2, 96, 16, 5), (1, 1, 8, 32, 2), (16, 1, 80, 32, 4), (40, 2, 64, 16, 4), (3, 3, 256, 16, 3),
    (5, 1, 200, 64, 2), (2, 1, 72, 128, 2), (8, 8, 64, 256, 2), (34, 2, 24, 16, 70)])
def test_attention_forward_and_gradient(lm, dtype, heads, kv, dim, block, width):
    gen = torch.Generator().manual_seed(heads * 1000 + dim + block)
    n = 83 if block < 128 else 300
    blocks = -(-n // block)
    if block >= 128:
        n, rows = 300, 37
    else:
        rows = n
    q, dout = rand(gen, rows, heads, dim, dtype=dtype), rand(gen, rows, heads, dim, dtype=dtype)
    k, v = rand(gen, n, kv, dim, dtype=dtype), rand(gen, n, kv, dim, dtype=dtype)
    idx = random_pattern(gen, rows, kv, width, blocks)
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.uniform(1, rows, n), None, block, None, True, dout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_sequences_and_wild_patterns(lm, dtype, causal):
    """Lengths of zero and one, fewer and more keys than queries, rows behind the last sequence, entries in any order, repeated and
    outside the sequence, rows that list nothing."""
    gen = torch.Generator().manual_seed(11)
    ql, kl = [1, 0, 33, 65, 7, 4], [1, 5, 33, 130, 0, 2]
    Tq, Tk = sum(ql) + 6, sum(kl) + 9
    H, G, D, B, W = 6, 3, 64, 16, 6
    q, dout = rand(gen, Tq, H, D, dtype=dtype), rand(gen, Tq, H, D, dtype=dtype)
    k, v = rand(gen, Tk, G, D, dtype=dtype), rand(gen, Tk, G, D, dtype=dtype)
    idx = random_pattern(gen, Tq, G, W, 9, wild=True)
    cu = lambda x: i32([sum(x[:i]) for i in range(len(x) + 1)]).to(DEV)
    seqs = lm.Seqs(len(ql), cu_q=cu(ql), cu_k=cu(kl))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.packed(ql, kl), seqs, B, 0.21, causal, dout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_padded_batch(lm, dtype):
    gen = torch.Generator().manual_seed(12)
    n, L, H, G, D, B, W = 4, 50, 4, 2, 64, 32, 3
    ql, kl = [50, 1, 0, 20], [50, 1, 7, 40]
    q, dout = rand(gen, n * L, H, D, dtype=dtype), rand(gen, n * L, H, D, dtype=dtype)
    k, v = rand(gen, n * L, G, D, dtype=dtype), rand(gen, n * L, G, D, dtype=dtype)
    for s in range(n):  # what stands in the padding is nobody's business
        q[s * L + ql[s]:(s + 1) * L] = math.nan
        dout[s * L + ql[s]:(s + 1) * L] = math.nan
        k[s * L + kl[s]:(s + 1) * L] = math.nan
        v[s * L + kl[s]:(s + 1) * L] = math.inf
    idx = random_pattern(gen, n * L, G, W, 2, wild=True)
    seqs = lm.Seqs(n, q_len=i32(ql).to(DEV), k_len=i32(kl).to(DEV))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.uniform(n, L, L, ql, kl), seqs, B, None, True, dout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_hidden_keys_may_hold_anything(lm, dtype):
    """NaN, infinities and the type's extremes in keys after the query and in blocks that no row lists."""
    gen = torch.Generator().manual_seed(13)
    n, H, G, D, B = 48, 4, 1, 64, 16
    q, k, v = rand(gen, n, H, D, dtype=dtype), rand(gen, n, G, D, dtype=dtype), rand(gen, n, G, D, dtype=dtype)
    k[16:32], v[16:32] = math.nan, -math.inf            # block 1 is listed by no row
    k[44:], v[44:] = torch.finfo(dtype).min, math.nan    # keys behind the last query asked about
    idx = i32([0, 2, -1]).expand(n, G, 3).contiguous()
    idx[16:32] = i32([0, -1, -1])
    rows = 44
    want = lo.attention(q[:rows], k[:rows], v[:rows], idx[:rows], lo.uniform(1, rows, rows), B, 0.125, True)
    out, lse = lm.block_attention(q.to(DEV), k.to(DEV), v.to(DEV), idx.to(DEV), block=B, scale=0.125, return_lse=True)
    every = torch.ones(rows, dtype=torch.bool)
    within(out[:rows], want["out"], want["tol_out"], every, "out")
    within(lse[:rows], want["lse"], want["tol_lse"], every, "lse")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_strided_tensors(lm, dtype):
    """q, k, v as slices of one fused projection, and heads before rows."""
    gen = torch.Generator().manual_seed(14)
    n, H, G, D, B, W = 70, 4, 2, 64, 16, 3
    fused = rand(gen, n, (H + 2 * G) * D, dtype=dtype).to(DEV)
    q = fused[:, :H * D].view(n, H, D)
    k = fused[:, H * D:(H + G) * D].view(n, G, D)
    v = rand(gen, G, n, D, dtype=dtype).to(DEV).transpose(0, 1)
    dout = rand(gen, n, H, D, dtype=dtype)
    idx = random_pattern(gen, n, G, W, 5)
    check_attention(lm, q, k, v, idx, lo.uniform(1, n, n), None, B, None, True, dout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads, kv, dim, block, page, width", [(8, 2, 128, 64, 64, 5), (4, 4, 64, 16, 48, 9), (16, 1, 96, 32, 32, 40),
                                                               (20, 1, 256, 16, 16, 4)])
def test_single_tokens_over_a_paged_cache(lm, dtype, heads, kv, dim, block, page, width):
    """Pages that end inside a block's tile, pages that are none, lengths zero and one, NaN behind the last key."""
    gen = torch.Generator().manual_seed(dim + page)
    lens = [1, 0, block, block + 1, 3 * page + 5, 150]
    per = -(-max(lens) // page)
    pages = len(lens) * per + 2
    deal = torch.randperm(pages, generator=gen)[:len(lens) * per].view(len(lens), per).tolist()
    k, v = rand(gen, pages, page, kv, dim, dtype=dtype), rand(gen, pages, page, kv, dim, dtype=dtype)
    for s, L in enumerate(lens):
        for j in range(L, per * page):
            k[deal[s][j // page], j % page] = math.nan
            v[deal[s][j // page], j % page] = math.nan
    deal[4][1] = -1
    deal[5][0] = pages
    q = rand(gen, len(lens), heads, dim, dtype=dtype)
    blocks = -(-max(lens) // block)
    idx = random_pattern(gen, len(lens), kv, width, blocks)
    idx[3, :, 0] = 0
    seqs = lm.Seqs(len(lens), k_len=i32(lens).to(DEV), page_table=i32(deal).to(DEV))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.paged(lens, deal, page, pages), seqs, block, None, True, None,
                    kv_flat=(k.view(-1, kv, dim), v.view(-1, kv, dim)))


def test_several_tokens_a_sequence_over_a_paged_cache(lm):
    """Three proposed tokens a sequence: positions are the last three."""
    gen = torch.Generator().manual_seed(17)
    lens, page, B, H, G, D = [2, 40, 95], 32, 16, 8, 2, 64
    k, v = rand(gen, 9, page, G, D, dtype=torch.bfloat16), rand(gen, 9, page, G, D, dtype=torch.bfloat16)
    deal = [[0, 3, 6], [1, 4, 7], [2, 5, 8]]
    q = rand(gen, 9, H, D, dtype=torch.bfloat16)
    idx = random_pattern(gen, 9, G, 4, 6)
    seqs = lm.Seqs(3, k_len=i32(lens).to(DEV), page_table=i32(deal).to(DEV))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.paged(lens, deal, page, 9, 3), seqs, B, None, True, None,
                    kv_flat=(k.view(-1, G, D), v.view(-1, G, D)))


def test_many_rows_take_the_form_without_split(lm):
    """Enough rows that a wavefront has a row to itself, against the form that splits rows: 3000 rows at once and row by row."""
    gen = torch.Generator().manual_seed(18)
    n, H, G, D, B, W = 3000, 4, 2, 64, 16, 4
    q, k, v = (rand(gen, n, h, D, dtype=torch.float32).to(DEV) for h in (H, G, G))
    idx = torch.sort(torch.randint(0, 188, (n, G, W), generator=gen, dtype=torch.int32), dim=2).values.to(DEV)
    out, lse = lm.block_attention(q, k, v, idx, block=B, return_lse=True)
    pick = [0, 1, 17, 1500, 2998, 2999]
    want = lo.attention(q.cpu()[pick], k.cpu(), v.cpu(), idx.cpu()[pick],
                        lo.Layout([(x, 1, list(range(t + 1))) for x, t in enumerate(pick)]), B, 0.125, True)
    every = torch.ones(len(pick), dtype=torch.bool)
    within(out[pick], want["out"], want["tol_out"], every, "out")
    within(lse[pick], want["lse"], want["tol_lse"], every, "lse")


def test_offsets_past_32_bits(lm):
    """A cache whose last pages begin behind 2^32 elements."""
    page, G, D, B = 4096, 8, 128, 64
    pages = 2 ** 32 // (page * G * D) + 2
    k = torch.zeros(pages, page, G, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    gen = torch.Generator().manual_seed(19)
    tail = rand(gen, page, G, D, dtype=torch.bfloat16), rand(gen, page, G, D, dtype=torch.bfloat16)
    k[-1], v[-1] = tail[0].to(DEV), tail[1].to(DEV)
    q = rand(gen, 1, 16, D, dtype=torch.bfloat16)
    lens, deal = [page], [[pages - 1]]
    idx = i32([0, 7, 63]).expand(1, G, 3).contiguous()
    seqs = lm.Seqs(1, k_len=i32(lens).to(DEV), page_table=i32(deal).to(DEV))
    check_attention(lm, q.to(DEV), k, v, idx, lo.paged(lens, [[0]], page, 1), seqs, B, None, True, None, kv_flat=tail)
    means = lm.block_means(k, block=B, seqs=seqs, last=B)
    assert torch.equal(means[-1].cpu(), tail[0][-B:].double().mean(0).to(torch.bfloat16))


# ---- gradient through autograd and against differences ----------------------------------------------------------------------------
def test_autograd_and_differences(lm):
    """The gradient that autograd returns, along a direction, against central differences of the 64-bit forward."""
    gen = torch.Generator().manual_seed(21)
    n, H, G, D, B, W = 40, 4, 2, 32, 16, 3
    host = [rand(gen, n, h, D) for h in (H, G, G)]
    idx = random_pattern(gen, n, G, W, 3)
    leaves = [x.to(DEV).requires_grad_() for x in host]
    dout = rand(gen, n, H, D)
    out = lm.block_attention(*leaves, idx.to(DEV), block=B)
    out.backward(dout.to(DEV))
    lay = lo.uniform(1, n, n)
    f = lambda x: (lo.attention(*x, idx, lay, B, 1 / math.sqrt(D), True)["out"] * dout.double()).sum()
    want = lo.attention(*host, idx, lay, B, 1 / math.sqrt(D), True, dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        step = rand(gen, *host[i].shape).double()
        h = 1e-5
        up, dn = [x.double() for x in host], [x.double() for x in host]
        up[i], dn[i] = up[i] + h * step, dn[i] - h * step
        diff = float((f(up) - f(dn)) / (2 * h))
        got = float((leaves[i].grad.cpu().double() * step).sum())
        # the kernel's bound summed along the direction, and the difference quotient's own 1e-6
        assert abs(diff - got) <= float((want["tol_" + name] * step.abs()).sum()) + 1e-6 * (1 + abs(diff)), name


def test_gradient_of_slices_and_expanded_heads(lm):
    """Leaves that reach the call as views: a fused projection, and one key head expanded to four."""
    gen = torch.Generator().manual_seed(22)
    n, D, B = 30, 32, 16
    fused = rand(gen, n, 8 * D).to(DEV).requires_grad_()
    one = rand(gen, n, 1, D).to(DEV).requires_grad_()
    idx = random_pattern(gen, n, 4, 2, 2).to(DEV)
    dout = rand(gen, n, 4, D).to(DEV)
    q, k = fused[:, :4 * D].view(n, 4, D), fused[:, 4 * D:].view(n, 4, D)
    lm.block_attention(q, k, one.expand(n, 4, D), idx, block=B).backward(dout)
    want = lo.attention(q.detach().cpu(), k.detach().cpu(), one.detach().cpu().expand(n, 4, D).contiguous(), idx.cpu(), lo.uniform(1, n, n), B,
                        1 / math.sqrt(D), True, dout.cpu())
    every = torch.ones(n, dtype=torch.bool)
    within(fused.grad[:, :4 * D].view(n, 4, D), want["dq"], want["tol_dq"], every, "dq")
    within(fused.grad[:, 4 * D:].view(n, 4, D), want["dk"], want["tol_dk"], every, "dk")
    # torch adds the four heads in 32 bits
    within(one.grad, want["dv"].sum(1, keepdim=True), want["tol_dv"].sum(1, keepdim=True) + 4 * lo.U32 * want["dv"].abs().sum(1, keepdim=True), every, "dv")


def test_gradients_do_not_depend_on_timing(lm):
    gen = torch.Generator().manual_seed(23)
    n, H, G, D, B = 500, 8, 2, 64, 16
    q, k, v, dout = (rand(gen, n, h, D, dtype=torch.bfloat16).to(DEV) for h in (H, G, G, H))
    idx = random_pattern(gen, n, G, 8, 32).to(DEV)
    out, lse = lm.block_attention(q, k, v, idx, block=B, return_lse=True)
    first = lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=B)
    for _ in range(3):
        again = lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=B)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- means and selection ------------------------------------------------------------------------------------------------------------
def check_means(got_row, want, dtype):
    # the sum in 64 bits, rounded once: half a step (and 2^-40 of it for the order of the 64-bit sum)
    d = (got_row.cpu().double() - want).abs()
    assert (d <= lo.u(dtype) * want.abs() * (1 + 2.0 ** -40) + torch.finfo(dtype).smallest_normal * lo.u(dtype) * 2).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim, block, heads, kv", [(64, 16, 4, 2), (128, 64, 8, 1), (200, 32, 3, 3), (8, 256, 2, 1)])
def test_selection_packed(lm, dtype, dim, block, heads, kv):
    gen = torch.Generator().manual_seed(dim + block)
    lens = [1, 0, block, 5 * block + 3, 9 * block]
    n = sum(lens)
    q = rand(gen, n + 2, heads, dim, dtype=dtype)
    k = rand(gen, n + 2, kv, dim, dtype=dtype)
    cu = i32([sum(lens[:i]) for i in range(len(lens) + 1)]).to(DEV)
    seqs = lm.Seqs(len(lens), cu_q=cu, cu_k=cu)
    lay = lo.packed(lens, lens)
    means = lm.block_means(k.to(DEV), block=block, seqs=seqs)
    held = {}
    for (s, b), want in lo.block_mean_rows(k, lay, block).items():
        row = sum(lens[:s]) // block + s + b
        check_means(means[row], want, dtype)
        held[s, b] = means[row].cpu()
    for width, first, local in ((3, 1, 1), (4, 0, 2), (2, 1, 1), (6, 2, 3), (16, 1, 1)):
        out = torch.full((n + 2, kv, width), -7, dtype=torch.int32, device=DEV)
        lm.select_blocks(q.to(DEV), means, block=block, width=width, first=first, local=local, k_rows=n + 2, seqs=seqs, out=out)
        assert torch.equal(out[:n].cpu(), lo.select(q[:n], held, lay, block, width, first, local, True)), (width, first, local)
        assert (out[n:] == -7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_selection_ties_and_values_that_are_no_numbers(lm, dtype):
    """Equal scores go to the lowest index; NaN is lowest; infinities order as numbers."""
    gen = torch.Generator().manual_seed(31)
    n, H, G, D, B = 20 * 16, 4, 2, 64, 16
    q = rand(gen, n, H, D, dtype=dtype)
    means = rand(gen, 20, G, D, dtype=dtype)
    means[5] = means[3]
    means[11] = means[3]
    means[7, 0, 3] = math.nan
    means[9, 1, 2] = math.inf
    means[13, 1, 2] = -math.inf
    q[100:140] = 0
    q[200, 0, 5] = math.nan
    q[201, 1, 5] = math.inf
    held = {(0, b): means[b] for b in range(20)}
    for causal in (True, False):
        for width in (4, 7):
            local = 1 if causal else 0
            got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=width, first=1, local=local, causal=causal, k_rows=n)
            assert torch.equal(got.cpu(), lo.select(q, held, lo.uniform(1, n, n), B, width, 1, local, causal))


def test_selection_of_scores_next_to_each_other(lm):
    """Means that differ in their last bits: the order must be that of the 64-bit scores."""
    gen = torch.Generator().manual_seed(32)
    B, nb, D = 16, 64, 128
    q = rand(gen, 40, 2, D)
    base = rand(gen, 1, 1, D)
    means = base * (1 + torch.randint(-3, 4, (nb, 1, D), generator=gen) * 2.0 ** -23)
    means = means.float().contiguous()
    seqs = lm.Seqs(1, q_len=i32([40]).to(DEV), k_len=i32([nb * B]).to(DEV))
    got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=9, first=0, local=0, causal=False, k_rows=nb * B, seqs=seqs)
    want = lo.select(q, {(0, b): means[b] for b in range(nb)}, lo.uniform(1, 40, nb * B), B, 9, 0, 0, False)
    assert torch.equal(got.cpu(), want)


def test_selection_over_very_many_blocks(lm):
    gen = torch.Generator().manual_seed(33)
    nb, B, D = 9001, 16, 64
    q = rand(gen, 3, 2, D)
    means = rand(gen, nb, 1, D)
    seqs = lm.Seqs(1)
    for width, first in ((64, 3), (256, 0)):
        got = lm.select_blocks(q.to(DEV), means.to(DEV), block=B, width=width, first=first, local=2, k_rows=nb * B, seqs=seqs)
        score = q.double().sum(1) @ means[:, 0].double().t()
        lay = lo.uniform(1, 3, nb * B)
        want = lo.select(q, {(0, b): means[b] for b in range(nb)}, lay, B, width, first, 2, True)
        assert torch.equal(got.cpu(), want) and score.shape == (3, nb)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_serving_step_over_a_paged_cache(lm, dtype):
    """Append a token, refresh the newest block's mean, select, attend: each against its plain form, several steps in a row."""
    gen = torch.Generator().manual_seed(34)
    H, G, D, B, page, W = 8, 2, 64, 16, 32, 4
    lens = [1, 15, 16, 100, 190]
    per, n = 7, 5
    pages = n * per
    deal = torch.randperm(pages, generator=gen).view(n, per)
    k = torch.full((pages, page, G, D), math.nan, dtype=dtype)
    v = torch.full_like(k, math.nan)
    for s in range(n):
        for j in range(lens[s]):
            k[deal[s, j // page], j % page] = rand(gen, G, D, dtype=dtype)
            v[deal[s, j // page], j % page] = rand(gen, G, D, dtype=dtype)
    kd, vd, table = k.to(DEV), v.to(DEV), deal.int().to(DEV)
    seqs = lm.Seqs(n, k_len=i32(lens).to(DEV), page_table=table)
    means = lm.block_means(kd, block=B, seqs=seqs)
    for step in range(4):
        q = rand(gen, n, H, D, dtype=dtype)
        for s in range(n):
            j = lens[s]
            lens[s] += 1
            k[deal[s, j // page], j % page], v[deal[s, j // page], j % page] = rand(gen, G, D, dtype=dtype), rand(gen, G, D, dtype=dtype)
        kd.copy_(k)
        vd.copy_(v)
        seqs.k_len.copy_(i32(lens))
        lm.block_means(kd, block=B, seqs=seqs, last=1, out=means)
        lay = lo.paged(lens, deal.tolist(), page, pages)
        held = {}
        for (s, b), want in lo.block_mean_rows(k.view(-1, G, D), lay, B).items():
            row = int(deal[s, b * B // page]) * (page // B) + b * B % page // B
            check_means(means[row], want, dtype)
            held[s, b] = means[row].cpu()
        idx = lm.select_blocks(q.to(DEV), means, block=B, width=W, first=1, local=2, k_rows=pages, seqs=seqs)
        assert torch.equal(idx.cpu(), lo.select(q, held, lay, B, W, 1, 2, True))
        check_attention(lm, q.to(DEV), kd, vd, idx.cpu(), lay, seqs, B, None, True, None, kv_flat=(k.view(-1, G, D), v.view(-1, G, D)))


def test_training_step_end_to_end(lm):
    """Means, selection, attention and its gradient as a layer runs them."""
    gen = torch.Generator().manual_seed(35)
    n, H, G, D, B, W = 130, 4, 2, 64, 16, 4
    q, k, v = (rand(gen, n, h, D, dtype=torch.bfloat16) for h in (H, G, G))
    dout = rand(gen, n, H, D, dtype=torch.bfloat16)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    means = lm.block_means(leaves[1].detach(), block=B)
    idx = lm.select_blocks(leaves[0].detach(), means, block=B, width=W, k_rows=n)
    lay = lo.uniform(1, n, n)
    assert torch.equal(idx.cpu(), lo.select(q, {(0, b): means[b].cpu() for b in range(9)}, lay, B, W, 1, 1, True))
    lm.block_attention(*leaves, idx, block=B).backward(dout.to(DEV))
    want = lo.attention(q, k, v, idx.cpu(), lay, B, 1 / math.sqrt(D), True, dout)
    every = torch.ones(n, dtype=torch.bool)
    for name, x in zip(("dq", "dk", "dv"), leaves):
        within(x.grad, want[name], want["tol_" + name], every, name)


# ---- routing ------------------------------------------------------------------------------------------------------------------------
def check_routing(lm, ids, experts, channels, dtype, gen):
    T, K = ids.shape
    offsets, order, place = lo.route(ids, experts)
    plan = lm.route(ids.to(DEV), experts)
    live = len(order)
    assert plan.offsets.cpu().tolist() == offsets
    assert torch.equal(plan.place.cpu(), place)
    assert plan.order[:live].cpu().tolist() == order
    x, y = rand(gen, T, channels, dtype=dtype), rand(gen, T * K, channels, dtype=dtype)
    w, dout, dxs = torch.rand(T, K, generator=gen), rand(gen, T, channels, dtype=dtype), rand(gen, T * K, channels, dtype=dtype)
    y[live:] = math.nan
    dxs[live:] = math.nan
    w[place < 0] = math.nan  # weights of dropped entries are not read
    xs = lm.gather_tokens(x.to(DEV), plan)
    tok = torch.tensor(order, dtype=torch.int64) // K if live else torch.zeros(0, dtype=torch.int64)
    assert torch.equal(xs[:live].cpu(), x[tok])
    ww = torch.nan_to_num(w.double()).reshape(-1)[order] if live else torch.zeros(0, dtype=torch.float64)
    zero = lambda: torch.zeros(T, channels, dtype=torch.float64)
    every = torch.ones(T, dtype=torch.bool)
    ut = lo.u(dtype)
    terms = ww[:, None] * y[:live].double()
    want, size = zero().index_add_(0, tok, terms), zero().index_add_(0, tok, terms.abs())
    within(lm.combine_tokens(y.to(DEV), plan, w.to(DEV)), want, 1.01 * ut * want.abs() + 2 * K * lo.U32 * size + 1e-30, every, "out")
    dx = lm.gather_tokens_backward(dxs.to(DEV), plan)
    want, size = zero().index_add_(0, tok, dxs[:live].double()), zero().index_add_(0, tok, dxs[:live].double().abs())
    within(dx, want, 1.01 * ut * want.abs() + K * lo.U32 * size + 1e-30, every, "dx")
    dy, dw = lm.combine_tokens_backward(dout.to(DEV), y.to(DEV), plan, w.to(DEV))
    want = ww[:, None] * dout.double()[tok]
    within(dy[:live], want, (ut + lo.U32) * 1.01 * want.abs() + 1e-12 * (dtype == torch.float16) + 1e-30 + torch.finfo(dtype).smallest_normal * ut * 2,
           torch.ones(live, dtype=torch.bool), "dy")
    prod = dout.double()[tok] * y[:live].double()
    want_w, size_w = torch.zeros(T * K, dtype=torch.float64), torch.zeros(T * K, dtype=torch.float64)
    want_w[order], size_w[order] = prod.sum(1), prod.abs().sum(1)
    # a lane adds channels / 64 products or more one after the other: every product and addition rounds once
    within(dw.reshape(-1), want_w, (channels / 64 + 16) * 2 * lo.U32 * size_w + 1e-30, torch.ones(T * K, dtype=torch.bool), "dw")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens, top, experts, channels", [(1, 1, 1, 1), (7, 2, 5, 64), (64, 8, 64, 1000), (100, 3, 24, 1023), (33, 4, 256, 4096),
                                                           (513, 8, 7, 24), (1100, 4, 16, 8)])
def test_routing(lm, dtype, tokens, top, experts, channels):
    gen = torch.Generator().manual_seed(tokens + channels)
    check_routing(lm, torch.randint(-1, experts + 1, (tokens, top), generator=gen, dtype=torch.int32), experts, channels, dtype, gen)


@pytest.mark.parametrize("experts", [1, 3, 1000, 1025, 2049, 4096])
def test_routing_of_many_entries(lm, experts):
    """Several chunks, every size class of the counters; the same expert several times in a token; all tokens at one expert."""
    gen = torch.Generator().manual_seed(experts)
    ids = torch.randint(0, experts, (3001, 5), generator=gen, dtype=torch.int32)
    check_routing(lm, ids, experts, 8, torch.float32, gen)
    check_routing(lm, torch.full((2500, 4), experts - 1, dtype=torch.int32), experts, 8, torch.float32, gen)
    check_routing(lm, torch.full((2500, 4), -1, dtype=torch.int32), experts, 8, torch.float32, gen)


def test_routing_of_nothing(lm):
    plan = lm.route(torch.zeros(0, 4, dtype=torch.int32, device=DEV), 6)
    assert plan.offsets.cpu().tolist() == [0] * 7 and plan.place.shape == (0, 4)
    assert lm.gather_tokens(torch.zeros(0, 16, device=DEV), plan).shape == (0, 16)
    assert lm.combine_tokens(torch.zeros(0, 16, device=DEV), plan, torch.zeros(0, 4, device=DEV)).shape == (0, 16)


def test_routing_through_autograd(lm):
    """A layer of experts (one scale each): gradients of tokens and weights against torch on the same graph in 64 bits."""
    gen = torch.Generator().manual_seed(41)
    T, K, E, C = 50, 3, 6, 40
    ids = torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32)
    ids[::7, 1] = -1
    x0, w0, s = rand(gen, T, C), torch.rand(T, K, generator=gen), rand(gen, E)
    dout = rand(gen, T, C)
    x, w = x0.to(DEV).requires_grad_(), w0.to(DEV).requires_grad_()
    plan = lm.route(ids.to(DEV), E)
    live = int(plan.offsets[-1])
    expert = torch.searchsorted(plan.offsets[1:].contiguous(), torch.arange(T * K, device=DEV, dtype=torch.int32), right=True).clamp(max=E - 1)
    row_scale = s.to(DEV)[expert] * (torch.arange(T * K, device=DEV) < live)
    xs = lm.gather_tokens(x, plan)
    xs = torch.where((torch.arange(T * K, device=DEV) < live)[:, None], xs, torch.zeros((), device=DEV))
    lm.combine_tokens(xs * row_scale[:, None], plan, w).backward(dout.to(DEV))
    x64, w64 = x0.double().requires_grad_(), w0.double().requires_grad_()
    keep = (ids >= 0).double()
    fac = (w64 * keep * s.double()[ids.clamp(min=0).long()]).sum(1)
    (fac[:, None] * x64).backward(dout.double())
    # every value passes at most 8 roundings in 32 bits, sums have K or C terms
    size = (w0.double() * keep * s.double()[ids.clamp(min=0).long()].abs()).sum(1)[:, None] * dout.double().abs()
    within(x.grad, x64.grad, 16 * lo.U32 * size + 1e-30, torch.ones(T, dtype=torch.bool), "dx")
    size = (dout.double() * x0.double()).abs().sum(1)[:, None] * s.double()[ids.clamp(min=0).long()].abs()
    within(w.grad, w64.grad, 64 * lo.U32 * size + 1e-30, torch.ones(T, dtype=torch.bool), "dw")


# ---- streams, graphs, refusals ----------------------------------------------------------------------------------------------------------
def test_on_another_stream(lm):
    gen = torch.Generator().manual_seed(51)
    q, k, v = (rand(gen, 64, h, 64, dtype=torch.bfloat16).to(DEV) for h in (4, 2, 2))
    idx = random_pattern(gen, 64, 2, 3, 4).to(DEV)
    want = lm.block_attention(q, k, v, idx, block=16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = lm.block_attention(q, k, v, idx, block=16)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def test_two_captured_graphs(lm):
    """Two graphs of the whole step, replayed in turn with new inputs and eager work between: every replay equals the eager call."""
    gen = torch.Generator().manual_seed(52)
    H, G, D, B, W, K, E = 4, 2, 64, 16, 3, 2, 8

    def step(q, k, v, dout, ids, w):
        means = lm.block_means(k, block=B)
        idx = lm.select_blocks(q, means, block=B, width=W, k_rows=k.shape[0])
        out, lse = lm.block_attention(q, k, v, idx, block=B, return_lse=True)
        grads = lm.block_attention_backward(dout, q, k, v, idx, out, lse, block=B)
        plan = lm.route(ids, E)
        xs = lm.gather_tokens(out.view(q.shape[0], -1), plan)
        y = lm.combine_tokens(xs, plan, w)
        dy, dw = lm.combine_tokens_backward(y, xs, plan, w)
        return (means, idx, out, lse, *grads, plan.offsets, plan.place, xs, y, dy, dw, lm.gather_tokens_backward(dy, plan))

    def inputs(n):
        return [rand(gen, n, H, D, dtype=torch.bfloat16), rand(gen, n, G, D, dtype=torch.bfloat16), rand(gen, n, G, D, dtype=torch.bfloat16),
                rand(gen, n, H, D, dtype=torch.bfloat16), torch.randint(0, E, (n, K), generator=gen, dtype=torch.int32), torch.rand(n, K, generator=gen)]

    held, graphs, outs = [], [], []
    for n in (100, 2100):
        x = [t.to(DEV) for t in inputs(n)]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(*x)
        torch.cuda.current_stream().wait_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(*x)
        held.append(x)
        graphs.append(g)
        outs.append(y)
    for turn in range(3):
        for x in held:
            for a, b in zip(x, inputs(x[0].shape[0])):
                a.copy_(b)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, outs):
            for a, b in zip(step(*x), y):
                assert torch.equal(a, b)


def test_refusals_on_the_gpu(lm):
    q = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device=DEV)
    idx = torch.zeros(8, 2, 2, dtype=torch.int32, device=DEV)
    ok = dict(block=16)
    for args in ((q, k, k.float(), idx), (q, k, k[:4], idx), (q.float(), k, k, idx), (q, k, k, idx.long()), (q, k, k, idx[:4]),
                 (q, k, k, idx[:, :1]), (q, k[..., :32], k[..., :32], idx), (q[:, :3], k, k, idx), (q.transpose(1, 2), k, k, idx),
                 (q.double(), k.double(), k.double(), idx), (q, k.cpu(), k, idx)):
        with pytest.raises(ValueError):
            lm.block_attention(*args, **ok)
    with pytest.raises(ValueError):
        lm.block_attention(q, k, k, idx, block=24)
    with pytest.raises(ValueError):
        lm.block_attention(q.requires_grad_(), k, k, idx, block=16, out=torch.empty_like(q))
    odd = torch.zeros(8 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(8, 4, 64)
    with pytest.raises(ValueError):
        lm.block_attention(odd, k, k, idx, **ok)
    with pytest.raises(ValueError):
        lm.select_blocks(q.detach(), torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV), block=16, width=2, k_rows=8)
    plan = lm.route(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 3)
    for bad in (torch.zeros(3, 8, device=DEV), torch.zeros(4, 8, device=DEV, dtype=torch.float64), torch.zeros(8, 4, device=DEV).t()):
        with pytest.raises(ValueError):
            lm.gather_tokens(bad, plan)
    with pytest.raises(ValueError):
        lm.combine_tokens(torch.zeros(8, 8, device=DEV), plan, torch.zeros(4, 2, device=DEV, dtype=torch.bfloat16))
