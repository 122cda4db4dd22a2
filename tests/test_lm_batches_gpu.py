"""Batches whose totals are large while their sequences are not, calls that mix prompts and single tokens, blocks that very many rows list."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")
import lm_oracle as lo  # noqa: E402
from test_lm_gpu import DEV, check_attention, i32, lm, rand, random_pattern, within  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def cu(lens):
    return i32([sum(lens[:i]) for i in range(len(lens) + 1)]).to(DEV)


@pytest.mark.parametrize("rows, dtype", [(4000, torch.bfloat16), (6000, torch.bfloat16), (4000, torch.float32)], ids=str)
def test_gradient_of_a_block_that_more_rows_list_than_are_walked_at_once(lm, rows, dtype):
    """Width 256 and these rows share a block out to items of 1024 and 2048 rows (by the pattern's size, not by its live entries), which do
    not begin at whole words of 64 and take the list in LDS more than once."""
    gen = torch.Generator().manual_seed(rows)
    D, B, W = 16, 16, 256
    q, k, v, dout = (rand(gen, rows, 1, D, dtype=dtype) for _ in range(4))
    idx = torch.full((rows, 1, W), -1, dtype=torch.int32)
    idx[:, 0, 0] = 0
    idx[::3, 0, 1] = torch.arange(rows, dtype=torch.int32)[::3] // B  # and some their own
    idx[:, 0, 1][idx[:, 0, 1] == 0] = -1
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lo.uniform(1, rows, rows), None, B, None, True, dout)


@pytest.mark.parametrize("n, each, block", [(130, 260, 16), (2300, 241, 16)])
def test_selection_of_many_short_sequences(lm, n, each, block):
    """More than 2048 and more than 32768 blocks in all, a few in each sequence."""
    gen = torch.Generator().manual_seed(n)
    H, G, D, W = 2, 1, 16, 4
    lens = [each - (s % 7) for s in range(n)]
    q_lens = [min(8, x) for x in lens]  # the last rows of each
    Tk = sum(lens)
    k = rand(gen, Tk, G, D, dtype=torch.bfloat16).to(DEV)
    q = rand(gen, sum(q_lens), H, D, dtype=torch.bfloat16)
    seqs = lm.Seqs(n, cu_q=cu(q_lens), cu_k=cu(lens))
    assert Tk // block > (32768 if n > 2000 else 2048)
    means = lm.block_means(k, block=block, seqs=seqs)
    got = lm.select_blocks(q.to(DEV), means, block=block, width=W, k_rows=Tk, first=1, local=1, seqs=seqs).cpu()
    held, starts = means.cpu(), torch.tensor([0] + lens).cumsum(0).tolist()
    for s in (0, 1, 5, n // 2, n - 2, n - 1):
        base = starts[s] // block + s
        rows = {(0, b): held[base + b] for b in range(-(-lens[s] // block))}
        a = sum(q_lens[:s])
        want = lo.select(q[a:a + q_lens[s]], rows, lo.Layout([(0, q_lens[s], list(range(lens[s])))]), block, W, 1, 1, True)
        assert torch.equal(got[a:a + q_lens[s]], want), s


@pytest.mark.parametrize("singles", [3, 40, 1100])
def test_a_prompt_and_single_tokens_in_one_call(lm, singles):
    """A piece of a prompt among conversations' next tokens: fewer than four rows a sequence on average, and more."""
    gen = torch.Generator().manual_seed(singles)
    H, G, D, B, W = 4, 2, 64, 16, 5
    ql = [1] * (singles // 2) + [150] + [1] * (singles - singles // 2)
    kl = [int(x) for x in torch.randint(1, 90, (len(ql),), generator=gen)]
    kl[singles // 2] = 260
    q, dout = (rand(gen, sum(ql), H, D, dtype=torch.bfloat16) for _ in range(2))
    k, v = (rand(gen, sum(kl), G, D, dtype=torch.bfloat16) for _ in range(2))
    seqs, lay = lm.Seqs(len(ql), cu_q=cu(ql), cu_k=cu(kl)), lo.packed(ql, kl)
    means = lm.block_means(k.to(DEV), block=B, seqs=seqs)
    idx = lm.select_blocks(q.to(DEV), means, block=B, width=W, k_rows=k.shape[0], seqs=seqs).cpu()
    held, starts = means.cpu(), torch.tensor([0] + kl).cumsum(0).tolist()
    rows = {(s, b): held[starts[s] // B + s + b] for s in range(len(kl)) for b in range(-(-kl[s] // B))}
    assert torch.equal(idx, lo.select(q, rows, lay, B, W, 1, 1, True))
    check_attention(lm, q.to(DEV), k.to(DEV), v.to(DEV), idx, lay, seqs, B, None, True, dout)


def test_calls_of_several_threads(lm):
    """Four threads, each on its own stream, through every operator and its gradient: as one thread by itself."""
    gen = torch.Generator().manual_seed(99)
    n, H, G, D, B, W, T, K, E, Ch = 700, 4, 2, 64, 16, 4, 300, 2, 8, 40
    work = []
    for _ in range(4):
        q, k, v = (rand(gen, n, h, D, dtype=torch.bfloat16).to(DEV).requires_grad_() for h in (H, G, G))
        x, w = rand(gen, T, Ch).to(DEV).requires_grad_(), torch.rand(T, K, generator=gen).to(DEV).requires_grad_()
        work.append((q, k, v, x, w, torch.randint(-1, E, (T, K), generator=gen, dtype=torch.int32).to(DEV)))

    def run(q, k, v, x, w, ids):
        with torch.no_grad():
            idx = lm.select_blocks(q, lm.block_means(k, block=B), block=B, width=W, k_rows=n)
        out, lse = lm.block_attention(q, k, v, idx, block=B, return_lse=True)
        plan = lm.route(ids, E)
        y = lm.combine_tokens(lm.gather_tokens(x, plan), plan, w)
        return (idx, out, lse, y, *torch.autograd.grad((out.float().sum() + lse.sum() + (y * y).sum()), (q, k, v, x, w)))

    want = [run(*a) for a in work]
    torch.cuda.synchronize()
    got, errors = [[] for _ in work], []

    def thread(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[i].append(run(*work[i]))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    for mine, ref in zip(got, want):
        assert all(torch.equal(a, b) for res in mine for a, b in zip(res, ref))
