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


def bounds_with_lse(q, k, v, idx, layout, B, scale, dout, dlse):
    """dq, dk, dv in 64 bits with a gradient dlse of the log-sum-exp beside dout, and bounds.

    ds = p (dp - delta + dlse): the part with dlse is scale p dlse k (or q), and the kernel computes p (dp - delta') with
    delta' = delta - dlse in 32 bits.  Beside lm_oracle's bounds for dout: p is off by rel_p of itself (its part of the oracle's bound for dv),
    the difference, the product with p and the scale by 6 steps of 32 bits of |dlse| (and of delta, which the oracle counts), their rounding
    to the type by 1.01 u, and the sums over keys (dq) and rows (dk) by a step a term.
    """
    T = q.dtype
    want = lo.attention(q, k, v, idx, layout, B, scale, True, dout)
    Q, K = q.double(), k.double()
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    add = {n: torch.zeros_like(want[n]) for n in ("dq", "dk")}
    tol = {n: torch.zeros_like(want[n]) for n in ("dq", "dk")}
    count = torch.zeros(k.shape[0], G, 1, dtype=torch.float64)
    ut, ta = lo.u(T), lo.tiny(T)
    for first, rows_q, rows_k in layout.seqs:
        for i in range(rows_q):
            t, L = first + i, len(rows_k)
            limit = min(L, L - rows_q + i + 1)
            for g in range(G):
                keys = [] if limit <= 0 else [rows_k[j] for b in lo.listed(idx[t, g].tolist(), limit, B) for j in range(b * B, min(b * B + B, limit))]
                if not keys:
                    continue
                hs = slice(g * (H // G), (g + 1) * (H // G))
                s = scale * Q[t, hs] @ K[keys, g].t()
                p = torch.softmax(s, 1)
                ds = (D + 4) * lo.U32 * abs(scale) * (Q[t, hs].abs() @ K[keys, g].abs().t()).max() + 2 * lo.U32 * (s.abs().max() + 1)
                rel_p = 2 * ds + 2.0 ** -21 + (len(keys) + 64) * lo.U32 + want["tol_lse"][t, hs].max()
                d = p * dlse[t, hs].double()[:, None]
                off = abs(scale) * d.abs() * (1.01 * ut + rel_p + 6 * lo.U32) * 1.02 + ta
                add["dq"][t, hs] += scale * d @ K[keys, g]
                add["dk"][keys, g] += scale * d.t() @ Q[t, hs]
                tol["dq"][t, hs] += (off + len(keys) * lo.U32 * abs(scale) * d.abs()) @ K[keys, g].abs()
                tol["dk"][keys, g] += (off + (layout_rows(layout) * H // G) * lo.U32 * abs(scale) * d.abs()).t() @ Q[t, hs].abs()
                count[keys, g] += 1
    for n in ("dq", "dk"):
        want["tol_" + n] = want["tol_" + n] + tol[n] + 1.01 * ut * add[n].abs()
        want[n] = want[n] + add[n]
    return want


def layout_rows(layout):
    return sum(n for _, n, _ in layout.seqs)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n, H, G, D, B, W", [(83, 8, 2, 64, 16, 4), (70, 6, 2, 96, 16, 3), (300, 4, 1, 128, 64, 2), (600, 2, 2, 64, 32, 12)])
def test_gradient_through_the_log_sum_exp(lm, dtype, n, H, G, D, B, W):
    """Few keys in a walk and many (delta is found in two ways), rows without a key whose gradient is no number."""
    gen = torch.Generator().manual_seed(n + D)
    q, k, v = (rand(gen, n, h, D, dtype=dtype) for h in (H, G, G))
    dout, dlse = rand(gen, n, H, D, dtype=dtype), 3 * rand(gen, n, H)
    idx = random_pattern(gen, n, G, W, -(-n // B))
    idx[5] = -1
    want = bounds_with_lse(q, k, v, idx, lo.uniform(1, n, n), B, 1 / math.sqrt(D), dout, dlse)
    dlse[5] = math.nan  # what a logarithm of nothing gives back
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    out, lse = lm.block_attention(*leaves, idx.to(DEV), block=B, return_lse=True)
    got = torch.autograd.grad((out, lse), leaves, (dout.to(DEV), dlse.to(DEV)))
    every = torch.ones(n, dtype=torch.bool)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x, want[name], want["tol_" + name], every, name)


def test_only_the_log_sum_exp_has_a_gradient(lm):
    """Against central differences of the 64-bit form along a direction; v has no part in it."""
    gen = torch.Generator().manual_seed(84)
    n, H, G, D, B, W = 40, 4, 2, 32, 16, 3
    host = [rand(gen, n, h, D) for h in (H, G, G)]
    idx, dlse = random_pattern(gen, n, G, W, 3), rand(gen, n, H)
    idx[:, :, 0] = 0  # every row has a key
    lay = lo.uniform(1, n, n)
    leaves = [x.to(DEV).requires_grad_() for x in host]
    _, lse = lm.block_attention(*leaves, idx.to(DEV), block=B, return_lse=True)
    (lse * dlse.to(DEV)).sum().backward()
    assert (leaves[2].grad == 0).all()
    want = bounds_with_lse(*host, idx, lay, B, 1 / math.sqrt(D), torch.zeros(n, H, D), dlse)
    f = lambda x: (lo.attention(*x, idx, lay, B, 1 / math.sqrt(D), True)["lse"] * dlse.double()).sum()
    for i, name in enumerate(("dq", "dk")):
        step, h = rand(gen, *host[i].shape).double(), 1e-5
        up, dn = [x.double() for x in host], [x.double() for x in host]
        up[i], dn[i] = up[i] + h * step, dn[i] - h * step
        diff = float((f(up) - f(dn)) / (2 * h))
        got = float((leaves[i].grad.cpu().double() * step).sum())
        assert abs(diff - got) <= float((want["tol_" + name] * step.abs()).sum()) + 1e-6 * (1 + abs(diff)), name


def spread(q, k, v, idx, B, scale, off_dout, off_dlse, out):
    """What gradients of one causal sequence are off by, at most, if dout and dlse are off by so much: the formulas with absolute values."""
    Q, K, V = q.double(), k.double(), v.double()
    n, H, D = Q.shape
    G = K.shape[1]
    r = [torch.zeros_like(x) for x in (Q, K, V)]
    for t in range(n):
        for g in range(G):
            keys = [j for b in lo.listed(idx[t, g].tolist(), t + 1, B) for j in range(b * B, min(b * B + B, t + 1))]
            if not keys:
                continue
            hs = slice(g * (H // G), (g + 1) * (H // G))
            p = torch.softmax(scale * Q[t, hs] @ K[keys, g].t(), 1)
            off = p * (off_dout[t, hs] @ V[keys, g].abs().t() + (off_dout[t, hs] * out[t, hs].abs()).sum(1, keepdim=True) + off_dlse[t, hs][:, None])
            r[0][t, hs] += scale * off @ K[keys, g].abs()
            r[1][keys, g] += scale * off.t() @ Q[t, hs].abs()
            r[2][keys, g] += p.t() @ off_dout[t, hs]
    return r


def test_two_halves_joined_by_their_log_sum_exp(lm):
    """Attention over two sets of blocks, joined by torch in 64 bits: output and gradients as of one call over both."""
    gen = torch.Generator().manual_seed(85)
    n, H, G, D, B = 96, 4, 2, 64, 16
    host = [rand(gen, n, h, D) for h in (H, G, G)]
    dout = rand(gen, n, H, D)
    scale, lay = 1 / math.sqrt(D), lo.uniform(1, n, n)
    blocks = torch.arange(6, dtype=torch.int32).expand(n, G, 6).contiguous()
    halves = [blocks[:, :, i::2].contiguous() for i in (0, 1)]
    leaves = [x.to(DEV).requires_grad_() for x in host]
    parts = [lm.block_attention(*leaves, x.to(DEV), block=B, return_lse=True) for x in halves]
    # the first half sees a key in every row; where the second sees none its weight is 0
    live = torch.arange(n, device=DEV)[:, None] >= B
    a, b = parts[0][1].double(), torch.where(live, parts[1][1].double(), 0.0)
    w1 = torch.where(live, torch.sigmoid(b - a), 0.0)
    out = (1 - w1)[:, :, None] * parts[0][0].double() + w1[:, :, None] * parts[1][0].double()
    got = torch.autograd.grad(out, leaves, dout.to(DEV).double())

    whole = lo.attention(*host, blocks, lay, B, scale, True, dout)
    ref = [lo.attention(*host, x, lay, B, scale, True) for x in halves]
    tol_out, tol = torch.zeros(n, H, D, dtype=torch.float64), [torch.zeros_like(x.double()) for x in host]
    # a weight is off by at most its share of what the two log-sum-exps are off by
    off_lse = ref[0]["tol_lse"] + torch.where(live.cpu(), ref[1]["tol_lse"], 0.0)
    weight = [torch.exp(r["lse"] - whole["lse"]) for r in ref]
    for w, r in zip(weight, ref):
        tol_out += 1.01 * (w[:, :, None] * r["tol_out"] + (w * off_lse)[:, :, None] * r["out"].abs())
    for w, r, x in zip(weight, ref, halves):
        do = w[:, :, None] * dout.double()
        dl = w * (dout.double() * (r["out"] - whole["out"])).sum(2)
        mine = bounds_with_lse(*host, x, lay, B, scale, do.float(), dl.float())
        # they come back in 32 bits: one rounding each, beside what weights and outputs are off by
        off_do = do.abs() * (lo.U32 + off_lse[:, :, None]) * 1.01
        off_dl = (dl.abs() * (lo.U32 + off_lse) + w * (dout.double().abs() * (r["tol_out"] + tol_out)).sum(2)) * 1.01
        for i, (name, s) in enumerate(zip(("dq", "dk", "dv"), spread(*host, x, B, scale, off_do, off_dl, r["out"]))):
            # the two halves' gradients are added in 32 bits; the oracle's own do and dl above were rounded once too
            tol[i] += 1.01 * (mine["tol_" + name] + 2 * s + lo.U32 * mine[name].abs())
    every = torch.ones(n, dtype=torch.bool)
    within(out, whole["out"], tol_out, every, "out")
    for i, name in enumerate(("dq", "dk", "dv")):
        within(got[i], whole[name], tol[i], every, name)


@pytest.mark.parametrize("op", ["gather", "combine"])
def test_a_plan_written_again_before_backward(lm, op):
    gen = torch.Generator().manual_seed(86)
    T, K, E, Ch = 12, 2, 4, 8
    plan = lm.route(torch.randint(0, E, (T, K), generator=gen, dtype=torch.int32).to(DEV), E)
    x, w = rand(gen, T * K if op == "combine" else T, Ch).to(DEV).requires_grad_(), torch.rand(T, K, generator=gen).to(DEV)
    out = lm.gather_tokens(x, plan) if op == "gather" else lm.combine_tokens(x, plan, w)
    plan.place.fill_(-1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.sum().backward()


def test_buffers_written_again_before_backward(lm):
    """A pattern, a tensor of keys and an output that a later call writes into: the graph that saved them refuses."""
    leaves, idx, dout, B = small(87, torch.bfloat16)
    q, k, v = (x.detach() for x in leaves)
    n = k.shape[0]
    means = lm.block_means(k, block=B)
    base = means.clone()  # means as keys of a second, coarser attention
    few = torch.zeros(n, k.shape[1], 1, dtype=torch.int32, device=DEV)
    writes = [(lambda: lm.select_blocks(q, means, block=B, width=idx.shape[2], k_rows=n, out=idx), lambda: lm.block_attention(*leaves, idx, block=B)),
              (lambda: lm.block_means(k, block=B, out=base), lambda: lm.block_attention(leaves[0], base, base, few, block=16, causal=False))]
    scaled, log = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    writes.append((lambda: lm.block_attention(q, k, v, idx, block=B, out=scaled), lambda: (scaled * leaves[0]).sum()))
    writes.append((lambda: lm.block_attention(q, k, v, idx, block=B, lse=log), lambda: (log[:, :, None] * leaves[0]).sum()))
    for write, use in writes:
        out = use()
        write()
        with pytest.raises(RuntimeError, match="inplace operation"):
            out.sum().backward()


def test_buffers_that_require_a_gradient_are_refused(lm):
    leaves, idx, _, B = small(88, torch.float32)
    q, k, v = (x.detach() for x in leaves)
    wants = torch.empty_like(q).requires_grad_()
    with pytest.raises(ValueError):
        lm.block_attention(q, k, v, idx, block=B, out=wants)
    with pytest.raises(ValueError):
        lm.block_means(k, block=B, out=torch.empty(-(-k.shape[0] // B), *k.shape[1:], device=DEV).requires_grad_())
    with torch.no_grad():
        lm.block_attention(q, k, v, idx, block=B, out=wants)
    assert torch.equal(wants.detach(), lm.block_attention(q, k, v, idx, block=B))
    with torch.inference_mode():
        out = torch.empty_like(q)
        lm.block_attention(q, k, v, idx, block=B, out=out)
        assert torch.equal(out, wants)


def test_capture_over_leaves_behind_other_operators(lm):
    """A weight in front of the call: an eager graph over it, made on the default stream, keeps a capture from starting; a deleted one does not."""
    leaves, idx, dout, B = small(89, torch.bfloat16)
    q, k, v = (x.detach() for x in leaves)
    w = torch.ones(1, dtype=torch.bfloat16, device=DEV, requires_grad=True)

    def forward():
        return lm.block_attention(q * w, k, v, idx, block=B)

    def step():
        out = forward()
        return (out.detach(), *torch.autograd.grad(out, [w], dout))

    alive = forward()
    with pytest.raises(RuntimeError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            forward()
    del alive
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        q.copy_(rand(torch.Generator().manual_seed(90), *q.shape, dtype=q.dtype))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want
