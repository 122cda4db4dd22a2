"""Sparse products whose pattern a language model chooses row by row: what is measured, and the plain forms.

Two families of operators (nsparse_amd.lm):
  * attention over blocks of keys that a cheap score selects for each query -- the selection (block means, scores, the
    best `width` blocks), attention over the selected blocks, its gradient, and the form for single tokens over a paged cache;
  * tokens sorted by expert and back with weights applied, and the gradient.

`own = False` computes the plain forms with elementary torch operations; `own = True` calls the framework.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a long prompt picks the blocks of every token: grouped heads, one sequence
        dict(name="select_prompt", op="select", lens="16384", paged=0, heads=32, kv=8, dim=128, block=64, width=16, first=1,
             local=2, type="bf16"),
        # one step of serving 16 conversations: the newest block's mean is refreshed in the cache, one query each selects
        dict(name="select_step", op="select", lens="32768,1,64,65,1000,20011,777,16384,5,31007,4096,12345,128,2500,8191,27000",
             paged=64, heads=32, kv=8, dim=128, block=64, width=16, first=1, local=2, type="bf16"),
        # a long prompt attends to its selected blocks
        dict(name="attend_prompt", op="attend", lens="8192", paged=0, heads=32, kv=8, dim=128, block=64, width=16, type="bf16"),
        # several prompts of uneven lengths in one call, smaller heads and blocks, half precision
        dict(name="attend_ragged", op="attend", lens="1,2047,333,64,1500", paged=0, heads=16, kv=4, dim=64, block=32, width=8,
             type="f16"),
        # the next token of one long conversation: latency
        dict(name="decode_one", op="attend", lens="30011", paged=64, heads=32, kv=8, dim=128, block=64, width=16, type="bf16"),
        # the next token of 64 conversations of very uneven lengths, pages of two blocks
        dict(name="decode_batch", op="attend", lens=_spread_lens(64, 32768), paged=128, heads=32, kv=8, dim=128, block=64,
             width=32, type="bf16"),
        # one training step of the attention: forward and gradients
        dict(name="train_prompt", op="train", lens="4096", paged=0, heads=32, kv=8, dim=128, block=64, width=16, type="bf16"),
        # packed sequences of odd lengths in single precision, a head size between the powers of two
        dict(name="train_ragged", op="train", lens="701,1,17,640,142", paged=0, heads=6, kv=2, dim=96, block=16, width=12,
             type="f32"),
        # a prompt through a wide layer of 64 experts: sort, gather, combine
        dict(name="route_prompt", op="route", tokens=16384, channels=4096, experts=64, top=8, dropped=0.0, type="bf16"),
        # a handful of decoded tokens: latency
        dict(name="route_few", op="route", tokens=7, channels=2048, experts=128, top=4, dropped=0.0, type="f16"),
        # one training step of the routing: forward and gradients
        dict(name="route_train", op="route_train", tokens=8192, channels=2048, experts=32, top=4, dropped=0.0, type="bf16"),
        # an odd row size, and experts that live on another device (their entries are dropped here)
        dict(name="route_train_odd", op="route_train", tokens=1003, channels=1023, experts=24, top=3, dropped=0.3, type="f32"),
    ]


def _spread_lens(n, longest):
    """n lengths spread evenly over the logarithm of 1..longest, as text."""
    return ",".join(str(max(1, round(longest ** (i / (n - 1))))) for i in range(n))


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, parts):
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng: random.Random):
    op = rng.choice(["select", "select", "attend", "attend", "attend", "train", "train", "route", "route_train"])
    ty = rng.choice(["bf16", "f16", "f32"])
    if op in ("route", "route_train"):
        tokens = _log_uniform(rng, 1, 16384 if op == "route" else 8192)
        top = rng.randint(1, 8)
        channels = _log_uniform(rng, 64, 4096) | rng.randint(0, 1)
        if op == "route_train":
            top, channels = min(top, 4), min(channels, 2048)
        if ty == "f32":
            channels = max(64, channels // 2)
        return dict(op=op, tokens=tokens, channels=channels, experts=_log_uniform(rng, max(top, 4), 256), top=top,
                    dropped=rng.choice([0.0, 0.0, 0.5]), type=ty)
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4])
    dim = rng.choice([64, 80, 96, 128])
    block = rng.choice([16, 32, 64])
    width = rng.randint(3, 16)
    case = dict(op=op, heads=kv * group, kv=kv, dim=dim, block=block, width=width, type=ty)
    if op == "select":
        case.update(first=rng.randint(0, 1), local=rng.randint(1, 2))
    if op != "train" and rng.random() < 0.5:
        n = rng.randint(1, 32)
        case.update(paged=block * rng.choice([1, 2]), lens=",".join(str(_log_uniform(rng, 1, 16384)) for _ in range(n)))
    else:
        total = _log_uniform(rng, 1, {"select": 8192, "attend": 4096, "train": 2048}[op])
        case.update(paged=0, lens=_split(rng, total, rng.randint(1, 6)))
    return case


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


# ---- inputs -------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    ty = _TYPES[case["type"]]
    st = dict(case=case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)

    if case["op"] in ("route", "route_train"):
        T, C, E, K = case["tokens"], case["channels"], case["experts"], case["top"]
        # a router's choice: K distinct experts a token, some experts liked better than others
        logits = normal(T, E) + 1.5 * normal(1, E)
        best = torch.topk(logits, K, dim=1)
        ids = best.indices.to(torch.int32)
        if case["dropped"] > 0:
            gone = torch.rand(T, K, generator=gen, device=dev) < case["dropped"]
            ids = torch.where(gone, torch.full_like(ids, -1), ids)
        st.update(ids=ids, weights=torch.softmax(best.values, dim=1).contiguous(), x=normal(T, C).to(ty))
        st["y"] = normal(T * K, C).to(ty)  # what the experts returned, row by row of the sorted order
        if case["op"] == "route_train":
            st["dout"] = normal(T, C).to(ty)
            st["dxs"] = normal(T * K, C).to(ty)
        return st

    lens = _lens(case)
    H, G, D, B = case["heads"], case["kv"], case["dim"], case["block"]
    n = len(lens)
    k_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    if case["paged"]:
        P = case["paged"]
        need = [(L + P - 1) // P for L in lens]
        pages = sum(need) + 3
        deal = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        table = torch.full((n, max(need)), -1, dtype=torch.int32, device=dev)
        at = 0
        for s, m in enumerate(need):
            table[s, :m] = deal[at:at + m]
            at += m
        kv_shape = (pages, P, G, D)
        st.update(table=table, k_len=k_len, cu=None)
        Tq = n
        row_seq = torch.arange(n, device=dev)
        row_pos = k_len.long() - 1
    else:
        total = sum(lens)
        kv_shape = (total, G, D)
        cu = torch.zeros(n + 1, dtype=torch.int32, device=dev)
        cu[1:] = torch.cumsum(k_len, 0)
        st.update(table=None, k_len=None, cu=cu)
        Tq = total
        row_seq = torch.searchsorted(cu[1:].long(), torch.arange(total, device=dev), right=True)
        row_pos = torch.arange(total, device=dev) - cu.long()[row_seq]
    st["q"] = normal(Tq, H, D).to(ty)
    st["k"] = normal(*kv_shape).to(ty)
    if case["op"] == "select":
        if case["paged"]:
            # the cache keeps the means beside the keys; the step refreshes the newest block of each conversation
            st["means"] = st["k"].view(kv_shape[0] * (case["paged"] // B), B, G, D).double().mean(1).to(ty)
    else:
        st["v"] = normal(*kv_shape).to(ty)
        # the selected blocks: the own one, the first, and others that stay alike over neighbouring queries
        nb = (max(lens) + B - 1) // B
        W = case["width"]
        slow = normal(Tq // 64 + 1, G, nb)
        idx = torch.empty(Tq, G, W, dtype=torch.int32, device=dev)
        blocks = torch.arange(nb, device=dev)
        for a in range(0, Tq, 2048):
            z = min(a + 2048, Tq)
            score = slow[torch.arange(a, z, device=dev) // 64] + 0.5 * normal(z - a, G, nb)
            own_block = (row_pos[a:z] // B)[:, None, None]
            score = torch.where((blocks == own_block) | (blocks == 0), score + 100.0, score)
            score = torch.where(blocks > own_block, torch.full_like(score, -math.inf), score)
            take = min(W, nb)
            top = torch.topk(score, take, dim=2)
            got = torch.where(torch.isinf(top.values), torch.full_like(top.indices, nb), top.indices).sort(dim=2).values
            idx[a:z, :, :take] = torch.where(got == nb, torch.full_like(got, -1), got).to(torch.int32)
            idx[a:z, :, take:] = -1
        st["idx"] = idx
        if case["op"] == "train":
            st["dout"] = normal(Tq, H, D).to(ty)
    if own:
        from nsparse_amd import lm
        if case["paged"]:
            st["seqs"] = lm.Seqs(n, k_len=k_len, page_table=st["table"])
        elif n > 1:
            st["seqs"] = lm.Seqs(n, cu_q=st["cu"], cu_k=st["cu"])
        else:
            st["seqs"] = None
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from nsparse_amd import lm
    case = st["case"]
    op = case["op"]
    if op in ("route", "route_train"):
        plan = lm.route(st["ids"], case["experts"])
        xs = lm.gather_tokens(st["x"], plan)
        out = lm.combine_tokens(st["y"], plan, st["weights"])
        res = dict(offsets=plan.offsets, place=plan.place, out=out)
        if case["dropped"] == 0:
            res.update(order=plan.order, xs=xs)
        else:
            # rows behind the last expert are nobody's: they are not part of the result
            res.update(order=_kept_rows(plan.order, plan.offsets), xs=_kept_rows(xs, plan.offsets))
        if op == "route_train":
            dy, dw = lm.combine_tokens_backward(st["dout"], st["y"], plan, st["weights"])
            dx = lm.gather_tokens_backward(st["dxs"], plan)
            res.update(dx=dx, dw=dw, dy=dy if case["dropped"] == 0 else _kept_rows(dy, plan.offsets))
        return res
    B = case["block"]
    if op == "select":
        if case["paged"]:
            means = lm.block_means(st["k"], block=B, seqs=st["seqs"], last=1, out=st["means"])
        else:
            means = lm.block_means(st["k"], block=B, seqs=st["seqs"])
        idx = lm.select_blocks(st["q"], means, block=B, width=case["width"], first=case["first"], local=case["local"],
                               k_rows=st["k"].shape[0], seqs=st["seqs"])
        return dict(means=means, idx=idx)
    out, lse = lm.block_attention(st["q"], st["k"], st["v"], st["idx"], block=B, seqs=st["seqs"], return_lse=True)
    if op == "attend":
        return dict(out=out, lse=lse)
    dq, dk, dv = lm.block_attention_backward(st["dout"], st["q"], st["k"], st["v"], st["idx"], out, lse, block=B,
                                             seqs=st["seqs"])
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


def _kept_rows(rows, offsets):
    """Rows behind offsets[-1] set to zero (a whole-tensor product a user's experts would do by masking)."""
    live = torch.arange(rows.shape[0], device=rows.device) < offsets[-1]
    return torch.where(live.view(-1, *([1] * (rows.dim() - 1))), rows, torch.zeros_like(rows))


def _run_plain(st):
    op = st["case"]["op"]
    if op in ("route", "route_train"):
        return _plain_route(st)
    if op == "select":
        return _plain_select(st)
    return _plain_attention(st)


def _plain_route(st):
    case = st["case"]
    ids, w, E = st["ids"], st["weights"], case["experts"]
    T, K = ids.shape
    N, ty = T * K, st["x"].dtype
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    srt = torch.sort(key, stable=True)
    order = srt.indices
    counts = (key[:, None] == torch.arange(E, device=key.device)).sum(0)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=key.device)
    offsets[1:] = torch.cumsum(counts, 0)
    live = srt.values < E
    place = torch.empty_like(order)
    place[order] = torch.arange(N, device=key.device)
    place = torch.where(key < E, place, torch.full_like(place, -1)).reshape(T, K)
    live_rows = live[:, None]
    xs = st["x"].float()[order // K] * live_rows
    at = place.clamp(min=0)
    picked = (place >= 0).float()
    y = st["y"].float()
    out = torch.zeros(T, y.shape[1], dtype=torch.float32, device=y.device)
    for j in range(K):
        out = out + torch.where((place[:, j] >= 0)[:, None], w[:, j, None] * y[at[:, j]], torch.zeros((), device=y.device))
    res = dict(offsets=offsets.to(torch.int32), place=place.to(torch.int32), out=out.to(ty),
               order=torch.where(live, order, torch.zeros_like(order)).to(torch.int32), xs=xs.to(ty))
    if case["op"] == "route_train":
        dout = st["dout"].float()
        dy = dout[order // K] * w.reshape(-1)[order][:, None] * live_rows
        dw = torch.stack([(dout * y[at[:, j]]).sum(1) * picked[:, j] for j in range(K)], dim=1)
        dx = torch.zeros_like(out)
        dxs = st["dxs"].float()
        for j in range(K):
            dx = dx + dxs[at[:, j]] * picked[:, j, None]
        res.update(dy=dy.to(ty), dw=dw, dx=dx.to(ty))
    return res


def _rows_of(st):
    """Sequence and position of every query row, length and first row of every sequence (device tensors)."""
    q = st["q"]
    dev = q.device
    if st["cu"] is None:
        seq = torch.arange(q.shape[0], device=dev)
        length = st["k_len"].long()
        return seq, length - 1, length, None
    cu = st["cu"].long()
    seq = torch.searchsorted(cu[1:], torch.arange(q.shape[0], device=dev), right=True)
    return seq, torch.arange(q.shape[0], device=dev) - cu[seq], cu[1:] - cu[:-1], cu[:-1]


def _plain_select(st):
    case = st["case"]
    B, W, G = case["block"], case["width"], case["kv"]
    q, k = st["q"], st["k"]
    seq, pos, length, start = _rows_of(st)
    n = length.shape[0]
    if case["paged"]:
        P = case["paged"]
        newest = (length - 1) // B
        row = st["table"].long()[torch.arange(n, device=q.device), newest * B // P]
        inside = (newest * B % P)[:, None] + torch.arange(B, device=q.device)
        keys = k[row[:, None], inside].double()
        live = (newest[:, None] * B + torch.arange(B, device=q.device)) < length[:, None]
        fresh = (keys * live[:, :, None, None]).sum(1) / live.sum(1)[:, None, None]
        means = st["means"]
        means[row * (P // B) + newest * B % P // B] = fresh.to(k.dtype)
    else:
        one = n == 1
        rows = (k.shape[0] + B - 1) // B if one else k.shape[0] // B + n
        where = (torch.zeros_like(seq) if one else start[seq] // B + seq) + pos // B
        total = torch.zeros(rows, G, k.shape[2], dtype=torch.float64, device=k.device)
        total.index_add_(0, where, k.double())
        count = torch.zeros(rows, dtype=torch.float64, device=k.device)
        count.index_add_(0, where, torch.ones_like(where, dtype=torch.float64))
        means = (total / count.clamp(min=1.0)[:, None, None]).to(k.dtype)
    qsum = q.double().view(q.shape[0], G, -1, q.shape[2]).sum(2)
    idx = torch.full((q.shape[0], G, W), -1, dtype=torch.int32, device=q.device)
    if case["paged"]:
        for s in range(n):
            nb = -(-_lens(case)[s] // B)
            b = torch.arange(nb, device=q.device)
            m = means[st["table"].long()[s, b * B // P] * (P // B) + b * B % P // B].double()
            _pick(case, qsum[s:s + 1], m, pos[s:s + 1], idx[s:s + 1])
    else:
        at = 0
        for s, L in enumerate(_lens(case)):
            nb = -(-L // B)
            if L:
                first = 0 if one else at // B + s
                for a in range(at, at + L, 8192):
                    z = min(a + 8192, at + L)
                    _pick(case, qsum[a:z], means[first:first + nb].double(), pos[a:z], idx[a:z])
            at += L
    return dict(means=means, idx=idx)


def _pick(case, qsum, means, pos, idx):
    """idx[rows, g, :] = the selected blocks of these rows, ascending, -1 behind."""
    nb = means.shape[0]
    W = min(case["width"], nb)
    own_block = (pos // case["block"])[:, None]
    b = torch.arange(nb, device=pos.device)
    rank = torch.where(b > own_block, 2, torch.where((b < case["first"]) | (b > own_block - case["local"]), 0, 1))
    for g in range(case["kv"]):
        score = qsum[:, g] @ means[:, g].t().contiguous()
        score = torch.where(torch.isnan(score), torch.full_like(score, -math.inf), score)
        by_score = torch.sort(score, dim=1, descending=True, stable=True).indices
        by_rank = torch.sort(rank.gather(1, by_score), dim=1, stable=True)
        got = by_score.gather(1, by_rank.indices)[:, :W]
        got = torch.where(by_rank.values[:, :W] == 2, torch.full_like(got, nb), got).sort(dim=1).values
        idx[:, g, :W] = torch.where(got == nb, torch.full_like(got, -1), got).to(torch.int32)


def _plain_attention(st):
    case = st["case"]
    q, idx, B, W, G = st["q"], st["idx"], case["block"], case["width"], case["kv"]
    D, H, Tq = q.shape[2], q.shape[1], q.shape[0]
    scale = 1.0 / math.sqrt(D)
    dev, ty = q.device, q.dtype
    seq, pos, length, start = _rows_of(st)
    k = st["k"].reshape(-1, G, D).float().transpose(0, 1).contiguous()
    v = st["v"].reshape(-1, G, D).float().transpose(0, 1).contiguous()
    heads = torch.arange(G, device=dev)[:, None, None]
    out = torch.zeros(Tq, H, D, dtype=torch.float32, device=dev)
    lse = torch.empty(Tq, H, dtype=torch.float32, device=dev)
    train = case["op"] == "train"
    if train:
        dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, (1 << 28) // (G * W * B * D))
    for a in range(0, Tq, step):
        z = min(a + step, Tq)
        r = z - a
        block = idx[a:z].long()
        j = block[:, :, :, None] * B + torch.arange(B, device=dev)
        live = (block >= 0)[:, :, :, None] & (j <= pos[a:z, None, None, None])
        j = torch.where(live, j, torch.zeros_like(j))
        if case["paged"]:
            P = case["paged"]
            row = st["table"].long()[seq[a:z, None, None, None], j // P].clamp(min=0) * P + j % P
        else:
            row = start[seq[a:z, None, None, None]] + j
        row = row.reshape(r, G, W * B).transpose(0, 1)
        live = live.reshape(r, G, W * B).transpose(0, 1)
        kg, vg = k[heads, row], v[heads, row]
        qg = q[a:z].float().view(r, G, H // G, D).transpose(0, 1).contiguous()
        s = torch.matmul(qg, kg.transpose(2, 3).contiguous()) * scale
        s = torch.where(live[:, :, None], s, torch.full_like(s, -math.inf))
        top = s.max(dim=3, keepdim=True).values
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        e = torch.exp(s - top)
        total = e.sum(3, keepdim=True)
        p = e / torch.where(total == 0, torch.ones_like(total), total)
        o = torch.matmul(p, vg)
        out[a:z] = o.transpose(0, 1).reshape(r, H, D)
        lse[a:z] = (torch.log(total) + top).squeeze(3).transpose(0, 1).reshape(r, H)
        if train:
            do = st["dout"][a:z].float().view(r, G, H // G, D).transpose(0, 1).contiguous()
            delta = (do * o).sum(3, keepdim=True)
            ds = p * (torch.matmul(do, vg.transpose(2, 3).contiguous()) - delta) * scale
            dq[a:z] = torch.matmul(ds, kg).transpose(0, 1).reshape(r, H, D)
            add_v = torch.matmul(p.transpose(2, 3).contiguous(), do)
            add_k = torch.matmul(ds.transpose(2, 3).contiguous(), qg)
            for g in range(G):
                dv[g].index_add_(0, row[g].reshape(-1), add_v[g].reshape(-1, D))
                dk[g].index_add_(0, row[g].reshape(-1), add_k[g].reshape(-1, D))
    res = dict(out=out.to(ty), lse=lse)
    if train:
        res.update(dq=dq.to(ty), dk=dk.transpose(0, 1).contiguous().to(ty), dv=dv.transpose(0, 1).contiguous().to(ty))
    return res


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    w = 4 if case["type"] == "f32" else 2
    if case["op"] in ("route", "route_train"):
        T, C, E, K = case["tokens"], case["channels"], case["experts"], case["top"]
        N = T * K * (1.0 - case["dropped"])
        ints = 4 * (2 * T * K + N + E + 1)
        fwd = w * C * (T + N + N + T) + 4 * N + ints  # x, xs, y, out
        if case["op"] == "route":
            return dict(bytes=int(fwd), flops=int(2 * N * C))
        # dout and y (again) in, dy and dw out; dxs in, dx out
        return dict(bytes=int(fwd + w * C * (T + N + N) + 8 * N + w * C * (N + T)), flops=int(6 * N * C))
    lens = _lens(case)
    H, G, D, B, W = case["heads"], case["kv"], case["dim"], case["block"], case["width"]
    Tq = len(lens) if case["paged"] else sum(lens)
    if case["op"] == "select":
        blocks = sum(-(-L // B) for L in lens)
        if case["paged"]:
            keys = sum((L - 1) % B + 1 for L in lens if L)
            pairs = blocks
        else:
            keys = sum(lens)
            pairs = sum(L * (-(-L // B) + 1) / 2 for L in lens)
        return dict(bytes=int(w * D * (keys * G + blocks * G + Tq * H) + 4 * Tq * G * W),
                    flops=int(2 * pairs * G * D + keys * G * D + Tq * H * D))
    # keys a row attends to: all it has, or what width blocks hold
    if case["paged"]:
        att = sum(min(L, W * B) for L in lens)
        keys = att
    else:
        att = 0
        for L in lens:
            full = min(L, W * B)
            att += full * (full + 1) / 2 + (L - full) * (W * B - B / 2)
        keys = sum(lens)
    rows = Tq * H
    byts = w * D * (2 * rows + 2 * keys * G) + 4 * rows + 4 * Tq * G * W
    if case["op"] == "attend":
        return dict(bytes=int(byts), flops=int(4 * att * H * D))
    byts += w * D * (2 * rows + 2 * keys * G)  # dout in, dq, dk, dv out
    return dict(bytes=int(byts), flops=int(14 * att * H * D))


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("route", "route_train"):
        return _exact_route(case, st)
    if case["op"] == "select":
        return _exact_select(case, st)
    return _exact_attention(case, st)


def _exact_route(case, st):
    ids = st["ids"].cpu().tolist()
    T, K, E, C = case["tokens"], case["top"], case["experts"], case["channels"]
    dev = st["x"].device
    buckets = [[] for _ in range(E)]
    for t, row in enumerate(ids):
        for j, e in enumerate(row):
            if 0 <= e < E:
                buckets[e].append(t * K + j)
    order = [e for b in buckets for e in b]
    offsets = [0]
    for b in buckets:
        offsets.append(offsets[-1] + len(b))
    place = [-1] * (T * K)
    for r, e in enumerate(order):
        place[e] = r
    live = len(order)
    ent = torch.tensor(order, dtype=torch.int64, device=dev)
    tok, w = ent // K, st["weights"].double().reshape(-1)[ent][:, None]
    xs = torch.zeros(T * K, C, dtype=torch.float64, device=dev)
    xs[:live] = st["x"].double()[tok]
    y = st["y"][:live].double()
    out = torch.zeros(T, C, dtype=torch.float64, device=dev).index_add_(0, tok, w * y)
    res = dict(offsets=torch.tensor(offsets, dtype=torch.int32, device=dev),
               place=torch.tensor(place, dtype=torch.int32, device=dev).reshape(T, K), out=out,
               order=torch.tensor(order + [0] * (T * K - live), dtype=torch.int32, device=dev), xs=xs)
    if case["op"] == "route_train":
        dout = st["dout"].double()[tok]
        dy = torch.zeros_like(xs)
        dy[:live] = w * dout
        dw = torch.zeros(T * K, dtype=torch.float64, device=dev)
        dw[ent] = (dout * y).sum(1)
        dx = torch.zeros_like(out).index_add_(0, tok, st["dxs"][:live].double())
        res.update(dy=dy, dw=dw.reshape(T, K), dx=dx)
    return res


def _sequences(case, st):
    """Per sequence: its query rows and its keys' rows in the flattened cache."""
    at = 0
    for s, L in enumerate(_lens(case)):
        if case["paged"]:
            P = case["paged"]
            j = torch.arange(L, device=st["q"].device)
            yield s, L, slice(s, s + 1), st["table"][s].long()[j // P] * P + j % P
        else:
            yield s, L, slice(at, at + L), torch.arange(at, at + L, device=st["q"].device)
        at += L


def _exact_select(case, st):
    B, W, G, H = case["block"], case["width"], case["kv"], case["heads"]
    q, k = st["q"], st["k"].reshape(-1, G, case["dim"])
    dev, lens = q.device, _lens(case)
    if case["paged"]:
        means = st["means"].double()
    else:
        rows = -(-lens[0] // B) if len(lens) == 1 else sum(lens) // B + len(lens)
        means = torch.zeros(rows, G, case["dim"], dtype=torch.float64, device=dev)
    idx = torch.full((q.shape[0], G, W), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, L, qs, rows in _sequences(case, st):
        if not L:
            continue
        nb = -(-L // B)
        if case["paged"]:
            where = rows[::B] // B
            means[where[-1]] = k[rows[(nb - 1) * B:]].double().mean(0)
            held = st["means"].double()[where]
            held[-1] = means[where[-1]].to(k.dtype).double()
        else:
            base = 0 if len(lens) == 1 else at // B + s
            fine = torch.stack([c.double().mean(0) for c in k[at:at + L].split(B)])
            means[base:base + nb] = fine
            held = fine.to(k.dtype).double()  # the scores are defined on the means as the cache holds them
        n = 1 if case["paged"] else L
        pos = torch.arange(L - n, L, device=dev)
        for a in range(0, n, 4096):
            p = pos[a:a + 4096]
            rows_q = q[qs][a:a + 4096].double()
            b = torch.arange(nb, device=dev)[None, :]
            own_block = (p // B)[:, None]
            forced = (b < case["first"]) | (b > own_block - case["local"])
            for g in range(G):
                score = torch.zeros(p.shape[0], nb, dtype=torch.float64, device=dev)
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    score += rows_q[:, h] @ held[:, g].t().contiguous()
                score = score.masked_fill(forced, math.inf).masked_fill(b > own_block, -math.inf)
                take = min(W, nb)
                best = torch.topk(score, take, dim=1)
                chosen = torch.zeros(p.shape[0], nb, dtype=torch.bool, device=dev)
                chosen.scatter_(1, best.indices, best.values > -math.inf)
                slot = torch.cumsum(chosen.int(), 1) - 1
                r, c = torch.nonzero(chosen, as_tuple=True)
                target = idx[qs][a:a + 4096]
                target[r, g, slot[r, c].long()] = c.to(torch.int32)
        at += L
    return dict(means=means, idx=idx)


def _exact_attention(case, st):
    B, G, H, D = case["block"], case["kv"], case["heads"], case["dim"]
    q, idx = st["q"], st["idx"]
    dev = q.device
    scale = 1.0 / math.sqrt(D)
    k, v = (st[x].reshape(-1, G, D).double() for x in ("k", "v"))
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=dev)
    train = case["op"] == "train"
    if train:
        dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
    for s, L, qs, rows in _sequences(case, st):
        if not L:
            continue
        n = 1 if case["paged"] else L
        nb = -(-L // B)
        late = torch.arange(L, device=dev)[None, :] > torch.arange(L - n, L, device=dev)[:, None]
        for g in range(G):
            kk, vv = k[rows, g], v[rows, g]
            listed_blocks = torch.zeros(n, nb + 1, dtype=torch.bool, device=dev)
            sel = idx[qs][:, g].long()
            listed_blocks.scatter_(1, torch.where(sel < 0, torch.full_like(sel, nb), sel), True)
            allowed = listed_blocks[:, :nb].repeat_interleave(B, dim=1)[:, :L] & ~late
            for h in range(g * (H // G), (g + 1) * (H // G)):
                qq = q[qs][:, h].double()
                z = (qq @ kk.t().contiguous() * scale).masked_fill(~allowed, -math.inf)
                norm = torch.logsumexp(z, dim=1, keepdim=True)
                p = torch.exp(z - norm).masked_fill(~allowed, 0.0)
                out[qs, h] = p @ vv
                lse[qs, h] = norm[:, 0]
                if train:
                    do = st["dout"][qs][:, h].double()
                    back = p * (do @ vv.t().contiguous() - (do * out[qs, h]).sum(1, keepdim=True)) * scale
                    dq[qs, h] = back @ kk
                    dk[rows, g] += back.t().contiguous() @ qq
                    dv[rows, g] += p.t().contiguous() @ do
    res = dict(out=out, lse=lse)
    if train:
        res.update(dq=dq, dk=dk, dv=dv)
    return res
