"""Plain 64-bit forms of the operators of include/nsparse_lm.h, on the CPU, and bounds of what a kernel may be off by.

Every bound counts roundings: u(T) = half a step of type T relative to the value, 2^-24 for one operation in 32 bits.
"""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step below the smallest normal number: what rounding to T may change there, whatever the value."""
    return torch.finfo(dtype).smallest_normal * u(dtype)


class Layout:
    """Sequences as lists: (first query row, query rows, key rows as an index list or None entries for hidden keys)."""

    def __init__(self, seqs):
        self.seqs = seqs


def packed(q_lens, k_lens):
    out, a, b = [], 0, 0
    for m, n in zip(q_lens, k_lens):
        out.append((a, m, list(range(b, b + n))))
        a, b = a + m, b + n
    return Layout(out)


def uniform(n, q_each, k_each, q_len=None, k_len=None):
    return Layout([(s * q_each, q_each if q_len is None else q_len[s],
                    list(range(s * k_each, s * k_each + (k_each if k_len is None else k_len[s])))) for s in range(n)])


def paged(k_len, table, page, pages, q_each=1):
    """Key j of sequence s is row table[s][j // page] * page + j % page of the flattened cache; -1 for a page that is none."""
    out = []
    for s, n in enumerate(k_len):
        rows = []
        for j in range(n):
            p = table[s][j // page]
            rows.append(p * page + j % page if 0 <= p < pages else -1)
        out.append((s * q_each, q_each, rows))
    return Layout(out)


def listed(row, limit, block):
    """The blocks of a pattern row that count: inside the visible keys and greater than every entry before."""
    seen, out = -1, []
    for e in row:
        if e > seen:
            if e * block < limit:
                out.append(e)
            seen = e
    return out


def attention(q, k, v, idx, layout, block, scale, causal, dout=None):
    """dict of out, lse (and dq, dk, dv with dout) and of tol_* bounds, all float64.  q, k, v in the kernel's type; k, v flattened rows."""
    T = q.dtype
    Q, K, V = q.double(), k.double(), v.double()
    n, H, D = Q.shape
    G = K.shape[1]
    ut, ta = u(T), tiny(T)
    out = torch.zeros(n, H, D, dtype=torch.float64)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64)
    tol_out, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    covered = torch.zeros(n, dtype=torch.bool)
    if dout is not None:
        dO = dout.double()
        dq, dk, dv = torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V)
        tq, tk, tv = torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V)
        size_k, size_v = torch.zeros_like(K), torch.zeros_like(K)
        terms = torch.zeros(K.shape[0], G, 1, dtype=torch.float64)
    for first, rows_q, rows_k in layout.seqs:
        L = len(rows_k)
        for i in range(rows_q):
            t = first + i
            covered[t] = True
            limit = min(L, L - rows_q + i + 1) if causal else L
            for g in range(G):
                if limit <= 0:
                    continue
                keys = [j for b in listed(idx[t, g].tolist(), limit, block) for j in range(b * block, min(b * block + block, limit))]
                keys = [rows_k[j] for j in keys if rows_k[j] >= 0]
                if not keys:
                    continue
                hs = slice(g * (H // G), (g + 1) * (H // G))
                kk, vv, qq = K[keys, g], V[keys, g], Q[t, hs]
                s = scale * qq @ kk.t()
                m = s.max(dim=1, keepdim=True).values
                e = torch.exp(s - m)
                tot = e.sum(1, keepdim=True)
                p = e / tot
                o = p @ vv
                N = len(keys)
                # a score is off by the roundings of a sum of D products, of the scale (rounded, times log2 e) and of its
                # subtraction from the running maximum; the exponential adds 2^-21 of its value
                ds = (D + 4) * U32 * abs(scale) * (qq.abs() @ kk.abs().t()).max() + 2 * U32 * (s.abs().max() + 1)
                rel = 2 * ds + 2.0 ** -21 + (N + 64) * U32
                out[t, hs], lse[t, hs] = o, (m + torch.log(tot)).squeeze(1)
                tol_out[t, hs] = ut * o.abs() * 1.01 + (1.01 * ut + 2 * rel) * (p @ vv.abs()) + ta * (vv.abs().sum(0) + 1)
                tol_lse[t, hs] = ds + rel + 4 * U32 * lse[t, hs].abs()
                if dout is None:
                    continue
                do = dO[t, hs]
                dp = do @ vv.t()
                delta = (do * o).sum(1, keepdim=True)
                d = p * (dp - delta)
                # p in the backward comes from the rounded log-sum-exp; delta from the rounded output
                rel_p = rel + tol_lse[t, hs].max()
                off_delta = (do.abs() * tol_out[t, hs]).sum(1, keepdim=True) + (D + 2) * U32 * (do.abs() * o.abs()).sum(1, keepdim=True)
                off_dp = (D + 2) * U32 * (do.abs() @ vv.abs().t())
                off_d = p * ((dp - delta).abs() * (1.01 * ut + rel_p + 6 * U32) + off_dp + off_delta) * 1.02
                dq[t, hs] = scale * d @ kk
                tq[t, hs] = (abs(scale) * (off_d + N * U32 * d.abs()) + ta) @ kk.abs() + 2 * U32 * dq[t, hs].abs()
                dk[keys, g] += scale * d.t() @ qq
                dv[keys, g] += p.t() @ do
                tk[keys, g] += (abs(scale) * off_d + ta).t() @ qq.abs()
                tv[keys, g] += (p * (1.01 * ut + rel_p) * 1.02 + ta).t() @ do.abs()
                terms[keys, g] += H // G
                size_k[keys, g] += abs(scale) * d.abs().t() @ qq.abs()
                size_v[keys, g] += p.t() @ do.abs()
    res = dict(out=out, lse=lse, tol_out=tol_out, tol_lse=tol_lse, covered=covered)
    if dout is not None:
        tk += (terms + 4) * U32 * size_k  # the sums over rows, in 32 bits
        tv += (terms + 4) * U32 * size_v
        res.update(dq=dq, dk=dk, dv=dv, tol_dq=tq + 1.01 * ut * dq.abs() + ta, tol_dk=tk + 1.01 * ut * dk.abs() + ta,
                   tol_dv=tv + 1.01 * ut * dv.abs() + ta)
    return res


def block_mean_rows(k, layout, block):
    """{(sequence, block): [kv_heads, head_dim] float64} over the keys that exist."""
    out = {}
    for s, (_, _, rows) in enumerate(layout.seqs):
        for b in range(-(-len(rows) // block)):
            part = rows[b * block:b * block + block]
            if all(r >= 0 for r in part):
                out[s, b] = k[part].double().mean(0)
    return out


def select(q, means, layout, block, width, first, local, causal):
    """means: {(sequence, block): [kv_heads, head_dim]} in the kernel's type; absent blocks score lowest."""
    n, H, D = q.shape
    G = next(iter(means.values())).shape[0] if means else 1
    idx = torch.full((n, G, width), -1, dtype=torch.int32)
    Q = q.double()
    for s, (start, rows_q, rows_k) in enumerate(layout.seqs):
        L = len(rows_k)
        for i in range(rows_q):
            pos = L - rows_q + i
            eligible = (0 if pos < 0 else pos // block + 1) if causal else -(-L // block)
            for g in range(G):
                qs = Q[start + i, g * (H // G):(g + 1) * (H // G)].sum(0)
                forced = [b for b in range(eligible) if b < first or b >= eligible - local]
                rest = []
                for b in range(eligible):
                    if b in forced:
                        continue
                    m = means.get((s, b))
                    x = -math.inf if m is None else float(qs @ m[g].double())
                    rest.append((math.inf if math.isnan(x) else -x, b))
                rest.sort()
                got = sorted(forced + [b for _, b in rest[:max(0, width - len(forced))]])[:width]
                idx[start + i, g, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return idx


def route(ids, experts):
    """offsets, order (list), place [tokens, top]"""
    T, K = ids.shape
    buckets = [[] for _ in range(experts)]
    for t in range(T):
        for j in range(K):
            e = int(ids[t, j])
            if 0 <= e < experts:
                buckets[e].append(t * K + j)
    order = [x for b in buckets for x in b]
    offsets = [0]
    for b in buckets:
        offsets.append(offsets[-1] + len(b))
    place = torch.full((T * K,), -1, dtype=torch.int32)
    for r, x in enumerate(order):
        place[x] = r
    return offsets, order, place.view(T, K)
