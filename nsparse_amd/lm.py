"""Sparse products of language models on torch tensors: include/nsparse_lm.h behind torch's allocator and streams.

  * attention over blocks of keys that a cheap score selects: block_means, select_blocks, block_attention
    (differentiable) and block_attention_backward; single tokens over a paged cache are the same calls;
  * tokens sorted by expert and back: route, gather_tokens, combine_tokens (both differentiable) and their *_backward.

Tensors live on one GPU; work is queued on that device's current stream and nothing synchronises, so every call may be captured
into a graph.  Refused arguments raise ValueError with the reason.  There is no fallback: a missing library raises.
"""
import ctypes as C
import math

import torch

from .capi import LmAttn, load_lm

__all__ = ["Seqs", "Route", "block_means", "select_blocks", "block_attention", "block_attention_backward", "route",
           "gather_tokens", "gather_tokens_backward", "combine_tokens", "combine_tokens_backward"]

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Seqs:
    """How query rows and key rows fall into `n` sequences (device int32 tensors; see nsparse_lm.h).

    cu_q / cu_k [n + 1]: packed rows; without them every sequence has the same number of rows.  q_len / k_len [n]: only that
    many of them count.  page_table [n, pages]: keys are a paged cache [pages, page_size, kv_heads, head_dim] (k_len required).
    """

    def __init__(self, n, cu_q=None, cu_k=None, q_len=None, k_len=None, page_table=None):
        self.n = int(n)
        if self.n < 1:
            raise ValueError("Seqs: n must be positive")
        for name, t, size in (("cu_q", cu_q, self.n + 1), ("cu_k", cu_k, self.n + 1), ("q_len", q_len, self.n), ("k_len", k_len, self.n)):
            if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous()):
                raise ValueError(f"Seqs: {name} must be a contiguous int32 tensor of {size} numbers")
        if page_table is not None and (page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != self.n
                                       or page_table.stride(1) != 1 and page_table.shape[1] > 1):
            raise ValueError("Seqs: page_table must be an int32 tensor [n, pages] with contiguous rows")
        self.cu_q, self.cu_k, self.q_len, self.k_len, self.page_table = cu_q, cu_k, q_len, k_len, page_table

    def _tensors(self):
        return [t for t in (self.cu_q, self.cu_k, self.q_len, self.k_len, self.page_table) if t is not None]


_ONE = Seqs(1)


def _check(rc):
    if rc < 0:
        raise ValueError(load_lm().nsparse_lm_last_error_string().decode())
    if rc > 0:
        raise RuntimeError(load_lm().nsparse_lm_last_error_string().decode())


def _on_gpu(*tensors):
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError("tensors must live on a GPU")
    for t in tensors:
        if t.device != dev:
            raise ValueError("all tensors must live on one device")
    return dev


def _ptr(t):
    return None if t is None else t.data_ptr()


def _contiguous(t, what, dtype=None, shape=None):
    if not t.is_contiguous() or (dtype is not None and t.dtype != dtype) or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{what} must be contiguous" + (f", {dtype}" if dtype is not None else "") +
                         (f", of shape {tuple(shape)}" if shape is not None else ""))


def _attn(seqs, block, *, q=None, k=None, v=None, q_heads=None, k_rows=None, width=1, causal=True, scale=0.0, first=0, local=0):
    """The argument block of a call."""
    a = LmAttn()
    some = k if k is not None else q
    if some.dtype not in _DTYPES:
        raise ValueError("tensors must be float32, float16 or bfloat16")
    a.dtype = _DTYPES[some.dtype]
    a.block, a.width, a.causal, a.n_seq = int(block), int(width), int(bool(causal)), seqs.n
    a.first, a.local, a.scale = int(first), int(local), float(scale)
    paged = seqs.page_table is not None
    if q is not None:
        if q.dim() != 3 or q.stride(2) != 1 and q.shape[2] > 1:
            raise ValueError("q must be [rows, heads, head_dim] with a contiguous head_dim")
        a.q_rows, a.heads, a.head_dim = q.shape
        a.q_stride[0], a.q_stride[1] = q.stride(0) if q.shape[0] > 1 else 0, q.stride(1) if q.shape[1] > 1 else 0
        a.kv_heads = a.heads
    if k is not None:
        for t, what in ((k, "k"), (v, "v")):
            if t is None:
                continue
            if t.dim() != (4 if paged else 3) or t.stride(-1) != 1 and t.shape[-1] > 1:
                raise ValueError(f"{what} must be [rows, kv_heads, head_dim], or [pages, page_size, kv_heads, head_dim] with a page table, "
                                 "with a contiguous head_dim")
            if t.shape != k.shape or t.dtype != k.dtype:
                raise ValueError("k and v must have one shape and type")
        a.k_rows, a.kv_heads = k.shape[0], k.shape[-2]
        if q is None:
            a.heads, a.head_dim = a.kv_heads, k.shape[-1]
            if not paged and seqs.cu_q is None:
                a.q_rows = 0
        elif q.shape[2] != k.shape[-1] or q.dtype != k.dtype:
            raise ValueError("q, k and v must have one head_dim and type")
        if paged:
            a.page_size = k.shape[1]
        for t, stride in ((k, a.k_stride), (v, a.v_stride)):
            if t is not None:
                if paged:
                    stride[0] = t.stride(0) if t.shape[0] > 1 else 0
                stride[1] = t.stride(-3) if t.shape[-3] > 1 else 0
                stride[2] = t.stride(-2) if t.shape[-2] > 1 else 0
    if k_rows is not None:
        a.k_rows = int(k_rows)
    if q_heads is not None:
        a.heads, a.kv_heads = q_heads
    if paged:
        a.table_stride = seqs.page_table.stride(0) if seqs.n > 1 else seqs.page_table.shape[1]
    a.cu_q, a.cu_k, a.q_len, a.k_len, a.page_table = (_ptr(seqs.cu_q), _ptr(seqs.cu_k), _ptr(seqs.q_len), _ptr(seqs.k_len),
                                                      _ptr(seqs.page_table))
    return a


class _Queue:
    """The device of a call made current, and its current stream."""

    def __init__(self, dev):
        self.guard = torch.cuda.device(dev)
        self.dev = dev

    def __enter__(self):
        self.guard.__enter__()
        return torch.cuda.current_stream(self.dev).cuda_stream

    def __exit__(self, *exc):
        return self.guard.__exit__(*exc)


def _empty_or_zeros(whole, *shape, dtype, device):
    """A new output: rows that no sequence has are left as they were by the kernels, so they start as zeros."""
    return (torch.empty if whole else torch.zeros)(*shape, dtype=dtype, device=device)


# ---- attention over selected blocks ---------------------------------------------------------------------------------------
def block_means(k, *, block, seqs=None, last=0, out=None):
    """Mean of every block of `block` keys, in the keys' type: [rows, kv_heads, head_dim], rows as nsparse_lm.h numbers them.

    out: a buffer kept from earlier calls (a serving cache keeps it beside the keys); last > 0 then refreshes only the
    blocks that hold the last `last` keys of each sequence.
    """
    seqs = seqs or _ONE
    dev = _on_gpu(k, *seqs._tensors(), *([out] if out is not None else []))
    a = _attn(seqs, block, k=k)
    a.cu_q = None
    a.q_len = None
    a.q_rows = 0
    lib = load_lm()
    rows = lib.nsparse_lm_mean_rows(C.byref(a))
    _check(min(rows, 0))
    shape = (rows, k.shape[-2], k.shape[-1])
    if out is None:
        whole = seqs.cu_k is None and seqs.k_len is None and last == 0
        out = _empty_or_zeros(whole, *shape, dtype=k.dtype, device=dev)
    else:
        _contiguous(out, "out", k.dtype, shape)
    with _Queue(dev) as st:
        _check(lib.nsparse_lm_block_means(C.byref(a), _ptr(k), _ptr(out), int(last), st))
    return out


def select_blocks(q, means, *, block, width, k_rows, first=1, local=1, causal=True, seqs=None, out=None):
    """int32 [rows, kv_heads, width]: the blocks that every query row selects for every key head, ascending, -1 behind.

    k_rows: rows (pages) of the keys that `means` stands for.  The first `first` and (causal) last `local` blocks up to the query's own are
    always taken, the rest by score.
    """
    seqs = seqs or _ONE
    dev = _on_gpu(q, means, *seqs._tensors(), *([out] if out is not None else []))
    if means.dim() != 3 or means.dtype != q.dtype or means.shape[2] != q.shape[-1]:
        raise ValueError("means must be [rows, kv_heads, head_dim] in q's type")
    _contiguous(means, "means")
    a = _attn(seqs, block, q=q, k_rows=k_rows, width=width, causal=causal, first=first, local=local)
    a.kv_heads = means.shape[1]
    lib = load_lm()
    if seqs.page_table is not None:
        if k_rows < 1 or means.shape[0] % k_rows:
            raise ValueError("means must have page_size / block rows a page")
        a.page_size = means.shape[0] // k_rows * int(block)
    rows = lib.nsparse_lm_mean_rows(C.byref(a))
    _check(min(rows, 0))
    if rows != means.shape[0]:
        raise ValueError(f"means must have {rows} rows for these keys")
    shape = (q.shape[0], means.shape[1], int(width))
    if out is None:
        whole = seqs.cu_q is None and seqs.q_len is None
        out = torch.empty(shape, dtype=torch.int32, device=dev) if whole else torch.full(shape, -1, dtype=torch.int32, device=dev)
    else:
        _contiguous(out, "out", torch.int32, shape)
    with _Queue(dev) as st:
        _check(lib.nsparse_lm_select_blocks(C.byref(a), _ptr(q), _ptr(means), _ptr(out), st))
    return out


def _attention(q, k, v, idx, block, scale, causal, seqs, out, lse):
    a = _attn(seqs, block, q=q, k=k, v=v, width=idx.shape[-1] if idx.dim() == 3 else 0, causal=causal, scale=scale)
    _contiguous(idx, "idx", torch.int32, (q.shape[0], a.kv_heads, a.width))
    whole = seqs.cu_q is None and seqs.q_len is None
    if out is None:
        out = _empty_or_zeros(whole, *q.shape, dtype=q.dtype, device=q.device)
    else:
        _contiguous(out, "out", q.dtype, q.shape)
    if lse is None:
        lse = _empty_or_zeros(whole, q.shape[0], q.shape[1], dtype=torch.float32, device=q.device)
    else:
        _contiguous(lse, "lse", torch.float32, q.shape[:2])
    with _Queue(q.device) as st:
        _check(load_lm().nsparse_lm_block_attention(C.byref(a), _ptr(q), _ptr(k), _ptr(v), _ptr(idx), _ptr(out), _ptr(lse), st))
    return out, lse


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, idx, block, scale, causal, seqs):
        out, lse = _attention(q, k, v, idx, block, scale, causal, seqs, None, None)
        ctx.save_for_backward(q, k, v, idx, out, lse, *seqs._tensors())
        ctx.rest = (block, scale, causal, seqs)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, idx, out, lse = ctx.saved_tensors[:6]
        block, scale, causal, seqs = ctx.rest
        dq, dk, dv = block_attention_backward(dout.contiguous(), q, k, v, idx, out, lse, block=block, scale=scale, causal=causal, seqs=seqs)
        return dq, dk, dv, None, None, None, None, None


def block_attention(q, k, v, idx, *, block, scale=None, causal=True, seqs=None, out=None, lse=None, return_lse=False):
    """softmax(scale q k^T) v over the keys of the listed blocks; scale defaults to head_dim ** -0.5.

    q [rows, heads, head_dim]; k, v [rows, kv_heads, head_dim] or a paged cache; idx int32 [rows, kv_heads, width] as select_blocks
    returns it.  Differentiable in q, k, v (not over a paged cache).  out, lse: buffers to write into (then not differentiable).
    """
    seqs = seqs or _ONE
    _on_gpu(q, k, v, idx, *seqs._tensors(), *[t for t in (out, lse) if t is not None])
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if out is not None or lse is not None:
            raise ValueError("out and lse do not go with tensors that require a gradient")
        if seqs.page_table is not None:
            raise ValueError("a paged cache has no gradient")
        o, s = _BlockAttention.apply(q, k, v, idx, block, scale, causal, seqs)
    else:
        o, s = _attention(q, k, v, idx, block, scale, causal, seqs, out, lse)
    return (o, s) if return_lse else o


def block_attention_backward(dout, q, k, v, idx, out, lse, *, block, scale=None, causal=True, seqs=None):
    """(dq, dk, dv) of block_attention from its output and log-sum-exp."""
    seqs = seqs or _ONE
    dev = _on_gpu(dout, q, k, v, idx, out, lse, *seqs._tensors())
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    a = _attn(seqs, block, q=q, k=k, v=v, width=idx.shape[-1] if idx.dim() == 3 else 0, causal=causal, scale=scale)
    _contiguous(idx, "idx", torch.int32, (q.shape[0], a.kv_heads, a.width))
    _contiguous(dout, "dout", q.dtype, q.shape)
    _contiguous(out, "out", q.dtype, q.shape)
    _contiguous(lse, "lse", torch.float32, q.shape[:2])
    lib = load_lm()
    need = lib.nsparse_lm_block_attention_bwd_workspace(C.byref(a))
    _check(min(need, 0))
    whole_q = seqs.cu_q is None and seqs.q_len is None
    whole_k = seqs.cu_k is None and seqs.k_len is None
    dq = _empty_or_zeros(whole_q, *q.shape, dtype=q.dtype, device=dev)
    dk = _empty_or_zeros(whole_k, *k.shape, dtype=q.dtype, device=dev)
    dv = _empty_or_zeros(whole_k, *k.shape, dtype=q.dtype, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with _Queue(dev) as st:
        _check(lib.nsparse_lm_block_attention_bwd(C.byref(a), _ptr(q), _ptr(k), _ptr(v), _ptr(idx), _ptr(out), _ptr(lse), _ptr(dout),
                                                  _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), need, st))
    return dq, dk, dv


# ---- tokens sorted by expert --------------------------------------------------------------------------------------------
class Route:
    """A sorted routing: offsets int32 [experts + 1], order int32 [tokens * top] (sorted row -> entry t * top + j; what stands behind
    offsets[experts] means nothing), place int32 [tokens, top] (entry -> sorted row, -1 where dropped)."""

    def __init__(self, offsets, order, place):
        self.offsets, self.order, self.place = offsets, order, place
        self.tokens, self.top = place.shape


def route(ids, experts):
    """Sort the entries of ids (int32 [tokens, top]) by expert, stable; ids outside [0, experts) are dropped."""
    dev = _on_gpu(ids)
    if ids.dim() != 2:
        raise ValueError("ids must be [tokens, top]")
    _contiguous(ids, "ids", torch.int32)
    lib = load_lm()
    tokens, top = ids.shape
    need = lib.nsparse_lm_route_workspace(tokens, top, int(experts))
    _check(min(need, 0))
    offsets = torch.empty(int(experts) + 1, dtype=torch.int32, device=dev)
    order = torch.empty(tokens * top, dtype=torch.int32, device=dev)
    place = torch.empty(tokens, top, dtype=torch.int32, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _Queue(dev) as st:
        _check(lib.nsparse_lm_route(_ptr(ids), tokens, top, int(experts), _ptr(offsets), _ptr(order), _ptr(place), _ptr(ws), need, st))
    return Route(offsets, order, place)


def _rows(t, what, rows):
    if t.dtype not in _DTYPES:
        raise ValueError("tensors must be float32, float16 or bfloat16")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{what} must be [{rows}, channels]")
    _contiguous(t, what)


def _weights(w, plan):
    if w is not None:
        _contiguous(w, "weights", torch.float32, (plan.tokens, plan.top))


def _gather(x, plan):
    dev = _on_gpu(x, plan.place)
    _rows(x, "x", plan.tokens)
    xs = torch.empty(plan.tokens * plan.top, x.shape[1], dtype=x.dtype, device=dev)
    with _Queue(dev) as st:
        _check(load_lm().nsparse_lm_gather_tokens(_DTYPES[x.dtype], _ptr(x), _ptr(plan.place), plan.tokens, plan.top, x.shape[1], _ptr(xs), st))
    return xs


def _combine(y, plan, weights):
    dev = _on_gpu(y, plan.place, *([weights] if weights is not None else []))
    _rows(y, "y", plan.tokens * plan.top)
    _weights(weights, plan)
    out = torch.empty(plan.tokens, y.shape[1], dtype=y.dtype, device=dev)
    with _Queue(dev) as st:
        _check(load_lm().nsparse_lm_combine_tokens(_DTYPES[y.dtype], _ptr(y), _ptr(plan.place), _ptr(weights), plan.tokens, plan.top, y.shape[1],
                                                   _ptr(out), st))
    return out


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _gather(x, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        return gather_tokens_backward(dxs.contiguous(), ctx.plan), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, plan, weights):
        ctx.plan = plan
        ctx.save_for_backward(y, weights)
        return _combine(y, plan, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights = ctx.saved_tensors
        dy, dw = _combine_backward(dout.contiguous(), y, ctx.plan, weights, fill=True)
        return dy, None, dw


def gather_tokens(x, plan):
    """xs [tokens * top, channels]: the tokens' rows expert by expert (rows behind offsets[experts] mean nothing).  Differentiable."""
    if torch.is_grad_enabled() and x.requires_grad:
        return _Gather.apply(x, plan)
    return _gather(x, plan)


def gather_tokens_backward(dxs, plan):
    """dx [tokens, channels]: the sum of each token's rows of dxs."""
    return _combine(dxs, plan, None)


def combine_tokens(y, plan, weights):
    """out [tokens, channels] = sum over a token's entries of weights [tokens, top] (float32) times their rows of y.  Differentiable."""
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _Combine.apply(y, plan, weights)
    return _combine(y, plan, weights)


def _combine_backward(dout, y, plan, weights, fill):
    dev = _on_gpu(dout, y, plan.place, weights)
    _rows(dout, "dout", plan.tokens)
    _rows(y, "y", plan.tokens * plan.top)
    if y.dtype != dout.dtype or y.shape[1] != dout.shape[1]:
        raise ValueError("dout and y must have one type and number of channels")
    _weights(weights, plan)
    dy = (torch.zeros_like if fill else torch.empty_like)(y)
    dw = torch.empty_like(weights)
    with _Queue(dev) as st:
        _check(load_lm().nsparse_lm_combine_tokens_bwd(_DTYPES[y.dtype], _ptr(dout), _ptr(y), _ptr(plan.place), _ptr(weights), plan.tokens,
                                                       plan.top, y.shape[1], _ptr(dy), _ptr(dw), st))
    return dy, dw


def combine_tokens_backward(dout, y, plan, weights):
    """(dy, dw) of combine_tokens; rows of dy behind offsets[experts] mean nothing."""
    return _combine_backward(dout, y, plan, weights, fill=False)
