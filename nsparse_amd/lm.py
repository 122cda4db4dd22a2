"""Sparse products of language models on torch tensors: include/nsparse_lm.h behind torch's allocator and streams.

  * attention over blocks of keys that a cheap score selects: block_means, select_blocks, block_attention
    (differentiable) and block_attention_backward; single tokens over a paged cache are the same calls;
  * tokens sorted by expert and back: route, gather_tokens, combine_tokens (both differentiable) and their *_backward.

Tensors live on one GPU; work is queued on that device's current stream and nothing synchronises, so every call may be captured
into a graph.  A backward pass is captured by calling the *_backward functions, or through autograd while no graph made outside of the
capture over the same leaves is alive (refused with RuntimeError where such a graph came from these functions, over their own inputs or, made
on the default stream, over leaves behind them).  Refused
arguments raise ValueError with the reason, tensors with a tangent (forward mode) NotImplementedError.  Block means, and so the selection,
have no derivative: they come without a graph.  There is no fallback: a missing library raises.
"""
import ctypes as C
import math
import struct
import threading
import weakref

import torch
from torch.autograd import forward_ad

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
        # a table cut out of a wider one: its rows count as long as they are apart, so the last one has to be there in full
        if page_table is not None and self.n > 1 and page_table.shape[1] > 0 and (
                page_table.stride(0) < page_table.shape[1] or
                page_table.storage_offset() + self.n * page_table.stride(0) > page_table.untyped_storage().nbytes() // 4):
            raise ValueError("Seqs: page_table's rows must not overlap, and a cut of a wider table must keep the last row's end")
        self.cu_q, self.cu_k, self.q_len, self.k_len, self.page_table = cu_q, cu_k, q_len, k_len, page_table

    # addresses, read at every call (0: none)
    ptr_cu_q = property(lambda self: 0 if self.cu_q is None else self.cu_q.data_ptr())
    ptr_cu_k = property(lambda self: 0 if self.cu_k is None else self.cu_k.data_ptr())
    ptr_q_len = property(lambda self: 0 if self.q_len is None else self.q_len.data_ptr())
    ptr_k_len = property(lambda self: 0 if self.k_len is None else self.k_len.data_ptr())
    # (a table without columns is not read, but has to be somewhere)
    ptr_table = property(lambda self: 0 if self.page_table is None else self.page_table.data_ptr() or self.ptr_k_len)

    def _tensors(self):
        return [t for t in (self.cu_q, self.cu_k, self.q_len, self.k_len, self.page_table) if t is not None]


_ONE = Seqs(1)


def _check(rc):
    if rc < 0:
        raise ValueError(load_lm().nsparse_lm_last_error_string().decode())
    if rc > 0:
        raise RuntimeError(load_lm().nsparse_lm_last_error_string().decode())


def _on_gpu(*tensors):
    """The index of the GPU that all tensors live on."""
    dev = tensors[0].get_device()
    if dev < 0:
        raise ValueError("tensors must live on a GPU")
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError("all tensors must live on one device")
    return dev


def _no_tangent(*tensors):
    """Forward mode is refused: a kernel reads a tensor's address, the tangent would be lost."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("there is no derivative in forward mode")


def _queued(dev, fn, *args):
    """fn(*args, stream) with the tensors' device current."""
    if torch.cuda.current_device() == dev:
        return fn(*args, _raw_stream(dev))
    with torch.cuda.device(dev):
        return fn(*args, _raw_stream(dev))


def _raw_stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _contiguous(t, what, dtype=None, shape=None):
    if not t.is_contiguous() or (dtype is not None and t.dtype != dtype) or (shape is not None and t.shape != shape):
        raise ValueError(f"{what} must be contiguous" + (f", {dtype}" if dtype is not None else "") +
                         (f", of shape {tuple(shape)}" if shape is not None else ""))


def _written(*buffers):
    """The caller's buffers that a kernel writes count as written in place: a graph that saved one of them refuses its backward."""
    for t in buffers:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("a buffer to write into must not require a gradient")
        torch.autograd.graph.increment_version(t)


# the fields of LmAttn in their order (an int of padding before the 64-bit ones is the struct module's)
_ATTN = struct.Struct("@11if3q5P8q")
assert _ATTN.size == C.sizeof(LmAttn)


def _attn(seqs, block, *, q=None, k=None, v=None, kv_heads=None, k_rows=None, page_size=0, width=1, causal=True, scale=0.0, first=0, local=0):
    """The argument block of a call, and its key heads.  Without q: for the keys alone."""
    some = q if k is None else k
    dtype = _DTYPES.get(some.dtype)
    if dtype is None:
        raise ValueError("tensors must be float32, float16 or bfloat16")
    table = seqs.page_table
    q_rows = heads = dim = q0 = q1 = 0
    if q is not None:
        if q.dim() != 3 or q.stride(2) != 1 and q.shape[2] > 1:
            raise ValueError("q must be [rows, heads, head_dim] with a contiguous head_dim")
        q_rows, heads, dim = q.shape
        q0, q1 = (q.stride(0) if q_rows > 1 else 0), (q.stride(1) if heads > 1 else 0)
    ks = vs = (0, 0, 0)
    if k is not None:
        ks = _key_strides(k, "k", table is not None)
        if v is not None:
            if v.shape != k.shape or v.dtype != k.dtype:
                raise ValueError("k and v must have one shape and type")
            vs = _key_strides(v, "v", table is not None)
        shape = k.shape
        k_rows, kv_heads = shape[0], shape[-2]
        if q is None:
            heads, dim = kv_heads, shape[-1]
        elif dim != shape[-1] or q.dtype != k.dtype:
            raise ValueError("q, k and v must have one head_dim and type")
        if table is not None:
            page_size = shape[1]
    table_stride = 0 if table is None else table.stride(0) if seqs.n > 1 and table.shape[1] else table.shape[1]
    try:
        packed = _ATTN.pack(
            dtype, heads, kv_heads, dim, int(block), int(width), 1 if causal else 0, seqs.n, page_size, int(first), int(local), scale, q_rows,
            int(k_rows), table_stride, 0 if q is None else seqs.ptr_cu_q,
            seqs.ptr_cu_k, 0 if q is None else seqs.ptr_q_len, seqs.ptr_k_len, seqs.ptr_table, q0, q1, *ks, *vs)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"an argument is out of range: {e}") from None
    return LmAttn.from_buffer_copy(packed), kv_heads


def _key_strides(t, what, paged):
    if t.dim() != (4 if paged else 3) or t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what} must be [rows, kv_heads, head_dim], or [pages, page_size, kv_heads, head_dim] with a page table, "
                         "with a contiguous head_dim")
    shape, stride = t.shape, t.stride()
    return (stride[0] if paged and shape[0] > 1 else 0, stride[-3] if shape[-3] > 1 else 0, stride[-2] if shape[-2] > 1 else 0)


def _empty_or_zeros(whole, *shape, dtype, device):
    """A new output: rows that no sequence has are left as they were by the kernels, so they start as zeros."""
    return (torch.empty if whole else torch.zeros)(*shape, dtype=dtype, device=device)


# ---- attention over selected blocks ---------------------------------------------------------------------------------------
def block_means(k, *, block, seqs=None, last=0, out=None):
    """Mean of every block of `block` keys, in the keys' type: [rows, kv_heads, head_dim], rows as nsparse_lm.h numbers them.  Without a
    derivative.  Sequences that share a page have to hold the same keys of a block that is computed.

    out: a buffer kept from earlier calls (a serving cache keeps it beside the keys); last > 0 then refreshes only the
    blocks that hold the last `last` keys of each sequence.
    """
    seqs = seqs or _ONE
    dev = _on_gpu(k, *seqs._tensors(), *([out] if out is not None else []))
    a, _ = _attn(seqs, block, k=k)
    lib = load_lm()
    ref = C.byref(a)
    rows = lib.nsparse_lm_mean_rows(ref)
    _check(min(rows, 0))
    shape = (rows, k.shape[-2], k.shape[-1])
    if out is None:
        whole = seqs.cu_k is None and seqs.k_len is None and last == 0
        out = _empty_or_zeros(whole, *shape, dtype=k.dtype, device=k.device)
    else:
        _contiguous(out, "out", k.dtype, shape)
        _written(out)
    _check(_queued(dev, lib.nsparse_lm_block_means, ref, k.data_ptr(), out.data_ptr(), int(last)))
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
    page_size = 0
    if seqs.page_table is not None:
        if k_rows < 1 or means.shape[0] % k_rows:
            raise ValueError("means must have page_size / block rows a page")
        page_size = means.shape[0] // k_rows * int(block)
    a, _ = _attn(seqs, block, q=q, kv_heads=means.shape[1], k_rows=k_rows, page_size=page_size, width=width, causal=causal, first=first, local=local)
    lib = load_lm()
    ref = C.byref(a)
    rows = lib.nsparse_lm_mean_rows(ref)
    _check(min(rows, 0))
    if rows != means.shape[0]:
        raise ValueError(f"means must have {rows} rows for these keys")
    shape = (q.shape[0], means.shape[1], int(width))
    if out is None:
        whole = seqs.cu_q is None and seqs.q_len is None
        out = torch.empty(shape, dtype=torch.int32, device=q.device) if whole else torch.full(shape, -1, dtype=torch.int32, device=q.device)
    else:
        _contiguous(out, "out", torch.int32, shape)
        _written(out)
    _check(_queued(dev, lib.nsparse_lm_select_blocks, ref, q.data_ptr(), means.data_ptr(), out.data_ptr()))
    return out


def _attention(dev, q, k, v, idx, block, scale, causal, seqs, out, lse):
    a, kv_heads = _attn(seqs, block, q=q, k=k, v=v, width=idx.shape[-1] if idx.dim() == 3 else 0, causal=causal, scale=scale)
    shape = q.shape
    _contiguous(idx, "idx", torch.int32, (shape[0], kv_heads, a.width))
    whole = seqs.cu_q is None and seqs.q_len is None
    if out is None:
        out = _empty_or_zeros(whole, *shape, dtype=q.dtype, device=q.device)
    else:
        _contiguous(out, "out", q.dtype, shape)
        _written(out)
    if lse is None:
        lse = _empty_or_zeros(whole, shape[0], shape[1], dtype=torch.float32, device=q.device)
    else:
        _contiguous(lse, "lse", torch.float32, shape[:2])
        _written(lse)
    _check(_queued(dev, load_lm().nsparse_lm_block_attention, C.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), idx.data_ptr(),
                   out.data_ptr(), lse.data_ptr()))
    return out, lse


# Autograd nodes that were made outside of a capture and are alive.  A leaf's gradient is accumulated on the stream on which the first
# of its living nodes was made: a backward pass captured while one of these lives would leave the capture, which ends the process.
# Refused are graphs over the call's own leaves, and those made on the default stream, which cannot join a capture, over leaves
# further back.
_eager = weakref.WeakSet()
_eager_lock = threading.RLock()  # a finalizer may make a node while its thread holds it


def _leaves_behind(*starts):
    """Ids of the leaves that these tensors or autograd nodes come from."""
    leaves, seen, todo = set(), set(), []
    for x in starts:
        if not isinstance(x, torch.Tensor):
            todo.append(x)
        elif x.requires_grad and x.is_leaf:
            leaves.add(id(x))
        elif x.requires_grad:
            todo.append(x.grad_fn)
    while todo:
        node = todo.pop()
        if node in seen:
            continue
        seen.add(node)
        try:
            before = [n for n, _ in node.next_functions if n is not None]
        except RuntimeError:  # another thread's graph has just gone
            continue
        if not before and hasattr(node, "variable"):
            leaves.add(id(node.variable))
        todo += before
    return leaves


def _may_capture(ctx, *inputs):
    wanted = [t for t in inputs if t.requires_grad]
    if not wanted:
        return
    ctx.leaves = [id(t) for t in wanted if t.is_leaf]
    ctx.on_default = _raw_stream(wanted[0].get_device()) == 0
    if not torch.cuda.is_current_stream_capturing():
        with _eager_lock:
            _eager.add(ctx)
        return
    with _eager_lock:
        alive = list(_eager)
    if not alive:
        return
    behind = _leaves_behind(*wanted)
    if any(x in node.leaves for node in alive for x in ctx.leaves) or behind & _leaves_behind(*[node for node in alive if node.on_default]):
        raise RuntimeError("a graph made outside of this capture over the same leaves is alive: delete its outputs before capturing")


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, idx, block, scale, causal, seqs):
        _may_capture(ctx, q, k, v)
        out, lse = _attention(q.get_device(), q, k, v, idx, block, scale, causal, seqs, None, None)
        ctx.save_for_backward(q, k, v, idx, out, lse, *seqs._tensors())
        ctx.rest = (block, scale, causal, seqs)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, idx, out, lse = ctx.saved_tensors[:6]
        block, scale, causal, seqs = ctx.rest
        dout = torch.zeros_like(out) if dout is None else dout.contiguous()
        if dout.data_ptr() % 16:  # a piece of a larger gradient may begin anywhere
            dout = dout.clone()
        dlse = None if dlse is None else dlse.contiguous()
        dq, dk, dv = block_attention_backward(dout, q, k, v, idx, out, lse, block=block, scale=scale, causal=causal, seqs=seqs, dlse=dlse)
        return dq, dk, dv, None, None, None, None, None


def block_attention(q, k, v, idx, *, block, scale=None, causal=True, seqs=None, out=None, lse=None, return_lse=False):
    """softmax(scale q k^T) v over the keys of the listed blocks; scale defaults to head_dim ** -0.5.

    q [rows, heads, head_dim]; k, v [rows, kv_heads, head_dim] or a paged cache; idx int32 [rows, kv_heads, width] as select_blocks
    returns it.  Differentiable in q, k, v (not over a paged cache), through the output and through the log-sum-exp [rows, heads] that
    return_lse adds.  out, lse: buffers to write into (then not differentiable).
    """
    seqs = seqs or _ONE
    dev = _on_gpu(q, k, v, idx, *seqs._tensors(), *[t for t in (out, lse) if t is not None])
    _no_tangent(q, k, v)
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if out is not None or lse is not None:
            raise ValueError("out and lse do not go with tensors that require a gradient")
        if seqs.page_table is not None:
            raise ValueError("a paged cache has no gradient")
        o, s = _BlockAttention.apply(q, k, v, idx, block, scale, causal, seqs)
    else:
        o, s = _attention(dev, q, k, v, idx, block, scale, causal, seqs, out, lse)
    return (o, s) if return_lse else o


def block_attention_backward(dout, q, k, v, idx, out, lse, *, block, scale=None, causal=True, seqs=None, dlse=None):
    """(dq, dk, dv) of block_attention from its output and log-sum-exp; dlse: the log-sum-exp's own gradient, if it has one."""
    seqs = seqs or _ONE
    some = [] if dlse is None else [dlse]
    dev = _on_gpu(dout, q, k, v, idx, out, lse, *some, *seqs._tensors())
    _no_tangent(dout, q, k, v, out, lse, *some)
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    a, kv_heads = _attn(seqs, block, q=q, k=k, v=v, width=idx.shape[-1] if idx.dim() == 3 else 0, causal=causal, scale=scale)
    shape = q.shape
    _contiguous(idx, "idx", torch.int32, (shape[0], kv_heads, a.width))
    _contiguous(dout, "dout", q.dtype, shape)
    _contiguous(out, "out", q.dtype, shape)
    _contiguous(lse, "lse", torch.float32, shape[:2])
    if dlse is not None:
        _contiguous(dlse, "dlse", torch.float32, shape[:2])
    lib = load_lm()
    ref = C.byref(a)
    need = lib.nsparse_lm_block_attention_bwd_workspace(ref)
    _check(min(need, 0))
    whole_q = seqs.cu_q is None and seqs.q_len is None
    whole_k = seqs.cu_k is None and seqs.k_len is None
    dq = _empty_or_zeros(whole_q, *shape, dtype=q.dtype, device=q.device)
    dk = _empty_or_zeros(whole_k, *k.shape, dtype=q.dtype, device=q.device)
    dv = _empty_or_zeros(whole_k, *k.shape, dtype=q.dtype, device=q.device)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _check(_queued(dev, lib.nsparse_lm_block_attention_lse_bwd, ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), idx.data_ptr(), out.data_ptr(),
                   lse.data_ptr(), dout.data_ptr(), _ptr(dlse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need))
    return dq, dk, dv


# ---- tokens sorted by expert --------------------------------------------------------------------------------------------
class Route:
    """A sorted routing: offsets int32 [experts + 1], order int32 [tokens * top] (sorted row -> entry t * top + j; what stands behind
    offsets[experts] means nothing), place int32 [tokens, top] (entry -> sorted row, -1 where dropped)."""

    def __init__(self, offsets, order, place):
        if place.dtype != torch.int32 or place.dim() != 2 or not place.is_contiguous():
            raise ValueError("place must be a contiguous int32 tensor [tokens, top]")
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
    offsets = torch.empty(int(experts) + 1, dtype=torch.int32, device=ids.device)
    order = torch.empty(tokens * top, dtype=torch.int32, device=ids.device)
    place = torch.empty(tokens, top, dtype=torch.int32, device=ids.device)
    ws = torch.empty(need, dtype=torch.uint8, device=ids.device) if need else None
    _check(_queued(dev, lib.nsparse_lm_route, ids.data_ptr(), tokens, top, int(experts), offsets.data_ptr(), order.data_ptr(), place.data_ptr(),
                   _ptr(ws), need))
    return Route(offsets, order, place)


def _rows(t, what, rows):
    if t.dtype not in _DTYPES:
        raise ValueError("tensors must be float32, float16 or bfloat16")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{what} must be [{rows}, channels]")
    _contiguous(t, what)


def _weights(w, place):
    if w is not None:
        _contiguous(w, "weights", torch.float32, place.shape)


def _gather(x, place):
    dev = _on_gpu(x, place)
    tokens, top = place.shape
    _rows(x, "x", tokens)
    xs = torch.empty(tokens * top, x.shape[1], dtype=x.dtype, device=x.device)
    _check(_queued(dev, load_lm().nsparse_lm_gather_tokens, _DTYPES[x.dtype], x.data_ptr(), place.data_ptr(), tokens, top, x.shape[1],
                   xs.data_ptr()))
    return xs


def _combine(y, place, weights):
    dev = _on_gpu(y, place, *([weights] if weights is not None else []))
    tokens, top = place.shape
    _rows(y, "y", tokens * top)
    _weights(weights, place)
    out = torch.empty(tokens, y.shape[1], dtype=y.dtype, device=y.device)
    _check(_queued(dev, load_lm().nsparse_lm_combine_tokens, _DTYPES[y.dtype], y.data_ptr(), place.data_ptr(), _ptr(weights), tokens, top,
                   y.shape[1], out.data_ptr()))
    return out


# The plan's rows are saved like any tensor that backward reads: torch tells when they were written again in between.
class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, place):
        _may_capture(ctx, x)
        ctx.save_for_backward(place)
        return _gather(x, place)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        _no_tangent(dxs)
        return _combine(dxs.contiguous(), *ctx.saved_tensors, None), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, place, weights):
        _may_capture(ctx, y, weights)
        ctx.save_for_backward(y, place, weights)
        return _combine(y, place, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        dy, dw = _combine_backward(dout.contiguous(), *ctx.saved_tensors, fill=True)
        return dy, None, dw


def gather_tokens(x, plan):
    """xs [tokens * top, channels]: the tokens' rows expert by expert (rows behind offsets[experts] mean nothing).  Differentiable."""
    _no_tangent(x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Gather.apply(x, plan.place)
    return _gather(x, plan.place)


def gather_tokens_backward(dxs, plan):
    """dx [tokens, channels]: the sum of each token's rows of dxs."""
    _no_tangent(dxs)
    return _combine(dxs, plan.place, None)


def combine_tokens(y, plan, weights):
    """out [tokens, channels] = sum over a token's entries of weights [tokens, top] (float32) times their rows of y.  Differentiable."""
    if weights is None:
        raise ValueError("weights must be given; a plain sum of a token's rows is gather_tokens_backward")
    _no_tangent(y, weights)
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _Combine.apply(y, plan.place, weights)
    return _combine(y, plan.place, weights)


def _combine_backward(dout, y, place, weights, fill):
    dev = _on_gpu(dout, y, place, weights)
    _no_tangent(dout, y, weights)
    tokens, top = place.shape
    _rows(dout, "dout", tokens)
    _rows(y, "y", tokens * top)
    if y.dtype != dout.dtype or y.shape[1] != dout.shape[1]:
        raise ValueError("dout and y must have one type and number of channels")
    _weights(weights, place)
    dy = (torch.zeros_like if fill else torch.empty_like)(y)
    dw = torch.empty_like(weights)
    _check(_queued(dev, load_lm().nsparse_lm_combine_tokens_bwd, _DTYPES[y.dtype], dout.data_ptr(), y.data_ptr(), place.data_ptr(),
                   weights.data_ptr(), tokens, top, y.shape[1], dy.data_ptr(), dw.data_ptr()))
    return dy, dw


def combine_tokens_backward(dout, y, plan, weights):
    """(dy, dw) of combine_tokens; rows of dy behind offsets[experts] mean nothing."""
    return _combine_backward(dout, y, plan.place, weights, fill=False)
