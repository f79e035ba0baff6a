"""Paged key/value caches and drafted trees.

The decode path of a server whose sequences have different lengths and whose
steps may verify several drafted tokens per sequence.  A step is

    plan = paged.plan(batch, parents)                    # once
    q    = paged.append(batch, plan, qkv, ...)           # per layer
    out  = paged.tree_attention(batch, plan, q, ...)     # per layer
    acc  = paged.tree_accept(batch, parents, tokens, predicted)

over a `PagedCache` (the pools of pages) and a `PagedBatch` (which pages and
how many positions each sequence has, and which rows of the step are its new
"nodes").  One node per sequence is plain decoding, `parents=None` a chunk of
a prompt, and parents a tree (or forest) of drafts.  The rules of each call
are those of include/affon_b200.h; the lengths, page table and indices are
device tensors that the kernels read when they run, so a captured graph can be
replayed on changed contents.  What the kernels find wrong with them is
reported by `Session.synchronize()`.

Calls run on the Session's device and on torch's current stream of it.
`tree_attention` and `tree_accept` use the Session's workspace: such calls of one
Session (and graphs captured from them) must not run at the same time on two
streams; make a Session per stream for that.  The reference has no counterpart: its
models use a fixed-capacity cache.
"""
import ctypes

import torch

from . import _lib
from .core import AffonError, check

_FLOAT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_BF16 = (torch.bfloat16,)


def _check(cond, message, code="invalid_shape"):
    if not cond:
        raise AffonError(code, message)


def _tensor(session, t, name, dtypes, dim, dense=False):
    """t must be a tensor of the Session's device with one of `dtypes` and `dim` axes, the last one dense."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    _check(t.device == session.torch_device, f"{name} is on {t.device}, Session on {session.torch_device}",
           "device_mismatch")
    _check(t.dtype in dtypes, f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}, not {t.dtype}",
           "invalid_dtype")
    _check(t.dim() == dim, f"{name} must have {dim} axes, not {t.dim()}")
    _check(t.is_contiguous() if dense else t.stride(-1) == 1 or t.shape[-1] == 1,
           f"{name} must be {'contiguous' if dense else 'dense along its last axis'}")
    return t


def _ints(session, t, name, shape):
    if _dense(t, torch.int32, shape, session.torch_device):
        return t
    _tensor(session, t, name, (torch.int32,), len(shape), dense=True)
    _check(tuple(t.shape) == shape, f"{name} must have shape {list(shape)}, not {list(t.shape)}")
    return t


def _dense(t, dtype, shape, device):
    """Whether t needs no closer look (the checks of a decode step's calls are most of their host time)."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device
            and t.is_contiguous())


def _rows_of(session, t, name, dtypes, rows, cols, more=False):
    """A [rows, cols] tensor, dense along its rows (`more`: with further columns); returns the elements between rows."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and _dense(t, t.dtype, (rows, cols), session.torch_device):
        return cols
    _tensor(session, t, name, dtypes, 2)
    _check(t.shape[0] == rows and (t.shape[1] == cols or more and t.shape[1] > cols),
           f"{name} must be [{rows}, {cols}{' or more' if more else ''}], not {list(t.shape)}")
    return t.stride(0) if rows > 1 else cols  # a lone row's stride is never used


def _ready(session):
    if session.disposed:
        raise AffonError("invalid_arg", "Session has been disposed")
    session.bind_stream()
    return _lib.lib()


def _tables(session, cos, sin, half):
    """Rotation tables [positions, half]; returns the positions."""
    for t, name in ((cos, "cos"), (sin, "sin")):
        if not (isinstance(t, torch.Tensor) and _dense(t, torch.float32, t.shape, session.torch_device) and t.dim() == 2):
            _tensor(session, t, name, (torch.float32,), 2, dense=True)
    _check(cos.shape == sin.shape and cos.shape[1] == half, f"cos and sin must be [positions, {half}]")
    return cos.shape[0]


class PagedCache:
    """Key and value pools, bf16 [layers, pages, kv_heads, page_size, head_dim] (or without the layer axis).

    The axes may lie in any order in memory as long as head_dim is dense and
    both pools have the same strides, so a contiguous [batch, kv_heads,
    capacity, head_dim] cache is one too: `PagedCache.from_contiguous`."""

    def __init__(self, session, k, v):
        bf16 = (torch.bfloat16,)
        dim = k.dim() if isinstance(k, torch.Tensor) and k.dim() == 4 else 5
        _tensor(session, k, "k", bf16, dim)
        _tensor(session, v, "v", bf16, dim)
        _check(k.shape == v.shape and k.stride() == v.stride(), "k and v must have the same shape and strides")
        _check(k.numel() > 0, "a cache needs at least one page")
        self.session = session
        self.k, self.v = (k, v) if dim == 5 else (k[None], v[None])
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = self.k.shape
        st = self.k.stride()
        self.layer_stride = st[0] if self.layers > 1 else 0
        # A stride of a one-element axis is never used.
        self.strides = (st[1] if self.pages > 1 else self.head_dim, st[2] if self.kv_heads > 1 else self.head_dim,
                        st[3])
        esz = self.k.element_size()
        base = (self.k.data_ptr(), self.v.data_ptr())
        self._ptrs = [tuple(ctypes.c_void_p(b + i * self.layer_stride * esz) for b in base)
                      for i in range(self.layers)]

    @classmethod
    def empty(cls, session, layers, pages, kv_heads, page_size, head_dim):
        """New pools (zeros) in the layout the kernels like best: a page's positions of one head are contiguous."""
        shape = (layers, pages, kv_heads, page_size, head_dim)
        make = lambda: torch.zeros(shape, dtype=torch.bfloat16, device=session.torch_device)
        return cls(session, make(), make())

    @classmethod
    def from_contiguous(cls, session, k, v, page_size):
        """A view of contiguous caches [layers, batch, kv_heads, capacity, head_dim] as pages of `page_size`
        positions, and the page table [batch, capacity/page_size] that names them in order."""
        for t, name in ((k, "k"), (v, "v")):
            _tensor(session, t, name, (torch.bfloat16,), 5, dense=True)
        layers, batch, heads, cap, hd = k.shape
        _check(page_size > 0 and cap % page_size == 0, "the capacity must be a multiple of the page size")
        per = cap // page_size
        # Page (b, head 0, j) starts (b*heads*per + j) pages of page_size*hd elements into the layer; a head further
        # is cap*hd on.  Pages that start in another head's run are not in the table.
        shape = (layers, batch * heads * per - (heads - 1) * per, heads, page_size, hd)
        st = (batch * heads * cap * hd, page_size * hd, cap * hd, hd, 1)
        cache = cls(session, k.as_strided(shape, st), v.as_strided(shape, st))
        table = (torch.arange(batch, device=k.device, dtype=torch.int32)[:, None] * (heads * per)
                 + torch.arange(per, device=k.device, dtype=torch.int32)[None, :])
        return cache, table.contiguous()

    def layer(self, index):
        """Base pointers of one layer's pools."""
        _check(isinstance(index, int) and 0 <= index < self.layers, f"layer {index} of {self.layers}", "invalid_arg")
        return self._ptrs[index]


class PagedBatch:
    """The sequences of a step: page_table int32 [seqs, pages per sequence], ctx_lens int32 [seqs] (cached
    positions), cu_nodes int32 [seqs+1] (first row of each sequence's nodes), `rows` rows in the step's buffers and
    at most `max_nodes` nodes per sequence.  `cache` gives the pools; a batch that only plans may give page_size and
    pages instead."""

    def __init__(self, session, page_table, ctx_lens, cu_nodes, rows, max_nodes, cache=None, page_size=None,
                 pages=None):
        _tensor(session, page_table, "page_table", (torch.int32,), 2, dense=True)
        seqs, per = page_table.shape
        _check(seqs >= 1 and per >= 1, "page_table must not be empty")
        _ints(session, ctx_lens, "ctx_lens", (seqs,))
        _ints(session, cu_nodes, "cu_nodes", (seqs + 1,))
        _check(isinstance(rows, int) and 0 <= rows < 2 ** 31, "rows must be a whole number from 0")
        _check(isinstance(max_nodes, int) and 1 <= max_nodes <= _lib.MAX_TREE_NODES,
               f"max_nodes must be 1 to {_lib.MAX_TREE_NODES}")
        alone = isinstance(page_size, int) and isinstance(pages, int)
        _check(alone if cache is None else page_size is None and pages is None,
               "give a cache, or page_size and pages", "invalid_arg")
        if cache is not None:
            _check(isinstance(cache, PagedCache) and cache.session is session, "cache must be a PagedCache of the Session",
                   "invalid_arg")
        self.session, self.cache = session, cache
        self.page_table, self.ctx_lens, self.cu_nodes = page_table, ctx_lens, cu_nodes
        self.seqs, self.rows, self.max_nodes = seqs, rows, max_nodes
        self.mask_words = -(-max_nodes // 32)
        hd = cache.head_dim if cache else 64
        strides = cache.strides if cache else (hd, hd, hd)
        d = self.desc = _lib.PagedDesc(
            ctypes.sizeof(_lib.PagedDesc), seqs, rows, max_nodes, cache.kv_heads if cache else 1, hd,
            cache.page_size if cache else page_size, self.mask_words, cache.pages if cache else pages, *strides, per)
        check(_lib.lib().affon_b200_paged_validate(ctypes.byref(d)), "PagedBatch")
        self._desc = ctypes.byref(d)
        self._descs = {}
        self._step = tuple(ctypes.c_void_p(t.data_ptr()) for t in (cu_nodes, ctx_lens, page_table))

    def _memo(self, desc, *fields):
        """A reference to the call descriptor with these fields (a step's calls repeat the same few)."""
        key = (desc,) + fields
        ref = self._descs.get(key)
        if ref is None:
            if len(self._descs) >= 64:
                self._descs.clear()
            ref = self._descs[key] = ctypes.byref(desc(ctypes.sizeof(desc), *fields))
        return ref

    def _pools(self, layer):
        _check(self.cache is not None, "the batch was made without a cache", "invalid_arg")
        return self.cache.layer(layer)


class TreePlan:
    """positions int32 [rows], slots int32 [rows] (-1: padding), mask int32 words [rows, mask_words] (None: chains)."""

    __slots__ = ("positions", "slots", "mask")

    def __init__(self, positions, slots, mask=None):
        self.positions, self.slots, self.mask = positions, slots, mask


def plan(batch, parents=None, out=None):
    """Rotation positions, cache slots and ancestor masks of the step's rows.

    parents: int32 [rows], the index within its sequence of the node that each
    node continues (negative: a root), or None when every node continues the
    one before it.  `out`: a TreePlan whose tensors are overwritten."""
    s = batch.session
    if parents is not None:
        _ints(s, parents, "parents", (batch.rows,))
    if out is None:
        new = batch.ctx_lens.new_empty
        out = TreePlan(new(batch.rows), new(batch.rows), new((batch.rows, batch.mask_words)))
    else:
        _check_plan(batch, out)
        _check(out.mask is not None, "plan needs a mask to write", "invalid_arg")
    L = _ready(s)
    cu, ctx, table = batch._step
    check(L.affon_b200_paged_plan(s._ctx, batch._desc, cu, None if parents is None else parents.data_ptr(), ctx, table,
                                  out.positions.data_ptr(), out.slots.data_ptr(), out.mask.data_ptr()))
    return out


def _check_plan(batch, p):
    _ints(batch.session, p.positions, "positions", (batch.rows,))
    _ints(batch.session, p.slots, "slots", (batch.rows,))
    if p.mask is not None:
        _ints(batch.session, p.mask, "mask", (batch.rows, batch.mask_words))


def append(batch, plan, qkv, q_heads, cos=None, sin=None, layer=0, rope="half", q_out=None):
    """Rotate the step's queries and keys and append keys and values to the cache; returns the rotated queries.

    qkv: f32 or bf16 [rows, (q_heads + 2*kv_heads)*head_dim], queries, keys
    and values in that order (more columns may follow).  cos, sin: f32
    [positions, head_dim/2].  rope: "half" (pairs d, d + head_dim/2),
    "interleaved" (pairs 2d, 2d + 1) or "none".  Padding rows of q_out are not
    written."""
    s, c = batch.session, batch.cache
    k, v = batch._pools(layer)
    hd, kv, rows = c.head_dim, c.kv_heads, batch.rows
    _check(isinstance(q_heads, int) and q_heads >= 0, "q_heads must be a whole number")
    ld = _rows_of(s, qkv, "qkv", _FLOAT, rows, (q_heads + 2 * kv) * hd, more=True)
    _ints(s, plan.slots, "slots", (rows,))
    mode = _lib.ROPE.get(rope)
    _check(mode is not None, "rope must be half, interleaved or none", "invalid_arg")
    length = 0
    if mode:
        _ints(s, plan.positions, "positions", (rows,))
        length = _tables(s, cos, sin, hd // 2)
    if q_out is None:
        q_out = torch.empty((rows, q_heads * hd), dtype=torch.bfloat16, device=s.torch_device)
    ld_q = _rows_of(s, q_out, "q_out", _BF16, rows, q_heads * hd)
    d = batch._memo(_lib.AppendDesc, _FLOAT[qkv.dtype], mode, q_heads, 0, q_heads * hd, (q_heads + kv) * hd, length, ld,
                    ld_q)
    L = _ready(s)
    check(L.affon_b200_paged_append(s._ctx, batch._desc, d, qkv.data_ptr(), cos.data_ptr() if mode else None,
                                    sin.data_ptr() if mode else None, plan.positions.data_ptr() if mode else None,
                                    plan.slots.data_ptr(), q_out.data_ptr(), k, v))
    return q_out


def tree_attention(batch, plan, q, q_heads, layer=0, scale=None, out=None, pair_order=False):
    """Attention of the step's nodes over their sequences' caches; returns bf16 [rows, q_heads*head_dim].

    q: rotated queries, bf16 [rows, q_heads*head_dim].  plan.mask (or None for
    chains) says which drafted nodes each node sees; scale defaults to
    head_dim**-0.5.  Padding rows of `out` are not written.  pair_order writes the 4-bit decode qmv's column order."""
    s, c = batch.session, batch.cache
    k, v = batch._pools(layer)
    _check(isinstance(q_heads, int) and q_heads > 0, "q_heads must be a positive whole number")
    cols = q_heads * c.head_dim
    ld_q = _rows_of(s, q, "q", _BF16, batch.rows, cols)
    mask = plan.mask if plan is not None else None
    if mask is not None:
        _ints(s, mask, "mask", (batch.rows, batch.mask_words))
    if out is None:
        out = torch.empty((batch.rows, cols), dtype=torch.bfloat16, device=s.torch_device)
    ld_out = _rows_of(s, out, "out", _BF16, batch.rows, cols)
    d = batch._memo(_lib.TreeAttnDesc, q_heads, c.head_dim ** -0.5 if scale is None else float(scale),
                    1 if pair_order else 0, ld_q, ld_out)
    L = _ready(s)
    cu, ctx, table = batch._step
    check(L.affon_b200_tree_attention(s._ctx, batch._desc, d, q.data_ptr(), cu, ctx, table,
                                      None if mask is None else mask.data_ptr(), k, v, out.data_ptr()))
    return out


class Accepted:
    """counts int32 [seqs], path int32 [seqs, max_nodes] (-1 behind the last), next_tokens int32 [seqs], lens int32
    [seqs] (cached positions after the step)."""

    __slots__ = ("counts", "path", "next_tokens", "lens")

    def __init__(self, counts, path, next_tokens, lens):
        self.counts, self.path, self.next_tokens, self.lens = counts, path, next_tokens, lens


def tree_accept(batch, parents, tokens, predicted, out=None):
    """Walk every drafted tree along the model's greedy predictions and move the accepted nodes' keys and values
    together in all layers of the cache.

    tokens, predicted: int32 [rows], each node's token and the model's next
    token after it.  Node 0 of a sequence is always accepted.  `out`: an
    Accepted whose tensors are overwritten; its lens may be the batch's
    ctx_lens, which then advance in place."""
    s, c = batch.session, batch.cache
    _check(c is not None, "the batch was made without a cache", "invalid_arg")
    if parents is not None:
        _ints(s, parents, "parents", (batch.rows,))
    _ints(s, tokens, "tokens", (batch.rows,))
    _ints(s, predicted, "predicted", (batch.rows,))
    if out is None:
        new, seqs = batch.ctx_lens.new_empty, batch.seqs
        out = Accepted(new(seqs), new((seqs, batch.max_nodes)), new(seqs), new(seqs))
    else:
        _ints(s, out.counts, "counts", (batch.seqs,))
        _ints(s, out.path, "path", (batch.seqs, batch.max_nodes))
        _ints(s, out.next_tokens, "next_tokens", (batch.seqs,))
        _ints(s, out.lens, "lens", (batch.seqs,))
    L = _ready(s)
    cu, ctx, table = batch._step
    k, v = c.layer(0)
    check(L.affon_b200_tree_accept(s._ctx, batch._desc, c.layers, c.layer_stride, cu,
                                   None if parents is None else parents.data_ptr(), tokens.data_ptr(),
                                   predicted.data_ptr(), table, ctx, k, v, out.counts.data_ptr(), out.path.data_ptr(),
                                   batch.max_nodes, out.next_tokens.data_ptr(), out.lens.data_ptr()))
    return out
