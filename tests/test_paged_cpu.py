"""The paged cache's host side without a GPU: descriptor layouts and rules,
refusals of the Python calls, views of contiguous caches, and the plain
restatements that the GPU tests compare with."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import paged_ref as ref
from affon_b200 import _lib, paged
from affon_b200.core import AffonError

HOST = SimpleNamespace(torch_device=torch.device("cpu"), disposed=False)


def desc(**kw):
    d = dict(seqs=2, rows=5, max_nodes=4, kv_heads=2, head_dim=128, page_size=16, mask_words=1, pages=9,
             page_stride=4096, head_stride=2048, token_stride=128, ld_table=3)
    d.update(kw)
    return _lib.PagedDesc(ctypes.sizeof(_lib.PagedDesc), *[d[k] for k, _ in _lib.PagedDesc._fields_[1:]])


def test_struct_layouts_match_header():
    assert ctypes.sizeof(_lib.PagedDesc) == 72 and _lib.PagedDesc.pages.offset == 32
    assert ctypes.sizeof(_lib.AppendDesc) == 48 and _lib.AppendDesc.ld_qkv.offset == 32
    assert ctypes.sizeof(_lib.TreeAttnDesc) == 32 and _lib.TreeAttnDesc.ld_q.offset == 16


@pytest.mark.parametrize("kw", [dict(), dict(head_dim=64), dict(page_size=256), dict(rows=0), dict(max_nodes=256, mask_words=8),
                                dict(kv_heads=1, head_stride=0), dict(pages=1, page_stride=3)])
def test_descriptor_accepts(kw):
    assert _lib.lib().affon_b200_paged_validate(ctypes.byref(desc(**kw))) == _lib.OK, _lib.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(seqs=0), _lib.INVALID_SHAPE), (dict(seqs=65537), _lib.INVALID_SHAPE), (dict(rows=-1), _lib.INVALID_SHAPE),
    (dict(max_nodes=0), _lib.INVALID_SHAPE), (dict(max_nodes=257, mask_words=9), _lib.INVALID_SHAPE),
    (dict(max_nodes=33), _lib.INVALID_SHAPE), (dict(mask_words=9), _lib.INVALID_SHAPE),
    (dict(kv_heads=0), _lib.INVALID_SHAPE), (dict(head_dim=96), _lib.UNSUPPORTED),
    (dict(page_size=24), _lib.UNSUPPORTED), (dict(page_size=512), _lib.UNSUPPORTED), (dict(page_size=0), _lib.UNSUPPORTED),
    (dict(pages=0), _lib.INVALID_SHAPE), (dict(pages=1 << 27), _lib.INVALID_SHAPE),
    (dict(ld_table=0), _lib.INVALID_SHAPE), (dict(ld_table=1 << 26), _lib.INVALID_SHAPE),
    (dict(token_stride=64), _lib.INVALID_SHAPE), (dict(token_stride=132), _lib.INVALID_SHAPE),
    (dict(head_stride=0), _lib.INVALID_SHAPE), (dict(page_stride=-4096), _lib.INVALID_SHAPE),
    (dict(page_stride=1 << 39), _lib.INVALID_SHAPE)])
def test_descriptor_refusals(kw, status):
    assert _lib.lib().affon_b200_paged_validate(ctypes.byref(desc(**kw))) == status
    assert _lib.last_error().startswith("paged:")


def test_bad_struct_size_and_null_context_are_refused():
    L = _lib.lib()
    d = desc()
    d.struct_size = 8
    assert L.affon_b200_paged_validate(ctypes.byref(d)) == _lib.INVALID_ARG
    assert L.affon_b200_paged_validate(None) == _lib.INVALID_ARG
    p = ctypes.byref(desc())
    assert L.affon_b200_paged_plan(None, p, *[None] * 7) == _lib.INVALID_ARG
    assert L.affon_b200_paged_append(None, p, None, *[None] * 8) == _lib.INVALID_ARG
    assert L.affon_b200_tree_attention(None, p, None, *[None] * 8) == _lib.INVALID_ARG
    assert L.affon_b200_tree_accept(None, p, 1, 0, *[None] * 10, 4, None, None) == _lib.INVALID_ARG


def cache(heads=2, page=16, hd=64, pages=5, layers=1):
    z = lambda: torch.zeros((layers, pages, heads, page, hd), dtype=torch.bfloat16)
    return paged.PagedCache(HOST, z(), z())


def batch(c=None, rows=5, max_nodes=4, **kw):
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)
    args = dict(page_table=torch.zeros((2, 3), dtype=torch.int32), ctx_lens=i32(3, 4), cu_nodes=i32(0, 2, 5))
    args.update({k: kw.pop(k) for k in list(kw) if k in args})
    return paged.PagedBatch(HOST, args["page_table"], args["ctx_lens"], args["cu_nodes"], rows, max_nodes,
                            cache=c if c is not None else cache(), **kw)


def refused(code, fn, *args, **kw):
    with pytest.raises(AffonError) as err:
        fn(*args, **kw)
    assert err.value.code == code, err.value


def test_cache_and_batch_refusals():
    z = torch.zeros((5, 2, 16, 64), dtype=torch.bfloat16)
    refused("invalid_dtype", paged.PagedCache, HOST, z.float(), z.float())
    refused("invalid_shape", paged.PagedCache, HOST, z, z[:4])
    refused("invalid_shape", paged.PagedCache, HOST, z.transpose(-1, -2), z.transpose(-1, -2))
    refused("invalid_shape", paged.PagedCache, HOST, z[:0], z[:0])
    refused("device_mismatch", paged.PagedCache, SimpleNamespace(torch_device=torch.device("cuda", 0)), z, z)
    with pytest.raises(TypeError):
        paged.PagedCache(HOST, None, z)
    refused("invalid_dtype", batch, ctx_lens=torch.zeros(2, dtype=torch.int64))
    refused("invalid_shape", batch, ctx_lens=torch.zeros(3, dtype=torch.int32))
    refused("invalid_shape", batch, page_table=torch.zeros((2, 6), dtype=torch.int32)[:, ::2])
    refused("invalid_shape", batch, max_nodes=257)
    refused("invalid_shape", batch, rows=-1)
    refused("unsupported_lowering", batch, cache(hd=80))
    refused("unsupported_lowering", batch, cache(page=24))
    refused("invalid_arg", batch, page_size=16)
    # a head stride that is no multiple of 16 bytes
    odd = torch.zeros(20000, dtype=torch.bfloat16).as_strided((5, 2, 16, 64), (2100, 1028, 64, 1))
    refused("invalid_shape", batch, paged.PagedCache(HOST, odd, odd))


def test_call_refusals():
    b = batch()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    p = paged.TreePlan(i32(5), i32(5), i32(5, 1))
    refused("invalid_shape", paged.plan, b, i32(4))
    refused("invalid_dtype", paged.plan, b, torch.zeros(5))
    refused("invalid_arg", paged.plan, b, out=paged.TreePlan(i32(5), i32(5)))
    cos = torch.zeros((9, 32))
    refused("invalid_shape", paged.append, b, p, bf(5, 511), 4, cos, cos)
    refused("invalid_shape", paged.append, b, p, bf(4, 512), 4, cos, cos)
    refused("invalid_dtype", paged.append, b, p, torch.zeros((5, 512), dtype=torch.float16), 4, cos, cos)
    refused("invalid_shape", paged.append, b, p, bf(5, 512), 4, cos, cos[:, :16])
    refused("invalid_arg", paged.append, b, p, bf(5, 512), 4, cos, cos, rope="partial")
    refused("invalid_arg", paged.append, b, p, bf(5, 512), 4, cos, cos, layer=1)
    with pytest.raises(TypeError):
        paged.append(b, p, bf(5, 512), 4)          # tables are missing
    refused("invalid_shape", paged.tree_attention, b, p, bf(5, 255), 4)
    refused("invalid_shape", paged.tree_attention, b, paged.TreePlan(None, None, i32(5, 2)), bf(5, 256), 4)
    refused("invalid_dtype", paged.tree_attention, b, p, torch.zeros((5, 256)), 4)
    refused("invalid_shape", paged.tree_attention, b, p, bf(5, 256), 4, out=bf(4, 256))
    refused("invalid_shape", paged.tree_accept, b, i32(5), i32(4), i32(5))
    refused("invalid_shape", paged.tree_accept, b, i32(5), i32(5), i32(5),
            out=paged.Accepted(i32(2), i32(2, 3), i32(2), i32(2)))
    only = paged.PagedBatch(HOST, i32(2, 3), i32(2), i32(3), 5, 4, page_size=16, pages=7)
    refused("invalid_arg", paged.tree_attention, only, p, bf(5, 256), 4)


def test_contiguous_cache_is_a_paged_one():
    layers, b, heads, cap, hd, page = 2, 3, 2, 64, 64, 16
    k = torch.arange(layers * b * heads * cap * hd).reshape(layers, b, heads, cap, hd).to(torch.bfloat16)
    v = k.clone()
    c, table = paged.PagedCache.from_contiguous(HOST, k, v, page)
    assert tuple(table.shape) == (b, cap // page) and int(table.max()) < c.pages
    for s in range(b):
        for j in range(cap // page):
            assert torch.equal(c.k[:, int(table[s, j])], k[:, s, :, j * page:(j + 1) * page])
    assert c.k.data_ptr() == k.data_ptr()
    refused("invalid_shape", paged.PagedCache.from_contiguous, HOST, k, v, 48)


def test_reference_attention_is_a_softmax_of_what_is_seen():
    """The restatement against torch's own softmax on a dense case, and its bound against a bf16 rounding of the
    probabilities."""
    st = ref.Step([5, 0], [3, 2], 16, seed=1)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((st.pages, 2, 16, 64), generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((5, 256), generator=g).to(torch.bfloat16)
    out, bound = ref.attention(st, q, k, v, 4, 0.125)
    for s in range(2):
        a, n, c = int(st.cu[s]), st.nodes[s], st.ctx[s]
        see = torch.from_numpy(ref.ancestors(st.parents[s]))
        for h in range(4):
            keys, vals = ref.gather(st, k, s, c + n)[h // 2], ref.gather(st, v, s, c + n)[h // 2]
            z = q[a:a + n, h * 64:(h + 1) * 64].double() @ keys.T * 0.125
            z[:, c:][~see] = -torch.inf
            p = torch.softmax(z, -1)
            want = p @ vals
            assert torch.allclose(out[a:a + n, h * 64:(h + 1) * 64], want, atol=1e-12)
            pr = torch.exp(z - z.amax(-1, keepdim=True)).to(torch.bfloat16).double()
            got = (pr @ vals / pr.sum(-1, keepdim=True)).to(torch.bfloat16).double()
            assert ((got - want).abs() <= bound[a:a + n, h * 64:(h + 1) * 64]).all()


def test_reference_accept_walks_the_lowest_fitting_child():
    st = ref.Step([7], [6], 16, parents=[np.array([-1, 0, 0, 2, 2, 4], dtype=np.int32)])
    tokens = np.array([9, 1, 2, 3, 3, 4])
    predicted = np.array([2, 0, 3, 7, 4, 5])
    counts, path, nxt, lens = ref.accept(st, tokens, predicted)
    assert counts.tolist() == [3] and path[0].tolist() == [0, 2, 3, -1, -1, -1]
    assert nxt.tolist() == [7] and lens.tolist() == [10]


def test_a_session_used_by_two_streams_keeps_neither(monkeypatch):
    """Another thread's call may come between a call's two steps, to read its stream and to set the context's: the
    next call sets its own again."""
    from affon_b200 import core
    seen = []
    streams = iter([1, 2, 1])
    s = object.__new__(core.Session)
    s._ctx, s.ordinal, s.disposed = None, 0, False

    def set_stream(ctx, raw):
        seen.append(raw)
        if len(seen) == 1:
            s.bind_stream()                                  # the other thread's whole call
        return _lib.OK
    monkeypatch.setattr(core._lib, "lib", lambda: SimpleNamespace(affon_b200_ctx_set_stream=set_stream))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda ordinal: next(streams), raising=False)
    s.bind_stream()
    s.bind_stream()
    assert seen == [1, 2, 1]


def test_a_context_without_a_workspace_is_refused():
    """What a failed growth of the workspace leaves: the kernels' status word and counters have no place."""
    L = _lib.lib()
    ctx = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)  # a context of zeros
    d, some = desc(), 4096                                   # buffers that are never read
    p = ctypes.byref(d)
    a = ctypes.byref(_lib.AppendDesc(ctypes.sizeof(_lib.AppendDesc), _lib.BF16, 0, 0, 0, 0, 256, 0, 512, 0))
    t = ctypes.byref(_lib.TreeAttnDesc(ctypes.sizeof(_lib.TreeAttnDesc), 4, 1.0, 0, 512, 512))
    for status in (L.affon_b200_paged_plan(ctx, p, *[some] * 7),
                   L.affon_b200_paged_append(ctx, p, a, *[some] * 8),
                   L.affon_b200_tree_attention(ctx, p, t, *[some] * 8),
                   L.affon_b200_tree_accept(ctx, p, 1, 0, *[some] * 10, 4, some, some)):
        assert status == _lib.UNSUPPORTED and "workspace" in _lib.last_error()


def test_a_lone_row_needs_no_aligned_stride():
    """The stride of a one-element axis is never used: one row may have any number of further columns."""
    bf = torch.zeros((1, 517), dtype=torch.bfloat16)
    assert paged._rows_of(HOST, bf, "qkv", (torch.bfloat16,), 1, 512, more=True) == 512
    assert paged._rows_of(HOST, bf[:, :512], "q", (torch.bfloat16,), 1, 512) == 512
    two = torch.zeros((2, 520), dtype=torch.bfloat16)
    assert paged._rows_of(HOST, two[:, :512], "q", (torch.bfloat16,), 2, 512) == 520
    assert paged._rows_of(HOST, two, "qkv", (torch.bfloat16,), 2, 512, more=True) == 520
