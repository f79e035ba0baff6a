"""The paged-cache operators on the GPU against their 64-bit restatements."""
import math

import numpy as np
import pytest
import torch

import paged_ref as ref
from affon_b200 import Session, paged
from affon_b200.core import AffonError

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def sess():
    with Session("cuda:0") as s:
        yield s


def dev(a):
    return torch.as_tensor(a).to(DEV)


def pools(st, heads, hd, seed, layers=1, nhd=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        t = torch.randn((layers, st.pages, heads, st.page, hd), generator=g).to(torch.bfloat16)
        # nhd: the heads of a position lie together
        out.append(t.transpose(2, 3).contiguous().to(DEV).transpose(2, 3) if nhd else t.to(DEV))
    return out


def batch(sess, st, k, v):
    c = paged.PagedCache(sess, k, v)
    return paged.PagedBatch(sess, dev(st.table), dev(np.asarray(st.ctx, dtype=np.int32)), dev(st.cu), st.rows,
                            st.max_nodes, cache=c)


def tables(rows, hd):
    inv = 500000.0 ** (-np.arange(hd // 2) * 2.0 / hd)
    ang = np.arange(rows)[:, None] * inv[None]
    return torch.from_numpy(np.cos(ang).astype(np.float32)), torch.from_numpy(np.sin(ang).astype(np.float32))


# ------------------------------------------------------------------- plan
@pytest.mark.parametrize("ctx,nodes,page,pad", [([0], [1], 16, 0), ([333], [13], 16, 3), ([5, 0, 70, 31], [33, 0, 64, 1], 32, 7),
                                                ([100, 7], [256, 255], 128, 0), ([15, 16, 17], [1, 1, 1], 16, 2)])
@pytest.mark.parametrize("kind", ["forest", "chain", "none"])
def test_plan_matches(sess, ctx, nodes, page, pad, kind):
    st = ref.Step(ctx, nodes, page, seed=len(nodes) + page, pad=pad, parents=None if kind == "forest" else "chain",
                  roots=kind == "forest")
    b = paged.PagedBatch(sess, dev(st.table), dev(np.asarray(ctx, dtype=np.int32)), dev(st.cu), st.rows, st.max_nodes,
                         page_size=page, pages=st.pages)
    p = paged.plan(b, None if kind == "none" else dev(st.flat_parents()))
    sess.synchronize()
    for got, want in zip((p.positions, p.slots, p.mask), st.plan()):
        assert torch.equal(got.cpu(), torch.from_numpy(want))


def test_plan_reports_bad_parents_pages_and_lengths(sess):
    st = ref.Step([5, 9, 3], [3, 4, 2], 16, parents="chain")
    make = lambda ctx=None, cu=None, table=None: paged.PagedBatch(
        sess, dev(st.table if table is None else table),
        dev(np.asarray(st.ctx if ctx is None else ctx, dtype=np.int32)),
        dev(st.cu if cu is None else np.asarray(cu, dtype=np.int32)), st.rows, st.max_nodes, page_size=16,
        pages=st.pages)
    want = [torch.from_numpy(a) for a in st.plan()]

    def run(b, parents):
        p = paged.plan(b, dev(parents))
        with pytest.raises(AffonError) as err:
            sess.synchronize()
        assert err.value.code == "invalid_arg"
        return p
    par = st.flat_parents().copy()
    par[4] = 3                                   # a parent behind its child: the node becomes a root
    p = run(make(), par)
    assert int(p.positions[4]) == 9 and int(p.mask[4, 0]) == 2
    assert torch.equal(p.slots.cpu(), want[1])
    # lengths that do not fit: the sequence's rows become padding, the others keep their slots
    for kw, lost in ((dict(ctx=[5, 9, -1]), [7, 8]), (dict(ctx=[5, 9, 2 ** 31 - 1]), [7, 8]),
                     (dict(cu=[0, 3, 7, 10]), [7, 8]), (dict(cu=[0, 3, 2, 2]), [2, 3, 4, 5, 6, 7, 8])):
        p = run(make(**kw), st.flat_parents())
        keep = [r for r in range(st.rows) if r not in lost and not (r == 2 and 2 in lost)]
        assert torch.equal(p.slots[keep].cpu(), want[1][keep])
        assert all(int(p.slots[r]) == -1 for r in lost if r != 2)
    table = st.table.copy()
    table[1, 0] = st.pages
    p = run(make(table=table), st.flat_parents())
    assert p.slots[3:7].cpu().tolist() == [-1] * 4 and torch.equal(p.slots[7:].cpu(), want[1][7:])
    paged.plan(make(), dev(st.flat_parents()))
    sess.synchronize()                           # the Session stays usable


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rope", ["half", "interleaved", "none"])
@pytest.mark.parametrize("ctx,nodes,page,heads,group,hd,nhd", [
    ([333], [1], 16, 8, 4, 128, False), ([0, 40, 7], [5, 0, 33], 32, 3, 7, 64, True), ([9, 200], [17, 64], 128, 1, 1, 128, True),
    ([1, 2, 3, 4], [2, 2, 2, 3], 16, 2, 16, 64, False)])
def test_append_matches(sess, dtype, rope, ctx, nodes, page, heads, group, hd, nhd):
    st = ref.Step(ctx, nodes, page, seed=3, pad=2)
    k, v = pools(st, heads, hd, 4, layers=2, nhd=nhd)
    k0, v0 = k.cpu(), v.cpu()
    b = batch(sess, st, k, v)
    qh = heads * group
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((st.rows, (qh + 2 * heads) * hd + 16), generator=g).to(dtype)
    qkv = dev(wide)[:, :-16]                     # rows that are not dense
    cos, sin = tables(max(ctx) + max(nodes), hd)
    pos, slots, _ = st.plan()
    q_out = torch.full((st.rows, qh * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    args = (dev(cos), dev(sin)) if rope != "none" else ()
    got = paged.append(b, paged.TreePlan(dev(pos), dev(slots)), qkv, qh, *args, layer=1, rope=rope, q_out=q_out)
    sess.synchronize()
    assert got is q_out
    real = torch.from_numpy(slots) >= 0
    x = wide[:, :-16].double().reshape(st.rows, qh + 2 * heads, hd)
    at = torch.from_numpy(pos).long()
    if rope == "none":
        y, mag = x.clone(), torch.zeros_like(x)
    else:
        y = torch.cat([ref.rotate(x[:, :qh + heads], cos.double()[at], sin.double()[at], rope), x[:, qh + heads:]], 1)
        mag = torch.cat([ref.rotate(x[:, :qh + heads].abs(), cos.double()[at].abs(), -sin.double()[at].abs(), rope).abs()
                         + ref.rotate(x[:, :qh + heads].abs(), cos.double()[at].abs(), sin.double()[at].abs(), rope).abs(),
                         torch.zeros_like(x[:, qh + heads:])], 1)
    # two f32 products and their sum (2^-23 of the magnitudes), one rounding to bf16 (half a step)
    tol = 2.0 ** -8 * y.abs() + 2.0 ** -22 * mag
    q = q_out.cpu().double().reshape(st.rows, qh, hd)
    assert ((q - y[:, :qh]).abs() <= tol[:, :qh])[real].all()
    assert (q[~real] == 7.0).all()               # padding rows stay
    kw, vw = k0.clone().double(), v0.clone()
    kt = torch.zeros_like(kw)
    for r in torch.nonzero(real).flatten().tolist():
        pg, off = slots[r] // page, slots[r] % page
        kw[1, pg, :, off], kt[1, pg, :, off] = y[r, qh:qh + heads], tol[r, qh:qh + heads]
        vw[1, pg, :, off] = x[r, qh + heads:].to(dtype).to(torch.bfloat16)
    assert ((k.cpu().double() - kw).abs() <= kt).all()     # every other element is exactly as it was
    assert torch.equal(v.cpu(), vw)


def test_append_without_queries_and_bad_rows(sess):
    st = ref.Step([3], [5], 16, parents="chain")
    k, v = pools(st, 2, 64, 1)
    k0 = k.clone()
    b = batch(sess, st, k, v)
    pos, slots, _ = st.plan()
    cos, sin = tables(8, 64)
    qkv = torch.randn((5, 4 * 64), device=DEV)
    empty = paged.append(b, paged.TreePlan(dev(pos), dev(slots)), qkv, 0, dev(cos), dev(sin))
    sess.synchronize()
    assert tuple(empty.shape) == (5, 0) and not torch.equal(k, k0)
    good = k.clone()
    for bad_pos, bad_slot in ((8, None), (-1, None), (None, -2), (None, st.pages * 16)):
        p2, s2 = pos.copy(), slots.copy()
        if bad_pos is not None:
            p2[2] = bad_pos
        if bad_slot is not None:
            s2[2] = bad_slot
        k.copy_(k0)
        paged.append(b, paged.TreePlan(dev(p2), dev(s2)), qkv, 0, dev(cos), dev(sin))
        with pytest.raises(AffonError) as err:
            sess.synchronize()
        assert err.value.code == "invalid_arg"
        want = good.clone()
        want[0, slots[2] // 16, :, slots[2] % 16] = k0[0, slots[2] // 16, :, slots[2] % 16]
        assert torch.equal(k, want)              # the bad row alone is skipped


# -------------------------------------------------------------- attention
def run_attention(sess, st, heads, group, hd, seed=0, nhd=False, scale=None, mask="plan", sharp=2.0, seen=None,
                  pair=False):
    k, v = pools(st, heads, hd, seed, nhd=nhd)
    qh = heads * group
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((st.rows, qh * hd), generator=g) * sharp).to(torch.bfloat16)
    b = batch(sess, st, k, v)
    words = st.plan()[2]
    if seen is not None:
        words = np.zeros_like(words)
        for s in range(st.seqs):
            words[st.cu[s]:st.cu[s + 1]] = ref.pack(seen[s], st.words)
    plan = paged.TreePlan(None, None, dev(words) if mask == "plan" else None)
    out = torch.full((st.rows, qh * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    got = paged.tree_attention(b, plan, dev(q), qh, scale=scale, out=out, pair_order=pair)
    sess.synchronize()
    want, bound = ref.attention(st, q, k[0].cpu(), v[0].cpu(), qh, hd ** -0.5 if scale is None else scale, seen)
    return got.cpu().double(), want, bound


def assert_close(st, got, want, bound):
    n = int(st.cu[-1])
    err = (got[:n] - want[:n]).abs()
    assert torch.isfinite(got[:n]).all()
    assert (err <= bound[:n]).all(), float((err / bound[:n]).max())
    assert (got[n:] == 7.0).all()                # padding rows stay


@pytest.mark.parametrize("ctx,nodes,page,heads,group,hd", [
    ([0], [1], 16, 1, 1, 128),                   # a first token
    ([333], [1], 16, 8, 4, 128),
    ([1, 0, 127, 128, 129, 64], [1, 1, 1, 1, 1, 0], 16, 2, 4, 64),
    ([700, 1300, 901], [1, 1, 1], 64, 8, 4, 128),
    ([1021, 2111, 5], [3, 7, 2], 16, 4, 8, 128),
    ([40, 0, 300], [33, 64, 5], 32, 3, 7, 64),
    ([120, 1000], [64, 64], 32, 2, 4, 128),      # 256 query rows a KV head
    ([130, 0], [256, 200], 128, 2, 8, 64),       # several row tiles
    ([5, 250], [129, 100], 256, 1, 3, 128),
    ([5000], [2], 16, 1, 16, 128),               # one KV head, many pieces
    ([17] * 40, [1] * 40, 16, 4, 1, 128),        # many short sequences
    ([3000, 1, 0, 2], [4, 0, 31, 1], 16, 5, 5, 128)])
def test_attention_matches(sess, ctx, nodes, page, heads, group, hd):
    st = ref.Step(ctx, nodes, page, seed=sum(ctx) + page, pad=3)
    assert_close(st, *run_attention(sess, st, heads, group, hd, seed=hd + page))


@pytest.mark.parametrize("ctx,nodes,page,heads,group,hd", [
    ([20000], [1], 64, 1, 8, 128),               # one unit in a piece per SM
    ([19000], [3], 16, 1, 20, 64),
    ([5900, 4100], [200, 228], 128, 8, 8, 64),   # many pieces a CTA, units of 256, 64 and 32 rows in turn
    ([900, 3, 2000], [70, 33, 129], 32, 3, 2, 128),
    ([60, 200], [2, 3], 16, 1, 300, 128),        # more heads per KV head than a unit has rows
    ([(i * 37) % 400 for i in range(300)], [1 + i % 5 if i % 7 else 0 for i in range(300)], 16, 2, 3, 64)])
def test_attention_divides_any_work(sess, ctx, nodes, page, heads, group, hd):
    st = ref.Step(ctx, nodes, page, seed=sum(nodes), pad=1)
    assert_close(st, *run_attention(sess, st, heads, group, hd, seed=hd + len(ctx)))


@pytest.mark.parametrize("ctx,nodes,page,heads,group,hd", [
    ([1021, 2111, 1500, 1800, 1207], [3, 7, 5, 4, 6], 16, 8, 8, 128),   # a piece for each CTA
    ([700 + 40 * i for i in range(16)], [1] * 16, 64, 8, 4, 128),       # whole units
    ([900, 1200], [64, 50], 32, 8, 4, 128),                             # two row tiles
    ([600, 0, 35, 2500], [9, 0, 129, 2], 64, 3, 2, 64),                 # sequences without nodes between
    ([250 + i for i in range(32)], [1] * 32, 32, 4, 2, 64),             # 32 sequences are weighed,
    ([250 + i for i in range(33)], [1] * 33, 32, 4, 2, 64)])            # 33 are not
def test_attention_of_few_units(sess, ctx, nodes, page, heads, group, hd):
    st = ref.Step(ctx, nodes, page, seed=sum(nodes) + 1, pad=2)
    assert_close(st, *run_attention(sess, st, heads, group, hd, seed=hd + len(ctx)))


def test_visible_nan_keys_make_the_row_nan(sess):
    st = ref.Step([150], [4], 16, parents=[np.array([-1, 0, 0, 2], dtype=np.int32)])
    k, v = (t.cpu() for t in pools(st, 1, 64, 1))
    pg, off = st.place(0, 152)                   # node 2, seen by nodes 2 and 3
    k[0, pg, 0, off, 5] = math.nan
    q = torch.randn((4, 64), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    b = batch(sess, st, dev(k), dev(v))
    got = paged.tree_attention(b, paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 1).cpu()
    sess.synchronize()
    assert torch.isfinite(got[:2]).all() and torch.isnan(got[2:]).all()


@pytest.mark.parametrize("kw", [dict(nhd=True), dict(scale=0.3), dict(scale=-0.05), dict(sharp=30.0), dict(sharp=0.0), dict(pair=True)])
def test_attention_variants(sess, kw):
    st = ref.Step([70, 400, 9], [9, 20, 1], 16, seed=8)
    got, want, bound = run_attention(sess, st, 2, 4, 128, seed=3, **kw)
    if kw.get("pair"):
        order = lambda t: t.reshape(st.rows, -1, 2, 4).transpose(-1, -2).reshape(st.rows, -1)
        want, bound = order(want), order(bound)
    assert_close(st, got, want, bound)


@pytest.mark.parametrize("rows", [1, 10, 40, 70])           # 4, 2 and 1 copies of the rows, two row tiles
@pytest.mark.parametrize("step", [0.02, 0.5, 11.0, -3.0])   # log2 units of a position: up by little, by tiles, by runs
def test_attention_of_climbing_scores(sess, rows, step):
    """The maximum rises (or falls) all the way, within runs, tiles and pieces."""
    st = ref.Step([1500], [rows], 32, seed=rows)
    k, v = (t.cpu() for t in pools(st, 1, 64, 2))
    q = torch.zeros((rows, 4 * 64), dtype=torch.bfloat16)
    q[:, ::64] = 1.0                             # scores are the keys' first dim
    for i in range(1500 + rows):
        pg, off = st.place(0, i)
        k[0, pg, 0, off, 0] = i * step * math.log(2)
    out = torch.full((rows, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    got = paged.tree_attention(batch(sess, st, dev(k), dev(v)), paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 4,
                               scale=1.0, out=out)
    sess.synchronize()
    assert_close(st, got.cpu().double(), *ref.attention(st, q, k[0], v[0], 4, 1.0))


def test_attention_without_mask_is_causal(sess):
    st = ref.Step([50, 3], [40, 130], 16, parents="chain")
    assert_close(st, *run_attention(sess, st, 2, 4, 128, mask=None))


def test_rows_that_see_nothing_are_zero(sess):
    """Any mask is allowed: rows that see no drafted node, rows that see later ones, and no cached position."""
    st = ref.Step([0, 0, 33], [5, 40, 3], 16, seed=2)
    rng = np.random.default_rng(0)
    seen = [rng.random((n, n)) < 0.4 for n in st.nodes]
    seen[0][2] = False
    seen[1][::3] = False
    seen[2][:] = False
    got, want, bound = run_attention(sess, st, 2, 4, 64, seen=seen)
    empty = [2] + [5 + i for i in range(0, 40, 3)]
    assert (got[empty] == 0).all()
    assert_close(st, got, want, bound)


def test_mask_bits_behind_the_last_node_mean_nothing(sess):
    st = ref.Step([20], [3], 16, parents="chain")
    k, v = pools(st, 1, 64, 0)
    b = batch(sess, st, k, v)
    q = torch.randn((3, 64), device=DEV).to(torch.bfloat16)
    words = dev(st.plan()[2])
    a = paged.tree_attention(b, paged.TreePlan(None, None, words), q, 1)
    c = paged.tree_attention(b, paged.TreePlan(None, None, words | -8), q, 1)
    sess.synchronize()
    assert torch.equal(a, c)


@pytest.mark.parametrize("hd,page,ctx,n", [(128, 16, 37, 6), (64, 64, 100, 40), (128, 128, 128, 3), (128, 32, 0, 130)])
def test_what_is_hidden_does_not_reach_the_result(sess, hd, page, ctx, n):
    """NaN and infinities behind the last position, in free pages, and in drafted nodes that a row does not see."""
    st = ref.Step([ctx, 8], [n, 2], page, seed=5)
    st.parents[0] = np.array([-1] + [0] * (n - 1), dtype=np.int32)   # siblings below one root
    k, v = (t.cpu() for t in pools(st, 2, hd, 1))
    used = torch.zeros((st.pages, page), dtype=torch.bool)
    for s in range(st.seqs):
        for i in range(st.ctx[s] + st.nodes[s]):
            used[st.place(s, i)] = True
    for t, fill in ((k, math.nan), (v, math.inf)):
        t[0].transpose(1, 2)[~used] = fill
    bad = [1, n - 1]
    for j, fill in zip(bad, (math.nan, -math.inf)):
        pg, off = st.place(0, ctx + j)
        k[0, pg, :, off] = fill
        v[0, pg, 1, off, ::3] = fill
    q = torch.randn((st.rows, 8 * hd), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    b = batch(sess, st, dev(k), dev(v))
    got = paged.tree_attention(b, paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 8)
    sess.synchronize()
    kc = torch.where(k[0].isfinite(), k[0], torch.zeros_like(k[0]))
    vc = torch.where(v[0].isfinite(), v[0], torch.zeros_like(v[0]))
    want, bound = ref.attention(st, q, kc, vc, 8, hd ** -0.5)
    clean = [r for r in range(st.rows) if r not in bad]
    got = got.cpu().double()
    assert torch.isfinite(got[clean]).all()
    assert ((got - want).abs() <= bound)[clean].all()


def test_visible_infinities_reach_the_rows_that_see_them(sess):
    st = ref.Step([30], [4], 16, parents=[np.array([-1, 0, 0, 2], dtype=np.int32)])
    k, v = (t.cpu() for t in pools(st, 1, 128, 1))
    pg, off = st.place(0, 32)                    # node 2, seen by nodes 2 and 3
    v[0, pg, 0, off, 5], v[0, pg, 0, off, 9] = math.inf, math.nan
    q = torch.randn((4, 128), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    b = batch(sess, st, dev(k), dev(v))
    got = paged.tree_attention(b, paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 1).cpu()
    sess.synchronize()
    assert torch.isfinite(got[:2]).all()
    for r in (2, 3):
        assert got[r, 5] == math.inf and math.isnan(got[r, 9])
        assert torch.isfinite(got[r, [i for i in range(128) if i not in (5, 9)]]).all()


def test_shared_pages_and_long_offsets(sess):
    """Two sequences that share a prefix's pages, in a pool whose last pages lie past 2^31 elements."""
    page, hd, heads = 256, 128, 4
    pages = (1 << 31) // (page * hd * heads) + 8
    k = torch.zeros((pages, heads, page, hd), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    ids = [pages - 1, pages - 3, 2, pages - 2]
    for i in ids:
        k[i].normal_()
        v[i].normal_()
    st = ref.Step([300, 300], [2, 3], page, seed=1)
    st.table = np.array([[ids[0], ids[1]], [ids[0], ids[3]]], dtype=np.int32)
    st.pages = pages
    q = torch.randn((5, 8 * hd), device=DEV).to(torch.bfloat16)
    b = batch(sess, st, k, v)
    got = paged.tree_attention(b, paged.TreePlan(None, None, dev(st.plan()[2])), q, 8)
    sess.synchronize()
    small = [t[ids].cpu() for t in (k, v)]
    st.table = np.array([[0, 1], [0, 3]], dtype=np.int32)
    want, bound = ref.attention(st, q.cpu(), *small, 8, hd ** -0.5)
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_bad_pages_and_lengths_are_reported(sess):
    st = ref.Step([40, 20], [2, 3], 16, seed=4)
    k, v = pools(st, 2, 64, 0)
    q = torch.randn((5, 4 * 64), device=DEV).to(torch.bfloat16)
    plan = paged.TreePlan(None, None, dev(st.plan()[2]))
    good = paged.tree_attention(batch(sess, st, k, v), plan, q, 4)
    sess.synchronize()
    for what, value in (("table", st.pages), ("table", -1), ("ctx", -5), ("ctx", 5000), ("cu", 1)):
        b = batch(sess, st, k, v)
        if what == "table":
            b.page_table[0, 1] = value
        elif what == "ctx":
            b.ctx_lens[0] = value
        else:
            b.cu_nodes[1] = -1
        out = torch.full_like(q, 7.0)
        paged.tree_attention(b, plan, q, 4, out=out)
        with pytest.raises(AffonError) as err:
            sess.synchronize()
        assert err.value.code == "invalid_arg"
        if what != "cu":
            assert torch.equal(out[2:], good[2:])        # the other sequence is untouched by it
        if what == "ctx":
            assert (out[:2] == 7.0).all()
    again = paged.tree_attention(batch(sess, st, k, v), plan, q, 4)
    sess.synchronize()
    assert torch.equal(again, good)


def test_attention_repeats_bit_for_bit_on_streams_and_in_graphs(sess):
    st = ref.Step([1500, 90, 700], [6, 1, 12], 16, seed=6)
    k, v = pools(st, 4, 128, 0)
    q = torch.randn((st.rows, 16 * 128), device=DEV).to(torch.bfloat16)
    b = batch(sess, st, k, v)
    plan = paged.TreePlan(None, None, dev(st.plan()[2]))
    first = paged.tree_attention(b, plan, q, 16).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged.tree_attention(b, plan, q, 16)
    torch.cuda.current_stream().wait_stream(side)
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.tree_attention(b, plan, q, 16, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
    torch.cuda.synchronize()
    sess.synchronize()
    assert torch.equal(first, other) and torch.equal(first, out)
    b.ctx_lens[0] = 800                          # the graph reads the lengths when it runs
    g.replay()
    want = paged.tree_attention(b, plan, q, 16)
    sess.synchronize()
    assert torch.equal(out, want) and not torch.equal(out, first)


def test_sessions_on_two_streams_do_not_disturb_each_other():
    """A Session per stream: both attend at once, neither sees the other's workspace."""
    st = ref.Step([2500, 900, 40], [5, 9, 1], 16, seed=6)
    k, v = pools(st, 4, 128, 0)
    q = torch.randn((st.rows, 16 * 128), device=DEV).to(torch.bfloat16)
    plan = paged.TreePlan(None, None, dev(st.plan()[2]))
    with Session("cuda:0") as one, Session("cuda:0") as two:
        want = paged.tree_attention(batch(one, st, k, v), plan, q, 16)
        one.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for s, stream in zip((one, two), streams):
            stream.wait_stream(torch.cuda.current_stream())
            b = batch(s, st, k, v)
            with torch.cuda.stream(stream):
                outs.append([paged.tree_attention(b, plan, q, 16) for _ in range(20)])
        for s in (one, two):
            s.synchronize()
        assert all(torch.equal(o, want) for group in outs for o in group)


def test_disposed_session_and_zero_scale_are_refused(sess):
    st = ref.Step([5], [1], 16)
    k, v = pools(st, 1, 64, 0)
    b = batch(sess, st, k, v)
    q = torch.zeros((1, 64), dtype=torch.bfloat16, device=DEV)
    for scale in (0.0, math.inf, math.nan):
        with pytest.raises(AffonError) as err:
            paged.tree_attention(b, None, q, 1, scale=scale)
        assert err.value.code == "invalid_arg"
    gone = Session("cuda:0")
    b = batch(gone, st, k, v)
    gone.dispose()
    with pytest.raises(AffonError):
        paged.tree_attention(b, None, q, 1)
    with pytest.raises(AffonError):
        gone.synchronize()


def test_scales_whose_log2_form_overflows_are_refused(sess):
    st = ref.Step([5], [1], 16)
    k, v = pools(st, 1, 64, 0)
    b = batch(sess, st, k, v)
    q = torch.zeros((1, 64), dtype=torch.bfloat16, device=DEV)
    for scale in (3.0e38, -3.0e38):
        with pytest.raises(AffonError) as err:
            paged.tree_attention(b, None, q, 1, scale=scale)
        assert err.value.code == "invalid_arg"
    v.normal_()
    want = v[0, int(st.table[0, 0]), 0, :6].double().mean(0)     # equal scores: the mean of the values
    for scale in (1.9e38, -1.9e38):
        out = paged.tree_attention(b, None, q, 1, scale=scale)
        sess.synchronize()
        # one rounding of the result (2^-8 of it, half a step with room) and an f32 sum
        assert ((out[0].double() - want).abs() <= 2 ** -8 * want.abs() + 1e-5).all()


def test_append_refuses_columns_past_31_bits(sess):
    import ctypes
    from affon_b200 import _lib
    st = ref.Step([5], [1], 16)
    k, v = pools(st, 1, 64, 0)
    b = batch(sess, st, k, v)
    d = _lib.AppendDesc(ctypes.sizeof(_lib.AppendDesc), _lib.BF16, 0, 1, 0, 64, 2 ** 31 - 64, 1, 2 ** 33, 64)
    status = _lib.lib().affon_b200_paged_append(sess._ctx, ctypes.byref(b.desc), ctypes.byref(d), *[None] * 8)
    assert status == _lib.INVALID_SHAPE


# ----------------------------------------------------------------- accept
def accept_case(st, rng, follow=0.8):
    """Tokens and predictions that accept paths of different lengths (with repeated sibling tokens)."""
    tokens = rng.integers(0, 4, size=st.rows).astype(np.int32)
    predicted = rng.integers(0, 4, size=st.rows).astype(np.int32)
    for s in range(st.seqs):
        for i in range(st.nodes[s]):
            kids = [j for j in range(st.nodes[s]) if st.parents[s][j] == i]
            if kids and rng.random() < follow:
                predicted[st.cu[s] + i] = tokens[st.cu[s] + rng.choice(kids)]
    return tokens, predicted


@pytest.mark.parametrize("ctx,nodes,page,heads,hd,layers,nhd,kind", [
    ([333], [13], 16, 8, 128, 2, False, None), ([5, 0, 70, 31], [33, 0, 64, 1], 32, 3, 64, 3, True, None),
    ([100, 7], [256, 255], 128, 1, 128, 1, False, "chain"), ([9] * 20, [7] * 20, 16, 2, 64, 5, False, None),
    ([15, 14], [40, 40], 16, 2, 128, 30, False, None), ([50], [30], 16, 8, 128, 2, True, None)])
@pytest.mark.parametrize("inplace", [False, True])
def test_accept_matches(sess, ctx, nodes, page, heads, hd, layers, nhd, kind, inplace):
    st = ref.Step(ctx, nodes, page, seed=sum(nodes), parents=kind, pad=2)
    rng = np.random.default_rng(page)
    tokens, predicted = accept_case(st, rng, 0.97 if kind else 0.8)
    k, v = pools(st, heads, hd, 2, layers=layers, nhd=nhd)
    k0, v0 = k.cpu(), v.cpu()
    b = batch(sess, st, k, v)
    out = None
    if inplace:
        new = lambda *s: torch.full(s, 99, dtype=torch.int32, device=DEV)
        out = paged.Accepted(new(st.seqs), new(st.seqs, st.max_nodes), new(st.seqs), b.ctx_lens)
    a = paged.tree_accept(b, None if kind == "chain" else dev(st.flat_parents()), dev(tokens), dev(predicted), out=out)
    sess.synchronize()
    counts, path, nxt, lens = ref.accept(st, tokens, predicted)
    assert counts.max() > 1 or nodes == [13]     # that one accepts its root alone
    for got, want in ((a.counts, counts), (a.path, path), (a.next_tokens, nxt), (a.lens, lens)):
        assert got.cpu().tolist() == want.tolist()
    assert b.ctx_lens.cpu().tolist() == (lens.tolist() if inplace else list(ctx))
    assert torch.equal(k.cpu(), ref.move_accepted(st, k0, path, counts))
    assert torch.equal(v.cpu(), ref.move_accepted(st, v0, path, counts))


# --------------------------------------------------------------- together
def test_drafted_steps_equal_plain_steps(sess):
    """Plan, append, attention and accept as a server runs them, captured once and replayed: the cache and outputs of
    drafted steps equal those of feeding the accepted tokens one by one."""
    heads, group, hd, page, seqs, n, cap = 2, 4, 64, 16, 3, 8, 96
    qh = heads * group
    vocab = 12
    rng = np.random.default_rng(0)
    g = torch.Generator().manual_seed(0)
    emb = (torch.randn((vocab, (qh + 2 * heads) * hd), generator=g)).to(torch.bfloat16).to(DEV)
    readout = torch.randn((qh * hd, vocab), generator=g).to(DEV)
    cos, sin = (t.to(DEV) for t in tables(cap, hd))
    per = cap // page

    def machine(rows_per):
        shape = (seqs, heads, cap, hd)
        k, v = torch.zeros((1,) + shape, dtype=torch.bfloat16, device=DEV), torch.zeros((1,) + shape, dtype=torch.bfloat16, device=DEV)
        cache, table = paged.PagedCache.from_contiguous(sess, k, v, page)
        ctx = torch.zeros(seqs, dtype=torch.int32, device=DEV)
        cu = torch.arange(seqs + 1, dtype=torch.int32, device=DEV) * rows_per
        b = paged.PagedBatch(sess, table, ctx, cu, seqs * rows_per, rows_per, cache=cache)
        return k, v, b

    def step(b, parents, tokens, plan):
        paged.plan(b, parents, out=plan)
        q = paged.append(b, plan, emb[tokens.long()], qh, cos, sin)
        o = paged.tree_attention(b, plan, q, qh)
        return o, (o.float() @ readout).argmax(-1).int()

    k1, v1, b1 = machine(1)
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    plan1 = paged.TreePlan(new(seqs), new(seqs), new(seqs, 1))
    acc1 = paged.Accepted(new(seqs), new(seqs, 1), new(seqs), b1.ctx_lens)
    tok = torch.tensor([1, 5, 7], dtype=torch.int32, device=DEV)
    said = [tok.cpu().tolist()]
    for _ in range(24):
        _, pred = step(b1, None, tok, plan1)
        paged.tree_accept(b1, None, tok, pred, out=acc1)
        tok = acc1.next_tokens.clone()
        said.append(tok.cpu().tolist())
    sess.synchronize()
    # the same with drafted trees: the right continuation hidden among wrong ones
    k2, v2, b2 = machine(n)
    plan2 = paged.TreePlan(new(seqs * n), new(seqs * n), new(seqs * n, 1))
    acc2 = paged.Accepted(new(seqs), new(seqs, n), new(seqs), b2.ctx_lens)
    parents, tokens = new(seqs * n), new(seqs * n)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            _, pred2 = step(b2, parents, tokens, plan2)
            paged.tree_accept(b2, parents, tokens, pred2, out=acc2)
    at = [0] * seqs
    for _ in range(12):
        par, tk = [], []
        for s in range(seqs):
            p = ref.random_forest(n, rng)
            t = rng.integers(0, vocab, size=n)
            t[0] = said[at[s]][s]
            cur = 0                              # one child of each node on a path is right
            for depth in range(1, 4):
                kids = [j for j in range(cur + 1, n) if p[j] == cur]
                if not kids or at[s] + depth >= len(said):
                    break
                cur = int(rng.choice(kids))
                t[cur] = said[at[s] + depth][s]
            par.append(p)
            tk.append(t)
        parents.copy_(dev(np.concatenate(par)))
        tokens.copy_(dev(np.concatenate(tk).astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        counts = acc2.counts.cpu().tolist()
        for s in range(seqs):
            at[s] += counts[s]
            if at[s] < len(said):
                assert int(acc2.next_tokens[s]) == said[at[s]][s]
        if max(at) >= 20:
            break
    sess.synchronize()
    assert max(at) > 12                          # drafts were accepted
    for s in range(seqs):
        m = min(at[s], 24)
        assert torch.equal(k2[0, s, :, :m], k1[0, s, :, :m]) and torch.equal(v2[0, s, :, :m], v1[0, s, :, :m])


# ------------------------------------------------- accepted nodes without a page
@pytest.mark.parametrize("layers", [0, 1, 40])               # no cache to move, one CTA a sequence, several
@pytest.mark.parametrize("hole", ["own", "root", "target"])
def test_accept_skips_a_sequence_whose_accepted_nodes_have_no_page(sess, layers, hole):
    """Their keys and values were never written (or have nowhere to go), so no length may pass them: the sequence's
    outputs and cache stay as they were, the others advance, and the next synchronize reports it."""
    st = ref.Step([20, 14, 40], [5, 20, 6], 16, seed=3, parents="chain", pad=1)
    st.parents[1] = np.array([-1, 0] + [1] * 17 + [18], dtype=np.int32)      # path 0, 1, 18, 19
    tokens = np.arange(st.rows, dtype=np.int32)
    predicted = np.full(st.rows, -7, dtype=np.int32)
    at = int(st.cu[1])
    for a, b in ((0, 1), (1, 18), (18, 19)):
        predicted[at + a] = tokens[at + b]
    predicted[at + 19] = 77
    predicted[:4] = tokens[1:5]                              # the first sequence's whole chain
    counts, path, nxt, lens = ref.accept(st, tokens, predicted)
    assert counts.tolist() == [5, 4, 1] and path[1, :4].tolist() == [0, 1, 18, 19]
    k, v = pools(st, 2, 64, 5, layers=max(1, layers))
    k0, v0 = k.clone(), v.clone()
    b = batch(sess, st, k, v)
    # positions 14 and 15 lie in its first page, 16 to 31 in the second, 32 and 33 (nodes 18 and 19) in the third
    b.page_table[1, {"own": 2, "root": 0, "target": 1}[hole]] = -1 if hole != "root" else st.pages
    new = lambda *s: torch.full(s, 99, dtype=torch.int32, device=DEV)
    out = paged.Accepted(new(3), new(3, st.max_nodes), new(3), b.ctx_lens)
    if layers:
        paged.tree_accept(b, dev(st.flat_parents()), dev(tokens), dev(predicted), out=out)
    else:                                                    # the C call alone takes no cache
        import ctypes
        from affon_b200 import _lib
        p = [dev(a) for a in (st.flat_parents(), tokens, predicted)]
        sess.bind_stream()
        assert _lib.lib().affon_b200_tree_accept(
            sess._ctx, ctypes.byref(b.desc), 0, 0, b.cu_nodes.data_ptr(), *[t.data_ptr() for t in p],
            b.page_table.data_ptr(), b.ctx_lens.data_ptr(), None, None, out.counts.data_ptr(), out.path.data_ptr(),
            st.max_nodes, out.next_tokens.data_ptr(), out.lens.data_ptr()) == _lib.OK
    with pytest.raises(AffonError) as err:
        sess.synchronize()
    assert err.value.code == "invalid_arg"
    for got, want in ((out.counts, counts), (out.path, path), (out.next_tokens, nxt)):
        assert got[[0, 2]].cpu().tolist() == want[[0, 2]].tolist() and (got[1] == 99).all()
    assert b.ctx_lens.cpu().tolist() == [int(lens[0]), 14, int(lens[2])]
    if layers:
        counts[1] = 0                                        # nothing of it moves
        assert torch.equal(k.cpu(), ref.move_accepted(st, k0.cpu(), path, counts))
        assert torch.equal(v.cpu(), ref.move_accepted(st, v0.cpu(), path, counts))


def test_accept_needs_no_page_for_what_it_does_not_accept(sess):
    st = ref.Step([14], [20], 16, seed=3, parents=[np.array([-1] + [0] * 19, dtype=np.int32)])
    tokens, predicted = np.arange(20, dtype=np.int32), np.full(20, 1, dtype=np.int32)
    k, v = pools(st, 1, 64, 5)
    b = batch(sess, st, k, v)
    b.page_table[0, 1:] = -1                                 # positions 16 and up: nodes 2 to 19
    a = paged.tree_accept(b, dev(st.flat_parents()), dev(tokens), dev(predicted))
    sess.synchronize()
    assert a.counts.tolist() == [2] and a.lens.tolist() == [16]
    assert a.path[0, :3].tolist() == [0, 1, -1] and a.next_tokens.tolist() == [1]


# ------------------------------------------------------- climbing and far scores
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("step", [0.02, 0.5, 11.0, -3.0])
def test_climbing_scores_of_one_copy_in_alternate_tiles(sess, hd, step):
    """100 query rows: one copy of the rows, whose streams take alternate tiles and rescale their own O."""
    st = ref.Step([1500], [25], 32, seed=25)
    k, v = (t.cpu() for t in pools(st, 1, hd, 2))
    q = torch.zeros((25, 4 * hd), dtype=torch.bfloat16)
    q[:, ::hd] = 1.0
    for i in range(1525):
        pg, off = st.place(0, i)
        k[0, pg, 0, off, 0] = i * step * math.log(2)
    out = torch.full((25, 4 * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    got = paged.tree_attention(batch(sess, st, dev(k), dev(v)), paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 4,
                               scale=1.0, out=out)
    sess.synchronize()
    assert_close(st, got.cpu().double(), *ref.attention(st, q, k[0], v[0], 4, 1.0))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 10, 25, 70])            # 4, 2 and 1 copies of the rows, two row tiles
def test_a_raise_between_far_scores_keeps_their_weights(sess, rows, hd):
    """Scores near 2^22 log2 units, where f32 steps by 1/4 below and 1/2 above: all positions score 5592401 but one
    5592413 at three quarters of the context, both exact in f32, times 0.75 log2 units.  Values are 1 and -1.

    The weights' ratio is 2^-9 up to the rounding of 0.75 (12 * 0.75 * 2^-23 of an exponent) and exp's, so the result
    is off by a probability's rounding to bf16 (2^-8 of sum p |v - o| = 1 - o^2) and its own."""
    st = ref.Step([2000 + 37 * s for s in range(8)], [rows] * 8, 64, seed=rows)
    heads, scale = 8, float(np.float32(0.75 * math.log(2)))
    k = torch.zeros((st.pages, heads, 64, hd), dtype=torch.bfloat16)
    v = torch.ones_like(k)
    k[..., 0], k[..., 1], k[..., 2] = 85 * 65536, 85 * 256, 81
    for s in range(8):
        pg, off = st.place(s, 1500)
        k[pg, :, off, 2], v[pg, :, off] = 93, -1
    q = torch.zeros((st.rows, heads * 4 * hd), dtype=torch.bfloat16)
    for d in range(3):
        q[:, d::hd] = 1.0
    got = paged.tree_attention(batch(sess, st, dev(k)[None], dev(v)[None]),
                               paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), heads * 4, scale=scale)
    sess.synchronize()
    got = got.cpu().double()
    for s in range(8):
        a = int(st.cu[s])
        seen = st.ctx[s] - 1 + torch.from_numpy(ref.ancestors(st.parents[s])).sum(-1).double()
        w = seen * 2.0 ** -9
        want = ((w - 1) / (w + 1))[:, None]
        tol = (2.0 ** -8 + 2.0 ** -12) * (1 - want ** 2) + 2.0 ** -8 * want.abs()
        err = (got[a:a + rows] - want).abs()
        assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("far", [2.0 ** 20, -2.0 ** 26, 7.0e8, -7.0e8])
@pytest.mark.parametrize("rows", [1, 25, 70])
def test_equal_far_scores_give_the_mean(sess, rows, far):
    """Up to the largest scores that are promised: every position has the same one, so the probabilities are equal
    whatever their rounding, and the result is off by the f32 sums and its own rounding to bf16."""
    st = ref.Step([700], [rows], 32, seed=rows)
    k, v = (t.cpu() for t in pools(st, 1, 64, 7))
    k.zero_()
    k[..., 0], k[..., 1] = 85 * 256, 81
    q = torch.zeros((rows, 4 * 64), dtype=torch.bfloat16)
    q[:, ::64], q[:, 1::64] = 1.0, 1.0
    scale = float(np.float32(far / (85 * 256 + 81)))
    got = paged.tree_attention(batch(sess, st, dev(k), dev(v)), paged.TreePlan(None, None, dev(st.plan()[2])), dev(q), 4,
                               scale=scale)
    sess.synchronize()
    want, _ = ref.attention(st, q, k[0], v[0], 4, 0.0)
    mag, _ = ref.attention(st, q, k[0], v[0].abs(), 4, 0.0)
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * mag).all()


def test_append_of_one_row_with_further_columns(sess):
    st = ref.Step([5], [1], 16)
    k, v = pools(st, 2, 64, 1)
    b = batch(sess, st, k, v)
    pos, slots, _ = st.plan()
    p = paged.TreePlan(dev(pos), dev(slots))
    wide = torch.randn((1, 8 * 64 + 5), device=DEV).to(torch.bfloat16)       # 517 columns: not a multiple of 16 bytes
    q = paged.append(b, p, wide, 4, rope="none")
    sess.synchronize()
    pg, off = st.place(0, 5)
    assert torch.equal(q, wide[:, :256])
    assert torch.equal(k[0, pg, :, off].flatten(), wide[0, 256:384])
    assert torch.equal(v[0, pg, :, off].flatten(), wide[0, 384:512])


# ------------------------------------------------------------- the merge gives up
def test_a_merge_that_gives_up_is_reported_and_the_next_call_is_right(sess):
    """A hook makes every merge wait (20 ms) for one piece more than there is."""
    from affon_b200 import _lib
    st = ref.Step([3000, 64, 900], [9, 2, 64], 16, seed=6)
    k, v = pools(st, 4, 128, 0)
    q = torch.randn((st.rows, 16 * 128), device=DEV).to(torch.bfloat16)
    b = batch(sess, st, k, v)
    plan = paged.TreePlan(None, None, dev(st.plan()[2]))
    want = paged.tree_attention(b, plan, q, 16)
    sess.synchronize()
    L = _lib.lib()
    L.affon_b200_debug_set_combine_wait(20_000_000, 1)
    try:
        out = torch.full_like(want, 7.0)
        paged.tree_attention(b, plan, q, 16, out=out)
        with pytest.raises(AffonError) as err:
            sess.synchronize()
        assert err.value.code == "timeout"
    finally:
        L.affon_b200_debug_set_combine_wait(0, 0)
    assert (out[0] == 7.0).all()                             # the long sequence's rows were to be merged
    for _ in range(2):
        assert torch.equal(paged.tree_attention(b, plan, q, 16), want)
        sess.synchronize()
