"""Measured cases of the paged-cache operators: the step plan of a forest of
drafted tokens, rotation and append into a paged key/value cache, attention
of drafted trees over that cache, and the acceptance of a drafted path.

`run` computes an operator in its plain form (elementary torch operations in
32 bits) where `own` is false, and through affon_b200.paged where it is true.
A case's ragged lengths follow from the case alone; all values follow from
the seed.
"""
import math

import numpy as np
import torch

own = False

ROPE_THETA = 500000.0
_SESSION = {}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One new token of one short sequence (interactive decoding): latency only.  8B head layout.
        {"name": "attention-one-token", "op": "attention", "seqs": 1, "ctx_lo": 333, "ctx_hi": 333, "nodes_lo": 1,
         "nodes_hi": 1, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 16},
        # A serving batch of plain single-token decoding: 16 sequences near 1024 positions, 8B head layout.
        {"name": "attention-batch", "op": "attention", "seqs": 16, "ctx_lo": 700, "ctx_hi": 1300, "nodes_lo": 1,
         "nodes_hi": 1, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 64},
        # Small drafted trees of a few sequences near 2048 positions: 70B head layout, odd tree sizes.
        {"name": "attention-trees", "op": "attention", "seqs": 5, "ctx_lo": 1021, "ctx_hi": 2111, "nodes_lo": 3,
         "nodes_hi": 7, "kv_heads": 8, "group": 8, "head_dim": 128, "page": 16},
        # Wide trees: 64 drafted tokens per sequence, so 256 query rows share every key (compute and bandwidth level).
        {"name": "attention-wide-trees", "op": "attention", "seqs": 8, "ctx_lo": 6011, "ctx_hi": 10007, "nodes_lo": 49,
         "nodes_hi": 64, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 32},
        # Long documents: the largest cache, 16 drafted tokens each, offsets past 2^31 bytes.
        {"name": "attention-long", "op": "attention", "seqs": 4, "ctx_lo": 120001, "ctx_hi": 131072, "nodes_lo": 16,
         "nodes_hi": 16, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 64},
        # Prompt chunks as chains of 256 tokens, 64-wide heads: many query rows per key (compute bound).
        {"name": "attention-chunks", "op": "attention", "seqs": 3, "ctx_lo": 1501, "ctx_hi": 5003, "nodes_lo": 200,
         "nodes_hi": 256, "kv_heads": 8, "group": 8, "head_dim": 64, "page": 128},
        # One row of an f32 projection into the cache: the smallest call.
        {"name": "append-one-token", "op": "append", "seqs": 1, "ctx_lo": 333, "ctx_hi": 333, "nodes_lo": 1,
         "nodes_hi": 1, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 16, "input": "f32", "rope": "half"},
        # Prompt chunks of many sequences at once: bandwidth bound.
        {"name": "append-chunks", "op": "append", "seqs": 64, "ctx_lo": 0, "ctx_hi": 900, "nodes_lo": 180,
         "nodes_hi": 256, "kv_heads": 8, "group": 4, "head_dim": 128, "page": 64, "input": "bf16", "rope": "half"},
        # The plan of one small tree: latency only.
        {"name": "plan-one-tree", "op": "plan", "seqs": 1, "ctx_lo": 333, "ctx_hi": 333, "nodes_lo": 13,
         "nodes_hi": 13, "page": 16},
        # The plan of a large step: 64 trees of up to 64 nodes.
        {"name": "plan-trees", "op": "plan", "seqs": 64, "ctx_lo": 100, "ctx_hi": 9000, "nodes_lo": 20,
         "nodes_hi": 64, "page": 32},
        # One small tree accepted, two layers.
        {"name": "accept-one-tree", "op": "accept", "seqs": 1, "ctx_lo": 333, "ctx_hi": 333, "nodes_lo": 13,
         "nodes_hi": 13, "kv_heads": 8, "head_dim": 128, "page": 16, "layers": 2},
        # A batch of wide trees accepted in all 32 layers of the 8B layout.
        {"name": "accept-trees", "op": "accept", "seqs": 32, "ctx_lo": 5, "ctx_hi": 90, "nodes_lo": 33,
         "nodes_hi": 64, "kv_heads": 8, "head_dim": 128, "page": 32, "layers": 32},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.4e15)


def draw(rng):
    """A case of the same ranges: any head layout, ragged or even lengths, costs up to the largest listed case's."""
    op = rng.choice(["attention", "attention", "append", "accept", "plan"])
    ctx_hi = _log_int(rng, 1, 131072 if op == "attention" else 4096)
    nodes_hi = _log_int(rng, 1, 256)
    case = {"op": op, "seqs": _log_int(rng, 1, 64), "ctx_lo": int(ctx_hi * rng.choice([0.0, 0.5, 0.9, 1.0])),
            "ctx_hi": ctx_hi, "nodes_lo": max(1, int(nodes_hi * rng.choice([0.1, 0.6, 1.0]))), "nodes_hi": nodes_hi,
            "page": rng.choice([16, 32, 64, 128])}
    if op == "plan":
        case["seqs"] = _log_int(rng, 1, 256)
        return case
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
    case["head_dim"] = rng.choice([64, 128, 128])
    if op != "accept":
        case["group"] = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    if op == "append":
        case["input"] = rng.choice(["bf16", "f32"])
        case["rope"] = rng.choice(["half", "half", "interleaved"])
        while _rows(case) * (case["group"] + 2) * case["kv_heads"] * case["head_dim"] > 1 << 27:
            case["seqs"] = max(1, case["seqs"] // 2)
            case["nodes_hi"] = max(case["nodes_lo"], case["nodes_hi"] // 2)
            case["nodes_lo"] = max(1, case["nodes_lo"] // 2)
    if op == "accept":
        case["layers"] = _log_int(rng, 1, 32)
        while case["layers"] * _pages(case) * case["page"] * case["kv_heads"] * case["head_dim"] > 1 << 28:
            if case["ctx_hi"] > 64:
                case["ctx_hi"], case["ctx_lo"] = case["ctx_hi"] // 2, case["ctx_lo"] // 2
            elif case["seqs"] > 1:
                case["seqs"] //= 2
            else:
                case["layers"] = max(1, case["layers"] // 2)
    if op == "attention":
        most = _cost(next(c for c in listed() if c["name"] == "attention-long"))
        while _cost(case) > most:
            if case["ctx_hi"] > 256:
                case["ctx_hi"], case["ctx_lo"] = case["ctx_hi"] // 2, case["ctx_lo"] // 2
            else:
                case["nodes_hi"], case["nodes_lo"] = -(-case["nodes_hi"] // 2), -(-case["nodes_lo"] // 2)
    return case


# ----------------------------------------------------- shapes of a case
def _spread(lo, hi, n, stride):
    """n whole numbers from lo to hi in a mixed order (the same for every seed)."""
    if n == 1:
        return [hi]
    even = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    step = next(s for s in range(max(1, n * stride // 100), 2 * n + 2) if math.gcd(s, n) == 1)
    return [even[i * step % n] for i in range(n)]


def _ctx(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["seqs"], 38)


def _nodes(case):
    return _spread(case["nodes_lo"], case["nodes_hi"], case["seqs"], 61)


def _rows(case):
    return sum(_nodes(case))


def _pages(case):
    return sum(-(-(c + n) // case["page"]) for c, n in zip(_ctx(case), _nodes(case)))


def _words(case):
    return -(-case["nodes_hi"] // 32)


def work(case):
    """Bytes and operations one pass cannot do without: every input read once, every output written once."""
    rows, seqs, op = _rows(case), case["seqs"], case["op"]
    ctx, nodes = _ctx(case), _nodes(case)
    table = 4 * _pages(case)
    if op == "plan":   # parents in; positions, slots and mask words out
        return {"bytes": 4 * rows * (3 + _words(case)) + 4 * (2 * seqs + 1) + table, "flops": 0}
    kh, hd = case["kv_heads"], case["head_dim"]
    if op == "accept":
        # parents, tokens and predictions in; every accepted row but the root's moves, in every layer
        moved = sum(_accept_depth(n) - 1 for n in nodes)
        return {"bytes": 12 * rows + 16 * seqs + moved * case["layers"] * kh * hd * 2 * 2 * 2, "flops": 0}
    qh = kh * case["group"]
    if op == "append":
        size = 2 if case["input"] == "bf16" else 4
        return {"bytes": rows * ((qh + 2 * kh) * hd * (size + 2) + hd * 4 + 8), "flops": 3 * rows * (qh + kh) * hd}
    cache = sum(c + n for c, n in zip(ctx, nodes)) * kh * hd * 4
    return {"bytes": cache + rows * qh * hd * 4 + rows * _words(case) * 4 + table + 4 * (2 * seqs + 1),
            "flops": sum(4 * n * qh * hd * (c + n) for c, n in zip(ctx, nodes))}


def _accept_depth(nodes):
    """Length of the path that a verification accepts here: 1 (the root) to 6, as the tree's size allows."""
    return 1 if nodes < 4 else min(6, 1 + nodes // 6)


# ------------------------------------------------------------------ inputs
def _trees(nodes, rng):
    """Parents of each tree, in draft order: node 0 is the root, each other node hangs below an earlier one, low
    depths first as a drafter grows them."""
    parents = []
    for n in nodes:
        par = np.full(n, -1, dtype=np.int32)
        for i in range(1, n):
            par[i] = rng.integers(max(0, i // 3 - 2), max(1, (2 * i) // 3 + (i < 3)))
        parents.append(par)
    return parents


def _masks(parents, words):
    """Ancestor-or-self bits of every row, packed in 32-bit words."""
    out = []
    for par in parents:
        m = np.zeros((len(par), words * 32), dtype=bool)
        for i, p in enumerate(par):
            if p >= 0:
                m[i] = m[p]
            m[i, i] = True
        out.append(m)
    bits = np.concatenate(out).reshape(-1, words, 32).astype(np.uint64)
    packed = (bits << np.arange(32, dtype=np.uint64)).sum(-1)
    return packed.astype(np.uint32).view(np.int32)


def _depths(parents):
    out = []
    for par in parents:
        d = np.zeros(len(par), dtype=np.int32)
        for i, p in enumerate(par):
            d[i] = d[p] + 1 if p >= 0 else 0
        out.append(d)
    return out


def _accepted_tree(n, rng):
    """A tree, its tokens, and predictions that accept a path whose nodes lie behind the places they move to."""
    length = _accept_depth(n)
    par = _trees([n], rng)[0]
    path = [0]
    if length > 1:   # the accepted path: one node per level, from the later drafts of the tree
        path += sorted(rng.choice(np.arange(length, n), size=length - 1, replace=False).tolist())
        for a, b in zip(path, path[1:]):
            par[b] = a
    tok = np.zeros(n, dtype=np.int32)
    seen = {}
    for i in range(n):   # siblings are distinct proposals
        used = seen.setdefault(int(par[i]), set())
        t = int(rng.integers(0, 128256))
        while t in used:
            t = (t + 1) % 128256
        used.add(t)
        tok[i] = t
    pred = rng.integers(0, 128256, size=n).astype(np.int32)
    for a, b in zip(path, path[1:]):
        pred[a] = tok[b]
    last = seen.get(path[-1], set())
    while int(pred[path[-1]]) in last:
        pred[path[-1]] = (pred[path[-1]] + 1) % 128256
    return par, tok, pred


def _session(device):
    """One Session per device, kept as a serving process keeps it."""
    key = str(device)
    if key not in _SESSION:
        from affon_b200 import Session
        _SESSION[key] = Session(key)
    return _SESSION[key]


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    op, page, seqs = case["op"], case["page"], case["seqs"]
    ctx, nodes, rows, words = _ctx(case), _nodes(case), _rows(case), _words(case)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=dev)
    normal = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)

    # The pages of every sequence, scattered over the pool as an allocator leaves them.
    need = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
    pages = sum(need) + 3
    order = rng.permutation(pages)
    table = np.zeros((seqs, max(need)), dtype=np.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    st = {"op": op, "case": dict(case), "ctx_host": ctx, "nodes_host": nodes, "page": page, "rows": rows,
          "words": words, "need": need,
          "table": up(table), "ctx": up(np.asarray(ctx, dtype=np.int32)), "cu": up(cu),
          "seq_of_row": up(np.repeat(np.arange(seqs), nodes)),
          "node_of_row": up(np.concatenate([np.arange(n) for n in nodes]).astype(np.int64))}
    if op == "accept":
        grown = [_accepted_tree(n, rng) for n in nodes]
        parents = [g[0] for g in grown]
        st["tokens"] = up(np.concatenate([g[1] for g in grown]))
        st["predicted"] = up(np.concatenate([g[2] for g in grown]))
        st["steps"] = max(_accept_depth(n) for n in nodes)
    else:
        parents = _trees(nodes, rng)
        if op == "attention" and case["nodes_lo"] >= 200:   # prompt chunks are chains
            parents = [np.arange(-1, n - 1, dtype=np.int32) for n in nodes]
    st["parents"] = up(np.concatenate(parents).astype(np.int32))
    st["deepest"] = int(max(d.max() for d in _depths(parents)))
    if op in ("append", "attention"):
        loc = np.concatenate([table[s, (ctx[s] + np.arange(n)) // page] * page + (ctx[s] + np.arange(n)) % page
                              for s, n in enumerate(nodes)])
        pos = np.concatenate([c + d for c, d in zip(ctx, _depths(parents))])
        st["slots"], st["positions"] = up(loc.astype(np.int32)), up(pos.astype(np.int32))
        st["mask"] = up(_masks(parents, words))
    if op != "plan":
        kh, hd, layers = case["kv_heads"], case["head_dim"], case.get("layers", 1)
        st["k"], st["v"] = normal(layers, pages, kh, page, hd), normal(layers, pages, kh, page, hd)
        qh = kh * case.get("group", 1)
        st["q_heads"], st["hd"], st["kh"] = qh, hd, kh
    if op == "append":
        dt = torch.bfloat16 if case["input"] == "bf16" else torch.float32
        st["qkv"] = randn(rows, (qh + 2 * kh) * hd).to(dt)
        most = max(ctx) + max(nodes)
        inv = ROPE_THETA ** (-np.arange(hd // 2, dtype=np.float64) * 2.0 / hd)
        ang = np.arange(most, dtype=np.float64)[:, None] * inv[None, :]
        st["cos"], st["sin"] = up(np.cos(ang).astype(np.float32)), up(np.sin(ang).astype(np.float32))
    if op == "attention":
        # heads differ in how sharply they look: score deviations from 0.5 to 3
        heat = torch.linspace(0.5, 3.0, qh, device=dev)
        st["q"] = (randn(rows, qh, hd) * heat[None, :, None]).to(torch.bfloat16).reshape(rows, qh * hd)
        st["scale"] = 1.0 / math.sqrt(hd)
        st["out"] = torch.zeros((rows, qh * hd), dtype=torch.bfloat16, device=dev)
    if own:
        from affon_b200 import paged
        sess = _session(dev)
        if op == "plan":
            shape = dict(page_size=page, pages=pages)
        else:
            st["cache"] = paged.PagedCache(sess, st["k"], st["v"])
            shape = dict(cache=st["cache"])
        st["batch"] = paged.PagedBatch(sess, st["table"], st["ctx"], st["cu"], rows=rows, max_nodes=max(nodes),
                                       **shape)
        if op in ("append", "attention"):
            st["plan"] = paged.TreePlan(st["positions"], st["slots"], st["mask"])
    return st


# --------------------------------------------------------------------- run
def run(st):
    return {"plan": _plan, "append": _append, "attention": _attention, "accept": _accept}[st["op"]](st)


def _plan(st):
    if own:
        from affon_b200 import paged
        p = paged.plan(st["batch"], st["parents"])
        return p.positions, p.slots, p.mask
    seq, node, page = st["seq_of_row"], st["node_of_row"], st["page"]
    first = st["cu"].long()[seq]
    row = torch.arange(st["rows"], device=seq.device)
    bit = torch.ones_like(row) << (node % 32)
    mask = torch.zeros((st["rows"], st["words"]), dtype=torch.int64, device=seq.device)
    mask[row, node // 32] = bit
    par = st["parents"].long()
    up = torch.where(par >= 0, first + par, row)       # a root points at itself
    depth = (par >= 0).long()
    for _ in range(max(1, math.ceil(math.log2(st["deepest"] + 1)))):   # doubling: ancestors of ancestors
        mask = mask | mask[up]
        depth = depth + depth[up]
        up = up[up]
    place = st["ctx"].long()[seq] + node
    slots = st["table"].long()[seq, place // page] * page + place % page
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask)
    return (st["ctx"].long()[seq] + depth).int(), slots.int(), mask.int()


def _append(st):
    if own:
        from affon_b200 import paged
        q = paged.append(st["batch"], st["plan"], st["qkv"], st["q_heads"], st["cos"], st["sin"],
                         rope=st["case"]["rope"])
        return q, st["k"], st["v"]
    return _append_plain(st, torch.float32)


def _append_plain(st, dt):
    rows, qh, kh, hd, page = st["rows"], st["q_heads"], st["kh"], st["hd"], st["page"]
    x = st["qkv"].to(dt).reshape(rows, qh + 2 * kh, hd)
    pos = st["positions"].long()
    c, s = st["cos"].to(dt)[pos][:, None, :], st["sin"].to(dt)[pos][:, None, :]
    r = x[:, :qh + kh]
    if st["case"]["rope"] == "half":
        a, b = r[..., :hd // 2], r[..., hd // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], dim=-1).reshape(rows, qh + kh, hd)
    slot = st["slots"].long()
    st["k"][0][slot // page, :, slot % page] = y[:, qh:].to(torch.bfloat16)
    st["v"][0][slot // page, :, slot % page] = x[:, qh + kh:].to(torch.bfloat16)
    return y[:, :qh].to(torch.bfloat16).reshape(rows, qh * hd), st["k"], st["v"]


def _visible(st, s, n):
    """Which drafted nodes each of sequence s's nodes sees, from the packed words."""
    r0 = sum(st["nodes_host"][:s])
    m = st["mask"][r0:r0 + n].long()
    bits = (m[:, :, None] >> torch.arange(32, device=m.device)) & 1
    return r0, bits.reshape(n, -1)[:, :n].bool()


def _attention(st):
    if own:
        from affon_b200 import paged
        return paged.tree_attention(st["batch"], st["plan"], st["q"], st["q_heads"], scale=st["scale"],
                                    out=st["out"])
    qh, kh, hd = st["q_heads"], st["kh"], st["hd"]
    g = qh // kh
    for s, (c, n) in enumerate(zip(st["ctx_host"], st["nodes_host"])):
        r0, seen = _visible(st, s, n)
        pages = st["table"][s, :st["need"][s]].long()
        keys = st["k"][0][pages].float().transpose(0, 1).reshape(kh, -1, hd)[:, :c + n]     # [kv head, position, dim]
        vals = st["v"][0][pages].float().transpose(0, 1).reshape(kh, -1, hd)[:, :c + n]
        q = st["q"][r0:r0 + n].float().reshape(n, kh, g, hd).permute(1, 2, 0, 3).reshape(kh, g * n, hd)
        sc = torch.matmul(q, keys.transpose(1, 2)).reshape(kh, g, n, c + n) * st["scale"]
        sc[..., c:] = torch.where(seen, sc[..., c:], torch.full_like(sc[..., c:], -math.inf))
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(p.reshape(kh, g * n, c + n), vals) / p.sum(-1).reshape(kh, g * n, 1)
        st["out"][r0:r0 + n] = o.reshape(kh, g, n, hd).permute(2, 0, 1, 3).reshape(n, qh * hd).to(torch.bfloat16)
    return st["out"]


def _accept(st):
    if own:
        from affon_b200 import paged
        a = paged.tree_accept(st["batch"], st["parents"], st["tokens"], st["predicted"])
        return a.counts, a.path, a.next_tokens, a.lens, st["k"], st["v"]
    page, dev = st["page"], st["ctx"].device
    seqs, most = len(st["nodes_host"]), max(st["nodes_host"])
    seq, node, first = st["seq_of_row"], st["node_of_row"], st["cu"].long()[:-1]
    par, tok, pred = st["parents"].long(), st["tokens"], st["predicted"]
    which = torch.arange(seqs, device=dev)
    cur = torch.zeros(seqs, dtype=torch.int64, device=dev)
    going = torch.ones(seqs, dtype=torch.bool, device=dev)
    counts = torch.ones(seqs, dtype=torch.int64, device=dev)
    path = torch.full((seqs, most), -1, dtype=torch.int64, device=dev)
    path[:, 0] = 0
    for step in range(1, st["steps"] + 1):
        fits = (par == cur[seq]) & (tok == pred[first + cur][seq])
        best = torch.full((seqs,), most, dtype=torch.int64, device=dev).scatter_reduce(
            0, seq, torch.where(fits, node, torch.full_like(node, most)), "amin")
        going = going & (best < most)
        cur = torch.where(going, best, cur)
        if step < most:
            path[which, step] = torch.where(going, cur, path[which, step])
        counts = counts + going.long()
    d = min(st["steps"], most)
    steps = torch.arange(d, device=dev)[None, :]
    live = steps < counts[:, None]
    src = st["ctx"].long()[:, None] + torch.where(live, path[:, :d], steps.expand(seqs, d).clamp(max=0))
    dst = st["ctx"].long()[:, None] + torch.where(live, steps.expand(seqs, d), torch.zeros_like(steps))
    table = st["table"].long()
    sp, so = table[which[:, None], src // page], src % page
    dp, do = table[which[:, None], dst // page], dst % page
    for t in (st["k"], st["v"]):
        t[:, dp, :, do] = t[:, sp, :, so].clone()
    nxt = pred[first + cur]
    return counts.int(), path.int(), nxt, (st["ctx"].long() + counts).int(), st["k"], st["v"]


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The operator's definition in 64 bits, head by head; None where the outputs are whole numbers and copies."""
    if case["op"] not in ("attention", "append"):
        return None
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    qh, kh, hd, page = st["q_heads"], st["kh"], st["hd"], st["page"]
    ctx, nodes = st["ctx_host"], st["nodes_host"]
    if case["op"] == "append":
        x, pos, slot = st["qkv"].double(), st["positions"].long(), st["slots"].long()
        cos, sin = st["cos"].double()[pos], st["sin"].double()[pos]
        q = torch.empty((st["rows"], qh * hd), dtype=torch.float64, device=x.device)
        k, v = st["k"].double(), st["v"].double()
        lo = torch.arange(hd // 2, device=x.device)
        first, second = (lo, lo + hd // 2) if case["rope"] == "half" else (2 * lo, 2 * lo + 1)
        for h in range(qh + kh):
            a, b = x[:, h * hd + first], x[:, h * hd + second]
            y = torch.empty((st["rows"], hd), dtype=torch.float64, device=x.device)
            y[:, first], y[:, second] = a * cos - b * sin, b * cos + a * sin
            if h < qh:
                q[:, h * hd:(h + 1) * hd] = y
            else:
                k[0][slot // page, h - qh, slot % page] = y
        for h in range(kh):
            v[0][slot // page, h, slot % page] = x[:, (qh + kh + h) * hd:(qh + kh + h + 1) * hd]
        return q, k, v
    out = torch.zeros((st["rows"], qh * hd), dtype=torch.float64, device=st["q"].device)
    g, r0 = qh // kh, 0
    for s, (c, n) in enumerate(zip(ctx, nodes)):
        words = st["mask"][r0:r0 + n].cpu().numpy().view(np.uint32)
        seen = torch.from_numpy(np.array([[words[i, j // 32] >> (j % 32) & 1 for j in range(n)] for i in range(n)],
                                         dtype=bool)).to(out.device)
        at = torch.arange(c + n, device=out.device)
        where, off = st["table"][s].long()[at // page], at % page
        for h in range(kh):
            keys, vals = st["k"][0][where, h, off].double(), st["v"][0][where, h, off].double()
            for i in range(g):
                col = slice((h * g + i) * hd, (h * g + i + 1) * hd)
                z = st["q"][r0:r0 + n, col].double() @ keys.T * st["scale"]
                z[:, c:].masked_fill_(~seen, -math.inf)
                out[r0:r0 + n, col] = torch.softmax(z, dim=-1) @ vals
        r0 += n
    return out
