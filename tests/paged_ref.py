"""Plain restatements, in 64 bits on the CPU, of the paged-cache operators,
and the cases that their tests build from them."""
import math

import numpy as np
import torch


def random_forest(n, rng, roots=False):
    """Parents of n nodes: each node hangs below any earlier one (with `roots`, some below none)."""
    par = np.full(n, -1, dtype=np.int32)
    for i in range(1, n):
        par[i] = rng.integers(-1 if roots else 0, i)
    return par


def ancestors(par):
    """bool [n, n]: node i sees j (itself or an ancestor)."""
    n = len(par)
    m = np.zeros((n, n), dtype=bool)
    for i in range(n):
        if par[i] >= 0:
            m[i] = m[par[i]]
        m[i, i] = True
    return m


def pack(seen, words):
    """bool [n, n] -> int32 words [n, words], bit j of word j/32."""
    n = seen.shape[0]
    bits = np.zeros((n, words * 32), dtype=np.uint64)
    bits[:, :n] = seen
    w = (bits.reshape(n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32).view(np.int32)


class Step:
    """A ragged step: lengths, trees and a scattered page table, all on the host."""

    def __init__(self, ctx, nodes, page, seed=0, parents=None, pad=0, spare=2, roots=False):
        rng = np.random.default_rng(seed)
        self.ctx, self.nodes, self.page, self.pad = list(ctx), list(nodes), page, pad
        self.seqs, self.rows = len(ctx), sum(nodes) + pad
        self.max_nodes = max(1, max(nodes))
        self.words = -(-self.max_nodes // 32)
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        need = [max(1, -(-(c + n) // page)) for c, n in zip(ctx, nodes)]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.zeros((self.seqs, max(need)), dtype=np.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = order[at:at + k]
            at += k
        if parents is None:
            parents = [random_forest(n, rng, roots) for n in nodes]
        elif isinstance(parents, str):   # "chain"
            parents = [np.arange(-1, n - 1, dtype=np.int32) for n in nodes]
        self.parents = parents

    def place(self, s, i):
        """(page, position) of cache position i of sequence s."""
        return int(self.table[s, i // self.page]), i % self.page

    def flat_parents(self):
        return np.concatenate(self.parents + [np.full(self.pad, -1, dtype=np.int32)]).astype(np.int32)

    def plan(self):
        positions = np.zeros(self.rows, dtype=np.int32)
        slots = np.full(self.rows, -1, dtype=np.int32)
        mask = np.zeros((self.rows, self.words), dtype=np.int32)
        for s in range(self.seqs):
            a, n = self.cu[s], self.nodes[s]
            seen = ancestors(self.parents[s])
            if n:
                mask[a:a + n] = pack(seen, self.words)
            for i in range(n):
                positions[a + i] = self.ctx[s] + seen[i].sum() - 1
                pg, off = self.place(s, self.ctx[s] + i)
                slots[a + i] = pg * self.page + off
        return positions, slots, mask


def gather(step, pool, s, length):
    """[kv_heads, length, head_dim] float64 of one sequence from a [pages, kv_heads, page, head_dim] pool."""
    at = torch.arange(length)
    pages = torch.from_numpy(step.table[s].astype(np.int64))[at // step.page]
    return pool[pages, :, at % step.page].double().transpose(0, 1)


def attention(step, q, k, v, q_heads, scale, seen=None):
    """(out, bound): exact attention in float64 [rows, q_heads*hd] (NaN in padding rows) and the largest error a
    kernel may make that rounds each probability to bf16 (half a step: 2^-8 relative), sums in f32, and rounds the
    result to bf16.

    With weights p (1 + d), |d| <= 2^-8 + eta, the quotient is off by sum p d (v - o) / sum p (1 + d); eta covers the
    f32 score (head_dim products: head_dim 2^-24 sum |q k| scale, as an absolute error of the exponent) and 2^-15
    for exp and the f32 sums; then one rounding of the result."""
    pages, kh, page, hd = k.shape
    g = q_heads // kh
    out = torch.full((step.rows, q_heads * hd), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for s in range(step.seqs):
        a, n, c = int(step.cu[s]), step.nodes[s], step.ctx[s]
        if n == 0:
            continue
        see = torch.from_numpy(ancestors(step.parents[s]) if seen is None else seen[s])
        keys, vals = gather(step, k, s, c + n), gather(step, v, s, c + n)
        for h in range(q_heads):
            cols = slice(h * hd, (h + 1) * hd)
            x = q[a:a + n, cols].double()
            kk, vv = keys[h // g], vals[h // g]
            z = x @ kk.T * scale
            full = torch.cat([torch.ones((n, c), dtype=torch.bool), see], dim=1)
            z = torch.where(full, z, torch.full_like(z, -math.inf))
            m = z.amax(-1, keepdim=True)
            p = torch.where(full, torch.exp(z - torch.where(m.isinf(), torch.zeros_like(m), m)), torch.zeros_like(z))
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, torch.ones_like(l), l)
            # hidden places contribute nothing, whatever they hold
            clean = lambda t: torch.where(t.isfinite(), t, torch.zeros_like(t))
            o = p @ clean(vv)
            for j in torch.nonzero(~vv.isfinite().all(-1)).flatten().tolist():
                o = torch.where(full[:, j:j + 1], o + torch.where(vv[j].isfinite(), torch.zeros_like(vv[j]), vv[j]), o)
            far = torch.einsum("nt,tnd->nd", p, (clean(vv)[:, None, :] - clean(o)[None]).abs()) if n * (c + n) * hd \
                < 1 << 24 else p @ clean(vv).abs() + clean(o).abs()
            eta = hd * 2.0 ** -24 * scale * float((x.abs() @ clean(kk).abs().T).nan_to_num(0, 0, 0).max()) + 2.0 ** -15
            out[a:a + n, cols] = o
            bound[a:a + n, cols] = (2.0 ** -8 + 2 * eta) * far * 1.01 + 2.0 ** -8 * o.abs() * 1.01 + 1e-30
    return out, bound


def rotate(x, cos, sin, mode):
    """float64 rotation of [rows, heads, hd] by per-row tables [rows, hd/2]."""
    c, s = cos[:, None, :], sin[:, None, :]
    hd = x.shape[-1]
    y = torch.empty_like(x)
    if mode == "half":
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        y[..., :hd // 2], y[..., hd // 2:] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y[..., 0::2], y[..., 1::2] = a * c - b * s, b * c + a * s
    return y


def accept(step, tokens, predicted):
    """(counts, path, next, lens) by the plain walk."""
    counts, nxt, lens = [], [], []
    path = np.full((step.seqs, step.max_nodes), -1, dtype=np.int32)
    for s in range(step.seqs):
        a, n = int(step.cu[s]), step.nodes[s]
        cur, got = (0 if n else -1), []
        while cur >= 0:
            got.append(cur)
            want = predicted[a + cur]
            cur = next((i for i in range(n) if step.parents[s][i] == cur and tokens[a + i] == want), -1)
        path[s, :len(got)] = got
        counts.append(len(got))
        nxt.append(int(predicted[a + got[-1]]) if got else -1)
        lens.append(step.ctx[s] + len(got))
    return np.array(counts), path, np.array(nxt), np.array(lens)


def move_accepted(step, pool, path, counts):
    """pool [layers, pages, kv_heads, page, hd] with the accepted rows moved together (a new tensor)."""
    out = pool.clone()
    for s in range(step.seqs):
        for i in range(int(counts[s])):
            sp, so = step.place(s, step.ctx[s] + int(path[s, i]))
            dp, do = step.place(s, step.ctx[s] + i)
            out[:, dp, :, do] = pool[:, sp, :, so]
    return out
