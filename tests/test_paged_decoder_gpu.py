"""The decoder over a paged cache: plain steps against the contiguous-cache
decoder of the same weights, drafted trees against a float32 restatement of
every node's path, and the graph-captured step."""
import math

import numpy as np
import pytest
import torch

import paged_ref as ref
from affon_b200.core import AffonError
from affon_b200.decoder import LlamaConfig, PagedDecoder, QuantizedDecoder
from test_decoder_gpu import bf16, normed_proj, rope

pytestmark = pytest.mark.gpu

SMALL = LlamaConfig(layers=2, d_model=512, q_heads=4, kv_heads=1, head_dim=128, ffn=1024, vocab=1000)
SMALL_G8 = LlamaConfig(layers=2, d_model=1024, q_heads=16, kv_heads=2, head_dim=128, ffn=2048, vocab=1000)
SMALL_8BIT = LlamaConfig(layers=2, d_model=512, q_heads=8, kv_heads=2, head_dim=128, ffn=1536, vocab=1000, bits=8)


def cached(dec, layer, seq, length):
    """Keys and values [kv_heads, length, hd] of a sequence, float32."""
    at = torch.arange(length, device=dec.device)
    pages = dec.page_table[seq].long()[at // dec.page_size]
    take = lambda pool: pool[layer][pages, :, at % dec.page_size].float().transpose(0, 1)
    return take(dec.k_cache), take(dec.v_cache)


def ref_tree(dec, seq, ctx, parents, tokens):
    """float32 residual rows, logits and bf16-rounded keys/values of a tree over a sequence's first ctx positions."""
    c = dec.cfg
    G, hd, n = c.q_heads // c.kv_heads, c.head_dim, len(tokens)
    seen = torch.from_numpy(ref.ancestors(parents)).to(dec.device)
    pos = ctx + seen.sum(-1) - 1
    cos, sin = dec.cos[pos][:, None], dec.sin[pos][:, None]
    h = dec.embed[torch.as_tensor(tokens, device=dec.device).long()].float()
    kept = []
    for li, lay in enumerate(dec.layers):
        qkv = bf16(normed_proj(h, lay["attn_norm"], lay["qkv"], c.eps))
        q = qkv[:, :c.q_heads * hd].reshape(n, c.q_heads, hd)
        k = qkv[:, c.q_heads * hd:(c.q_heads + c.kv_heads) * hd].reshape(n, c.kv_heads, hd)
        v = qkv[:, (c.q_heads + c.kv_heads) * hd:].reshape(n, c.kv_heads, hd)
        q, k = bf16(rope(q, cos, sin)), bf16(rope(k, cos, sin))
        kept.append((k, v))
        pk, pv = cached(dec, li, seq, ctx)
        keys = torch.cat([pk, k.transpose(0, 1)], 1).repeat_interleave(G, 0)
        vals = torch.cat([pv, v.transpose(0, 1)], 1).repeat_interleave(G, 0)
        z = torch.einsum("nhd,htd->nht", q, keys) / math.sqrt(hd)
        z[:, :, ctx:] = z[:, :, ctx:].masked_fill(~seen[:, None, :], -math.inf)
        attn = bf16(torch.einsum("nht,htd->nhd", torch.softmax(z, -1), vals).reshape(n, -1))
        h = h + attn @ lay["o"].dequantized().T
        gu = normed_proj(h, lay["ffn_norm"], lay["gate_up"], c.eps).reshape(n, -1, 2, 8)
        act = bf16(torch.nn.functional.silu(gu[:, :, 0].reshape(n, -1)) * gu[:, :, 1].reshape(n, -1))
        h = h + act @ lay["down"].dequantized().T
    return h, normed_proj(h, dec.final_norm, dec.lm_head, c.eps), kept


def clear(logits):
    top = torch.topk(logits, 2, dim=-1)
    return (top.values[:, 0] - top.values[:, 1]) > 2e-2 * top.values[:, 0].abs().clamp(min=1), top.indices[:, 0]


@pytest.mark.parametrize("cfg,rows,nodes,page", [(SMALL, 16, [5, 8, 1], 16), (SMALL_G8, 32, [12, 0, 20], 32),
                                                 (SMALL_8BIT, 8, [3, 4], 64)], ids=["4q", "8q-empty", "8bit"])
def test_drafted_step_matches_float32_reference(cfg, rows, nodes, page):
    seqs = len(nodes)
    rng = np.random.default_rng(rows)
    d = PagedDecoder(cfg, seqs, rows, "cuda:0", capacity=192, pages=seqs * 192 // page, page_size=page, seed=2)
    try:
        lens = [37, 0, 90][:seqs]
        d.prefill([rng.integers(0, cfg.vocab, size=n).tolist() for n in lens])
        d.synchronize()
        assert d.ctx_lens.tolist() == lens
        parents = [ref.random_forest(n, rng) for n in nodes]
        tokens = [rng.integers(0, cfg.vocab, size=n) for n in nodes]
        want = [ref_tree(d, s, lens[s], parents[s], tokens[s]) if nodes[s] else None for s in range(seqs)]
        for s in range(seqs):
            # some drafts right: a child of the root is what the reference predicts there
            ok, best = clear(want[s][1]) if nodes[s] > 1 else (torch.zeros(1, dtype=torch.bool), None)
            kids = [j for j in range(nodes[s]) if parents[s][j] == 0]
            if ok[0] and kids:
                tokens[s][kids[-1]] = int(best[0])
                want[s] = ref_tree(d, s, lens[s], parents[s], tokens[s])
        for s in range(seqs):
            d.reserve(s, lens[s] + nodes[s])
        d.set_step(nodes, np.concatenate(parents), np.concatenate(tokens))
        d.step_eager()
        d.synchronize()
        predicted, at = d.predicted.cpu().numpy(), 0
        for s, n in enumerate(nodes):
            if n == 0:
                assert int(d.accepted.counts[s]) == 0 and int(d.ctx_lens[s]) == lens[s]
                continue
            h, logits, kept = want[s]
            got = d.h[at:at + n]
            assert float((got - h).abs().max()) <= 2e-2 * float(h.abs().max())
            ok, best = clear(logits)
            assert torch.equal(torch.from_numpy(predicted[at:at + n]).to(best.device)[ok].long(), best[ok])
            step = ref.Step([lens[s]], [n], page, parents=[parents[s]])
            counts, path, nxt, new = ref.accept(step, tokens[s], predicted[at:at + n])
            assert d.accepted.counts[s] == counts[0] and d.ctx_lens[s] == new[0]
            assert d.accepted.path[s, :n].tolist() == path[0].tolist() and int(d.accepted.next_tokens[s]) == nxt[0]
            line = path[0][:counts[0]].tolist()
            for li in range(cfg.layers):
                k, v = cached(d, li, s, int(new[0]))
                for pool, exact in ((k, kept[li][0]), (v, kept[li][1])):
                    rows_ = exact[line].transpose(0, 1)
                    assert float((pool[:, lens[s]:] - rows_).abs().max()) <= 2e-2 * max(1.0, float(rows_.abs().max()))
            at += n
    finally:
        d.close()


def test_plain_steps_fill_the_first_layer_like_the_contiguous_decoder():
    """Same weights, the same tokens at the same positions: the first layer's keys and values come from the same
    projection bits, so values are equal and keys (each a rotation in f32 rounded once to bf16: half a step, 2^-8
    relative, and 2^-22 of the rotated pair's magnitudes) differ by at most two such errors.  Deeper layers differ by
    the two attentions' roundings and are compared with a float32 restatement above."""
    B, T = 4, 21
    gen = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, SMALL.vocab, (T, B), generator=gen)
    a = QuantizedDecoder(SMALL, batch=B, capacity=64, device="cuda:0", seed=7, max_steps=16)
    b = PagedDecoder(SMALL, B, B, "cuda:0", capacity=64, pages=2 * B, page_size=32, seed=7)
    try:
        a.prefill(prompt)
        b.prefill([prompt[:, s].tolist() for s in range(B)])
        for step in range(6):
            toks = torch.randint(0, SMALL.vocab, (B,), generator=gen, dtype=torch.int32)
            a.tokens.copy_(toks)
            for s in range(B):
                b.reserve(s, T + step + 1)
            b.set_step([1] * B, tokens=toks.tolist())
            a.step_eager()
            b.step_eager()
        a.synchronize()
        b.synchronize()
        assert b.ctx_lens.tolist() == [T + 6] * B and int(a.pos) == T + 6
        for s in range(B):
            k, v = cached(b, 0, s, T + 6)
            ka, va = (t[0][s, :, :T + 6].float() for t in (a.k_cache, a.v_cache))
            assert torch.equal(v, va)
            pair = ka.abs() + ka.roll(64, -1).abs()
            assert ((k - ka).abs() <= 2 * (2.0 ** -8 * ka.abs() * 1.01 + 2.0 ** -21 * pair)).all()
    finally:
        a.close()
        b.close()


@pytest.mark.parametrize("overlap", [False, True])
def test_captured_steps_equal_eager_ones(overlap):
    outs = []
    for captured in (False, True):
        d = PagedDecoder(SMALL, 3, 12, "cuda:0", capacity=128, pages=24, page_size=16, seed=5, overlap=overlap)
        try:
            rng = np.random.default_rng(1)
            d.prefill([rng.integers(0, SMALL.vocab, size=n).tolist() for n in (9, 30, 2)])
            for s in range(3):
                d.reserve(s, 100)
            if captured:
                d.set_step([4, 4, 4], tokens=[0] * 12)
                d.capture()
            seen = []
            for _ in range(4):
                par = np.concatenate([ref.random_forest(4, rng) for _ in range(3)])
                d.set_step([4, 4, 4], par, rng.integers(0, SMALL.vocab, size=12))
                d.replay() if captured else d.step_eager()
                d.synchronize()
                seen += [d.predicted.clone(), d.accepted.counts.clone(), d.ctx_lens.clone(), d.h.clone()]
            outs.append(seen + [d.k_cache.clone(), d.v_cache.clone()])
        finally:
            d.close()
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_pages_are_shared_out_and_overruns_reported():
    d = PagedDecoder(SMALL, 2, 4, "cuda:0", capacity=64, pages=3, page_size=16, seed=5)
    try:
        d.reserve(0, 30)
        with pytest.raises(ValueError):
            d.reserve(1, 30)                     # one page is left
        with pytest.raises(ValueError):
            d.reserve(1, 65)
        with pytest.raises(ValueError):
            d.set_step([3, 2])
        with pytest.raises(ValueError):
            d.set_step([2, 2], parents=[-1])
        with pytest.raises(ValueError):
            d.set_step([2, 2], tokens=[1, 2, 3])
        d.release(0)
        d.reserve(1, 48)
        d.prefill([[], list(range(48))])
        d.synchronize()
        assert d.ctx_lens.tolist() == [0, 48]
        # pages that a sequence gave back are not its any more, whatever its length says
        d.release(1)
        d.reserve(1, 10)
        d.reserve(0, 10)
        k0 = d.k_cache.clone()
        d.ctx_lens[1] = 20
        d.set_step([0, 1], tokens=[1])
        d.step_eager()
        with pytest.raises(AffonError):
            d.synchronize()
        assert torch.equal(d.k_cache, k0)
        d.reset()
        k0 = d.k_cache.clone()
        d.ctx_lens[1] = 62                       # three more nodes pass the page table's end
        d.set_step([0, 3], tokens=[1, 2, 3])
        d.step_eager()
        with pytest.raises(AffonError) as err:
            d.synchronize()
        assert err.value.code == "invalid_arg"
        assert torch.equal(d.k_cache, k0) and int(d.ctx_lens[1]) == 62
    finally:
        d.close()


def test_no_length_passes_nodes_without_a_page():
    d = PagedDecoder(SMALL, 2, 6, "cuda:0", capacity=64, pages=3, page_size=16, seed=5)
    try:
        d.prefill([list(range(1, 15)), [1, 2, 3]])
        d.synchronize()
        d.set_step([3, 2], tokens=[1, 2, 3, 4, 5])           # the first one's third node is position 16
        d._accept, d._follow = False, torch.tensor([2, 3, -1, 5, -1, 0], dtype=torch.int32, device=d.device)
        k0 = d.k_cache.clone()
        d.step_eager()
        with pytest.raises(AffonError):
            d.synchronize()
        assert d.ctx_lens.tolist() == [14, 5]
        free = [p for p in range(3) if p not in d._pages_of[0] + d._pages_of[1]]
        assert torch.equal(d.k_cache[:, free], k0[:, free])
    finally:
        d.close()


def state(d):
    """Every device tensor that a decoder's next steps or its user read."""
    a, p = d.accepted, d.plan
    return [d.k_cache, d.v_cache, d.ctx_lens, d.cu_nodes, d.parents, d.tokens, d.predicted, d.page_table, d.h, d.ss,
            d.xq, d.qkv, d.q, d.attn, d.act, d.amax, d.pos, d.step_ctr, p.positions, p.slots, p.mask, a.counts, a.path,
            a.next_tokens]


def drafted(d, nodes, rng):
    d.set_step(nodes, np.concatenate([ref.random_forest(n, rng) for n in nodes]),
               rng.integers(0, d.cfg.vocab, size=sum(nodes)))


def test_timing_the_roles_leaves_the_paged_cache_as_it_was():
    """step_breakdown between steps, with no page to spare behind the last node."""
    d = PagedDecoder(SMALL, 3, 12, "cuda:0", capacity=128, pages=24, page_size=16, seed=5)
    try:
        rng = np.random.default_rng(1)
        d.prefill([rng.integers(0, SMALL.vocab, size=n).tolist() for n in (9, 30, 2)])
        for nodes in ([4, 4, 4], [1, 6, 0]):
            for s, n in enumerate(nodes):
                d.reserve(s, int(d.ctx_lens[s]) + n)
            drafted(d, nodes, rng)
            d.step_eager()
            d.synchronize()
            before = [t.clone() for t in state(d)]
            parts = d.step_breakdown()
            d.synchronize()                      # nothing was reported
            for t, was in zip(state(d), before):
                assert torch.equal(t, was)
            assert {"plan", "append", "attn", "accept", "qkv", "embed", "finalize"} <= set(parts)
            assert all(ms > 0 for ms, _ in parts.values())
            assert sum(n for _, n in parts.values()) == d.launches_per_step()
    finally:
        d.close()


def test_timing_the_roles_of_a_decoder_without_pages():
    d = PagedDecoder(SMALL, 2, 4, "cuda:0", capacity=64, pages=3, page_size=16, seed=5)
    try:
        before = [t.clone() for t in state(d)]
        for role in ("plan", "append", "attn", "accept"):
            assert d.role_time_ms(role) > 0
        d.set_step([3, 1], tokens=[1, 2, 3, 4])
        d.reserve(0, 2)
        after = [t.clone() for t in state(d)]
        for role in ("plan", "append", "attn", "accept"):
            assert d.role_time_ms(role) > 0
        d.synchronize()
        for t, was, now in zip(state(d), before, after):
            assert torch.equal(t, now)
        assert torch.equal(d.k_cache, before[0])
    finally:
        d.close()


def test_a_capacity_that_ends_inside_a_page():
    """Sequences hold whole pages: steps across the capacity asked for are those of a decoder that was asked for the
    whole page, and steps across the last page leave everything as it was."""
    outs = []
    for capacity in (100, 128):
        d = PagedDecoder(SMALL, 1, 4, "cuda:0", capacity=capacity, pages=2, page_size=64, seed=5)
        try:
            rng = np.random.default_rng(1)
            d.prefill([rng.integers(0, SMALL.vocab, size=99).tolist()])
            d.set_step([3], tokens=[5, 6, 7])
            d.step_eager()
            d.synchronize()
            got = [t.clone() for t in state(d)]
            assert got[2].tolist() == [99 + int(d.accepted.counts[0])]
            outs.append(got)
            d.ctx_lens[0] = 126
            k0, v0 = d.k_cache.clone(), d.v_cache.clone()
            d.step_eager()
            with pytest.raises(AffonError) as err:
                d.synchronize()
            assert err.value.code == "invalid_arg" and d.ctx_lens.tolist() == [126]
            assert torch.equal(d.k_cache, k0) and torch.equal(d.v_cache, v0)
            with pytest.raises(ValueError):
                d.reserve(0, 129)
        finally:
            d.close()
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_a_prompt_joins_running_sequences():
    """prefill(keep=True) feeds prompts to some sequences and leaves the others, their next tokens included; the joined
    sequence holds, bit for bit, what it holds when it is alone."""
    rng = np.random.default_rng(4)
    first, second, more = (rng.integers(0, SMALL.vocab, size=n).tolist() for n in (21, 30, 7))
    made = lambda: PagedDecoder(SMALL, 2, 8, "cuda:0", capacity=128, pages=16, page_size=16, seed=5)
    d, alone = made(), made()
    try:
        d.prefill([first, []])
        for _ in range(3):
            d.reserve(0, int(d.ctx_lens[0]) + 1)
            d.set_step([1, 0], tokens=[int(d.accepted.next_tokens[0])])
            d.step_eager()
        d.synchronize()
        k, v = cached(d, 1, 0, 24)
        nxt = int(d.accepted.next_tokens[0])
        d.prefill([[], second], keep=True)
        d.synchronize()
        alone.prefill([[], second])
        alone.synchronize()
        assert d.ctx_lens.tolist() == [24, 30]
        assert d.accepted.next_tokens.tolist() == [nxt, int(alone.accepted.next_tokens[1])]
        for got, want in zip(cached(d, 1, 0, 24), (k, v)):
            assert torch.equal(got, want)
        d.prefill([[], more], keep=True)                     # a sequence's own prompt goes on, too
        alone.prefill([[], more], keep=True)
        d.synchronize()
        alone.synchronize()
        for li in range(SMALL.layers):
            for got, want in zip(cached(d, li, 1, 37), cached(alone, li, 1, 37)):
                assert torch.equal(got, want)
        # what does not fit is refused before anything is lost
        for prompts, keep in (([[1] * 129, []], False), ([[1] * 105, []], True), ([[1]], True)):
            with pytest.raises(ValueError):
                d.prefill(prompts, keep=keep)
        assert d.ctx_lens.tolist() == [24, 37]
        # captured steps go on as they were
        d.reserve(0, 25)
        d.reserve(1, 38)
        d.set_step([1, 1], tokens=d.accepted.next_tokens.tolist())
        d.capture()
        d.replay()
        d.synchronize()
        assert d.ctx_lens.tolist() == [25, 38]
    finally:
        d.close()
        alone.close()
