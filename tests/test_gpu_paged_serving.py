"""The paged cache's and the beam search's operators together, as a program that
serves uses them: prompts and steps appended, attended to, evicted; beams
selected, reordered, gone on with."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import U, UB, Cache, attention, attention_slack, bf16, f64
from test_gpu_kv_paged import plain_evict

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _rope_tab(positions, dim):
    tab = ca.Buffer(positions * dim * 4)
    ca.rope_table_f32(ca.Buffer.from_array(ca.rope_inv_freq(dim, 10000.0)), tab, positions, dim)
    ca.synchronize()
    return tab


def test_bounded_cache_over_many_steps():
    """Two layers' prompts and 40 steps in a cache of 64 slots a row with 48 kept:
    every call against the plain form of what the device holds before it."""
    say("bounded cache")
    rng = np.random.default_rng(41)
    rows, heads, kvh, dim, page, pages, budget, recent, prompt, steps = 3, 6, 2, 64, 16, 4, 48, 8, 40, 40
    group, scale, slots = heads // kvh, dim ** -0.5, page * pages
    tab = _rope_tab(prompt + steps, dim)
    layers = [Cache(rng, [0] * rows, kvh, dim, page, pages) for _ in range(2)]
    for c in layers:
        c.upload()
        c.accb = ca.Buffer.from_array(np.full((rows, kvh, slots), -1, np.float32))
        c.posb = ca.Buffer.from_array(np.full((rows, kvh, slots), 9999, np.uint32))
        c.next = ca.Buffer(4 * rows)
        c.work = ca.Buffer(max(ca.attn_paged_plan(c.kv, heads, True)[1], ca.kv_evict_paged_plan(c.kv, budget), 16))
    seen = np.zeros(rows, np.uint32)
    seenb = ca.Buffer.from_array(seen)
    q, o = ca.Buffer(rows * prompt * heads * dim * 2), ca.Buffer(rows * heads * dim * 4)
    evictions = 0
    for step in range(steps + 1):
        tq = prompt if step == 0 else 1
        seen += tq
        seenb.write(seen)
        for c in layers:
            c.lens = c.lens + np.uint32(tq)
            c.lb.write(c.lens)
            qkv = ca.Buffer.from_array(rng.standard_normal((rows * tq, (heads + 2 * kvh) * dim)).astype(np.float32))
            ca.rope_qkv_paged_bf16(c.kv, qkv, tab, prompt + steps, c.lb, seenb, q, tq, heads, c.accb, c.posb)
            acc, pos = c.accb.read(np.float32, (rows, kvh, slots)), c.posb.read(np.uint32, (rows, kvh, slots))
            c.k, c.v = c.download()
            n = int(c.lens[0])
            assert np.all(acc[:, :, n - tq:n] == 0)
            assert np.array_equal(pos[:, :, n - tq:n], np.broadcast_to(np.arange(seen[0] - tq, seen[0]), (rows, kvh, tq)))
            # the last token's query attends
            q16 = q.read(np.uint16, (rows, tq, heads, dim))[:, -1]
            last = ca.Buffer.from_array(q16)
            ca.attn_paged_bf16(c.kv, last, c.lb, o, heads, scale, c.work, True, c.accb, c.accb)
            got, acc2 = o.read(np.float32, (rows, heads, dim)), c.accb.read(np.float32, (rows, kvh, slots))
            for r in range(rows):
                k, v = f64(c.get(c.k, r, n)), f64(c.get(c.v, r, n))
                for h in range(kvh):
                    mine = slice(h * group, (h + 1) * group)
                    want, p, pv, es = attention(f64(q16[r, mine]), k[h], v[h], scale)
                    slack = attention_slack(es, n)
                    assert np.all(np.abs(got[r, mine] - want) <= slack * pv + U * np.abs(want))
                    total = acc[r, h, :n] + p.sum(0)
                    assert np.all(np.abs(acc2[r, h, :n] - total) <= p.sum(0) * (slack + (group + 2) * U) + U * np.abs(total))
            if n < slots:
                continue
            evictions += 1
            ca.kv_evict_paged_bf16(c.kv, c.lb, seenb, c.accb, c.posb, c.next, c.accb, c.posb, budget, recent, c.work)
            k2, v2 = c.download()
            acc3, pos3 = c.accb.read(np.float32, acc.shape), c.posb.read(np.uint32, pos.shape)
            for r in range(rows):
                for h in range(kvh):
                    to, src = plain_evict(acc2[r, h], pos[r, h], n, int(seen[r]), budget, recent)
                    acc2[r, h, to], pos[r, h, to] = acc2[r, h, src], pos[r, h, src]
                    for pool in (c.k, c.v):
                        pool[c.table[r, to // page], h, to % page] = pool[c.table[r, src // page], h, src % page]
                    # the last positions are all there
                    assert set(range(int(seen[r]) - recent, int(seen[r]))) <= set(pos3[r, h, :budget].tolist())
            assert np.array_equal(acc3, acc2) and np.array_equal(pos3, pos)
            assert np.array_equal(k2, c.k) and np.array_equal(v2, c.v)
            c.lens = c.next.read(np.uint32)
            assert np.all(c.lens == budget)
            c.lb.write(c.lens)
    assert evictions == 4


def test_beam_search_over_shared_pages():
    """Two groups of three beams through 37 steps and three pages, two layers under
    one table that only the device's calls change: every beam's pages hold what
    its own history of tokens appends to a contiguous cache, bit by bit."""
    say("beam search over shared pages")
    rng = np.random.default_rng(42)
    groups, beams, vocab, heads, dim, page, pages, layers, prompt, steps = 2, 3, 96, 2, 64, 16, 4, 2, 11, 37
    rows, wide, eos, slots, scale = groups * beams, 3 * heads * dim, 5, page * pages, dim ** -0.5
    positions = prompt + steps + 1
    tab, inv = _rope_tab(positions, dim), ca.Buffer.from_array(ca.rope_inv_freq(dim, 10000.0))
    # a layer's q | k | v of a token is a row of its embedding; logits come from the first layer's attention
    embed16 = bf16(rng.standard_normal((layers, vocab, wide)))
    embed = [ca.Buffer.from_array(e) for e in embed16]
    lm = ca.Buffer.from_array(bf16(rng.standard_normal((heads * dim, vocab)) * 0.3))
    caches = [Cache(rng, [0] * rows, heads, dim, page, pages, spare=rows) for _ in range(layers)]
    for c in caches:
        c.upload()
    tables = [ca.Buffer.from_array(caches[0].table), ca.Buffer(caches[0].table.nbytes)]
    spares = [ca.Buffer.from_array(caches[0].spare), ca.Buffer(4 * rows)]
    lens2, lensb = ca.Buffer(4 * rows), ca.Buffer(4 * rows)
    kvs = [ca.PagedKV(c.kb.ptr, c.vb.ptr, tables[0].ptr, c.num_pages, page, rows, pages, heads, dim) for c in caches]
    pools = [b for c in caches for b in (c.kb, c.vb)]
    x, q, o16 = ca.Buffer(rows * prompt * wide * 4), ca.Buffer(rows * prompt * heads * dim * 2), ca.Buffer(rows * heads * dim * 2)
    logits, work = ca.Buffer(rows * vocab * 4), ca.Buffer(max(ca.beam_select_plan(groups, beams, vocab), ca.attn_paged_plan(kvs[0], heads)[1], 16))
    tokens, parents, done = (ca.Buffer.from_array(np.zeros(rows, np.uint32)) for _ in range(3))
    first = np.full((groups, beams), -np.inf, np.float32)
    first[:, 0] = 0
    scores = ca.Buffer.from_array(first)
    history = np.repeat(rng.integers(6, vocab, (groups, prompt)), beams, 0).astype(np.uint32)
    tokens_now, shared = history, 0
    for step in range(steps + 1):
        tq = tokens_now.shape[1]
        n = history.shape[1]
        lensb.write(np.full(rows, n, np.uint32))
        ids = ca.Buffer.from_array(np.ascontiguousarray(tokens_now))
        for layer, kv in enumerate(kvs):
            kv.table = tables[0].ptr
            ca.embed_bf16(ids, embed[layer], x, rows * tq, vocab, wide)
            ca.rope_qkv_paged_bf16(kv, x, tab, positions, lensb, None, q, tq, heads)
            if layer == 0:
                q1 = ca.Buffer.from_array(q.read(np.uint16, (rows, tq, heads, dim))[:, -1])
                ca.attn_paged_bf16(kv, q1, lensb, o16, heads, scale, work)
        # every beam's pages against a contiguous cache of its own history
        flat_ids, flat_x = ca.Buffer.from_array(history), ca.Buffer(rows * n * wide * 4)
        fq, fk, fv = ca.Buffer(rows * n * heads * dim * 2), ca.Buffer(rows * heads * slots * dim * 2), ca.Buffer(rows * heads * slots * dim * 2)
        table = tables[0].read(np.uint32, (rows, pages))
        for layer, c in enumerate(caches):
            ca.embed_bf16(flat_ids, embed[layer], flat_x, rows * n, vocab, wide)
            ca.rope_qkv_bf16(flat_x, inv, lensb, fq, fk, fv, rows, n, heads, dim, slots)
            c.table = table
            flats = [b.read(np.uint16, (rows, heads, slots, dim)) for b in (fk, fv)]
            if layer == 0:
                flat0 = [*flats, fq.read(np.uint16, (rows, n, heads, dim))]
            for pool, flat in zip(c.download(), flats):
                for r in range(rows):
                    assert np.array_equal(c.get(pool, r, n), flat[r, :, :n]), (step, layer, r)
        # pages that beams share are filled ones; the page that a row writes is its own
        used = [set(table[r, : -(-n // page)].tolist()) for r in range(rows)]
        tails = [int(table[r, (n - 1) // page]) for r in range(rows)] if n % page else []
        assert len(set(tails)) == len(tails) and not any(t in used[r] for i, t in enumerate(tails) for r in range(rows) if r != i)
        shared += sum(len(used[0] & used[r]) for r in range(1, beams))
        got = f64(o16.read(np.uint16, (rows, heads, dim)))
        ca.gemm_bf16(o16, lm, logits, rows, vocab, heads * dim, True)
        k, v = (f64(flat0[i])[:, :, :n] for i in range(2))
        qq = f64(flat0[2][:, -1])
        for r in range(rows):
            for h in range(heads):
                want, _, pv, es = attention(qq[r, h:h + 1], k[r, h], v[r, h], scale)
                slack = attention_slack(es, n)
                assert np.all(np.abs(got[r, h] - want[0]) <= ((slack + 2.0 ** -16) * pv + UB * (np.abs(want) + slack * pv))[0])
        if step == steps:
            break
        before, lg = scores.read(np.float32, (groups, beams)).astype(np.float64), logits.read(np.float32, (groups, beams, vocab)).astype(np.float64)
        over = done.read(np.uint32, (groups, beams)) != 0
        ca.beam_select_f32(logits, scores, done, tokens, parents, scores, done, groups, beams, vocab, eos, work)
        ca.beam_reorder_paged_bf16(kvs[0], pools, lensb, parents, spares[0], tables[1], lens2, spares[1])
        tables.reverse(), spares.reverse()
        t, p = tokens.read(np.uint32), parents.read(np.uint32)
        assert np.all(lens2.read(np.uint32) == n)
        # the scores are those of the continuations named, and none that was left out is above them
        top = lg.max(-1, keepdims=True)
        total = before[..., None] + lg - top - np.log(np.exp(lg - top).sum(-1, keepdims=True))
        total[over] = -np.inf
        total[over, eos] = before[over]
        after = scores.read(np.float32, (groups, beams))
        for g in range(groups):
            named = total[g, p[g * beams:(g + 1) * beams] - g * beams, t[g * beams:(g + 1) * beams]]
            assert np.all(np.abs(after[g] - named) <= (2 * 64 + 18) * U + U * np.abs(named))
            assert np.all(np.diff(after[g]) <= 0)
            left = total[g].copy()
            left[p[g * beams:(g + 1) * beams] - g * beams, t[g * beams:(g + 1) * beams]] = -np.inf
            assert left.max() <= after[g].min() + 300 * U
        tokens_now = t[:, None]
        history = np.concatenate([history[p], tokens_now], 1)
    assert shared > 0


def test_prompt_attends_over_pages():
    """A prompt's tokens as rows of their own whose tables are the sequence's: causal
    attention over the pages that the append has just filled."""
    say("prompt over pages")
    rng = np.random.default_rng(43)
    heads, kvh, dim, page, pages, tq, old = 6, 2, 128, 32, 5, 70, 33
    cache = Cache(rng, [old + tq], kvh, dim, page, pages)
    kv = cache.upload()
    tab = _rope_tab(old + tq, dim)
    q, o = ca.Buffer(tq * heads * dim * 2), ca.Buffer(tq * heads * dim * 2)
    qkv = ca.Buffer.from_array(rng.standard_normal((tq, (heads + 2 * kvh) * dim)).astype(np.float32))
    ca.rope_qkv_paged_bf16(kv, qkv, tab, old + tq, cache.lb, None, q, tq, heads)
    tables = ca.Buffer.from_array(np.repeat(cache.table, tq, 0))
    lens = ca.Buffer.from_array(np.arange(old + 1, old + tq + 1, dtype=np.uint32))
    each = ca.PagedKV(kv.k, kv.v, tables.ptr, kv.num_pages, page, tq, pages, kvh, dim)
    work = ca.Buffer(max(ca.attn_paged_plan(each, heads)[1], 16))
    ca.attn_paged_bf16(each, q, lens, o, heads, dim ** -0.5, work)
    got, q16 = f64(o.read(np.uint16, (tq, heads, dim))), f64(q.read(np.uint16, (tq, heads, dim)))
    k, v = (f64(cache.get(pool, 0, old + tq)) for pool in cache.download())
    group = heads // kvh
    for t in range(tq):
        n = old + t + 1
        for h in range(kvh):
            mine = slice(h * group, (h + 1) * group)
            want, _, pv, es = attention(q16[t, mine], k[h, :n], v[h, :n], dim ** -0.5)
            slack = attention_slack(es, n)
            assert np.all(np.abs(got[t, mine] - want) <= (slack + 2.0 ** -16) * pv + UB * (np.abs(want) + slack * pv)), (t, h)
