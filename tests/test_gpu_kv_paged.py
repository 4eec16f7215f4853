"""Upkeep of a cache in pages: append, eviction and reordering against plain
forms on the host.  Rotations are held to the framework's own append bit by
bit, moves and tables are whole numbers."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from paged_util import U, UB, Cache, bf16, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _table(positions, dim):
    theta = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(dim // 2) / (dim // 2))
    return np.stack([np.cos(theta), np.sin(theta)], -1).astype(np.float32)


def _rotated(x, tab):
    """x [..., dim] in 64 bits by tab [..., dim/2, 2], and the bound of its bf16
    form: three f32 roundings and one to bf16."""
    a, b = np.split(x, 2, -1)
    c, s = tab[..., 0].astype(np.float64), tab[..., 1].astype(np.float64)
    y = np.concatenate([a * c - b * s, b * c + a * s], -1)
    big = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    return y, UB * np.abs(y) + 3 * U * big


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("heads,kvh,dim,page,pages,tq,lens,ahead", [
    (16, 16, 128, 16, 3, 1, [1, 16, 17, 48], 0),
    (8, 2, 64, 32, 2, 1, [1, 33, 64], 900),
    (7, 1, 128, 64, 3, 40, [40, 41, 100, 190], 5),       # tokens that cross pages
    (64, 8, 128, 16, 40, 500, [500, 640], 0),            # more than one workgroup a token
    (3, 3, 64, 16, 2, 20, [20, 32], 1),
])
def test_append(heads, kvh, dim, page, pages, tq, lens, ahead):
    say(f"append heads {heads}/{kvh} dim {dim} page {page} tq {tq}")
    rng = np.random.default_rng(heads * tq + dim)
    cache = Cache(rng, lens, kvh, dim, page, pages)
    rows = len(lens)
    qkv = rng.standard_normal((rows, tq, heads + 2 * kvh, dim)).astype(np.float32)
    seen = cache.lens + np.uint32(ahead)
    tab = _table(int(seen.max()), dim)
    acc = rng.random((rows, kvh, cache.slots)).astype(np.float32)
    where = rng.integers(0, 1000, acc.shape).astype(np.uint32)
    kv = cache.upload()
    accb, posb, q = ca.Buffer.from_array(acc), ca.Buffer.from_array(where), ca.Buffer(rows * tq * heads * dim * 2)
    ca.rope_qkv_paged_bf16(kv, ca.Buffer.from_array(qkv), ca.Buffer.from_array(tab), len(tab), cache.lb,
                           ca.Buffer.from_array(seen) if ahead else None, q, tq, heads, accb, posb)
    got_q = f64(q.read(np.uint16, (rows, tq, heads, dim)))
    k, v = cache.download()
    acc2, pos2 = accb.read(np.float32, acc.shape), posb.read(np.uint32, acc.shape)
    want_k, want_v = cache.k.copy(), cache.v.copy()
    for r, n in enumerate(lens):
        slots, pos = np.arange(n - tq, n), np.arange(n - tq, n) + ahead
        y, tol = _rotated(qkv[r, :, :heads + kvh].astype(np.float64), tab[pos][:, None])
        assert np.all(np.abs(got_q[r] - y[:, :heads]) <= tol[:, :heads])
        at = (cache.table[r, slots // page], slice(None), slots % page)
        assert np.all(np.abs(f64(k[at]) - y[:, heads:]) <= tol[:, heads:])
        assert np.array_equal(v[at], bf16(qkv[r, :, heads + kvh:]))
        want_k[at], want_v[at] = k[at], v[at]
        acc[r, :, slots] = 0
        where[r, :, slots] = pos[:, None]
    # and nothing else changed
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)
    assert np.array_equal(acc2, acc) and np.array_equal(pos2, where)


def test_append_matches_the_contiguous_append():
    """One kv head a head, the stdlib's rotation table: the bits of
    rope_qkv_bf16."""
    say("append against rope_qkv_bf16")
    rng = np.random.default_rng(3)
    rows, tq, heads, dim, max_len = 3, 5, 4, 128, 48
    lens = np.array([5, 21, 48], np.uint32)
    qkv = ca.Buffer.from_array(rng.standard_normal((rows * tq, 3 * heads * dim)).astype(np.float32))
    inv = ca.Buffer.from_array(ca.rope_inv_freq(dim, 10000.0))
    lb = ca.Buffer.from_array(lens)
    q1, k1, v1 = ca.Buffer(rows * tq * heads * dim * 2), ca.Buffer(rows * heads * max_len * dim * 2), ca.Buffer(rows * heads * max_len * dim * 2)
    ca.rope_qkv_bf16(qkv, inv, lb, q1, k1, v1, rows, tq, heads, dim, max_len)
    tab = ca.Buffer(max_len * dim * 4)
    ca.rope_table_f32(inv, tab, max_len, dim)
    cache = Cache(rng, [0, 0, 0], heads, dim, 16, 3)
    kv = cache.upload()
    q2 = ca.Buffer(q1.nbytes)
    ca.rope_qkv_paged_bf16(kv, qkv, tab, max_len, lb, None, q2, tq, heads)
    assert np.array_equal(q1.read(np.uint16), q2.read(np.uint16))
    k, v = cache.download()
    for pool, flat in ((k, k1), (v, v1)):
        flat = flat.read(np.uint16, (rows, heads, max_len, dim))
        for r, n in enumerate(lens):
            assert np.array_equal(cache.get(pool, r, int(n))[:, n - tq:], flat[r, :, n - tq:n])


def test_append_without_a_place():
    """Slots outside the table, positions outside the rotations, pages outside
    the pool: q alone, turned by the first position where there is no other."""
    say("append without a place")
    rng = np.random.default_rng(4)
    kvh, dim, tq = 2, 64, 2
    cache = Cache(rng, [1, 40, 18, 20, 10], kvh, dim, 16, 2)  # shorter than tq; past 32 slots; a bad page; past the rotations; good
    seen = np.array([1, 40, 18, 600, 10], np.uint32)
    cache.table[2, 1] = cache.num_pages
    tab = _table(100, dim)
    qkv = rng.standard_normal((5, tq, 2 * kvh + 4, dim)).astype(np.float32)
    acc = rng.random((5, kvh, 32)).astype(np.float32)
    kv = cache.upload()
    accb, posb, q = ca.Buffer.from_array(acc), ca.Buffer.from_array(np.full(acc.shape, 9, np.uint32)), ca.Buffer(5 * tq * 4 * dim * 2)
    ca.rope_qkv_paged_bf16(kv, ca.Buffer.from_array(qkv), ca.Buffer.from_array(tab), 100, cache.lb,
                           ca.Buffer.from_array(seen), q, tq, 4, accb, posb)
    got = f64(q.read(np.uint16, (5, tq, 4, dim)))
    for r, pos in enumerate(([0, 0], [0, 0], [16, 17], [0, 0], [8, 9])):
        y, tol = _rotated(qkv[r, :, :4].astype(np.float64), tab[pos][:, None])
        assert np.all(np.abs(got[r] - y) <= tol), r
    k, v = cache.download()
    slots = np.array([8, 9])
    at = (cache.table[4, slots // 16], slice(None), slots % 16)
    for new, old in ((k, cache.k), (v, cache.v)):
        assert not np.array_equal(new[at], old[at])
        new[at] = old[at]
        assert np.array_equal(new, old)
    acc[4, :, slots] = 0
    assert np.array_equal(accb.read(np.float32, acc.shape), acc)
    where = np.full(acc.shape, 9, np.uint32)
    where[4, :, slots] = slots[:, None]
    assert np.array_equal(posb.read(np.uint32, acc.shape), where)


# ---------------------------------------------------------------- eviction

def plain_evict(acc, pos, n, seen, budget, recent):
    """(slots filled, slots they are filled from) of one (row, kv head)."""
    late = seen - min(recent, seen)
    w = acc[:n].astype(np.float64)
    first = np.where(pos[:n] >= late, 0, np.where(np.isnan(w), 2, 1))
    weight = np.where(first == 1, w, 0.0)
    order = np.lexsort((np.arange(n), -weight, first))
    keep = np.zeros(n, bool)
    keep[order[:min(n, budget)]] = True
    slots = np.arange(n)
    return slots[(slots < budget) & ~keep], slots[(slots >= budget) & keep]


class Evict:
    def __init__(self, cache, acc, pos, seen, budget, recent, in_place):
        self.c, self.acc, self.pos, self.seen, self.budget, self.recent, self.in_place = cache, acc, pos, seen, budget, recent, in_place
        self.kv = cache.upload()
        self.seenb, self.accb, self.posb = (ca.Buffer.from_array(x) for x in (seen, acc, pos))
        self.acc2 = self.accb if in_place else ca.Buffer.from_array(np.full_like(acc, -3))
        self.pos2 = self.posb if in_place else ca.Buffer.from_array(np.full_like(pos, 77))
        self.lens2 = ca.Buffer.from_array(np.full_like(cache.lens, 5))
        self.work = ca.Buffer.from_array(np.full(ca.kv_evict_paged_plan(self.kv, budget), 0xFF, np.uint8))

    def __call__(self):
        ca.kv_evict_paged_bf16(self.kv, self.c.lb, self.seenb, self.accb, self.posb, self.lens2, self.acc2, self.pos2,
                               self.budget, self.recent, self.work)

    def check(self):
        c = self.c
        k, v = c.download()
        acc, pos, lens = self.acc2.read(np.float32, self.acc.shape), self.pos2.read(np.uint32, self.pos.shape), self.lens2.read(np.uint32)
        want_k, want_v = c.k.copy(), c.v.copy()
        want_acc, want_pos = (self.acc.copy(), self.pos.copy()) if self.in_place else (np.full_like(self.acc, -3), np.full_like(self.pos, 77))
        for r in range(len(c.lens)):
            n = min(int(c.lens[r]), c.slots)
            assert lens[r] == min(n, self.budget)
            for h in range(c.kv_heads):
                to, src = plain_evict(self.acc[r, h], self.pos[r, h], n, int(self.seen[r]), self.budget, self.recent)
                assert len(to) == len(src)
                stay = np.arange(min(n, self.budget))
                want_acc[r, h, stay], want_pos[r, h, stay] = self.acc[r, h, stay], self.pos[r, h, stay]
                want_acc[r, h, to], want_pos[r, h, to] = self.acc[r, h, src], self.pos[r, h, src]
                for want, pool in ((want_k, c.k), (want_v, c.v)):
                    want[c.table[r, to // c.page], h, to % c.page] = pool[c.table[r, src // c.page], h, src % c.page]
        assert np.array_equal(pos, want_pos)
        assert np.array_equal(acc, want_acc, equal_nan=True)
        assert np.array_equal(k, want_k) and np.array_equal(v, want_v)


def _weights(rng, kind, shape, slots):
    if kind == "spread":
        return np.exp(1.5 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    if kind == "few values":
        return rng.integers(0, 4, shape).astype(np.float32)
    acc = rng.standard_normal(shape).astype(np.float32)  # anything at all
    for value in (np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-40, -1e-40):
        acc[rng.random(shape) < 0.08] = value
    return acc


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["spread", "equal", "few values", "anything"])
@pytest.mark.parametrize("kvh,dim,page,pages,budget,recent,lens", [
    (2, 128, 16, 5, 32, 8, [80, 33, 32, 31, 1, 0, 64]),
    (3, 64, 16, 4, 1, 0, [64, 2, 1]),
    (1, 128, 16, 4, 48, 48, [64, 50]),             # the last positions alone
    (2, 64, 32, 3, 40, 90, [96, 95, 200]),         # more of them than the budget; past the table
    (4, 128, 64, 10, 511, 100, [640, 512, 513]),   # one slot, and many
    (1, 64, 16, 200, 1000, 64, [3200, 1500]),
    (2, 128, 16, 3, 48, 4, [48, 20]),              # a budget of the whole table
    (2, 64, 16, 100, 1200, 7, [1201, 1600, 1202]), # one slot, two and many of a longer row
    (2, 128, 16, 20, 128, 16, [320, 250, 140]),    # as many moves as the choosing workgroup makes
    (1, 64, 32, 50, 1472, 9, [1600, 1500]),
])
def test_evict(kvh, dim, page, pages, budget, recent, lens, kind, in_place):
    say(f"evict budget {budget} recent {recent} {kind} in place {in_place}")
    rng = np.random.default_rng(budget * 7 + recent)
    cache = Cache(rng, lens, kvh, dim, page, pages)
    shape = (len(lens), kvh, cache.slots)
    seen = np.full(len(lens), 5 * cache.slots, np.uint32)
    pos = np.stack([np.stack([rng.permutation(5 * cache.slots)[:cache.slots] for _ in range(kvh)]) for _ in lens]).astype(np.uint32)
    case = Evict(cache, _weights(rng, kind, shape, cache.slots), pos, seen, budget, recent, in_place)
    case()
    case.check()


@pytest.mark.parametrize("budget", [50000, 70000])
def test_evict_long_row(budget):
    """More slots than a workgroup holds, heads that differ; one slot too many."""
    say(f"evict long row {budget}")
    rng = np.random.default_rng(21)
    cache = Cache(rng, [70001], 2, 64, 1024, 69)
    pos = np.stack([rng.permutation(cache.slots) for _ in range(2)])[None].astype(np.uint32)
    case = Evict(cache, _weights(rng, "spread", (1, 2, cache.slots), cache.slots), pos, np.array([cache.slots], np.uint32), budget, 3000, False)
    case()
    case.check()


def test_evict_skips_pages_that_are_not_there():
    """K and V of a slot without a page neither move nor are overwritten; the
    weights and positions do."""
    say("evict unknown pages")
    rng = np.random.default_rng(22)
    cache = Cache(rng, [64], 1, 64, 16, 4)
    good = cache.table.copy()
    acc, pos = np.arange(64, 0, -1, dtype=np.float32)[None, None], np.arange(64, dtype=np.uint32)[None, None]
    acc[0, 0, [3, 20, 5]] = 0          # given up: 3 and 5 in a good page, 20 in a bad one
    acc[0, 0, 32:] = 0
    acc[0, 0, [33, 50, 51]] = 100      # kept: 33 and 51 in good pages, 50 too
    case = Evict(cache, acc, pos, np.array([64], np.uint32), 32, 0, False)
    bad = good.copy()
    bad[0, 1] = cache.num_pages        # slots 16 .. 31
    cache.tb.write(bad)
    case()
    k, _ = cache.download()
    assert np.array_equal(case.pos2.read(np.uint32, (64,))[[3, 5, 20]], [33, 50, 51])
    want = cache.k.copy()
    for to, src in ((3, 33), (5, 50)):
        want[good[0, to // 16], 0, to % 16] = cache.k[good[0, src // 16], 0, src % 16]
    assert np.array_equal(k, want)


def test_evict_captured_and_replayed():
    """A replay sees the lengths, weights and positions of its own time."""
    say("evict graph")
    rng = np.random.default_rng(23)
    cache = Cache(rng, [200, 90], 2, 64, 16, 13)
    shape = (2, 2, cache.slots)
    pos = np.broadcast_to(np.arange(cache.slots, dtype=np.uint32), shape).copy()
    seen = np.array([200, 90], np.uint32)
    case = Evict(cache, _weights(rng, "spread", shape, cache.slots), pos, seen, 64, 10, False)
    replay = captured(case)
    other = Evict(Cache(rng, [48], 1, 128, 16, 3), rng.random((1, 1, 48)).astype(np.float32),
                  np.arange(48, dtype=np.uint32)[None, None], np.array([48], np.uint32), 16, 2, True)
    for trip in range(3):
        acc = _weights(rng, "few values" if trip == 1 else "spread", shape, cache.slots)
        cache.kb.write(cache.k), cache.vb.write(cache.v), case.accb.write(acc)
        case.acc2.write(np.full_like(acc, -3)), case.pos2.write(np.full_like(pos, 77))
        replay()
        other()
        case.acc = acc
        case.check()


# ---------------------------------------------------------------- reorder

class Reorder:
    def __init__(self, rng, rows, kvh, dim, page, pages, lens, parents, pools):
        self.c = Cache(rng, lens, kvh, dim, page, pages, spare=rows)
        self.kv = self.c.upload()
        self.parents = np.asarray(parents, np.uint32)
        self.pools = [bf16(rng.standard_normal(self.c.k.shape)) for _ in range(pools)]
        self.dev = [ca.Buffer.from_array(p) for p in self.pools]
        self.pb, self.sb = ca.Buffer.from_array(self.parents), ca.Buffer.from_array(self.c.spare)
        self.t2, self.l2, self.s2 = ca.Buffer(self.c.table.nbytes), ca.Buffer(4 * rows), ca.Buffer(4 * rows)

    def __call__(self):
        ca.beam_reorder_paged_bf16(self.kv, self.dev, self.c.lb, self.pb, self.sb, self.t2, self.l2, self.s2)

    def check(self, given_up=()):
        c = self.c
        table, spare, lens = c.table.copy(), c.spare.copy(), c.lens.copy()
        want = [p.copy() for p in self.pools]
        for r, p in enumerate(self.parents):
            if r in given_up:
                table[r], lens[r] = 0xFFFFFFFF, 0
                continue
            if p == r:
                continue
            last, used = divmod(int(c.lens[p]), c.page)
            table[r, :last] = c.table[p, :last]
            if used:
                table[r, last], spare[r] = c.spare[r], c.table[r, last]
                for w, pool in zip(want, self.pools):
                    w[c.spare[r], :, :used] = pool[c.table[p, last], :, :used]
        assert np.array_equal(self.t2.read(np.uint32, table.shape), table)
        assert np.array_equal(self.l2.read(np.uint32), lens)
        assert np.array_equal(self.s2.read(np.uint32), spare)
        for w, dev in zip(want, self.dev):
            assert np.array_equal(dev.read(np.uint16, w.shape), w)


@pytest.mark.parametrize("kvh,dim,page,pages,n,pools", [
    (2, 128, 16, 4, 33, 2), (1, 64, 16, 4, 32, 2), (3, 64, 32, 3, 96, 4), (2, 128, 64, 2, 1, 1), (4, 64, 16, 3, 0, 2),
    (1, 128, 1024, 1, 1000, 3), (1, 64, 16, 2, 17, 131), (2, 64, 16, 2, 20, 0),
])
def test_reorder(kvh, dim, page, pages, n, pools):
    say(f"reorder page {page} len {n} pools {pools}")
    rng = np.random.default_rng(n + pools)
    parents = [0, 0, 3, 2, 6, 6, 6, 4, 8]  # itself, shared, exchanged, chains
    case = Reorder(rng, 9, kvh, dim, page, pages, [n] * 9, parents, pools)
    case()
    case.check()


def test_reorder_gives_up_rows_without_a_parent():
    say("reorder without a parent")
    rng = np.random.default_rng(31)
    case = Reorder(rng, 6, 1, 64, 16, 3, [20, 20, 21, 60, 60, 20], [1, 6, 0, 4, 3, 0xFFFFFFFF], 2)
    case()
    case.check(given_up=(1, 2, 3, 4, 5))  # no such row twice, another length, past the table


def test_reorder_captured_and_replayed():
    say("reorder graph")
    rng = np.random.default_rng(32)
    case = Reorder(rng, 4, 2, 64, 16, 4, [37] * 4, [1, 1, 0, 2], 4)
    replay = captured(case)
    for parents in ([1, 1, 0, 2], [3, 0, 0, 3], [0, 1, 2, 3]):
        case.parents = np.asarray(parents, np.uint32)
        case.pb.write(case.parents)
        for dev, pool in zip(case.dev, case.pools):
            dev.write(pool)
        replay()
        case.check()


# ---------------------------------------------------------------- append, rows that share pages

def test_append_of_rows_shorter_than_the_call():
    """A row of fewer slots, or fewer positions, than the call has tokens a row takes
    none of them, those that would have a slot included; its q is turned by the first
    position.  (The tokens of prompts of different lengths are rows of one token.)"""
    say("append to short rows")
    rng = np.random.default_rng(5)
    heads, kvh, dim, tq = 4, 2, 128, 5
    cache = Cache(rng, [3, 9, 4, 5], kvh, dim, 16, 2)
    seen = np.array([3, 4, 60, 7], np.uint32)  # too few slots; positions; slots again; good
    tab = _table(80, dim)
    qkv = rng.standard_normal((4, tq, heads + 2 * kvh, dim)).astype(np.float32)
    acc = rng.random((4, kvh, 32)).astype(np.float32)
    kv = cache.upload()
    accb, posb, q = ca.Buffer.from_array(acc), ca.Buffer.from_array(np.full(acc.shape, 9, np.uint32)), ca.Buffer(4 * tq * heads * dim * 2)
    ca.rope_qkv_paged_bf16(kv, ca.Buffer.from_array(qkv), ca.Buffer.from_array(tab), len(tab), cache.lb,
                           ca.Buffer.from_array(seen), q, tq, heads, accb, posb)
    got = f64(q.read(np.uint16, (4, tq, heads, dim)))
    for r, pos in enumerate(([0] * 5, [0] * 5, [0] * 5, [2, 3, 4, 5, 6])):
        y, tol = _rotated(qkv[r, :, :heads].astype(np.float64), tab[pos][:, None])
        assert np.all(np.abs(got[r] - y) <= tol), r
    k, v = cache.download()
    slots = np.arange(5)
    at = (cache.table[3, slots // 16], slice(None), slots % 16)
    assert np.array_equal(v[at], bf16(qkv[3, :, heads + kvh:]))
    for new, old in ((k, cache.k), (v, cache.v)):
        new[at] = old[at]
        assert np.array_equal(new, old)
    acc[3, :, slots] = 0
    assert np.array_equal(accb.read(np.float32, acc.shape), acc)
    where = np.full(acc.shape, 9, np.uint32)
    where[3, :, slots] = slots[:, None] + 2
    assert np.array_equal(posb.read(np.uint32, acc.shape), where)


def test_append_of_prompts_of_different_lengths():
    """Their tokens as rows of one token, whose tables are their sequence's: rows
    that write different slots of one page, the same as a call a prompt."""
    say("append of ragged prompts")
    rng = np.random.default_rng(6)
    heads, kvh, dim, prompts = 6, 2, 64, [1, 37, 16, 50, 33]
    whole = Cache(rng, [0] * len(prompts), kvh, dim, 16, 4)
    tab = ca.Buffer.from_array(_table(64, dim))
    qkv = rng.standard_normal((sum(prompts), heads + 2 * kvh, dim)).astype(np.float32)
    kv = whole.upload()
    begins = np.cumsum([0] + prompts)
    want_q = []
    for r, n in enumerate(prompts):
        table, q = ca.Buffer.from_array(whole.table[r]), ca.Buffer(n * heads * dim * 2)
        one = ca.PagedKV(kv.k, kv.v, table.ptr, kv.num_pages, 16, 1, 4, kvh, dim)
        ca.rope_qkv_paged_bf16(one, ca.Buffer.from_array(qkv[begins[r]:begins[r + 1]]), tab, 64,
                               ca.Buffer.from_array(np.array([n], np.uint32)), None, q, n, heads)
        want_q.append(q.read(np.uint16, (n, heads, dim)))
    want = whole.download()
    kv = whole.upload()  # the pages as they were
    rows = np.repeat(np.arange(len(prompts)), prompts)
    table = ca.Buffer.from_array(whole.table[rows])
    lens = np.concatenate([np.arange(1, n + 1) for n in prompts]).astype(np.uint32)
    q = ca.Buffer(sum(prompts) * heads * dim * 2)
    each = ca.PagedKV(kv.k, kv.v, table.ptr, kv.num_pages, 16, sum(prompts), 4, kvh, dim)
    ca.rope_qkv_paged_bf16(each, ca.Buffer.from_array(qkv), tab, 64, ca.Buffer.from_array(lens), None, q, 1, heads)
    assert np.array_equal(q.read(np.uint16, (sum(prompts), heads, dim)), np.concatenate(want_q))
    for got, pool in zip(whole.download(), want):
        assert np.array_equal(got, pool)


# ---------------------------------------------------------------- eviction, ties in long rows, windows

@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["equal", "few values", "anything"])
@pytest.mark.parametrize("budget,recent", [(50000, 3000), (9000, 100), (65000, 0), (30000, 30000), (70000, 500)])
def test_evict_equal_weights_in_long_rows(budget, recent, kind, in_place):
    """The lower slot where weights are equal, where the last one that is kept lies in
    any of a row's tiles of 8192."""
    say(f"evict long row, {kind}, budget {budget} recent {recent} in place {in_place}")
    rng = np.random.default_rng(budget + recent)
    cache = Cache(rng, [70001, 69000], 1, 64, 1024, 69)
    pos = np.stack([rng.permutation(2 * cache.slots)[:cache.slots] for _ in range(2)])[:, None].astype(np.uint32)
    case = Evict(cache, _weights(rng, kind, (2, 1, cache.slots), cache.slots), pos, np.full(2, 2 * cache.slots, np.uint32),
                 budget, recent, in_place)
    case()
    case.check()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page,pages,budget,recent,lens", [
    (16, 8, 40, 300, [128, 100, 41, 40, 7]),       # in LDS; one slot too many; none
    (16, 8, 1, 2000, [128, 2]),                    # the newest alone
    (16, 100, 700, 1 << 31, [1600, 1500, 701]),    # every position there was
    (16, 90, 400, 4000, [1440, 1200, 1100]),
    (1024, 20, 5000, 50000, [20001, 15000, 5001]), # tiles of 8192
])
def test_evict_keeps_the_newest_of_many_recent_positions(page, pages, budget, recent, lens, in_place):
    """More slots of the last positions than the budget: the newest are kept, whatever
    slots they are in."""
    say(f"evict window, budget {budget} recent {recent} in place {in_place}")
    rng = np.random.default_rng(budget)
    cache = Cache(rng, lens, 2, 64, page, pages)
    shape = (len(lens), 2, cache.slots)
    seen = 3 * cache.slots
    pos = np.broadcast_to(rng.permutation(seen)[:cache.slots].astype(np.uint32), shape).copy()
    acc = _weights(rng, "anything", shape, cache.slots)
    for r, n in enumerate(lens):  # one row after the other: its window is its own
        one = Cache(rng, [n], 2, 64, page, pages)
        case = Evict(one, acc[r:r + 1], pos[r:r + 1], np.array([seen], np.uint32), budget, recent, in_place)
        case()
        late = np.sort(pos[r, 0, :n][pos[r, 0, :n].astype(np.int64) >= seen - recent])[::-1]
        assert len(late) > budget or r > 0  # fewer in a shorter row: all are kept, then by weight
        if len(late) > budget:
            case.recent = seen - int(late[budget - 1])  # the same said with no more of them than the budget
        case.check()


# ---------------------------------------------------------------- reorder, pages that are not there

def test_reorder_of_pages_that_are_not_there():
    """A parent whose partly filled page does not exist: absent for its children too,
    and their own pages' old rows are not in its place.  A spare page that does not
    exist takes no rows."""
    say("reorder unknown pages")
    rng = np.random.default_rng(33)
    parents = [0, 0, 1, 0, 4]
    case = Reorder(rng, 5, 2, 64, 16, 4, [37] * 5, parents, 3)
    table, spare = case.c.table.copy(), case.c.spare.copy()
    table[1, 2], table[4, 2] = case.c.num_pages, 0xFFFFFFFF  # the parent of 2; its own parent
    table[0, 1] = 0xFFFFFFFF                                 # a filled page: of 0, 1 and 3
    spare[3] = case.c.num_pages + 5
    case.c.tb.write(table)
    case.sb.write(spare)
    case()
    got, num = case.t2.read(np.uint32, table.shape), case.c.num_pages
    want, want_spare, pools = table.copy(), spare.copy(), [p.copy() for p in case.pools]
    want[1, :2], want[1, 2], want_spare[1] = table[0, :2], spare[1], table[1, 2]
    want[2, :2] = table[1, :2]
    want[3, :2], want[3, 2], want_spare[3] = table[0, :2], spare[3], table[3, 2]
    for pool in pools:
        pool[spare[1], :, :5] = pool[table[0, 2], :, :5]
    assert got[2, 2] >= num
    got[2, 2] = want[2, 2]
    assert np.array_equal(got, want)
    assert np.array_equal(case.s2.read(np.uint32), want_spare)
    assert np.array_equal(case.l2.read(np.uint32), [37] * 5)
    for pool, dev in zip(pools, case.dev):
        assert np.array_equal(dev.read(np.uint16, pool.shape), pool)
