"""Pages and slot maps of a step (kv_admit_paged, kv_release_paged) against a plain loop
over rows: every output is a whole number, so all have to be equal."""
import numpy as np
import pytest

import catena_amd as ca
import requests_util as plain
from gpu_util import captured, say
from paged_util import geometry

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Step:
    """Rows of `lens` slots that hold their pages, `spare` pages on the stack."""

    def __init__(self, rng, lens, page, max_pages, spare, extra_held=0):
        self.lens, self.page, self.max_pages = np.asarray(lens, np.uint32), page, max_pages
        rows = len(self.lens)
        self.held = np.minimum(-(-self.lens.astype(np.int64) // page) + extra_held, max_pages).astype(np.uint32)
        self.num_pages = max(int(self.held.sum()) + spare, 1)
        order = rng.permutation(self.num_pages).astype(np.uint32)
        self.table = np.full((rows, max_pages), 0xFFFFFFFF, np.uint32)
        self.table[np.arange(max_pages) < self.held[:, None]] = order[: int(self.held.sum())]
        self.free = np.concatenate([order[int(self.held.sum()):], np.full(int(self.held.sum()), 77, np.uint32)])[: self.num_pages]
        self.count = min(spare, self.num_pages)
        self.seen = (self.lens + rng.integers(0, 50, rows)).astype(np.uint32)
        self.kv = geometry(k=0, v=0, table=0, num_pages=self.num_pages, page_size=page, rows=rows, max_pages=max_pages, kv_heads=1)

    def admit(self, want, max_tokens, seen=True):
        up = ca.Buffer.from_array
        rows = len(self.lens)
        one = np.array([self.count], np.uint32)
        b = [up(x) for x in (self.table, self.lens, self.held, np.asarray(want, np.uint32), self.free, one)]
        out = [ca.Buffer(4 * rows), ca.Buffer(4 * rows), ca.Buffer(4 * (rows + 1)), ca.Buffer(4), ca.Buffer(max(4 * max_tokens, 4)),
               ca.Buffer(max(8 * max_tokens, 8))]
        s = (up(self.seen), ca.Buffer(4 * rows)) if seen else (None, None)
        ca.kv_admit_paged(self.kv, *b, *out, max_tokens, *s)
        got = (b[0].read(np.uint32, self.table.shape), out[0].read(np.uint32), out[1].read(np.uint32), out[2].read(np.uint32),
               int(out[3].read(np.uint32)[0]), out[4].read(np.uint32)[:max_tokens], out[5].read(np.uint64)[:max_tokens])
        return got + ((s[1].read(np.uint32),) if seen else ()), b[4].read(np.uint32)

    def check(self, want, max_tokens, seen=True):
        got, free = self.admit(want, max_tokens, seen)
        exp = plain.admit(self.table, self.lens, self.held, np.asarray(want, np.uint32), self.free, self.count, self.page, max_tokens,
                          self.seen if seen else None)
        for name, x, y in zip(("table", "lens", "held", "starts", "count", "pos", "slots", "seen"), got, exp):
            assert np.array_equal(np.asarray(x, np.uint64), np.asarray(y).astype(np.uint64)), name
        assert np.array_equal(free, self.free)
        return got


@pytest.mark.parametrize("rows,page,most,tokens", [(1, 16, 1, 1), (1, 1024, 1500, 1500), (3, 16, 40, 64), (64, 16, 1, 64), (65, 32, 3, 100),
                                                   (255, 64, 200, 5000), (256, 16, 33, 4096), (1024, 16, 2, 1024), (1025, 128, 9, 3000),
                                                   (2500, 16, 60, 70000), (5, 16, 30000, 131072)])
@pytest.mark.parametrize("seen", [False, True])
def test_admit(rows, page, most, tokens, seen):
    say(f"admit {rows} x {page}, up to {most} of {tokens}")
    rng = np.random.default_rng(rows * 7 + page)
    max_pages = max(4, -(-(3 * most) // page))
    lens = rng.integers(0, max_pages * page + 1, rows)
    lens[rng.random(rows) < 0.2] = 0
    want = rng.integers(0, most + 1, rows)
    want[0] = most
    lens[0] = rng.integers(0, page)
    need = int(np.maximum(-(-(lens + want) // page) - -(-lens // page), 0).sum())
    s = Step(rng, lens, page, max_pages, need + 3)
    s.check(want, tokens, seen)


@pytest.mark.parametrize("spare", [0, 1, 7, 40])
@pytest.mark.parametrize("rows", [30, 1500])
def test_admit_when_pages_run_out(rows, spare):
    say(f"pages run out: {rows} rows, {spare} pages")
    rng = np.random.default_rng(spare)
    s = Step(rng, rng.integers(1, 60, rows), 16, 8, spare)
    got = s.check(rng.integers(0, 40, rows), 100000)
    assert got[4] >= 0 and np.any(got[1] > s.lens)  # rows that need no page go on
    s.check(np.ones(rows), rows)


@pytest.mark.parametrize("tokens", [0, 1, 50, 51, 3000])
def test_admit_when_the_list_is_full(tokens):
    say(f"a list of {tokens}")
    rng = np.random.default_rng(tokens)
    s = Step(rng, rng.integers(0, 100, 1200), 16, 16, 2000)
    s.check(rng.integers(0, 5, 1200), tokens)


def test_admit_odd_rows():
    """Requests past the table, none at all, sums past 32 bits, rows that hold more or
    fewer pages than their slots need."""
    say("odd rows")
    rng = np.random.default_rng(5)
    lens = np.array([64, 60, 0, 10, 0, 33, 16, 0], np.uint32)
    want = np.array([1, 5, 64, 0, 65, 0xFFFFFFFF, 16, 4], np.uint32)
    s = Step(rng, lens, 16, 4, 20)
    s.check(want, 200)
    Step(rng, lens, 16, 4, 20, extra_held=1).check(want, 200)
    few = Step(rng, lens, 16, 4, 20)
    few.held = np.array([4, 2, 0, 0, 0, 1, 0, 0], np.uint32)
    few.check(want, 200)
    many = Step(rng, np.zeros(9, int), 1024, 1 << 20, 3)
    many.check(np.full(9, 1 << 30), 5000)  # 2^33 tokens asked for
    none = Step(rng, np.zeros(0, int), 16, 4, 3)
    got, _ = none.admit(np.zeros(0), 4, False)
    assert got[3].tolist() == [0] and got[4] == 3 and got[5].tolist() == [0] * 4 and set(got[6].tolist()) == {2 ** 64 - 1}
    # a count past the pool is cut to it; a page that is not there is no place
    bad = Step(rng, np.array([3, 40]), 16, 4, 5)
    bad.count, bad.table[0, 0] = bad.num_pages + 9, 0xFFFFFFFF
    got, _ = bad.admit(np.array([2, 1]), 4, False)
    assert got[6][0] == got[6][1] == 2 ** 64 - 1 and got[4] == bad.num_pages
    slot = int(bad.table[1, 2]) * 16 + 8
    assert got[6][2] == slot


@pytest.mark.parametrize("rows,max_pages", [(1, 4), (7, 3), (300, 40), (1300, 5), (2, 20000)])
def test_release(rows, max_pages):
    say(f"release {rows} x {max_pages}")
    rng = np.random.default_rng(rows)
    s = Step(rng, rng.integers(0, 16 * max_pages + 1, rows), 16, max_pages, 11)
    done = rng.integers(0, 2, rows).astype(np.uint32) * 5
    done[0] = 1
    up = ca.Buffer.from_array
    b = [up(x) for x in (s.table, s.lens, s.held, done, s.free, np.array([s.count], np.uint32))]
    out = [ca.Buffer(4 * rows), ca.Buffer(4 * rows), ca.Buffer(4)]
    ca.kv_release_paged(s.kv, *b, *out)
    back = [int(p) for r in range(rows) if done[r] for p in s.table[r, : s.held[r]]]
    free = s.free.copy()
    free[s.count:s.count + len(back)] = back
    table = s.table.copy()
    for r in np.flatnonzero(done):
        table[r, : s.held[r]] = 0xFFFFFFFF
    assert np.array_equal(b[4].read(np.uint32), free) and np.array_equal(b[0].read(np.uint32, table.shape), table)
    assert int(out[2].read(np.uint32)[0]) == s.count + len(back)
    assert np.array_equal(out[0].read(np.uint32), np.where(done, 0, s.lens)) and np.array_equal(out[1].read(np.uint32), np.where(done, 0, s.held))


def test_admit_and_release_captured():
    """A graph of both over state that goes round: admitted, ended, admitted again, with
    eager work between the replays; no page is lost or given twice."""
    say("captured admission")
    rng = np.random.default_rng(9)
    rows, page, max_pages, tokens = 40, 16, 6, 512
    s = Step(rng, np.zeros(rows, int), page, max_pages, 130)
    up = ca.Buffer.from_array
    table, free = up(s.table), up(s.free)
    lens, held, count = [up(s.lens), ca.Buffer(4 * rows)], [up(s.held), ca.Buffer(4 * rows)], [up(np.array([130], np.uint32)), ca.Buffer(4)]
    want, done, starts, pos, slots = ca.Buffer(4 * rows), ca.Buffer(4 * rows), ca.Buffer(4 * (rows + 1)), ca.Buffer(4 * tokens), ca.Buffer(8 * tokens)

    def step():
        ca.kv_admit_paged(s.kv, table, lens[0], held[0], want, free, count[0], lens[1], held[1], starts, count[1], pos, slots, tokens)
        ca.kv_release_paged(s.kv, table, lens[1], held[1], done, free, count[1], lens[0], held[0], count[0])

    replay = captured(step)
    now = (s.table.copy(), s.lens.copy(), s.held.copy(), s.free.copy(), 130)
    for _ in range(12):
        w, d = rng.integers(0, 30, rows).astype(np.uint32), (rng.random(rows) < 0.3).astype(np.uint32)
        want.write(w)
        done.write(d)
        replay()
        ca.synchronize()
        exp = plain.admit(now[0], now[1], now[2], w, now[3], now[4], page, tokens)
        assert np.array_equal(pos.read(np.uint32), exp[5]) and np.array_equal(slots.read(np.uint64), exp[6])
        t, n, h, c, f = exp[0], exp[1], exp[2], exp[4], now[3].copy()
        for r in np.flatnonzero(d):
            f[c:c + h[r]] = t[r, : h[r]]
            c += int(h[r])
            t[r, : h[r]] = 0xFFFFFFFF
        now = (t, np.where(d, 0, n), np.where(d, 0, h), f, c)
        assert np.array_equal(table.read(np.uint32, t.shape), t) and int(count[0].read(np.uint32)[0]) == c
        assert np.array_equal(free.read(np.uint32)[:c], f[:c])
        assert np.array_equal(lens[0].read(np.uint32), now[1]) and np.array_equal(held[0].read(np.uint32), now[2])
        pages = sorted(f[:c].tolist() + [int(p) for r in range(rows) for p in t[r, : now[2][r]]])
        assert pages == sorted(s.free[:130].tolist())
