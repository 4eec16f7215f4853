"""Causal attention of packed sequences against 64 bits. p is rounded to bf16, p_i (1 +
d_i) with |d_i| <= 2^-8, in the sum over v and in that of p alike, so that the result

    sum p_i (1 + d_i) v_i / sum p_i (1 + d_i) = o + sum p_i d_i (v_i - o) / (1 + sum p_i d_i)

is off by 2^-8 (sum p |v| + |o|) at most (1 + 2^-7 for the divisor); it is
rounded to bf16 itself."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from paged_util import NAN16, UB, Cache, attention, bf16, f64
from requests_util import prompt_slack

pytestmark = pytest.mark.gpu
MARK = 0x4242  # what places of no row keep


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _bound(es, n, pv, want):
    off = prompt_slack(es, n) * pv + UB * (1 + 2 * UB) * (pv + np.abs(want))
    return off + UB * (np.abs(want) + off)


class Prompt:
    """Rows of n new tokens behind `ctx` slots, in pages or (page 0) packed."""

    def __init__(self, rng, n, ctx, heads, kvh, dim, page, pad=0, gap=0, scale=1.0, stride=0):
        self.n, self.ctx, self.heads, self.kvh, self.dim, self.page = list(n), list(ctx), heads, kvh, dim, page
        self.rows, self.lens = len(self.n), np.array(self.n, np.int64) + np.array(self.ctx, np.int64)
        self.starts = np.concatenate([[gap], gap + np.cumsum(self.n)]).astype(np.uint32)
        self.tokens = int(self.starts[-1]) + pad
        self.q = bf16(rng.standard_normal((self.tokens, heads, dim)) * scale)
        self.scale = dim ** -0.5
        if page:
            self.cache = Cache(rng, self.lens, kvh, dim, page, max(1, -(-int(self.lens.max(initial=0)) // page)), lazy=True, scale=scale)
        else:
            self.stride = stride or kvh * dim
            self.k, self.v = (np.full((max(self.tokens, 1), self.stride), NAN16, np.uint16) for _ in range(2))
            for x in (self.k, self.v):
                x[gap:self.starts[-1], : kvh * dim] = bf16(rng.standard_normal((int(self.starts[-1]) - gap, kvh * dim)) * scale)

    def run(self, again=1):
        up = ca.Buffer.from_array
        self.o = up(np.full((self.tokens + 1, self.heads, self.dim), MARK, np.uint16))
        qb, sb, lb = up(self.q), up(self.starts), up(self.lens.astype(np.uint32))
        if self.page:
            kv = self.cache.upload()
            work = ca.Buffer(max(ca.attn_prompt_plan(kv, self.tokens, self.heads), 16))
            self.call = lambda: ca.attn_prompt_bf16(kv, qb, sb, lb, self.o, self.tokens, self.heads, self.scale, work)
        else:
            kb, vb = up(self.k), up(self.v)
            work = ca.Buffer(max(ca.attn_packed_plan(self.rows, self.tokens, self.heads, self.kvh, self.dim), 16))
            self.keep = (kb, vb)
            self.call = lambda: ca.attn_packed_bf16(qb, kb, vb, sb, self.o, self.rows, self.tokens, self.heads, self.kvh, self.dim, self.scale, work,
                                                    0 if self.stride == self.kvh * self.dim else self.stride)
        self.more = (qb, sb, lb, work)
        for _ in range(again):
            self.call()
        return self.read()

    def read(self):
        got = self.o.read(np.uint16, (self.tokens + 1, self.heads, self.dim))
        assert np.all(got[self.starts[-1]:] == MARK) and np.all(got[: self.starts[0]] == MARK)
        return got

    def kv_of(self, r):
        n = int(self.lens[r])
        if self.page:
            return f64(self.cache.get(self.cache.k, r, n)), f64(self.cache.get(self.cache.v, r, n))
        a, b = int(self.starts[r]), int(self.starts[r + 1])
        return tuple(f64(x[a:b, : self.kvh * self.dim]).reshape(b - a, self.kvh, self.dim).transpose(1, 0, 2) for x in (self.k, self.v))

    def check(self, got, tokens=None):
        group = self.heads // self.kvh
        for r in range(self.rows):
            if not self.n[r]:
                continue
            k, v = self.kv_of(r)
            for t in (range(self.n[r]) if tokens is None else sorted({x % self.n[r] for x in tokens})):
                n = self.ctx[r] + t + 1
                at = int(self.starts[r]) + t
                for h in range(self.kvh):
                    mine = slice(h * group, (h + 1) * group)
                    want, _, pv, es = attention(f64(self.q[at, mine]), k[h, :n], v[h, :n], self.scale)
                    assert np.all(np.abs(f64(got[at, mine]) - want) <= _bound(es, n, pv, want)), (r, t, h)


SHAPES = [
    # new tokens, slots before, heads, kv heads, dim, page
    ([1], [0], 1, 1, 64, 16), ([1], [0], 8, 1, 128, 16), ([2, 1], [0, 63], 4, 4, 128, 16), ([64], [0], 2, 2, 128, 64),
    ([65, 63, 128, 1], [0, 1, 0, 127], 4, 2, 128, 32), ([33, 0, 7], [5, 0, 300], 8, 2, 64, 16), ([130, 17], [0, 40], 7, 1, 128, 128),
    ([1, 1, 1, 1, 1], [0, 15, 16, 700, 64], 32, 8, 128, 16), ([200], [1000], 16, 1, 64, 1024), ([0, 0, 3], [0, 4, 0], 5, 5, 128, 16),
    ([31, 97], [0, 0], 48, 2, 128, 16), ([257], [0], 3, 3, 64, 32), ([40], [88], 40, 1, 128, 64),
]


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", SHAPES)
@pytest.mark.parametrize("packed", [False, True])
def test_prompt(n, ctx, heads, kvh, dim, page, packed):
    say(f"prompt {n} {ctx} {heads} {kvh} {dim} {page} {packed}")
    rng = np.random.default_rng(sum(n) + heads)
    p = Prompt(rng, n, [0] * len(n) if packed else ctx, heads, kvh, dim, 0 if packed else page, pad=3, gap=len(n) % 3)
    p.check(p.run())


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", [([1500], [0], 8, 2, 128, 16), ([300, 1], [5000, 20000], 8, 1, 128, 64),
                                                      ([700, 900, 11], [0, 100, 3000], 4, 4, 64, 32), ([5], [33000], 4, 1, 64, 16)])
def test_long(n, ctx, heads, kvh, dim, page):
    say(f"long {n} {ctx} {heads} {kvh} {dim} {page}")
    rng = np.random.default_rng(sum(ctx))
    p = Prompt(rng, n, ctx, heads, kvh, dim, page)
    got = p.run()
    p.check(got, [0, 1, 63, 64, 127, 128, 255, 299, 640, 1023, 1400, -1])
    assert np.array_equal(p.run(again=3), got)


def test_many_rows():
    say("many rows")
    rng = np.random.default_rng(4)
    p = Prompt(rng, rng.integers(0, 6, 150), rng.integers(0, 90, 150), 4, 2, 64, 16)
    p.check(p.run())
    p = Prompt(rng, rng.integers(0, 9, 70), [0] * 70, 4, 2, 64, 0)
    p.check(p.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_scales(scale):
    say(f"scale {scale}")
    rng = np.random.default_rng(6)
    p = Prompt(rng, [70, 3], [20, 0], 4, 2, 128, 16)
    p.scale = scale
    p.check(p.run())


def test_stride():
    say("keys and values inside wider rows")
    rng = np.random.default_rng(7)
    for dim in (64, 128):
        p = Prompt(rng, [70, 130], [0, 0], 6, 2, dim, 0, stride=10 * dim)
        p.check(p.run())


def test_odd_starts():
    """lens below the new tokens (the first see nothing: 0), starts past the list or
    falling (cut; no tokens), lens past the table (the table's)."""
    say("odd starts")
    rng = np.random.default_rng(11)
    p = Prompt(rng, [40, 30], [0, 0], 4, 2, 128, 16)
    p.lens = np.array([25, 30])
    got = p.run()
    assert np.all(f64(got[:15]) == 0)
    k, v = (f64(p.cache.get(x, 0, 25)) for x in (p.cache.k, p.cache.v))
    want, _, pv, es = attention(f64(p.q[39, :2]), k[0], v[0], p.scale)
    slack = prompt_slack(es, 25) + UB
    assert np.all(np.abs(f64(got[39, :2]) - want) <= slack * pv + UB * (np.abs(want) + slack * pv))
    first = Prompt(rng, [40, 30], [0, 0], 4, 2, 128, 16)
    exp = first.run()
    sb = first.more[1]
    first.o.write(np.full_like(exp, MARK))
    sb.write(np.array([0, 40, 0xFFFFFFF0], np.uint32))  # the second row is cut to the list: 30 tokens
    first.call()
    assert np.array_equal(first.o.read(np.uint16, exp.shape), exp)
    first.o.write(np.full_like(exp, MARK))
    sb.write(np.array([40, 0, 0], np.uint32))
    first.call()
    assert np.all(first.o.read(np.uint16, exp.shape) == MARK)
    past = Prompt(rng, [16], [0], 4, 2, 128, 16)
    exp = past.run()
    past.more[2].write(np.array([1000], np.uint32))
    past.call()
    assert np.array_equal(past.o.read(np.uint16, exp.shape), exp)


def test_absent_pages():
    say("absent pages")
    rng = np.random.default_rng(12)
    p = Prompt(rng, [20, 9], [140, 23], 4, 2, 128, 16)
    p.cache.table[0, 3] = 0xFFFFFFFF
    p.cache.table[0, 8] = p.cache.num_pages
    p.cache.table[1] = 0xFFFFFFF0
    got = p.run()
    assert np.all(np.isnan(f64(got[20:29])))
    p.cache.table[0, [3, 8]] = p.cache.table[0, 0]  # (any page that is there, for reading)
    keep = np.ones(160, bool)
    keep[48:64] = keep[128:144] = False
    k, v = (f64(p.cache.get(x, 0, 160)) for x in (p.cache.k, p.cache.v))
    for t in (0, 3, 4, 19):
        seen = keep & (np.arange(160) < 141 + t)
        want, _, pv, es = attention(f64(p.q[t, 2:]), k[1, seen], v[1, seen], p.scale)
        assert np.all(np.abs(f64(got[t, 2:]) - want) <= _bound(es, 160, pv, want))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_seen_does_not_count(dim, packed):
    """Infinities and NaN in keys and values of later tokens change no bit of earlier
    ones; from their own token on they show as they do in the formula."""
    say(f"not seen {dim} {packed}")
    rng = np.random.default_rng(13)
    n, at = 150, 70
    p = Prompt(rng, [n], [0], 4, 2, dim, 0 if packed else 32)
    base = p.run()

    def put(which, slot, head, col, bits):
        if packed:
            (p.k if which == "k" else p.v)[slot, head * dim + col] = bits
        else:
            pool = p.cache.k if which == "k" else p.cache.v
            pool[p.cache.table[0, slot // 32], head, slot % 32, col] = bits

    put("v", at, 0, 5, 0x7F80)       # inf
    put("v", at + 3, 0, 6, 0xFF80)   # -inf
    put("v", at + 5, 0, 7, NAN16)
    put("v", at + 8, 0, 5, 0xFF80)   # -inf beside the inf
    put("k", at + 20, 1, 3, NAN16)
    got = p.run()[:n]  # (without the place behind the list)
    base = base[:n]
    assert np.array_equal(got[:at], base[:at])
    x = f64(got)
    assert np.all(np.isposinf(x[at:at + 8, :2, 5])) and np.all(np.isnan(x[at + 8:, :2, 5]))
    assert np.all(np.isneginf(x[at + 3:, :2, 6])) and np.all(np.isfinite(x[at:at + 3, :2, 6]))
    assert np.all(np.isnan(x[at + 5:, :2, 7])) and np.all(np.isfinite(x[: at + 5, :2, 7]))
    # no other column, and the other kv head until its key is NaN
    other = [c for c in range(dim) if c not in (5, 6, 7)]
    assert np.array_equal(got[:, :2][..., other], base[:, :2][..., other])
    assert np.array_equal(got[: at + 20, 2:], base[: at + 20, 2:]) and np.all(np.isnan(x[at + 20:, 2:]))


def test_large_values():
    say("large values")
    rng = np.random.default_rng(14)
    p = Prompt(rng, [90], [200], 4, 2, 128, 16)
    p.cache.v[...] = np.where(p.cache.v == NAN16, NAN16, 0x7F00)  # 2^127, whose sums f32 does not hold
    got = f64(p.run()[:90])
    assert np.all(np.abs(got - 2.0 ** 127) <= (2 * UB + prompt_slack(2.0 ** -10, 290)) * 2.0 ** 127)
    p = Prompt(rng, [90], [200], 4, 2, 128, 16, scale=12.0)  # scores of some thousands: one slot has all the weight
    p.check(p.run())


def test_captured():
    """One graph over lists whose lengths change, with eager calls between its replays."""
    say("captured")
    rng = np.random.default_rng(15)
    p = Prompt(rng, [60, 200, 9], [100, 0, 700], 8, 2, 128, 16)
    exp = p.run()
    replay = captured(p.call)
    for n in ([60, 200, 9], [1, 30, 9], [60, 0, 0], [2, 260, 7]):
        p.n, p.starts = n, np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
        p.lens = np.minimum(np.array([160, 200, 709]), p.cache.slots)
        p.ctx = [int(x) - y for x, y in zip(p.lens, n)]
        if min(p.ctx) < 0:
            p.lens, p.ctx = np.maximum(p.lens, n), [max(x, 0) for x in p.ctx]
            p.lens[1], p.n[1], p.ctx[1] = 200, 200, 0
            p.starts = np.concatenate([[0], np.cumsum(p.n)]).astype(np.uint32)
        p.more[1].write(p.starts)
        p.more[2].write(p.lens.astype(np.uint32))
        results = []
        for go in (replay, p.call, replay):
            p.o.write(np.full((p.tokens + 1, p.heads, p.dim), MARK, np.uint16))
            go()
            ca.synchronize()
            results.append(p.read())
        assert np.array_equal(results[0], results[1]) and np.array_equal(results[1], results[2])
        p.check(results[0], [0, 5, 59, 64, 130, -1])
    assert exp.shape == results[0].shape


# Lists of units: where some row may have more than 1024 slots

def test_list_of_many_rows():
    say("list of many rows")
    rng = np.random.default_rng(16)
    n, ctx = rng.integers(0, 3, 1100), rng.integers(0, 40, 1100)
    n[[7, 1030, 1099]], ctx[[7, 1030, 1099]] = [300, 40, 9], [2500, 1500, 1100]
    p = Prompt(rng, n, ctx, 8, 2, 64, 16, pad=5, gap=2)
    got = p.run()
    p.check(got, [0, 1, 8, 39, 130, 299])
    assert np.array_equal(p.run(again=2), got)
    n = rng.integers(0, 4, 1300)
    n[[0, 1299]] = [700, 65]
    p = Prompt(rng, n, [0] * 1300, 8, 2, 128, 0)
    p.check(p.run(), [0, 1, 2, 64, 300, 699])


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", [
    ([33, 34, 64, 65], [2000, 1000, 3, 1300], 2, 2, 64, 16), ([9, 16, 17, 1], [1500, 4000, 0, 2222], 8, 2, 128, 32),
    ([1, 2, 3], [9000, 1, 70], 40, 1, 128, 16), ([513, 1, 1, 255], [600, 3000, 1, 1000], 6, 3, 128, 128),
])
def test_list(n, ctx, heads, kvh, dim, page):
    """Units of up to 32, 64 and more query rows, cut or not."""
    say(f"list {n} {ctx} {heads} {kvh} {dim} {page}")
    p = Prompt(np.random.default_rng(sum(ctx)), n, ctx, heads, kvh, dim, page)
    got = p.run()
    p.check(got, [0, 1, 8, 15, 31, 32, 33, 63, 64, 254, 300, -1])
    assert np.array_equal(p.run(again=2), got)


@pytest.mark.parametrize("dim", [64, 128])
def test_list_what_is_not_seen(dim):
    """As above: for a wide unit, one of 60 query rows and one of two."""
    say(f"list, not seen {dim}")
    rng = np.random.default_rng(17)
    p = Prompt(rng, [300, 30, 1, 1], [1000, 1500, 3000, 2000], 4, 2, dim, 16)
    base = p.run()
    first = p.starts[:-1].astype(int)

    def put(which, row, slot, head, col, bits):
        pool = p.cache.k if which == "k" else p.cache.v
        pool[p.cache.table[row, slot // 16], head, slot % 16, col] = bits

    put("v", 0, 1150, 0, 5, 0x7F80)  # inf, from token 150 on
    put("v", 0, 1180, 0, 6, 0xFF80)  # -inf, from token 180 on
    put("k", 0, 1200, 1, 3, NAN16)   # from token 200 on
    put("v", 1, 1510, 1, 9, NAN16)   # from token 10 on
    put("v", 1, 1520, 1, 5, 0x7F80)  # from token 20 on
    put("v", 2, 700, 0, 5, 0x7F80)   # seen
    got = p.run()[:332]
    x, base = f64(got), base[:332]
    assert np.array_equal(got[:150], base[:150]) and np.array_equal(got[first[3]], base[first[3]])
    assert np.all(np.isposinf(x[150:300, :2, 5])) and np.all(np.isneginf(x[180:300, :2, 6])) and np.all(np.isfinite(x[150:180, :2, 6]))
    assert np.array_equal(got[150:200, 2:], base[150:200, 2:]) and np.all(np.isnan(x[200:300, 2:]))
    assert np.array_equal(got[300:310], base[300:310]) and np.array_equal(got[300:330, :2], base[300:330, :2])
    assert np.all(np.isnan(x[310:330, 2:, 9])) and np.all(np.isposinf(x[320:330, 2:, 5])) and np.all(np.isfinite(x[310:320, 2:, 5]))
    assert np.all(np.isposinf(x[first[2], :2, 5])) and np.array_equal(got[first[2], 2:], base[first[2], 2:])
    other = [c for c in range(dim) if c not in (5, 6, 9)]
    assert np.array_equal(got[:200][..., other], base[:200][..., other]) and np.array_equal(got[300:][..., other], base[300:][..., other])


def test_list_absent_pages():
    say("list, absent pages")
    rng = np.random.default_rng(18)
    p = Prompt(rng, [100, 10], [1400, 2000], 4, 2, 128, 16)
    gone = np.zeros((2, 2016), bool)
    for row, pages in ((0, [3, 50, 92]), (1, [0, 1, 2, 3, 4, 5, 6, 7, 60, 125])):
        p.cache.table[row, pages] = 0xFFFFFFFF
        for g in pages:
            gone[row, 16 * g:16 * g + 16] = True
    got = p.run()
    for r in range(2):
        n = int(p.lens[r])
        p.cache.table[r] = np.where(p.cache.table[r] == 0xFFFFFFFF, p.cache.table[0, 0], p.cache.table[r])  # (any, for reading)
        k, v = (f64(p.cache.get(x, r, n)) for x in (p.cache.k, p.cache.v))
        for t in (0, 5, 9) + ((63, 70, 99) if r == 0 else ()):
            at = int(p.starts[r]) + t
            seen = ~gone[r, :n] & (np.arange(n) <= p.ctx[r] + t)
            for h in range(2):
                mine = slice(2 * h, 2 * h + 2)
                want, _, pv, es = attention(f64(p.q[at, mine]), k[h, seen], v[h, seen], p.scale)
                assert np.all(np.abs(f64(got[at, mine]) - want) <= _bound(es, n, pv, want)), (r, t, h)


def test_list_captured():
    """Two graphs that share a workspace, over lists whose lengths change, with eager calls between."""
    say("list captured")
    rng = np.random.default_rng(19)
    p = Prompt(rng, [60, 300, 9, 1], [1200, 900, 700, 3000], 8, 2, 128, 16)
    p.run()
    graphs = [captured(p.call), captured(p.call)]
    for n in ([60, 300, 9, 1], [1, 1, 1, 1], [0, 200, 9, 1], [300, 0, 0, 70]):
        p.n, p.starts = n, np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
        p.ctx = [int(x) - y for x, y in zip(p.lens, n)]
        p.more[1].write(p.starts)
        results = []
        for go in (graphs[0], p.call, graphs[1], graphs[0]):
            p.o.write(np.full((p.tokens + 1, p.heads, p.dim), MARK, np.uint16))
            go()
            ca.synchronize()
            results.append(p.read())
        assert all(np.array_equal(results[0], x) for x in results[1:])
        p.check(results[0], [0, 8, 59, 64, 130, -1])


def test_list_overlapping_rows():
    """Which is not allowed: what comes out is anything, and places of no row stay."""
    say("list, rows that overlap")
    rng = np.random.default_rng(20)
    p = Prompt(rng, [2] + [0] * 39, [6400] + [3000] * 39, 2, 2, 64, 16, pad=1)
    p.starts = np.array([0, 2] * 20 + [0], np.uint32)
    p.lens[:] = 3000
    p.lens[0] = 6402
    up = ca.Buffer.from_array
    o = up(np.full((4, 2, 64), MARK, np.uint16))
    kv = p.cache.upload()
    keep = [up(p.q), up(p.starts), up(p.lens.astype(np.uint32)), ca.Buffer(ca.attn_prompt_plan(kv, 3, 2))]
    ca.attn_prompt_bf16(kv, keep[0], keep[1], keep[2], o, 3, 2, p.scale, keep[3])
    assert np.all(o.read(np.uint16, (4, 2, 64))[2:] == MARK)


def test_most_rows_and_heads():
    say("most rows and heads")
    rng = np.random.default_rng(21)
    p = Prompt(rng, [1] * 5000, rng.integers(0, 5, 5000), 2, 1, 64, 16)
    p.check(p.run())
    p = Prompt(rng, [1] * 8, [0] * 8, 131072, 1, 64, 0)  # 512 units a row
    got = p.run()
    for t in range(8):  # one slot: its value
        assert np.array_equal(got[t], np.broadcast_to(p.v[t], got[t].shape))


@pytest.mark.parametrize("heads,kvh,dim", [(16, 8, 64), (6, 3, 128), (80, 5, 64)])
def test_many_narrow_units(heads, kvh, dim):
    """So many that a workgroup takes several kv heads' of them: also where these do not come out even, units of one
    and two blocks of 32 query rows, parts, rows that see nothing, wide units beside them."""
    say(f"many narrow units {heads} {kvh} {dim}")
    rng = np.random.default_rng(22)
    rows = 2100 // kvh + 1
    n, ctx = rng.integers(0, 3, rows) + 1, rng.integers(0, 70, rows)
    n[:4], ctx[:4] = [200, 1, 4, 2], [100, 2300, 1500, 1100]
    p = Prompt(rng, n, ctx, heads, kvh, dim, 16, gap=1, pad=2)
    p.lens[5] = 1  # of n tokens: the last sees the slot
    n5, p.ctx[5] = p.n[5], 1 - p.n[5]
    got = p.run()
    at = int(p.starts[5])
    assert np.all(f64(got[at:at + n5 - 1]) == 0)
    p.n[5] = 0
    p.check(got, [0, 1, 2, 3, 100, 199])
    p.n[5] = n5
    assert np.array_equal(p.run(again=2), got)
