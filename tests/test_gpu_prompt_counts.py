"""Causal attention of packed sequences where every slot counts: a slot's key says which of a
few kinds it is, its value is 1 in one column, and a query row asks for one kind. So o's
columns are counts of slots over the number of the kind, and a slot that is left out, taken
twice or taken for another changes a column of some query row by one of at most 100, of a
tile by tens of percent.

The base-2 scores are 24 for the kind and 0 for the others (scale ln 2, keys and queries
whole numbers), so every p is a power of two, which bf16 holds: the result is off by f32's
sums (at most n + 200 roundings) and its own rounding alone."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import U, UB, bf16, f64
from test_gpu_attn_prompt import Prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Counted(Prompt):
    def __init__(self, rng, n, ctx, heads, kvh, dim, page, **kw):
        super().__init__(rng, n, ctx, heads, kvh, dim, page, **kw)
        self.scale = float(np.float32(np.log(2.0)))
        group = heads // kvh
        self.kinds, self.columns, self.of = [], [], []
        q = np.zeros((self.tokens, heads, dim), np.float32)
        for r in range(self.rows):
            slots, new = int(self.lens[r]), self.n[r]
            kinds = max(1, min(16, group * new))
            kind, column = rng.integers(0, kinds, slots), rng.integers(0, dim, slots)
            self.kinds.append(kinds), self.of.append(kind), self.columns.append(column)
            k, v = np.zeros((kvh, slots, dim), np.float32), np.zeros((kvh, slots, dim), np.float32)
            for h in range(kvh):
                k[h, np.arange(slots), (kind + h) % kinds] = 1  # (another kind for every kv head)
                v[h, np.arange(slots), (column + 5 * h) % dim] = 1
            if page:
                for pool, x in ((self.cache.k, k), (self.cache.v, v)):
                    self.cache.put(pool, r, np.arange(slots), bf16(x))
            else:
                a, b = int(self.starts[r]), int(self.starts[r + 1])
                for pool, x in ((self.k, k), (self.v, v)):
                    pool[a:b, : kvh * dim] = bf16(x.transpose(1, 0, 2)).reshape(b - a, kvh * dim)
            for t in range(new):
                for h in range(heads):
                    q[int(self.starts[r]) + t, h, (t * group + h % group) % kinds] = 24
        self.q = bf16(q)

    def check(self, got, tokens=None):
        group = self.heads // self.kvh
        for r in range(self.rows):
            for t in (range(self.n[r]) if tokens is None else sorted({x % self.n[r] for x in tokens} if self.n[r] else ())):
                n, at = self.ctx[r] + t + 1, int(self.starts[r]) + t
                kinds = self.kinds[r]
                table = np.zeros((kinds, self.dim))
                np.add.at(table, (self.of[r][:n], self.columns[r][:n]), 1)
                for h in range(self.heads):
                    asked = (t * group + h % group - h // group) % kinds
                    mine = table[asked]
                    other = table.sum(0) - mine
                    want = (mine + other * 2.0 ** -24) / (mine.sum() + other.sum() * 2.0 ** -24)
                    want = np.roll(want, 5 * (h // group))
                    bound = want * (UB + (n + 200) * U * (1 + UB))
                    assert np.all(np.abs(f64(got[at, h]) - want) <= bound), (r, t, h)


LAST = list(range(-17, 0))


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", [
    ([1500], [0], 8, 2, 128, 16), ([300, 1], [5000, 20000], 8, 1, 128, 64), ([700, 900, 11], [0, 100, 3000], 4, 4, 64, 32),
    ([5], [33000], 4, 1, 64, 16), ([20], [20000], 1, 1, 128, 128), ([600, 64, 33, 1], [3000, 2000, 9000, 4096], 2, 1, 64, 16),
    ([513, 1, 1, 255], [600, 3000, 1, 1000], 6, 3, 128, 128), ([1, 2, 3], [9000, 1, 70], 40, 1, 128, 16), ([100], [9000], 16, 2, 64, 1024),
])
def test_long(n, ctx, heads, kvh, dim, page):
    """Wide and narrow units, cut and joined."""
    say(f"counts {n} {ctx} {heads} {kvh} {dim} {page}")
    p = Counted(np.random.default_rng(sum(ctx) + dim), n, ctx, heads, kvh, dim, page)
    p.check(p.run(), [0, 1, 31, 32, 63, 64, 65, 127, 128, 255, 256, 299, 640, 1023, 1400] + LAST)


@pytest.mark.parametrize("n,heads,kvh,dim", [([2500], 4, 1, 64), ([1100, 70, 3], 6, 3, 128), ([64, 65, 130, 16], 2, 2, 64), ([33, 127], 4, 4, 128)])
def test_packed(n, heads, kvh, dim):
    say(f"counts, packed {n} {heads} {kvh} {dim}")
    p = Counted(np.random.default_rng(sum(n)), n, [0] * len(n), heads, kvh, dim, 0, pad=2, gap=1)
    p.check(p.run(), [0, 1, 31, 32, 63, 64, 65, 127, 128, 255, 256, 1023, 2047] + LAST)


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", [([1] * 5 + [40, 100], [0, 15, 16, 700, 64, 300, 500], 16, 4, 128, 16),
                                                      ([70, 3], [200, 900], 8, 2, 64, 32)])
def test_without_a_list(n, ctx, heads, kvh, dim, page):
    say(f"counts, no list {n} {ctx} {heads} {kvh} {dim} {page}")
    p = Counted(np.random.default_rng(sum(ctx)), n, ctx, heads, kvh, dim, page)
    p.check(p.run())


@pytest.mark.parametrize("heads,kvh,dim", [(16, 8, 64), (32, 8, 128)])
def test_many_narrow_units(heads, kvh, dim):
    """So many that two waves share one, some long enough to be cut, wide ones beside them."""
    say(f"counts, many narrow units {heads} {kvh} {dim}")
    rng = np.random.default_rng(heads)
    rows = 2100 // kvh + 1
    n, ctx = rng.integers(1, 4, rows), rng.integers(0, 70, rows)
    n[:6], ctx[:6] = [200, 1, 4, 2, 8, 1], [100, 2300, 1500, 1100, 4000, 9000]
    p = Counted(rng, n, ctx, heads, kvh, dim, 16, gap=1, pad=2)
    p.check(p.run(), [0, 1, 2, 3, 63, 64, 100] + LAST)
