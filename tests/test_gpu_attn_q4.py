"""Attention of one new token a row over a cache held in 4 bits, against 64 bits on the
values that the codes stand for. p v_scale is taken in two bf16 terms, 2^-16 of it; the
result is rounded to bf16 once."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from paged_util import U, UB, attention, bf16, f64
from requests_util import NAN16, Cache4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _slack(es, n):
    """e^(error of a score) above and below the fraction; 200 u for the exponential, its
    argument (up to 126: 90 u), p's factors and those between partial sums; sums of n terms
    whose longest chain is n / 16 + 64 adds, twice; p's terms."""
    return 2 * es + (200 + 2 * (n / 16 + 64)) * U + 2.0 ** -16


class Rows:
    def __init__(self, rng, lens, heads, kvh, dim, page, max_pages, **kw):
        self.c = Cache4(rng, lens, kvh, dim, page, max_pages, **kw)
        self.heads, self.scale = heads, dim ** -0.5
        self.q = bf16(rng.standard_normal((len(lens), heads, dim)))

    def run(self, again=1):
        kv = self.c.upload()
        self.qb, self.o = ca.Buffer.from_array(self.q), ca.Buffer.from_array(np.full(self.q.shape, 7, np.uint16))
        self.work = ca.Buffer(max(ca.attn_paged_q4_plan(kv, self.heads)[1], 16))
        self.call = lambda: ca.attn_paged_q4(kv, self.qb, self.c.lb, self.o, self.heads, self.scale, self.work)
        for _ in range(again):
            self.call()
        return self.o.read(np.uint16, self.q.shape)

    def check(self, got, keep=None):
        group = self.heads // self.c.kv_heads
        for r, n in enumerate(np.minimum(self.c.lens, self.c.slots).astype(int)):
            if n == 0:
                assert np.all(f64(got[r]) == 0)
                continue
            k, v = self.c.get(r, n)
            seen = np.ones(n, bool) if keep is None else keep[r][:n]
            for h in range(self.c.kv_heads):
                mine = slice(h * group, (h + 1) * group)
                want, _, pv, es = attention(f64(self.q[r, mine]), k[h, seen], v[h, seen], self.scale)
                slack = _slack(es, n)
                err = np.abs(f64(got[r, mine]) - want)
                assert np.all(err <= slack * pv + UB * (np.abs(want) + slack * pv)), (r, h, err.max())


SHAPES = [
    ([1], 1, 1, 64, 16, 1), ([1, 0, 15, 16, 17], 8, 2, 128, 16, 2), ([31, 32, 33, 64, 127, 128, 129], 4, 4, 64, 32, 5),
    ([500, 3, 640, 511], 16, 16, 128, 16, 40), ([1000, 1, 77], 40, 1, 128, 64, 16), ([2048], 24, 1, 64, 1024, 2),
    ([5000, 4999, 0, 130], 8, 8, 128, 128, 40), ([700] * 9, 35, 5, 64, 16, 44), ([300, 40000], 4, 1, 128, 16, 2500),
    ([9000, 12], 32, 8, 64, 32, 300), ([3000, 600, 513], 12, 1, 128, 32, 100), ([4096, 1537], 34, 2, 64, 64, 100),
    ([7000] + [1, 20, 37] * 170, 8, 8, 64, 128, 55),
]


@pytest.mark.parametrize("lens,heads,kvh,dim,page,pages", SHAPES)
def test_q4(lens, heads, kvh, dim, page, pages):
    say(f"q4 {lens} {heads} {kvh} {dim} {page}")
    rng = np.random.default_rng(sum(lens) + heads)
    x = Rows(rng, lens, heads, kvh, dim, page, pages, lazy=True)
    got = x.run()
    x.check(got)
    assert np.array_equal(x.run(again=3), got)


def test_ragged_batch():
    say("ragged batch")
    rng = np.random.default_rng(2)
    lens = rng.integers(0, 2000, 70)
    lens[[3, 50]] = 0
    x = Rows(rng, lens, 8, 2, 128, 16, 125, lazy=True)
    x.check(x.run())
    short = Rows(rng, rng.integers(0, 40, 70), 8, 2, 64, 16, 125, lazy=True)  # whole units though the table is long
    short.check(short.run())


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(scale):
    say(f"scale {scale}")
    rng = np.random.default_rng(3)
    x = Rows(rng, [130, 1000], 4, 2, 128, 32, 32)
    x.scale = scale
    x.check(x.run())


def test_absent_pages():
    say("absent pages")
    rng = np.random.default_rng(4)
    for pages in (12, 400):
        x = Rows(rng, [190, 150], 4, 2, 128, 16, pages)
        x.c.table[0, [3, 11]] = [0xFFFFFFFF, x.c.num_pages]
        x.c.table[1] = 0xFFFFFFF0
        got = x.run()
        assert np.all(np.isnan(f64(got[1])))
        keep = np.ones(190, bool)
        keep[48:64] = keep[176:] = False
        x.c.table[0, [3, 11]] = x.c.table[0, 0]
        x.c.lens = np.array([190, 0], np.uint32)
        got[1] = 0
        x.check(got, [keep, None])


@pytest.mark.parametrize("dim", [64, 128])
def test_scales_of_blocks(dim):
    """The least block scales (2^-127: nothing), large ones, a slot whose value scale is
    0, slots of very different value scales; a NaN block or scale shows in its own kv head
    alone."""
    say(f"block scales {dim}")
    rng = np.random.default_rng(5)
    x = Rows(rng, [200], 4, 2, dim, 16, 13)
    at = lambda s: (x.c.table[0, s // 16], s % 16)  # noqa: E731
    for s, byte in ((3, 0), (70, 0), (71, 130), (150, 124)):
        p, i = at(s)
        x.c.k_scale[p, :, :, i] = byte
    for s, bits in ((5, 0), (6, bf16(np.float32(1e-30)).item()), (90, bf16(np.float32(300.0)).item()), (91, 0x0001)):
        p, i = at(s)
        x.c.v_scale[p, :, i] = bits
    got = x.run()
    x.check(got)
    p, i = at(120)
    x.c.k_scale[p, 0, dim // 32 - 1, i] = 255
    x.c.v_scale[p, 1, i] = NAN16
    both = f64(x.run())
    assert np.all(np.isnan(both))
    x.c.v_scale[p, 1, i] = bf16(np.float32(0.5)).item()
    one = x.run()
    assert np.all(np.isnan(f64(one[:, :2]))) and np.all(np.isfinite(f64(one[:, 2:])))


def test_large_values():
    say("large values")
    rng = np.random.default_rng(6)
    x = Rows(rng, [300, 5000], 4, 2, 128, 16, 320)
    x.c.v[...] = 0x77
    x.c.v_scale[...] = np.where(x.c.v_scale == NAN16, NAN16, 0x7E2A)  # 6 of it: near the type's largest
    got = f64(x.run())
    want = 6 * f64(np.array([0x7E2A], np.uint16))[0]
    assert np.all(np.abs(got - want) <= (UB + 2.0 ** -15) * want)


def test_captured():
    say("captured")
    rng = np.random.default_rng(7)
    x = Rows(rng, [900, 33, 2000], 8, 2, 128, 16, 125)
    x.run()
    replay = captured(x.call)
    for lens in ([900, 33, 2000], [1, 0, 5], [1999, 640, 16]):
        x.c.lb.write(np.array(lens, np.uint32))
        res = []
        for go in (replay, x.call, replay):
            x.o.write(np.full(x.q.shape, 7, np.uint16))
            go()
            ca.synchronize()
            res.append(x.o.read(np.uint16, x.q.shape))
        assert np.array_equal(res[0], res[1]) and np.array_equal(res[1], res[2])
        if lens[0] == 900:
            x.check(res[0])
