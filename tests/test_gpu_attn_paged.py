"""Attention of one new token over a cache in pages, against the formula in 64
bits: every place that no slot in use has holds NaN, so a read that counts for
something shows."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from paged_util import U, UB, Cache, attention, attention_slack, bf16, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Call:
    """One attention call's buffers; run() gives (o, acc or None)."""

    def __init__(self, cache, q16, heads, scale, out_f32, acc=None):
        self.c, self.heads, self.scale, self.out_f32 = cache, heads, scale, out_f32
        self.kv = cache.upload()
        rows = len(cache.lens)
        self.shape = (rows, heads, cache.dim)
        self.q = ca.Buffer.from_array(q16)
        self.o = ca.Buffer(rows * heads * cache.dim * 4)
        self.acc = None if acc is None else ca.Buffer.from_array(acc)
        self.acc_out = None if acc is None else ca.Buffer.from_array(np.full_like(acc, -7.0))
        self.parts, nbytes = ca.attn_paged_plan(self.kv, heads, acc is not None)
        # no byte of the workspace counts before it is written
        self.work = ca.Buffer.from_array(np.full(max(nbytes, 16), 0xFF, np.uint8))

    def __call__(self):
        ca.attn_paged_bf16(self.kv, self.q, self.c.lb, self.o, self.heads, self.scale, self.work, self.out_f32,
                           self.acc, self.acc_out)

    def bits(self):
        o = self.o.read(np.uint32 if self.out_f32 else np.uint16, self.shape)
        return o, None if self.acc is None else self.acc_out.read(np.float32, (*self.shape[:1], self.c.kv_heads, self.c.slots))

    def run(self):
        self()
        o, acc = self.bits()
        return (o.view(np.float32).astype(np.float64) if self.out_f32 else f64(o)), acc


def check(cache, q16, heads, scale, got, out_f32, acc=None, got_acc=None, present=None):
    """Every row against the formula; present: slots that have a page, per row."""
    group = heads // cache.kv_heads
    for r in range(len(cache.lens)):
        n = min(int(cache.lens[r]), cache.slots)
        there = np.arange(n) if present is None else np.flatnonzero(present[r][:n])
        k, v = f64(cache.get(cache.k, r, n))[:, there], f64(cache.get(cache.v, r, n))[:, there]
        for h in range(cache.kv_heads):
            mine = slice(h * group, (h + 1) * group)
            if n == 0:
                assert np.array_equal(got[r, mine], np.zeros((group, cache.dim)))
            else:
                o, p, pv, es = attention(f64(q16[r, mine]), k[h], v[h], scale)
                slack = attention_slack(es, n)
                # a bf16 output: p in two terms (2^-16) and one rounding
                tol = slack * pv + U * np.abs(o) if out_f32 else (slack + 2.0 ** -16) * pv + UB * (np.abs(o) + slack * pv)
                assert np.all(np.abs(got[r, mine] - o) <= tol + 1e-37), (r, h, np.abs(got[r, mine] - o).max())
            if acc is not None:
                want = acc[r, h].astype(np.float64).copy()
                bound = np.zeros(cache.slots)
                if n:
                    want[there] += p.sum(0)
                    bound[there] = p.sum(0) * (slack + (group + 2) * U)
                bound[:n] += U * np.abs(want[:n])
                assert np.all(np.abs(got_acc[r, h, :n] - want[:n]) <= bound[:n] + 1e-37), (r, h)
                assert np.all(got_acc[r, h, n:] == -7.0)  # behind the row's end: as they were


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 127, 128, 129, 200, 255, 256]
CASES = [
    # heads, kv heads, dim, page, max pages, lens
    (4, 4, 128, 16, 16, EDGES),
    (8, 2, 64, 16, 16, EDGES),
    (7, 1, 128, 32, 9, [288, 287, 1, 33, 0, 400]),       # a length past the table: the table's
    (16, 1, 128, 64, 5, [320, 257, 19]),
    (34, 2, 64, 32, 11, [352, 351, 3, 161]),             # 17 query heads a kv head
    (40, 1, 128, 128, 3, [384, 300]),
    (2, 2, 128, 1024, 2, [2048, 1500, 1]),
    (12, 4, 128, 16, 321, [5136, 5001]),                 # runs
    (32, 8, 128, 32, 650, [20800]),
    (3, 3, 64, 16, 700, [11200, 1, 40, 10000]),          # short rows of a long table
    (1, 1, 128, 16, 1, [16]),
    (5, 5, 128, 16, 3, [33] * 130),                      # more pairs than workgroups a round
    (2, 1, 64, 16, 200, [(37 * i) % 211 for i in range(149)] + [3200]),  # many rows on one line, some without slots
    (34, 2, 64, 32, 100, [3200, 1777, 0]),               # cut rows of 17 query heads a kv head
    (4, 2, 128, 32, 60, [1920] * 3 + [64, 32, 31, 96]),  # parts that end with units
]
SHORT_ROWS = [  # of long tables: whole units, more than there are workgroups, or fewer; none
    (8, 8, 64, 16, 256, [(13 * i) % 91 for i in range(70)]),
    (34, 2, 64, 32, 64, [900, 1, 0, 513]),               # two tiles of heads
    (8, 2, 128, 64, 1024, [400, 33]),
    (4, 4, 128, 16, 512, [0, 0, 0]),
]
CASES += SHORT_ROWS


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("out_f32", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_formula(case, out_f32, weights):
    heads, kvh, dim, page, pages, lens = CASES[case]
    say(f"attn_paged case {case} heads {heads}/{kvh} dim {dim} page {page} slots {page * pages} f32 {out_f32} weights {weights}")
    rng = np.random.default_rng(100 + case)
    cache = Cache(rng, lens, kvh, dim, page, pages, lazy=CASES[case] in SHORT_ROWS)
    q = bf16(rng.standard_normal((len(lens), heads, dim)))
    acc = rng.random((len(lens), kvh, cache.slots)).astype(np.float32) if weights else None
    scale = dim ** -0.5
    got, got_acc = Call(cache, q, heads, scale, out_f32, acc).run()
    check(cache, q, heads, scale, got, out_f32, acc, got_acc)


@pytest.mark.parametrize("spread", [0.0, 3.0, 40.0])
def test_running_maximum(spread):
    """Scores of any spread, rising along the row so that the maximum moves in
    every tile, and falling: the same sums."""
    say(f"attn_paged spread {spread}")
    rng = np.random.default_rng(7)
    cache = Cache(rng, [1000, 1000], 2, 128, 16, 63)
    q = bf16(np.abs(rng.standard_normal((2, 4, 128))) + 0.5)
    ramp = np.linspace(-1, 1, 1000)[None, :, None] * spread / 8
    for r, sign in enumerate((1, -1)):
        cache.put(cache.k, r, np.arange(1000), bf16(rng.standard_normal((2, 1000, 128)) * 0.1 + sign * ramp))
    got, _ = Call(cache, q, 4, 128 ** -0.5, True).run()
    check(cache, q, 4, 128 ** -0.5, got, True)


def test_pages_that_the_pool_does_not_have():
    """Their slots are absent: the others' softmax; a row whose every page is
    unknown has nothing to divide by."""
    say("attn_paged unknown pages")
    rng = np.random.default_rng(8)
    cache = Cache(rng, [200, 130, 64], 2, 128, 16, 13)
    acc = rng.random((3, 2, cache.slots)).astype(np.float32)
    q = bf16(rng.standard_normal((3, 8, 128)))
    whole = cache.table.copy()
    present = np.ones((3, cache.slots), bool)
    call = Call(cache, q, 8, 0.1, True, acc)
    for r, entries in ((0, [0, 5, 12]), (1, [8])):
        for e in entries:
            cache.table[r, e] = cache.num_pages if e else 0xFFFFFFFF
            present[r, 16 * e:16 * e + 16] = False
    cache.table[2, :] = 0x80000000
    call.c.tb.write(cache.table)
    got, got_acc = call.run()
    assert np.all(np.isnan(got[2]))
    cache.table, cache.lens = whole, cache.lens[:2]
    check(cache, q, 8, 0.1, got, True, acc, got_acc, present)


def test_infinities_and_nan_in_use():
    """As the formula has them: NaN in a key or +inf in a score gives NaN, -inf
    in a score weighs nothing, a row of -inf alone NaN, an infinite value its sum."""
    say("attn_paged specials")
    rng = np.random.default_rng(9)
    cache = Cache(rng, [70] * 6, 1, 128, 16, 5)
    q = bf16(np.abs(rng.standard_normal((6, 2, 128))) + 0.1)
    everywhere = np.arange(70)

    def fill(row, slots, bits, pool):
        cache.put(pool, row, np.asarray(slots), np.full((1, len(slots), 128), bits, np.uint16))

    fill(0, [3], 0x7FC0, cache.k)          # NaN
    fill(1, [40], 0x7F80, cache.k)         # +inf
    fill(2, [0, 17, 69], 0xFF80, cache.k)  # -inf
    fill(3, everywhere, 0xFF80, cache.k)
    fill(4, [66], 0x7F80, cache.v)
    got, _ = Call(cache, q, 2, 0.05, True).run()
    for r in (0, 1, 3):
        assert np.all(np.isnan(got[r])), r
    assert np.all(np.isposinf(got[4]))
    # row 2: as without those slots; row 5: untouched
    for r, kept in ((2, np.setdiff1d(everywhere, [0, 17, 69])), (5, everywhere)):
        k, v = f64(cache.get(cache.k, r, 70))[0][kept], f64(cache.get(cache.v, r, 70))[0][kept]
        o, _, pv, es = attention(f64(q[r]), k, v, 0.05)
        assert np.all(np.abs(got[r] - o) <= attention_slack(es, 70) * pv + U * np.abs(o))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("out_f32", [True, False])
def test_values_of_the_largest_size_that_weigh_nothing(dim, out_f32):
    """Slots far below the maximum (e^-300), their values near the type's largest:
    nothing of them is in the sum."""
    say(f"attn_paged large values dim {dim} f32 {out_f32}")
    rng = np.random.default_rng(13)
    cache = Cache(rng, [80], 1, dim, 16, 5)
    q = np.zeros((1, 3, dim), np.float32)
    q[..., 0] = 1
    k = 0.5 * rng.standard_normal((1, 80, dim))
    light = np.arange(3, 80, 7)
    k[:, light, 0] = -300
    v = rng.standard_normal((1, 80, dim))
    v[:, light] = 3e38
    cache.put(cache.k, 0, np.arange(80), bf16(k))
    cache.put(cache.v, 0, np.arange(80), bf16(v))
    got, _ = Call(cache, bf16(q), 3, 1.0, out_f32).run()
    check(cache, bf16(q), 3, 1.0, got, out_f32)


def test_offsets_past_32_bits():
    """Pages behind 2^32 elements of a pool."""
    say("attn_paged large pool")
    rng = np.random.default_rng(10)
    page, kvh, dim = 1024, 8, 128
    one = kvh * page * dim * 2
    far = [4100, 2049, 4108]
    pool = ca.Buffer(4109 * one)
    k = bf16(rng.standard_normal((3, kvh, page, dim)))
    for i, p in enumerate(far):
        pool.write(k[i], p * one)
    table = ca.Buffer.from_array(np.array([far], np.uint32))
    lens = ca.Buffer.from_array(np.array([2500], np.uint32))
    q16 = bf16(rng.standard_normal((1, kvh, dim)))
    q, o = ca.Buffer.from_array(q16), ca.Buffer(kvh * dim * 4)
    kv = ca.PagedKV(pool.ptr, pool.ptr, table.ptr, 4109, page, 1, 3, kvh, dim)
    work = ca.Buffer(max(16, ca.attn_paged_plan(kv, kvh)[1]))
    ca.attn_paged_bf16(kv, q, lens, o, kvh, 0.09, work, True)
    got = o.read(np.float32, (kvh, dim))
    flat = f64(k).transpose(1, 0, 2, 3).reshape(kvh, 3 * page, dim)[:, :2500]
    for h in range(kvh):
        want, _, pv, es = attention(f64(q16[0, h:h + 1]), flat[h], flat[h], 0.09)
        assert np.all(np.abs(got[h] - want[0]) <= (attention_slack(es, 2500) * pv + U * np.abs(want))[0])
    pool.close()
    ca.lib().catena_pool_trim()


def test_in_place_weights_and_repeated_calls():
    """acc_out = acc_in, call after call: the weights add up; the same call gives
    the same bits."""
    say("attn_paged in place")
    rng = np.random.default_rng(11)
    cache = Cache(rng, [777, 300], 2, 64, 16, 49)
    q = bf16(rng.standard_normal((2, 6, 64)))
    call = Call(cache, q, 6, 0.125, False, np.zeros((2, 2, cache.slots), np.float32))
    call()
    o1, once = call.bits()
    call()
    o2, again = call.bits()
    assert np.array_equal(o1, o2) and np.array_equal(once, again)
    call.acc_out = call.acc
    for _ in range(3):
        call()
    _, three = call.bits()
    for r, n in enumerate((777, 300)):
        # three adds, each off by half a step at most
        assert np.all(np.abs(three[r, :, :n] - 3.0 * once[r, :, :n]) <= 3 * U * 3 * once[r, :, :n])
        assert np.all(three[r, :, n:] == 0)
        # three heads a kv head, three times; off by 3 u a slot, and u for each of n adds here
        assert np.all(np.abs(three[r, :, :n].astype(np.float64).sum(-1) - 9) <= 9 * (attention_slack(1e-4, n) + 4 * U))


def test_captured_and_replayed():
    """A graph's replays, between eager calls of another shape on workspaces of
    their own, give the eager bits."""
    say("attn_paged graph")
    rng = np.random.default_rng(12)
    one = Call(Cache(rng, [900, 17, 0], 2, 128, 16, 60), bf16(rng.standard_normal((3, 8, 128))), 8, 0.1, True,
               np.zeros((3, 2, 960), np.float32))
    two = Call(Cache(rng, [4000], 1, 128, 32, 125), bf16(rng.standard_normal((1, 4, 128))), 4, 0.1, False)
    assert one.parts > 1 and two.parts > 1
    want = []
    for call in (one, two):
        call()
        want.append(call.bits())
    replay = [captured(one), captured(two)]
    for _ in range(4):
        for call, again in zip((one, two), replay):
            call.o.write(np.full(call.o.nbytes, 0xEE, np.uint8))
            again()
        two()
        for call, (o, acc) in zip((one, two), want):
            got_o, got_acc = call.bits()
            assert np.array_equal(got_o, o)
            assert acc is None or np.array_equal(got_acc, acc)


@pytest.mark.parametrize("weights", [False, True])
def test_replayed_with_other_lengths(weights):
    """One graph, lengths that change between replays: cut rows, whole units of
    short rows, no slots at all."""
    say(f"attn_paged graph, lengths change, weights {weights}")
    rng = np.random.default_rng(14)
    cache = Cache(rng, [4096, 4096, 4096], 2, 64, 32, 128)
    q = bf16(rng.standard_normal((3, 8, 64)))
    acc = rng.random((3, 2, cache.slots)).astype(np.float32) if weights else None
    call = Call(cache, q, 8, 0.125, True, acc)
    assert call.parts > 0
    replay = captured(call)
    for lens in ([4096, 1, 2000], [90, 0, 33], [0, 0, 0], [31, 4096, 700], [4096, 1, 2000]):
        cache.lens = np.array(lens, np.uint32)
        cache.lb.write(cache.lens)
        if weights:
            call.acc_out.write(np.full_like(acc, -7.0))
        call.o.write(np.full(call.o.nbytes, 0xEE, np.uint8))
        replay()
        o, got_acc = call.bits()
        check(cache, q, 8, 0.125, o.view(np.float32).astype(np.float64), True, acc, got_acc)


LARGE = [
    # heads, kv heads, dim, page, max pages, lens
    (3, 1, 128, 16, 5, [2, 80]),                    # whole units
    (34, 2, 64, 16, 5, [80, 33, 16]),               # two tiles of heads
    (2, 1, 64, 16, 1024, [16384]),                  # cut rows, by the parts a unit has: many,
    (4, 4, 128, 32, 128, [4096] * 8 + [70, 5]),     # some,
    (8, 8, 64, 32, 128, [4096] * 8 + [31] * 60),    # few
]


@pytest.mark.parametrize("out_f32", [True, False])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_values_near_the_largest_that_weigh(case, out_f32):
    """Values near the type's largest, all of one sign in a column and all of
    weight: their mean is as large as they are, no sum on the way larger.  Scores
    rise along the row, so that many weights are formed below their maximum."""
    heads, kvh, dim, page, pages, lens = LARGE[case]
    say(f"attn_paged values of weight near the largest, case {case} f32 {out_f32}")
    rng = np.random.default_rng(200 + case)
    cache = Cache(rng, lens, kvh, dim, page, pages, lazy=True)
    q = np.zeros((len(lens), heads, dim), np.float32)
    q[..., 0] = 1
    sign = np.where(rng.random((kvh, 1, dim)) < 0.5, -1.0, 1.0)
    for r, n in enumerate(lens):
        k = 0.1 * rng.standard_normal((kvh, n, dim))
        k[:, :, 0] += np.linspace(0, 6, n)
        cache.put(cache.k, r, np.arange(n), bf16(k))
        cache.put(cache.v, r, np.arange(n), bf16(sign * (3.2e38 + 1e37 * rng.random((kvh, n, dim)))))
    call = Call(cache, bf16(q), heads, 1.0, out_f32, rng.random((len(lens), kvh, cache.slots)).astype(np.float32))
    assert (call.parts > 0) == (case >= 2 or case == 1)  # weights of two tiles of heads are joined
    got, acc = call.run()
    assert np.all(np.isfinite(got))
    check(cache, bf16(q), heads, 1.0, got, out_f32, call.acc.read(np.float32, acc.shape), acc)


CUT = [  # full rows are longer than what is taken whole
    # heads, kv heads, dim, page, max pages, lens
    # more than 64 rows on one line, several without slots before longer ones
    (8, 4, 128, 32, 50, [0, 0, 1600] + [(29 * i) % 180 for i in range(60)] + [0, 1600, 0, 0, 1590] + [0, 7] * 10 + [1600, 0, 64]),
    # the join without pieces, by few long rows
    (8, 8, 64, 64, 64, [4096] + [100, 0, 1, 33, 900] * 7 + [4096, 3000, 0, 2]),
    # long parts: 16384 tiles, of few units (128 wide and 64), of more than there are CUs
    (8, 8, 128, 1024, 64, [65536]),
    (16, 8, 64, 1024, 65, [66560]),
    (8, 8, 128, 64, 64, [1650] * 39 + [4096]),
    # more rows than the join's grid: with a piece a head, without pieces
    (128, 8, 128, 32, 65, [2080, 0, 31] + [97 * i for i in range(1, 16)]),
    (16, 8, 64, 1024, 9, [9216] + [(7 * i) % 40 for i in range(298)] + [9000]),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("case", range(len(CUT)))
def test_cut_rows(case, weights):
    heads, kvh, dim, page, pages, lens = CUT[case]
    say(f"attn_paged cut rows, case {case} heads {heads}/{kvh} dim {dim} rows {len(lens)} weights {weights}")
    rng = np.random.default_rng(300 + case)
    cache = Cache(rng, lens, kvh, dim, page, pages, lazy=True)
    q = bf16(rng.standard_normal((len(lens), heads, dim)))
    acc = rng.random((len(lens), kvh, cache.slots)).astype(np.float32) if weights else None
    out_f32 = case % 2 == 0
    call = Call(cache, q, heads, dim ** -0.5, out_f32, acc)
    # a plan of parts for a table's full rows, and full rows: cut, whatever the others' lengths
    units, tiles = len(lens) * kvh, kvh * sum(-(-n // 32) for n in lens)
    parts = ca.attn_paged_plan(cache.kv, heads)[0]
    assert parts > 0 and call.parts > 0 and max(lens) == cache.slots
    assert [len(lens) > 64 and parts <= 2 * units, parts <= 2 * units and len(lens) <= 64, parts == 256 and tiles >= 16384,
            parts == 256 and tiles >= 16384, parts > 256 and tiles >= 16384, 2 * units < parts <= 16 * units,
            parts <= 2 * units and len(lens) > 256][case]
    got, got_acc = call.run()
    check(cache, q, heads, dim ** -0.5, got, out_f32, acc, got_acc)


@pytest.mark.parametrize("size", [1e-33, 1e-25, 1e18, 1e35])
@pytest.mark.parametrize("lens", [[80], [16384]])
def test_values_of_any_size(lens, size):
    """The mean of small values and of large ones, over few slots and many."""
    say(f"attn_paged values near {size}, {lens[0]} slots")
    rng = np.random.default_rng(15)
    cache = Cache(rng, lens, 1, 64, 16, lens[0] // 16)
    cache.put(cache.v, 0, np.arange(lens[0]), bf16(size * rng.standard_normal((1, lens[0], 64))))
    q = bf16(rng.standard_normal((1, 3, 64)))
    got, _ = Call(cache, q, 3, 0.125, True).run()
    check(cache, q, 3, 0.125, got, True)


@pytest.mark.parametrize("out_f32", [True, False])
@pytest.mark.parametrize("lens", [[80], [4096]])
def test_infinite_values_of_little_weight(lens, out_f32):
    """Slots of weight 2^-65, of whose bits nothing is left for a second term, with
    infinite values: infinity, as in the formula, not the NaN of a term that is 0."""
    say(f"attn_paged infinite value of little weight, {lens[0]} slots, f32 {out_f32}")
    rng = np.random.default_rng(16)
    cache = Cache(rng, lens, 1, 128, 16, lens[0] // 16)
    q = np.zeros((1, 2, 128), np.float32)
    q[..., 0] = 1
    k = 0.5 * rng.standard_normal((1, lens[0], 128))
    k[..., 0] = 0
    k[:, [5, lens[0] - 2], 0] = -65
    cache.put(cache.k, 0, np.arange(lens[0]), bf16(k))
    cache.put(cache.v, 0, np.array([5, lens[0] - 2]), np.full((1, 2, 128), 0x7F80, np.uint16))
    got, _ = Call(cache, bf16(q), 2, np.log(2.0), out_f32).run()  # scores in base 2 as they are
    assert np.all(np.isposinf(got))
