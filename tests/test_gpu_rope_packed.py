"""Packed rotation and append, in bf16 and 4 bits, and its table. The rotation's
operations are rounded one by one and the codes are the nearest ones, so outputs are
equal bit by bit to the plain form's."""
import numpy as np
import pytest

import catena_amd as ca
import requests_util as plain
from gpu_util import say
from paged_util import NAN16, U, Cache, bf16, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _f32(bits):
    return f64(bits).astype(np.float32)


class Batch:
    """tokens at random slots of a pool; a few of them nowhere, or past the table of rotations."""

    def __init__(self, rng, tokens, heads, kvh, dim, page, rot, wide, positions=50, data=None):
        self.tokens, self.heads, self.kvh, self.dim, self.page, self.rot = tokens, heads, kvh, dim, page, rot
        self.pages = -(-tokens // page) + 2
        self.slots = rng.permutation(self.pages * page)[:tokens].astype(np.uint64)
        self.pos = rng.integers(0, positions, tokens).astype(np.uint32)
        if tokens > 4:
            self.slots[rng.integers(0, tokens, 2)] = [2 ** 64 - 1, self.pages * page]
            self.pos[rng.integers(0, tokens)] = positions
            self.slots[-1] = (1 << 40) + 3
        self.tab = rng.standard_normal((positions, rot // 2, 2)).astype(np.float32)
        x = rng.standard_normal((tokens, heads + 2 * kvh, dim)) if data is None else data
        self.x = x.astype(np.float32) if wide else bf16(x)
        self.wide = wide
        known = self.pos < positions
        self.at = np.where(known, self.pos, 0)
        self.there = known & (self.slots < self.pages * page)

    def expected(self, interleaved):
        x = self.x if self.wide else _f32(self.x)
        k0, v0 = self.heads, self.heads + self.kvh
        tab = self.tab[self.at]
        return plain.turn(x[:, :k0], tab, self.rot, interleaved), plain.turn(x[:, k0:v0], tab, self.rot, interleaved), bf16(x[:, v0:])

    def run(self, kv, interleaved, copies, slots=True):
        up = ca.Buffer.from_array
        q = ca.Buffer.from_array(np.full((self.tokens + 1, self.heads, self.dim), 7, np.uint16))
        out = [up(np.full((self.tokens, self.kvh, self.dim), 7, np.uint16)) for _ in range(2)] if copies else [None, None]
        self.keep = [up(self.x), up(self.tab), up(self.pos), up(self.slots)]
        call = ca.rope_packed_q4 if isinstance(kv, ca.PagedKV4) else ca.rope_packed_bf16
        call(kv, self.keep[0], self.wide, self.keep[1], len(self.tab), self.rot, interleaved, self.keep[2], self.keep[3] if slots else None,
             q, self.tokens, self.heads, *out)
        got = q.read(np.uint16, (self.tokens + 1, self.heads, self.dim))
        assert np.all(got[-1] == 7)
        return got[:-1], [b.read(np.uint16, (self.tokens, self.kvh, self.dim)) for b in out] if copies else None


CASES = [(1, 1, 1, 64, 16, 64), (1, 32, 8, 128, 16, 128), (5, 4, 2, 128, 16, 32), (33, 7, 7, 64, 32, 16), (70, 8, 1, 128, 64, 64),
         (129, 20, 5, 128, 1024, 128), (200, 2, 2, 64, 128, 48), (40, 64, 32, 128, 16, 112)]


@pytest.mark.parametrize("tokens,heads,kvh,dim,page,rot", CASES)
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_packed_bf16(tokens, heads, kvh, dim, page, rot, wide, interleaved):
    say(f"rope bf16 {tokens} {heads} {kvh} {dim} {page} {rot} {wide} {interleaved}")
    rng = np.random.default_rng(tokens + rot)
    b = Batch(rng, tokens, heads, kvh, dim, page, rot, wide)
    pools = [np.full((b.pages, kvh, page, dim), 9, np.uint16) for _ in range(2)]
    bufs = [ca.Buffer.from_array(p) for p in pools]
    kv = ca.PagedKV(bufs[0].ptr, bufs[1].ptr, 0, b.pages, page, 1, 1, kvh, dim)
    q, copies = b.run(kv, interleaved, tokens % 2 == 1)
    eq, ek, ev = b.expected(interleaved)
    assert np.array_equal(q, eq)
    if copies:
        assert np.array_equal(copies[0], ek) and np.array_equal(copies[1], ev)
    at = b.slots[b.there].astype(np.int64)
    pools[0][at // page, :, at % page], pools[1][at // page, :, at % page] = ek[b.there], ev[b.there]
    for buf, p in zip(bufs, pools):
        assert np.array_equal(buf.read(np.uint16, p.shape), p)


def _same4(cache, exp):
    for name in ("k", "v", "k_scale", "v_scale"):
        assert np.array_equal(getattr(cache, name), getattr(exp, name)), name


class Pools4:
    def __init__(self, pages, kvh, dim, page):
        self.k, self.v = np.full((pages, kvh, page, dim // 2), 9, np.uint8), np.full((pages, kvh, dim // 2, page), 9, np.uint8)
        self.k_scale, self.v_scale = np.full((pages, kvh, dim // 32, page), 9, np.uint8), np.full((pages, kvh, page), 9, np.uint16)
        self.page = page

    def upload(self, kvh, dim):
        self.bufs = [ca.Buffer.from_array(x) for x in (self.k, self.v, self.k_scale, self.v_scale)]
        return ca.PagedKV4(*[b.ptr for b in self.bufs], 0, len(self.k), self.page, 1, 1, kvh, dim)

    def write(self, slots, k16, v16):
        at, place = slots // self.page, slots % self.page
        code, scale, _ = plain.quantise_k(k16)
        self.k[at, :, place], self.k_scale[at, :, :, place] = plain.pack(code), scale
        code, scale, _ = plain.quantise_v(v16)
        self.v[at, :, :, place], self.v_scale[at, :, place] = plain.pack(code), scale

    def check(self):
        for b, x in zip(self.bufs, (self.k, self.v, self.k_scale, self.v_scale)):
            assert np.array_equal(b.read(x.dtype, x.shape), x)


def _check4(b, interleaved, copies):
    pools = Pools4(b.pages, b.kvh, b.dim, b.page)
    kv = pools.upload(b.kvh, b.dim)
    q, out = b.run(kv, interleaved, copies)
    eq, ek, ev = b.expected(interleaved)
    assert np.array_equal(q, eq)
    if copies:
        for got, bits, cut in zip(out, (ek, ev), (plain.quantise_k, plain.quantise_v)):
            value = cut(bits)[2]
            exp = bf16(value)
            exp[np.isnan(value)] = NAN16
            same = (got == exp) | ((got & 0x7FFF) > 0x7F80) & np.isnan(value) | ((got | exp) == 0x8000) & (value == 0)
            assert np.all(same)
    pools.write(b.slots[b.there].astype(np.int64), ek[b.there], ev[b.there])
    pools.check()


@pytest.mark.parametrize("tokens,heads,kvh,dim,page,rot", CASES)
@pytest.mark.parametrize("wide,interleaved", [(True, False), (False, True)])
def test_rope_packed_q4(tokens, heads, kvh, dim, page, rot, wide, interleaved):
    say(f"rope q4 {tokens} {heads} {kvh} {dim} {page} {rot} {wide} {interleaved}")
    rng = np.random.default_rng(tokens + rot + 1)
    _check4(Batch(rng, tokens, heads, kvh, dim, page, rot, wide), interleaved, True)


@pytest.mark.parametrize("dim", [64, 128])
def test_codes_of_odd_values(dim):
    """Zeros, signed zeros, ties, the type's largest and smallest values, infinities and
    NaN, blocks whose largest value is 6, 6.03 and 7.97 of a power of two."""
    say(f"odd values {dim}")
    rng = np.random.default_rng(3)
    tokens, kvh = 24, 2
    x = rng.standard_normal((tokens, 2 + 2 * kvh, dim))
    x[0] = 0
    x[1] = -0.0
    x[2] = np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0], dim // 16)
    x[3] = x[2] * 2.0 ** 100
    x[4] = x[2] * 2.0 ** -110
    x[5, :, ::32] = 3.3895e38  # the largest bf16
    x[6] *= 2.0 ** -130
    x[7, :, 5] = np.inf
    x[8, :, 40] = -np.inf
    x[9, :, 33] = np.nan
    x[10] = np.where(np.arange(dim) % 32 == 0, 6.03125, x[10])
    x[11] = np.where(np.arange(dim) % 32 == 0, 7.96875, x[11])
    x[12] = np.where(np.arange(dim) % 32 == 31, -6.0, x[12])
    x[13] *= 1e30
    x[14] *= 1e-30
    x[15] = 2.0 ** -126
    x[16, :, :32] = 0
    b = Batch(rng, tokens, 2, kvh, dim, 16, 16, False, data=x)
    b.tab[..., 0], b.tab[..., 1] = 1, 0  # as they are (but for an infinity beside a 0)
    b.slots, b.pos = rng.permutation(b.pages * 16)[:tokens].astype(np.uint64), np.zeros(tokens, np.uint32)
    b.there, b.at = np.ones(tokens, bool), b.pos
    _check4(b, False, True)


def test_no_slots_at_all():
    say("no slots")
    rng = np.random.default_rng(8)
    b = Batch(rng, 9, 4, 2, 64, 16, 64, True)
    kv = ca.PagedKV(0, 0, 0, 1, 16, 1, 1, 2, 64)
    q, copies = b.run(kv, True, True, slots=False)
    for got, exp in zip((q, *copies), b.expected(True)):
        assert np.array_equal(got, exp)
    kv4 = ca.PagedKV4(0, 0, 0, 0, 0, 1, 16, 1, 1, 2, 64)
    q, copies = b.run(kv4, True, True, slots=False)
    assert np.array_equal(q, b.expected(True)[0])
    assert np.array_equal(f64(copies[0]), plain.quantise_k(b.expected(True)[1])[2])


@pytest.mark.parametrize("first,n,rot,mscale", [(0, 1, 2, 1.0), (0, 300, 128, 1.0), (1 << 20, 257, 64, 1.25), (0xFFFFFF00, 255, 16, 1.0)])
def test_table(first, n, rot, mscale):
    """cos and sin in double of an angle whose product is rounded once (2^-53 of it), the
    functions to a few 2^-52, then one rounding to f32."""
    say(f"table {first} {n} {rot}")
    f = ca.rope_inv_freq_scaled(rot, 10000.0, ca.ROPE_LINEAR, 2.0)
    tab = ca.Buffer(n * rot * 4)
    ca.rope_table_scaled_f32(ca.Buffer.from_array(f), tab, first, n, rot, mscale)
    got = tab.read(np.float32, (n, rot // 2, 2))
    angle = (first + np.arange(n, dtype=np.float64))[:, None] * f
    want = mscale * np.stack([np.cos(angle), np.sin(angle)], -1)
    assert np.all(np.abs(got - want) <= U * np.abs(want) + mscale * (2.0 ** -52 * angle[..., None] + 2.0 ** -50))
