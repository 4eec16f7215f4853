"""Plain forms of the operators for requests of different lengths, in numpy, for the
tests (not collected by pytest)."""
import numpy as np

import catena_amd as ca
import oracle
from paged_util import U, bf16, f64

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([GRID, -GRID])
NAN16 = 0x7FC0


def admit(table, lens, held, want, free, count, page, max_tokens, seen=None):
    """What kv_admit_paged does, row by row; num_pages: as many as there are entries in `free`."""
    table, lens, held = table.copy(), lens.astype(np.int64), held.astype(np.int64)
    slots = table.shape[1] * page
    seen = lens if seen is None else seen.astype(np.int64)
    starts, pos, place = [0], [], []
    tokens = pages = taken = 0
    lens_out, held_out = lens.copy(), held.copy()
    for r in range(len(lens)):
        t = int(want[r]) if lens[r] + int(want[r]) <= slots else 0
        p = max(0, -(-(int(lens[r]) + t) // page) - int(held[r])) if t else 0
        tokens, pages = tokens + t, pages + p
        if tokens > max_tokens or (p and pages > count):
            t = p = 0
        for i in range(p):
            table[r, held[r] + i] = free[count - 1 - taken - i]
        taken += p
        lens_out[r] += t
        held_out[r] += p
        starts.append(starts[-1] + t)
        for i in range(t):
            slot = int(lens[r]) + i
            pos.append(int(seen[r]) + i)
            place.append(int(table[r, slot // page]) * page + slot % page)
    rest = max_tokens - len(pos)
    return (table, lens_out, held_out, np.array(starts), count - taken, np.array(pos + [0] * rest, np.int64),
            np.array(place + [2 ** 64 - 1] * rest, np.uint64), seen + (lens_out - lens))


def turn(x, tab, rot, interleaved):
    """Heads x [tokens][heads][dim] f32 turned by tab [tokens][rot / 2][2] f32, each operation rounded, to bf16 bits."""
    y = x.astype(np.float32).copy()
    cos, sin = tab[:, None, :, 0], tab[:, None, :, 1]
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    with np.errstate(all="ignore"):
        x1, x2 = y[..., a].copy(), y[..., b].copy()
        y[..., a] = x1 * cos - x2 * sin
        y[..., b] = x2 * cos + x1 * sin
    return bf16(y)


def codes(x, unit):
    """The nearest codes of x / unit (f64), of two the even one; 0 where unit is 0."""
    with np.errstate(all="ignore"):
        a = np.where(unit > 0, np.abs(x) / np.where(unit > 0, unit, 1), 0)
    d = np.abs(a[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    near = d == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(near.sum(-1) > 1, even.argmax(-1), near.argmax(-1))
    return np.where((unit > 0) & np.signbit(x), code + 8, code).astype(np.uint8)


def quantise_k(bits):
    """(codes, scale bytes, values in f64) of bf16 bits [..., dim]."""
    x = f64(bits).reshape(*bits.shape[:-1], bits.shape[-1] // 32, 32)
    odd = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(odd, 0, x)
    top = np.abs(x).max(-1, keepdims=True)
    e = np.full(top.shape, -127)
    for k in range(-127, 128):  # the smallest power of two with top <= 6 of them
        e = np.where(top > 6 * 2.0 ** k, k + 1, e)
    unit = 2.0 ** e
    code = np.where(odd, 0, codes(x, np.broadcast_to(unit, x.shape)))
    value = np.where(odd, np.nan, VALUES[code] * unit)
    return code.reshape(bits.shape).astype(np.uint8), np.where(odd, 255, e + 127)[..., 0].astype(np.uint8), value.reshape(bits.shape)


def quantise_v(bits):
    """(codes, scale in bf16 bits, values in f64) of bf16 bits [..., dim]."""
    x = f64(bits)
    odd = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(odd, 0, x)
    with np.errstate(all="ignore"):
        sixth = (np.abs(x).max(-1, keepdims=True) / 6).astype(np.float32)
    s16 = ((sixth.view(np.uint32).astype(np.uint64) + 0xFFFF) >> 16).astype(np.uint16)
    unit = f64(s16)
    code = np.where(odd, 0, codes(x, np.broadcast_to(unit, x.shape)))
    value = np.where(odd, np.nan, VALUES[code] * unit)
    return code.astype(np.uint8), np.where(odd, NAN16, s16)[..., 0].astype(np.uint16), value


def pack(code):
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)


class Cache4:
    """rows of `lens` slots in pages of 4 bits, anything in every other place."""

    def __init__(self, rng, lens, kv_heads, dim, page, max_pages, lazy=False, scale=1.0):
        self.lens = np.asarray(lens, np.uint32)
        rows = len(self.lens)
        self.page, self.max_pages, self.kv_heads, self.dim, self.slots = page, max_pages, kv_heads, dim, page * max_pages
        used = np.minimum(-(-self.lens.astype(np.int64) // page), max_pages) if lazy else np.full(rows, max_pages)
        self.num_pages = max(int(used.sum()), 1)
        order = rng.permutation(self.num_pages).astype(np.uint32)
        self.table = np.full((rows, max_pages), 0xFFFFFFFF, np.uint32)
        self.table[np.arange(max_pages) < used[:, None]] = order[: int(used.sum())]
        # what no slot in use has: any codes, scales that are NaN
        self.k = rng.integers(0, 256, (self.num_pages, kv_heads, page, dim // 2)).astype(np.uint8)
        self.v = rng.integers(0, 256, (self.num_pages, kv_heads, dim // 2, page)).astype(np.uint8)
        self.k_scale = np.full((self.num_pages, kv_heads, dim // 32, page), 255, np.uint8)
        self.v_scale = np.full((self.num_pages, kv_heads, page), NAN16, np.uint16)
        self.values = []
        for r in range(rows):
            n = min(int(self.lens[r]), self.slots)
            k16, v16 = (bf16(rng.standard_normal((kv_heads, n, dim)) * s) for s in (scale * np.exp(0.7 * rng.standard_normal((kv_heads, 1, dim))), 1.0))
            self.put(r, np.arange(n), k16, v16)

    def put(self, r, slots, k16, v16):
        """bf16 keys and values [kv heads][slots][dim] into a row's slots."""
        at, place = self.table[r, slots // self.page], slots % self.page
        code, scale, _ = quantise_k(k16)
        self.k[at, :, place] = pack(code).transpose(1, 0, 2)
        self.k_scale[at, :, :, place] = scale.transpose(1, 0, 2)
        code, scale, _ = quantise_v(v16)
        self.v[at, :, :, place] = pack(code).transpose(1, 0, 2)
        self.v_scale[at, :, place] = scale.T

    def get(self, r, n):
        """The values [kv heads][n][dim] of a row's first n slots, f64."""
        slots = np.arange(n)
        at, place = self.table[r, slots // self.page], slots % self.page
        out = []
        for pool, unit in ((self.k[at, :, place], 2.0 ** (self.k_scale[at, :, :, place].astype(np.float64) - 127)),
                           (self.v[at, :, :, place], f64(self.v_scale[at, :, place])[..., None])):
            unit = np.where(self.k_scale[at, :, :, place] == 255, np.nan, unit) if unit.shape[-1] > 1 else unit
            x = VALUES[np.stack([pool & 15, pool >> 4], -1).reshape(n, self.kv_heads, self.dim)]
            out.append((x.reshape(n, self.kv_heads, unit.shape[-1], -1) * unit[..., None]).reshape(x.shape).transpose(1, 0, 2))
        return out

    def upload(self):
        self.bufs = [ca.Buffer.from_array(x) for x in (self.k, self.v, self.k_scale, self.v_scale, self.table, self.lens)]
        self.lb = self.bufs[5]
        self.kv = ca.PagedKV4(*[b.ptr for b in self.bufs[:5]], self.num_pages, self.page, len(self.lens), self.max_pages,
                              self.kv_heads, self.dim)
        return self.kv

    def download(self):
        for b, x in zip(self.bufs[:4], (self.k, self.v, self.k_scale, self.v_scale)):
            x[...] = b.read(x.dtype, x.shape)


def prompt_slack(es, n):
    """Relative error of a sum weighted by the probabilities of n slots: e^(error of a
    score) above and below the fraction, sums of n terms whose longest chain is n / 2 +
    64 adds each, and 200 u for the exponential, its argument (up to 126 in base 2, so 90
    u), and the factors between partial sums."""
    return 2 * es + (200 + n + 128) * U
