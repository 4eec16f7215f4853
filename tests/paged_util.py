"""Caches in pages for the tests: built on the host, with NaN in every place that
no slot in use has, and read back the same way (not collected by pytest)."""
import numpy as np

import catena_amd as ca
import oracle

U = 2.0 ** -24     # f32 unit roundoff
UB = 2.0 ** -8     # bf16: half a step relative to the value
NAN16 = 0x7FC0


def bf16(x) -> np.ndarray:
    return oracle.f32_to_bf16_bits_np(np.ascontiguousarray(x, np.float32))


def f64(bits) -> np.ndarray:
    return oracle.bf16_bits_to_f32(np.ascontiguousarray(bits)).astype(np.float64)


class Cache:
    """rows of `lens` slots in pages, each row's pages anywhere in the pool; lazy:
    pages for the slots in use alone, table entries behind them name none."""

    def __init__(self, rng, lens, kv_heads, dim, page, max_pages, spare=0, scale=1.0, lazy=False):
        self.lens = np.asarray(lens, np.uint32)
        rows = len(self.lens)
        self.page, self.max_pages, self.kv_heads, self.dim = page, max_pages, kv_heads, dim
        self.slots = page * max_pages
        used = np.minimum(-(-self.lens // page), max_pages) if lazy else np.full(rows, max_pages)
        num = max(int(used.sum()) + spare, 1)
        order = rng.permutation(num).astype(np.uint32)
        self.table = np.full((rows, max_pages), 0xFFFFFFFF, np.uint32)
        self.table[np.arange(max_pages) < used[:, None]] = order[: int(used.sum())]
        self.spare = order[int(used.sum()):].copy()
        self.num_pages = num
        self.k = np.full((num, kv_heads, page, dim), NAN16, np.uint16)
        self.v = self.k.copy()
        for r in range(rows):
            n = min(int(self.lens[r]), self.slots)
            for pool in (self.k, self.v):
                self.put(pool, r, np.arange(n), bf16(rng.standard_normal((kv_heads, n, dim)) * scale))

    def put(self, pool, row, slots, values):
        """values [kv_heads][len(slots)][dim] into a row's slots."""
        pool[self.table[row, slots // self.page], :, slots % self.page] = values.transpose(1, 0, 2)

    def get(self, pool, row, n):
        """[kv_heads][n][dim] bits of a row's first n slots."""
        slots = np.arange(n)
        return pool[self.table[row, slots // self.page], :, slots % self.page].transpose(1, 0, 2)

    def upload(self):
        self.bufs = [ca.Buffer.from_array(x) for x in (self.k, self.v, self.table, self.lens)]
        self.kb, self.vb, self.tb, self.lb = self.bufs
        self.kv = ca.PagedKV(self.kb.ptr, self.vb.ptr, self.tb.ptr, self.num_pages, self.page, len(self.lens),
                             self.max_pages, self.kv_heads, self.dim)
        return self.kv

    def download(self):
        shape = self.k.shape
        return self.kb.read(np.uint16, shape), self.vb.read(np.uint16, shape)


def geometry(**over) -> ca.PagedKV:
    """A cache's handle whose pointers are never followed (refusals)."""
    kv = ca.PagedKV(1 << 20, 1 << 21, 1 << 22, 64, 16, 4, 16, 4, 128)
    for name, value in over.items():
        setattr(kv, name, value)
    return kv


def refused(status, call, *args, **kw):
    try:
        call(*args, **kw)
    except ca.CatenaError as e:
        assert e.status == status, str(e)
        assert ca.last_error()
        return
    raise AssertionError("the call was not refused")


def attention(q, k, v, scale):
    """(o, p, sum p |v|, bound on a score's error) of one kv head's queries in 64
    bits: q [group][dim], k / v [n][dim].

    A score is a sum of dim products in f32 (any order: at most dim + 1
    roundings on the way of each) times two rounded constants: (dim + 4) u of
    the sum of magnitudes."""
    with np.errstate(all="ignore"):
        s = (q @ k.T) * scale
        e = np.exp(s - s.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
        es = (q.shape[1] + 4) * U * (np.abs(q) @ np.abs(k).T).max() * abs(scale)
        return p @ v, p, p @ np.abs(v), es


def attention_slack(es, n):
    """Relative error of a probability, and of a sum weighted by it: e^(error of
    a score) above and below the fraction, 2 u of the exponential and 4 of the
    factors between partial sums each, and f32 sums of n terms whose longest
    chain is n / 16 + 64 adds."""
    return 2 * es + (12 + 2 * (n / 16 + 64)) * U
