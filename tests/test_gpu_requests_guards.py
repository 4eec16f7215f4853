"""Workspaces and outputs of exactly the size that the calls ask for, with marked bytes
behind them that have to stay, and workspaces that hold anything (all bits set) before."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import UB, attention, bf16, f64
from requests_util import Cache4
from test_gpu_attn_prompt import _bound
from test_gpu_attn_q4 import _slack

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Guarded:
    """nbytes of `fill`, and marks behind them."""

    def __init__(self, nbytes, fill=0xFF):
        self.n = int(nbytes)
        self.buf = ca.Buffer(self.n + GUARD)
        self.buf.write(np.concatenate([np.full(self.n, fill, np.uint8), np.arange(GUARD, dtype=np.uint32).astype(np.uint8)]))
        self.ptr = self.buf.ptr

    @property
    def _as_parameter_(self):
        return self.ptr

    def kept(self):
        return np.array_equal(self.buf.read(np.uint8, (GUARD,), self.n), np.arange(GUARD, dtype=np.uint32).astype(np.uint8))

    def read(self, dtype, shape):
        return self.buf.read(dtype, shape)


class Shared:
    """Rows that all read the same `slots` slots, a table of their own pages each row alike."""

    def __init__(self, rng, rows, slots, kvh, dim, page):
        pages = -(-slots // page)
        self.k, self.v = (bf16(rng.standard_normal((pages, kvh, page, dim))) for _ in range(2))
        self.table = np.tile(rng.permutation(pages).astype(np.uint32), (rows, 1))
        self.bufs = [ca.Buffer.from_array(x) for x in (self.k, self.v, self.table)]
        self.kv = ca.PagedKV(*[b.ptr for b in self.bufs], pages, page, rows, pages, kvh, dim)

    def get(self, h, n):
        return (f64(x[self.table[0], h].reshape(-1, x.shape[-1])[:n]) for x in (self.k, self.v))


# rows, new tokens of each, slots of each, heads, kv heads, dim: every unit of a share just
# above a CU's, so that all are cut in two (wide: the most places of parts that there can
# be), a few narrow units in many parts, both beside each other, so many narrow ones that two
# waves share each, wide ones that are not cut, and no list
PROMPTS = [(85, [64] * 85, [9600] * 85, 16, 4, 64), (1, [1], [130000], 32, 8, 64), (3, [64, 16, 1], [9000, 20000, 30000], 16, 4, 128),
           (300, [1] * 300, [600] * 299 + [9000], 16, 8, 64), (5, [700, 300, 65, 64, 3], [700] * 5, 4, 4, 128), (4, [70, 3, 1, 0], [900] * 4, 8, 2, 128)]


@pytest.mark.parametrize("rows,n,lens,heads,kvh,dim", PROMPTS)
def test_prompt(rows, n, lens, heads, kvh, dim):
    say(f"guards, prompt {rows} {sum(n)} {max(lens)} {heads} {kvh} {dim}")
    rng = np.random.default_rng(rows)
    c = Shared(rng, rows, max(max(lens), 1100 if rows != 4 else 0), kvh, dim, 16)
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    tokens, group = int(starts[-1]), heads // kvh
    q = bf16(rng.standard_normal((tokens, heads, dim)))
    need = ca.attn_prompt_plan(c.kv, tokens, heads)
    assert (need == 0) == (rows == 4)
    work, o = Guarded(max(need, 16)), Guarded(q.nbytes)
    up = [ca.Buffer.from_array(x) for x in (q, starts, np.array(lens, np.uint32))]
    ca.attn_prompt_bf16(c.kv, *up, o, tokens, heads, dim ** -0.5, (work.ptr, need))
    got = o.read(np.uint16, q.shape)
    assert work.kept() and o.kept()
    for r in sorted({0, rows // 2, rows - 2, rows - 1} & set(range(rows))):
        for t in sorted({0, n[r] // 2, n[r] - 1} & set(range(n[r]))):
            at, slots = int(starts[r]) + t, lens[r] - n[r] + t + 1
            for h in {0, kvh - 1}:
                k, v = c.get(h, slots)
                mine = slice(h * group, (h + 1) * group)
                want, _, pv, es = attention(f64(q[at, mine]), k, v, dim ** -0.5)
                assert np.all(np.abs(f64(got[at, mine]) - want) <= _bound(es, slots, pv, want)), (r, t, h)


@pytest.mark.parametrize("n,heads,kvh,dim", [([1500, 40, 1], 8, 2, 128), ([300] * 30, 2, 2, 64), ([60, 70], 4, 1, 128)])
def test_packed(n, heads, kvh, dim):
    say(f"guards, packed {n[:3]} {heads} {kvh} {dim}")
    rng = np.random.default_rng(heads)
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    tokens = int(starts[-1])
    q, k, v = (bf16(rng.standard_normal((tokens, h, dim))) for h in (heads, kvh, kvh))
    need = ca.attn_packed_plan(len(n), tokens, heads, kvh, dim)
    work, o = Guarded(max(need, 16)), Guarded(q.nbytes)
    up = [ca.Buffer.from_array(x) for x in (q, k, v, starts)]
    ca.attn_packed_bf16(*up, o, len(n), tokens, heads, kvh, dim, dim ** -0.5, (work.ptr, need))
    got = o.read(np.uint16, q.shape)
    assert work.kept() and o.kept()
    a, last, group = int(starts[0]), n[0] - 1, heads // kvh
    want, _, pv, es = attention(f64(q[last, :group]), f64(k[a:a + n[0], 0]), f64(v[a:a + n[0], 0]), dim ** -0.5)
    assert np.all(np.abs(f64(got[last, :group]) - want) <= _bound(es, n[0], pv, want))


@pytest.mark.parametrize("lens,heads,kvh,dim,pages", [([7000], 8, 8, 64, 440), ([40000, 1], 24, 1, 128, 2500), ([9000] + [3] * 130, 16, 4, 128, 600)])
def test_q4(lens, heads, kvh, dim, pages):
    """Cut rows; in the last case more workgroups than parts."""
    say(f"guards, 4 bits {lens[:2]} {heads} {kvh} {dim}")
    rng = np.random.default_rng(dim)
    c = Cache4(rng, lens, kvh, dim, 16, pages, lazy=True)
    kv = c.upload()
    parts, need = ca.attn_paged_q4_plan(kv, heads)
    assert parts > 0
    q = bf16(rng.standard_normal((len(lens), heads, dim)))
    qb, work, o = ca.Buffer.from_array(q), Guarded(need), Guarded(q.nbytes)
    ca.attn_paged_q4(kv, qb, c.lb, o, heads, dim ** -0.5, (work.ptr, need))
    got = o.read(np.uint16, q.shape)
    assert work.kept() and o.kept()
    group = heads // kvh
    for r in (0, len(lens) - 1):
        k, v = c.get(r, lens[r])
        for h in {0, kvh - 1}:
            mine = slice(h * group, (h + 1) * group)
            want, _, pv, es = attention(f64(q[r, mine]), k[h], v[h], dim ** -0.5)
            slack = _slack(es, lens[r])
            assert np.all(np.abs(f64(got[r, mine]) - want) <= slack * pv + UB * (np.abs(want) + slack * pv))


@pytest.mark.parametrize("four", [False, True])
def test_rotation(four):
    say(f"guards, rotation {four}")
    rng = np.random.default_rng(3)
    heads, kvh, dim, tokens, pages, page = 10, 5, 64, 37, 6, 16
    qkv = bf16(rng.standard_normal((tokens, heads + 2 * kvh, dim)))
    cells = pages * kvh * page
    sizes = (cells * dim // 2, cells * dim // 2, cells * dim // 32, cells * 2) if four else (cells * dim * 2,) * 2
    pools = [Guarded(n, 0) for n in sizes]
    q, k_out, v_out = (Guarded(tokens * h * dim * 2) for h in (heads, kvh, kvh))
    tab = rng.standard_normal((50, dim // 2, 2)).astype(np.float32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.uint64)
    slots[[3, 36]] = [2 ** 64 - 1, pages * page]  # no place, and the one behind the pool
    up = [ca.Buffer.from_array(x) for x in (qkv, tab, rng.integers(0, 52, tokens).astype(np.uint32), slots)]
    kv = (ca.PagedKV4 if four else ca.PagedKV)(*[p.ptr for p in pools], 0, pages, page, 1, 1, kvh, dim)
    call = ca.rope_packed_q4 if four else ca.rope_packed_bf16
    call(kv, up[0], False, up[1], 50, 32, False, up[2], up[3], q, tokens, heads, k_out, v_out)
    ca.synchronize()
    assert all(x.kept() for x in pools + [q, k_out, v_out])
    # what does not turn is there as it was
    assert np.array_equal(q.read(np.uint16, (tokens, heads, dim))[..., 32:], qkv[:, :heads, 32:])


def test_admission():
    say("guards, admission and release")
    rng = np.random.default_rng(4)
    rows, page, max_pages, tokens, pages = 1030, 16, 5, 3000, 4000
    lens = rng.integers(0, 70, rows).astype(np.uint32)
    held = (-(-lens.astype(int) // page)).astype(np.uint32)
    order = rng.permutation(pages).astype(np.uint32)
    table = np.full((rows, max_pages), 0xFFFFFFFF, np.uint32)
    table[np.arange(max_pages) < held[:, None]] = order[: int(held.sum())]
    free = order[int(held.sum()):]
    kv = ca.PagedKV(0, 0, 0, pages, page, rows, max_pages, 1, 128)
    up = lambda x: ca.Buffer.from_array(np.asarray(x, np.uint32))  # noqa: E731
    t, stack = Guarded(table.nbytes), Guarded(4 * pages)
    t.buf.write(table)
    stack.buf.write(free)
    out = [Guarded(4 * n) for n in (rows, rows, rows + 1, 1, tokens)] + [Guarded(8 * tokens)]
    ins = [up(x) for x in (lens, held, rng.integers(0, 6, rows), [len(free)], lens + 9, rng.integers(0, 2, rows))]
    seen = Guarded(4 * rows)
    ca.kv_admit_paged(kv, t, *ins[:3], stack, ins[3], *out, tokens, ins[4], seen)
    back = [Guarded(4 * n) for n in (rows, rows, 1)]
    ca.kv_release_paged(kv, t, out[0], out[1], ins[5], stack, out[3], *back)
    ca.synchronize()
    assert all(x.kept() for x in [t, stack, seen] + out + back)
    assert int(out[3].read(np.uint32, (1,))[0]) <= len(free) and int(out[2].read(np.uint32, (rows + 1,))[-1]) <= tokens
