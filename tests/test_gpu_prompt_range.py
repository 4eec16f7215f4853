"""The ends of prompt attention's range: values so small that products of them with p are
below the smallest normal number, infinities of small weight. Wide units, seen whole or
not, and narrow ones."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import attention, bf16, f64
from test_gpu_attn_prompt import Prompt, _bound

pytestmark = pytest.mark.gpu
SHAPES = [([90], [200]), ([2], [290]), ([300, 1], [1200, 1500])]  # rows of 4 x 2 heads: wide, narrow, both from a list


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


def _prompt(rng, n, ctx, dim, packed):
    return Prompt(rng, n, [0] * len(n) if packed else ctx, 4, 2, dim, 0 if packed else 16)


@pytest.mark.parametrize("size", [-70, -80, -100])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,ctx", SHAPES)
def test_tiny_values(n, ctx, dim, size):
    """Products below 2^-126 may be lost: of a row's slots 2 each (p's terms) and fewer sums
    than that, 6 n at most with the roundings around them, over a sum of p 2^-ease >= 2^-11 / n
    (the largest p is above 1/2, ease at most 10 + log2 n): n^2 2^-113 of o."""
    say(f"tiny values {n} {ctx} {dim} {size}")
    p = _prompt(np.random.default_rng(dim), n, ctx, dim, False)
    p.cache.v = np.where(p.cache.v == 0x7FC0, 0x7FC0, bf16(f64(p.cache.v).astype(np.float32) * np.float32(2.0 ** size))).astype(np.uint16)
    got = p.run()
    for r in range(p.rows):
        k, v = p.kv_of(r)
        for t in sorted({0, n[r] // 2, n[r] - 1}):
            slots, at = p.ctx[r] + t + 1, int(p.starts[r]) + t
            for h in range(2):
                mine = slice(2 * h, 2 * h + 2)
                want, _, pv, es = attention(f64(p.q[at, mine]), k[h, :slots], v[h, :slots], p.scale)
                bound = _bound(es, slots, pv, want) + float(p.lens[r]) ** 2 * 2.0 ** -113
                assert np.all(np.abs(f64(got[at, mine]) - want) <= bound), (r, t, h)


@pytest.mark.parametrize("n,ctx,weight", [(n, ctx, w) for n, ctx in SHAPES for w in (-20, -60, -80)] + [(*SHAPES[0], -100)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("packed", [False, True])
def test_infinities_of_small_weight(n, ctx, dim, packed, weight):
    """One slot of each row has a weight of 2^weight beside the others' 1 and an infinity in its value: its column is
    infinite from its own token on, all others as without it."""
    say(f"infinity of weight 2^{weight}: {n} {ctx} {dim} {packed}")
    p = _prompt(np.random.default_rng(dim), n, ctx, dim, packed)
    p.scale = float(np.float32(np.log(2.0)))
    q = np.zeros(p.q.shape, np.float32)
    q[..., 3] = -weight
    p.q = bf16(q)
    at = [min(70, int(x) - 1) for x in p.lens]

    def put(bits):
        for r in range(p.rows):
            length = int(p.lens[r])
            k = np.zeros((2, length, dim), np.float32)
            k[:, at[r], 3] = -1
            k = bf16(k)
            if packed:
                a = int(p.starts[r])
                p.k[a:a + length, : 2 * dim] = k.transpose(1, 0, 2).reshape(length, -1)
                p.v[a + at[r], 5] = bits
            else:
                p.cache.put(p.cache.k, r, np.arange(length), k)
                p.cache.v[p.cache.table[r, at[r] // 16], 0, at[r] % 16, 5] = bits
    put(0x3F80)
    base = p.run()
    for bits, sign in ((0x7F80, 1.0), (0xFF80, -1.0)):
        put(bits)
        got = p.run()
        x, same = f64(got[: p.starts[-1]]), np.ones((int(p.starts[-1]), 4, dim), bool)
        for r in range(p.rows):
            first = int(p.starts[r]) + max(0, at[r] - p.ctx[r])  # the first token that sees it
            last = int(p.starts[r + 1])
            assert np.all(x[first:last, :2, 5] == sign * np.inf), r
            same[first:last, :2, 5] = False
        assert np.array_equal(got[: p.starts[-1]][same], base[: p.starts[-1]][same])
