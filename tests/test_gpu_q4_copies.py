"""The copies that rope_packed_q4 writes beside a cache in 4 bits: k's are what the cache holds,
v's that rounded to bf16, half a step (2^-8 of it) at most."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import UB, bf16, f64
from requests_util import VALUES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_copies_are_what_the_cache_holds(dim):
    say(f"copies {dim}")
    ca.init(0)
    rng = np.random.default_rng(dim)
    tokens, kvh, page, pages = 50, 3, 16, 5
    qkv = bf16(rng.standard_normal((tokens, 4 * kvh, dim)) * np.exp2(rng.integers(-100, 100, (tokens, 1, 1))))
    shapes = ((pages, kvh, page, dim // 2), (pages, kvh, dim // 2, page), (pages, kvh, dim // 32, page))
    pools = [ca.Buffer.from_array(np.zeros(s, np.uint8)) for s in shapes] + [ca.Buffer.from_array(np.zeros((pages, kvh, page), np.uint16))]
    slots = rng.permutation(page * pages)[:tokens].astype(np.uint64)
    up = [ca.Buffer.from_array(x) for x in (qkv, rng.standard_normal((9, dim // 2, 2)).astype(np.float32), rng.integers(0, 9, tokens).astype(np.uint32), slots)]
    q, k_out, v_out = (ca.Buffer(tokens * h * dim * 2) for h in (2 * kvh, kvh, kvh))
    kv = ca.PagedKV4(*[p.ptr for p in pools], 0, pages, page, 1, 1, kvh, dim)
    ca.rope_packed_q4(kv, up[0], False, up[1], 9, dim, False, up[2], up[3], q, tokens, 2 * kvh, k_out, v_out)
    at, place = (slots // page).astype(int), (slots % page).astype(int)
    k, v, ks, vs = (p.read(t, s) for p, t, s in zip(pools, (np.uint8,) * 3 + (np.uint16,), shapes + ((pages, kvh, page),)))
    values = lambda x: VALUES[np.stack([x & 15, x >> 4], -1).reshape(tokens, kvh, dim)]  # noqa: E731
    held = values(k[at, :, place]) * np.repeat(np.exp2(ks[at, :, :, place].astype(np.float64) - 127), 32, -1)
    assert np.array_equal(f64(k_out.read(np.uint16, (tokens, kvh, dim))), held)
    held = values(v[at, :, :, place]) * f64(vs[at, :, place])[..., None]
    copies = f64(v_out.read(np.uint16, (tokens, kvh, dim)))
    assert np.all(np.abs(copies - held) <= UB * np.abs(held)) and np.any(copies != held)
