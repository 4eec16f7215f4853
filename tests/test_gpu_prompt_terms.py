"""Units of up to 64 query rows take p in two bf16 terms, as attention of one token over pages
does: the upper half of p's bits and what it leaves over, rounded, off by 2^-16 of p at most
(2^-20 more where the second term would be 0); the sum of p is that of the whole ones. So
their results are off by that of sum p |v| and their own rounding, not by 2^-8 of it."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import say
from paged_util import UB, attention, f64
from requests_util import prompt_slack
from test_gpu_attn_prompt import Prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Fine(Prompt):
    def check(self, got, rows=None):
        group = self.heads // self.kvh
        for r in range(self.rows) if rows is None else rows:
            k, v = self.kv_of(r)
            first = max(self.n[r] * group - 1, 0) // 256 * 256  # query row of the last unit; the others are wide
            if self.n[r] * group - first > 64:
                continue
            for t in range(-(-first // group), self.n[r]):
                n, at = self.ctx[r] + t + 1, int(self.starts[r]) + t
                for h in range(self.kvh):
                    mine = slice(h * group, (h + 1) * group)
                    want, _, pv, es = attention(f64(self.q[at, mine]), k[h, :n], v[h, :n], self.scale)
                    off = (prompt_slack(es, n) + 2.0 ** -16 + 2.0 ** -20) * pv
                    assert np.all(np.abs(f64(got[at, mine]) - want) <= off + UB * (np.abs(want) + off)), (r, t, h)


@pytest.mark.parametrize("n,ctx,heads,kvh,dim,page", [
    ([1], [900], 8, 1, 128, 16), ([16, 1, 5], [500, 90, 0], 8, 2, 64, 32), ([64], [700], 2, 2, 128, 64),  # no list
    ([1, 7, 16], [20000, 3000, 5000], 32, 8, 128, 16), ([5], [33000], 4, 1, 64, 16), ([33, 64, 2], [2000, 1500, 7], 1, 1, 64, 64),
    ([260, 1], [1100, 2000], 3, 3, 128, 16),  # the last unit of a row with wide ones
])
def test_pages(n, ctx, heads, kvh, dim, page):
    say(f"terms {n} {ctx} {heads} {kvh} {dim} {page}")
    p = Fine(np.random.default_rng(sum(ctx)), n, ctx, heads, kvh, dim, page)
    p.check(p.run())


@pytest.mark.parametrize("n,heads,kvh,dim", [([64, 1, 30], 2, 2, 64), ([16, 9], 32, 8, 128), ([320, 1000, 60], 1, 1, 64)])
def test_packed(n, heads, kvh, dim):
    say(f"terms, packed {n} {heads} {kvh} {dim}")
    p = Fine(np.random.default_rng(sum(n)), n, [0] * len(n), heads, kvh, dim, 0)
    p.check(p.run())


def test_many_narrow_units():
    say("terms, many narrow units")
    rng = np.random.default_rng(8)
    n, ctx = rng.integers(1, 4, 300), rng.integers(0, 600, 300)
    ctx[3] = 5000
    p = Fine(rng, n, ctx, 16, 8, 64, 16)
    p.check(p.run(), [0, 1, 3, 50, 299])


def test_as_attention_of_one_token():
    """Rows of one token each, also by attn_paged_bf16: values that differ by some 2^-17 of the largest
    terms, which are as large as o where p is even, round to neighbours in bf16 (steps of 2^-7 to 2^-8)
    in one case of 2^9 or so; rounded p, 2^-9 of the terms, does in about half of them."""
    say("single tokens by both calls")
    rng = np.random.default_rng(9)
    p = Fine(rng, [1] * 6, [0, 40, 700, 5000, 63, 2000], 16, 4, 128, 16)
    got = p.run()
    p.check(got)
    kv = p.cache.upload()
    work, o, q = ca.Buffer(max(ca.attn_paged_plan(kv, 16)[1], 16)), ca.Buffer(p.q.nbytes), ca.Buffer.from_array(p.q)
    ca.attn_paged_bf16(kv, q, p.cache.lb, o, 16, p.scale, work)
    assert (got[:6] != o.read(np.uint16, p.q.shape)).mean() < 0.05
