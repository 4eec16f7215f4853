"""A request that asks for more pages than are free, in front of requests that run: who is
stopped, how a caller sees it, and that taking the request back lets the others go on, in one
captured step."""
import numpy as np

import pytest

import catena_amd as ca
import requests_util as plain
from gpu_util import captured, say
from paged_util import geometry

pytestmark = pytest.mark.gpu


def test_a_request_that_waits_in_front():
    say("admission in the order of rows")
    ca.init(0)
    page, max_pages, spare = 16, 64, 5
    lens = np.array([0, 16, 31, 48, 5], np.uint32)  # the second and fourth need a page for their next token
    held = (-(-lens.astype(int) // page)).astype(np.uint32)
    rows, num = len(lens), int(held.sum()) + spare
    order = np.random.default_rng(0).permutation(num).astype(np.uint32)
    table = np.full((rows, max_pages), 0xFFFFFFFF, np.uint32)
    table[np.arange(max_pages) < held[:, None]] = order[: held.sum()]
    free = order[held.sum():]
    up = lambda x: ca.Buffer.from_array(np.asarray(x, np.uint32))  # noqa: E731
    kv = geometry(k=0, v=0, table=0, num_pages=num, page_size=page, rows=rows, max_pages=max_pages, kv_heads=1)
    t, ins, want, stack, count = up(table), (up(lens), up(held)), up(np.zeros(rows)), up(np.concatenate([free, np.zeros(num - spare)])), up([spare])
    out = [ca.Buffer(4 * rows), ca.Buffer(4 * rows), ca.Buffer(4 * (rows + 1)), ca.Buffer(4), ca.Buffer(4 * 200), ca.Buffer(8 * 200)]
    step = captured(lambda: ca.kv_admit_paged(kv, t, *ins, want, stack, count, *out, 200))
    for ask, expect in (([6 * page, 1, 1, 1, 1], [0, 0, 1, 0, 1]),  # 6 pages of 5: who needs a page waits too
                        ([0, 1, 1, 1, 1], [0, 1, 1, 1, 1]),         # taken back: all others go on
                        ([5 * page, 1, 1, 1, 1], [5 * page, 0, 1, 0, 1]),
                        ([201, 1, 1, 1, 1], [0] * 5)):              # more than the list: nobody behind it
        t.write(table)
        want.write(np.array(ask, np.uint32))
        step()
        ca.synchronize()
        got = out[0].read(np.uint32).astype(int) - lens
        assert got.tolist() == expect
        starts = out[2].read(np.uint32)
        assert starts[rows] == sum(expect) and (starts[rows] < sum(ask)) == (expect != ask)
        exp = plain.admit(table, lens, held, np.array(ask, np.uint32), free, spare, page, 200)
        assert np.array_equal(t.read(np.uint32, table.shape), exp[0]) and int(out[3].read(np.uint32)[0]) == exp[4]
        assert np.array_equal(out[5].read(np.uint64), exp[6])
