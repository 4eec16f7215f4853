"""One graph of attention over a 4-bit cache whose lengths change, every replay against the
formula: the cache is filled for the longest of them."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from test_gpu_attn_q4 import Rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


@pytest.mark.parametrize("heads,kvh,dim,most,all_lens", [
    (8, 2, 128, [1999, 640, 2000], [[900, 33, 2000], [1, 0, 5], [1999, 640, 16], [1999, 640, 2000], [0, 640, 513]]),
    (12, 1, 64, [9000, 100], [[9000, 100], [1, 100], [0, 0], [513, 1], [8999, 99]]),  # cut for some lengths, whole for others
])
def test_replays_are_right(heads, kvh, dim, most, all_lens):
    say(f"q4 replays {heads} {kvh} {dim}")
    x = Rows(np.random.default_rng(dim), most, heads, kvh, dim, 16, -(-max(most) // 16))
    x.run()
    replay = captured(x.call)
    for lens in all_lens:
        x.c.lens = np.array(lens, np.uint32)
        x.c.lb.write(x.c.lens)
        for go in (replay, x.call, replay):
            x.o.write(np.full(x.q.shape, 7, np.uint16))
            go()
            ca.synchronize()
            x.check(x.o.read(np.uint16, x.q.shape))
