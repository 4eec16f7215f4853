"""Beam search's selection against the formula in 64 bits.  Places are whole
numbers: inputs are drawn until neighbouring scores differ by more than the
calculation can be off, so that the order is the formula's."""
import numpy as np
import pytest

import catena_amd as ca
from gpu_util import captured, say
from paged_util import U

pytestmark = pytest.mark.gpu
EOS = 2


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Select:
    def __init__(self, logits, scores, done, eos=EOS):
        self.logits, self.scores, self.done, self.eos = logits, scores, done, eos
        self.groups, self.beams, self.vocab = logits.shape
        self.lb, self.sb = ca.Buffer.from_array(logits), ca.Buffer.from_array(scores)
        self.db = None if done is None else ca.Buffer.from_array(done)
        self.out = [ca.Buffer.from_array(np.full(scores.shape, 0xABABABAB, np.uint32)) for _ in range(4)]
        self.work = ca.Buffer.from_array(np.full(ca.beam_select_plan(*logits.shape), 0xFF, np.uint8))

    def __call__(self):
        t, p, s, d = self.out
        ca.beam_select_f32(self.lb, self.sb, self.db, t, p, s, d, self.groups, self.beams, self.vocab, self.eos, self.work)

    def read(self):
        t, p, s, d = self.out
        shape = self.scores.shape
        return t.read(np.uint32, shape), p.read(np.uint32, shape), s.read(np.float32, shape), d.read(np.uint32, shape)

    def want(self):
        """(tokens, parents, scores, done, smallest distance of a chosen score to
        the next of another beam)."""
        g, w, v = self.logits.shape
        x = self.logits.astype(np.float64)
        with np.errstate(all="ignore"):
            top = x.max(-1, keepdims=True)
            lse = top + np.log(np.exp(x - top).sum(-1, keepdims=True))
            total = self.scores.astype(np.float64)[..., None] + (x - lse)
            total[~np.isfinite(lse[..., 0])] = -np.inf
        total[~np.isfinite(total)] = -np.inf
        if self.done is not None:
            over = self.done != 0
            total[over] = -np.inf
            total[over, self.eos] = np.where(np.isfinite(self.scores), self.scores, -np.inf)[over]
        tokens, parents, done = (np.zeros((g, w), np.uint32) for _ in range(3))
        scores = np.full((g, w), -np.inf)
        near = np.inf
        for i in range(g):
            flat = total[i].reshape(-1)
            few = np.argpartition(-flat, min(w + 1, flat.size - 1))[: w + 2] if flat.size > 4 * w else np.arange(flat.size)
            # equal ones at the edge belong too
            edge = np.sort(flat[few])[::-1][min(w, len(few)) - 1]
            few = np.flatnonzero(flat >= edge) if np.isfinite(edge) else np.flatnonzero(np.isfinite(flat))
            order = few[np.lexsort((few, -flat[few]))]
            rest = flat[np.setdiff1d(np.argpartition(-flat, min(2 * w, flat.size - 1))[: 2 * w + 1], order[:w])]
            chosen = flat[order[:w]]
            beams = order[:w] // v
            for a in range(len(chosen)):
                others = np.concatenate([chosen[(np.arange(len(chosen)) != a) & (beams != beams[a])], rest])
                gaps = np.abs(others[np.isfinite(others)] - chosen[a])
                near = min(near, gaps[gaps > 0].min(initial=np.inf))
            for j in range(w):
                parents[i, j] = i * w + j
                if j < len(order):
                    b, t = divmod(int(order[j]), v)
                    tokens[i, j], parents[i, j], scores[i, j] = t, i * w + b, flat[order[j]]
                    done[i, j] = t == self.eos or (self.done is not None and self.done[i, b] != 0)
        return tokens, parents, scores, done, near

    def check(self, tied=False):
        tokens, parents, scores, done, near = self.want()
        if not tied:
            assert near > 1e-6, near  # between beams; far beyond what their log sums, off alike, differ by
        got = self.read()
        assert np.array_equal(got[0], tokens)
        assert np.array_equal(got[1], parents)
        assert np.array_equal(got[3], done)
        fine = np.isfinite(scores)
        assert np.array_equal(np.isfinite(got[2]), fine) and np.all(got[2][~fine] == -np.inf)
        # an exponential is off by u of |x - max| log2 e (below 2^6 where it counts, log2 e in f32 and the
        # product's rounding each) and 2 of itself, a sum of 16 by 16 u; one rounding of the result
        bound = (2 * 64 + 18) * U
        assert np.all(np.abs(got[2][fine] - scores[fine]) <= bound + U * np.abs(scores[fine]))


def _draw(seed, groups, beams, vocab, done_share=0.2, scale=2.5, eos=EOS):
    """Inputs whose order the calculation cannot miss."""
    for trial in range(20):
        rng = np.random.default_rng(1000 * seed + trial)
        logits = (scale * rng.standard_normal((groups, beams, vocab))).astype(np.float32)
        scores = (-4 - 8 * rng.random((groups, beams))).astype(np.float32)
        done = (rng.random((groups, beams)) < done_share).astype(np.uint32) if eos != ca.BEAM_NO_EOS else None
        case = Select(logits, scores, done, eos)
        if case.want()[4] > 1e-6:
            return case
    raise AssertionError("no such inputs")


@pytest.mark.parametrize("groups,beams,vocab", [
    (1, 1, 1), (1, 4, 3), (2, 32, 40), (3, 4, 32000), (1, 8, 4096), (1, 8, 4097), (2, 5, 4095), (1, 32, 12289), (7, 3, 1000),
    (1, 1, 300000), (2, 2, 64), (64, 2, 33), (1, 16, 50021),
])
def test_against_the_formula(groups, beams, vocab):
    say(f"beam_select {groups} x {beams} x {vocab}")
    case = _draw(beams + vocab, groups, beams, vocab, eos=min(EOS, vocab - 1))
    case()
    case.check()


def test_no_end_token():
    say("beam_select without an end token")
    case = _draw(5, 2, 4, 5000, eos=ca.BEAM_NO_EOS)
    case()
    case.check()
    assert not case.read()[3].any()


def test_first_step():
    """Every beam but the first at -inf: the first one's best tokens."""
    say("beam_select first step")
    case = _draw(6, 3, 6, 9000)
    scores = np.full((3, 6), -np.inf, np.float32)
    scores[:, 0] = 0
    case = Select(case.logits, scores, np.zeros((3, 6), np.uint32))
    case()
    case.check()
    assert np.all(case.read()[1] == 6 * np.arange(3)[:, None])


@pytest.mark.parametrize("vocab", [50, 4096, 9001])
def test_equal_logits(vocab):
    """Whole rows of one value, more equal logits than the list holds, and few
    values: the lower beam, then the lower token."""
    say(f"beam_select equal logits {vocab}")
    rng = np.random.default_rng(vocab)
    logits = np.zeros((4, 5, vocab), np.float32)
    logits[1] = rng.integers(0, 3, (5, vocab))
    logits[2, :, ::2] = -0.0
    logits[3] = np.where(rng.random((5, vocab)) < 0.5, 7.0, -3.0)
    scores = np.zeros((4, 5), np.float32)
    scores[3] = [-1, -1, -2, -1, -1]
    # rows of groups 1 and 3 must not tie between beams by rounding alone
    case = Select(logits[[0, 2]], scores[[0, 2]], None, ca.BEAM_NO_EOS)
    case()
    case.check(tied=True)
    for i in (1, 3):
        one = Select(np.repeat(logits[i:i + 1, :1], 5, 1), scores[i:i + 1], None, ca.BEAM_NO_EOS)  # equal sums too
        one()
        one.check(tied=True)


def test_masked_and_odd_logits():
    """-inf offers nothing; fewer offered than beams leave places empty; NaN, +inf
    or -inf alone take a beam out; so does a score that is not finite."""
    say("beam_select masked logits")
    case = _draw(8, 8, 4, 6000, done_share=0)
    x, s, d = case.logits.copy(), case.scores.copy(), case.done.copy()
    x[0, :, 10:] = -np.inf               # ten tokens a beam are allowed
    x[1] = -np.inf                       # none
    x[2] = -np.inf
    x[2, 1, 77], x[2, 3, 5000] = 1.0, -2.0  # two in all
    x[3, 0, 4500] = np.nan
    x[4, 2, 3] = np.inf
    x[5, 0], x[5, 1, 5] = np.nan, -np.inf
    s[6] = [np.nan, -np.inf, np.inf, -1]
    d[7] = [1, 1, 0, 1]
    s[7] = [-3, -np.inf, -90, np.nan]    # a done beam far ahead, two of no score
    case = Select(x, s, d)
    case()
    case.check()
    tokens, parents, scores, done = case.read()
    assert np.array_equal(parents[1], 4 + np.arange(4)) and np.all(scores[1] == -np.inf) and not tokens[1].any()
    assert np.sum(np.isfinite(scores[2])) == 2
    assert tokens[7, 0] == EOS and done[7, 0] == 1 and scores[7, 0] == -3


def test_far_logits_beside_a_masked_run():
    """Logits near -2000, and near +2000, in a row of which whole runs are masked:
    the references of the other runs alone count."""
    say("beam_select far logits")
    case = _draw(17, 2, 3, 40000, done_share=0)
    x = case.logits.copy()
    x[0] -= 2000
    x[1] += 2000
    x[:, :, :9000] = -np.inf
    x[:, 1, 17000:] = -np.inf
    case = Select(x, case.scores, case.done)
    case()
    case.check()


def test_every_beam_done():
    say("beam_select all done")
    case = _draw(9, 2, 4, 3000)
    case = Select(case.logits, case.scores, np.full((2, 4), 7, np.uint32))
    case()
    case.check()
    assert np.all(case.read()[3] == 1) and np.all(case.read()[0] == EOS)
    assert np.array_equal(-np.sort(-case.scores, -1), case.read()[2])


def test_in_place_and_replayed():
    """scores_out = scores and done_out = done, step after step; and a graph that
    is replayed on new logits."""
    say("beam_select in place, graph")
    first = _draw(10, 2, 4, 5000)
    first.out[2], first.out[3] = first.sb, first.db
    for seed in (11, 12):
        first()
        first.check()
        _, _, s, d = first.read()
        nxt = _draw(seed, 2, 4, 5000)
        first.logits, first.scores, first.done = nxt.logits, s, d
        first.lb.write(nxt.logits)
    case = _draw(13, 2, 4, 5000)
    replay = captured(case)
    other = _draw(14, 1, 8, 2000)
    for seed in (13, 15, 16):
        nxt = _draw(seed, 2, 4, 5000)
        case.logits, case.scores, case.done = nxt.logits, nxt.scores, nxt.done
        for buf, value in ((case.lb, nxt.logits), (case.sb, nxt.scores), (case.db, nxt.done)):
            buf.write(value)
        for o in case.out:
            o.write(np.full(o.nbytes, 0xEE, np.uint8))
        replay()
        other()
        case.check()
        other.check()


@pytest.mark.parametrize("groups,beams,vocab", [
    (64, 2, 8191), (32, 4, 8192), (16, 4, 16385), (8, 32, 4097), (256, 1, 4096), (1, 16, 70001), (1, 32, 200001), (300, 1, 100),
])
def test_wide_runs(groups, beams, vocab):
    """Batches large enough for runs of 4096 logits: their borders, what is left behind
    the last whole one, and (32 beams) more lists than are joined at once."""
    say(f"beam_select wide runs {groups} x {beams} x {vocab}")
    assert groups * beams * -(-vocab // 4096) >= 256
    case = _draw(beams + vocab, groups, beams, vocab)
    case()
    case.check()


@pytest.mark.parametrize("groups,beams,vocab", [(64, 4, 5000), (1, 32, 200001)])
def test_equal_logits_in_wide_runs(groups, beams, vocab):
    """More equal logits than a run's list or the join's holds, chunk after chunk of
    lists: the lower beam, then the larger logit, then the lower token."""
    say(f"beam_select equal logits, wide runs {groups} x {beams} x {vocab}")
    rng = np.random.default_rng(vocab)
    logits = np.zeros((groups, 1, vocab), np.float32)
    if groups > 1:
        logits[1], logits[2, :, ::2] = rng.integers(0, 3, vocab), -0.0
        logits[3] = np.where(rng.random(vocab) < 0.5, 7.0, -3.0)
    # a group's beams alike, so that their sums are
    case = Select(np.repeat(logits, beams, 1), np.zeros((groups, beams), np.float32), None, ca.BEAM_NO_EOS)
    case()
    case.check(tied=True)
    late = np.zeros((1, beams, vocab), np.float32)
    late[0, :, vocab - 40:] = 1  # the best in the last run of all
    case = Select(late, np.zeros((1, beams), np.float32), None, ca.BEAM_NO_EOS)
    case()
    case.check(tied=True)


@pytest.mark.parametrize("groups,vocab", [(1, 5000), (1, 128000), (40, 32000)])
def test_beams_of_different_shape_close_together(groups, vocab):
    """One logit far above many equal ones, all alike, and a spread: sums that are off
    by different amounts.  An exponential is off by 2.3 u of |x - max| (the
    difference, its product with log2 e, log2 e itself) and 2 u, a sum of 16 of them by 5
    u; the mean of |x - max| under the row's probabilities is at most ln(vocab), 18: 3e-6
    in all, and the result's rounding.  No continuation comes before one that is 6e-6
    above it."""
    say(f"beam_select shapes {groups} x {vocab}")
    rng = np.random.default_rng(vocab)
    beams, offset = 6, 0.3125
    x = np.zeros((groups, beams, vocab), np.float32)
    x[:, 0, 11] = 8.59
    x[:, 1] = offset
    x[:, 2] = 2.5 * rng.standard_normal((groups, vocab))
    x[:, 3, :7] = 12.2
    x[:, 4] = rng.random((groups, vocab))
    x[:, 5, ::3] = -9.7
    best = x.astype(np.float64).max(-1)
    lse = best + np.log(np.exp(x - best[..., None].astype(np.float64)).sum(-1))
    # the beams' best continuations 8e-6 apart, in any order, their scores as far as f32 has them
    place = np.argsort(rng.random((groups, beams)), -1)
    scores = (-1.0 - 8e-6 * place - (best - lse)).astype(np.float32)
    exact = scores.astype(np.float64) + (best - lse)
    case = Select(x, scores, np.zeros((groups, beams), np.uint32))
    case()
    tokens, parents, got, _ = case.read()
    for g in range(groups):
        order = np.sort(exact[g])[::-1]
        assert abs(got[g, 0] - order[0]) <= 3e-6 + U * abs(order[0])
        first = parents[g, 0] - g * beams
        assert exact[g, first] >= order[0] - 6e-6
    # every score is its continuation's
    x64 = x.astype(np.float64)
    for g in range(groups):
        w = parents[g] - g * beams
        want = scores[g, w].astype(np.float64) + x64[g, w, tokens[g]] - lse[g, w]
        assert np.all(np.abs(got[g] - want) <= 3e-6 + U * np.abs(want))
        # and what comes before another is not behind it by more than both are off
        assert np.all(np.diff(want) <= 6e-6)
