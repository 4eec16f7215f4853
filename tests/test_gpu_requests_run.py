"""Requests of different lengths served step by step, as a program would: pages are
given out, tokens turned and stored, attention over what the pages hold, pages given
back. State against the plain form, outputs against 64 bits on the values that the cache
holds; single steps, and a whole step captured once and replayed."""
import numpy as np
import pytest

import catena_amd as ca
import requests_util as plain
from gpu_util import captured, say
from paged_util import UB, attention, bf16, f64
from requests_util import prompt_slack

pytestmark = pytest.mark.gpu

ROWS, HEADS, KVH, PAGE, MAX_PAGES, POSITIONS = 6, 8, 2, 16, 10, 160
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module", autouse=True)
def _init():
    say("init device 0")
    ca.init(0)


class Server:
    """The program's buffers, and the same state on the host: table, lengths, pages held,
    the stack of free pages, and every row's keys and values."""

    def __init__(self, rng, dim, rot, four_bits, num_pages, max_tokens):
        self.rng, self.dim, self.rot, self.four_bits, self.max_tokens = rng, dim, rot, four_bits, max_tokens
        up = ca.Buffer.from_array
        self.table = np.full((ROWS, MAX_PAGES), NONE, np.uint32)
        self.lens, self.held = np.zeros(ROWS, np.int64), np.zeros(ROWS, np.int64)
        self.free = rng.permutation(num_pages).astype(np.uint32)
        self.count = num_pages
        self.keys, self.values = ([np.zeros((KVH, 0, dim)) for _ in range(ROWS)] for _ in range(2))
        self.b = {"table": up(self.table), "free": up(self.free), "want": up(np.zeros(ROWS, np.uint32)), "finished": up(np.zeros(ROWS, np.uint32)),
                  "starts": up(np.zeros(ROWS + 1, np.uint32)), "pos": up(np.zeros(max_tokens, np.uint32)), "map": up(np.zeros(max_tokens, np.uint64)),
                  "qkv": up(np.zeros((max_tokens, HEADS + 2 * KVH, dim), np.float32))}
        for name, n in (("lens", ROWS), ("held", ROWS), ("count", 1)):
            for i in range(2):
                self.b[f"{name}{i}"] = up(np.full(n, num_pages if name == "count" else 0, np.uint32))
        for name, heads in (("q", HEADS), ("o", HEADS), ("o1", HEADS), ("k", KVH), ("v", KVH)):
            self.b[name] = up(np.full((max_tokens, heads, dim), 0x7FC0, np.uint16))
        self.tab = ca.Buffer(POSITIONS * (rot // 2) * 8)
        freq = ca.rope_inv_freq_scaled(rot, 10000.0, ca.ROPE_PARTS, 4.0, 64, 1.0, 8.0)
        ca.rope_table_scaled_f32(up(freq), self.tab, 0, POSITIONS, rot, 1.1)
        shape = (num_pages, KVH, PAGE, dim)
        if four_bits:
            pools = [np.full((num_pages, KVH, PAGE, dim // 2), 0x77, np.uint8), np.full((num_pages, KVH, dim // 2, PAGE), 0x77, np.uint8),
                     np.full((num_pages, KVH, dim // 32, PAGE), 255, np.uint8), np.full((num_pages, KVH, PAGE), 0x7FC0, np.uint16)]
            self.pools = [up(p) for p in pools]
            self.kv = ca.PagedKV4(*[p.ptr for p in self.pools], self.b["table"].ptr, num_pages, PAGE, ROWS, MAX_PAGES, KVH, dim)
            work = [ca.attn_packed_plan(ROWS, max_tokens, HEADS, KVH, dim), ca.attn_paged_q4_plan(self.kv, HEADS)[1]]
        else:
            self.pools = [up(np.full(shape, 0x7FC0, np.uint16)) for _ in range(2)]
            self.kv = ca.PagedKV(self.pools[0].ptr, self.pools[1].ptr, self.b["table"].ptr, num_pages, PAGE, ROWS, MAX_PAGES, KVH, dim)
            work = [ca.attn_prompt_plan(self.kv, max_tokens, HEADS), ca.attn_paged_plan(self.kv, HEADS)[1]]
        self.sizes = ca.PagedKV(0, 0, self.b["table"].ptr, num_pages, PAGE, ROWS, MAX_PAGES, KVH, dim)
        self.work = ca.Buffer(max(16, *work))  # one for all of them
        self.scale = dim ** -0.5

    def admit(self):
        b = self.b
        ca.kv_admit_paged(self.sizes, b["table"], b["lens0"], b["held0"], b["want"], b["free"], b["count0"], b["lens1"], b["held1"], b["starts"],
                          b["count1"], b["pos"], b["map"], self.max_tokens)

    def turn(self):
        b = self.b
        call = ca.rope_packed_q4 if self.four_bits else ca.rope_packed_bf16
        call(self.kv, b["qkv"], True, self.tab, POSITIONS, self.rot, False, b["pos"], b["map"], b["q"], self.max_tokens, HEADS,
             *((b["k"], b["v"]) if self.four_bits else ()))

    def attend(self, kind):
        """prompt: all new tokens over the pages; packed: over the step's own keys; one: a token a row."""
        b = self.b
        if kind == "prompt":
            ca.attn_prompt_bf16(self.kv, b["q"], b["starts"], b["lens1"], b["o"], self.max_tokens, HEADS, self.scale, self.work)
        elif kind == "packed":
            ca.attn_packed_bf16(b["q"], b["k"], b["v"], b["starts"], b["o"], ROWS, self.max_tokens, HEADS, KVH, self.dim, self.scale, self.work)
        elif self.four_bits:
            ca.attn_paged_q4(self.kv, b["q"], b["lens1"], b["o1"], HEADS, self.scale, self.work)
        else:
            ca.attn_paged_bf16(self.kv, b["q"], b["lens1"], b["o1"], HEADS, self.scale, workspace=self.work)

    def release(self):
        b = self.b
        ca.kv_release_paged(self.sizes, b["table"], b["lens1"], b["held1"], b["finished"], b["free"], b["count1"], b["lens0"], b["held0"], b["count0"])

    def feed(self, want, finished):
        """What the step works on, to the device; what has to come out, on the host."""
        self.want, self.finished = np.array(want, np.uint32), np.array(finished, np.uint32)
        x = self.rng.standard_normal((self.max_tokens, HEADS + 2 * KVH, self.dim)).astype(np.float32)
        self.b["want"].write(self.want)
        self.b["finished"].write(self.finished)
        self.b["qkv"].write(x)
        self.table, lens, self.held, self.starts, self.count, pos, self.map, _ = plain.admit(
            self.table, self.lens, self.held, self.want, self.free, self.count, PAGE, self.max_tokens)
        tab = self.tab.read(np.float32, (POSITIONS, self.rot // 2, 2))[pos]
        self.q = plain.turn(x[:, :HEADS], tab, self.rot, False)
        k, v = plain.turn(x[:, HEADS:HEADS + KVH], tab, self.rot, False), bf16(x[:, HEADS + KVH:])
        k, v = (plain.quantise_k(k)[2], plain.quantise_v(v)[2]) if self.four_bits else (f64(k), f64(v))
        self.copies = [f64(bf16(x)).transpose(1, 0, 2) for x in (k, v)]  # (a code times a scale of 8 bits has up to 10)
        for r in range(ROWS):
            mine = slice(self.starts[r], self.starts[r + 1])
            self.keys[r] = np.concatenate([self.keys[r], k[mine].transpose(1, 0, 2)], 1)
            self.values[r] = np.concatenate([self.values[r], v[mine].transpose(1, 0, 2)], 1)
        self.lens = lens

    def check(self, kinds):
        """prompt, packed: p is rounded to bf16, p_i (1 + d_i) with |d_i| <= 2^-8, in the sum over v and in that of p,
        so that o is off by sum p_i d_i (v_i - o), at most 2^-8 (sum p |v| + |o|); one: p in two terms, 2^-16."""
        b, n = self.b, int(self.starts[-1])
        assert np.array_equal(b["starts"].read(np.uint32, (ROWS + 1,)), self.starts)
        assert np.array_equal(b["map"].read(np.uint64, (self.max_tokens,)), self.map)
        assert np.array_equal(b["lens1"].read(np.uint32, (ROWS,)), self.lens) and np.array_equal(b["held1"].read(np.uint32, (ROWS,)), self.held)
        assert b["count1"].read(np.uint32, (1,))[0] == self.count
        assert np.array_equal(b["q"].read(np.uint16, self.q.shape)[:n], self.q[:n])
        group = HEADS // KVH
        for kind in kinds:
            o = b["o1" if kind == "one" else "o"].read(np.uint16, (self.max_tokens, HEADS, self.dim))
            for r in range(ROWS):
                new = int(self.starts[r + 1] - self.starts[r])
                for t in range(new):
                    seen, at = int(self.lens[r]) - new + t + 1, int(self.starts[r]) + t
                    keys, values = (x[r][:, :seen] for x in (self.keys, self.values))
                    if kind == "packed":
                        keys, values = (x[:, self.starts[r]:at + 1] for x in self.copies)
                    for h in range(KVH):
                        mine = slice(h * group, (h + 1) * group)
                        want, _, pv, es = attention(f64(self.q[at, mine]), keys[h], values[h], self.scale)
                        p_bits = 2.0 ** -16 if kind == "one" else UB
                        slack = prompt_slack(es, seen) * pv + p_bits * (1 + 2 * p_bits) * (pv + np.abs(want))
                        over = np.abs(f64(o[at, mine]) - want) - slack - UB * (np.abs(want) + slack)
                        assert over.max() <= 0, (kind, r, t, h)

    def ended(self):
        """The rows that have ended, on the host: their pages on the stack, in order."""
        for r in np.flatnonzero(self.finished):
            pages = self.table[r, :self.held[r]].copy()
            self.free[self.count:self.count + len(pages)] = pages
            self.count += len(pages)
            self.table[r, :self.held[r]] = NONE
            self.held[r] = self.lens[r] = 0
            self.keys[r], self.values[r] = (np.zeros((KVH, 0, self.dim)) for _ in range(2))

    def check_ended(self):
        self.ended()
        b = self.b
        assert np.array_equal(b["table"].read(np.uint32, self.table.shape), self.table)
        assert np.array_equal(b["lens0"].read(np.uint32, (ROWS,)), self.lens) and np.array_equal(b["held0"].read(np.uint32, (ROWS,)), self.held)
        assert b["count0"].read(np.uint32, (1,))[0] == self.count
        assert np.array_equal(b["free"].read(np.uint32, self.free.shape)[:self.count], self.free[:self.count])


# new tokens a row asks for, rows that end with the step: prompts beside single tokens, a row that waits for pages or for
# a place in the list, one that asks for more than its table holds, rows that come back
STEPS = [([40, 3, 0, 0, 17, 1], []), ([1, 1, 70, 0, 1, 1], []), ([1, 1, 1, 90, 1, 1], [1]), ([1, 33, 1, 60, 1, 30], [2, 4]),
         ([1, 1, 64, 1, 20, 1], [0]), ([200, 1, 1, 1, 1, 1], [0, 1, 2, 3, 4, 5]), ([0, 0, 0, 0, 0, 0], []), ([16, 15, 17, 1, 32, 31], []),
         ([1, 1, 1, 1, 1, 1], [])]


@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 96)])
@pytest.mark.parametrize("graph", [False, True])
def test_chunks_and_single_tokens(dim, rot, graph):
    say(f"serve {dim} {rot} {graph}")
    x = Server(np.random.default_rng(dim + graph), dim, rot, False, 22, 150)

    def step():
        x.admit()
        x.turn()
        x.attend("prompt")
        x.release()

    run = captured(step) if graph else step
    for want, end in STEPS:
        x.feed(want, [r in end for r in range(ROWS)])
        run()
        x.check(["prompt"])
        x.check_ended()


@pytest.mark.parametrize("four_bits", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_then_single_tokens(dim, four_bits):
    """Both attentions of a token a row where every row has one: the workspace and the pages are the same. Two graphs
    of the step, replayed in turn with eager steps between."""
    say(f"decode {dim} {four_bits}")
    x = Server(np.random.default_rng(dim), dim, dim, four_bits, ROWS * MAX_PAGES, 120)
    first = "packed" if four_bits else "prompt"

    def step(kinds):
        x.admit()
        x.turn()
        for kind in kinds:
            x.attend(kind)
        x.release()

    x.feed([30, 1, 16, 17, 44, 2], [0] * ROWS)
    step([first])
    x.check([first])
    x.check_ended()
    kinds = ["one"] if four_bits else ["one", "prompt"]
    graphs = [captured(lambda: step(kinds)), captured(lambda: step(kinds[::-1]))]
    for i in range(7):
        x.feed([1] * ROWS, [0] * ROWS)
        (graphs[i % 3] if i % 3 < 2 else lambda: step(kinds))()
        x.check(kinds)
        x.check_ended()
