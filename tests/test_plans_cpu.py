"""The plans' arithmetic at the largest sizes that the calls accept, with the functions of
paged.h that the kernels use, built for the host."""
import os
import subprocess
import textwrap

import pytest

import catena_amd as ca
from paged_util import geometry, refused
from test_paged_cpu import INVALID, UNSUPPORTED
from test_requests_cpu import geometry4, release, rope

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "catena-lang_amd", "csrc", "kernels")
HEAD = """
    #include "paged.h"
    #include <cstdio>
    #define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\\n", __LINE__, #x); return 1; } } while (0)
"""


def on_host(tmp_path, body, *args):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(textwrap.dedent(HEAD) + textwrap.dedent(body))
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", KERNELS, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


STRETCHES = """
    #include <cstdlib>
    int main(int n, char** v) {
      // tiles of all units, workgroups that share them out, workgroups of the grid
      for (int i = 1; i + 2 < n; i += 3) {
        const uint64_t tiles = std::strtoull(v[i], 0, 10), blocks = std::strtoull(v[i + 1], 0, 10), grid = std::strtoull(v[i + 2], 0, 10);
        CHECK(tiles < 1ull << 31 && grid >= blocks);
        const uint32_t per = (uint32_t)((tiles + blocks - 1) / blocks);
        uint64_t next = 0;
        for (uint64_t b = 0; b < grid; ++b) {
          const Stretch s = stretch_of((uint32_t)tiles, per, (uint32_t)blocks, (uint32_t)b);
          CHECK(s.beg <= s.end && s.end <= tiles);
          if (s.beg == s.end) continue;
          CHECK(b < blocks);  // who stores parts has a place for them
          CHECK(s.beg == next && s.end - s.beg <= per);
          next = s.end;
        }
        CHECK(next == tiles);
      }
      std::puts("ok");
      return 0;
    }
"""


def test_every_tile_of_a_line_has_one_workgroup(tmp_path):
    """Attention over 4 bits starts a workgroup a unit also where units are cut: those behind
    the plan's have no tile, whatever 32 bits make of their place."""
    args = []
    # rows x slots of caches of so many kv heads and columns, and a row's slots in use (None: all)
    for rows, kvh, dim, slots, used in ((16384, 32, 64, 6656, None), (8192, 64, 64, 7168, None), (140000, 8, 128, 8192, 1024),
                                        (1, 1, 128, 1 << 20, None), (64, 8, 128, 8192, None), (3, 2, 64, 16384, 600)):
        parts, nbytes = ca.attn_paged_q4_plan(geometry4(rows=rows, kv_heads=kvh, head_dim=dim, max_pages=slots // 16, page_size=16), kvh)
        assert parts > 0 and nbytes >= 2 * parts * (dim + 2) * 4
        tiles = rows * kvh * -(-(used or slots) // 512)
        for blocks in {parts, min(parts, 512), min(parts, 256)}:
            args += [tiles, blocks, max(rows * kvh, parts)]
    args += [2 ** 31 - 1, 512, 512, 2 ** 31 - 1, 256, 512, 2 ** 31 - 1, 768, (1 << 24) - 1, 5, 3, 700, 1, 1, 1]
    on_host(tmp_path, STRETCHES, *args)


PARTS = """
    #include <algorithm>
    #include <random>
    #include <vector>
    struct Units {
      uint32_t cost;
      bool narrow;
      uint64_t n;
    };
    // parts of all kv heads of all units, at the places that the workspace has
    bool fits(const std::vector<Units>& units, uint64_t kv_heads) {
      uint64_t work = 0, places = 0, cut = 0;
      for (const Units& u : units) work += u.n * u.cost;
      const PromptCut c = prompt_cut(work * kv_heads);
      for (const Units& u : units) {
        const uint64_t parts = prompt_parts(c, u.cost, u.narrow);
        if (parts < 1 || parts > std::max(1u, u.cost)) return false;
        if (parts > 1) places += u.n * parts * prompt_places(u.narrow), cut += u.n;
      }
      return places * kv_heads <= kPromptParts && cut <= std::max<uint64_t>(1, kPromptParts / 2 / kv_heads);
    }
    int main() {
      std::mt19937_64 r(1);
      auto log_to = [&](double most) { return (uint64_t)std::exp(std::uniform_real_distribution<double>(0, std::log(most))(r)); };
      uint64_t most_places = 0;
      for (int i = 0; i < 300000; ++i) {
        const uint64_t kv = log_to(512);
        std::vector<Units> u;
        for (int kinds = 1 + i % 5; kinds > 0; --kinds) u.push_back({(uint32_t)log_to(1 << 26), r() % 2 == 0, log_to(i % 3 ? 400 : 1 << 23)});
        if (i % 2) {  // costs that are just above what is not cut
          uint64_t work = 0;
          for (const Units& x : u) work += x.n * x.cost;
          const PromptCut c = prompt_cut(work * kv);
          for (Units& x : u)  // (a unit has no more than 2^25 tiles)
            x.cost = (uint32_t)std::min<uint64_t>(1u << 26, (x.narrow ? c.most_narrow : c.most) * (1 + r() % 3) + 1 + r() % 3);
        }
        CHECK(fits(u, kv));
      }
      // one cost for every number of units: the shares that one unit passes by the least
      for (uint64_t n = 1; n <= 2100; ++n)
        for (uint32_t cost = 1; cost < 3000; cost += 1 + cost / 40)
          for (int narrow = 0; narrow < 2; ++narrow) {
            CHECK(fits({{cost, narrow != 0, n}}, 1));
            const PromptCut c = prompt_cut(n * cost);
            const uint64_t parts = prompt_parts(c, cost, narrow != 0);
            if (parts > 1) most_places = std::max(most_places, n * parts * prompt_places(narrow != 0));
          }
      CHECK(most_places > kPromptParts / 2);  // (so the bound is near)
      CHECK(fits({{1u << 26, false, 1}}, 65535) && fits({{1u << 26, true, 1u << 23}}, 1));
      std::puts("ok");
      return 0;
    }
"""


def test_parts_of_prompts_have_their_places(tmp_path):
    on_host(tmp_path, "#include <cmath>\n" + textwrap.dedent(PARTS))


@pytest.mark.parametrize("kv", [geometry(kv_heads=1), geometry4(kv_heads=1)])
def test_rotation_counts_in_32_bits(kv):
    """Threads go through a token's (heads + 2) * 8 runs of 16 values 256 apart: the number that ends
    the walk may not lie within 256 of 2^32, where the walk would begin again."""
    most = (2 ** 32 - 1 - 256) // 8 - 2
    assert (most + 2) * 8 + 256 < 2 ** 32
    for heads in (most + 1, 2 ** 29 - 3, 2 ** 32 - 1):
        refused(UNSUPPORTED, rope, kv, heads=heads)
    rope(kv, heads=most, tokens=0)


def test_release_counts_pages_in_32_bits():
    """A table of 2^32 entries or more could give back more pages than its sums hold, and entries
    behind them would stay."""
    for rows, pages in ((1 << 20, 1 << 12), (1 << 12, 1 << 20), (1 << 31, 16)):
        refused(UNSUPPORTED, release, geometry(rows=rows, max_pages=pages))
    refused(INVALID, release, geometry(rows=1 << 20, max_pages=(1 << 12) - 1), held=0)  # not for its size


def _prompt_bytes(rows, tokens, heads, kvh, dim, slots):
    """What prompt attention's list and parts take, in whole numbers of any size; None: refused."""
    group = heads // kvh
    units = tokens * group // 256 + min(rows, tokens)  # 256 query rows each, a row's last one any number
    if tokens * group > 2 ** 31 - 1 or units * kvh > (2 ** 32 - 1) // 512:
        return None
    if slots <= 1024 and units <= 256:
        return 0
    places, at_once = 4096, min(64, tokens * group)
    return 128 + 32 * (units + places) + 32 * min(units, max(1, places // 2 // kvh)) + places * at_once * (8 + 4 * dim)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_plans_up_to_the_largest_sizes(dim):
    sizes = [(1, 2 ** 31 - 1, 1, 1), (1, 2 ** 31, 1, 1), (1, 2 ** 30, 2, 1), (1, 2 ** 30 - 1, 2, 1), (2 ** 31 - 1, 2 ** 23, 1, 1),
             (2 ** 31 - 1, 2 ** 23 - 2 ** 16, 1, 1), (1, 1, 65535, 65535), (128, 256, 65535, 65535), (126, 256, 65535, 65535),
             (8, 2 ** 28 - 1, 64, 8), (1000, 10 ** 6, 128, 8), (5, 3, 7, 7), (300, 300, 16, 8), (1, 12000, 32, 8)]
    for rows, tokens, heads, kvh in sizes:
        for max_pages in (1, 64, 65, 2 ** 27 - 1):
            kv = geometry(rows=rows, kv_heads=kvh, head_dim=dim, max_pages=max_pages, page_size=16)
            want = _prompt_bytes(rows, tokens, heads, kvh, dim, 16 * max_pages)
            if tokens == 2 ** 31 or want is None:
                refused(UNSUPPORTED, ca.attn_prompt_plan, kv, tokens, heads)
            else:
                assert ca.attn_prompt_plan(kv, tokens, heads) == want, (rows, tokens, heads, kvh, max_pages)
        want = _prompt_bytes(rows, tokens, heads, kvh, dim, tokens)
        if tokens == 2 ** 31 or want is None:
            refused(UNSUPPORTED, ca.attn_packed_plan, rows, tokens, heads, kvh, dim)
        else:
            assert ca.attn_packed_plan(rows, tokens, heads, kvh, dim) == want
