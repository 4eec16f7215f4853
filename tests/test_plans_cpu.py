"""The plans' arithmetic at the largest sizes that the calls accept, with the functions of
paged.h that the kernels use, built for the host."""
import os
import subprocess
import textwrap

import catena_amd as ca
from test_requests_cpu import geometry4

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
