"""CPU checks of the cache in pages: what is refused before a device is looked
for, the plans, and the one function that turns a slot into an address, built
for the host and called with page numbers that the pool does not have."""
import os
import subprocess
import textwrap

import pytest

import catena_amd as ca
from paged_util import geometry, refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 16  # a pointer that is never followed
INVALID, UNSUPPORTED = 1, 2
BAD_GEOMETRY = [
    (UNSUPPORTED, dict(page_size=8)), (UNSUPPORTED, dict(page_size=48)), (UNSUPPORTED, dict(page_size=2048)),
    (UNSUPPORTED, dict(page_size=0)), (UNSUPPORTED, dict(head_dim=96)), (UNSUPPORTED, dict(head_dim=0)),
    (INVALID, dict(kv_heads=0)), (INVALID, dict(num_pages=0)), (INVALID, dict(max_pages=0)),
    (UNSUPPORTED, dict(max_pages=1 << 27)), (UNSUPPORTED, dict(kv_heads=1 << 17)),
    (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(table=0)), (INVALID, dict(k=(1 << 20) + 8)),
    (INVALID, dict(v=(1 << 20) + 2)), (INVALID, dict(table=(1 << 20) + 2)),
]


def attn(kv, heads=8, q=P, lens=P, o=P, work=(P, 1 << 40), acc_in=None, acc_out=None):
    ca.attn_paged_bf16(kv, q, lens, o, heads, 1.0, work, True, acc_in, acc_out)


@pytest.mark.parametrize("status,over", BAD_GEOMETRY)
def test_attention_refuses_a_bad_cache(status, over):
    refused(status, attn, geometry(**over))


def test_attention_refuses_bad_arguments():
    kv = geometry()
    for over in (dict(heads=0), dict(heads=6), dict(q=0), dict(lens=0), dict(o=0), dict(q=P + 8), dict(o=P + 4),
                 dict(lens=P + 1), dict(acc_in=P), dict(acc_out=P), dict(acc_in=P + 2, acc_out=P)):
        refused(INVALID, attn, kv, **over)
    need = ca.attn_paged_plan(kv, 8)[1]
    assert need > 0
    for work in (None, (0, need), (P, need - 1), (P + 8, need)):
        refused(INVALID, attn, kv, work=work)
    refused(UNSUPPORTED, attn, geometry(rows=1 << 31, kv_heads=4))


def test_attention_plan():
    kv = geometry(rows=1, max_pages=8192, kv_heads=8)
    splits, nbytes = ca.attn_paged_plan(kv, 32)
    assert splits > 1 and nbytes >= splits * 32 * (128 + 2) * 4
    # the scores of every head and slot beside it, where weights are wanted
    assert ca.attn_paged_plan(kv, 32, True)[1] >= nbytes + 32 * kv.slots * 4
    # many rows: whole, without a workspace
    assert ca.attn_paged_plan(geometry(rows=1024, kv_heads=8), 8) == (1, 0)
    # neither the pointers nor a device matter
    assert ca.attn_paged_plan(geometry(rows=1, max_pages=8192, kv_heads=8, k=0, v=0, table=0), 32) == (splits, nbytes)
    refused(INVALID, ca.attn_paged_plan, kv, 12)
    refused(UNSUPPORTED, ca.attn_paged_plan, geometry(page_size=24), 8)


def test_slot_to_address(tmp_path):
    """paged.h on the host: every place inside the pool, none for a slot past the
    table or a page that is not there, 64-bit offsets."""
    src = tmp_path / "place.cpp"
    src.write_text(textwrap.dedent("""
        #include "paged.h"
        #include <cstdio>
        #include <vector>
        #define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\\n", __LINE__, #x); return 1; } } while (0)
        int main() {
          const uint32_t num = 7, heads = 3, dim = 64, max_pages = 4, rows = 2;
          std::vector<uint32_t> table = {6, 0, 7, 3, 0xFFFFFFFFu, 5, 0x80000000u, 2};
          PagedKv kv{nullptr, nullptr, table.data(), num, 4, rows, max_pages, heads, dim};
          const uint64_t size = (uint64_t)num * heads * 16 * dim;
          CHECK(paged_slots(kv) == 64);
          CHECK(paged_len(kv, 0) == 0 && paged_len(kv, 63) == 63 && paged_len(kv, 0xFFFFFFFFu) == 64);
          for (uint32_t r = 0; r < rows; ++r)
            for (uint32_t h = 0; h < heads; ++h)
              for (uint32_t s = 0; s < 80; ++s) {
                uint64_t at = ~0ull;
                const bool here = paged_place(kv, r, h, s, &at);
                const bool want = s < 64 && table[r * max_pages + s / 16] < num;
                CHECK(here == want);
                if (here) CHECK(at + dim <= size);
                if (here) CHECK(at == (((uint64_t)table[r * max_pages + s / 16] * heads + h) * 16 + s % 16) * dim);
                if (!here) CHECK(at == ~0ull);
              }
          PagedKv big{nullptr, nullptr, nullptr, 1u << 20, 10, 1, 1, 64, 128};
          CHECK(paged_offset(big, (1u << 20) - 1, 63, 1023) == ((1ull << 20) * 64 * 1024 - 1) * 128);
          std::puts("ok");
          return 0;
        }
    """))
    exe = tmp_path / "place"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "catena-lang_amd", "csrc", "kernels"),
                    str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
