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
    long = geometry(rows=1, max_pages=8192)
    need = ca.attn_paged_plan(long, 8)[1]
    assert need > 0
    for work in (None, (0, need), (P, need - 1), (P + 8, need)):
        refused(INVALID, attn, long, work=work)
    refused(UNSUPPORTED, attn, geometry(rows=1 << 31, kv_heads=4))
    refused(UNSUPPORTED, attn, geometry(rows=1 << 16, kv_heads=64, max_pages=1 << 14), heads=64)
    # more slots than the strips of weights in a grid cover; without weights there are none
    long = geometry(rows=1, kv_heads=1, page_size=1024, max_pages=1 << 16)
    assert ca.attn_paged_plan(long, 1)[0] > 0
    refused(UNSUPPORTED, ca.attn_paged_plan, long, 1, True)
    refused(UNSUPPORTED, attn, long, heads=1, acc_in=P, acc_out=P)
    refused(UNSUPPORTED, ca.attn_paged_plan, geometry(rows=1, kv_heads=1), 1 << 14)  # heads of one kv head


def test_attention_plan():
    kv = geometry(rows=1, max_pages=8192, kv_heads=8)
    parts, nbytes = ca.attn_paged_plan(kv, 32)
    assert parts > 1 and nbytes >= parts * 2 * 4 * (128 + 2) * 4
    # the scores of every head and slot beside it, where weights are wanted
    assert ca.attn_paged_plan(kv, 32, True)[1] >= nbytes + 32 * kv.slots * 4
    # short rows: whole, without a workspace but for the scores
    short = geometry(rows=1024, kv_heads=8)
    assert ca.attn_paged_plan(short, 8) == (0, 0)
    assert ca.attn_paged_plan(short, 8, True)[0] == 0 and ca.attn_paged_plan(short, 8, True)[1] >= 8 * 1024 * short.slots * 4
    # neither the pointers nor a device matter
    assert ca.attn_paged_plan(geometry(rows=1, max_pages=8192, kv_heads=8, k=0, v=0, table=0), 32) == (parts, nbytes)
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


def append(kv, qkv=P, tab=P, positions=64, lens=P, seen=None, q=P, tq=1, heads=8, acc=None, slot_pos=None):
    ca.rope_qkv_paged_bf16(kv, qkv, tab, positions, lens, seen, q, tq, heads, acc, slot_pos)


def evict(kv, lens=P, seen=P, acc=P, pos=P, lens_out=2 * P, acc_out=P, pos_out=P, budget=8, recent=2, work=(P, 1 << 40)):
    ca.kv_evict_paged_bf16(kv, lens, seen, acc, pos, lens_out, acc_out, pos_out, budget, recent, work)


def reorder(kv, pools=(P, P), lens=P, parents=P, spare=P, table_out=P, lens_out=2 * P, spare_out=2 * P):
    ca.beam_reorder_paged_bf16(kv, list(pools), lens, parents, spare, table_out, lens_out, spare_out)


@pytest.mark.parametrize("call", [append, evict, reorder])
@pytest.mark.parametrize("status,over", BAD_GEOMETRY)
def test_upkeep_refuses_a_bad_cache(call, status, over):
    if call is reorder and ("k" in over or "v" in over):
        return  # reads the sizes and the table alone
    refused(status, call, geometry(**over))


def test_append_refuses_bad_arguments():
    kv = geometry()
    for over in (dict(heads=0), dict(heads=6), dict(qkv=0), dict(tab=0), dict(lens=0), dict(q=0), dict(positions=0),
                 dict(qkv=P + 4), dict(tab=P + 8), dict(q=P + 2), dict(lens=P + 2), dict(seen=P + 1), dict(acc=P),
                 dict(slot_pos=P), dict(acc=P + 2, slot_pos=P), dict(acc=P, slot_pos=P + 2)):
        refused(INVALID, append, kv, **over)
    for rows, tq in ((1 << 20, 1 << 12), (1 << 12, 1 << 12), (1 << 24, 1)):
        refused(UNSUPPORTED, append, geometry(rows=rows), tq=tq)


def test_evict_refuses_bad_arguments():
    kv = geometry()
    need = ca.kv_evict_paged_plan(kv, 8)
    assert need == 16 * 4 * (1 + 2 * 8)
    for name in ("lens", "seen", "acc", "pos", "lens_out", "acc_out", "pos_out"):
        refused(INVALID, evict, kv, **{name: 0})
        refused(INVALID, evict, kv, **{name: P + 2})
    for name in ("acc", "pos", "acc_out", "pos_out"):
        refused(INVALID, evict, kv, **{name: P + 8})
    refused(INVALID, evict, kv, seen=2 * P)  # the new lengths' place
    for rows, pages in ((1 << 22, 16), (1 << 20, 80)):  # more workgroups than a grid takes
        refused(UNSUPPORTED, evict, geometry(rows=rows, max_pages=pages))
        refused(UNSUPPORTED, ca.kv_evict_paged_plan, geometry(rows=rows, max_pages=pages), 8)
    for over in (dict(budget=0), dict(lens_out=P), dict(work=None), dict(work=(0, need)), dict(work=(P, need - 1)), dict(work=(P + 4, need))):
        refused(INVALID, evict, kv, **over)
    refused(INVALID, ca.kv_evict_paged_plan, kv, 0)
    refused(UNSUPPORTED, ca.kv_evict_paged_plan, geometry(max_pages=1 << 24), 1 << 26)
    # a budget of the whole table needs the counts alone
    assert ca.kv_evict_paged_plan(kv, 1 << 20) == 16 * 4


def test_reorder_refuses_bad_arguments():
    kv = geometry()
    for name in ("lens", "parents", "spare", "table_out", "lens_out", "spare_out"):
        refused(INVALID, reorder, kv, **{name: 0})
        refused(INVALID, reorder, kv, **{name: P + 1})
    refused(UNSUPPORTED, reorder, geometry(rows=1 << 24))
    for over in (dict(pools=(P, 0)), dict(pools=(P, P + 8)), dict(table_out=1 << 22), dict(lens_out=P), dict(spare_out=P)):
        refused(INVALID, reorder, kv, **over)


def test_beam_selection_refuses_bad_arguments():
    good = dict(logits=P, scores=P, done=P, tokens=P, parents=P, scores_out=P, done_out=P, groups=2, beams=4, vocab=100, eos=2,
                workspace=(P, 1 << 30))
    need = ca.beam_select_plan(2, 4, 100)
    assert need >= 8 * (4 * 8 + 8 + 4)
    for name in ("logits", "scores", "tokens", "parents", "scores_out"):
        refused(INVALID, ca.beam_select_f32, **{**good, name: 0})
    for name in ("logits", "scores", "done", "tokens", "parents", "scores_out", "done_out"):
        refused(INVALID, ca.beam_select_f32, **{**good, name: P + 1})
    for over in (dict(beams=0), dict(vocab=0), dict(eos=100), dict(eos=ca.BEAM_NO_EOS), dict(workspace=None),
                 dict(workspace=(P, need - 1)), dict(workspace=(P + 8, need)), dict(workspace=(0, need))):
        refused(INVALID, ca.beam_select_f32, **{**good, **over})
    for over in (dict(beams=33), dict(vocab=(1 << 26) + 1), dict(groups=1 << 29), dict(groups=1 << 22)):
        refused(UNSUPPORTED, ca.beam_select_f32, **{**good, **over})
        refused(UNSUPPORTED, ca.beam_select_plan, *({**good, **over}[n] for n in ("groups", "beams", "vocab")))
