"""CPU checks of the calls for requests of different lengths: what is refused before a
device is looked for, the plans, the scaled frequencies."""
import numpy as np
import pytest

import catena_amd as ca
from paged_util import geometry, refused
from test_paged_cpu import BAD_GEOMETRY, INVALID, UNSUPPORTED, P

SIZES = [(s, o) for s, o in BAD_GEOMETRY if not set(o) & {"k", "v", "table"}]


def geometry4(**over) -> ca.PagedKV4:
    kv = ca.PagedKV4(1 << 20, 1 << 21, 1 << 23, 1 << 24, 1 << 22, 64, 16, 4, 16, 4, 128)
    for name, value in over.items():
        setattr(kv, name, value)
    return kv


# pointers that are never followed, each its own
ADMIT = dict(table=P, lens=P + 4, held=P + 8, want=P + 12, free_pages=P + 16, free_count=P + 20, lens_out=P + 24, held_out=P + 28,
             starts=P + 32, free_count_out=P + 36, token_pos=P + 40, slot_map=P + 48, max_tokens=64)
RELEASE = dict(table=P, lens=P + 4, held=P + 8, finished=P + 12, free_pages=P + 16, free_count=P + 20, lens_out=P + 24,
               held_out=P + 28, free_count_out=P + 32)


def admit(kv, **over):
    ca.kv_admit_paged(kv, **{**ADMIT, **over})


def release(kv, **over):
    ca.kv_release_paged(kv, **{**RELEASE, **over})


def rope(kv, qkv=P, wide=True, tab=P, positions=8, rot=64, pos=P, slots=P, q=P, tokens=3, heads=8, k_out=None, v_out=None):
    call = ca.rope_packed_q4 if isinstance(kv, ca.PagedKV4) else ca.rope_packed_bf16
    call(kv, qkv, wide, tab, positions, rot, False, pos, slots, q, tokens, heads, k_out, v_out)


def prompt(kv, q=P, starts=P, lens=P, o=P, tokens=32, heads=8, work=(P, 1 << 40)):
    ca.attn_prompt_bf16(kv, q, starts, lens, o, tokens, heads, 1.0, work)


def packed(q=P, k=P, v=P, starts=P, o=P, rows=4, tokens=32, heads=8, kv_heads=4, dim=128, stride=0, work=(P, 1 << 40)):
    ca.attn_packed_bf16(q, k, v, starts, o, rows, tokens, heads, kv_heads, dim, 1.0, work, stride)


def q4(kv, q=P, lens=P, o=P, heads=8, work=(P, 1 << 40)):
    ca.attn_paged_q4(kv, q, lens, o, heads, 1.0, work)


@pytest.mark.parametrize("status,over", SIZES)
def test_bad_sizes_are_refused(status, over):
    for call in (admit, release, rope, prompt):
        refused(status, call, geometry(**over))
    for call in (rope, q4):
        refused(status, call, geometry4(**over))


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "table"])
def test_missing_pools_are_refused(name):
    for value in (0, (1 << 20) + 2):
        refused(INVALID, q4, geometry4(**{name: value}))
        if name in ("k", "v", "table"):
            refused(INVALID, prompt, geometry(**{name: value}))
        if name != "table":
            refused(INVALID, rope, geometry4(**{name: value}))
        if name in ("k", "v"):
            refused(INVALID, rope, geometry(**{name: value}))


def test_admission_refuses_bad_arguments():
    kv = geometry()
    for name in ADMIT:
        if name == "max_tokens":
            continue
        refused(INVALID, admit, kv, **{name: 0})
        refused(INVALID, admit, kv, **{name: ADMIT[name] + 2})
    for name in ("lens", "held", "want", "free_pages", "free_count"):
        for out in ("table", "lens_out", "held_out", "starts", "free_count_out", "token_pos"):
            refused(INVALID, admit, kv, **{out: ADMIT[name]})
    refused(INVALID, admit, kv, seen=P + 64)
    refused(INVALID, admit, kv, seen_out=P + 64)
    refused(INVALID, admit, kv, seen=P + 64, seen_out=P + 64)
    refused(INVALID, admit, kv, slot_map=P + 4)
    refused(UNSUPPORTED, admit, kv, max_tokens=1 << 31)
    refused(UNSUPPORTED, admit, geometry(rows=1 << 31))
    for name in RELEASE:
        refused(INVALID, release, kv, **{name: 0})
        refused(INVALID, release, kv, **{name: RELEASE[name] + 1})
    for name in ("lens", "held", "finished", "free_count"):
        for out in ("table", "lens_out", "held_out", "free_pages", "free_count_out"):
            refused(INVALID, release, kv, **{out: RELEASE[name]})
    refused(UNSUPPORTED, release, geometry(rows=1 << 31))


@pytest.mark.parametrize("kv", [geometry(), geometry4()])
def test_rotation_refuses_bad_arguments(kv):
    for over in (dict(qkv=0), dict(tab=0), dict(pos=0), dict(q=0), dict(qkv=P + 8), dict(tab=P + 8), dict(q=P + 8), dict(pos=P + 2),
                 dict(slots=P + 4), dict(positions=0), dict(heads=0), dict(heads=6), dict(k_out=P), dict(v_out=P),
                 dict(k_out=P + 8, v_out=P), dict(k_out=P, v_out=P + 4)):
        refused(INVALID, rope, kv, **over)
    for rot in (0, 8, 24, 130, 144):
        refused(UNSUPPORTED, rope, kv, rot=rot)
    refused(UNSUPPORTED, rope, kv, tokens=1 << 32)
    rope(kv, tokens=0)  # nothing to do, and no device to do it


def test_rotation_in_4_bits_refuses_more_heads_than_its_workgroup_holds():
    refused(UNSUPPORTED, rope, geometry4(kv_heads=129), heads=129)


def test_prompt_attention_refuses_bad_arguments():
    kv = geometry()
    for over in (dict(q=0), dict(starts=0), dict(lens=0), dict(o=0), dict(q=P + 8), dict(o=P + 8), dict(starts=P + 2), dict(lens=P + 1),
                 dict(heads=0), dict(heads=6)):
        refused(INVALID, prompt, kv, **over)
    refused(UNSUPPORTED, prompt, kv, tokens=1 << 31)
    refused(UNSUPPORTED, prompt, kv, tokens=1 << 30, heads=64)
    for over in (dict(q=0), dict(k=0), dict(v=0), dict(starts=0), dict(o=0), dict(q=P + 8), dict(k=P + 8), dict(v=P + 8), dict(o=P + 8),
                 dict(starts=P + 2), dict(heads=0), dict(heads=6), dict(kv_heads=0), dict(stride=504), dict(stride=516)):
        refused(INVALID, packed, **over)
    for over in (dict(dim=96), dict(dim=0), dict(tokens=1 << 31), dict(stride=(1 << 25) + 8), dict(kv_heads=1 << 16, heads=1 << 16)):
        refused(UNSUPPORTED, packed, **over)
    for call in (lambda: prompt(kv, tokens=0), lambda: prompt(geometry(rows=0)), lambda: packed(rows=0), lambda: packed(tokens=0)):
        call()  # nothing to do
    need = ca.attn_prompt_plan(kv, 32, 8)
    assert need == ca.attn_prompt_plan(geometry(k=0, v=0, table=0), 32, 8)
    if need:
        for work in (None, (0, need), (P, need - 1), (P + 8, need)):
            refused(INVALID, prompt, kv, work=work)
    need = ca.attn_packed_plan(4, 32, 8, 4, 128)
    if need:
        for work in (None, (0, need), (P, need - 1), (P + 8, need)):
            refused(INVALID, packed, work=work)


def test_attention_over_4_bits_refuses_bad_arguments():
    kv = geometry4()
    for over in (dict(q=0), dict(lens=0), dict(o=0), dict(q=P + 8), dict(o=P + 4), dict(lens=P + 1), dict(heads=0), dict(heads=6)):
        refused(INVALID, q4, kv, **over)
    long = geometry4(rows=1, max_pages=8192)
    parts, need = ca.attn_paged_q4_plan(long, 8)
    assert parts > 1 and need >= parts * 2 * 2 * (128 + 2) * 4
    for work in (None, (0, need), (P, need - 1), (P + 8, need)):
        refused(INVALID, q4, long, work=work)
    assert ca.attn_paged_q4_plan(geometry4(rows=1, max_pages=8192, k=0, v=0, k_scale=0, v_scale=0, table=0), 8) == (parts, need)
    refused(INVALID, ca.attn_paged_q4_plan, kv, 6)
    refused(UNSUPPORTED, q4, geometry4(rows=1 << 31, kv_heads=4))


@pytest.mark.parametrize("rot", [2, 16, 64, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_scaled_frequencies(rot, base):
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    eps = 2.0 ** -45  # a few roundings of a power in double
    plain = ca.rope_inv_freq_scaled(rot, base)
    assert np.all(np.abs(plain - f) <= eps * f)
    assert np.all(np.abs(ca.rope_inv_freq_scaled(rot, base, ca.ROPE_LINEAR, 4.0) - f / 4) <= eps * f)
    if rot > 2:
        raised = ca.rope_inv_freq_scaled(rot, base, ca.ROPE_BASE, 8.0)
        # the highest frequency stays, the lowest is an eighth
        assert raised[0] == 1.0 and abs(raised[-1] - f[-1] / 8) <= 64 * eps * f[-1]
    parts = ca.rope_inv_freq_scaled(rot, base, ca.ROPE_PARTS, 8.0, 8192.0, 1.0, 4.0)
    turns = 8192.0 * f / (2 * np.pi)
    keep = np.clip((turns - 1.0) / 3.0, 0, 1)
    assert np.all(np.abs(parts - (keep * f + (1 - keep) * f / 8)) <= 8 * eps * f)
    assert np.all(parts[turns >= 4] == plain[turns >= 4])


def test_scaled_frequencies_refuse_bad_arguments():
    for args in ((0, 1e4), (15, 1e4), (64, 0.0), (64, -1.0), (64, float("inf")), (64, float("nan")), (64, 1e4, ca.ROPE_LINEAR, 0.0),
                 (64, 1e4, ca.ROPE_LINEAR, float("nan")), (2, 1e4, ca.ROPE_BASE, 2.0), (64, 1e4, ca.ROPE_PARTS, 2.0, 0.0, 1.0, 4.0),
                 (64, 1e4, ca.ROPE_PARTS, 2.0, 8192.0, 4.0, 4.0), (64, 1e4, ca.ROPE_PARTS, 2.0, 8192.0, -1.0, 4.0)):
        refused(INVALID, ca.rope_inv_freq_scaled, *args)
    refused(UNSUPPORTED, ca.rope_inv_freq_scaled, 64, 1e4, 4, 2.0)
    refused(INVALID, ca.rope_table_scaled_f32, 0, P, 0, 4, 64)
    refused(INVALID, ca.rope_table_scaled_f32, P, 0, 0, 4, 64)
    refused(INVALID, ca.rope_table_scaled_f32, P + 4, P, 0, 4, 64)
    refused(INVALID, ca.rope_table_scaled_f32, P, P, 0, 4, 63)
    refused(UNSUPPORTED, ca.rope_table_scaled_f32, P, P, 0xFFFFFFFF, 4, 64)
    ca.rope_table_scaled_f32(P, P, 0, 0, 64)
