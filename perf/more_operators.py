"""The operators of a step over requests of different lengths, as measurable cases.

Every case is one pass through one operator, on inputs already resident on the
device:

  admit   kv_admit_paged: pages handed out, block table and slot map of a step
  rope    rope_packed_bf16 / rope_packed_q4: rotation of packed tokens, and their
          keys and values written to the slots of a slot map, in bf16 or 4 bits
  prompt  attn_prompt_bf16 / attn_packed_bf16: causal attention of packed
          sequences, over a cache in pages or over packed keys and values
  q4      attn_paged_q4: one new token of every row over a cache held in 4 bits

`own` chooses between the operators' plain form and the framework's calls.
`listed()` names the cases, `draw(rng)` gives more of the same ranges.
"""
import math
import os
import sys

import torch

own = False


def listed():
    return [
        # a decode step of a small batch: one token a request, now and then a new page
        {"name": "admit_step", "op": "admit", "rows": 64, "page": 16, "slots": 4096, "prompts": 0, "most": 1, "tokens": 64, "seen": False},
        # a full batch that takes prompts in: long ones beside requests that go on, some evicted before
        {"name": "admit_prompts", "op": "admit", "rows": 1024, "page": 16, "slots": 16384, "prompts": 64, "most": 2048, "tokens": 131072, "seen": True},
        # a decode step's q, k and v, 8 of the 64 places empty
        {"name": "rope_step", "op": "rope", "rows": 56, "tokens": 64, "most": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "pairs": "half", "page": 16, "slots": 4096, "wide": False, "q4": False, "copies": False},
        # prompts in f32, part of the head rotated, neighbouring pairs
        {"name": "rope_prompts", "op": "rope", "rows": 12, "tokens": 8192, "most": 900, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "pairs": "next", "page": 32, "slots": 2048, "wide": True, "q4": False, "copies": False},
        # prompts into a cache of 4 bits, with the values that it then holds for the prompts' own attention
        {"name": "rope_prompts_q4", "op": "rope", "rows": 12, "tokens": 8192, "most": 900, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "pairs": "half", "page": 32, "slots": 2048, "wide": False, "q4": True, "copies": True},
        # a few short prompts without a cache behind them: latency
        {"name": "prompt_short", "op": "prompt", "rows": 5, "most": 130, "even": False, "singles": 0, "ctx": 0, "heads": 16, "kv_heads": 16, "dim": 64, "page": 0},
        # ragged prompts of up to 4096 tokens
        {"name": "prompt_batch", "op": "prompt", "rows": 8, "most": 4096, "even": False, "singles": 0, "ctx": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # one long prompt
        {"name": "prompt_long", "op": "prompt", "rows": 1, "most": 12000, "even": True, "singles": 0, "ctx": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # chunks of prompts beside single tokens, all of them over what their pages hold already
        {"name": "prompt_mixed", "op": "prompt", "rows": 32, "most": 500, "even": True, "singles": 28, "ctx": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
        # one sequence of a 16-head decoder
        {"name": "q4_one", "op": "q4", "rows": 1, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16, "slots": 640, "ragged": False},
        # a serving batch, grouped heads, lengths from one token to the whole cache
        {"name": "q4_batch", "op": "q4", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "slots": 8192, "ragged": True},
        # one long document
        {"name": "q4_long", "op": "q4", "rows": 1, "heads": 32, "kv_heads": 8, "dim": 64, "page": 64, "slots": 131072, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _slots(rng, lo, hi, page):
    return max(1, -(-_log(rng, lo, hi) // page)) * page


def draw(rng):
    op = rng.choice(["admit", "rope", "rope", "prompt", "prompt", "q4", "q4"])
    page, dim = rng.choice([16, 32, 64, 128]), rng.choice([128, 128, 64])
    if op == "admit":
        rows = _log(rng, 1, 1024)
        prompts = rng.randint(0, min(64, rows))
        slots = _slots(rng, 512, 16384, page)
        return {"op": op, "rows": rows, "page": page, "slots": slots, "prompts": prompts, "most": _log(rng, 1, min(2048, slots)), "tokens": _log(rng, rows, 131072), "seen": rng.random() < 0.5}
    if op == "rope":
        while True:
            kv_heads, group = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 1, 2, 4, 7, 8])
            rows, most = _log(rng, 1, 64), rng.choice([1, _log(rng, 2, 2000)])
            c = {"op": op, "rows": rows, "tokens": rows * most + rng.choice([0, 0, 3]), "most": most, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                 "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "pairs": rng.choice(["half", "next"]), "page": page, "slots": _slots(rng, most, 2 * most + 1000, page),
                 "wide": rng.random() < 0.5, "q4": rng.random() < 0.4, "copies": rng.random() < 0.4}
            if c["heads"] <= 64 and c["tokens"] * (c["heads"] + 2 * kv_heads) * dim <= 8192 * 48 * 128 and rows * c["slots"] * kv_heads * dim <= 12 * 2048 * 8 * 128:
                return c
    if op == "prompt":
        while True:
            kv_heads, group = rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([1, 1, 2, 4, 7, 8, 16])
            rows, most = _log(rng, 1, 32), _log(rng, 1, 12000)
            packed = rng.random() < 0.3
            ctx = 0 if packed or rng.random() < 0.4 else _log(rng, 16, 65536)
            c = {"op": op, "rows": rows, "most": most, "singles": rng.choice([0, 0, rng.randint(0, rows)]), "even": rng.random() < 0.5, "ctx": ctx, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": 0 if packed else page}
            if c["heads"] <= 64 and rows * c["heads"] * most * (most + ctx) <= 32 * 12000 * 12000 and rows * (most + ctx) * kv_heads <= 1 << 21 and rows * c["heads"] * most <= 1 << 20:
                return c
    while True:
        kv_heads, group = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 1, 2, 4, 7, 8, 16, 24])
        c = {"op": op, "rows": _log(rng, 1, 64), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "slots": _slots(rng, 16, 131072, page), "ragged": rng.random() < 0.5}
        if c["heads"] <= 64 and c["rows"] * c["slots"] * kv_heads <= 64 * 8192 * 8 and c["rows"] * c["slots"] * c["heads"] <= 64 * 8192 * 32:
            return c


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _arange(n):
    return torch.arange(n, device="cuda")


def _i32(x):
    return x.to(torch.int32).contiguous()


def _table(g, rows, max_pages, extra=0):
    """A table of every row's own pages in any order, and `extra` pages in none."""
    order = _i32(torch.randperm(rows * max_pages + extra, generator=g, device="cuda"))
    return order[: rows * max_pages].view(rows, max_pages).contiguous(), order[rows * max_pages:].contiguous()


def _least(case):
    return case["most"] - case["most"] // 16 if case.get("even") else case["most"] // 4


def _places(case):
    """Places for the tokens of packed sequences: as many as they may need, whatever they need this time."""
    return (case["rows"] - case["singles"]) * case["most"] + case["singles"]


def _lengths(case, g):
    """New tokens of every row, and how many slots it had before."""
    rows, most = case["rows"], case["most"]
    n = _ints(g, max(1, _least(case)), most + 1, rows)
    n = torch.where(_arange(rows) < rows - case.get("singles", 0), n, torch.ones_like(n))
    return n[torch.randperm(rows, generator=g, device="cuda")], _ints(g, 0, case.get("ctx", 0) + 1, rows)


def _starts(n):
    return torch.cat([torch.zeros_like(n[:1]), n.cumsum(0)])


def _quantised(x):
    """(codes 0 .. 15, block scales, values) of keys x [..., dim] in 4 bits: 32 values share a power of two."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [1/2, 1): the smallest power of two with top <= 6 of them
    e = torch.where(top > 0, (e - 3 + (m > 0.75).to(e.dtype)).clamp(min=-127), -127)
    unit = _pow2(e)
    code = _codes(b, unit)
    return code.flatten(-2), (e + 127).squeeze(-1).to(torch.uint8), (_value(code) * unit).flatten(-2)


def _quantised_v(x):
    """(codes, scale in bf16, values) of values x [..., dim] in 4 bits: one scale for all of them."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    unit = top / torch.full_like(top, 6.0)
    unit = ((unit.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)  # up to bf16
    code = _codes(x, unit)
    return code, unit.squeeze(-1).to(torch.bfloat16), _value(code) * unit


def _pow2(e):
    """2 to whole numbers from -127 on, exactly."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _codes(x, unit):
    """The nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 units, of two the one with an even code; 8 and up below zero."""
    a = x.abs()
    code = (a > 0.25 * unit).int() + (a >= 0.75 * unit) + (a > 1.25 * unit) + (a >= 1.75 * unit) + (a > 2.5 * unit) + (a >= 3.5 * unit) + (a > 5.0 * unit)
    return torch.where(unit > 0, code + 8 * torch.signbit(x), torch.zeros_like(code))


def _value(code):
    m = code & 7
    a = torch.where(m < 5, m * 0.5, torch.where(m == 5, 3.0, torch.where(m == 6, 4.0, 6.0)))
    return torch.where(code >= 8, -a, a)


def _pack(code):
    """Two codes a byte, the first in the lower half."""
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)


def _unpack(byte):
    return torch.stack([byte & 15, byte >> 4], -1).flatten(-2).int()


def _pool4(case, g, pages):
    """Pools of a cache in 4 bits: k [pages][heads][page][dim / 2], its scales [..][dim / 32][page], v [..][dim / 2][page], its scales [..][page]."""
    kvh, page, dim = case["kv_heads"], case["page"], case["dim"]
    spread = _normal(g, kvh, 1, dim, scale=0.7).exp_()  # some channels of the keys are larger
    out = {"k": torch.empty(pages, kvh, page, dim // 2, device="cuda", dtype=torch.uint8), "k_scale": torch.empty(pages, kvh, dim // 32, page, device="cuda", dtype=torch.uint8),
           "v": torch.empty(pages, kvh, dim // 2, page, device="cuda", dtype=torch.uint8), "v_scale": torch.empty(pages, kvh, page, device="cuda", dtype=torch.bfloat16)}
    step = max(1, (1 << 27) // (kvh * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        code, scale, _ = _quantised(_normal(g, n, kvh, page, dim) * spread)
        out["k"][at:at + n], out["k_scale"][at:at + n] = _pack(code), scale.transpose(-1, -2)
        code, scale, _ = _quantised_v(_normal(g, n, kvh, page, dim, dtype=torch.bfloat16))
        out["v"][at:at + n], out["v_scale"][at:at + n] = _pack(code).transpose(-1, -2), scale
    return out


def _held4(x):
    """The values that the pools of 4 bits stand for, [pages][heads][page][dim] each."""
    k = _value(_unpack(x["k"])).unflatten(-1, (-1, 32)) * _pow2(x["k_scale"].int() - 127).transpose(-1, -2)[..., None]
    v = _value(_unpack(x["v"].transpose(-1, -2))) * x["v_scale"].float()[..., None]
    return k.flatten(-2), v


def _inputs(case, seed):
    """The case's inputs as torch tensors on the device, from the seed alone."""
    g, op, bf16 = _gen(seed), case["op"], torch.bfloat16
    rows = case["rows"]
    if op == "admit":
        page, max_pages = case["page"], case["slots"] // case["page"]
        new = _arange(rows) < case["prompts"]
        new = new[torch.randperm(rows, generator=g, device="cuda")]
        lens = torch.where(new, 0, _ints(g, 1, case["slots"] + 1, rows))
        want = torch.where(new, _ints(g, 1, case["most"] + 1, rows), (torch.rand(rows, generator=g, device="cuda") < 0.95).long())
        held = (lens + page - 1) // page
        need = ((lens + want + page - 1) // page - held).clamp(min=0)
        extra = int(need.sum()) + 8
        table, free = _table(g, rows, max_pages, extra)
        count = _ints(g, extra // 2, extra + 1, 1) if seed % 4 == 3 else torch.full((1,), extra, device="cuda")  # now and then pages run out
        return {"table": table, "free": free, "count": _i32(count), "lens": _i32(lens), "held": _i32(held), "want": _i32(want), "seen": _i32(lens + _ints(g, 0, 100, rows))}
    if op == "rope":
        page, kvh, dim, rot, tokens = case["page"], case["kv_heads"], case["dim"], case["rot"], case["tokens"]
        n, _ = _lengths(case, g)
        before = (torch.rand(rows, generator=g, device="cuda") * (case["slots"] - n + 1)).long()
        table, _ = _table(g, rows, case["slots"] // page)
        starts = _starts(n)
        row = (_arange(tokens)[:, None] >= starts[1:]).sum(-1)
        live, row = row < rows, row.clamp(max=rows - 1)
        slot = torch.where(live, before[row] + _arange(tokens) - starts[row], 0)
        x = {"pos": _i32(slot), "slots": torch.where(live, table[row, slot // page].long() * page + slot % page, -1), "table": table,
             "qkv": _normal(g, tokens, (case["heads"] + 2 * kvh) * dim, dtype=torch.float32 if case["wide"] else bf16)}
        # positions stretched by four beyond the length that a model was trained on
        theta = _arange(case["slots"]).double()[:, None] / 4 * 500000.0 ** (-_arange(rot // 2).double() / (rot // 2))
        x["rope_tab"] = torch.stack([theta.cos(), theta.sin()], -1).float()
        pages = table.numel()
        if case["q4"]:
            return {**x, **_pool4(case, g, pages)}
        return {**x, "k": _normal(g, pages, kvh, page, dim, dtype=bf16), "v": _normal(g, pages, kvh, page, dim, dtype=bf16)}
    if op == "prompt":
        kvh, dim = case["kv_heads"], case["dim"]
        n, ctx = _lengths(case, g)
        starts = _starts(n)
        x = {"starts": _i32(starts), "lens": _i32(n + ctx), "q": _normal(g, _places(case), case["heads"], dim, dtype=bf16)}
        if case["page"]:
            max_pages = -(-(case["most"] + case["ctx"]) // case["page"])
            x["table"], _ = _table(g, rows, max_pages)
            shape = (rows * max_pages, kvh, case["page"], dim)
        else:
            shape = (_places(case), kvh, dim)
        return {**x, "k": _normal(g, *shape, dtype=bf16), "v": _normal(g, *shape, dtype=bf16)}
    max_pages = case["slots"] // case["page"]
    table, _ = _table(g, rows, max_pages)
    lens = _ints(g, 1, case["slots"] + 1, rows) if case["ragged"] else torch.full((rows,), case["slots"], device="cuda")
    return {"table": table, "lens": _i32(lens), "q": _normal(g, rows, case["heads"], case["dim"], dtype=bf16), **_pool4(case, g, rows * max_pages)}


def _handles(case, s):
    """What a program keeps for the framework's calls: the cache's handle, output buffers and the workspace."""
    sys.path.insert(0, os.path.join(os.getcwd(), "catena-lang_amd"))
    import catena_amd as ca

    ca.init(0)
    op, ptr, dev = case["op"], torch.Tensor.data_ptr, {"device": "cuda"}
    rows, heads, kvh, dim, page = (case.get(name, 1) for name in ("rows", "heads", "kv_heads", "dim", "page"))
    s["ca"], nbytes = ca, 0
    if op == "admit":
        s["kv"] = ca.PagedKV(0, 0, 0, s["table"].numel() + s["free"].numel(), page, rows, s["table"].shape[1], 1, 128)
        s["lens_out"], s["held_out"], s["seen_out"], s["count_out"] = (torch.zeros_like(s[name]) for name in ("lens", "held", "seen", "count"))
        s["starts"] = torch.zeros(rows + 1, dtype=torch.int32, **dev)
        s["pos"] = torch.zeros(case["tokens"], dtype=torch.int32, **dev)
        s["slots"] = torch.zeros(case["tokens"], dtype=torch.int64, **dev)
    elif op == "rope":
        if case["q4"]:
            s["kv"] = ca.PagedKV4(ptr(s["k"]), ptr(s["v"]), ptr(s["k_scale"]), ptr(s["v_scale"]), ptr(s["table"]), s["k"].shape[0], page, rows, s["table"].shape[1], kvh, dim)
        else:
            s["kv"] = ca.PagedKV(ptr(s["k"]), ptr(s["v"]), ptr(s["table"]), s["k"].shape[0], page, rows, s["table"].shape[1], kvh, dim)
        s["q"] = torch.zeros(case["tokens"], heads, dim, dtype=torch.bfloat16, **dev)
        s["k_out"], s["v_out"] = (torch.zeros(case["tokens"], kvh, dim, dtype=torch.bfloat16, **dev) for _ in range(2))
    elif op == "prompt":
        s["o"] = torch.zeros_like(s["q"])
        if page:
            s["kv"] = ca.PagedKV(ptr(s["k"]), ptr(s["v"]), ptr(s["table"]), s["k"].shape[0], page, rows, s["table"].shape[1], kvh, dim)
            nbytes = ca.attn_prompt_plan(s["kv"], _places(case), heads)
        else:
            nbytes = ca.attn_packed_plan(rows, _places(case), heads, kvh, dim)
    else:
        s["kv"] = ca.PagedKV4(ptr(s["k"]), ptr(s["v"]), ptr(s["k_scale"]), ptr(s["v_scale"]), ptr(s["table"]), s["k"].shape[0], page, rows, s["table"].shape[1], kvh, dim)
        s["o"] = torch.zeros_like(s["q"])
        nbytes = ca.attn_paged_q4_plan(s["kv"], heads)[1]
    s["work"] = torch.zeros(max(nbytes, 16), dtype=torch.uint8, **dev)
    s["work_bytes"] = nbytes


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:
        _handles(case, s)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls

def _call(s):
    c, ca = s["case"], s["ca"]
    op, ptr, work = c["op"], torch.Tensor.data_ptr, (s["work"].data_ptr(), s["work_bytes"])
    if op == "admit":
        seen = (ptr(s["seen"]), ptr(s["seen_out"])) if c["seen"] else (None, None)
        ca.kv_admit_paged(s["kv"], ptr(s["table"]), ptr(s["lens"]), ptr(s["held"]), ptr(s["want"]), ptr(s["free"]), ptr(s["count"]), ptr(s["lens_out"]), ptr(s["held_out"]),
                          ptr(s["starts"]), ptr(s["count_out"]), ptr(s["pos"]), ptr(s["slots"]), c["tokens"], *seen)
        return {"table": s["table"], "lens": s["lens_out"], "held": s["held_out"], "starts": s["starts"], "count": s["count_out"], "pos": s["pos"], "slots": s["slots"],
                **({"seen": s["seen_out"]} if c["seen"] else {})}
    if op == "rope":
        copies = (ptr(s["k_out"]), ptr(s["v_out"])) if c["copies"] else (None, None)
        call = ca.rope_packed_q4 if c["q4"] else ca.rope_packed_bf16
        call(s["kv"], ptr(s["qkv"]), c["wide"], ptr(s["rope_tab"]), s["rope_tab"].shape[0], c["rot"], c["pairs"] == "next", ptr(s["pos"]), ptr(s["slots"]), ptr(s["q"]),
             c["tokens"], c["heads"], *copies)
        return {"q": s["q"], **{name: s[name] for name in ("k", "v", "k_scale", "v_scale") if name in s}, **({"k_out": s["k_out"], "v_out": s["v_out"]} if c["copies"] else {})}
    if op == "prompt":
        if c["page"]:
            ca.attn_prompt_bf16(s["kv"], ptr(s["q"]), ptr(s["starts"]), ptr(s["lens"]), ptr(s["o"]), _places(c), c["heads"], c["dim"] ** -0.5, work)
        else:
            ca.attn_packed_bf16(ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["starts"]), ptr(s["o"]), c["rows"], _places(c), c["heads"], c["kv_heads"], c["dim"], c["dim"] ** -0.5, work)
        return {"o": s["o"]}
    ca.attn_paged_q4(s["kv"], ptr(s["q"]), ptr(s["lens"]), ptr(s["o"]), c["heads"], c["dim"] ** -0.5, work)
    return {"o": s["o"]}


# ------------------------------------------------------------------ the plain forms

def _plain_admit(s):
    c = s["case"]
    page, rows, max_pages = c["page"], c["rows"], s["table"].shape[1]
    lens, held, want, count = (s[name].long() for name in ("lens", "held", "want", "count"))
    want = torch.where(lens + want <= max_pages * page, want, 0)
    need = ((lens + want + page - 1) // page - held).clamp(min=0)
    need = torch.where(want > 0, need, 0)
    upto, pages = want.cumsum(0), need.cumsum(0)
    fits = (upto <= c["tokens"]) & ((need == 0) | (pages <= count))
    first = pages - need
    want, need = torch.where(fits, want, 0), torch.where(fits, need, 0)
    starts = _starts(want)
    at = _arange(max_pages) - held[:, None]
    given = (at >= 0) & (at < need[:, None])
    fresh = s["free"][(count - 1 - first[:, None] - at).clamp(0, s["free"].numel() - 1)]
    table = torch.where(given, fresh, s["table"])
    token = _arange(c["tokens"])
    row = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    live, row = row < rows, row.clamp(max=rows - 1)
    back = token - starts[row]
    slot = torch.where(live, lens[row] + back, 0)
    seen = s["seen"].long() if c["seen"] else lens
    return {"table": table, "lens": _i32(lens + want), "held": _i32(held + need), "starts": _i32(starts), "count": _i32(count - need.sum()),
            "pos": _i32(torch.where(live, seen[row] + back, 0)), "slots": torch.where(live, table[row, slot // page].long() * page + slot % page, -1),
            **({"seen": _i32(seen + want)} if c["seen"] else {})}


def _plain_rope(s):
    c = s["case"]
    heads, kvh, dim, rot, page = c["heads"], c["kv_heads"], c["dim"], c["rot"], c["page"]
    q, k, v = s["qkv"].view(c["tokens"], heads + 2 * kvh, dim).float().split([heads, kvh, kvh], 1)
    cos, sin = s["rope_tab"][s["pos"].long()].unsqueeze(1).unbind(-1)

    def turn(x):
        part, rest = x[..., :rot], x[..., rot:]
        x1, x2 = part.chunk(2, -1) if c["pairs"] == "half" else (part[..., 0::2], part[..., 1::2])
        y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
        part = torch.cat([y1, y2], -1) if c["pairs"] == "half" else torch.stack([y1, y2], -1).flatten(-2)
        return torch.cat([part, rest], -1).to(torch.bfloat16)

    q, k, v = turn(q), turn(k), v.to(torch.bfloat16)
    live = s["slots"] >= 0
    place = torch.where(live, s["slots"], 0)
    at = (place // page)[live], (place % page)[live]
    out = {"q": q}
    if c["q4"]:
        code, scale, k = _quantised(k)
        s["k"][at[0], :, at[1]], s["k_scale"][at[0], :, :, at[1]] = _pack(code)[live], scale[live]
        code, scale, v = _quantised_v(v)
        s["v"][at[0], :, :, at[1]], s["v_scale"][at[0], :, at[1]] = _pack(code)[live], scale[live]
        out |= {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    else:
        s["k"][at[0], :, at[1]], s["v"][at[0], :, at[1]] = k[live], v[live]
    if c["copies"]:
        out |= {"k_out": k.to(torch.bfloat16), "v_out": v.to(torch.bfloat16)}
    return {**out, "k": s["k"], "v": s["v"]}


def _attend(q, k, v, seen):
    """q [rows][kv heads][queries][dim] over k, v [rows][kv heads][slots][dim] where `seen` [rows][1][queries][slots] or alike is true."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(q.shape[-1] ** -0.5)
    x.masked_fill_(~seen, -math.inf)
    x.sub_(x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    return torch.matmul(x, v).div_(x.sum(-1, keepdim=True))


def _plain_prompt(s):
    c = s["case"]
    rows, heads, kvh, dim, most = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["most"]
    group, starts, lens = heads // kvh, s["starts"].long(), s["lens"].long()
    n = starts[1:] - starts[:-1]
    t = _arange(most)
    live = t < n[:, None]
    token = torch.where(live, starts[:-1, None] + t, 0)
    q = s["q"].float()[token].view(rows, most, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(rows, kvh, most * group, dim)
    if c["page"]:
        k, v = (s[name][s["table"].long()].transpose(2, 3).reshape(rows, -1, kvh, dim).transpose(1, 2).float() for name in "kv")
    else:
        k, v = (s[name][token].transpose(1, 2).float() for name in "kv")
    last = (lens - n)[:, None] + t  # the last slot that a token sees, its own
    seen = _arange(k.shape[2]) <= last.repeat_interleave(group, 1)[..., None]
    o = _attend(q, k, v, seen[:, None]).view(rows, kvh, most, group, dim).permute(0, 2, 1, 3, 4).reshape(rows, most, heads, dim)
    out = torch.zeros_like(s["q"])  # what lies behind the last sequence stays as it was
    out[token[live]] = o[live].to(torch.bfloat16)
    return {"o": out}


def _plain_q4(s):
    c = s["case"]
    rows, heads, kvh, dim, slots = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["slots"]
    k, v = (x[s["table"].long()].transpose(1, 2).reshape(rows, kvh, slots, dim) for x in _held4(s))
    q = s["q"].float().view(rows, kvh, heads // kvh, dim)
    seen = _arange(slots) < s["lens"][:, None, None, None]
    return {"o": _attend(q, k, v, seen).view(rows, heads, dim).to(torch.bfloat16)}


def run(s):
    if own:
        return _call(s)
    return {"admit": _plain_admit, "rope": _plain_rope, "prompt": _plain_prompt, "q4": _plain_q4}[s["case"]["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def _mean(case):
    """A row's new tokens, and the slots that it sees, on average."""
    n = (max(1, _least(case)) + case["most"]) / 2
    return n, n * n / 2 + n * case["ctx"] / 2


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "admit":
        new = case["prompts"] * case["most"] / 2
        return {"bytes": int(28 * rows + 12 * case["tokens"] + 8 * (new / case["page"] + rows / case["page"])), "flops": 0}
    if op == "rope":
        heads, kvh, dim, tokens = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
        cell = dim / 2 + (dim // 32 + 2) / 2 if case["q4"] else 2 * dim  # bytes of a key or a value, scales by half
        out = heads * dim * 2 + 2 * kvh * cell + (4 * kvh * dim if case["copies"] else 0)
        return {"bytes": int(tokens * ((heads + 2 * kvh) * dim * (4 if case["wide"] else 2) + out + 12) + case["slots"] * case["rot"] * 4),
                "flops": int(tokens * 3 * (heads + kvh) * case["rot"])}
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "prompt":
        n, pairs = _mean(case)
        many, one = rows - case["singles"], case["singles"]
        tokens, slots = many * n + one, many * (n + case["ctx"] / 2) + one * (1 + case["ctx"] / 2)
        return {"bytes": int(tokens * heads * dim * 4 + slots * kvh * dim * 4), "flops": int(4 * heads * dim * (many * pairs + one * (1 + case["ctx"] / 2)))}
    n = rows * case["slots"] * (0.5 if case["ragged"] else 1.0)  # ragged lengths: half the cache on average
    return {"bytes": int(n * kvh * (dim + dim // 32 + 2) + rows * heads * dim * 4), "flops": int(4 * n * heads * dim)}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_rope(case, x):
    heads, kvh, dim, rot, page = case["heads"], case["kv_heads"], case["dim"], case["rot"], case["page"]
    y = x["qkv"].double().view(case["tokens"], heads + 2 * kvh, dim).clone()
    tab = x["rope_tab"].double()[x["pos"].long()]
    angle = torch.complex(tab[..., 0], tab[..., 1])[:, None]
    i = torch.arange(rot // 2, device="cuda")
    first, second = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(y[:, : heads + kvh, first], y[:, : heads + kvh, second]) * angle
    y[:, : heads + kvh, first], y[:, : heads + kvh, second] = z.real, z.imag
    out = {"q": y[:, :heads], "k": None, "v": None, "k_scale": None, "v_scale": None, "k_out": None, "v_out": None}
    if case["q4"]:
        return out
    k, v = x["k"].double(), x["v"].double()
    keep = (x["slots"] >= 0).nonzero()[:, 0]
    slot = x["slots"][keep]
    k[slot // page, :, slot % page], v[slot // page, :, slot % page] = y[keep, heads:heads + kvh], y[keep, heads + kvh:]
    return {"q": y[:, :heads], "k": k, "v": v, **({"k_out": y[:, heads:heads + kvh], "v_out": y[:, heads + kvh:]} if case["copies"] else {})}


def _exact_prompt(case, x):
    heads, kvh, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    o = torch.zeros(_places(case), heads, dim, device="cuda", dtype=torch.float64)
    starts, lens = x["starts"].tolist(), x["lens"].tolist()
    for r in range(case["rows"]):
        a, b, n = starts[r], starts[r + 1], lens[r]
        for h in range(kvh):
            if page:
                pages = x["table"][r, : -(-n // page)].long()
                k, v = (x[name][pages, h].reshape(-1, dim)[:n].double() for name in "kv")
            else:
                k, v = (x[name][a:b, h].double() for name in "kv")
            late = torch.ones(b - a, n, device="cuda", dtype=torch.bool).triu(n - (b - a) + 1)
            for j in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                p = torch.softmax(((x["q"][a:b, j].double() @ k.T) / math.sqrt(dim)).masked_fill_(late, -math.inf), -1)
                o[a:b, j] = p @ v
    return {"o": o}


def _exact_q4(case, x):
    rows, heads, kvh, dim, page = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    o = torch.zeros(rows, heads, dim, device="cuda", dtype=torch.float64)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda", dtype=torch.float64)
    for r in range(rows):
        n = int(x["lens"][r])
        pages = x["table"][r, : -(-n // page)].long()
        for h in range(kvh):
            byte, unit = x["k"][pages, h].flatten(0, 1)[:n].long(), x["k_scale"][pages, h].transpose(-1, -2).flatten(0, 1)[:n].double()
            k = torch.stack([grid[byte % 16], grid[byte // 16]], -1).view(n, dim) * (2.0 ** (unit - 127)).repeat_interleave(32, 1)
            byte, unit = x["v"][pages, h].transpose(-1, -2).flatten(0, 1)[:n].long(), x["v_scale"][pages, h].flatten()[:n].double()
            v = torch.stack([grid[byte % 16], grid[byte // 16]], -1).view(n, dim) * unit[:, None]
            mine = slice(h * (heads // kvh), (h + 1) * (heads // kvh))
            o[r, mine] = torch.softmax((x["q"][r, mine].double() @ k.T) / math.sqrt(dim), -1) @ v
    return {"o": o}


def exact(case, seed):
    if case["op"] == "admit":
        return None  # whole numbers alone
    return {"rope": _exact_rope, "prompt": _exact_prompt, "q4": _exact_q4}[case["op"]](case, _inputs(case, seed))
