"""The paged cache's and the beam search's operators, as measurable cases.

Every case is one pass through one operator, on inputs already resident on the
device:

  attn     attn_paged_bf16: one new token of every row over a cache in pages,
           with or without the accumulated attention weights
  append   rope_qkv_paged_bf16: rotation, and the new rows written into pages
  evict    kv_evict_paged_bf16: the slots of least accumulated weight given up
  select   beam_select_f32: the best continuations over beams and vocabulary
  reorder  beam_reorder_paged_bf16: page tables and last pages of the parents

`own` chooses between the operators' plain form and the framework's calls.
`listed()` names the cases, `draw(rng)` gives more of the same ranges.
"""
import math
import os
import sys

import torch

own = False

EOS = 2  # the token that ends a beam


def listed():
    return [
        # one sequence of a 16-head decoder, a short cache: latency alone
        {"name": "attn_one_row", "op": "attn", "rows": 1, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16, "slots": 640, "ragged": False, "weights": False, "out": "f32"},
        # a serving batch, grouped heads, lengths from one token to the whole cache
        {"name": "attn_batch", "op": "attn", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "slots": 4096, "ragged": True, "weights": False, "out": "bf16"},
        # one long document: few rows, so the work is split over the length
        {"name": "attn_long", "op": "attn", "rows": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "slots": 131072, "ragged": False, "weights": False, "out": "bf16"},
        # a bounded cache that gathers the weights its eviction goes by; an odd length
        {"name": "attn_weights", "op": "attn", "rows": 8, "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "slots": 5152, "ragged": True, "weights": True, "out": "bf16"},
        # a decode step of 8 sequences
        {"name": "append_step", "op": "append", "rows": 8, "tq": 1, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16, "slots": 640, "tracked": True},
        # prompts of 500 tokens into pages
        {"name": "append_prompt", "op": "append", "rows": 8, "tq": 500, "heads": 16, "kv_heads": 16, "dim": 128, "page": 32, "slots": 640, "tracked": False},
        # every step gives up one slot of a full cache
        {"name": "evict_step", "op": "evict", "rows": 8, "kv_heads": 16, "dim": 128, "page": 16, "slots": 528, "budget": 512, "recent": 64, "over": 1},
        # now and then a fifth of a long cache
        {"name": "evict_fifth", "op": "evict", "rows": 32, "kv_heads": 8, "dim": 128, "page": 32, "slots": 5120, "budget": 4096, "recent": 512, "over": 1024},
        # one request of four beams
        {"name": "select_request", "op": "select", "groups": 1, "beams": 4, "vocab": 32000, "first": False},
        # a full batch over a large vocabulary
        {"name": "select_batch", "op": "select", "groups": 32, "beams": 8, "vocab": 128000, "first": False},
        # one request of four beams in a one-layer decoder
        {"name": "reorder_request", "op": "reorder", "groups": 1, "beams": 4, "layers": 1, "kv_heads": 16, "dim": 128, "page": 16, "slots": 640, "len": 333},
        # a full batch, sixteen layers
        {"name": "reorder_batch", "op": "reorder", "groups": 8, "beams": 8, "layers": 16, "kv_heads": 8, "dim": 128, "page": 64, "slots": 320, "len": 241},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _slots(rng, lo, hi, page):
    return max(1, -(-_log(rng, lo, hi) // page)) * page


def draw(rng):
    op = rng.choice(["attn", "attn", "append", "evict", "select", "reorder"])
    page, dim = rng.choice([16, 32, 64, 128]), rng.choice([128, 128, 64])
    if op == "attn":
        while True:
            kv_heads, group = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 1, 2, 4, 7, 8, 16, 24])
            c = {"op": op, "rows": _log(rng, 1, 64), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "slots": _slots(rng, 16, 131072, page),
                 "ragged": rng.random() < 0.5, "weights": rng.random() < 0.3, "out": rng.choice(["bf16", "f32"])}
            if c["heads"] <= 64 and c["rows"] * c["slots"] * kv_heads <= 64 * 4096 * 8 and c["rows"] * c["slots"] * c["heads"] <= 64 * 4096 * 32:
                return c
    if op == "append":
        while True:
            kv_heads, group, tq = rng.choice([1, 4, 8, 16, 32]), rng.choice([1, 2, 4, 7]), rng.choice([1, 1, _log(rng, 2, 2000)])
            c = {"op": op, "rows": _log(rng, 1, 64), "tq": tq, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "slots": _slots(rng, tq, 2 * tq + 1000, page),
                 "tracked": rng.random() < 0.5}
            if c["heads"] <= 64 and c["rows"] * tq * (c["heads"] + 2 * kv_heads) <= 8 * 500 * 48 and c["rows"] * c["slots"] * kv_heads <= 1 << 20:
                return c
    if op == "evict":
        while True:
            budget, rows, kv_heads = _log(rng, 64, 8192), _log(rng, 1, 64), rng.choice([1, 4, 8, 16])
            over = rng.choice([1, 1, _log(rng, 2, budget)])
            c = {"op": op, "rows": rows, "kv_heads": kv_heads, "dim": dim, "page": page, "slots": -(-(budget + over) // page) * page, "budget": budget,
                 "recent": rng.randint(0, budget), "over": over}
            if rows * kv_heads * c["slots"] <= 32 * 8 * 5120:
                return c
    if op == "select":
        while True:
            c = {"op": op, "groups": _log(rng, 1, 64), "beams": rng.choice([1, 2, 3, 4, 5, 8, 10, 16]), "vocab": _log(rng, 1000, 128000), "first": rng.random() < 0.25}
            if c["groups"] * c["beams"] * c["vocab"] <= 32 * 8 * 128000:
                return c
    while True:
        c = {"op": op, "groups": _log(rng, 1, 16), "beams": rng.randint(2, 16), "layers": _log(rng, 1, 16), "kv_heads": rng.choice([1, 4, 8, 16]), "dim": dim, "page": page,
             "slots": _slots(rng, 64, 1024, page)}
        c["len"] = rng.randint(1, c["slots"])
        if c["groups"] * c["beams"] * c["layers"] * c["kv_heads"] * c["dim"] * (c["slots"] + page) <= 64 * 16 * 8 * 128 * 384:
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


def _pool(case, g, extra=0):
    """The geometry, page pools of K and V, and a table of every row's own pages in any order."""
    rows = case["rows"] if "rows" in case else case["groups"] * case["beams"]
    per_row = case["slots"] // case["page"]
    pages = rows * per_row + extra
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    return shape, {"table": order[: rows * per_row].view(rows, per_row).contiguous(), "spare": order[rows * per_row:].contiguous()}


def _inputs(case, seed):
    """The case's inputs as torch tensors on the device, from the seed alone."""
    g, op, bf16 = _gen(seed), case["op"], torch.bfloat16
    if op == "select":
        groups, w, v = case["groups"], case["beams"], case["vocab"]
        scores = -torch.rand(groups, w, generator=g, device="cuda") * 8 - 4
        done = (torch.rand(groups, w, generator=g, device="cuda") < 0.1).to(torch.int32)
        if case["first"]:  # the prompt's beams are alike: the first of them alone counts
            scores = torch.where(_arange(w) == 0, torch.zeros_like(scores), torch.full_like(scores, -math.inf))
            done = torch.zeros_like(done)
        return {"logits": _normal(g, groups, w, v, scale=2.5), "scores": scores, "done": done}
    if op == "reorder":
        groups, w, rows = case["groups"], case["beams"], case["groups"] * case["beams"]
        shape, x = _pool(case, g, rows)
        x["caches"] = torch.empty(2 * case["layers"], *shape, device="cuda", dtype=bf16)
        for one in x["caches"]:
            one.copy_(torch.randn(shape, generator=g, device="cuda", dtype=bf16))
        x["parents"] = (_ints(g, 0, w, groups, w) + w * _arange(groups)[:, None]).reshape(rows).to(torch.int32)
        x["lens"] = torch.full((rows,), case["len"], device="cuda", dtype=torch.int32)
        return x
    rows, kvh, dim, slots = case["rows"], case["kv_heads"], case["dim"], case["slots"]
    shape, x = _pool(case, g)
    x["k"], x["v"] = (_normal(g, *shape, dtype=bf16) for _ in range(2))
    if op == "attn":
        x["q"] = _normal(g, rows, case["heads"], dim, dtype=bf16)
        lens = _ints(g, 1, slots + 1, rows) if case["ragged"] else torch.full((rows,), slots, device="cuda")
        x["lens"] = lens.to(torch.int32)
        if case["weights"]:
            x["acc"] = torch.rand(rows, kvh, slots, generator=g, device="cuda")
    elif op == "append":
        tq = case["tq"]
        x["qkv"] = _normal(g, rows * tq, (case["heads"] + 2 * kvh) * dim)
        x["lens"] = _ints(g, tq, slots + 1, rows).to(torch.int32)
        x["seen"] = (x["lens"] + 100).to(torch.int32)  # a hundred positions were given up before
        theta = _arange(slots + 100).double()[:, None] * 10000.0 ** (-_arange(dim // 2).double() / (dim // 2))
        x["rope_tab"] = torch.stack([theta.cos(), theta.sin()], -1).float()
        if case["tracked"]:
            x["acc"] = torch.rand(rows, kvh, slots, generator=g, device="cuda")
            x["slot_pos"] = _ints(g, 0, slots, rows, kvh, slots).to(torch.int32)
    else:
        n = case["budget"] + case["over"]
        x["lens"] = torch.full((rows,), n, device="cuda", dtype=torch.int32)
        x["acc"] = _normal(g, rows, kvh, slots, scale=1.5).exp_()
        # positions that are left of a longer text, in the order that earlier evictions gave them
        gaps = torch.where(_arange(slots) < n - case["recent"], _ints(g, 1, 4, rows, kvh, slots), 1)
        pos = gaps.cumsum(-1)
        x["seen"] = torch.full((rows,), 4 * slots, device="cuda", dtype=torch.int32)
        pos = pos - pos[..., n - 1:n] + 4 * slots - 1
        mixed = torch.argsort(torch.rand(rows, kvh, slots, generator=g, device="cuda") + (_arange(slots) >= n), -1)
        x["slot_pos"] = pos.gather(-1, mixed).to(torch.int32)
    return x


def _handles(case, s):
    """What a program keeps for the framework's calls: the cache's handle, output buffers and the workspace."""
    sys.path.insert(0, os.path.join(os.getcwd(), "catena-lang_amd"))
    import catena_amd as ca

    ca.init(0)
    op, dev = case["op"], {"device": "cuda"}
    s["ca"] = ca
    if op != "select":
        pool = s["caches"][0] if op == "reorder" else s["k"]
        k, v = (0, 0) if op == "reorder" else (s["k"].data_ptr(), s["v"].data_ptr())
        rows, max_pages = s["table"].shape
        s["kv"] = ca.PagedKV(k, v, s["table"].data_ptr(), pool.shape[0], case["page"], rows, max_pages, case["kv_heads"], case["dim"])
    nbytes = 0
    if op == "attn":
        s["o"] = torch.zeros(s["q"].shape, dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float32, **dev)
        nbytes = ca.attn_paged_plan(s["kv"], case["heads"], case["weights"])[1]
        if case["weights"]:
            s["acc_out"] = s["acc"].clone()
    elif op == "append":
        s["q"] = torch.zeros(case["rows"], case["tq"], case["heads"], case["dim"], dtype=torch.bfloat16, **dev)
    elif op == "evict":
        s["lens_out"], s["acc_out"], s["pos_out"] = torch.zeros_like(s["lens"]), s["acc"].clone(), s["slot_pos"].clone()
        nbytes = ca.kv_evict_paged_plan(s["kv"], case["budget"])
    elif op == "select":
        shape = (case["groups"], case["beams"])
        s["tokens"], s["parents"], s["done_out"] = (torch.zeros(shape, dtype=torch.int32, **dev) for _ in range(3))
        s["scores_out"] = torch.zeros(shape, **dev)
        nbytes = ca.beam_select_plan(*shape, case["vocab"])
    else:
        s["table_out"], s["lens_out"], s["spare_out"] = torch.zeros_like(s["table"]), torch.zeros_like(s["lens"]), torch.zeros_like(s["spare"])
        s["pools"] = [one.data_ptr() for one in s["caches"]]
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
    if op == "attn":
        acc = (ptr(s["acc"]), ptr(s["acc_out"])) if c["weights"] else (None, None)
        ca.attn_paged_bf16(s["kv"], ptr(s["q"]), ptr(s["lens"]), ptr(s["o"]), c["heads"], c["dim"] ** -0.5, work, c["out"] == "f32", *acc)
        return {"o": s["o"], **({"acc": s["acc_out"]} if c["weights"] else {})}
    if op == "append":
        extra = (ptr(s["acc"]), ptr(s["slot_pos"])) if c["tracked"] else (None, None)
        ca.rope_qkv_paged_bf16(s["kv"], ptr(s["qkv"]), ptr(s["rope_tab"]), s["rope_tab"].shape[0], ptr(s["lens"]), ptr(s["seen"]), ptr(s["q"]), c["tq"], c["heads"], *extra)
        return {"q": s["q"], "k": s["k"], "v": s["v"], **({"acc": s["acc"], "slot_pos": s["slot_pos"]} if c["tracked"] else {})}
    if op == "evict":
        ca.kv_evict_paged_bf16(s["kv"], ptr(s["lens"]), ptr(s["seen"]), ptr(s["acc"]), ptr(s["slot_pos"]), ptr(s["lens_out"]), ptr(s["acc_out"]), ptr(s["pos_out"]),
                               c["budget"], c["recent"], work)
        return {"k": s["k"], "v": s["v"], "acc": s["acc_out"], "slot_pos": s["pos_out"], "lens": s["lens_out"]}
    if op == "select":
        ca.beam_select_f32(ptr(s["logits"]), ptr(s["scores"]), ptr(s["done"]), ptr(s["tokens"]), ptr(s["parents"]), ptr(s["scores_out"]), ptr(s["done_out"]),
                           c["groups"], c["beams"], c["vocab"], EOS, work)
        return {"tokens": s["tokens"], "parents": s["parents"], "scores": s["scores_out"], "done": s["done_out"]}
    ca.beam_reorder_paged_bf16(s["kv"], s["pools"], ptr(s["lens"]), ptr(s["parents"]), ptr(s["spare"]), ptr(s["table_out"]), ptr(s["lens_out"]), ptr(s["spare_out"]))
    return {"caches": s["caches"], "table": s["table_out"], "lens": s["lens_out"], "spare": s["spare_out"]}


# ------------------------------------------------------------------ the plain forms

def _places(s, slot):
    """(page, place in the page) of slots [rows, ..., n] of every row."""
    page = s["case"]["page"]
    rows = _arange(slot.shape[0]).view(-1, *[1] * (slot.dim() - 1))
    return s["table"][rows, slot // page].long(), slot % page


def _plain_attn(s):
    c = s["case"]
    rows, kvh, dim, slots, heads = c["rows"], c["kv_heads"], c["dim"], c["slots"], c["heads"]
    table = s["table"].long()
    k, v = (s[name][table].transpose(1, 2).reshape(rows, kvh, slots, dim).float() for name in "kv")
    q = s["q"].float().view(rows, kvh, heads // kvh, dim)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * dim**-0.5
    valid = _arange(slots) < s["lens"][:, None, None, None]
    x = x.masked_fill(~valid, -math.inf)
    e = torch.where(valid, (x - x.amax(-1, keepdim=True)).exp(), 0.0)
    p = e / e.sum(-1, keepdim=True)
    o = torch.where((s["lens"] > 0)[:, None, None, None], torch.matmul(p, v), 0.0).view(rows, heads, dim)
    out = {"o": o.to(torch.bfloat16 if c["out"] == "bf16" else torch.float32)}
    if c["weights"]:
        out["acc"] = s["acc"] + torch.where(valid, p, 0.0).sum(2)
    return out


def _plain_append(s):
    c = s["case"]
    rows, tq, heads, kvh, dim = c["rows"], c["tq"], c["heads"], c["kv_heads"], c["dim"]
    back = _arange(tq) - tq
    slot, pos = s["lens"][:, None] + back, s["seen"][:, None] + back
    q, k, v = s["qkv"].view(rows, tq, heads + 2 * kvh, dim).split([heads, kvh, kvh], 2)
    cos, sin = s["rope_tab"][pos].unsqueeze(2).unbind(-1)

    def rope(x):
        x1, x2 = x.chunk(2, -1)
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).to(torch.bfloat16)

    page, place = _places(s, slot)
    s["k"][page, :, place] = rope(k)
    s["v"][page, :, place] = v.to(torch.bfloat16)
    out = {"q": rope(q), "k": s["k"], "v": s["v"]}
    if c["tracked"]:
        row = _arange(rows)[:, None].expand_as(slot)
        s["acc"][row, :, slot] = 0.0
        s["slot_pos"][row, :, slot] = pos[..., None].expand(rows, tq, kvh).to(torch.int32)
        out |= {"acc": s["acc"], "slot_pos": s["slot_pos"]}
    return out


def _plain_evict(s):
    c = s["case"]
    slots, budget = c["slots"], c["budget"]
    slot, lens = _arange(slots), s["lens"].long()
    valid = slot < lens[:, None, None]
    late = s["slot_pos"] >= (s["seen"] - c["recent"])[:, None, None]
    key = torch.where(valid, torch.where(late, math.inf, s["acc"]), -1.0)
    rank = torch.empty_like(key, dtype=torch.int64)
    rank.scatter_(-1, torch.sort(key, dim=-1, descending=True, stable=True)[1], slot.expand_as(rank).contiguous())
    new = lens.clamp(max=budget)
    keep = rank < new[:, None, None]
    hole, mover = ~keep & (slot < new[:, None, None]), keep & (slot >= budget)
    spot = torch.where(mover, mover.cumsum(-1) - 1, slots)  # the i-th mover's slot at i, the others in a bin of their own
    movers = torch.zeros(*key.shape[:2], slots + 1, device="cuda", dtype=torch.int64).scatter_(-1, spot, slot.expand_as(spot).contiguous())
    src = torch.where(hole, movers.gather(-1, torch.where(hole, hole.cumsum(-1) - 1, slots)), slot)
    head = _arange(c["kv_heads"])[None, :, None]
    (to_page, to_place), (page, place) = (_places(s, i.expand_as(src)[..., :budget]) for i in (slot, src))
    s["k"][to_page, head, to_place] = s["k"][page, head, place]
    s["v"][to_page, head, to_place] = s["v"][page, head, place]
    return {"k": s["k"], "v": s["v"], "acc": s["acc"].gather(-1, src), "slot_pos": s["slot_pos"].gather(-1, src), "lens": new.to(torch.int32)}


def _plain_select(s):
    c = s["case"]
    groups, w, v = c["groups"], c["beams"], c["vocab"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    score = s["scores"].double()[..., None]
    done = (s["done"] != 0)[..., None]
    total = torch.where(done, torch.where(_arange(v) == EOS, score, -math.inf), score + (x - lse))
    # a stable order of the few best of every beam gives that of all: ties go to the lower index
    best, token = torch.sort(total, dim=-1, descending=True, stable=True)
    best, token = (t[..., : min(w, v)].reshape(groups, -1) for t in (best, token))
    best, at = torch.sort(best, dim=-1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    beam, token = at // min(w, v), token.gather(-1, at)
    live = best > -math.inf
    beam = torch.where(live, beam, _arange(w))
    token = torch.where(live, token, 0)
    ends = (s["done"].gather(-1, beam) != 0) | (token == EOS)
    return {"tokens": token.to(torch.int32), "parents": (beam + w * _arange(groups)[:, None]).to(torch.int32), "scores": best.float(),
            "done": torch.where(live, ends, False).to(torch.int32)}


def _plain_reorder(s):
    c = s["case"]
    rows, page = s["table"].shape[0], c["page"]
    parent, own_row = s["parents"].long(), _arange(rows)
    n = s["lens"].long()[parent]
    last, used, moved = n // page, n % page, parent != own_row
    at = _arange(s["table"].shape[1])
    partly = (used > 0) & moved
    table = torch.where(at < last[:, None], s["table"][parent], s["table"])
    table = torch.where(partly[:, None] & (at == last[:, None]), s["spare"][:, None], table)
    table = torch.where(moved[:, None], table, s["table"])
    edge = last.clamp(max=at.numel() - 1)
    tail, mine = s["table"][parent, edge].long(), s["table"][own_row, edge]
    spare = s["spare"].long()
    copied = (_arange(page)[None, None, :, None] < used[:, None, None, None]) & partly[:, None, None, None]
    s["caches"][:, spare] = torch.where(copied, s["caches"][:, tail], s["caches"][:, spare])
    return {"caches": s["caches"], "table": table, "lens": n.to(torch.int32), "spare": torch.where(partly, mine, s["spare"])}


def run(s):
    if own:
        return _call(s)
    return {"attn": _plain_attn, "append": _plain_append, "evict": _plain_evict, "select": _plain_select, "reorder": _plain_reorder}[s["case"]["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "attn":
        n = case["rows"] * case["slots"] * (0.5 if case["ragged"] else 1.0)  # ragged lengths: half the cache on average
        cache = n * case["kv_heads"] * case["dim"] * 4
        small = case["rows"] * case["heads"] * case["dim"] * (2 + (2 if case["out"] == "bf16" else 4))
        return {"bytes": int(cache + small + (8 * n * case["kv_heads"] if case["weights"] else 0)), "flops": int(4 * n * case["heads"] * case["dim"])}
    if op == "append":
        n, wide = case["rows"] * case["tq"], case["heads"] + 2 * case["kv_heads"]
        return {"bytes": int(n * (wide * case["dim"] * 6 + (8 * case["kv_heads"] if case["tracked"] else 0)) + 4 * case["tq"] * case["dim"]),
                "flops": int(n * 3 * (case["heads"] + case["kv_heads"]) * case["dim"])}
    if op == "evict":
        n, budget = case["budget"] + case["over"], case["budget"]
        pairs, moves = case["rows"] * case["kv_heads"], case["over"] * budget / n  # slots are given up anywhere
        return {"bytes": int(pairs * (8 * (n + budget) + moves * 8 * case["dim"])), "flops": 0}
    if op == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * n, "flops": 3 * n}
    rows, moved = case["groups"] * case["beams"], 1 - 1 / case["beams"]
    tail = rows * moved * (case["len"] % case["page"]) * case["kv_heads"] * case["dim"] * 2
    return {"bytes": int(2 * case["layers"] * 2 * tail + rows * (8 * (case["slots"] // case["page"]) + 16)), "flops": 0}


# ------------------------------------------------------------------ the same in 64 bits

def _row_cache(x, pool, case, r):
    """Row r's slots of one pool in 64 bits, [kv heads][slots][dim]."""
    return torch.cat([x[pool][int(i)].double() for i in x["table"][r]], 1)


def _exact_attn(case, x):
    rows, kvh, dim = case["rows"], case["kv_heads"], case["dim"]
    o = torch.zeros(rows, case["heads"], dim, device="cuda", dtype=torch.float64)
    acc = x["acc"].double() if case["weights"] else None
    for r in range(rows):
        n = int(x["lens"][r])
        k, v = (_row_cache(x, pool, case, r)[:, :n] for pool in "kv")
        for h in range(kvh):
            mine = slice(h * (case["heads"] // kvh), (h + 1) * (case["heads"] // kvh))
            p = torch.softmax((x["q"][r, mine].double() @ k[h].T) / math.sqrt(dim), -1)
            o[r, mine] = p @ v[h]
            if case["weights"]:
                acc[r, h, :n] += p.sum(0)
    return {"o": o, **({"acc": acc} if case["weights"] else {})}


def _exact_append(case, x):
    rows, tq, heads, kvh, dim = case["rows"], case["tq"], case["heads"], case["kv_heads"], case["dim"]
    qkv, tab = x["qkv"].double().view(rows, tq, -1, dim), x["rope_tab"].double()
    k, v = x["k"].double(), x["v"].double()
    turned = torch.empty(rows, tq, heads + kvh, dim, device="cuda", dtype=torch.float64)
    for r in range(rows):
        n, seen = int(x["lens"][r]), int(x["seen"][r])
        angle = tab[seen - tq:seen, :, 0] + 1j * tab[seen - tq:seen, :, 1]
        z = (qkv[r, :, : heads + kvh, : dim // 2] + 1j * qkv[r, :, : heads + kvh, dim // 2:]) * angle[:, None]
        turned[r] = torch.cat([z.real, z.imag], -1)
        slot = torch.arange(n - tq, n, device="cuda")
        page = x["table"][r, slot // case["page"]].long()
        k[page, :, slot % case["page"]] = turned[r, :, heads:]
        v[page, :, slot % case["page"]] = qkv[r, :, heads + kvh:]
        if case["tracked"]:
            x["acc"][r, :, n - tq:n] = 0
    return {"q": turned[:, :, :heads], "k": k, "v": v, **({"acc": x["acc"].double(), "slot_pos": None} if case["tracked"] else {})}


def _exact_evict(case, x):
    page, budget = case["page"], case["budget"]
    pools, acc = {name: x[name].double() for name in "kv"}, x["acc"].double().cpu()
    pos, table = x["slot_pos"].cpu().tolist(), x["table"].cpu().tolist()
    to, source = [], []
    for r in range(case["rows"]):
        n, seen = int(x["lens"][r]), int(x["seen"][r])
        for h in range(case["kv_heads"]):
            weight = acc[r, h].tolist()
            best = sorted(range(n), key=lambda j: (pos[r][h][j] < seen - case["recent"], -weight[j] if pos[r][h][j] < seen - case["recent"] else 0, j))
            kept = set(best[:budget])
            holes = [j for j in range(min(n, budget)) if j not in kept]
            for j, i in zip(holes, sorted(i for i in kept if i >= budget)):
                to.append((table[r][j // page], h, j % page))
                source.append((table[r][i // page], h, i % page))
                acc[r, h, j] = weight[i]
    if to:
        t, f = (torch.tensor(z, device="cuda").T for z in (to, source))
        for p in pools.values():
            p[t[0], t[1], t[2]] = p[f[0], f[1], f[2]]
    return {**pools, "acc": acc, "slot_pos": None, "lens": None}


def _exact_select(case, x):
    groups, w, v = case["groups"], case["beams"], case["vocab"]
    scores = torch.empty(groups, w, dtype=torch.float64)
    for i in range(groups):
        every = torch.log_softmax(x["logits"][i].double(), -1) + x["scores"][i].double()[:, None]
        every[x["done"][i] != 0] = -math.inf
        ended = x["scores"][i].double()[x["done"][i] != 0]
        scores[i] = torch.cat([every.reshape(-1), ended]).topk(w)[0].cpu()
    return {"tokens": None, "parents": None, "scores": scores, "done": None}


def _exact_reorder(case, x):
    page, caches = case["page"], x["caches"]
    table, spare, parents = (x[name].tolist() for name in ("table", "spare", "parents"))
    last, used = case["len"] // page, case["len"] % page
    new = caches.clone()
    for r, p in enumerate(parents):
        if p != r and used:
            new[:, spare[r], :, :used] = caches[:, table[p][last], :, :used]
    return {"caches": new, "table": None, "lens": None, "spare": None}


def exact(case, seed):
    return {"attn": _exact_attn, "append": _exact_append, "evict": _exact_evict, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](case, _inputs(case, seed))
