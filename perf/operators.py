"""Attention of a batch whose requests share a long prefix, by which the operators of ds41rt_b200.ops.prefix are followed.

A server that answers many requests over one system prompt, or several answers to one question, keeps the pages of the common
part once; every request's page table begins with them.  A decode pass has one row per request.  The operators read the common
pages once for all rows instead of once per row:

  "grouped": grouped-query attention over cached keys and values, with chunked visibility and a sigmoid gate per head;
  "latent":  attention over one cached latent row per token (queries already multiplied by the key expansion), with a sink.

A case names the pass: `rows` requests over `prefixes` different common parts (the longest `prefix` tokens, the next half of
that, and so on), of which the last `alone` share nothing and `pads` more rows own no slot; every request has up to `own` tokens
after the common part.  Positions follow from the row number, pages and values from the seed.
"""
from __future__ import annotations

import math

import torch

own = False


# ---------------------------------------------------------------------------------------------------- the cases
def _grouped(name, rows, prefix, tail, heads=32, kv_heads=8, dim=128, vdim=128, prefixes=1, alone=0, pads=0, page=64, chunk=0,
             dtype="bf16"):
    return {"name": name, "kind": "grouped", "rows": rows, "prefix": prefix, "own": tail, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "vdim": vdim, "prefixes": prefixes, "alone": alone, "pads": pads, "page": page, "chunk": chunk,
            "dtype": dtype}


def _latent(name, rows, prefix, tail, heads=32, latent=512, rot=64, prefixes=1, alone=0, pads=0, page=64, dtype="bf16"):
    return {"name": name, "kind": "latent", "rows": rows, "prefix": prefix, "own": tail, "heads": heads, "kv_heads": 1,
            "dim": latent + rot, "vdim": latent, "prefixes": prefixes, "alone": alone, "pads": pads, "page": page, "chunk": 0,
            "dtype": dtype}


def listed():
    return [
        # four answers to one short question: the smallest call, where launches count
        _grouped("grouped 4 x 300", 4, 300, 40, heads=16, kv_heads=4),
        # a server's ordinary step: 32 requests over a system prompt of a few thousand tokens
        _grouped("grouped 32 x 4096", 32, 4096, 400),
        # many requests over one long document
        _grouped("grouped 200 x 16000", 200, 16000, 700),
        # chunked visibility: rows behind a chunk's border see a part of the common part, or nothing of it
        _grouped("grouped 40 x 7500 chunked", 40, 7500, 1500, chunk=8192, page=32),
        # odd heads and widths, two common parts, requests without one, rows without a slot
        _grouped("grouped 37 x 1501 mixed", 37, 1501, 150, heads=6, kv_heads=2, dim=32, vdim=48, prefixes=2, alone=5, pads=3),
        # the 32-bit form
        _grouped("grouped 8 x 1000 f32", 8, 1000, 100, heads=16, kv_heads=4, dtype="f32"),
        # the same calls of latent attention
        _latent("latent 4 x 300", 4, 300, 40, heads=16),
        _latent("latent 32 x 4096", 32, 4096, 400),
        _latent("latent 128 x 16000", 128, 16000, 700),
        _latent("latent 48 x 6000 three", 48, 6000, 300, heads=16, prefixes=3, alone=2),
        _latent("latent 19 x 777 narrow", 19, 777, 90, heads=5, latent=64, rot=32, pads=2, page=32),
        _latent("latent 6 x 500 f32", 6, 500, 60, heads=16, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["grouped", "latent"])
    dtype = "f32" if rng.random() < 0.1 else "bf16"
    rows = _spread(rng, 2, 24) if dtype == "f32" else _spread(rng, 2, 200 if kind == "grouped" else 128)
    prefix = _spread(rng, 64, 2000) if dtype == "f32" else _spread(rng, 64, 16000)
    prefixes = rng.choice([1, 1, 1, 2, 3])
    more = dict(prefixes=min(prefixes, rows // 2), alone=rng.choice([0, 0, 1, rows // 6]), pads=rng.choice([0, 0, 3]),
                page=rng.choice([32, 64, 64, 128]), dtype=dtype)
    tail = _spread(rng, 2, 700)
    if kind == "grouped":
        heads, kv_heads = rng.choice([(16, 4), (32, 8), (32, 8), (6, 2), (8, 8), (12, 1), (20, 4)])
        dim, vdim = rng.choice([(128, 128), (128, 128), (64, 64), (32, 48), (192, 128)])
        c = _grouped("", rows, prefix, tail, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim,
                     chunk=rng.choice([0, 0, 8192, 96]), **more)
    else:
        latent, rot = rng.choice([(512, 64), (512, 64), (256, 64), (64, 32)])
        c = _latent("", rows, prefix, tail, heads=rng.choice([16, 32, 32, 5, 8]), latent=latent, rot=rot, **more)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- what a pass looks like
def _layout(case):
    """Of every request: the common part it continues (-1: none), that part's tokens in whole pages, and its last position."""
    part, shared, last = [], [], []
    for i in range(case["rows"]):
        j = -1 if i >= case["rows"] - case["alone"] else i % case["prefixes"]
        tokens = max(1, case["prefix"] >> max(j, 0))
        part.append(j)
        shared.append(0 if j < 0 else tokens // case["page"] * case["page"])
        last.append(tokens + (i * 7919 + 13) % case["own"])
    return part, shared, last


def _first(case, pos):
    return pos - pos % case["chunk"] if case["chunk"] else 0


def work(case):
    part, shared, last = _layout(case)
    size = 2 if case["dtype"] == "bf16" else 4
    row = case["kv_heads"] * (case["dim"] + case["vdim"]) if case["kind"] == "grouped" else case["dim"]
    seen, keys, reach = 0, 0, {}
    for j, s, p in zip(part, shared, last):
        lo = _first(case, p)
        seen += p + 1 - lo
        keys += p + 1 - max(lo, s)
        if lo < s:
            reach[j] = max(reach.get(j, 0), s - lo)
    keys += sum(reach.values())
    wide = case["heads"] * (case["dim"] + case["vdim"])
    gates = 4 * case["rows"] * case["heads"] if case["kind"] == "grouped" else 4 * case["heads"]
    return {"bytes": size * (keys * row + (case["rows"] + case["pads"]) * wide) + gates, "flops": 2 * wide * seen}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    part, shared, last = _layout(case)
    n, P, H = case["rows"], case["page"], case["heads"]
    row = case["kv_heads"] * (case["dim"] + case["vdim"]) if case["kind"] == "grouped" else case["dim"]
    max_pages = max(last) // P + 2
    slots = torch.randperm(n + 1, generator=cpu)[:n]
    tables = torch.full((n + 1, max_pages), -1, dtype=torch.int32)
    need = sum((p // P + 1) - s // P for p, s in zip(last, shared)) + sum(s // P for _, s in set(zip(part, shared)))
    free = torch.randperm(need + 3, generator=cpu).to(torch.int32)
    at, common = 0, {}
    for i in range(n):
        k, whole = shared[i] // P, last[i] // P + 1
        if part[i] not in common:
            common[part[i]] = free[at:at + k]
            at += k
        tables[slots[i], :k] = common[part[i]]
        tables[slots[i], k:whole] = free[at:at + whole - k]
        at += whole - k
    pads = case["pads"]
    row_slot = torch.cat([slots.to(torch.int32), torch.full((pads,), -1, dtype=torch.int32)])
    s = {"case": case, "pool": rnd((need + 3) * P, row), "tables": tables.cuda(), "row_slot": row_slot.cuda(),
         "row_pos": torch.tensor(last + [0] * pads, dtype=torch.int32).cuda()}
    if case["kind"] == "grouped":
        s["q"] = rnd(n + pads, H, case["dim"]) * 1.5
        s["gate"] = torch.randn(n + pads, H, generator=gen, device="cuda")
    else:
        q = rnd(n + pads, H, case["dim"]) * 1.5
        s["q_abs"], s["q_rot"] = q[..., :case["vdim"]].contiguous(), q[..., case["vdim"]:].contiguous()
        s["sink"] = torch.randn(H, generator=gen, device="cuda") * 0.5
    s["out"] = torch.empty(n + pads, H, case["vdim"], dtype=dt, device="cuda")
    # the pass's rows by common part; a program that keeps such pages knows whom it gave them to
    s["groups"] = []
    for j in sorted(set(part)):
        rows = [i for i in range(n) if part[i] == j]
        s["groups"].append((torch.tensor(rows, device="cuda"), shared[rows[0]], max(last[i] for i in rows) + 1))
    if own:
        from ds41rt_b200.ops import prefix
        # workspace; the division of a pass's work is a part of the pass.  A program keeps its page table on the host, too
        s["plan"] = prefix.PrefixPlan(case["kind"], rows=n + pads, heads=H, kv_heads=case["kv_heads"], vdim=case["vdim"],
                                      page_tokens=P, device="cuda", dtype=dt)
        s["host"] = (row_slot.tolist(), tables)
    return s


def _scale(case):
    return (192 if case["kind"] == "latent" else case["dim"]) ** -0.5


def _split(case, rows):
    """Cache rows [..., row] -> keys [..., kv_heads, dim], values [..., kv_heads, vdim]."""
    if case["kind"] == "latent":
        return rows.unsqueeze(-2), rows[..., None, :case["vdim"]]
    G, D = case["kv_heads"], case["dim"]
    return rows[..., :G * D].unflatten(-1, (G, D)), rows[..., G * D:].unflatten(-1, (G, case["vdim"]))


# ---------------------------------------------------------------------------------------------------- one pass
def _plain_rows(s, rows, shared, end):
    """The rows of one common part of `shared` tokens: scores against its keys in one product, against their own keys (up to position
    `end`) in another."""
    case, P = s["case"], s["case"]["page"]
    q = s["q"] if case["kind"] == "grouped" else torch.cat([s["q_abs"], s["q_rot"]], -1)
    q = q[rows].float().unflatten(1, (case["kv_heads"], -1))                               # [b, g, n, d]
    table, pos = s["tables"][s["row_slot"][rows].long()].long(), s["row_pos"][rows].long()
    first = pos - pos % case["chunk"] if case["chunk"] else torch.zeros_like(pos)
    at = torch.arange(shared, device="cuda")
    k, v = _split(case, s["pool"][table[0, at // P] * P + at % P].float())
    far = torch.einsum("bgnd,kgd->bgnk", q, k) * _scale(case)
    far = far.masked_fill((at[None] < first[:, None])[:, None, None], -math.inf)
    at = torch.arange(shared, end, device="cuda")
    page = table[:, at // P].clamp(min=0)
    mk, mv = _split(case, s["pool"][page * P + at % P].float())
    near = torch.einsum("bgnd,bkgd->bgnk", q, mk) * _scale(case)
    near = near.masked_fill(((at[None] < first[:, None]) | (at[None] > pos[:, None]))[:, None, None], -math.inf)
    z = torch.cat([far, near], -1)
    top = z.amax(-1, keepdim=True)
    sink = None
    if case["kind"] == "latent":
        sink = s["sink"].view(1, 1, -1, 1)
        top = torch.maximum(top, sink)
    w = torch.exp(z - top)
    den = w.sum(-1, keepdim=True) + (0 if sink is None else torch.exp(sink - top))
    o = torch.einsum("bgnk,kgv->bgnv", w[..., :shared], v) + torch.einsum("bgnk,bkgv->bgnv", w[..., shared:], mv)
    return (o / den).flatten(1, 2)


def run(s):
    case = s["case"]
    if own:
        from ds41rt_b200.ops import prefix
        s["plan"].set(*s["host"])
        if case["kind"] == "grouped":
            return prefix.group_attend(s["q"], s["pool"], s["tables"], s["row_pos"], s["row_slot"], s["plan"], scale=_scale(case),
                                       chunk=case["chunk"], gate=s["gate"], out=s["out"])
        return prefix.latent_attend(s["q_abs"], s["q_rot"], s["pool"], s["tables"], s["row_pos"], s["row_slot"], s["plan"],
                                    scale=_scale(case), sink=s["sink"], out=s["out"])
    out = torch.zeros(s["out"].shape, device="cuda")
    for rows, shared, end in s["groups"]:
        out[rows] = _plain_rows(s, rows, shared, end)
    if case["kind"] == "grouped":
        out = out / (1 + torch.exp(-s["gate"]))[..., None]
    return out.to(s["out"].dtype)


def exact(case, seed):
    """Every request by itself over its own page table, in 64 bits."""
    s = prepare(case, seed)
    P, G, H, V = case["page"], case["kv_heads"], case["heads"], case["vdim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for i, (slot, pos) in enumerate(zip(s["row_slot"].tolist(), s["row_pos"].tolist())):
        if slot < 0:
            continue
        places = torch.arange(_first(case, pos), pos + 1, device="cuda")
        rows = s["pool"][s["tables"][slot].long()[places // P] * P + places % P].double()
        for g in range(G):
            heads = slice(g * H // G, (g + 1) * H // G)
            if case["kind"] == "grouped":
                query = s["q"][i, heads].double()
                keys = rows[:, g * case["dim"]:(g + 1) * case["dim"]]
                values = rows[:, G * case["dim"] + g * V:G * case["dim"] + (g + 1) * V]
            else:
                query = torch.cat([s["q_abs"][i], s["q_rot"][i]], -1).double()
                keys, values = rows, rows[:, :V]
            logits = query @ keys.T * _scale(case)
            if case["kind"] == "latent":
                logits = torch.cat([logits, s["sink"].double()[:, None]], 1)
            share = torch.softmax(logits, 1)[:, :len(places)] @ values
            if case["kind"] == "grouped":
                share = share * torch.sigmoid(s["gate"][i, heads].double())[:, None]
            out[i, heads] = share
    return out
