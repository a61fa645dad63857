"""A pass of several requests with several new tokens each, by which the operators of ds41rt_b200.ops.ragged are followed.

A server that batches continuously runs prompts' portions and decode rows in one pass: request i brings `new` tokens, stands at
`length` tokens with them and keeps its keys and values in the pages of its slot.  Of such a pass

  "describe": positions, slots and cache rows of all new tokens, from the requests' lengths on the GPU;
  "heads":    RMS norm of every query and key head, rotation by position, keys and values into their cache rows;
  "attend":   grouped-query attention of the new tokens over the paged cache: everything before them, or a window of positions and a
              few first tokens that stay visible; a sigmoid gate and an extra logit per head where a model has them.  The pass's
              description is a part of it;
  "layer":    the three, one after the other, as a layer of a model has them.

A case names the pass: `decodes` requests with one new token and `prompts` with up to `new`, over up to `context` earlier tokens; `idle`
requests bring nothing, `apart` ones have no slot, and `pads` rows lie behind the last request's.  Lengths follow from a request's number,
pages and values from the seed.
"""
from __future__ import annotations

import math

import torch

own = False


# ---------------------------------------------------------------------------------------------------- the cases
def _case(name, kind, decodes=0, prompts=0, new=1, context=0, heads=32, kv_heads=8, dim=128, vdim=128, rot=128, page=64, window=0,
          first=0, gate=False, sink=False, idle=0, apart=0, pads=0, dtype="bf16"):
    return {"name": name, "kind": kind, "decodes": decodes, "prompts": prompts, "new": new, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "rot": rot, "page": page, "window": window, "first": first, "gate": gate,
            "sink": sink, "idle": idle, "apart": apart, "pads": pads, "dtype": dtype}


def listed():
    return [
        # a decode step's rows: the smallest call, of launches only
        _case("describe 4 decodes", "describe", decodes=4, context=300),
        # a full batch: prompts' portions of every length among decode rows, requests without tokens, rows behind the last
        _case("describe 200 + 40 x 500", "describe", decodes=200, prompts=40, new=500, context=20000, idle=7, apart=2, pads=100),
        # queries and keys of a decode step
        _case("heads 16 decodes", "heads", decodes=16, context=4000),
        # a prompt's portion of 8192 tokens
        _case("heads 8192", "heads", prompts=1, new=8192, context=40000),
        # odd heads, a rotation of a part of the head, 32 bits
        _case("heads 5 x 199 f32", "heads", prompts=5, new=199, context=777, heads=6, kv_heads=2, dim=32, vdim=48, rot=16, page=32,
              apart=1, pads=3, dtype="f32"),
        # few short requests: latency
        _case("attend 4 x 300", "attend", decodes=4, context=300, heads=16, kv_heads=4, gate=True),
        # a server's decode step over long contexts: every key once
        _case("attend 64 x 8192", "attend", decodes=64, context=8192),
        # the same in a model with windows, whose requests are long: first tokens and a window of each
        _case("attend 200 x 30000 window", "attend", decodes=200, context=30000, window=1024, first=4, sink=True),
        # portions of prompts beside decode rows
        _case("attend 60 + 12 x 300 mixed", "attend", decodes=60, prompts=12, new=300, context=6000, heads=16, kv_heads=4, page=32,
              idle=2, apart=1, pads=9, gate=True),
        # a long prompt at once
        _case("attend 8192", "attend", prompts=1, new=8192),
        # 32 bits, odd heads
        _case("attend 3 + 2 x 50 f32", "attend", decodes=3, prompts=2, new=50, context=500, heads=6, kv_heads=2, dim=32, vdim=48,
              window=200, first=2, gate=True, dtype="f32"),
        # a layer's share of a pass with a window
        _case("layer 30 + 3 x 2000 window", "layer", decodes=30, prompts=3, new=2000, context=5000, window=2048, first=16),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, size = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        kind = rng.choice(["describe", "heads", "heads", "attend", "attend", "attend", "attend", "layer"])
        dtype = "f32" if rng.random() < 0.15 else "bf16"
        small = dtype == "f32" and kind != "heads"
        heads, kv_heads = rng.choice([(16, 4), (32, 8), (32, 8), (6, 2), (8, 8), (12, 1), (20, 4)])
        dim, vdim, rot = rng.choice([(128, 128, 128), (128, 128, 128), (128, 128, 64), (64, 64, 64), (32, 48, 16), (192, 128, 64)])
        windowed = rng.random() < 0.5
        decodes, prompts = rng.choice([(1, 0), (0, 1), (1, 1), (1, 1)])
        c = _case("", kind, decodes=decodes * _spread(rng, 1, 16 if small else 200), prompts=prompts * _spread(rng, 1, 4 if small else 40),
                  new=_spread(rng, 2, 100 if small else 8192), context=_spread(rng, 1, 1000 if small else 30000), heads=heads,
                  kv_heads=kv_heads, dim=dim, vdim=vdim, rot=rot, page=rng.choice([16, 32, 64, 64, 128]),
                  window=_spread(rng, 16, 4096) if windowed else 0, first=rng.choice([0, 1, 4, 16, 100]) if windowed else 0,
                  gate=rng.random() < 0.5, sink=rng.random() < 0.3, idle=rng.choice([0, 0, 1, 5]), apart=rng.choice([0, 0, 1]),
                  pads=rng.choice([0, 0, 1, 50]), dtype=dtype)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= size and sum(_layout(c)[1]) <= 16384:
            del c["name"]
            return c


# ---------------------------------------------------------------------------------------------------- what a pass looks like
def _part(i):
    return 1 - ((i * 37) % 64) / 128


def _layout(case):
    """Of every request: whether it has a slot, how many new tokens, and its length with them."""
    leased, new, length = [], [], []
    for i in range(case["decodes"] + case["prompts"]):
        n = 1 if i < case["decodes"] else max(1, round(case["new"] * _part(i - case["decodes"])))
        leased.append(True)
        new.append(n)
        length.append(n + int(case["context"] * _part(3 * i)))
    for j in range(case["idle"]):
        at = (5 * j + 1) % (len(new) + 1)
        for lst, x in ((leased, True), (new, 0), (length, 40 * j)):
            lst.insert(at, x)
    for j in range(case["apart"]):
        at = (3 * j + 2) % (len(new) + 1)
        for lst, x in ((leased, False), (new, 2 + j), (length, 9)):
            lst.insert(at, x)
    return leased, new, length


def _ranges(case, p0, p1):
    """Positions that some of the rows at p0 .. p1 see: those of the first tokens that lie before the window, and the rest."""
    low = max(0, p0 - case["window"] + 1) if case["window"] else 0
    return min(case["first"], low), low, p1 + 1


def work(case):
    leased, new, length = _layout(case)
    size = 2 if case["dtype"] == "bf16" else 4
    H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    rows, n = sum(x for x, l in zip(new, leased) if l), len(new)
    describe = {"bytes": 12 * n + 4 * n + 12 * (sum(new) + case["pads"]), "flops": 4 * rows}
    values = rows * ((H + G) * D + G * V)
    heads = {"bytes": 2 * size * values + 8 * rows, "flops": 8 * values}
    keys = pairs = 0
    for l, x, total in zip(leased, new, length):
        if l and x:
            a, low, end = _ranges(case, total - x, total - 1)
            keys += a + end - low
            if not case["window"]:
                pairs += x * (2 * (total - x) + x + 1) // 2
            else:
                for p in range(total - x, total):
                    b, lo, e = _ranges(case, p, p)
                    pairs += b + e - lo
    attend = {"bytes": size * (keys * G * (D + V) + rows * H * (D + V)) + (4 * rows * H if case["gate"] else 0),
              "flops": 2 * H * (D + V) * pairs}
    parts = {"describe": [describe], "heads": [heads], "attend": [describe, attend], "layer": [describe, heads, attend]}[case["kind"]]
    return {k: sum(p[k] for p in parts) for k in ("bytes", "flops")}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    leased, new, length = _layout(case)
    n, P, H, G, D, V = len(new), case["page"], case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    R = sum(new) + case["pads"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    order = torch.randperm(n + 1, generator=cpu)[:n].tolist()
    slots = [s if l else -1 for s, l in zip(order, leased)]
    width = max(length) // P + 2
    tables = torch.full((n + 1, width), -1, dtype=torch.int32)
    need = [-(-t // P) if l else 0 for t, l in zip(length, leased)]
    pages = sum(need) + 3
    free, at = torch.randperm(pages, generator=cpu).to(torch.int32), 0
    for s, k in zip(slots, need):
        if s >= 0:
            tables[s, :k] = free[at:at + k]
            at += k
    s = {"case": case, "rows": R, "slots": i32(slots), "new": i32(new), "lengths": i32(length), "tables": tables.cuda(), "pages": pages,
         "host": (slots, new, length)}
    if case["kind"] == "describe":
        return s
    # the rows' values as a projection leaves them: queries, keys and values of all heads side by side
    s["pool"] = rnd(pages * P, G * (D + V))
    if case["kind"] in ("heads", "layer"):
        s["qkv"] = rnd(R, (H + G) * D + G * V)
        s["q_norm"], s["k_norm"] = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda") for _ in range(2))
        s["freq"] = 500000.0 ** -(torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float32) * 2 / case["rot"])
        s["q_out"] = rnd(R, H, D)
    else:
        s["q"] = rnd(R, H, D) * 1.5
    if case["kind"] != "heads":
        s["out"] = rnd(R, H, V)
        s["gate"] = torch.randn(R, H, generator=gen, device="cuda") if case["gate"] else None
        s["sink"] = torch.randn(H, generator=gen, device="cuda") if case["sink"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "heads":
        s["row_pos"], s["row_place"] = _plain_rows(s)[0::2]
    if own and case["kind"] != "heads":
        from ds41rt_b200.ops import ragged
        # the pass's arrays and workspace, which a program keeps from pass to pass
        s["pass"] = ragged.RaggedPass(rows=s["rows"], requests=len(s["host"][0]), heads=case["heads"], kv_heads=case["kv_heads"],
                                      dim=case["dim"], vdim=case["vdim"], page_tokens=case["page"], window=case["window"],
                                      first=case["first"], device="cuda",
                                      dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def _plain_rows(s):
    """Position, slot and cache row of every row."""
    P, new = s["case"]["page"], s["new"]
    end = new.long().cumsum(0)
    r = torch.arange(s["rows"], device="cuda")
    i = (r[:, None] >= end[None]).sum(1)
    live = i < len(new)
    i = i.clamp(max=len(new) - 1)
    slot = torch.where(live, s["slots"][i], -1)
    pos = torch.where(live, s["lengths"][i] - new[i] + (r - (end - new)[i]), 0)
    page = s["tables"][slot.clamp(min=0).long(), (pos // P).long()]
    place = torch.where((slot >= 0) & (page >= 0), page * P + pos % P, -1)
    return pos.int(), slot.int(), place.int()


def _plain_heads(s, pos, place):
    case = s["case"]
    H, G, D, V, half = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["rot"] // 2
    rows = (place >= 0).nonzero()[:, 0]
    x = s["qkv"][rows].float()
    angle = pos[rows].double()[:, None] * s["freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    q, k, v = x.split([H * D, G * D, G * V], 1)
    s["q_out"][rows] = turned(q.unflatten(1, (H, D)), s["q_norm"]).to(s["q_out"].dtype)
    k = turned(k.unflatten(1, (G, D)), s["k_norm"]).flatten(1)
    s["pool"][place[rows].long()] = torch.cat([k, v], 1).to(s["pool"].dtype)
    return s["q_out"]


def _plain_attend(s, q):
    case, P, out = s["case"], s["case"]["page"], s["out"]
    G, D, V, g = case["kv_heads"], case["dim"], case["vdim"], case["heads"] // case["kv_heads"]
    r0 = 0
    for slot, new, length in zip(*s["host"]):
        if slot < 0:
            out[r0:r0 + new] = 0
        for a in range(0, new if slot >= 0 else 0, 1024):
            b = min(a + 1024, new)
            pos = torch.arange(length - new + a, length - new + b, device="cuda")
            f, low, end = _ranges(case, length - new + a, length - new + b - 1)
            at = torch.cat([torch.arange(f, device="cuda"), torch.arange(low, end, device="cuda")])
            kv = s["pool"][s["tables"][slot, at // P].long() * P + at % P].float()
            k, v = kv[:, :G * D].unflatten(1, (G, D)).transpose(0, 1), kv[:, G * D:].unflatten(1, (G, V)).transpose(0, 1)
            x = q[r0 + a:r0 + b].float().unflatten(1, (G, g)).permute(1, 0, 2, 3).flatten(1, 2)        # [G, rows * g, D]
            z = (x @ k.transpose(1, 2) * D ** -0.5).unflatten(1, (b - a, g))
            seen = at[None] <= pos[:, None]
            if case["window"]:
                seen &= (at[None] > pos[:, None] - case["window"]) | (at[None] < case["first"])
            z = z.masked_fill(~seen[:, None], -math.inf)
            top = z.amax(-1, keepdim=True)
            if s["sink"] is not None:
                sink = s["sink"].view(G, 1, g, 1)
                top = torch.maximum(top, sink)
            z = torch.exp(z - top)
            den = z.sum(-1, keepdim=True)
            if s["sink"] is not None:
                den = den + torch.exp(sink - top)
            o = (z.flatten(1, 2) @ v).unflatten(1, (b - a, g)) / den
            o = o.permute(1, 0, 2, 3).flatten(1, 2)
            if s["gate"] is not None:
                o = o / (1 + torch.exp(-s["gate"][r0 + a:r0 + b]))[..., None]
            out[r0 + a:r0 + b] = o.to(out.dtype)
        r0 += new
    return out


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        from ds41rt_b200.ops import ragged
        if kind != "heads":
            rows = s["pass"].describe(s["slots"], s["new"], s["lengths"], s["tables"], s["pages"])
        if kind == "describe":
            return list(rows)
        if kind != "attend":
            H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
            q, k, v = s["qkv"].split([H * D, G * D, G * V], 1)
            pos, place = (s["row_pos"], s["row_place"]) if kind == "heads" else (rows[0], rows[2])
            ragged.heads_to_cache(q.view(-1, H, D), k.view(-1, G, D), v.view(-1, G, V), pos, place, s["pool"], q_norm=s["q_norm"],
                                  k_norm=s["k_norm"], eps=1e-6, freq=s["freq"], out=s["q_out"])
        if kind == "heads":
            return [s["q_out"], s["pool"]]
        q = s["q"] if kind == "attend" else s["q_out"]
        out = ragged.attend(q, s["pool"], s["tables"], s["pass"], scale=case["dim"] ** -0.5, sink=s["sink"], gate=s["gate"], out=s["out"])
        return [out] if kind == "attend" else [s["q_out"], s["pool"], out]
    if kind == "attend":
        return [_plain_attend(s, s["q"])]
    if kind == "describe":
        return list(_plain_rows(s))
    pos, place = (s["row_pos"], s["row_place"]) if kind == "heads" else _plain_rows(s)[0::2]
    q = _plain_heads(s, pos, place)
    return [q, s["pool"]] if kind == "heads" else [q, s["pool"], _plain_attend(s, q)]


def exact(case, seed):
    """Every request by itself, in 64 bits; what is stored in between has the type that it is stored in."""
    if case["kind"] == "describe":
        return None
    s = _inputs(case, seed)
    P, H, G, D, V = case["page"], case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    half, dt = case["rot"] // 2, s["pool"].dtype
    wide = torch.float64
    stored = s["pool"].to(wide)
    places, r0 = [], 0
    for slot, new, length in zip(*s["host"]):
        at = torch.arange(length, device="cuda")
        places.append((slot, r0, new, length, None if slot < 0 else s["tables"][slot].long()[at // P] * P + at % P))
        r0 += new
    outputs = []
    if case["kind"] != "attend":
        query = s["q_out"].to(wide)
        for slot, a, new, length, place in places:
            if slot < 0 or new == 0:
                continue
            x = s["qkv"][a:a + new].to(wide)
            turn = torch.polar(torch.ones((), dtype=wide, device="cuda"),
                               torch.arange(length - new, length, device="cuda").to(wide).outer(s["freq"].to(wide)))
            for h in range(H + G):
                y = x[:, h * D:(h + 1) * D]
                y = y * (y.square().mean(1) + 1e-6).rsqrt()[:, None] * (s["q_norm"] if h < H else s["k_norm"]).to(wide)
                c = torch.complex(y[:, :half].contiguous(), y[:, half:2 * half].contiguous()) * turn
                y = torch.cat([c.real, c.imag, y[:, 2 * half:]], 1)
                if h < H:
                    query[a:a + new, h] = y
                else:
                    stored[place[length - new:], (h - H) * D:(h - H + 1) * D] = y
            stored[place[length - new:], G * D:] = x[:, (H + G) * D:]
        outputs = [query, stored]
        if case["kind"] == "heads":
            return outputs
        query, stored = query.to(dt).to(wide), stored.to(dt).to(wide)
    else:
        query = s["q"].to(wide)
    out = s["out"].to(wide)
    for slot, a, new, length, place in places:
        out[a:a + new] = 0
        for t in range(0, new if slot >= 0 else 0, 512):
            b = min(t + 512, new)
            p = torch.arange(length - new + t, length - new + b, device="cuda")[:, None]
            lo, hi = 0, length - new + b
            if case["window"] and case["first"] == 0:
                lo = max(0, length - new + t - case["window"] + 1)
            j = torch.arange(lo, hi, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden |= (p - j >= case["window"]) & (j >= case["first"])
            rows = stored[place[lo:hi]]
            for h in range(H):
                kv = h // (H // G)
                logits = query[a + t:a + b, h] @ rows[:, kv * D:(kv + 1) * D].T / math.sqrt(D)
                logits[hidden] = -math.inf
                if s["sink"] is not None:
                    logits = torch.cat([logits, s["sink"][h].to(wide).expand(b - t, 1)], 1)
                o = torch.softmax(logits, 1)[:, :hi - lo] @ rows[:, G * D + kv * V:G * D + (kv + 1) * V]
                if s["gate"] is not None:
                    o = o * torch.sigmoid(s["gate"][a + t:a + b, h].to(wide))[:, None]
                out[a + t:a + b, h] = o
    return outputs + [out]
