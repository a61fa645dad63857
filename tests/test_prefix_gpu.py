"""Attention over a shared prefix against its definition in 64 bits, row by row over the row's own page table.

Tolerances, per value, from the arithmetic (u = 2^-8 for bf16, 2^-24 for fp32: a rounding's largest relative error; w, v: the
row's attention weights and values, A = sum w |v|):
  scores   a product of D fp32 terms is off by at most (D + 2) 2^-23 sum |q k| (tensor cores may truncate: one bit more than a
           rounding each), scaled; a weight by twice that, relative, as its denominator moves too: 2 d A with d the largest over keys
  weights  bf16: rounded as the operand of the second product, u A; the exponential is good to 2^-21: 2^-20 A with the denominator
  sums     n fp32 terms: n 2^-23 A, twice for the denominator; joining `parts` parts: inside that
  result   u |o| of the rounding that it leaves with
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def prefix():
    from ds41rt_b200.ops import prefix as m
    return m


class Pass:
    """A random pass: rows over prefixes of `pages` whole pages (one entry per prefix), then own tokens."""

    def __init__(self, kind, *, heads, kv_heads=1, dim, vdim, groups, P=64, alone=0, pads=0, own=70, chunk=0, dtype=BF16, seed=0,
                 per_slot=1, poison=False, sharp=1.5, early=False):
        rng, gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.kind, self.H, self.G, self.D, self.V, self.P, self.chunk, self.dtype = kind, heads, kv_heads, dim, vdim, P, chunk, dtype
        self.row = kv_heads * (dim + vdim) if kind == "grouped" else dim
        lead, slots = [], 0
        for rows, pages in groups:
            lead += [(slots, pages)] * rows
            slots += 1
        lead += [(-1 - i, 0) for i in range(alone)]
        n = len(lead)
        ids = list(range(3000))
        rng.shuffle(ids)
        take = iter(ids)
        common = {g: [next(take) for _ in range(pages)] for g, pages in set(lead)}
        length = [pages * P + rng.randint(0 if pages and not early else 1, own) for _, pages in lead]
        if early:                                     # rows that stand inside the prefix themselves
            length = [max(1, rng.randint(1, max(1, pages * P + own))) for _, pages in lead]
        width = max(max((x + own) // P + 2, p + 1) for x, (_, p) in zip(length, lead)) + 1
        self.slot_ids = rng.sample(range(n + 2), n)
        self.tables = torch.full((n + 2, width), -1, dtype=torch.int32)
        rows = []
        for s, (g, pages), m in zip(self.slot_ids, lead, length):
            need = max(pages, (m + per_slot - 1) // P + 1)
            row = common[g] + [next(take) for _ in range(need - pages)]
            self.tables[s, :need] = torch.tensor(row, dtype=torch.int32)
            rows += [(s, m + i) for i in range(per_slot)]
        blocks = [rows[i:i + per_slot] for i in range(0, len(rows), per_slot)]
        rng.shuffle(blocks)                           # rows of a slot stay adjacent, slots stand in any order
        rows = [r for b in blocks for r in b]
        for _ in range(pads):
            rows.insert(rng.choice(range(0, len(rows) + 1, per_slot)), (-1, rng.randint(0, 50)))
        self.R = len(rows)
        self.row_slot = [s for s, _ in rows]
        self.row_pos = [p for _, p in rows]
        self.pages = int(self.tables.max()) + 2
        rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")
        self.pool = rnd(self.pages * P, self.row).to(dtype)
        if poison:                                    # what no row sees may be anything
            seen = torch.zeros(self.pages * P, dtype=torch.bool)
            for s, p in rows:
                if s >= 0:
                    at = torch.arange(p + 1)
                    seen[self.tables[s].long()[at // P] * P + at % P] = True
            bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
            hidden = (~seen).nonzero().flatten().cuda()
            self.pool[hidden] = bad[hidden % 3][:, None].to(dtype)
        self.q = (rnd(self.R, heads, dim) * sharp).to(dtype)
        self.gate, self.sink = rnd(self.R, heads), rnd(heads)
        self.scale = dim ** -0.5
        self.dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.d_tables, self.d_pos, self.d_slot = self.tables.cuda(), self.dev(self.row_pos), self.dev(self.row_slot)

    def plan(self, rows=None, **kw):
        plan = prefix().PrefixPlan(self.kind, rows=rows or self.R, heads=self.H, kv_heads=self.G, vdim=self.V, page_tokens=self.P,
                                   device="cuda", dtype=self.dtype, **kw)
        plan.set(self.row_slot, self.tables)
        return plan

    def run(self, plan, gate=True, **kw):
        a = (self.pool, self.d_tables, self.d_pos, self.d_slot, plan)
        if self.kind == "grouped":
            return prefix().group_attend(self.q, *a, scale=self.scale, chunk=self.chunk, gate=self.gate if gate else None, **kw)
        q_rot = self.q[..., self.V:].contiguous() if self.D > self.V else None
        return prefix().latent_attend(self.q[..., :self.V].contiguous(), q_rot, *a, scale=self.scale, sink=self.sink if gate else None, **kw)

    def expected(self, gate=True):
        """(values, tolerances) in 64 bits."""
        u = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24
        out = torch.zeros(self.R, self.H, self.V, dtype=torch.float64, device="cuda")
        tol = torch.full_like(out, 1e-300)
        for r, (s, p) in enumerate(zip(self.row_slot, self.row_pos)):
            if s < 0:
                continue
            lo = p - p % self.chunk if self.chunk else 0
            at = torch.arange(lo, p + 1)
            x = self.pool[(self.tables[s].long()[at // self.P] * self.P + at % self.P).cuda()].double()
            for g in range(self.G):
                hs = slice(g * self.H // self.G, (g + 1) * self.H // self.G)
                q = self.q[r, hs].double()
                if self.kind == "grouped":
                    k = x[:, g * self.D:(g + 1) * self.D]
                    v = x[:, self.G * self.D + g * self.V:self.G * self.D + (g + 1) * self.V]
                else:
                    k, v = x, x[:, :self.V]
                z = q @ k.T * self.scale
                d = ((q.abs() @ k.abs().T).amax(1) * self.scale * (self.D + 2) * 2.0 ** -23)[:, None]
                if self.kind == "latent" and gate:
                    z = torch.cat([z, self.sink[hs].double()[:, None]], 1)
                w = torch.softmax(z, 1)[:, :len(at)]
                o, A = w @ v, w @ v.abs()
                t = (2 * d * (1 + d) + 2.0 ** -20 + 2 * len(at) * 2.0 ** -23 + (u if self.dtype == BF16 else 0)) * A
                if self.kind == "grouped" and gate:
                    f = torch.sigmoid(self.gate[r, hs].double())[:, None]
                    o, t = o * f, (t + 2.0 ** -21 * o.abs()) * f
                out[r, hs], tol[r, hs] = o, t + u * (o.abs() + t) + 1e-30
        return out, tol

    def check(self, plan=None, gate=True, **kw):
        plan = plan or self.plan()
        got = self.run(plan, gate, **kw)
        torch.cuda.synchronize()
        plan.check_status()
        want, tol = self.expected(gate)
        far = (got.double() - want).abs() / tol
        worst = float(far.max())
        assert worst <= 1 and torch.isfinite(got).all(), (worst, (far > 1).nonzero()[:5].tolist(), got.isnan().sum().item())
        return got


GROUPED = [
    dict(heads=16, kv_heads=4, dim=128, vdim=128, groups=[(4, 4)]),
    dict(heads=32, kv_heads=8, dim=128, vdim=128, groups=[(33, 20)], own=200),
    dict(heads=32, kv_heads=8, dim=128, vdim=128, groups=[(70, 9)], P=128),
    dict(heads=6, kv_heads=2, dim=32, vdim=48, groups=[(9, 30), (7, 3), (2, 1)], P=32, alone=3, pads=2),
    dict(heads=8, kv_heads=8, dim=64, vdim=64, groups=[(5, 7)], pads=1),
    dict(heads=12, kv_heads=1, dim=64, vdim=64, groups=[(25, 11)], alone=1),
    dict(heads=20, kv_heads=4, dim=192, vdim=128, groups=[(13, 6)]),
    dict(heads=4, kv_heads=2, dim=256, vdim=256, groups=[(6, 5)]),
    dict(heads=4, kv_heads=2, dim=128, vdim=256, groups=[(6, 5)]),
    dict(heads=4, kv_heads=2, dim=16, vdim=16, groups=[(3, 40)], P=8),
    dict(heads=4, kv_heads=2, dim=80, vdim=112, groups=[(3, 3)], P=256),
    dict(heads=4, kv_heads=2, dim=64, vdim=64, groups=[(5, 9)], P=48),
    dict(heads=40, kv_heads=1, dim=64, vdim=64, groups=[(9, 9)]),
    dict(heads=160, kv_heads=1, dim=64, vdim=64, groups=[(3, 9)]),
    dict(heads=8, kv_heads=2, dim=64, vdim=64, groups=[(30, 12)], chunk=256, own=300),
    dict(heads=8, kv_heads=2, dim=64, vdim=64, groups=[(30, 12)], chunk=100, own=300, P=32),
    dict(heads=8, kv_heads=2, dim=64, vdim=64, groups=[(20, 12)], early=True),
    dict(heads=8, kv_heads=2, dim=64, vdim=64, groups=[(12, 12)], per_slot=3),
    dict(heads=16, kv_heads=4, dim=128, vdim=128, groups=[(6, 7)], dtype=F32),
    dict(heads=6, kv_heads=2, dim=32, vdim=48, groups=[(5, 9), (3, 4)], P=32, alone=2, pads=1, dtype=F32, chunk=96),
    dict(heads=2, kv_heads=2, dim=512, vdim=512, groups=[(3, 3)], dtype=F32),
]
LATENT = [
    dict(heads=16, dim=576, vdim=512, groups=[(4, 4)]),
    dict(heads=32, dim=576, vdim=512, groups=[(33, 20)], own=200),
    dict(heads=32, dim=576, vdim=512, groups=[(21, 9)], P=128),
    dict(heads=16, dim=576, vdim=512, groups=[(9, 30), (7, 3), (2, 1)], P=32, alone=3, pads=2),
    dict(heads=5, dim=96, vdim=64, groups=[(19, 12)], P=32, pads=2),
    dict(heads=8, dim=320, vdim=256, groups=[(30, 8)]),
    dict(heads=4, dim=96, vdim=64, groups=[(40, 3)], P=8),
    dict(heads=3, dim=528, vdim=448, groups=[(6, 5)], P=48),
    dict(heads=128, dim=576, vdim=512, groups=[(3, 9)]),
    dict(heads=130, dim=96, vdim=64, groups=[(3, 9)]),
    dict(heads=16, dim=128, vdim=128, groups=[(5, 9)]),
    dict(heads=2, dim=656, vdim=592, groups=[(5, 3)]),
    dict(heads=16, dim=576, vdim=512, groups=[(20, 12)], early=True),
    dict(heads=16, dim=576, vdim=512, groups=[(12, 12)], per_slot=3),
    dict(heads=16, dim=576, vdim=512, groups=[(6, 7)], dtype=F32),
    dict(heads=5, dim=96, vdim=64, groups=[(5, 9), (3, 4)], P=32, alone=2, pads=1, dtype=F32),
]


@pytest.mark.parametrize("i", range(len(GROUPED)))
def test_grouped(i):
    Pass("grouped", seed=i, **GROUPED[i]).check()


@pytest.mark.parametrize("i", range(len(LATENT)))
def test_latent(i):
    Pass("latent", seed=100 + i, **LATENT[i]).check()


SMALL = {"grouped": dict(heads=8, kv_heads=2, dim=64, vdim=64), "latent": dict(heads=8, dim=192, vdim=128)}
KINDS = ("grouped", "latent")


@pytest.mark.parametrize("kind", KINDS)
def test_hidden_places_may_hold_anything(kind):
    Pass(kind, groups=[(9, 5), (3, 2)], alone=1, pads=1, poison=True, own=150, **SMALL[kind]).check()


@pytest.mark.parametrize("rows", [2, 20, 60])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_inside_a_prefix_do_not_see_what_follows_them(kind, rows):
    """Shared pages whose last positions nobody stands behind yet."""
    for seed in range(4):
        Pass(kind, groups=[(rows, 9), (3, 4)], early=True, poison=True, seed=seed, P=(64, 32, 128, 16)[seed], **SMALL[kind]).check()
    Pass(kind, groups=[(rows, 9)], early=True, poison=True, dtype=F32, **SMALL[kind]).check()
    if kind == "grouped":
        Pass(kind, groups=[(rows, 9)], early=True, poison=True, chunk=200, **SMALL[kind]).check()


# rings of one to eight tiles, blocks that come to the list many times, walks that several pieces of a range share
DEPTHS = [("grouped", dict(heads=8, kv_heads=4, dim=256, vdim=128, groups=[(9, 12)], own=200)),
          ("grouped", dict(heads=8, kv_heads=4, dim=256, vdim=64, groups=[(9, 12)], own=200)),
          ("grouped", dict(heads=8, kv_heads=4, dim=16, vdim=32, groups=[(9, 12)], own=200)),
          ("grouped", dict(heads=32, kv_heads=8, dim=64, vdim=64, groups=[(130, 2), (60, 1), (40, 3)], own=80)),
          ("grouped", dict(heads=32, kv_heads=8, dim=128, vdim=128, groups=[(150, 3)], own=80, P=16)),
          ("grouped", dict(heads=32, kv_heads=4, dim=128, vdim=128, groups=[(64, 40)], own=30, P=32, chunk=700)),
          ("grouped", dict(heads=32, kv_heads=32, dim=64, vdim=64, groups=[(40, 2)], own=300)),
          ("latent", dict(heads=64, dim=576, vdim=512, groups=[(100, 2), (60, 1)], own=80)),
          ("latent", dict(heads=16, dim=64, vdim=64, groups=[(150, 3)], own=300, P=16))]


@pytest.mark.parametrize("i", range(len(DEPTHS)))
def test_many_units_and_rings_of_every_depth(i):
    kind, kw = DEPTHS[i]
    Pass(kind, seed=200 + i, **kw).check()


@pytest.mark.parametrize("kind", KINDS)
def test_scores_that_differ_widely(kind):
    """Scores of hundreds: parts whose weights vanish beside another part's, and a running maximum that grows late."""
    for seed in range(3):
        Pass(kind, groups=[(10, 9)], own=200, sharp=60.0, seed=seed, **SMALL[kind]).check()


@pytest.mark.parametrize("chunk,P", [(256, 64), (100, 32), (1000, 16)])
def test_plans_that_leave_out_earlier_chunks(chunk, P):
    p = Pass("grouped", groups=[(20, 700 // P), (5, 90 // P)], alone=2, pads=1, own=600, chunk=chunk, P=P, **SMALL["grouped"])
    plan = p.plan(chunk=chunk)
    p.check(plan)
    plan.set(p.row_slot, p.tables, [x + 1 for x in p.row_pos])
    p.check(plan)
    p.row_pos = [x + 1 if x // P == (x + 1) // P else x for x in p.row_pos]         # where the page is leased
    p.d_pos = p.dev(p.row_pos)
    p.check(plan)
    with pytest.raises(ValueError, match="chunk of"):
        p.chunk = 0
        p.run(plan)


@pytest.mark.parametrize("kind", KINDS)
def test_without_gate_or_sink(kind):
    Pass(kind, groups=[(5, 6)], **SMALL[kind]).check(gate=False)


@pytest.mark.parametrize("kind", KINDS)
def test_nothing_shared_and_no_rows_alive(kind):
    Pass(kind, groups=[], alone=4, **SMALL[kind]).check()
    Pass(kind, groups=[(1, 4)], **SMALL[kind]).check()
    p = Pass(kind, groups=[(3, 4)], **SMALL[kind])
    p.row_slot = [-1] * p.R
    p.d_slot = p.dev(p.row_slot)
    assert not p.check().any()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_beyond_the_pass_and_strided_arguments(kind):
    p = Pass(kind, groups=[(7, 6)], **SMALL[kind])
    want = p.run(p.plan())
    m, R, H, V = prefix(), p.R, p.H, p.V
    plan = p.plan(rows=R + 9)
    wide = torch.full((R + 3, H * V + 24), 7.0, dtype=BF16, device="cuda")
    out = wide[:R, 8:8 + H * V].unflatten(1, (H, V))
    a = (p.pool, p.d_tables, p.d_pos, p.d_slot, plan)
    if kind == "grouped":
        q = torch.randn(R, H * p.D + 40, device="cuda").to(BF16)
        q[:, 16:16 + H * p.D] = p.q.flatten(1)
        gate = torch.randn(R, H + 5, device="cuda")
        gate[:, 2:2 + H] = p.gate
        m.group_attend(q[:, 16:16 + H * p.D].unflatten(1, (H, p.D)), *a, scale=p.scale, gate=gate[:, 2:2 + H], out=out)
    else:
        both = torch.randn(R, H, p.D + 8, device="cuda").to(BF16)
        both[..., 8:] = p.q
        qa = torch.randn(R, H * V + 16, device="cuda").to(BF16)
        qa[:, 16:] = p.q[..., :V].flatten(1)
        m.latent_attend(qa[:, 16:].unflatten(1, (H, V)), both[..., 8 + V:], *a, scale=p.scale, sink=p.sink, out=out)
    assert torch.equal(out, want)
    assert (wide[R:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 8 + H * V:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,groups,alone", [(1, [], 1), (1, [(3, 4)], 0), (8, [], 1)])
def test_one_row_or_one_head_with_any_stride(kind, heads, groups, alone):
    """A dimension of one entry has no neighbour: its stride means nothing."""
    p = Pass(kind, heads=heads, dim=64, vdim=64 if kind == "grouped" else 48, groups=groups, alone=alone)
    plan, (R, H, V) = p.plan(), (p.R, p.H, p.V)
    want, tol = p.expected()
    odd = lambda t: t.as_strided(t.shape, tuple(s if n > 1 else 12345 + 2 * k for k, (n, s) in enumerate(zip(t.shape, t.stride()))))
    a, out = (p.pool, p.d_tables, p.d_pos, p.d_slot, plan), odd(torch.empty(R, H, V, dtype=BF16, device="cuda"))
    if kind == "grouped":
        prefix().group_attend(odd(p.q), *a, scale=p.scale, gate=odd(p.gate), out=out)
    else:
        prefix().latent_attend(odd(p.q[..., :V].contiguous()), odd(p.q[..., V:].contiguous()), *a, scale=p.scale, sink=p.sink, out=out)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_repeated_calls_agree_bit_for_bit(kind, dtype):
    p = Pass(kind, groups=[(9, 8)], dtype=dtype, **SMALL[kind])
    plan = p.plan()
    first = p.run(plan)
    for _ in range(5):
        assert torch.equal(p.run(plan), first)
    assert torch.equal(p.run(p.plan()), first)


@pytest.mark.parametrize("kind", KINDS)
def test_captured_calls_follow_the_plan_and_the_rows(kind):
    """A graph that was captured while nothing was shared serves a batch that shares, other rows, and nothing shared again."""
    a = Pass(kind, groups=[], alone=12, own=500, seed=1, **SMALL[kind])
    b = Pass(kind, groups=[(8, 7), (4, 3)], own=60, seed=2, **SMALL[kind])
    c = Pass(kind, groups=[(11, 2)], alone=1, own=300, seed=3, **SMALL[kind])
    width, slots = max(x.tables.shape[1] for x in (a, b, c)), max(x.tables.shape[0] for x in (a, b, c))
    pages = max(x.pages for x in (a, b, c))
    for x in (a, b, c):                                # one cache for the three passes
        t = torch.full((slots, width), -1, dtype=torch.int32)
        t[:x.tables.shape[0], :x.tables.shape[1]] = x.tables
        x.tables = t
        pool = torch.zeros(pages * x.P, x.row, dtype=BF16, device="cuda")
        pool[:x.pool.shape[0]] = x.pool
        x.pool = pool
    live = Pass(kind, groups=[], alone=12, own=500, seed=1, **SMALL[kind])
    live.tables, live.pool, live.d_tables = a.tables, a.pool.clone(), a.tables.cuda()
    plan = a.plan()
    out = torch.empty(12, live.H, live.V, dtype=BF16, device="cuda")
    qa, qr = live.q[..., :live.V].contiguous(), live.q[..., live.V:].contiguous()

    def enqueue():
        args = (live.pool, live.d_tables, live.d_pos, live.d_slot, plan)
        if kind == "grouped":
            prefix().group_attend(live.q, *args, scale=live.scale, gate=live.gate, out=out)
        else:
            prefix().latent_attend(qa, qr, *args, scale=live.scale, sink=live.sink, out=out)

    enqueue()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        enqueue()
    for x in (b, a, c, b):
        for name in ("pool", "d_pos", "d_slot", "q", "gate", "sink"):
            getattr(live, name).copy_(getattr(x, name))
        live.d_tables.copy_(x.tables)
        qa.copy_(x.q[..., :live.V])
        qr.copy_(x.q[..., live.V:])
        plan.set(x.row_slot, x.tables)
        g.replay()
        torch.cuda.synchronize()
        plan.check_status()
        want, tol = x.expected()
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_with_a_plan_each(kind):
    a, b = (Pass(kind, groups=[(9, 12)], seed=s, **SMALL[kind]) for s in (1, 2))
    pa, pb = a.plan(), b.plan()
    wa, wb = a.run(pa), b.run(pb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            ga = a.run(pa)
        with torch.cuda.stream(s2):
            gb = b.run(pb)
        torch.cuda.synchronize()
        assert torch.equal(ga, wa) and torch.equal(gb, wb)


@pytest.mark.parametrize("kind", KINDS)
def test_a_step_of_both_operators_in_turn(kind):
    """Growing contexts under one plan: every step writes a cache row per request and attends, as a decode loop does."""
    p = Pass(kind, groups=[(6, 5), (3, 2)], alone=1, own=40, **SMALL[kind])
    plan = p.plan()
    for step in range(3):
        p.row_pos = [x + 7 for x in p.row_pos]
        for r, (s, pos) in enumerate(zip(p.row_slot, p.row_pos)):
            while p.tables[s, pos // p.P] < 0:         # a page at the table's end leaves the plan as it is
                k = int((p.tables[s] < 0).nonzero()[0])
                p.tables[s, k] = p.pages
                p.pages += 1
        extra = torch.randn(p.pages * p.P - p.pool.shape[0], p.row, device="cuda").to(p.dtype)
        p.pool = torch.cat([p.pool, extra])
        p.d_pos, p.d_tables = p.dev(p.row_pos), p.tables.cuda()
        p.check(plan)
