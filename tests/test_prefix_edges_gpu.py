"""Attention over a shared prefix where a row's window, its numbers or its plan are out of the ordinary.

Tolerances and expected values are those of test_prefix_gpu.Pass.
"""
import math

import pytest
import torch

from test_prefix_gpu import BF16, F32, SMALL, Pass

pytestmark = pytest.mark.gpu


def poison_unseen(p):
    """NaN and infinities wherever no row of the pass sees: behind its position, and before its chunk."""
    seen = torch.zeros(p.pages * p.P, dtype=torch.bool)
    for s, pos in zip(p.row_slot, p.row_pos):
        if s >= 0:
            at = torch.arange(pos - pos % p.chunk if p.chunk else 0, pos + 1)
            seen[p.tables[s].long()[at // p.P] * p.P + at % p.P] = True
    hidden = (~seen).nonzero().flatten().cuda()
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
    p.pool[hidden] = bad[hidden % 3][:, None].to(p.dtype)
    return hidden.numel()


WIDE = dict(heads=32, kv_heads=8, dim=128, vdim=128)
ODD = dict(heads=6, kv_heads=2, dim=32, vdim=48)
CHUNKS = [
    (SMALL["grouped"], dict(chunk=96, P=64, groups=[(1, 1)], own=60)),
    (SMALL["grouped"], dict(chunk=100, P=32, groups=[(20, 9)], own=300)),
    (SMALL["grouped"], dict(chunk=100, P=32, groups=[(60, 9), (3, 2)], early=True)),
    (SMALL["grouped"], dict(chunk=200, P=64, groups=[(70, 5)], early=True, own=150)),
    (SMALL["grouped"], dict(chunk=96, P=128, groups=[(9, 3)], early=True)),
    (SMALL["grouped"], dict(chunk=40, P=256, groups=[(40, 2)], early=True)),
    (SMALL["grouped"], dict(chunk=100, P=16, groups=[(33, 20)], early=True, pads=2, alone=2)),
    (SMALL["grouped"], dict(chunk=30, P=8, groups=[(12, 30)], own=90)),
    (SMALL["grouped"], dict(chunk=50, P=64, groups=[(12, 4)], per_slot=3)),
    (SMALL["grouped"], dict(chunk=7, P=64, groups=[(130, 6)], early=True)),
    (WIDE, dict(chunk=300, P=64, groups=[(65, 12)], early=True)),
    (WIDE, dict(chunk=1000, P=64, groups=[(40, 15)], own=300)),
    (ODD, dict(chunk=96, P=32, groups=[(90, 9)], early=True, alone=3)),
    (dict(heads=8, kv_heads=8, dim=64, vdim=64), dict(chunk=100, P=64, groups=[(130, 5)], early=True)),
    (SMALL["grouped"], dict(chunk=100, P=48, groups=[(20, 5)], early=True)),
    (SMALL["grouped"], dict(chunk=100, P=32, groups=[(20, 9)], early=True, dtype=F32)),
]


@pytest.mark.parametrize("i", range(len(CHUNKS)))
def test_places_outside_every_chunk_may_hold_anything(i):
    """A chunk's border inside a page, and gaps between the windows of rows that share a range."""
    sizes, kw = CHUNKS[i]
    p = Pass("grouped", seed=300 + i, **sizes, **kw)
    assert poison_unseen(p) > 0
    plan = p.plan()
    p.check(plan)
    later = p.plan(chunk=p.chunk)                            # a plan that leaves out what lies before the rows' chunks
    later.set(p.row_slot, p.tables, [x + 1 for x in p.row_pos])
    p.check(later)


FORMS = [("grouped", dict(SMALL["grouped"])), ("grouped", dict(SMALL["grouped"], P=48)), ("grouped", dict(SMALL["grouped"], dtype=F32)),
         ("grouped", dict(WIDE)), ("latent", dict(SMALL["latent"])), ("latent", dict(heads=16, dim=576, vdim=512)),
         ("latent", dict(SMALL["latent"], P=48)), ("latent", dict(heads=4, dim=48, vdim=32, dtype=F32))]


@pytest.mark.parametrize("i", range(len(FORMS)))
def test_results_that_are_no_numbers_are_not_hidden(i):
    """NaN and infinities in a query, in a request's only own key, in a value, in a sink or gate: the definition's NaN, and nobody else's."""
    kind, sizes = FORMS[i]
    for case in range(6):
        p = Pass(kind, groups=[(9, 5), (4, 2)], alone=2, pads=1, own=130, seed=10 * i + case, **sizes)
        live = [r for r, s in enumerate(p.row_slot) if s >= 0]
        a, b = live[0], live[-1]
        none = p.row_slot.index(-1)                          # a row without a slot gives zeros whatever stands in it
        p.q[none], p.gate[none] = math.nan, math.nan
        if case == 0:
            p.q[a, 1] = math.nan
            p.q[b] = math.nan
        elif case == 1:
            p.q[a, :, 3] = math.inf
            p.q[b, 0, 0] = -math.inf
        elif case == 2:                                      # the request's own part is this key alone
            r = next(r for r in live if p.row_pos[r] > 2 * p.P)
            lead = p.tables[p.row_slot[r]].tolist()
            shared = next(k for k, page in enumerate(lead) if not any(page == int(p.tables[s][k]) for s in p.row_slot if s >= 0 and s != p.row_slot[r]))
            p.row_pos[r] = shared * p.P
            p.d_pos = p.dev(p.row_pos)
            p.pool[lead[shared] * p.P] = math.nan
        elif case == 3:
            s, pos = p.row_slot[a], p.row_pos[a]
            p.pool[int(p.tables[s, pos // p.P]) * p.P + pos % p.P, -1 if kind == "grouped" else 5] = math.nan
        elif kind == "latent":
            p.sink[:3] = torch.tensor([math.nan, -math.inf, math.inf] if case == 4 else [1e30, -1e30, 80.0])
        else:
            p.gate[a, 0], p.gate[b, 1], p.gate[b, 0] = (math.nan, math.inf, -math.inf) if case == 4 else (1e30, -1e30, 80.0)
        plan = p.plan()
        got = p.run(plan)
        plan.check_status()
        want, tol = p.expected()
        assert case == 5 or want.isnan().any()
        assert torch.equal(got.isnan(), want.isnan()), (case, got.isnan().sum().item(), want.isnan().sum().item())
        assert ((got.double() - want).abs() <= tol)[~want.isnan()].all(), case


@pytest.mark.parametrize("groups,P,heads", [([(40, 90)], 64, 32), ([(3, 150), (2, 70)], 32, 16), ([(1, 200)], 64, 128)])
def test_exchanged_scores_are_read_before_they_are_overwritten(groups, P, heads):
    """Long walks of CTA pairs, again and again: each call gives the bits of the first, which are right."""
    p = Pass("latent", heads=heads, dim=576, vdim=512, groups=groups, P=P, own=400, seed=5)
    plan = p.plan()
    first = p.check(plan)
    for _ in range(40):
        assert torch.equal(p.run(plan), first)


@pytest.mark.parametrize("i", range(len(FORMS)))
def test_rows_of_other_slots_than_the_plan_says_are_reported(i):
    from ds41rt_b200.ops.lib import KernelError
    kind, sizes = FORMS[i]
    p = Pass(kind, groups=[(9, 5)], alone=2, pads=1, own=130, seed=i, **sizes)
    plan, none = p.plan(), p.row_slot.index(-1)
    a, b, c = [r for r, s in enumerate(p.row_slot) if s >= 0][:3]
    out = torch.empty(p.R, p.H, p.V, dtype=p.dtype, device="cuda")
    want, tol = p.expected()
    p.run(plan, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.run(plan, out=out)
    for call in (lambda: p.run(plan, out=out), g.replay):
        p.d_slot[c] = -1                                     # a row that the plan knows may have no slot
        call()
        plan.check_status()
        assert not out[c].any()
        for rows, slots in (((a, b), (p.row_slot[b], p.row_slot[a])), ((none,), (p.row_slot[a],))):
            p.d_slot[list(rows)] = p.dev(slots)
            call()
            with pytest.raises(KernelError, match="bad argument"):
                plan.check_status()
            plan.status.zero_()
            assert out[list(rows)].isnan().all()
            right = [r for r in range(p.R) if r not in rows and r != c]
            assert ((out.double() - want).abs() <= tol)[right].all()
            p.d_slot[:] = p.dev(p.row_slot)
            p.d_slot[c] = -1
        p.d_slot[:] = p.dev(p.row_slot)
        call()
        plan.check_status()
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("page", [-1, "n", 1 << 25, (1 << 31) - 1, -(1 << 31)])
@pytest.mark.parametrize("i", range(len(FORMS)))
def test_pages_that_the_pool_does_not_have(i, page):
    """A page inside what a row sees that is not leased, or whose number is none of the pool's: not there, or zeros in tensor-core forms."""
    kind, sizes = FORMS[i]
    p = Pass(kind, groups=[(5, 3)], alone=2, own=200, seed=i, **sizes)
    plan = p.plan()
    tiled = p.dtype == BF16 and p.P == 64
    r = next(r for r, s in enumerate(p.row_slot) if p.row_pos[r] >= 4 * p.P)
    s, hole = p.row_slot[r], 3                               # behind the common pages, before the row's last one
    want, tol = p.expected()
    p.d_tables[s, hole] = p.pool.shape[0] // p.P if page == "n" else page
    got = p.run(plan)
    torch.cuda.synchronize()
    plan.check_status()
    others = [x for x in range(p.R) if x != r]
    assert ((got.double() - want).abs() <= tol)[others].all()
    at = torch.arange(p.row_pos[r] + 1)
    rows = p.pool[(p.tables[s].long()[at // p.P] * p.P + at % p.P).cuda()].double()
    gone = (at // p.P == hole).cuda()
    rows[gone] = 0
    n = p.H // p.G
    for h in range(p.H):
        g = h // n
        k, v = (rows[:, g * p.D:(g + 1) * p.D], rows[:, p.G * p.D + g * p.V:p.G * p.D + (g + 1) * p.V]) if kind == "grouped" else (rows, rows[:, :p.V])
        z = k @ p.q[r, h].double() * p.scale
        if not tiled:
            z[gone] = -math.inf
        if kind == "latent":
            z = torch.cat([z, p.sink[h:h + 1].double()])
        w = torch.softmax(z, 0)[:len(at)]
        o, A = w @ v, w @ v.abs()
        u = 2.0 ** -8 if p.dtype == BF16 else 2.0 ** -24
        d = float((k.abs() @ p.q[r, h].double().abs()).max()) * p.scale * (p.D + 2) * 2.0 ** -23
        t = (2 * d * (1 + d) + 2.0 ** -20 + 2 * len(at) * 2.0 ** -23 + (u if p.dtype == BF16 else 0)) * A
        if kind == "grouped":
            f = torch.sigmoid(p.gate[r, h].double())
            o, t = o * f, (t + 2.0 ** -21 * o.abs()) * f
        assert ((got[r, h].double() - o).abs() <= t + u * (o.abs() + t) + 1e-30).all(), h


def test_graphs_are_captured_right_behind_a_long_prompt():
    """The rows of the last set_rows() took the long form, which needs no plan; the captured pass over them does."""
    import test_belasun_gpu as belasun
    from ds41rt_b200.runtime.session import DecodeSession
    from test_stack_gpu import close
    e = belasun.engine("tiles", "bf16", shared_prefix=True, page_tokens=32)
    toks = belasun.tokens("tiles", 110, seed=12)
    want, spread = belasun.reference("tiles", toks, "bf16")[:2]
    assert e.cache.ensure(0, 200)
    e.set_rows(toks[:100], list(range(100)), [0] * 100)
    e.forward_rows(100, head=False)
    e.set_rows(toks[:80], list(range(80)), [0] * 80)
    ses = DecodeSession(e)
    assert ses.graph(80) is not None
    for at in range(100, 110):
        ses.step([toks[at]], [at], [0])
        close(e.logits_rows(1).cpu().double(), want[at:at + 1], "bf16", spread[at:at + 1])
    e.check_status()


@pytest.mark.parametrize("kind", ["grouped", "latent"])
def test_plans_are_made_while_the_gpu_is_busy(kind):
    """set() orders its copies on the stream and does not wait for it; a later call takes the plan, an earlier one had its own."""
    a = Pass(kind, groups=[(9, 12)], seed=1, **SMALL[kind])
    b = Pass(kind, groups=[(5, 3)], alone=4, seed=2, **SMALL[kind])
    width, slots = max(x.tables.shape[1] for x in (a, b)), max(x.tables.shape[0] for x in (a, b))
    for x in (a, b):
        t = torch.full((slots, width), -1, dtype=torch.int32)
        t[:x.tables.shape[0], :x.tables.shape[1]] = x.tables
        x.tables, x.d_tables = t, t.cuda()
    plan = a.plan()
    a.run(plan), b.plan()                                    # pinned memory and kernels are there
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)
    busy = torch.cuda.Event()
    busy.record()
    got = []
    for _ in range(4):
        for x in (a, b):
            plan.set(x.row_slot, x.tables)
            got.append((x, x.run(plan)))
    assert not busy.query()
    torch.cuda.synchronize()
    plan.check_status()
    for x, out in got:
        want, tol = x.expected()
        assert ((out.double() - want).abs() <= tol).all()


def test_plans_are_not_set_inside_a_capture():
    p = Pass("grouped", groups=[(3, 4)], **SMALL["grouped"])
    plan = p.plan()
    out = torch.empty(p.R, p.H, p.V, dtype=BF16, device="cuda")
    p.run(plan, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            plan.set(p.row_slot, p.tables)
        p.run(plan, out=out)
    g.replay()
    torch.cuda.synchronize()
    want, tol = p.expected()
    assert ((out.double() - want).abs() <= tol).all()


def test_a_device_loop_gives_the_logits_of_its_own_tokens():
    """Steps that feed themselves across pages, as requests outgrow the lengths that the plan was made with, against the plain CPU statement
    of the tokens that came out."""
    import test_belasun_gpu as belasun
    from ds41rt_b200.runtime.session import DecodeSession
    from test_stack_gpu import close, feed
    e = belasun.engine("tiles", "bf16", shared_prefix=True, page_tokens=32)
    common = belasun.tokens("tiles", 130, seed=8)
    feed(e, 0, common, 0, [1024])
    snap = e.cache.snapshot(0, 130)
    assert e.cache.restore(1, snap) and all(e.cache.ensure(s, 300) for s in (0, 1))
    ses = DecodeSession(e)
    e.set_rows([3, 200], [130, 130], [0, 1])
    toks, seen = [[3], [200]], {}
    for step in range(120):
        ses.run_device_loop(2, 1)
        if step % 13 == 0 or step == 119:
            seen[130 + step] = e.logits_rows(2).cpu().double()
        for t, new in zip(toks, e.in_tokens[:2].tolist()):
            t.append(new)
    e.check_status()
    assert e.row_pos[:2].tolist() == [250, 250]
    for r in range(2):
        want, spread = belasun.reference("tiles", common + toks[r][:120], "bf16")[:2]
        for at, got in seen.items():
            close(got[r:r + 1], want[at:at + 1], "bf16", spread[at:at + 1])
