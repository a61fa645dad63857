"""Plans of attention over a shared prefix: which rows share what, how the keys are divided, and what the calls refuse (no GPU)."""
import itertools
import random

import numpy as np
import pytest
import torch

from ds41rt_b200.ops import prefix
from ds41rt_b200.ops.prefix import PrefixPlan, common_runs

BF16 = torch.bfloat16


def table(*rows, width=12):
    t = np.full((len(rows), width), -1, dtype=np.int32)
    for i, r in enumerate(rows):
        t[i, :len(r)] = r
    return t


def test_rows_are_grouped_by_their_leading_pages():
    t = table([1, 2, 3, 4, 5], [1, 2, 3, 7, 8, 9], [1, 2, 3, 11], [1, 20, 21], [30, 31, 32], [30, 31, 33, 34], [])
    got = {tuple(sorted(rows)): pages for rows, pages in common_runs(t)}
    assert got == {(0, 1, 2): 3, (4, 5): 2}


def test_one_row_that_shares_little_does_not_cost_the_others_their_prefix():
    t = table(*[[1, 2, 3, 4, 5, 6, 7, 8, 100 + i] for i in range(6)], [1, 200, 201])
    assert [(sorted(r), p) for r, p in common_runs(t)] == [(list(range(6)), 8)]


def test_leading_pages_alone_count_and_free_places_never_do():
    assert common_runs(table([1, 2, 3], [4, 2, 3])) == []
    assert common_runs(table([], [])) == []
    assert common_runs(table([5])) == []
    assert common_runs(table([1, 2], [1, 2], width=2)) == [([0, 1], 2)]


def best_saving(t):
    """Most page reads that any division of the rows into groups saves, by trying them all."""
    n = len(t)

    def run(rows):
        k = 0
        while k < t.shape[1] and t[rows[0], k] >= 0 and all(t[r, k] == t[rows[0], k] for r in rows):
            k += 1
        return k

    best = 0
    for size in range(2, n + 1):
        for rows in itertools.combinations(range(n), size):
            best = max(best, (size - 1) * run(rows))
    return best


@pytest.mark.parametrize("seed", range(40))
def test_the_first_group_saves_most_and_groups_are_true(seed):
    rng = random.Random(seed)
    rows = []
    for _ in range(rng.randint(2, 7)):                       # paths of a small random tree
        rows.append([10 * d + rng.randint(0, 1 + d // 3) for d in range(rng.randint(0, 6))])
    t = table(*rows)
    groups = common_runs(t)
    seen = [r for g, _ in groups for r in g]
    assert len(seen) == len(set(seen))
    for members, pages in groups:
        assert len(members) > 1 and pages > 0
        assert all((t[m, :pages] == t[members[0], :pages]).all() and (t[m, :pages] >= 0).all() for m in members)
    assert max([(len(m) - 1) * p for m, p in groups], default=0) == best_saving(t)


@pytest.mark.parametrize("seed", range(30))
def test_units_cover_every_position_of_every_row_once(seed):
    rng = random.Random(seed)
    P = rng.choice([32, 64, 128])
    kind, heads, kv, vdim = rng.choice([("grouped", 16, 4, 64), ("grouped", 6, 2, 64), ("latent", 16, 1, 512), ("latent", 5, 1, 64)])
    rows = rng.randint(2, 90)
    width = 80
    t = np.full((rows + 4, width), -1, dtype=np.int32)
    pages = iter(rng.sample(range(100000), 20000))
    slots = rng.sample(range(rows + 4), rows)
    parts = [[next(pages) for _ in range(rng.randint(1, 70))] for _ in range(rng.randint(1, 4))]
    for s in slots:
        lead = rng.choice(parts + [[]])
        row = lead + [next(pages) for _ in range(rng.randint(1, width - len(lead)))]
        t[s, :len(row)] = row
    row_slots = [s if rng.random() < 0.9 else -1 for s in slots]
    if seed % 3 == 0:                                          # several rows of a request
        row_slots = [s for s in row_slots[:rows // 3] for _ in range(3)]
    lengths = [rng.randint(1, width * P) for _ in row_slots] if seed % 2 else None
    plan = PrefixPlan(kind, rows=rows, heads=heads, kv_heads=kv, vdim=vdim, page_tokens=P, device="cpu")
    plan.set(row_slots, torch.from_numpy(t), lengths)
    d = plan.data.numpy()
    units, turns, order, cell, count = (d[a:b] for a, b in zip(plan._at, plan._at[1:] + [len(d)]))
    assert d[0] == plan.n_units <= plan.max_units and not units[8 * plan.n_units:].any()
    listed = units.reshape(plan.max_turns, plan.grid, -1, 8)[..., 2].any(2)
    assert (listed == (np.arange(plan.max_turns)[:, None] < turns[None])).all()          # a block's turns are its first places
    covered, used = {}, set()
    for slot, first, n, k0, k1, part, tail, head in units[:8 * plan.n_units].reshape(-1, 8).tolist():
        if n == 0:                                             # a place that was not dealt
            continue
        assert 0 < n <= plan.rows_per_unit and 0 <= k0 < k1 and k0 % P == 0 and k1 % P == 0 and 0 <= head < kv
        for r in range(first, first + n) if tail else order[first:first + n].tolist():
            s = row_slots[r]
            assert s >= 0 and (t[s, :k1 // P] == t[slot, :k1 // P]).all() and (not tail or s == slot)
            assert part < count[r]
            cells = (int(cell[r]) + part, head)
            assert cells not in used and cells[0] < plan.max_cells       # no cell has two writers
            used.add(cells)
            covered.setdefault((r, head), []).append((k0, k1, part))
    for r, s in enumerate(row_slots):
        for head in range(kv):
            got = sorted(covered.get((r, head), []))
            assert [x[2] for x in got] == list(range(count[r]))
            assert [x[0] for x in got] + [width * P] == [0] + [x[1] for x in got] if s >= 0 else not got


def test_a_new_plan_replaces_the_old_one_whole():
    t = table([1, 2, 3, 4], [1, 2, 3, 5], [9, 8])
    plan = PrefixPlan("grouped", rows=3, heads=4, kv_heads=2, vdim=16, page_tokens=64, device="cpu")
    plan.set([0, 1, 2], t)
    assert plan.n_units > 0 and plan.shared == [([0, 1], 192)]
    plan.set([0, 2], t)
    assert plan.shared == []
    plan.set([-1, -1], t)
    assert plan.n_units == 0 and int(plan.data.abs().sum()) == 0


def test_rows_of_one_slot_share_with_other_slots_only():
    t = table([1, 2, 3, 4], [1, 2, 3, 5])
    plan = PrefixPlan("latent", rows=4, heads=4, vdim=16, page_tokens=64, device="cpu")
    plan.set([0, 0, 0], t)
    assert plan.shared == []
    plan.set([0, 0, 1, -1], t)
    assert plan.shared == [([0, 1, 2], 192)]


def test_short_prefixes_are_left_to_the_rows():
    t = table([1, 2], [1, 3])
    plan = PrefixPlan("grouped", rows=2, heads=4, kv_heads=2, vdim=16, page_tokens=32, device="cpu", min_tokens=64)
    plan.set([0, 1], t)
    assert plan.shared == []


@pytest.mark.parametrize("kind,P", [("grouped", 32), ("grouped", 48), ("grouped", 192), ("latent", 16), ("latent", 160)])
def test_key_ranges_are_whole_pages_and_fit_the_plan(kind, P):
    for rows, pages in ((2, 3), (2, 40), (90, 30), (150, 600)):
        shared = list(range(1, pages + 1))
        t = table(*[shared + [100000 + 10 * i] for i in range(rows)], width=pages + 4)
        plan = PrefixPlan(kind, rows=rows, heads=8, kv_heads=2 if kind == "grouped" else 1, vdim=64, page_tokens=P, device="cpu")
        plan.set(range(rows), t)
        assert plan.span > 0 and plan.span % P == 0 and 0 < plan.n_units <= plan.max_units
        units = plan.data[4:4 + 8 * plan.n_units].reshape(-1, 8)
        assert bool((units[:, 3] % P == 0).all()) and bool((units[:, 4] % P == 0).all())


def test_short_requests_are_not_divided_and_long_ones_are():
    t = table(*[[10 * i + k for k in range(1, 3)] for i in range(4)], list(range(1000, 1700)), width=800)
    plan = PrefixPlan("grouped", rows=5, heads=8, kv_heads=2, vdim=128, page_tokens=64, device="cpu")
    plan.set(range(5), t)
    at = plan._at[4]
    assert plan.data[at:at + 5].tolist()[:4] == [1, 1, 1, 1] and plan.data[at + 4] > 8


@pytest.mark.parametrize("kw", [dict(kind="other"), dict(heads=0), dict(heads=6, kv_heads=4), dict(vdim=24), dict(rows=0),
                                dict(kind="latent", kv_heads=2), dict(dtype=torch.float16), dict(page_tokens=0)])
def test_plans_refuse_what_they_cannot_describe(kw):
    args = dict(kind="grouped", rows=4, heads=8, kv_heads=2, vdim=32, page_tokens=64, device="cpu")
    args.update(kw)
    if args["kind"] == "latent" and "kv_heads" not in kw:
        args["kv_heads"] = 1
    with pytest.raises(ValueError):
        PrefixPlan(args.pop("kind"), **args)


@pytest.mark.parametrize("slots,tables", [([0] * 5, table([1])), ([1], table([1])), ([0], table([1]).astype(np.int64)),
                                          ([0], table([1])[0]), ([[0]], table([1]))])
def test_plans_refuse_rows_and_tables_that_do_not_fit(slots, tables):
    plan = PrefixPlan("grouped", rows=4, heads=8, kv_heads=2, vdim=32, page_tokens=64, device="cpu")
    with pytest.raises(ValueError):
        plan.set(slots, tables)
    with pytest.raises(ValueError):
        plan.set([0], table([1]), [1, 2])


def call(kind="grouped", **change):
    """A call that is right but for its device (everything lies on the CPU), with some arguments changed."""
    H, D, V, P, R = 8, 32, 32, 64, 3
    G = 2 if kind == "grouped" else 1
    plan = PrefixPlan(kind, rows=4, heads=H, kv_heads=G, vdim=V, page_tokens=P, device="cpu")
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)
    a = dict(page_table=z(4, 5, dtype=torch.int32), row_pos=z(R, dtype=torch.int32), row_slot=z(R, dtype=torch.int32), plan=plan,
             scale=1.0, out=z(R, H, V))
    if kind == "grouped":
        a.update(q=z(R, H, D), pool=z(10 * P, G * (D + V)), gate=z(R, H, dtype=torch.float32))
        fn = prefix.group_attend
    else:
        a.update(q_abs=z(R, H, V), q_rot=z(R, H, 16), pool=z(10 * P, V + 16), sink=z(H, dtype=torch.float32))
        fn = prefix.latent_attend
    for k, v in change.items():
        a[k] = v(a[k]) if callable(v) else v
    return fn(**a)


COMMON = [
    (dict(page_table=lambda t: t.long()), "32-bit"), (dict(row_pos=lambda t: t.float()), "32-bit"),
    (dict(row_slot=lambda t: t[:2]), "entry per row"), (dict(page_table=lambda t: t[0]), "slots, pages"),
    (dict(page_table=lambda t: t.t()), "contiguous"), (dict(pool=lambda t: t[:100]), "whole pages"),
    (dict(pool=lambda t: t[:, :-1]), "contiguous rows"), (dict(pool=lambda t: t.float()), "pool is"),
    (dict(out=lambda t: t[:2]), "out must be"), (dict(out=lambda t: t.float()), "out is"),
    (dict(out=lambda t: t.transpose(0, 1)), "out must be"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(), "current CUDA device"),
]


@pytest.mark.parametrize("kind", ["grouped", "latent"])
@pytest.mark.parametrize("change,why", COMMON)
def test_calls_refuse_what_does_not_fit(kind, change, why):
    if not change and torch.cuda.is_available():
        pytest.skip("the device check is the one that is asked here")
    with pytest.raises(ValueError, match=why):
        call(kind, **change)


@pytest.mark.parametrize("change", [
    dict(q=lambda t: t.float()), dict(q=lambda t: t[:, :4]), dict(q=lambda t: t[..., :24]), dict(q=lambda t: t[..., ::2]),
    dict(q=lambda t: t[0]), dict(q=lambda t: torch.zeros(5, 8, 32, dtype=BF16)), dict(q=lambda t: torch.zeros(0, 8, 32, dtype=BF16)),
    dict(q=lambda t: torch.zeros(3 * 8 * 32 + 1, dtype=BF16)[1:].view(3, 8, 32)), dict(q=lambda t: t[:1].expand(3, 8, 32)),
    dict(q=lambda t: torch.zeros(3, 8, 48, dtype=BF16)[..., :32]),
    dict(gate=lambda t: t.to(BF16)), dict(gate=lambda t: t[:2]), dict(gate=lambda t: t.t().contiguous().t()), dict(chunk=-1),
    dict(plan=lambda p: PrefixPlan("latent", rows=4, heads=8, vdim=32, page_tokens=64, device="cpu"))])
def test_grouped_calls_refuse(change):
    with pytest.raises(ValueError):
        call("grouped", **change)


@pytest.mark.parametrize("change", [
    dict(q_abs=lambda t: t[..., :16]), dict(q_abs=lambda t: t.float()), dict(q_rot=lambda t: t[:2]), dict(q_rot=lambda t: t[..., :8]),
    dict(q_rot=None), dict(sink=lambda t: t[:4]), dict(sink=lambda t: t.to(BF16)), dict(sink=lambda t: torch.zeros(16)[::2]),
    dict(plan=lambda p: PrefixPlan("grouped", rows=4, heads=8, kv_heads=1, vdim=32, page_tokens=64, device="cpu"))])
def test_latent_calls_refuse(change):
    with pytest.raises(ValueError):
        call("latent", **change)


class Leases:
    """What StackEngine.describe() asks of an engine and its cache."""
    from ds41rt_b200.models.stack import StackEngine
    describe, settle = StackEngine.describe, StackEngine.settle

    def __init__(self):
        from ds41rt_b200.models.paged import PagedSlots
        self.cache = PagedSlots()
        self.cache._init_pages(4, 1024, "cpu", 64, 40)
        self.attn_rows, self._planned, self._plan_from, self._plan_until, self._undescribed = 3, None, [], 0, None
        self.prefix_plans = {"x": PrefixPlan("grouped", rows=3, heads=4, kv_heads=2, vdim=16, page_tokens=64, device="cpu")}
        self.plan, self.sets = self.prefix_plans["x"], 0
        real = self.plan.set

        def counted(*a):
            self.sets += 1
            real(*a)
        self.plan.set = counted

    def share(self, slot, n):
        """A lease of the first n pages of slot 0."""
        pages = self.cache.alloc.retain(0, self.cache._gen(0), n)
        self.cache.alloc.share(slot, self.cache._gen(slot), pages)
        self.cache._publish(slot)


def test_plans_of_an_engine_follow_its_rows_and_their_leases():
    e = Leases()
    assert e.cache.ensure(0, 300)
    e.share(1, 3)
    e.share(2, 2)
    assert e.cache.ensure(1, 400) and e.cache.ensure(2, 400)
    e.describe([300, 301, 302], [0, 1, 2])
    assert e.sets == 1 and e.plan.shared == [([0, 1, 2], 128)]
    e.describe(np.array([301, 302, 303]), np.array([0, 1, 2]))         # the same requests a step later
    assert e.cache.ensure(0, 700)                                      # pages appended to a lease
    e.describe([302, 303, 304], [0, 1, 2])
    assert e.sets == 1
    e.describe([600, 303, 304], [0, 1, 2])                             # longer by a few tiles
    assert e.sets == 2
    e.describe([599, 303, 304], [0, 1, 2])                             # one goes back
    assert e.sets == 3
    e.sets = 2
    e.describe([601, 304], [0, 1])
    assert e.sets == 3 and e.plan.shared == [([0, 1], 192)]
    e.describe([304, 601], [1, 0])
    assert e.sets == 4
    e.cache.release(1)                                                 # the slot's next request shares nothing
    assert e.cache.ensure(1, 400)
    e.describe([304, 601], [1, 0])
    assert e.sets == 5 and e.plan.shared == []
    e.describe([1, 2, 3, 4], [0, 0, 0, 0])                             # more rows than passes of this form have
    assert e.sets == 6 and int(e.plan.data[e.plan._at[4]:].count_nonzero()) == 3
    e.describe([], [])
    assert e.plan.n_units == 0


def test_rows_that_need_no_plan_are_described_when_one_is():
    e = Leases()
    assert e.cache.ensure(0, 300)
    e.describe([1], [0])
    e.settle()
    assert e.sets == 1
    e._undescribed = ([2, 3], [0, 0])
    e.settle()
    e.settle()
    assert e.sets == 2 and e._undescribed is None and e.plan.n_rows == 2
    e._undescribed = ([2, 3], [0, 0])
    e.describe([4], [0])                                     # other rows are there now
    e.settle()
    assert e.sets == 3 and e.plan.n_rows == 1


def test_engines_without_plans_ignore_the_rows():
    e = Leases()
    e.prefix_plans = {}
    e.describe([1], [0])
    assert e.sets == 0


def test_only_layer_stacks_are_served_with_shared_prefixes():
    from ds41rt_b200.models.registry import FAMILIES
    assert {n for n, f in FAMILIES.items() if f.shared_prefix} == {"genesun", "belasun"}


def matching(plan, monkeypatch, rows, shape, capturing=False):
    """The last of a call's checks, which stand behind that of the device."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(plan, "device", torch.device("cuda"))
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype)
    pool, out = z(128, 32, dtype=BF16), z(rows, 4, 16, dtype=BF16)
    prefix._check(plan, "latent", rows, out, None, None, pool, z(*shape), z(rows), z(rows), out, 32, 1.0)


def test_calls_match_the_rows_and_the_table_of_their_plan(monkeypatch):
    plan = PrefixPlan("latent", rows=6, heads=4, vdim=16, page_tokens=64, device="cpu")
    with pytest.raises(ValueError, match="set for 0 rows"):
        matching(plan, monkeypatch, 3, (3, 5))
    t = table([1, 2], [1, 3], [4], width=5)
    plan.set([0, 1, 2], t)
    matching(plan, monkeypatch, 3, (3, 5))
    for rows, shape in ((2, (3, 5)), (4, (3, 5)), (3, (2, 5)), (3, (3, 6)), (3, (3, 4))):
        with pytest.raises(ValueError, match="set for 3 rows"):
            matching(plan, monkeypatch, rows, shape)


def test_plans_of_captured_calls_do_not_outgrow_them(monkeypatch):
    plan = PrefixPlan("latent", rows=6, heads=4, vdim=16, page_tokens=64, device="cpu")
    t = table([1, 2], [1, 3], [4], width=5)
    plan.set([0, 1, 2, -1], t)
    matching(plan, monkeypatch, 4, (3, 5))
    plan.set([0, 1, 2, -1, -1], t)
    matching(plan, monkeypatch, 5, (3, 5), capturing=True)
    plan.set([0, 1, 2], t)
    matching(plan, monkeypatch, 3, (3, 5), capturing=True)
    with pytest.raises(ValueError, match="captured call has 3 rows"):
        plan.set([0, 1, 2, -1], t)
    with pytest.raises(ValueError, match="captured"):
        plan.set([0, 1, 2], table([1, 2], [1, 3], [4], [5], width=5))
    plan.set([2, -1], t)
    assert plan.n_rows == 2


@pytest.mark.parametrize("seed", range(20))
def test_plans_with_a_chunk_leave_out_what_no_row_sees(seed):
    rng = random.Random(seed)
    P, chunk, width = rng.choice([(32, 256), (64, 100), (64, 1024), (16, 50)]) + (60,)
    rows = rng.randint(2, 40)
    lead = list(range(1, 1 + rng.randint(1, 40)))
    t = np.full((rows, width), -1, dtype=np.int32)
    for i in range(rows):
        own = rng.randint(1, width - len(lead))
        t[i, :len(lead) + own] = lead + [1000 + 100 * i + k for k in range(own)]
    slots = list(range(rows)) if seed % 2 else [i // 2 for i in range(rows)]          # two rows of a request
    lengths = [rng.randint(1, width * P) for _ in slots] if seed % 2 else [n + k for n in [rng.randint(1, width * P - 1)
                                                                              for _ in range(rows)] for k in range(2)][:rows]
    plan = PrefixPlan("grouped", rows=rows, heads=8, kv_heads=2, vdim=64, page_tokens=P, device="cpu", chunk=chunk)
    plan.set(slots, t, lengths)
    d = plan.data.numpy()
    units, turns, order, cell, count = (d[a:b] for a, b in zip(plan._at, plan._at[1:] + [len(d)]))
    covered = {}
    for slot, first, n, k0, k1, part, tail, head in units[:8 * plan.n_units].reshape(-1, 8).tolist():
        for r in range(first, first + n) if tail else order[first:first + n].tolist():
            assert part < count[r] and (t[slots[r], :k1 // P] == t[slot, :k1 // P]).all() and (not tail or slots[r] == slot)
            covered.setdefault((r, head), []).append((k0, k1, part))
    for r in range(rows):
        for head in range(2):
            got = sorted(covered[r, head])
            assert [x[2] for x in got] == list(range(count[r]))
            assert [x[0] for x in got[1:]] + [width * P] == [x[1] for x in got]         # no gap to the table's end
            assert got[0][0] <= (lengths[r] - 1) // chunk * chunk
    plan.set(slots, t)                                       # without lengths nothing is left out
    first = plan.data[4:4 + 8 * plan.n_units].reshape(-1, 8)
    assert int(first[first[:, 2] > 0][:, 3].min()) == 0
    with pytest.raises(ValueError):
        PrefixPlan("latent", rows=2, heads=4, vdim=16, page_tokens=64, device="cpu", chunk=64)


@pytest.mark.parametrize("args,want", [
    (("grouped", 32, 8, 128, 128, 64), True), (("grouped", 32, 8, 256, 128, 16), True), (("grouped", 32, 8, 128, 144, 64), False),
    (("grouped", 160, 1, 64, 64, 64), False), (("grouped", 32, 8, 272, 64, 64), False), (("grouped", 32, 8, 64, 64, 48), False),
    (("grouped", 32, 8, 64, 64, 4), False), (("grouped", 32, 8, 64, 64, 192), True), (("grouped", 32, 8, 64, 64, 96), False),
    (("latent", 128, 1, 576, 512, 64), True), (("latent", 130, 1, 576, 512, 64), False), (("latent", 16, 1, 592, 528, 64), False),
    (("latent", 16, 1, 592, 512, 64), False), (("latent", 16, 1, 512, 512, 8), True)])
def test_which_shapes_engines_plan_for(args, want):
    assert prefix.tiled(*args) is want
