"""Plans of attention over a shared prefix around captures, and the division of the work (no GPU)."""
import contextlib

import pytest
import torch

from ds41rt_b200.models.base import RowsEngine


class Rows(RowsEngine):
    """An engine whose last rows were a prompt's, so that its plan is made when a pass asks for it."""

    def __init__(self):
        self.log, self.capturing, self.undescribed = [], False, True
        self.in_tokens = self.row_pos = self.row_slot = torch.zeros(4, dtype=torch.int32)
        self.long = True                                     # the first pass takes the form without a plan

    def settle(self):
        if self.undescribed:
            self.log.append("plan in capture" if self.capturing else "plan")
            self.undescribed = False

    def forward(self):
        if not self.long:
            self.settle()
        self.long = False
        self.log.append("captured" if self.capturing else "eager")


def test_plans_are_made_before_a_capture(monkeypatch):
    e = Rows()

    @contextlib.contextmanager
    def graph(g):
        e.capturing = True
        yield
        e.capturing = False

    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    e.capture(e.forward)
    assert e.log == ["plan", "eager", "captured"]


def many(rows=200, pages=250, own=11, width=266):
    """A page table of requests over one long prefix."""
    import numpy as np
    t = np.full((rows, width), -1, dtype=np.int32)
    t[:, :pages] = np.arange(pages)
    t[:, pages:pages + own] = pages + np.arange(rows * own).reshape(rows, own)
    return t


def plan(**kw):
    from ds41rt_b200.ops.prefix import PrefixPlan
    args = dict(kind="grouped", rows=200, heads=32, kv_heads=8, vdim=128, page_tokens=64, device="cpu")
    args.update(kw)
    return PrefixPlan(args.pop("kind"), **args)


def test_a_plan_is_made_in_a_fraction_of_a_step():
    """Batches that change are planned between their steps.  The largest of these took 14 ms once, 0.4 ms now."""
    import time
    t, p = many(), plan()
    best = 1.0
    for _ in range(5):
        start = time.perf_counter()
        p.set(range(200), t)
        best = min(best, time.perf_counter() - start)
    assert p.shared == [(list(range(200)), 16000)] and best < 3e-3


@pytest.mark.parametrize("lengths", [[-5, 0, 1, 3000], [1 << 60, 1 << 40, 64 * 266, 64 * 266 + 1], [-(1 << 62)] * 4])
@pytest.mark.parametrize("chunk", [0, 100])
def test_lengths_beyond_what_a_request_can_have(lengths, chunk):
    p, t = plan(rows=4, chunk=chunk), many(4)
    p.set(range(4), t, lengths)
    d = p.data.numpy()
    units = d[4:4 + 8 * p.n_units].reshape(-1, 8)
    units = units[units[:, 2] > 0]
    assert (units[:, 3] >= 0).all() and (units[:, 3] < units[:, 4]).all() and (units[:, 4] <= 266 * 64).all()
    for r in range(4):                                       # the table's end belongs to a unit of every row
        assert any(u[4] == 266 * 64 and u[6] and u[1] <= r < u[1] + u[2] for u in units)


def test_tables_in_other_orders_and_too_long_ones():
    import numpy as np
    t, p, q = many(6), plan(rows=6), plan(rows=6)
    p.set(range(6), t)
    q.set(range(6), np.asfortranarray(t))
    assert torch.equal(p.data, q.data)
    q.set(range(6), torch.from_numpy(np.repeat(t, 2, 0))[::2])
    assert torch.equal(p.data, q.data)
    with pytest.raises(ValueError, match="2\\^31"):
        plan(page_tokens=1 << 24).set(range(6), t)


def test_heads_whose_units_do_not_come_in_twos():
    """An odd number of items per head, and more heads than a block has turns at a time."""
    for kv in (1, 3, 64, 300):
        p = plan(rows=3, heads=kv, kv_heads=kv, vdim=16)
        p.set(range(3), many(3, pages=3, own=1, width=5))
        units = p.data[4:4 + 8 * p.n_units].reshape(-1, 8)
        seen = {}
        for slot, first, n, k0, k1, part, tail, head in units[units[:, 2] > 0].tolist():
            for i in range(first, first + n):
                r = i if tail else int(p.data[p._at[2] + i])
                seen.setdefault((r, head), []).append((k0, k1))
        assert len(seen) == 3 * kv
        for spans in seen.values():
            spans.sort()
            assert spans[0][0] == 0 and spans[-1][1] == 320 and all(a[1] == b[0] for a, b in zip(spans, spans[1:]))


def test_the_memory_of_plans_is_known_before_they_are_made():
    from types import SimpleNamespace as N
    from ds41rt_b200.models.registry import FAMILIES
    from ds41rt_b200.models.stack import prefix_plan_bytes, prefix_plan_sizes
    from ds41rt_b200.ops.prefix import PrefixPlan
    shapes = [("grouped", 32, 8, 128, 128, 0), ("grouped", 32, 8, 128, 128, 8192), ("grouped", 32, 8, 128, 128, 0),
              ("latent", 16, 1, 576, 512, 0), ("latent", 4, 1, 96, 64, 0), ("grouped", 4, 2, 320, 64, 0)]
    layers = [N(mixer=N(prefix_shape=lambda s=s: s)) for s in shapes] + [N(mixer=N())]
    w = N(dtype="bf16", layers=layers)
    sizes = prefix_plan_sizes(w, 40, 64)
    assert set(sizes) == set(shapes[:5])                     # wide keys are read row by row
    made = [PrefixPlan(device="cpu", **s) for s in sizes.values()]
    assert prefix_plan_bytes(w, 40) == sum(t.numel() * t.element_size() for p in made for t in (p.data, p.part_o, p.part_ml, p.status))
    assert prefix_plan_bytes(w, 5000) == prefix_plan_bytes(w, 256) > prefix_plan_bytes(w, 40)
    assert prefix_plan_bytes(N(dtype="f32", layers=layers), 40) == 0
    assert FAMILIES["belasun"].shared_prefix_bytes(w, 40) == prefix_plan_bytes(w, 40) and FAMILIES["ds41"].shared_prefix_bytes(w, 40) == 0


def test_blocks_that_come_back_very_often():
    """Thousands of heads: each block takes its turns by the thousand, and no place is dealt twice."""
    p = plan(rows=40, heads=8192, kv_heads=8192, vdim=16)
    p.set(range(40), many(40, pages=2, own=3, width=6))
    d = p.data.numpy()
    units = d[4:4 + 8 * p.n_units].reshape(-1, 8)
    alive = units[units[:, 2] > 0]
    assert len({(u[1], u[3], u[6], u[7]) for u in alive.tolist()}) == len(alive)
    turns = d[p._at[1]:p._at[2]]
    assert turns.max() <= p.max_turns and int(turns.sum()) >= len(alive) // 2 and turns.max() - turns.min() <= 2
