"""Ragged passes where they could go wrong: graphs, streams, strides, far places, pages that are not there, NaN and infinities, requests
that cannot be.  Values are compared as in test_ragged_gpu.py, whose passes these are."""
import math
import random

import pytest
import torch

from test_ragged_gpu import BF16, F32, I32, Batch, ragged

pytestmark = pytest.mark.gpu
FORMS = [dict(heads=8, kv_heads=2, dim=64, vdim=64, P=64), dict(heads=8, kv_heads=2, dim=64, vdim=64, P=24),
         dict(heads=8, kv_heads=2, dim=64, vdim=64, P=32, dtype=F32), dict(heads=8, kv_heads=2, dim=64, vdim=192, P=64)]
MIXED = [(1, 700), (37, 5), None, (0, 40), (130, 129), (1, 63), (2, 126)]


def run(b, **kw):
    b.describe()
    out = b.attend(**kw)
    b.p.check_status()
    return out


@pytest.mark.parametrize("form", FORMS)
def test_rows_behind_the_last_and_between_are_left_as_they_were(form):
    b = Batch(MIXED, pads=5, **form)
    out = torch.full((b.R, b.H, b.V), 7.0, dtype=b.dtype, device="cuda")
    assert run(b, out=out) is out
    b.check(out)
    assert (out[b.total:] == 7).all()


@pytest.mark.parametrize("form", FORMS)
def test_capacity_beyond_the_rows(form):
    """A pass for more rows and requests than it has."""
    b = Batch(MIXED, pads=300, **form)
    out = run(b, out=torch.zeros(b.R, b.H, b.V, dtype=b.dtype, device="cuda"))
    b.check(out)
    empty = torch.zeros(0, dtype=I32, device="cuda")
    pos, slot, place = b.p.describe(empty, empty, empty, b.d_tables, b.pages)
    assert (slot == -1).all() and (place == -1).all() and (pos == 0).all()
    kept = out.clone()
    assert torch.equal(b.attend(out=out), kept)
    b.p.check_status()


@pytest.mark.parametrize("form", FORMS)
def test_described_by_rows(form):
    b = Batch(MIXED, pads=3, spare=2, **form)             # its three rows without a slot are a request each
    first = [x.clone() for x in b.describe()]
    want = b.attend()
    n = b.total
    pos, slot = first[0].clone(), first[1].clone()
    again = b.p.describe_rows(pos[:n], slot[:n], b.d_tables, b.pages)
    assert all(torch.equal(x, y) for x, y in zip(again, first))
    b.p.check_status()
    b.check(b.attend())
    assert torch.equal(b.attend()[:n], want[:n])


def test_rows_of_more_requests_than_the_pass_takes():
    m = ragged()
    p = m.RaggedPass(rows=20, requests=3, heads=4, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cuda")
    table = torch.arange(10, dtype=I32, device="cuda").view(5, 2)
    dev = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    pos, slot, place = p.describe_rows(dev([5, 6, 7, 70, 3, 4, 1, 2]), dev([0, 0, 0, 1, 2, 2, 3, 3]), table, 10)
    assert slot.tolist()[:8] == [0, 0, 0, 1, 2, 2, -1, -1] and pos.tolist()[:6] == [5, 6, 7, 70, 3, 4]
    assert place.tolist()[:6] == [5, 6, 7, 3 * 64 + 6, 4 * 64 + 3, 4 * 64 + 4]
    from ds41rt_b200.ops.lib import KernelError
    with pytest.raises(KernelError, match="1 requests"):
        p.check_status()
    # one slot twice, apart, and positions that do not follow one another: requests of their own
    pos, slot, place = p.describe_rows(dev([5, 7, 1]), dev([0, 0, 1]), table, 10)
    assert p.header[1].item() == 3
    p.check_status()


def test_rows_without_a_slot_are_one_request():
    m = ragged()
    p = m.RaggedPass(rows=900, requests=3, heads=4, kv_heads=2, dim=64, vdim=64, page_tokens=64, device="cuda")
    table = torch.arange(10, dtype=I32, device="cuda").view(5, 2)
    pos = torch.arange(900, dtype=I32, device="cuda") * 7919 % 2000
    slot = torch.full_like(pos, -1)
    pos[600:640], slot[600:640] = torch.arange(50, 90, device="cuda", dtype=I32), 2
    got_pos, got_slot, place = p.describe_rows(pos, slot, table, 10)
    p.check_status()
    assert torch.equal(got_pos, pos) and torch.equal(got_slot, slot) and (place[slot < 0] == -1).all()
    assert place[600:640].tolist() == [4 * 64 + i for i in range(50, 90)]
    assert p.header[1].item() == 900
    slot[700:701] = 1                       # a fourth and a fifth
    pos[700:701] = 3
    got_pos, got_slot, place = p.describe_rows(pos, slot, table, 10)
    assert (got_slot[700:] == -1).all() and got_slot[639].item() == 2 and p.header[1].item() == 700
    with pytest.raises(ValueError, match="copies"):
        p.describe_rows(p.row_pos, slot, table, 10)


def test_requests_that_cannot_be():
    from ds41rt_b200.ops.lib import KernelError
    b = Batch([(3, 10), (2, 60), (4, 0)])
    for what, tensor, value in (("negative", b.d_new, -1), ("too short", b.d_length, 1), ("too long", b.d_length, 1 << 29), ("slot", b.d_slots, 5)):
        kept = tensor.clone()
        tensor[1] = value
        pos, slot, place = b.describe()
        with pytest.raises(KernelError, match="number 1"):
            b.p.check_status()
        rows = 2 if tensor is not b.d_new else 0
        assert slot.tolist()[:3 + rows] == [b.slots[0]] * 3 + [-1] * rows and place[3:3 + rows].tolist() == [-1] * rows, what
        out = b.attend()
        assert (out[3:3 + rows] == 0).all()
        tensor.copy_(kept)
    b.describe()
    b.p.check_status()
    b.check(b.attend())
    # more tokens than the pass has rows
    b.d_new[2] = 1 << 30
    b.d_length[2] = (1 << 30) + 1
    pos, slot, place = b.describe()
    with pytest.raises(KernelError, match="number 2"):
        b.p.check_status()
    assert b.p.header[1].item() == b.R
    b.attend()
    torch.cuda.synchronize()


@pytest.mark.parametrize("form", FORMS)
def test_strides(form):
    """Queries, gates and results inside wider tensors; queries whose heads stand apart."""
    b = Batch(MIXED, pads=2, gate=True, **form)
    R, H, D, V = b.R, b.H, b.D, b.V
    wide = torch.randn(R, H + 3, D + 16, device="cuda").to(b.dtype)
    wide[:, 2:2 + H, :D] = b.q
    b.q = wide[:, 2:2 + H, :D]
    gates = torch.randn(R, H + 5, device="cuda")
    gates[:, 1:1 + H] = b.gate
    b.gate = gates[:, 1:1 + H]
    store = torch.full((R, H * V + 24), 3.0, device="cuda").to(b.dtype)
    out = store[:, 8:8 + H * V].unflatten(1, (H, V))
    run(b, out=out)
    b.check(out)
    assert (store[:, :8] == 3).all() and (store[:, 8 + H * V:] == 3).all()


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (64, 256), (128, 160)])
def test_results_at_any_16_bytes(dim, vdim):
    """Rows of the result that begin at 16 bytes but not at 32; requests in one piece and in many."""
    b = Batch([(1, 9000), (100, 30), (7, 4000), (1, 0)], heads=8, kv_heads=2, dim=dim, vdim=vdim, pads=1, sink=True)
    b.describe()
    assert b.p.units.view(-1, ragged().UNIT)[:b.p.header[0].item(), 8].max() > 1
    want = b.attend()
    b.check(want)
    wide = torch.full((b.R, 8 * vdim + 24), 7.0, dtype=BF16, device="cuda")
    out = wide[:, 8:8 + 8 * vdim].unflatten(1, (8, vdim))
    b.attend(out=out)
    assert torch.equal(out[:b.total], want[:b.total])
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + 8 * vdim:] == 7).all() and (wide[b.total:] == 7).all()


@pytest.mark.parametrize("form", FORMS)
def test_pages_that_are_not_leased_read_as_zeros(form):
    """Of a visible page without a number, or with one that the pool does not have."""
    b = Batch([(1, 200), (70, 300)], **form)
    P = b.P
    for s, pg, number in ((b.slots[0], 1, -1), (b.slots[1], 2, b.pages + 7), (b.slots[1], 0, -1)):
        b.tables[s, pg] = number
    b.d_tables = b.tables.cuda()
    out = run(b)
    # the same with a page of zeros
    zero = int(set(range(b.pages)).difference(b.tables.flatten().tolist()).pop())
    b.pool[zero * P:(zero + 1) * P] = 0
    t = b.tables.clone()
    t[b.slots[0], 1] = t[b.slots[1], 2] = t[b.slots[1], 0] = zero
    b.tables, b.d_tables = t, t.cuda()
    b.check(out)
    pos, slot, place = b.describe()
    b.tables[b.slots[1], 5] = -1
    last = b.describe()[2].clone()
    assert (last >= -1).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("window,first", [(0, 0), (70, 4), (200, 130)])
def test_nan_and_infinities(form, window, first):
    """What a row meets is in its result and in no other request's; what nobody sees is in nobody's."""
    runs = [(1, 300), (40, 100), (1, 7), (90, 60)]
    b = Batch(runs, window=window, first=first, poison=True, sink=True, **form)
    clean = run(b).clone()
    b.check(clean)
    g = b.H // b.G
    ends = [0]
    for n in b.new:
        ends.append(ends[-1] + n)
    place = lambda i, at: int(b.tables[b.slots[i], at // b.P]) * b.P + at % b.P
    # a query
    kept = b.q.clone()
    b.q[ends[1] + 3, 5] = math.nan
    out = run(b)
    assert out[ends[1] + 3, 5].isnan().all()
    out[ends[1] + 3, 5] = clean[ends[1] + 3, 5]
    assert torch.equal(out, clean)
    b.q = kept
    # a key of key/value head 1 of request 3, at a position that the last row sees
    at = place(3, b.length[3] - 2)
    kept = b.pool[at].clone()
    b.pool[at, b.D:b.D + 3] = math.nan
    out = run(b)
    r = ends[4] - 1
    assert out[r, g:].isnan().all() and not out[r, :g].isnan().any()
    assert torch.equal(out[:ends[3]], clean[:ends[3]])
    before = slice(ends[3], ends[4] - 2)                  # rows that stand before it
    assert torch.equal(out[before], clean[before])
    b.pool[at] = kept
    # a value: its column of its rows; others of the block may have it
    b.pool[at, b.G * b.D + b.V + 2] = math.inf
    out = run(b)
    assert (out[r, g:, 2].isinf() | out[r, g:, 2].isnan()).all() and torch.equal(out[r, :g], clean[r, :g])
    assert torch.equal(out[:ends[3]], clean[:ends[3]])
    b.pool[at] = kept
    # gate and sink
    b.gate[ends[2], 1] = math.nan
    b.sink[2] = math.nan
    out = run(b)
    assert out[ends[2], 1].isnan().all() and out[:, 2].isnan().all() and torch.equal(out[:, 3:], clean[:, 3:])
    # scores of minus infinity alone: 0 / 0
    b = Batch([(1, 0)], gate=False, **form)
    b.q[0, 0] = 0
    b.q[0, 0, 0] = 1
    b.pool[place_of(b, 0), 0] = -math.inf
    assert run(b)[0, 0].isnan().all()


def place_of(b, at):
    return int(b.tables[b.slots[0], at // b.P]) * b.P + at % b.P


@pytest.mark.parametrize("form", FORMS)
def test_scores_of_hundreds(form):
    """Maxima that rise from tile to tile, and first keys that outweigh all others."""
    b = Batch([(1, 1500), (60, 700), (200, 0)], sharp=1.0, gate=False, **form)
    for s, n in zip(b.slots, b.length):
        at = torch.arange(n)
        rows = b.tables[s].long()[at // b.P] * b.P + at % b.P
        scale = torch.linspace(0.1, 12, n, device="cuda") if s != b.slots[1] else torch.linspace(12, 0.1, n, device="cuda")
        b.pool[rows.cuda(), :b.G * b.D] *= scale[:, None].to(b.dtype)
    b.check(run(b))


@pytest.mark.parametrize("form", FORMS)
def test_twice_the_same(form):
    """Bit for bit, from a workspace that other passes have used."""
    b = Batch([(1, 4000), (1, 90), (20, 2500), (1, 6000)], sink=True, **form)
    outs = []
    for _ in range(4):
        outs.append(run(b).clone())
        b.p.part_o.fill_(math.nan)
        b.p.part_ml.fill_(math.nan)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    assert not b.p.counters.any()
    b.check(outs[0])


@pytest.mark.parametrize("form", FORMS)
def test_captured_and_replayed_over_other_requests(form):
    """Description, heads and attention in one graph, which follows its tensors."""
    m = ragged()
    b = Batch([(1, 300), (9, 100), (0, 10), (2, 0)], pads=30, **form)
    slots, new, length, tables = b.d_slots.clone(), b.d_new.clone(), b.d_length.clone(), b.d_tables.clone()
    H, G, D, V = b.H, b.G, b.D, b.V
    qkv = torch.randn(b.R, (H + G) * D + G * V, device="cuda").to(b.dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x, d in zip(qkv.split([H * D, G * D, G * V], 1), (D, D, V)))
    freq = 100.0 ** -(torch.arange(D // 2, device="cuda", dtype=F32) / (D // 2))
    w = torch.rand(D, device="cuda") + 0.5
    turned, out = torch.zeros(b.R, H, D, dtype=b.dtype, device="cuda"), torch.zeros(b.R, H, V, dtype=b.dtype, device="cuda")

    def layer():
        pos, _, place = b.p.describe(slots, new, length, tables, b.pages)
        m.heads_to_cache(q, k, v, pos, place, b.pool, q_norm=w, k_norm=w, freq=freq, out=turned)
        m.attend(turned, b.pool, tables, b.p, scale=b.scale, gate=b.gate, out=out)

    layer()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    order = [2, 0, 3, 1]
    for trial in range(3):
        # other tokens, other lengths, another order
        b.new = [4, 1, 0, 11] if trial == 0 else [0, 2, 7, 1] if trial == 1 else [1, 1, 1, 1]
        b.length = [n + x for n, x in zip(b.new, [7, 250, 64, 60] if trial != 1 else [0, 90, 0, 99])]
        b.slots = [b.slots[i] for i in order]
        grow = torch.full_like(b.tables, -1)
        free = list(range(b.pages))
        for s, x in zip(b.slots, b.length):
            for pg in range(-(-x // b.P)):
                grow[s, pg] = free.pop()
        b.tables, b.total = grow, sum(b.new)
        dev = lambda x: torch.tensor(x, dtype=I32, device="cuda")
        slots.copy_(dev(b.slots)), new.copy_(dev(b.new)), length.copy_(dev(b.length)), tables.copy_(grow)
        qkv.copy_(torch.randn_like(qkv, dtype=F32).to(b.dtype))
        graph.replay()
        torch.cuda.synchronize()
        b.p.check_status()
        b.q, b.d_tables = turned, tables
        b.check(out)


def test_two_streams_with_a_pass_each():
    a = Batch([(1, 3000), (40, 900), (1, 5)], seed=1)
    b = Batch([(100, 700), (1, 2000)], seed=2, window=300, first=5)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, x in ((one, a), (two, b)):
            with torch.cuda.stream(s):
                x.describe()
                outs.append((x, x.attend()))
    torch.cuda.synchronize()
    for x, out in outs[-4:]:
        x.check(out)


def test_far_places():
    """A pool of more than 2^31 values and pages at its end; a position behind a hundred thousand others."""
    b = Batch([(1, 100000), (3, 500)], heads=16, kv_heads=8, dim=128, vdim=128, window=500, first=3)
    more = (1 << 31) // (2048 * 64) + 200
    pool = torch.empty(more * 64, 2048, dtype=BF16, device="cuda")
    pool[-b.pages * 64:] = b.pool
    shift = more - b.pages
    b.tables = torch.where(b.tables >= 0, b.tables + shift, -1)
    b.pool, b.d_tables, b.pages = pool, b.tables.cuda(), more
    b.check(run(b))
    pos, slot, place = b.p.describe(b.d_slots, b.d_new, b.d_length, b.d_tables, b.pages)
    k, v = (torch.randn(b.R, 8, 128, device="cuda").to(BF16) for _ in range(2))
    ragged().heads_to_cache(b.q, k, v, pos, place, pool)
    assert torch.equal(pool[place[0].item()], torch.cat([k[0].flatten(), v[0].flatten()]))


def test_heads_in_place():
    """Queries over themselves."""
    m = ragged()
    for dtype, D, rot in ((BF16, 128, 128), (F32, 64, 32), (BF16, 24, 10)):
        q, k, v = (torch.randn(50, h, D, device="cuda").to(dtype) for h in (6, 2, 2))
        pos = torch.arange(50, dtype=I32, device="cuda") * 1000
        place = torch.arange(50, dtype=I32, device="cuda")
        freq = torch.rand(rot // 2, device="cuda")
        w = torch.rand(D, device="cuda")
        pools = [torch.zeros(64, 2 * 2 * D, dtype=dtype, device="cuda") for _ in range(2)]
        want = m.heads_to_cache(q, k, v, pos, place, pools[0], q_norm=w, k_norm=w, freq=freq)
        got = m.heads_to_cache(q, k, v, pos, place, pools[1], q_norm=w, k_norm=w, freq=freq, out=q)
        assert got is q and torch.equal(got, want) and torch.equal(*pools)


def test_heads_of_padded_width():
    """Heads of 40 values in 48, the rest zeros, normed over the 40; no norm on the keys."""
    m = ragged()
    q = torch.randn(9, 4, 48, device="cuda")
    q[..., 40:] = 0
    k, v = q[:, :2].contiguous(), torch.randn(9, 2, 16, device="cuda")
    pool = torch.zeros(16, 2 * 64, device="cuda")
    at = torch.arange(9, dtype=I32, device="cuda")
    w = torch.rand(48, device="cuda")
    got = m.heads_to_cache(q, k, v, at, at, pool, q_norm=w, eps=1e-5, width=40)
    want = q.double() / (q[..., :40].double().square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
    assert ((got - want).abs() <= want.abs() * 2 ** -18 + 1e-30).all()
    assert torch.equal(pool[:9, :96].view(9, 2, 48), k)


@pytest.mark.parametrize("name", ["freq", "q", "norm"])
def test_heads_keep_nan(name):
    m = ragged()
    q, k, v = (torch.randn(5, h, 64, device="cuda") for h in (2, 1, 1))
    at, pool = torch.arange(5, dtype=I32, device="cuda"), torch.zeros(8, 128, device="cuda")
    freq, w = torch.rand(32, device="cuda"), torch.rand(64, device="cuda")
    if name == "freq":
        freq[3] = math.inf
    elif name == "q":
        q[2, 1, 7] = math.nan
    else:
        w[9] = math.nan
    out = m.heads_to_cache(q, k, v, at, at, pool, q_norm=w, freq=freq)
    bad = out.isnan()
    want = torch.zeros_like(bad)
    if name == "freq":
        want[:, :, [3, 35]] = True
    elif name == "q":
        want[2, 1] = True
    else:
        want[:, :, [9, 41]] = True
    assert torch.equal(bad, want)


def test_random_passes():
    """Whatever comes: sizes, windows, mixtures."""
    rng = random.Random(11)
    for trial in range(25):
        heads, kv = rng.choice([(8, 2), (16, 4), (6, 2), (5, 5), (12, 1), (28, 4)])
        dim, vdim = rng.choice([(64, 64), (128, 128), (32, 48), (80, 16), (192, 128), (16, 112)])
        window = rng.choice([0, 0, 1, 17, 128, 700])
        runs = [(rng.choice([1, 1, 1, 2, rng.randint(1, 300)]), rng.choice([0, rng.randint(0, 3000)])) for _ in range(rng.choice([1, 4, 20]))]
        b = Batch(runs, heads=heads, kv_heads=kv, dim=dim, vdim=vdim, P=rng.choice([16, 32, 64, 128, 48]), window=window,
                  first=rng.choice([0, 1, 5, 64, 200]) if window else 0, seed=trial, poison=rng.random() < 0.5, sink=rng.random() < 0.5,
                  gate=rng.random() < 0.5, pads=rng.choice([0, 2]), dtype=rng.choice([BF16, BF16, F32]) if sum(n for n, _ in runs) < 400 else BF16)
        b.check(run(b))
