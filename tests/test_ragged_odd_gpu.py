"""Heads of odd widths and odd numbers, and of the largest that a call takes, against the definition in 64 bits.

Tolerances as in test_ragged_gpu.py: a mean of D squares and its root, D 2^-24 + 2^-21, relative; a rotation 2^-20 of |a| + |b|; a rounding
to the type, 2^-24 or 2^-8."""
import pytest
import torch

from test_ragged_gpu import Batch

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def check(R, H, G, D, V, rot, dtype):
    from ds41rt_b200.ops import ragged as m
    gen = torch.Generator(device="cuda").manual_seed(H + D)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")
    qkv = rnd(R, (H + G) * D + G * V).to(dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x, d in zip(qkv.split([H * D, G * D, G * V], 1), (D, D, V)))
    pos = torch.arange(R, dtype=I32, device="cuda") * 977
    place = torch.arange(R, dtype=I32, device="cuda").flip(0)
    w = 1 + 0.3 * rnd(D)
    freq = 10000.0 ** -(torch.arange(rot // 2, device="cuda", dtype=F32) / max(1, rot // 2))
    pool = torch.zeros(R, G * (D + V), dtype=dtype, device="cuda")
    out = m.heads_to_cache(q, k, v, pos, place, pool, q_norm=w, k_norm=w, eps=1e-5, freq=freq)
    u, half = 2 ** -8 if dtype == BF16 else 2 ** -24, rot // 2

    def reference(x):
        x = x.double()
        x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        rel = D * 2 ** -24 + 2 ** -21
        angle = pos.double()[:, None, None] * freq.double()
        a, b = x[..., :half], x[..., half:rot]
        y = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., rot:]], -1)
        tol = x.abs() * rel
        tol[..., :half] = tol[..., half:rot] = (a.abs() + b.abs()) * (rel + 2 ** -20)
        return y, tol + u * y.abs() + 1e-30

    y, tol = reference(q)
    assert ((out.double() - y).abs() <= tol).all()
    rows = pool[place.long()]
    y, tol = reference(k)
    assert ((rows[:, :G * D].double().unflatten(1, (G, D)) - y).abs() <= tol).all()
    assert torch.equal(rows[:, G * D:], v.flatten(1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,D,V,rot", [(2, 1, 15, 8, 8), (2, 1, 7, 3, 6), (1, 2, 9, 1, 2), (4, 1, 33, 16, 32), (3, 2, 1, 1, 0), (1, 1, 17, 5, 16)])
def test_odd_heads(H, G, D, V, rot, dtype):
    check(37, H, G, D, V, rot, dtype)


@pytest.mark.parametrize("H,G,D,rot", [(64, 2, 768, 768), (48, 1, 1024, 1024), (64, 2, 768, 0), (395, 1, 128, 128), (4000, 224, 12, 12)])
def test_rows_of_the_most_head_values(H, G, D, rot):
    """Up to 50688 values, and all of them turned."""
    check(3, H, G, D, 4, rot, BF16)


@pytest.mark.parametrize("form", [dict(heads=8, kv_heads=2, dim=128, vdim=128, P=64), dict(heads=8, kv_heads=2, dim=64, vdim=64, P=24),
                                  dict(heads=8, kv_heads=2, dim=256, vdim=256, P=32, dtype=F32)])
def test_attention_in_place_of_its_queries(form):
    """Requests in many pieces, blocks of many rows and of few."""
    b = Batch([(1, 9000), (300, 200), (7, 500), (65, 0), (1, 3)], window=0, sink=True, **form)
    b.describe()
    want = b.attend()
    q = b.q.clone()
    assert b.attend(out=b.q) is b.q and torch.equal(b.q, want)
    b.q = q
    b.check(want)


@pytest.mark.parametrize("dtype,more", [(F32, 4), (F32, 12), (BF16, 8)])
def test_attention_of_rows_at_16_bytes(dtype, more):
    b = Batch([(1, 900), (70, 20), (5, 64)], heads=6, kv_heads=2, dim=64, vdim=48, P=32, dtype=dtype, pads=1)
    b.describe()
    want = b.attend()
    b.check(want)
    wide = torch.full((b.R, b.H, b.D + more), 5.0, dtype=dtype, device="cuda")
    wide[..., :b.D] = b.q
    b.q = wide[..., :b.D]
    store = torch.full((b.R, b.H * b.V + more), 3.0, dtype=dtype, device="cuda")
    out = store[:, :b.H * b.V].unflatten(1, (b.H, b.V))
    b.attend(out=out)
    assert torch.equal(out[:b.total], want[:b.total]) and (store[:, b.H * b.V:] == 3).all() and (store[b.total:] == 3).all()


@pytest.mark.parametrize("by_rows", [False, True])
@pytest.mark.parametrize("window,first", [(0, 0), (300, 70)])
def test_the_largest_description(window, first, by_rows):
    """As many rows, requests and blocks as a pass takes: every row's numbers, and every (row, head) in one block's pieces."""
    from ds41rt_b200.ops import ragged as m
    R, n, P, G = 1 << 18, 4096, 64, 2
    p = m.RaggedPass(rows=R, requests=n, heads=4 * G, kv_heads=G, dim=64, vdim=64, page_tokens=P, window=window, first=first, device="cuda")
    assert p.max_blocks == m.MOST_BLOCKS and p.unit_tokens == 64
    gen = torch.Generator().manual_seed(2)
    new = torch.randint(0, 129, (n,), generator=gen)
    new[new.cumsum(0) > R] = 0
    new[17] = 0
    new[-1] += R - new.sum() if new.sum() < R else 0
    assert new.sum() == R
    before = torch.randint(0, 3000, (n,), generator=gen)
    length = new + before
    width = int(length.max()) // P + 1
    slots = torch.randperm(n, generator=gen)
    table = torch.randperm(n * width, generator=gen).view(n, width).to(I32).cuda()
    of = torch.repeat_interleave(torch.arange(n), new)
    start = new.cumsum(0) - new
    at = before[of] + torch.arange(R) - start[of]
    dev = lambda x: x.to(I32).cuda()
    if by_rows:
        got = p.describe_rows(dev(at), dev(slots[of]), table, n * width)
    else:
        got = p.describe(dev(slots), dev(new), dev(length), table, n * width)
    p.check_status()
    pos, slot = dev(at), dev(slots[of])
    place = table[slot.long(), (pos // P).long()] * P + pos % P
    assert all(torch.equal(x, y) for x, y in zip(got, (pos, slot, place)))
    count, total = p.header[:2].tolist()
    assert total == R and 0 < count <= p.max_units
    u = p.units.view(-1, m.UNIT)[:count].cpu().long()
    s, row0, tokens, pos0, head, tile0, tiles, piece, pieces, cell, counter, step = u.T
    assert (tokens > 0).all() and (tokens <= 64).all() and (s == slots[of[row0]]).all() and (pos0 == at[row0]).all()
    assert (of[row0] == of[row0 + tokens - 1]).all() and (counter < p.counters.numel()).all()
    begins = torch.zeros(G * (R + 1), dtype=torch.long)
    first_piece = piece == 0
    begins.index_add_(0, (head * (R + 1) + row0)[first_piece], torch.ones_like(row0[first_piece]))
    begins.index_add_(0, (head * (R + 1) + row0 + tokens)[first_piece], -torch.ones_like(row0[first_piece]))
    assert (begins.view(G, -1).cumsum(1)[:, :R] == 1).all()
    assert first_piece.sum() == (1 / pieces.double()).sum().round() and ((cell + (piece + 1) * step)[pieces > 1] <= p.max_cells).all()
