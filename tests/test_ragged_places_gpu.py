"""New tokens whose own page is not leased.  Values are compared as in test_ragged_gpu.py, whose passes these are."""
import math

import pytest
import torch

from test_ragged_gpu import BF16, F32, I32, Batch, ragged

pytestmark = pytest.mark.gpu
FORMS = [dict(heads=8, kv_heads=2, dim=64, vdim=64, P=64), dict(heads=8, kv_heads=2, dim=64, vdim=64, P=24),
         dict(heads=8, kv_heads=2, dim=64, vdim=64, P=32, dtype=F32), dict(heads=8, kv_heads=2, dim=64, vdim=192, P=64),
         dict(heads=32, kv_heads=1, dim=128, vdim=128, P=16)]
# decode in many pieces, a prompt's portion over three pages or more, a few tokens, a whole request
MISSING = [(0, 9000), (1, 130), (1, 259), (3, 70), (4, 2)]


def taken_out(**form):
    """A pass with new tokens on pages that are not leased, or have a number that the pool does not have, and which rows those are."""
    b = Batch([(1, 9000), (200, 100), (1, 511), (4, 67), (3, 0), (1, 20)], pads=2, sink=True, **form)
    whole = b.tables.clone()
    for j, (i, at) in enumerate(MISSING):
        b.tables[b.slots[i], at // b.P] = -1 if j % 2 == 0 else b.pages + j
    b.d_tables = b.tables.cuda()
    lost = torch.tensor([not 0 <= int(b.tables[b.slots[i], at // b.P]) < b.pages for i, at in b.rows] + [False] * 2, device="cuda")
    # what is read of them: zeros
    zero = int(set(range(b.pages)).difference(whole.flatten().tolist()).pop())
    b.pool[zero * b.P:(zero + 1) * b.P] = 0
    read = torch.where((b.tables >= 0) & (b.tables < b.pages), b.tables, zero)
    return b, lost, torch.where(whole >= 0, read, -1)


def same(b, out, lost, read):
    """Zeros where a token has no place, and what others see of those positions is zeros."""
    assert lost.any() and (out[lost] == 0).all()
    live = torch.arange(b.R, device="cuda") < b.total
    assert not out[live].isnan().any()
    a, kept, checked = 0, b.d_tables, out.clone()
    b.d_tables = read.cuda()
    gate, b.gate = b.gate, b.gate.clone()
    b.gate[lost] = -math.inf                  # of these the definition is zero as well
    b.q = torch.where(lost[:, None, None], torch.zeros_like(b.q), b.q)
    b.check(checked)
    b.d_tables, b.gate = kept, gate


@pytest.mark.parametrize("form", FORMS)
def test_queries_that_nobody_made(form):
    """Whatever lies where the query of a token without a place would be, its result is zeros and nobody else's is moved."""
    b, lost, read = taken_out(**form)
    b.q[lost] = math.nan
    b.describe()
    out = torch.full((b.R, b.H, b.V), math.nan, dtype=b.dtype, device="cuda")
    b.attend(out=out)
    assert out[b.total:].isnan().all()
    same(b, out, lost, read)


@pytest.mark.parametrize("window,first", [(0, 0), (150, 5)])
@pytest.mark.parametrize("form", FORMS)
def test_heads_and_attention_together(form, window, first):
    """Queries into a buffer of NaN, keys and values into the pool, and the attention of both."""
    m = ragged()
    b, lost, read = taken_out(window=window, first=first, **form)
    H, G, D, V = b.H, b.G, b.D, b.V
    qkv = torch.randn(b.R, (H + G) * D + G * V, device="cuda").to(b.dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x, d in zip(qkv.split([H * D, G * D, G * V], 1), (D, D, V)))
    w = torch.rand(D, device="cuda") + 0.5
    freq = 100.0 ** -(torch.arange(D // 2, device="cuda", dtype=F32) / (D // 2))
    turned = torch.full((b.R, H, D), math.nan, dtype=b.dtype, device="cuda")
    pos, slot, place = b.describe()
    m.heads_to_cache(q, k, v, pos, place, b.pool, q_norm=w, k_norm=w, freq=freq, out=turned)
    assert turned[lost].isnan().all() and not turned[:b.total][~lost[:b.total]].isnan().any()
    b.q = turned
    out = torch.full((b.R, H, V), math.nan, dtype=b.dtype, device="cuda")
    b.attend(out=out)
    same(b, out, lost, read)


@pytest.mark.parametrize("by_rows", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_places(form, by_rows):
    """A token whose page has no number, or one that the pool does not have, has place -1; every other one has its own; and it is told."""
    from ds41rt_b200.ops.lib import KernelError
    b, lost, read = taken_out(**form)
    n = b.total
    at = torch.tensor([p for _, p in b.rows], dtype=I32, device="cuda")
    of = torch.tensor([b.slots[i] for i, _ in b.rows], dtype=I32, device="cuda")
    pos, slot, place = b.p.describe_rows(at, of, b.d_tables, b.pages) if by_rows else b.describe()
    assert torch.equal(pos[:n], at) and torch.equal(slot[:n], of)
    want = b.d_tables[of.long(), (at // b.P).long()] * b.P + at % b.P
    assert torch.equal(place[:n], torch.where(lost[:n], -1, want)) and (place[n:] == -1).all()
    b.p.describe(b.d_slots[:0], b.d_new[:0], b.d_length[:0], b.d_tables, b.pages)          # a pass that has none
    rows = lost.nonzero().flatten().tolist()
    with pytest.raises(KernelError, match=f"{len(rows)} new tokens are on pages that are not leased, the lowest row of them {rows[0]}"):
        b.p.check_status()
    b.p.check_status()


def test_an_engine_tells_of_pages_that_are_not_leased():
    """A pass beyond a slot's lease and one within it: told once; what the second gives is as if the first had not been."""
    from ds41rt_b200.ops.lib import KernelError
    from test_ragged_engine_gpu import Model, close, config, engine, tokens
    model = Model(config())
    for dtype in ("f32", "bf16"):
        e = engine(model, dtype)
        t = tokens(32, 4)
        e.cache.ensure(0, 32)                       # a page of 32
        for n in (40, 32):
            e.set_rows((t + t)[:n], range(n), [0] * n)
            e.forward_rows(n, head=False)
            got = e.logits_at(range(n))
            assert not got.isnan().any() and close(got[31], model.logits(t)[-1], dtype)
        with pytest.raises(KernelError, match="8 new tokens are on pages that are not leased, the lowest row of them 32"):
            e.check_status()
        e.check_status()
