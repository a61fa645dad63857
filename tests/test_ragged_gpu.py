"""Ragged passes against their definitions in 64 bits, request by request.

Tolerances, per value, from the arithmetic (u = 2^-8 for bf16, 2^-24 for fp32: a rounding's largest relative error; w, v: the row's
attention weights and values, A = sum w |v|):
  scores   a product of D fp32 terms is off by at most (D + 2) 2^-23 sum |q k| (tensor cores may truncate: one bit more than a rounding
           each), scaled; a weight by twice that, relative, as its denominator moves too: 2 d A with d the largest over keys
  weights  the tensor-core form rounds them to bf16 as the operand of the second product, 2^-8 A; the exponential's argument (below 2^4
           where its weight counts) and value are good to 2^-20: 2^-19 A with the denominator
  sums     n fp32 terms: n 2^-23 A, twice for the denominator; joining parts: inside that
  result   u |o| of the rounding that it leaves with; the gate's factor 2^-20 |o|
Heads: a mean of D squares and its root, D 2^-24 + 2^-22, relative; two products and the factors of a rotation 2^-21 of |a| + |b|, sine and
cosine good to 2^-22; a rounding to the type.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def ragged():
    from ds41rt_b200.ops import ragged as m
    return m


class Batch:
    """`requests`: (new tokens, tokens before them) of each; None: one without a slot."""

    def __init__(self, requests, *, heads=8, kv_heads=2, dim=64, vdim=64, P=64, window=0, first=0, dtype=BF16, seed=0, pads=0, poison=False,
                 sharp=1.5, gate=True, sink=False, spare=0):
        rng, gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.H, self.G, self.D, self.V, self.P, self.window, self.first, self.dtype = heads, kv_heads, dim, vdim, P, window, first, dtype
        n = len(requests)
        self.new = [0 if r is None else r[0] for r in requests]
        for i, r in enumerate(requests):
            if r is None:
                self.new[i] = 3
        self.length = [5 if r is None else r[0] + r[1] for r in requests]
        ids = rng.sample(range(n + 2), n)
        self.slots = [-1 if r is None else s for s, r in zip(ids, requests)]
        self.total = sum(self.new)
        self.R = self.total + pads
        width = max(x // P + 1 for x in self.length) + 1
        self.tables = torch.full((n + 2, width), -1, dtype=I32)
        need = [0 if s < 0 else -(-x // P) for s, x in zip(self.slots, self.length)]
        self.pages = sum(need) + 3
        free = list(range(self.pages))
        rng.shuffle(free)
        for s, k in zip(self.slots, need):
            if s >= 0:
                self.tables[s, :k] = torch.tensor([free.pop() for _ in range(k)], dtype=I32)
        self.rows = []                                    # (request, position) of every row
        for i in range(n):
            self.rows += [(i, self.length[i] - self.new[i] + t) for t in range(self.new[i])]
        rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")
        self.pool = rnd(self.pages * P, kv_heads * (dim + vdim)).to(dtype)
        if poison:                                        # what no row of a request sees may be anything
            seen = torch.zeros(self.pages * P, dtype=torch.bool)
            for i, s in enumerate(self.slots):
                if s >= 0 and self.new[i]:
                    at = torch.arange(self.length[i])
                    low = max(0, self.length[i] - self.new[i] - window + 1) if window else 0
                    at = at[(at >= low) | (at < first)]
                    seen[self.tables[s].long()[at // P] * P + at % P] = True
            bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
            hidden = (~seen).nonzero().flatten().cuda()
            self.pool[hidden] = bad[hidden % 3][:, None].to(dtype)
        self.q = (rnd(self.R, heads, dim) * sharp).to(dtype)
        self.gate = rnd(self.R, heads) if gate else None
        self.sink = rnd(heads) if sink else None
        self.scale = dim ** -0.5
        dev = lambda x: torch.tensor(x, dtype=I32, device="cuda")
        self.d_slots, self.d_new, self.d_length, self.d_tables = dev(self.slots), dev(self.new), dev(self.length), self.tables.cuda()
        self.p = ragged().RaggedPass(rows=self.R, requests=n + spare, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, page_tokens=P,
                                     window=window, first=first, device="cuda", dtype=dtype)

    def describe(self):
        return self.p.describe(self.d_slots, self.d_new, self.d_length, self.d_tables, self.pages)

    def attend(self, **kw):
        return ragged().attend(self.q, self.pool, self.d_tables, self.p, scale=self.scale, gate=self.gate, sink=self.sink, **kw)

    def visible(self, pos, length):
        at = torch.arange(length, device="cuda")[None]
        p = pos[:, None]
        return (at <= p) & ((at > p - self.window) | (at < self.first)) if self.window else at <= p

    def check(self, out, form=None):
        """`out` [R, H, V] against 64 bits; rows behind the last are not looked at."""
        tiled = self.p.tiled if form is None else form
        u, G, D, V, g = (2 ** -8 if self.dtype == BF16 else 2 ** -24), self.G, self.D, self.V, self.H // self.G
        a = 0
        worst = 0.0
        for i, s in enumerate(self.slots):
            n, length = self.new[i], self.length[i]
            rows = slice(a, a + n)
            a += n
            if n == 0:
                continue
            if s < 0:
                assert (out[rows] == 0).all()
                continue
            at = torch.arange(length, device="cuda")
            kv = self.pool[self.d_tables[s].long()[at // self.P] * self.P + at % self.P].double()
            pos = torch.arange(length - n, length, device="cuda")
            seen = self.visible(pos, length)
            kv = torch.where(seen.any(0)[:, None], kv, 0.0)
            for h in range(self.H):
                k, v = kv[:, h // g * D:(h // g + 1) * D], kv[:, G * D + h // g * V:G * D + (h // g + 1) * V]
                q = self.q[rows, h].double()
                z = (q @ k.T * self.scale).masked_fill(~seen, -math.inf)
                d = ((q.abs() @ k.abs().T) * seen).amax(1) * self.scale * (D + 2) * 2 ** -23
                logits = z if self.sink is None else torch.cat([z, self.sink[h].double().expand(n, 1)], 1)
                w = torch.softmax(logits, 1)[:, :length]
                o, A = w @ v, w @ v.abs()
                tol = (2 * d[:, None] + 2 ** -19 + 3 * length * 2 ** -23) * A
                if tiled:
                    tol = tol + 2 ** -8 * A
                f = 1.0 if self.gate is None else torch.sigmoid(self.gate[rows, h].double())[:, None]
                o, tol = o * f, tol * f
                tol = tol + (u + 2 ** -20) * o.abs() + 2 ** -24 * A + 1e-30
                err = (out[rows, h].double() - o).abs()
                worst = max(worst, (err / tol).nan_to_num(math.inf).max().item())
                assert (err <= tol).all(), (i, h, worst, err.max().item())
        return worst


RUNS = {
    "one": [(1, 0)],
    "decode": [(1, 299), (1, 64), (1, 0), (1, 511)],
    "prompt": [(300, 0)],
    "mixed": [(1, 700), (37, 5), None, (0, 40), (130, 129), (1, 63), (2, 126), (64, 64)],
    "many": [(1 + (i * 5) % 7, (i * 131) % 900) for i in range(40)],
}
# (heads, kv_heads, dim, vdim, page): those of the tensor-core form, then others
TILED = [(8, 2, 64, 64, 64), (32, 8, 128, 128, 64), (6, 2, 32, 48, 32), (12, 1, 128, 128, 16), (4, 4, 192, 128, 128), (20, 4, 80, 16, 256),
         (128, 1, 64, 128, 64), (3, 1, 256, 32, 32), (5, 5, 256, 128, 16), (4, 1, 128, 256, 64), (8, 2, 256, 256, 64), (6, 3, 48, 160, 32)]
OTHERS = [(8, 2, 64, 64, 24), (4, 1, 128, 240, 64), (2, 2, 16, 16, 4), (200, 1, 32, 32, 64)]


def test_describe_rows_and_units():
    """Every row's numbers, and that the units have every (row, head, key) that is to be seen once."""
    m = ragged()
    rng = random.Random(5)
    for trial in range(30):
        heads, kv_heads, dim, vdim, P = rng.choice(TILED + OTHERS)
        window = rng.choice([0, 0, 1, 20, 130, 1000])
        b = Batch([None if rng.random() < 0.1 else (rng.choice([0, 1, 1, rng.randint(1, 400)]), rng.choice([0, rng.randint(0, 5000)]))
                   for _ in range(rng.choice([1, 3, 17, 200]))], heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, P=P, seed=trial, window=window,
                  first=rng.choice([0, 1, 70, 300]) if window else 0, pads=rng.choice([0, 1, 5]) + 1)
        pos, slot, place = (x.tolist() for x in b.describe())
        b.p.check_status()
        for r in range(b.R):
            if r >= b.total:
                assert (pos[r], slot[r], place[r]) == (0, -1, -1)
                continue
            i, at = b.rows[r]
            s = b.slots[i]
            want = -1 if s < 0 else int(b.tables[s, at // P]) * P + at % P
            assert (pos[r], slot[r], place[r]) == (at, s, want)
        n_units, total = b.p.header.tolist()[:2]
        assert total == b.total and n_units <= b.p.max_units
        units = b.p.units.view(-1, m.UNIT)[:n_units].tolist()
        group, align = heads // kv_heads, min(P, b.p.key_tile)
        pieces, cells = {}, []
        for s, row0, tokens, pos0, head, tile0, tiles, piece, of, cell, counter, step in units:
            assert 0 < tokens <= b.p.unit_tokens and step == tokens * group
            assert (slot[row0], pos[row0]) == (s, pos0) and b.rows[row0][0] == b.rows[row0 + tokens - 1][0]
            pieces.setdefault((row0, tokens, head), []).append((piece, of, tile0, tiles, cell, counter))
            if of > 1:
                cells.append((cell + piece * step, step))
        covered = {h: [0] * b.total for h in range(kv_heads * b.p.v_parts)}
        for (row0, tokens, head), found in pieces.items():
            found.sort()
            of = found[0][1]
            assert [f[0] for f in found] == list(range(of)) and len({f[4:] for f in found}) == 1
            at = 0
            for _, _, tile0, tiles, _, counter in found:
                assert tile0 == at and 0 <= counter < b.p.counters.numel()
                at += tiles
            for r in range(row0, row0 + tokens):
                covered[head][r] += 1
            if slot[row0] < 0:
                assert at == 0
                continue
            p0, p1 = pos[row0], pos[row0] + tokens - 1
            low = max(0, p0 - b.window + 1) if b.window else 0
            base = low // align * align
            lead = -(-min(b.first, p1 + 1) // align) * align if b.first else 0
            if lead and lead >= base:
                lead = base = 0
            if not b.first:
                lead = 0
            assert at == -(-(lead + p1 + 1 - base) // b.p.key_tile)
        assert all(c == 1 for h in covered.values() for c in h)
        cells.sort()
        assert all(a + n <= c for (a, n), (c, _) in zip(cells, cells[1:])) and all(c + n <= b.p.max_cells for c, n in cells)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", [(8, 2, 64, 64, 64, 64), (32, 8, 128, 128, 128, 64), (6, 2, 32, 48, 16, 32), (5, 1, 24, 7, 10, 8),
                                   (4, 4, 192, 128, 64, 16), (2, 1, 128, 128, 0, 64), (1, 1, 256, 256, 256, 64)])
@pytest.mark.parametrize("norm", ["shared", "own", "none"])
def test_heads(dtype, sizes, norm):
    m = ragged()
    H, G, D, V, rot, P = sizes
    gen = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")
    R, rows_pool = 45, 40 * P
    source = dtype if norm != "own" else (F32 if dtype == BF16 else BF16)
    qkv = rnd(R, (H + G) * D + G * V + 8).to(source)
    q, k, v = (x.unflatten(1, (-1, d)) for x, d in zip(qkv[:, :(H + G) * D + G * V].split([H * D, G * D, G * V], 1), (D, D, V)))
    pos = torch.tensor([0, 1, 2, 1 << 20, (1 << 24) + 1, 2 ** 31 - 5] + [37 * i for i in range(R - 6)], dtype=I32, device="cuda")
    place = torch.randperm(rows_pool, generator=torch.Generator().manual_seed(1))[:R].to(I32).cuda()
    place[[3, 9, R - 1]] = -1
    w = {"shared": lambda h: 1 + 0.3 * rnd(D), "own": lambda h: 1 + 0.3 * rnd(h, D), "none": lambda h: None}[norm]
    wq, wk = w(H), w(G)
    freq = 10000.0 ** -(torch.arange(rot // 2, device="cuda", dtype=F32) / max(1, rot // 2)) if rot else None
    pool = rnd(rows_pool, G * (D + V)).to(dtype)
    kept, out = pool.clone(), rnd(R, H, D).to(dtype)
    before = out.clone()
    got = m.heads_to_cache(q, k, v, pos, place, pool, q_norm=wq, k_norm=wk, eps=1e-5, freq=freq, out=out)
    assert got is out
    u = 2 ** -8 if dtype == BF16 else 2 ** -24

    def reference(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * weight.double()
        rel = (D * 2 ** -24 + 2 ** -21) if weight is not None else 0.0
        y, tol = x.clone(), x.abs() * rel
        if rot:
            h = rot // 2
            angle = pos.double()[:, None, None] * freq.double()
            a, b = x[..., :h], x[..., h:rot]
            y[..., :h], y[..., h:rot] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
            both = (a.abs() + b.abs()) * (rel + 2 ** -20)
            tol[..., :h], tol[..., h:rot] = both, both
        return y, tol + u * y.abs() + 1e-30

    live = place >= 0
    y, tol = reference(q, wq)
    assert ((out.double() - y).abs() <= tol)[live].all()
    assert torch.equal(out[~live], before[~live])
    y, tol = reference(k, wk)
    rows = pool[place[live].long()]
    assert ((rows[:, :G * D].double().unflatten(1, (G, D)) - y[live]).abs() <= tol[live]).all()
    assert torch.equal(rows[:, G * D:], v[live].flatten(1).to(dtype))
    kept[place[live].long()] = rows
    assert torch.equal(pool, kept)


@pytest.mark.parametrize("run", sorted(RUNS))
@pytest.mark.parametrize("sizes", OTHERS[:2] + [(8, 2, 64, 64, 64)])
def test_attend_32_bit(run, sizes):
    H, G, D, V, P = sizes
    b = Batch(RUNS[run], heads=H, kv_heads=G, dim=D, vdim=V, P=P, dtype=F32, pads=2, sink=True)
    b.describe()
    b.check(b.attend())
    b.p.check_status()


@pytest.mark.parametrize("run", ["decode", "mixed"])
@pytest.mark.parametrize("sizes", OTHERS)
def test_attend_other_sizes(run, sizes):
    H, G, D, V, P = sizes
    b = Batch(RUNS[run], heads=H, kv_heads=G, dim=D, vdim=V, P=P, window=100, first=3)
    assert not b.p.tiled
    b.describe()
    b.check(b.attend())


@pytest.mark.parametrize("run", sorted(RUNS))
@pytest.mark.parametrize("sizes", TILED)
def test_attend_tiled(run, sizes):
    H, G, D, V, P = sizes
    b = Batch(RUNS[run], heads=H, kv_heads=G, dim=D, vdim=V, P=P, pads=2, sink=run == "mixed", gate=run != "prompt")
    assert b.p.tiled
    b.describe()
    out = b.attend()
    b.p.check_status()
    b.check(out)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (50, 4), (64, 0), (65, 64), (128, 100), (300, 1000), (257, 2), (10000, 3)])
@pytest.mark.parametrize("sizes", [(8, 2, 64, 64, 64), (12, 1, 128, 128, 16), (6, 2, 32, 48, 32), (8, 2, 128, 128, 256), (4, 2, 64, 192, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_windows(window, first, sizes, dtype):
    H, G, D, V, P = sizes
    runs = [(1, 900), (70, 0), (200, 333), (1, 0), (5, 1200), (0, 9), None]
    b = Batch(runs, heads=H, kv_heads=G, dim=D, vdim=V, P=P, window=window, first=first, dtype=dtype, poison=True, sink=True)
    b.describe()
    out = b.attend()
    b.p.check_status()
    b.check(out)
