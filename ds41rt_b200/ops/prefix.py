"""Attention of a batch whose requests share a prefix (csrc/kernels/prefix_attn.cu, prefix_group.cu, prefix_latent.cu).

Requests that continue the same tokens keep the pages of the common part once: their page tables begin with the same pages.
`group_attend` and `latent_attend` give every row of a pass what `ds41_group_attend` and `ds41_latent_attend` give it (its
attention over all cached positions up to its own, or over its chunk of them), but read the common pages once for all rows that
share them; each row reads only what follows by itself, and the parts are joined by their maxima and sums.

Which rows share what is a `PrefixPlan`, made on the host from the page tables.  It holds as long as the rows belong to the same
slots and those keep their leading pages: pages added at a table's end leave it valid, so a decode loop makes it once for a batch.
It also holds the workspace of the calls, so calls with one plan follow one another on one stream; concurrent streams, or graphs
that replay at the same time, need a plan each.  A captured call reads the plan from device memory: after `set()` a replay uses the
new one.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import lib
from . import stack as S

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SMS = 148                # of a B200: plans do not depend on the device found
ITEM = 8                 # numbers of an item (ds41_prefix_plan)
MAX_PARTS = 160          # parts of a row's prefix that a join takes
MAX_OWN = 32             # splits of a row's own keys (latent attention)


class PlanArgs(C.Structure):
    _fields_ = [("items", C.c_void_p), ("n_items", C.c_void_p), ("order", C.c_void_p), ("own", C.c_void_p), ("cell", C.c_void_p),
                ("parts", C.c_void_p), ("part_o", C.c_void_p), ("part_ml", C.c_void_p), ("max_items", C.c_int),
                ("rows_per_item", C.c_int), ("grid", C.c_int)]


def common_runs(tables: np.ndarray) -> List[Tuple[List[int], int]]:
    """Groups of rows of a page table that begin with the same leased pages: (rows, common pages), a row in one group at most.

    Sorted, rows with a common beginning stand next to each other, and a range of them shares the least of the runs between
    neighbours.  The range that saves most reads, (rows - 1) x pages, is a group; the rows on either side of it are divided again."""
    order = sorted(range(len(tables)), key=lambda i: tables[i].tobytes())
    t = tables[order]
    same = (t[1:] == t[:-1]) & (t[1:] >= 0)
    runs = np.where(same.all(1), t.shape[1], same.argmin(1)) if len(t) > 1 else np.zeros(0, dtype=np.int64)
    out, todo = [], [(0, len(runs))]
    while todo:
        lo, hi = todo.pop()
        best = (0, 0, 0, 0)
        rising: List[Tuple[int, int]] = []               # (first run, height) of the ranges that are still open
        for i in range(lo, hi + 1):
            h, at = (int(runs[i]) if i < hi else 0), i
            while rising and rising[-1][1] >= h:
                at, top = rising.pop()
                best = max(best, ((i - at) * top, top, at, i))
            rising.append((at, h))
        gain, pages, a, b = best
        if gain == 0:
            continue
        out.append(([order[i] for i in range(a, b + 1)], pages))
        todo += [(lo, max(lo, a - 1)), (min(hi, b + 1), hi)]
    return out


def key_span(work: Sequence[Tuple[int, int]], budget: int, unit: int) -> int:
    """Keys of an item, where `work` lists (pieces, keys) of every prefix and `budget` items run at once: the shortest range that
    keeps one wave of items, or of two waves where shorter ones win by more than an item's fixed cost."""
    longest = max(keys for _, keys in work)
    best = None
    for waves in (1, 2):
        lo, hi = 1, -(-longest // unit)
        if sum(n for n, _ in work) > budget * waves:
            continue
        while lo < hi:
            mid = (lo + hi) // 2
            if sum(n * -(-keys // (mid * unit)) for n, keys in work) <= budget * waves:
                hi = mid
            else:
                lo = mid + 1
        cost = waves * (lo * unit + ITEM_COST)
        if best is None or cost < best[0]:
            best = (cost, lo * unit)
    return max(best[1] if best else longest, -(-longest // (MAX_PARTS * unit)) * unit)


ITEM_COST = 512          # fixed cost of an item, in keys


class PrefixPlan:
    """Rows that share leading pages, how their attention is divided, and the workspace of the calls.

    `kind`: "grouped" or "latent"; `rows`: most rows of a pass; `heads`, `kv_heads`, `vdim`: of the attention (latent: one key / value
    head, `vdim` the padded latent width)."""

    def __init__(self, kind: str, *, rows: int, heads: int, vdim: int, page_tokens: int, device, kv_heads: int = 1, dtype=BF16,
                 min_tokens: int = 64):
        if kind not in ("grouped", "latent"):
            raise ValueError(f"a prefix plan is grouped or latent, not {kind!r}")
        if min(rows, heads, kv_heads, vdim, page_tokens) <= 0 or heads % kv_heads or vdim % 16:
            raise ValueError("sizes must be positive, kv_heads must divide heads, the value width must be a multiple of 16")
        if kind == "latent" and kv_heads != 1:
            raise ValueError("latent attention has one key / value head")
        if dtype not in (BF16, F32):
            raise ValueError(f"cache rows are bf16 or fp32, not {dtype}")
        self.kind, self.rows, self.heads, self.kv_heads, self.vdim = kind, rows, heads, kv_heads, vdim
        self.page_tokens, self.dtype, self.device = page_tokens, dtype, torch.device(device)
        self.min_tokens = min_tokens
        per_lane = heads // kv_heads
        self.rows_per_item = max(1, (256 if kind == "grouped" else 128) // per_lane)
        pair = kind == "latent" and vdim > 256               # two CTAs to an item
        self.budget = max(1, (SMS // 2 if pair else SMS) // kv_heads)
        self.max_items = 2 * self.budget + rows
        self.max_cells = 2 * self.budget * min(self.rows_per_item, rows) + rows
        self.own_cells = rows * self._own_splits(rows, 1 << 30) if kind == "latent" else 0
        z = lambda n, d: torch.zeros(max(n, 4), dtype=d, device=self.device)
        # [count, 3 unused | items | order | own | cell | parts]
        self._at = np.cumsum([4, ITEM * self.max_items, rows, rows, rows]).tolist()
        self.data = z(self._at[-1] + rows, I32)
        self.part_o, self.part_ml = z(self.max_cells * heads * vdim, F32), z(self.max_cells * heads * 2, F32)
        self.own_o, self.own_ml = z(self.own_cells * heads * vdim, F32), z(self.own_cells * heads * 2, F32)
        self.status = lib.new_status(self.device)
        self.n_items = 0
        self.shared: List[Tuple[List[int], int]] = []      # rows and tokens of every prefix
        self.least_own = 0
        a, base = PlanArgs(), self.data.data_ptr()
        a.n_items, (a.items, a.order, a.own, a.cell, a.parts) = base, (base + 4 * x for x in self._at)
        a.part_o, a.part_ml = self.part_o.data_ptr(), self.part_ml.data_ptr()
        a.max_items, a.rows_per_item = self.max_items, self.rows_per_item
        a.grid = min(self.max_items * kv_heads, SMS)
        self.args = a

    def _own_splits(self, rows: int, tokens: int) -> int:
        return max(1, min(2 * SMS // (rows * -(-self.heads // 32)), MAX_OWN, -(-tokens // 64)))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.data, self.part_o, self.part_ml, self.own_o, self.own_ml))

    def set(self, slots: Sequence[int], tables) -> None:
        """`slots`: the slot of every row of the passes to come (-1: none); `tables`: the page table on the host, [slots, pages],
        negative where no page is leased."""
        t = tables.numpy() if isinstance(tables, torch.Tensor) else np.asarray(tables)
        s = np.asarray(slots, dtype=np.int64)
        if t.ndim != 2 or t.dtype != np.int32:
            raise ValueError("the page table is a matrix of 32-bit integers")
        if s.ndim != 1 or len(s) > self.rows:
            raise ValueError(f"a plan for {self.rows} rows does not take {s.shape}")
        if len(s) and int(s.max()) >= len(t):
            raise ValueError(f"slot {int(s.max())} of {len(t)}")
        of = {}                                                # rows of every slot
        for r, slot in enumerate(s.tolist()):
            if slot >= 0:
                of.setdefault(slot, []).append(r)
        keep = list(of)
        runs = common_runs(t[keep]) if len(keep) > 1 else []
        self.shared = [(sorted(r for i in members for r in of[keep[i]]), pages * self.page_tokens) for members, pages in runs
                       if pages * self.page_tokens >= self.min_tokens]
        self._lay_out(s)

    def _lay_out(self, slots: np.ndarray) -> None:
        host = np.zeros(self.data.numel(), dtype=np.int32)
        items, order, own, cell, parts = (host[a:b] for a, b in zip(self._at, self._at[1:] + [len(host)]))
        pieces = [-(-len(rows) // self.rows_per_item) for rows, _ in self.shared]
        n = at = cells = 0
        if self.shared:
            span = key_span([(p, tokens) for p, (_, tokens) in zip(pieces, self.shared)], self.budget, max(128, self.page_tokens))
            todo = []
            for p, (rows, tokens) in zip(pieces, self.shared):
                count = -(-tokens // span)
                order[at:at + len(rows)] = rows
                own[rows], parts[rows] = tokens, count
                cell[rows] = cells + count * np.arange(len(rows))
                cells += count * len(rows)
                for i in range(p):
                    lo, hi = (len(rows) * j // p for j in (i, i + 1))
                    todo += [(int(slots[rows[0]]), at + lo, hi - lo, k * span, min(tokens, (k + 1) * span), k, 0, 0) for k in range(count)]
                at += len(rows)
            todo.sort(key=lambda x: x[3] - x[4])               # the longest ranges first
            n = len(todo)
            assert n <= self.max_items and cells <= self.max_cells, (n, cells)
            items[:ITEM * n] = np.asarray(todo, dtype=np.int32).ravel()
        host[0] = self.n_items = n
        live = [r for r in range(len(slots)) if slots[r] >= 0]
        self.least_own = int(own[live].min()) if live else 0
        self.data.copy_(torch.from_numpy(host))

    def check_status(self, what: str = "attention over a shared prefix"):
        lib.raise_on_status(self.status, what)


# ---------------------------------------------------------------------------------------------------- launches
def launch_group(a: S.GroupAttendArgs, plan: PrefixPlan) -> None:
    """Both launches of grouped attention; `a` as for ds41_group_attend."""
    k, st = lib.kernels("stack"), lib.stream()
    if plan.n_items or torch.cuda.is_current_stream_capturing():
        lib.check(k.ds41_prefix_group_shared(C.byref(a), C.byref(plan.args), st), "ds41_prefix_group_shared")
    lib.check(k.ds41_prefix_group_own(C.byref(a), C.byref(plan.args), st), "ds41_prefix_group_own")


def launch_latent(a: S.LatentAttendArgs, plan: PrefixPlan, n_pages: int, sink, out: torch.Tensor, ld_out: int) -> None:
    """The launches of latent attention; `a` as for ds41_latent_attend, whose partial results lie in the plan."""
    k, st = lib.kernels("stack"), lib.stream()
    tokens = a.max_pages * a.page_tokens - (plan.least_own if not torch.cuda.is_current_stream_capturing() else 0)
    a.n_splits = plan._own_splits(a.rows, max(tokens, 1))
    a.part_o, a.part_ml = plan.own_o.data_ptr(), plan.own_ml.data_ptr()
    if plan.n_items or torch.cuda.is_current_stream_capturing():
        lib.check(k.ds41_prefix_latent_shared(C.byref(a), C.byref(plan.args), n_pages, st), "ds41_prefix_latent_shared")
    lib.check(k.ds41_prefix_latent_own(C.byref(a), C.byref(plan.args), st), "ds41_prefix_latent_own")
    lib.check(k.ds41_prefix_latent_merge(lib.ptr(plan.own_o), lib.ptr(plan.own_ml), lib.ptr(sink), C.byref(plan.args), a.n_splits, a.rows,
                                         a.heads, a.kv_pad, lib.ptr(out), ld_out, a.f32, st), "ds41_prefix_latent_merge")


def own_cluster(rows: int, heads: int, kv_heads: int, tokens: int) -> int:
    """CTAs that share a row's own keys in grouped attention."""
    blocks = rows * kv_heads * -(-(heads // kv_heads) // 16)
    n = max(1, min(SMS // blocks, 16, -(-tokens // 128)))
    return n if n <= 8 else (16 if n == 16 and blocks <= 4 else 8)


# ---------------------------------------------------------------------------------------------------- front end
def _check(plan: PrefixPlan, kind: str, q: torch.Tensor, pool, page_table, row_pos, row_slot, out, width: int, scale: float,
           named) -> int:
    if plan.kind != kind:
        raise ValueError(f"the plan is for {plan.kind} attention")
    if not scale > 0:
        raise ValueError("scale must be positive")
    R = q.shape[0]
    if not 0 < R <= plan.rows:
        raise ValueError(f"a pass has 1 to {plan.rows} rows, not {R}")
    for name, t in (("pool", pool), ("out", out)) + named:
        if t is not None and t.dtype != (F32 if name in ("gate", "sink") else plan.dtype):
            raise ValueError(f"{name} is {t.dtype}")
    for name, t in (("page_table", page_table), ("row_pos", row_pos), ("row_slot", row_slot)):
        if t.dtype != I32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous 32-bit integers")
    if page_table.dim() != 2 or row_pos.dim() != 1 or row_slot.dim() != 1 or row_pos.numel() < R or row_slot.numel() < R:
        raise ValueError("page_table is [slots, pages], row_pos and row_slot have an entry per row")
    if pool.dim() != 2 or not pool.is_contiguous() or pool.shape[1] != width or pool.shape[0] == 0 or pool.shape[0] % plan.page_tokens:
        raise ValueError(f"pool must be contiguous rows of {width} values, whole pages of {plan.page_tokens} of them")
    if pool.shape[0] >= 1 << 31:
        raise ValueError("a pool has fewer than 2^31 rows")
    if out.shape != (R, plan.heads, plan.vdim) or out.stride(2) != 1 or out.stride(1) != plan.vdim or out.stride(0) % 8:
        raise ValueError(f"out must be [{R}, {plan.heads}, {plan.vdim}], a row's heads side by side and rows at multiples of 8 values")
    if out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    here = torch.device("cuda", torch.cuda.current_device()) if plan.device.type == "cuda" and torch.cuda.is_available() else None
    for name, t in (("pool", pool), ("out", out), ("page_table", page_table), ("row_pos", row_pos), ("row_slot", row_slot),
                    ("plan", plan.data)) + named:
        if t is not None and t.device != here:
            raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")
    return R


def _heads(name: str, q: torch.Tensor, heads: int, dtype):
    if q.dim() != 3 or q.shape[1] != heads or q.dtype != dtype or q.shape[2] % 16 or q.shape[2] == 0:
        raise ValueError(f"{name} must be [rows, {heads}, a multiple of 16] of {dtype}")
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16 or q.stride(0) < q.stride(1) * (heads - 1) + q.shape[2]:
        raise ValueError(f"{name}: values of a head side by side, rows and heads at multiples of 8 values, 16-byte aligned")


def group_attend(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, row_pos: torch.Tensor, row_slot: torch.Tensor,
                 plan: PrefixPlan, *, scale: float, chunk: int = 0, gate: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of a pass over a paged cache, common pages read once: [rows, heads, vdim].

    q [rows, heads, dim]; pool [pages * page_tokens, kv_heads * (dim + vdim)]: keys of all key/value heads, then their values; row r
    stands at row_pos[r] of slot row_slot[r] (negative: the row's result is zero) and sees the positions up to its own, within its
    chunk of `chunk` of them where that is not 0.  `gate` [rows, heads] fp32: a head's result times sigmoid(gate)."""
    _heads("q", q, plan.heads, plan.dtype)
    R, H, D = q.shape
    if q.stride(1) != D:
        raise ValueError("q: a row's heads must lie side by side")
    if out is None:
        out = torch.empty(R, H, plan.vdim, dtype=plan.dtype, device=q.device)
    _check(plan, "grouped", q, pool, page_table, row_pos, row_slot, out, plan.kv_heads * (D + plan.vdim), scale,
           (("q", q), ("gate", gate)))
    if chunk < 0:
        raise ValueError("chunk must not be negative")
    if gate is not None and (gate.shape != (R, H) or gate.stride(1) != 1):
        raise ValueError(f"gate must be [{R}, {H}] with a row's values side by side")
    a = S.GroupAttendArgs()
    a.q, a.pool, a.out, a.status = lib.ptr(q), lib.ptr(pool), lib.ptr(out), lib.ptr(plan.status)
    a.page_table, a.row_pos, a.row_slot = lib.ptr(page_table), lib.ptr(row_pos), lib.ptr(row_slot)
    a.gate = S.Proj(gate, gate.stride(0)).args() if gate is not None else S.NO_PROJ
    a.u, a.taps, a.slots = S.NO_PROJ, 1, page_table.shape[0]
    a.ld_q, a.ld_out, a.scale, a.chunk = q.stride(0), out.stride(0), scale, chunk
    a.rows, a.heads, a.kv_heads, a.dim_pad, a.vdim_pad = R, H, plan.kv_heads, D, plan.vdim
    a.max_pages, a.page_tokens, a.f32, a.n_pages = page_table.shape[1], plan.page_tokens, int(plan.dtype == F32), \
        pool.shape[0] // plan.page_tokens
    span = a.max_pages * plan.page_tokens - (0 if torch.cuda.is_current_stream_capturing() else plan.least_own)
    a.n_splits = own_cluster(R, H, plan.kv_heads, max(1, min(span, chunk or span)))
    launch_group(a, plan)
    return out


def latent_attend(q_abs: torch.Tensor, q_rot: Optional[torch.Tensor], pool: torch.Tensor, page_table: torch.Tensor,
                  row_pos: torch.Tensor, row_slot: torch.Tensor, plan: PrefixPlan, *, scale: float,
                  sink: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Latent attention of a pass over a paged cache, common pages read once: [rows, heads, latent width].

    q_abs [rows, heads, latent], q_rot [rows, heads, rot] (None: no rotated part); pool [pages * page_tokens, latent + rot]: a
    position's latent, which is key and value of every head, and its rotated key part.  `sink` [heads] fp32: an extra logit in a
    head's denominator."""
    _heads("q_abs", q_abs, plan.heads, plan.dtype)
    R, H, V = q_abs.shape
    if V != plan.vdim:
        raise ValueError(f"q_abs: {V} latent values, the plan has {plan.vdim}")
    if q_abs.stride(1) != V:
        raise ValueError("q_abs: a row's heads must lie side by side")
    if q_rot is not None:
        _heads("q_rot", q_rot, H, plan.dtype)
        if q_rot.shape[0] != R:
            raise ValueError("q_rot must have as many rows as q_abs")
    rot = 0 if q_rot is None else q_rot.shape[2]
    if out is None:
        out = torch.empty(R, H, V, dtype=plan.dtype, device=q_abs.device)
    _check(plan, "latent", q_abs, pool, page_table, row_pos, row_slot, out, V + rot, scale,
           (("q_abs", q_abs), ("q_rot", q_rot), ("sink", sink)))
    if sink is not None and (sink.shape != (H,) or not sink.is_contiguous()):
        raise ValueError(f"sink must be {H} contiguous values")
    a = S.LatentAttendArgs()
    a.q_abs, a.ld_q_abs = lib.ptr(q_abs), q_abs.stride(0)
    if q_rot is not None:
        a.q_rot, a.ld_q_rot, a.q_rot_stride = lib.ptr(q_rot), q_rot.stride(0), q_rot.stride(1)
    a.pool, a.page_table, a.row_pos, a.row_slot = lib.ptr(pool), lib.ptr(page_table), lib.ptr(row_pos), lib.ptr(row_slot)
    a.scale, a.rows, a.heads, a.kv_pad, a.row_len = scale, R, H, V, V + rot
    a.max_pages, a.page_tokens, a.f32, a.status = page_table.shape[1], plan.page_tokens, int(plan.dtype == F32), lib.ptr(plan.status)
    launch_latent(a, plan, pool.shape[0] // plan.page_tokens, sink, out, out.stride(0))
    return out
