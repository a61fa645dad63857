"""Attention of a batch whose requests share a prefix (csrc/kernels/prefix_attn.cu, prefix_group.cu, prefix_latent.cu).

Requests that continue the same tokens keep the pages of the common part once: their page tables begin with the same pages.
`group_attend` and `latent_attend` give every row of a pass what `ds41_group_attend` and `ds41_latent_attend` give it (its
attention over all cached positions up to its own, or over its chunk of them), but read the common pages once for all rows that
share them; each row reads only what follows by itself, and the parts are joined by their maxima and sums.

Which rows share what is a `PrefixPlan`, made on the host from the page tables.  It holds as long as the rows belong to the same
slots and those keep their leading pages: pages added at a table's end leave it valid, so a decode loop makes it once for a batch.
It also holds the workspace of the calls, so calls with one plan, and `set()`, follow one another on one stream; concurrent streams,
or graphs that replay at the same time, need a plan each.  A captured call reads the plan from device memory: after `set()` a replay
uses the new one, which may not have more rows than the call that was captured.  A row that belongs to another slot than its plan says
gets NaN, and check_status() raises; that a slot's leading pages are the ones it was set for is the caller's to see to.

The pages of what a row sees have to be leased, by numbers that the pool has; those that are not are left out where products are 32-bit
and read as zeros by the tensor-core forms, as in the operators that read row by row.
What no row of a pass sees may hold anything, NaN included.  A NaN that a row does meet, in its query, a key, a value, a gate or a
sink, is in its result; one in a value that only some rows of a range see may be in the others' as well, as the tensor cores multiply
it by their weight of zero.
"""
from __future__ import annotations

import ctypes as C
from typing import List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import lib
from . import stack as S
from .stack import ceil_to

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SMS = 148                # of a B200: plans do not depend on the device found
UNIT = 8                 # numbers of a unit (ds41_prefix_plan)


class PlanArgs(C.Structure):
    _fields_ = [("units", C.c_void_p), ("n_units", C.c_void_p), ("turns", C.c_void_p), ("order", C.c_void_p), ("cell", C.c_void_p), ("owner", C.c_void_p), ("parts", C.c_void_p),
                ("part_o", C.c_void_p), ("part_ml", C.c_void_p), ("max_units", C.c_int), ("rows_per_unit", C.c_int), ("grid", C.c_int)]


class PlanShape(C.Structure):
    """What the host's division of the work goes by (csrc/core/prefix_plan.cc)."""
    _fields_ = [(n, C.c_int) for n in ("rows", "heads", "kv_heads", "vdim", "page_tokens", "chunk", "rows_per_unit", "together", "grid",
                                       "min_tokens", "max_turns", "max_units", "max_cells", "extra", "least_span", "reserved")] + \
               [(n, C.c_double) for n in ("turn", "row", "longer", "shorter", "byte", "part")]


def _failed(err: int):
    raise (MemoryError("no memory to divide the work of a pass") if err == -2 else RuntimeError("a plan's arrays do not hold its rows' division"))


def common_runs(tables: np.ndarray) -> List[Tuple[List[int], int]]:
    """Groups of rows of a page table that begin with the same leased pages: (rows, common pages), a row in one group at most.  Which
    they are: find_groups() of csrc/core/prefix_plan.cc."""
    t = np.ascontiguousarray(tables, dtype=np.int32)
    n, width = t.shape
    order, bounds, pages = (np.zeros(max(n, 1) * k, dtype=np.int32) for k in (1, 2, 1))
    count = lib.core().ds41_prefix_groups(C.c_void_p(t.ctypes.data), n, width, *(C.c_void_p(x.ctypes.data) for x in (order, bounds, pages)))
    if count < 0:
        _failed(count)
    return [(order[bounds[2 * i]:bounds[2 * i + 1]].tolist(), int(pages[i])) for i in range(count)]


def tiled(kind: str, heads: int, kv_heads: int, dim: int, vdim: int, page_tokens: int) -> bool:
    """Do bf16 calls of these sizes take the tensor-core forms?  The one for everything else, whose products are 32-bit, is for sizes that
    are small or rare: reading common pages once does not make up for it.  `dim`: of a key (latent: with its rotated part)."""
    if page_tokens < 8 or max(page_tokens, 64) % min(page_tokens, 64):
        return False
    if kind == "grouped":
        return heads // kv_heads <= 128 and vdim <= 128 and dim <= 256
    return heads <= 128 and vdim <= 512 and dim - vdim <= 64


class Cost(NamedTuple):
    """What a plan goes by, in us (measured on units of 64 to 16000 keys): of a block's turn, of a row of its units, of a key of the
    longer of the units that it has at a time and of one of the shorter, of a byte of partial results on their way to the join and of a
    part of the row that has most of them."""
    turn: float
    row: float
    longer: float
    shorter: float
    byte: float
    part: float = 0.2


COSTS = {"grouped": Cost(1.4, 0.10, 0.0105, 0.0055, 1 / 6e6), "latent": Cost(4.0, 0.0, 0.0205, 0.0, 1 / 8e6)}
COST_F32 = Cost(1.0, 0.0, 0.3, 0.3, 1 / 6e6)


class PrefixPlan:
    """Rows that share leading pages, how their attention is divided, and the workspace of the calls.

    `kind`: "grouped" or "latent"; `rows`: most rows of a pass; `heads`, `kv_heads`, `vdim`: of the attention (latent: one key / value
    head, `vdim` the padded latent width).  Prefixes shorter than `min_tokens` are left to the rows.  `chunk`: the calls' chunk, if the
    plan is to leave out what lies before the rows' chunks (see set())."""

    def __init__(self, kind: str, *, rows: int, heads: int, vdim: int, page_tokens: int, device, kv_heads: int = 1, dtype=BF16,
                 min_tokens: int = 64, chunk: int = 0):
        if kind not in ("grouped", "latent"):
            raise ValueError(f"a prefix plan is grouped or latent, not {kind!r}")
        if min(rows, heads, kv_heads, vdim, page_tokens) <= 0 or heads % kv_heads or vdim % 16:
            raise ValueError("sizes must be positive, kv_heads must divide heads, the value width must be a multiple of 16")
        if kind == "latent" and kv_heads != 1:
            raise ValueError("latent attention has one key / value head")
        if chunk < 0 or (chunk and kind == "latent"):
            raise ValueError("chunk must not be negative, and latent attention has none")
        if dtype not in (BF16, F32):
            raise ValueError(f"cache rows are bf16 or fp32, not {dtype}")
        self.kind, self.rows, self.heads, self.kv_heads, self.vdim = kind, rows, heads, kv_heads, vdim
        self.page_tokens, self.dtype, self.device, self.chunk = page_tokens, dtype, torch.device(device), chunk
        self.min_tokens, self.cost = min_tokens, COSTS[kind] if dtype == BF16 else COST_F32
        self._sizes(kind, rows, heads, vdim, kv_heads)
        self.data = torch.zeros(self._size, dtype=I32, device=self.device)
        # parts without a weight are not read
        self.part_o = torch.empty(self.max_cells * heads * vdim, dtype=F32, device=self.device)
        self.part_ml = torch.empty(self.max_cells * heads * 2, dtype=F32, device=self.device)
        self.status = lib.new_status(self.device)
        self.n_units = self.span = 0
        self.n_rows, self.table_shape = 0, None            # of the last set(): what calls have to match
        self.captured: Optional[int] = None                # least rows of the calls that graphs hold
        # prefixes: {rows, tokens, first of them that is seen} of each, then their rows; {places, length of the ranges, prefixes}
        self._groups, self._result = np.zeros(4 * rows, dtype=np.int32), np.zeros(3, dtype=np.int32)
        # one copy of everything costs less than two of what is used, if it is small (64 KB: 3 us of the host, 7 with the slices of two)
        self._whole = self._size <= 1 << 14
        self._used = 0
        shape = PlanShape(rows=rows, heads=heads, kv_heads=kv_heads, vdim=vdim, page_tokens=page_tokens, chunk=chunk,
                          rows_per_unit=self.rows_per_unit, together=self.together, grid=self.grid, min_tokens=min_tokens,
                          max_turns=self.max_turns, max_units=self.max_units, max_cells=self.max_cells, extra=self.extra,
                          least_span=ceil_to(128 if dtype == BF16 else 32, page_tokens), **self.cost._asdict())
        at = (C.c_int32 * 5)(*self._at)
        self._divide = lib.core().ds41_prefix_divide
        self._shape = (shape, at, C.byref(shape), C.c_void_p(self._groups.ctypes.data), C.c_void_p(self._result.ctypes.data))
        a, base = PlanArgs(), self.data.data_ptr()
        a.n_units, (a.units, a.turns, a.order, a.cell, a.parts) = base, (base + 4 * x for x in self._at)
        a.owner = a.cell + 4 * rows
        a.part_o, a.part_ml = self.part_o.data_ptr(), self.part_ml.data_ptr()
        a.max_units, a.rows_per_unit, a.grid = self.max_units, self.rows_per_unit, self.grid
        self.args, self.args_ref = a, C.byref(a)

    def _sizes(self, kind: str, rows: int, heads: int, vdim: int, kv_heads: int):
        self.rows_per_unit = max(1, 128 // (heads // kv_heads))
        self.together = 2 if kind == "grouped" else 1            # units that a block (latent, wide: two blocks) has at a time
        self.grid = SMS // 2 if kind == "latent" and vdim > 256 else SMS               # two CTAs to a unit
        self.extra = 3 * -(-self.grid * self.together // kv_heads)      # items beyond one for every piece of a prefix and every request
        self.max_items = self.extra + 2 * rows
        # a head's items go in twos (one may stay alone), the heads are dealt one like the other
        self.max_turns = -(-(self.max_items + 1) * kv_heads // (self.grid * self.together)) + 2
        self.max_units = self.max_turns * self.grid * self.together
        self.max_cells = self.extra * min(self.rows_per_unit, rows) + 2 * rows
        # [count, 3 unused | units | turns | order | cell, owner | parts]
        self._at = np.cumsum([4, UNIT * self.max_units, self.grid, rows, 2 * rows]).tolist()
        self._size = self._at[-1] + rows

    @classmethod
    def nbytes(cls, kind: str, *, rows: int, heads: int, vdim: int, kv_heads: int = 1, **_) -> int:
        """Device memory that a plan of these sizes takes."""
        p = cls.__new__(cls)
        p._sizes(kind, rows, heads, vdim, kv_heads)
        return 4 * (p._size + p.max_cells * heads * (vdim + 2) + 4)

    @property
    def shared(self) -> List[Tuple[List[int], int]]:
        """Rows and tokens of every prefix."""
        out, n_groups = [], int(self._result[2])
        at = 3 * n_groups
        for i in range(n_groups):
            n, tokens = self._groups[3 * i:3 * i + 2].tolist()
            out.append((self._groups[at:at + n].tolist(), tokens))
            at += n
        return out

    def set(self, slots: Sequence[int], tables, lengths: Optional[Sequence[int]] = None) -> None:
        """`slots`: the slot of every row of the passes to come (-1: none); `tables`: the page table on the host, [slots, pages],
        negative where no page is leased.  `lengths`: how many tokens each row's request has now (default: what its pages hold); the
        division of the work goes by it.  A plan with a `chunk` also leaves out the keys before the chunk of a row's last token, if it
        is given lengths: until the next set() such a row may go on, but not back behind that chunk's beginning.  Not inside a capture;
        the device's copy is made on the current stream, and the host does not wait for it."""
        t = tables.numpy() if isinstance(tables, torch.Tensor) else np.asarray(tables)
        s = np.ascontiguousarray(slots, dtype=np.int64)
        if t.ndim != 2 or t.dtype != np.int32:
            raise ValueError("the page table is a matrix of 32-bit integers")
        n, (n_slots, width) = len(s), t.shape
        if s.ndim != 1 or n > self.rows:
            raise ValueError(f"a plan for {self.rows} rows does not take {s.shape}")
        if n and int(s.max()) >= n_slots:
            raise ValueError(f"slot {int(s.max())} of {n_slots}")
        if lengths is not None and len(lengths) != n:
            raise ValueError("lengths has an entry per row")
        if width * self.page_tokens >= 1 << 31:
            raise ValueError("a request has fewer than 2^31 tokens")
        if self.captured is not None and (n > self.captured or t.shape != self.table_shape):
            raise ValueError(f"a captured call has {self.captured} rows and a page table of {tuple(self.table_shape)}")
        t = np.ascontiguousarray(t)
        have = np.ascontiguousarray(lengths, dtype=np.int64) if lengths is not None else None
        cuda = self.data.is_cuda
        if cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a plan is not set inside a capture")
        # torch keeps a pinned buffer until the copies from it are done
        to = torch.empty(self._size, dtype=I32, pin_memory=True) if cuda else self.data
        _, at, shape, groups, result = self._shape
        err = self._divide(shape, C.c_void_p(t.ctypes.data), n_slots, width, C.c_void_p(s.ctypes.data), n,
                           C.c_void_p(have.ctypes.data if have is not None else 0), self.max_units if self._whole else self._used,
                           C.c_void_p(to.data_ptr()), at, groups, result)
        if err:
            _failed(err)
        self.n_units, self.span, _ = self._result.tolist()
        self.n_rows, self.table_shape = n, t.shape
        if cuda and self._whole:
            self.data.copy_(to, non_blocking=True)
        elif cuda:
            a, b = self._at[0] + UNIT * max(self.n_units, self._used), self._at[1]
            self.data[:a].copy_(to[:a], non_blocking=True)
            self.data[b:].copy_(to[b:], non_blocking=True)
        self._used = self.n_units

    def check_status(self, what: str = "attention over a shared prefix"):
        lib.raise_on_status(self.status, what)


# ---------------------------------------------------------------------------------------------------- launches
def _stream() -> int:
    """The current stream's handle, without the object that torch.cuda.current_stream() makes for it (3 us, a sixth of a call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def launch_group(a: S.GroupAttendArgs, plan: PrefixPlan) -> None:
    """Grouped attention; `a` as for ds41_group_attend."""
    lib.check(lib.kernels("stack").ds41_prefix_group(C.byref(a), plan.args_ref, C.c_void_p(_stream())), "ds41_prefix_group")


def launch_latent(a: S.LatentAttendArgs, plan: PrefixPlan, n_pages: int, sink, out: torch.Tensor, ld_out: int) -> None:
    """Latent attention and the join of its parts; `a` as for ds41_latent_attend."""
    lib.check(lib.kernels("stack").ds41_prefix_latent(C.byref(a), plan.args_ref, n_pages, lib.ptr(sink), lib.ptr(out), ld_out,
                                                      C.c_void_p(_stream())), "ds41_prefix_latent")


# ---------------------------------------------------------------------------------------------------- front end
def _check(plan: PrefixPlan, kind: str, rows: int, q, q_rot, extra, pool, page_table, row_pos, row_slot, out, width: int,
           scale: float) -> None:
    """`extra`: the gate or the sink.  What is asked of every tensor is asked at once, as it is a call's host time; which one it is that
    does not fit is found afterwards."""
    if plan.kind != kind:
        raise ValueError(f"the plan is for {plan.kind} attention")
    if not scale > 0:
        raise ValueError("scale must be positive")
    if not 0 < rows <= plan.rows:
        raise ValueError(f"a pass has 1 to {plan.rows} rows, not {rows}")
    dtype = plan.dtype
    if pool.dtype is not dtype or out.dtype is not dtype or page_table.dtype is not I32 or row_pos.dtype is not I32 \
            or row_slot.dtype is not I32 or (extra is not None and extra.dtype is not F32):
        for name, t, want in (("pool", pool, dtype), ("out", out, dtype), ("page_table", page_table, I32), ("row_pos", row_pos, I32),
                              ("row_slot", row_slot, I32), ("gate" if kind == "grouped" else "sink", extra, F32)):
            if t is not None and t.dtype != want:
                raise ValueError(f"{name} must be 32-bit integers, not {t.dtype}" if want == I32 else f"{name} is {t.dtype}")
    if not (page_table.is_contiguous() and row_pos.is_contiguous() and row_slot.is_contiguous()):
        raise ValueError("page_table, row_pos and row_slot must be contiguous")
    if page_table.dim() != 2 or row_pos.dim() != 1 or row_slot.dim() != 1 or row_pos.numel() < rows or row_slot.numel() < rows:
        raise ValueError("page_table is [slots, pages], row_pos and row_slot have an entry per row")
    shape = pool.shape
    if len(shape) != 2 or not pool.is_contiguous() or shape[1] != width or shape[0] == 0 or shape[0] % plan.page_tokens:
        raise ValueError(f"pool must be contiguous rows of {width} values, whole pages of {plan.page_tokens} of them")
    if shape[0] >= 1 << 31:
        raise ValueError("a pool has fewer than 2^31 rows")
    if out.shape != (rows, plan.heads, plan.vdim):
        raise ValueError(f"out must be [{rows}, {plan.heads}, {plan.vdim}]")
    step, head, one = _steps(out)
    if one != 1 or head != plan.vdim or step % 8 or step < plan.heads * plan.vdim or out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned, a row's heads side by side and rows apart, at multiples of 8 values")
    here = torch.cuda.current_device() if plan.device.type == "cuda" else None
    if not (pool.get_device() == here and out.get_device() == here and page_table.get_device() == here and row_pos.get_device() == here
            and row_slot.get_device() == here and q.get_device() == here and (q_rot is None or q_rot.get_device() == here)
            and (extra is None or extra.get_device() == here) and plan.data.get_device() == here):
        for name, t in (("pool", pool), ("out", out), ("page_table", page_table), ("row_pos", row_pos), ("row_slot", row_slot), ("q", q),
                        ("q_rot", q_rot), ("gate" if kind == "grouped" else "sink", extra), ("the plan", plan.data)):
            if t is not None and t.get_device() != here:
                raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")
    if rows != plan.n_rows or page_table.shape != plan.table_shape:
        raise ValueError(f"the plan was set for {plan.n_rows} rows and a page table of {plan.table_shape and tuple(plan.table_shape)}")
    if torch.cuda.is_current_stream_capturing():
        plan.captured = rows if plan.captured is None else min(rows, plan.captured)


def _steps(t: torch.Tensor) -> Tuple[int, int, int]:
    """Strides of [rows, heads, values]; a dimension of one entry may have any, and gets that of entries side by side."""
    row, head, one = t.stride()
    rows, heads, values = t.shape
    head = values if heads == 1 else head
    return (heads * head if rows == 1 else row), head, one


def _heads(name: str, q: torch.Tensor, heads: int, dtype) -> Tuple[int, int]:
    """Values between a tensor's rows and between a row's heads."""
    shape = q.shape
    if len(shape) != 3 or shape[1] != heads or q.dtype != dtype or shape[2] % 16 or shape[2] == 0:
        raise ValueError(f"{name} must be [rows, {heads}, a multiple of 16] of {dtype}")
    row, head, one = _steps(q)
    if one != 1 or row % 8 or head % 8 or q.data_ptr() % 16 or row < head * (heads - 1) + shape[2]:
        raise ValueError(f"{name}: values of a head side by side, rows and heads at multiples of 8 values, 16-byte aligned")
    return row, head


def group_attend(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, row_pos: torch.Tensor, row_slot: torch.Tensor,
                 plan: PrefixPlan, *, scale: float, chunk: int = 0, gate: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of a pass over a paged cache, common pages read once: [rows, heads, vdim].

    q [rows, heads, dim]; pool [pages * page_tokens, kv_heads * (dim + vdim)]: keys of all key/value heads, then their values; row r
    stands at row_pos[r] of slot row_slot[r] (negative: the row's result is zero) and sees the positions up to its own, within its
    chunk of `chunk` of them where that is not 0.  `gate` [rows, heads] fp32: a head's result times sigmoid(gate)."""
    (ld_q, step), dtype = _heads("q", q, plan.heads, plan.dtype), plan.dtype
    R, H, D = q.shape
    if step != D:
        raise ValueError("q: a row's heads must lie side by side")
    if out is None:
        out = torch.empty(R, H, plan.vdim, dtype=dtype, device=q.device)
    _check(plan, "grouped", R, q, None, gate, pool, page_table, row_pos, row_slot, out, plan.kv_heads * (D + plan.vdim), scale)
    if chunk < 0 or (plan.chunk and chunk != plan.chunk):
        raise ValueError(f"the plan is for a chunk of {plan.chunk}" if plan.chunk else "chunk must not be negative")
    if gate is not None and (gate.shape != (R, H) or (H > 1 and gate.stride(1) != 1)):
        raise ValueError(f"gate must be [{R}, {H}] with a row's values side by side")
    slots, max_pages = page_table.shape
    a = S.GroupAttendArgs(q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), row_pos.data_ptr(), row_slot.data_ptr(), out.data_ptr(),
                          plan.status.data_ptr(), S.ProjArgs(gate.data_ptr(), 0, gate.stride(0), 1, 0, 0) if gate is not None else S.NO_PROJ, S.NO_PROJ, None,
                          ld_q, scale, R, H, plan.kv_heads, D, plan.vdim, chunk, 1, slots, 0, _steps(out)[0], max_pages, plan.page_tokens,
                          int(dtype == F32), pool.shape[0] // plan.page_tokens, 0)
    launch_group(a, plan)
    return out


def latent_attend(q_abs: torch.Tensor, q_rot: Optional[torch.Tensor], pool: torch.Tensor, page_table: torch.Tensor,
                  row_pos: torch.Tensor, row_slot: torch.Tensor, plan: PrefixPlan, *, scale: float,
                  sink: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Latent attention of a pass over a paged cache, common pages read once: [rows, heads, latent width].

    q_abs [rows, heads, latent], q_rot [rows, heads, rot] (None: no rotated part); pool [pages * page_tokens, latent + rot]: a
    position's latent, which is key and value of every head, and its rotated key part.  `sink` [heads] fp32: an extra logit in a
    head's denominator."""
    (ld_abs, step), dtype = _heads("q_abs", q_abs, plan.heads, plan.dtype), plan.dtype
    R, H, V = q_abs.shape
    if V != plan.vdim:
        raise ValueError(f"q_abs: {V} latent values, the plan has {plan.vdim}")
    if step != V:
        raise ValueError("q_abs: a row's heads must lie side by side")
    rot = ld_rot = rot_head = 0
    if q_rot is not None:
        ld_rot, rot_head = _heads("q_rot", q_rot, H, dtype)
        if q_rot.shape[0] != R:
            raise ValueError("q_rot must have as many rows as q_abs")
        rot = q_rot.shape[2]
    if out is None:
        out = torch.empty(R, H, V, dtype=dtype, device=q_abs.device)
    _check(plan, "latent", R, q_abs, q_rot, sink, pool, page_table, row_pos, row_slot, out, V + rot, scale)
    if sink is not None and (sink.shape != (H,) or not sink.is_contiguous()):
        raise ValueError(f"sink must be {H} contiguous values")
    a = S.LatentAttendArgs()
    a.q_abs, a.ld_q_abs, a.q_rot, a.ld_q_rot, a.q_rot_stride = q_abs.data_ptr(), ld_abs, q_rot.data_ptr() if rot else None, ld_rot, rot_head
    a.pool, a.page_table, a.row_pos, a.row_slot = pool.data_ptr(), page_table.data_ptr(), row_pos.data_ptr(), row_slot.data_ptr()
    a.scale, a.rows, a.heads, a.kv_pad, a.row_len = scale, R, H, V, V + rot
    a.max_pages, a.page_tokens, a.f32, a.status = page_table.shape[1], plan.page_tokens, int(dtype == F32), plan.status.data_ptr()
    launch_latent(a, plan, pool.shape[0] // plan.page_tokens, sink, out, _steps(out)[0])
    return out
