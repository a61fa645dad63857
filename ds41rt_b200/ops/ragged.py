"""Passes of several requests with any number of new tokens each, over a paged cache (csrc/kernels/ragged.cu, ragged_attend.cu).

A server that batches continuously runs portions of prompts and decode rows in one pass.  Request i brings `new[i]` tokens, the last of
`lengths[i]`, and keeps its keys and values in the pages of slot `slots[i]`; its rows follow those of request i - 1.

`RaggedPass.describe` makes positions, slots and cache rows of all new tokens from the lengths, on the device and without the host, and
divides the attention's work; `heads_to_cache` norms every query and key head by itself, rotates them and stores keys and values;
`attend` is the attention of the new tokens over everything before them, or over a window of positions and a few first tokens that stay
visible.  One description serves all layers of a pass whose attention has the pass's sizes and window.

A pass holds the workspace of its calls: they follow one another on one stream; concurrent streams, or graphs that replay at the same
time, need a pass each.  Everything can be captured, `describe` included: a replay follows what the tensors of slots, tokens, lengths and
pages then hold.

Rows behind the last request's are left as they were, in every output but the description, where they have position 0, slot -1 and place
-1.  Requests without a slot (negative) have rows, too: their attention is zero, they have no place in the cache.  The pages of what a row
sees have to be leased, by numbers that the pool has; others read as zeros, and nothing is stored in them.  A new token whose own page is
not leased has no place, either: `heads_to_cache` leaves its query out, its attention is zero, and check_status() tells of it.  What no
row of a request's block of tokens sees may hold anything, NaN included.  A NaN that a row does meet is in its result; one in a value that
only some rows of a block see may be in the others' as well, as the tensor cores multiply it by their weight of zero.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import lib
from . import stack as S
from .prefix import _steps

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SMS = 148                       # of a B200: passes do not depend on the device found
_raw_stream = torch._C._cuda_getCurrentRawStream      # without the object that torch.cuda.current_stream() makes for it (3 us)
UNIT = 12                       # numbers of a unit (ds41_ragged_pass)
MOST_ROWS, MOST_REQUESTS, MOST_BLOCKS, MOST_UNITS = 1 << 18, 4096, 8192, 1 << 22
MOST_HEAD_VALUES = 50688        # of a row's queries and keys


class PassArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("header", "row_pos", "row_slot", "row_place", "units", "counters", "part_o", "part_ml", "status",
                                       "report")] + \
               [(n, C.c_int) for n in ("rows", "requests", "heads", "kv_heads", "dim", "vdim", "page_tokens", "window", "first", "f32", "tiled",
                                       "unit_tokens", "key_tile", "turn_rows", "max_blocks", "max_units", "max_cells", "grid", "v_parts")]


class HeadsArgs(C.Structure):
    _fields_ = [(n, S.ProjArgs) for n in ("q", "k", "v")] + \
               [(n, C.c_void_p) for n in ("q_norm", "k_norm", "freq", "row_pos", "row_place", "q_out", "pool")] + \
               [("ld_q", C.c_longlong), ("eps", C.c_float)] + \
               [(n, C.c_int) for n in ("q_norm_stride", "k_norm_stride", "width", "rows", "heads", "kv_heads", "dim", "vdim", "rot_dim",
                                       "pool_rows", "f32")]


class AttendArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "pool", "page_table", "out")] + [("gate", S.ProjArgs), ("sink", C.c_void_p)] + \
               [(n, C.c_longlong) for n in ("q_row", "q_head", "out_row")] + \
               [("scale", C.c_float), ("q_rows", C.c_int), ("max_pages", C.c_int), ("n_pages", C.c_int)]


def packed(arguments) -> struct.Struct:
    """A C structure's layout, by which its bytes are made in a fifth of the time that its object takes (1 us instead of 5)."""
    letters = {C.c_void_p: "P", C.c_longlong: "q", C.c_int: "i", C.c_float: "f"}
    form = lambda a: "".join(letters[t] if t in letters else form(t) for _, t in a._fields_)
    return struct.Struct("@" + form(arguments))


_HEADS_BYTES, _ATTEND_BYTES = packed(HeadsArgs), packed(AttendArgs)
_NO_GATE = (0, 0, 0, 0, 0, 0)


def tiled(heads: int, kv_heads: int, dim: int, vdim: int, page_tokens: int) -> bool:
    """Do bf16 calls of these sizes take the tensor-core form (pages of 16, 32, 64, 128 or whole 128s)?  The one for everything else
    multiplies in 32 bits, and takes many times as long in large calls."""
    pages = page_tokens >= 16 and not (128 % page_tokens if page_tokens < 128 else page_tokens % 128)
    return pages and heads // kv_heads <= 128 and dim <= 256 and (vdim <= 128 or (vdim <= 256 and vdim % 32 == 0))


class RaggedPass:
    """Description and workspace of passes of up to `rows` new tokens of up to `requests` requests.

    `heads`, `kv_heads`, `dim`, `vdim`: of the attention.  `window`, `first`: a row at position p sees the positions j <= p with
    j > p - window (0: all of them) or j < first."""

    def __init__(self, *, rows: int, requests: int, heads: int, kv_heads: int, dim: int, vdim: int, page_tokens: int, device, window: int = 0,
                 first: int = 0, dtype=BF16):
        if min(rows, requests, heads, kv_heads, dim, vdim, page_tokens) <= 0 or heads % kv_heads:
            raise ValueError("sizes must be positive, and kv_heads must divide heads")
        if dim % 16 or vdim % 16 or max(dim, vdim) > 256:
            raise ValueError("heads have a multiple of 16 values, at most 256")
        if rows > MOST_ROWS or requests > MOST_REQUESTS or heads // kv_heads > 1024:
            raise ValueError(f"at most {MOST_ROWS} rows, {MOST_REQUESTS} requests and 1024 query heads to a key/value head")
        if window < 0 or first < 0 or max(window, first) >= 1 << 31 or page_tokens >= 1 << 24:
            raise ValueError("window and first are numbers of tokens, a page has fewer than 2^24")
        if dtype not in (BF16, F32):
            raise ValueError(f"cache rows are bf16 or fp32, not {dtype}")
        self.rows, self.requests, self.heads, self.kv_heads, self.dim, self.vdim = rows, requests, heads, kv_heads, dim, vdim
        self.page_tokens, self.window, self.first, self.dtype, self.device = page_tokens, window, first, dtype, torch.device(device)
        self.columns = kv_heads * (dim + vdim)
        self._sizes()
        i32 = lambda n: torch.zeros(n, dtype=I32, device=self.device)
        self.header, self.units, self.counters = i32(16), i32(UNIT * self.max_units), i32(2 * self.max_blocks * kv_heads * self.v_parts)
        self.described = i32(3 * rows)
        self.row_pos, self.row_slot, self.row_place = self.described.view(3, rows)
        self._own = self.described.data_ptr(), self.described.data_ptr() + 12 * rows
        self.part_o = torch.empty(self.max_cells * (vdim // self.v_parts), dtype=F32, device=self.device)     # what is read was written before
        self.part_ml = torch.empty(self.max_cells * 2, dtype=F32, device=self.device)
        self.status, self.report = lib.new_status(self.device), self.header[4:8]
        self.table_shape: Optional[Tuple[int, ...]] = None           # of the last describe(): what attend has to match
        self.n_pages = 0
        a = PassArgs(*(t.data_ptr() for t in (self.header, self.row_pos, self.row_slot, self.row_place, self.units, self.counters,
                                              self.part_o, self.part_ml, self.status, self.report)),
                     rows, requests, heads, kv_heads, dim, vdim, page_tokens, window, first, int(dtype == F32), int(self.tiled),
                     self.unit_tokens, self.key_tile, self.turn_rows, self.max_blocks, self.max_units, self.max_cells, SMS, self.v_parts)
        self.args, self.args_ref = a, C.byref(a)

    def _sizes(self):
        group = self.heads // self.kv_heads
        self.tiled = self.dtype == BF16 and tiled(self.heads, self.kv_heads, self.dim, self.vdim, self.page_tokens)
        self.unit_tokens = 2 * (128 // group) if self.tiled else max(1, 64 // group)
        self.key_tile = 128 if self.tiled else 32
        self.v_parts = 2 if self.tiled and self.vdim > 128 else 1
        columns = self.vdim // self.v_parts
        # of the tensor-core form: blocks of so few rows have them in both of a CTA's tiles, which take the keys in turn
        self.turn_rows = min(64, -(-self.dim // 64) * 16384 // (4 * columns)) if self.tiled else 0
        self.max_blocks = self.rows // self.unit_tokens + min(self.requests, self.rows)
        if self.max_blocks > MOST_BLOCKS:
            raise ValueError(f"{self.rows} rows of {group} heads to a key/value head are more than a pass divides")
        self.max_units = self.max_blocks * self.kv_heads * self.v_parts + 8 * SMS
        if self.max_units >= MOST_UNITS:
            raise ValueError(f"{self.rows} rows of {self.requests} requests with {self.kv_heads} key/value heads are more than a pass divides")
        self.max_cells = min(2 * SMS * self.unit_tokens * group, 64 * self.rows * self.heads * self.v_parts)

    def tell(self, status: torch.Tensor, report: torch.Tensor):
        """Where kernels report from now on: four numbers each, on the device."""
        self.status, self.report = status, report
        self.args.status, self.args.report = status.data_ptr(), report.data_ptr()

    def nbytes(self) -> int:
        """Device memory that the pass takes."""
        return sum(t.numel() * t.element_size() for t in (self.header, self.units, self.counters, self.row_pos, self.row_slot, self.row_place,
                                                          self.part_o, self.part_ml, self.status))

    def describe(self, slots: torch.Tensor, new: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor, n_pages: int):
        """`slots`, `new`, `lengths`: 32-bit integers, one per request, on the device: page table row (negative: none), new tokens, tokens
        with them.  `page_table` [slots, pages]; the pool has `n_pages`.  Returns (row_pos, row_slot, row_place) [rows] each: the pass's
        own tensors, which the next call overwrites.  A request whose lengths cannot be, or whose slot there is not, counts as one without
        a slot, and rows beyond the pass's are left out; the next check_status() raises, whatever was described in between."""
        n = slots.numel()
        for name, t in (("slots", slots), ("new", new), ("lengths", lengths)):
            if t.dtype is not I32 or t.shape != (n,) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous 32-bit integers, one per request")
        if n > self.requests:
            raise ValueError(f"a pass for {self.requests} requests does not take {n}")
        here = torch.cuda.current_device()
        if not (slots.get_device() == here and new.get_device() == here and lengths.get_device() == here):
            _elsewhere(here, (("slots", slots), ("new", new), ("lengths", lengths)))
        slots_at, new_at, lengths_at = slots.data_ptr(), new.data_ptr(), lengths.data_ptr()
        self._apart(n, slots_at, new_at, lengths_at)
        n_slots, width = self._table(page_table, n_pages, here)
        err = lib.kernels("stack").ds41_ragged_describe(self.args_ref, C.c_void_p(slots_at), C.c_void_p(new_at),
                                                        C.c_void_p(lengths_at), n, C.c_void_p(page_table.data_ptr()), n_slots,
                                                        width, n_pages, C.c_void_p(_raw_stream(here)))
        if err:
            lib.check(err, "ds41_ragged_describe")
        self.table_shape, self.n_pages = (n_slots, width), n_pages
        return self.row_pos, self.row_slot, self.row_place

    def describe_rows(self, row_pos: torch.Tensor, row_slot: torch.Tensor, page_table: torch.Tensor, n_pages: int):
        """The same from the positions and slots of rows, 32-bit integers on the device, as other operators take them: adjacent rows of
        one slot at consecutive positions are a request's, and adjacent rows without a slot one that nothing is done for.  More
        requests than the pass takes are left out, and the next check_status() raises."""
        n = row_pos.numel()
        if n > self.rows or row_pos.dtype is not I32 or row_slot.dtype is not I32 or row_pos.shape != (n,) or row_slot.shape != (n,) \
                or not (row_pos.is_contiguous() and row_slot.is_contiguous()):
            raise ValueError(f"row_pos and row_slot must be contiguous 32-bit integers, one per row, of at most {self.rows} rows")
        here = torch.cuda.current_device()
        if not (row_pos.get_device() == here and row_slot.get_device() == here):
            _elsewhere(here, (("row_pos", row_pos), ("row_slot", row_slot)))
        self._apart(n, row_pos.data_ptr(), row_slot.data_ptr())
        n_slots, width = self._table(page_table, n_pages, here)
        err = lib.kernels("stack").ds41_ragged_describe_rows(self.args_ref, C.c_void_p(row_pos.data_ptr()), C.c_void_p(row_slot.data_ptr()), n,
                                                             C.c_void_p(page_table.data_ptr()), n_slots, width, n_pages,
                                                             C.c_void_p(_raw_stream(here)))
        if err:
            lib.check(err, "ds41_ragged_describe_rows")
        self.table_shape, self.n_pages = (n_slots, width), n_pages
        return self.row_pos, self.row_slot, self.row_place

    def _apart(self, n: int, *places: int):
        """`places`: of n numbers each, which some blocks read while others write the description."""
        low, high = self._own
        for at in places:
            if at < high and at + 4 * n > low:
                raise ValueError("a description is not made from its own row_pos, row_slot and row_place: copies of them")

    def _table(self, page_table: torch.Tensor, n_pages: int, here: int) -> Tuple[int, int]:
        n_slots, width = page_table.shape if page_table.dim() == 2 else (0, 0)
        if page_table.dtype is not I32 or n_slots == 0 or width == 0 or not page_table.is_contiguous():
            raise ValueError("page_table is a contiguous matrix of 32-bit integers, [slots, pages]")
        if n_pages <= 0 or n_pages * self.page_tokens >= 1 << 31 or width * self.page_tokens > 1 << 30:
            raise ValueError("a pool has fewer than 2^31 rows, a request at most 2^30")
        if not (page_table.get_device() == here and self.header.get_device() == here):
            _elsewhere(here, (("page_table", page_table), ("the pass", self.header)))
        return n_slots, width

    def check_status(self, what: str = "ragged pass"):
        """Raises if a wait gave up, or if a description since the last check had requests that cannot be, or new tokens on pages that
        are not leased."""
        lib.raise_on_status(self.status, what)
        found = told(self.report.tolist())
        if found:
            self.report.zero_()
            raise lib.KernelError(f"{what}: {found}")


def told(report) -> str:
    """What descriptions have reported (ds41_ragged_pass), in words; nothing: ""."""
    bad, first, lost, lowest = report
    parts = [f"{bad} requests of the description cannot be, the first of them number {first}"] if bad else []
    if lost:
        parts += [f"{lost} new tokens are on pages that are not leased, the lowest row of them {2 ** 31 - 1 - lowest}"]
    return "; ".join(parts)


def _elsewhere(here: int, tensors):
    for name, t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")


def _projection(name: str, x: torch.Tensor, rows: int, heads: int, dim: int) -> Tuple[int, int, int, int, int, int]:
    shape, dtype = x.shape, x.dtype
    if shape != (rows, heads, dim) or (dtype is not BF16 and dtype is not F32):
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}] of bf16 or fp32")
    row, head, one = x.stride()
    if one != 1 or head != dim or row < heads * dim or row >= 1 << 31:
        row, head, one = _steps(x)
        if one != 1 or head != dim or row < heads * dim or row >= 1 << 31:
            raise ValueError(f"{name}: a row's heads must lie side by side")
    return x.data_ptr(), 0, row, 1, dtype is BF16, 0


def _weight(name: str, w: torch.Tensor, heads: int, dim: int) -> Tuple[int, int]:
    shape = w.shape
    if w.dtype is not F32 or not w.is_contiguous() or (shape != (dim,) and shape != (heads, dim)):
        raise ValueError(f"{name} must be contiguous fp32, [{dim}] or [{heads}, {dim}]")
    return w.data_ptr(), dim if len(shape) == 2 else 0


def heads_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, row_pos: torch.Tensor, row_place: torch.Tensor, pool: torch.Tensor, *,
                   q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   freq: Optional[torch.Tensor] = None, width: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Queries [rows, heads, dim] as attention reads them; keys and values go into `pool`.

    q, k [rows, kv_heads, dim], v [rows, kv_heads, vdim]: bf16 or fp32, a row's heads side by side.  Every head of q and k becomes
    x / sqrt(mean(x^2) + eps) * weight where a weight (fp32, [dim], or [heads, dim]) is given, the mean over `width` values
    (0: all; the others are padding, zeros); its values j and j + len(freq), j < len(freq), are then turned by row_pos * freq[j].
    pool [pages * page_tokens, kv_heads * (dim + vdim)], bf16 or fp32: row row_place[r] becomes the keys of all heads, then the values.
    Rows with a negative place are left out.  Two rows with one place leave a mixture of theirs."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v are [rows, heads, values]")
    (R, H, D), G, V = q.shape, k.shape[1], v.shape[2]
    if min(H, G, D, V) == 0 or D > 1024 or max(H, G) > 4096 or (H + G) * D > MOST_HEAD_VALUES:
        raise ValueError(f"heads of 1 to 1024 values, of all queries and keys at most {MOST_HEAD_VALUES}")
    dtype, (pool_rows, columns) = pool.dtype, pool.shape if pool.dim() == 2 else (0, 0)
    if (dtype is not BF16 and dtype is not F32) or columns != G * (D + V) or not pool.is_contiguous() or not 0 < pool_rows < 1 << 31 \
            or columns >= 1 << 31:
        raise ValueError(f"pool must be contiguous rows of {G * (D + V)} values, bf16 or fp32, fewer than 2^31 rows and values of a row")
    a_q, a_k, a_v = _projection("q", q, R, H, D), _projection("k", k, R, G, D), _projection("v", v, R, G, V)
    q_weight, q_stride = (0, 0) if q_norm is None else _weight("q_norm", q_norm, H, D)
    k_weight, k_stride = (0, 0) if k_norm is None else _weight("k_norm", k_norm, G, D)
    half = 0
    if freq is not None:
        half = freq.numel()
        if freq.dtype is not F32 or freq.dim() != 1 or not freq.is_contiguous() or 2 * half > D:
            raise ValueError(f"freq must be at most {D // 2} contiguous fp32 values")
    if not 0 <= width <= D or not eps >= 0:
        raise ValueError(f"width is 0 to {D}, eps is not negative")
    for name, t in (("row_pos", row_pos), ("row_place", row_place)):
        if t.dtype is not I32 or t.dim() != 1 or t.numel() < R or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous 32-bit integers, one per row")
    if out is None:
        out = torch.empty(R, H, D, dtype=dtype, device=q.device)
    if out.shape != (R, H, D) or out.dtype is not dtype:
        raise ValueError(f"out must be [{R}, {H}, {D}] of the pool's type")
    row, head, one = out.stride()
    if one != 1 or head != D or row < H * D:
        row, head, one = _steps(out)
    if one != 1 or head != D or row < H * D:
        raise ValueError("out: a row's heads must lie side by side, rows apart")
    here = torch.cuda.current_device()
    if not (q.get_device() == here and k.get_device() == here and v.get_device() == here and row_pos.get_device() == here
            and row_place.get_device() == here and pool.get_device() == here and out.get_device() == here
            and (q_norm is None or q_norm.get_device() == here) and (k_norm is None or k_norm.get_device() == here)
            and (freq is None or freq.get_device() == here)):
        _elsewhere(here, (("q", q), ("k", k), ("v", v), ("row_pos", row_pos), ("row_place", row_place), ("pool", pool), ("out", out),
                          ("q_norm", q_norm), ("k_norm", k_norm), ("freq", freq)))
    if R == 0:
        return out
    a = _HEADS_BYTES.pack(*a_q, *a_k, *a_v, q_weight, k_weight, freq.data_ptr() if half else 0, row_pos.data_ptr(), row_place.data_ptr(),
                          out.data_ptr(), pool.data_ptr(), row, eps, q_stride, k_stride, width or D, R, H, G, D, V, 2 * half, pool_rows,
                          dtype is F32)
    err = lib.kernels("stack").ds41_ragged_heads(a, C.c_void_p(_raw_stream(here)))
    if err:
        lib.check(err, "ds41_ragged_heads")
    return out


def attend(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, described: RaggedPass, *, scale: float,
           sink: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of a described pass over a paged cache: [rows, heads, vdim].

    q [rows, heads, dim]; pool [pages * page_tokens, kv_heads * (dim + vdim)]: keys of all key/value heads, then their values, the new
    tokens' among them.  `sink` [heads] fp32: an extra logit in a head's denominator; `gate` [rows, heads] fp32: a head's result times
    sigmoid(gate).  Rows behind the last request's are left as `out` has them.  `out` may be `q` itself, but for bf16 values of more than
    128 columns in the tensor-core form.  Rows whose number in the pass's row_place is negative become zeros."""
    p = described
    R, H, D, V, dtype = p.rows, p.heads, p.dim, p.vdim, p.dtype
    if q.shape != (R, H, D) or q.dtype is not dtype:
        raise ValueError(f"q must be [{R}, {H}, {D}] of {dtype}")
    q_row, q_head, one = _steps(q)
    few = 7 if dtype is BF16 else 3               # rows and heads at multiples of 16 bytes
    if one != 1 or q_row & few or q_head & few or q.data_ptr() % 16 or q_row < q_head * (H - 1) + D:
        raise ValueError("q: values of a head side by side, rows and heads at multiples of 16 bytes")
    table_shape = page_table.shape
    if p.table_shape is None:
        raise ValueError("the pass has not been described")
    pool_rows, columns = pool.shape if pool.dim() == 2 else (0, 0)
    if pool.dtype is not dtype or columns != p.columns or not pool.is_contiguous() or pool.data_ptr() % 16:
        raise ValueError(f"pool must be contiguous rows of {p.columns} values of {dtype}, 16-byte aligned")
    if pool_rows != p.n_pages * p.page_tokens or tuple(table_shape) != p.table_shape:
        raise ValueError(f"the pass was described for {p.n_pages} pages and a page table of {p.table_shape}")
    if page_table.dtype is not I32 or not page_table.is_contiguous():
        raise ValueError("page_table is a contiguous matrix of 32-bit integers, [slots, pages]")
    if not scale > 0:
        raise ValueError("scale must be positive")
    if out is None:
        out = torch.empty(R, H, V, dtype=dtype, device=q.device)
    if out.shape != (R, H, V) or out.dtype is not dtype:
        raise ValueError(f"out must be [{R}, {H}, {V}] of {dtype}")
    step, head, one = _steps(out)
    out_at = out.data_ptr()
    if one != 1 or head != V or step & few or step < H * V or out_at % 16:
        raise ValueError("out: a row's heads side by side, rows apart and at multiples of 16 bytes")
    if p.v_parts > 1 and out_at == q.data_ptr():
        raise ValueError("out cannot be q where values have more than 128 columns: two units read a query, at different times")
    sink_at, gates = 0, _NO_GATE
    if sink is not None:
        if sink.dtype is not F32 or sink.shape != (H,) or not sink.is_contiguous():
            raise ValueError(f"sink must be {H} contiguous fp32 values")
        sink_at = sink.data_ptr()
    if gate is not None:
        gate_row, one = gate.stride() if gate.dim() == 2 else (0, 0)
        if gate.dtype is not F32 or gate.shape != (R, H) or (H > 1 and one != 1) or (R > 1 and not H <= gate_row < 1 << 31):
            raise ValueError(f"gate must be fp32 [{R}, {H}] with a row's values side by side")
        gates = gate.data_ptr(), 0, gate_row if R > 1 else H, 1, 0, 0
    here = torch.cuda.current_device()
    if not (q.get_device() == here and pool.get_device() == here and page_table.get_device() == here and out.get_device() == here
            and p.header.get_device() == here and (sink is None or sink.get_device() == here) and (gate is None or gate.get_device() == here)):
        _elsewhere(here, (("q", q), ("pool", pool), ("page_table", page_table), ("out", out), ("the pass", p.header), ("sink", sink),
                          ("gate", gate)))
    a = _ATTEND_BYTES.pack(q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), out_at, *gates, sink_at, q_row, q_head, step, scale, R,
                           table_shape[1], p.n_pages)
    err = lib.kernels("stack").ds41_ragged_attend(a, p.args_ref, C.c_void_p(_raw_stream(here)))
    if err:
        lib.check(err, "ds41_ragged_attend")
    return out
