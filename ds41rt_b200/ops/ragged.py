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
sees have to be leased, by numbers that the pool has; others read as zeros, and nothing is stored in them.  What no row of a request's
block of tokens sees may hold anything, NaN included.  A NaN that a row does meet is in its result; one in a value that only some rows of
a block see may be in the others' as well, as the tensor cores multiply it by their weight of zero.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import lib
from . import stack as S
from .prefix import _heads, _steps, _stream

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SMS = 148                       # of a B200: passes do not depend on the device found
UNIT = 12                       # numbers of a unit (ds41_ragged_pass)
MOST_ROWS, MOST_REQUESTS, MOST_BLOCKS = 1 << 18, 4096, 12288


class PassArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("header", "row_pos", "row_slot", "row_place", "units", "counters", "part_o", "part_ml", "status")] + \
               [(n, C.c_int) for n in ("rows", "requests", "heads", "kv_heads", "dim", "vdim", "page_tokens", "window", "first", "f32", "tiled",
                                       "unit_tokens", "key_tile", "max_blocks", "max_units", "max_cells", "grid")]


class HeadsArgs(C.Structure):
    _fields_ = [(n, S.ProjArgs) for n in ("q", "k", "v")] + \
               [(n, C.c_void_p) for n in ("q_norm", "k_norm", "freq", "row_pos", "row_place", "q_out", "pool")] + \
               [("ld_q", C.c_longlong), ("eps", C.c_float)] + \
               [(n, C.c_int) for n in ("q_norm_stride", "k_norm_stride", "width", "rows", "heads", "kv_heads", "dim", "vdim", "rot_dim",
                                       "pool_rows", "f32")]


class AttendArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "pool", "page_table", "out", "gate", "sink")] + \
               [(n, C.c_longlong) for n in ("q_row", "q_head", "out_row", "gate_row")] + \
               [("scale", C.c_float), ("q_rows", C.c_int), ("max_pages", C.c_int), ("n_pages", C.c_int)]


def tiled(heads: int, kv_heads: int, dim: int, vdim: int, page_tokens: int) -> bool:
    """Do bf16 calls of these sizes take the tensor-core form?  The one for everything else multiplies in 32 bits."""
    pages = page_tokens >= 16 and not (128 % page_tokens if page_tokens < 128 else page_tokens % 128)
    return pages and heads // kv_heads <= 128 and dim <= 256 and vdim <= 128


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
        self._sizes()
        i32 = lambda n: torch.zeros(n, dtype=I32, device=self.device)
        self.header, self.units, self.counters = i32(16), i32(UNIT * self.max_units), i32(2 * self.max_blocks * kv_heads)
        self.row_pos, self.row_slot, self.row_place = i32(rows), i32(rows), i32(rows)
        self.part_o = torch.empty(self.max_cells * vdim, dtype=F32, device=self.device)     # what is read was written before
        self.part_ml = torch.empty(self.max_cells * 2, dtype=F32, device=self.device)
        self.status = lib.new_status(self.device)
        self.table_shape: Optional[Tuple[int, ...]] = None           # of the last describe(): what attend has to match
        self.n_pages = 0
        a = PassArgs(*(t.data_ptr() for t in (self.header, self.row_pos, self.row_slot, self.row_place, self.units, self.counters,
                                              self.part_o, self.part_ml, self.status)),
                     rows, requests, heads, kv_heads, dim, vdim, page_tokens, window, first, int(dtype == F32), int(self.tiled),
                     self.unit_tokens, self.key_tile, self.max_blocks, self.max_units, self.max_cells, SMS)
        self.args, self.args_ref = a, C.byref(a)

    def _sizes(self):
        group = self.heads // self.kv_heads
        self.tiled = self.dtype == BF16 and tiled(self.heads, self.kv_heads, self.dim, self.vdim, self.page_tokens)
        self.unit_tokens = 2 * (128 // group) if self.tiled else max(1, 64 // group)
        self.key_tile = 128 if self.tiled else 32
        self.max_blocks = self.rows // self.unit_tokens + min(self.requests, self.rows)
        if self.max_blocks > MOST_BLOCKS:
            raise ValueError(f"{self.rows} rows of {group} heads to a key/value head are more than a pass divides")
        self.max_units = self.max_blocks * self.kv_heads + 8 * SMS
        self.max_cells = min(2 * SMS * self.unit_tokens * group, 64 * self.rows * self.heads)

    def nbytes(self) -> int:
        """Device memory that the pass takes."""
        return sum(t.numel() * t.element_size() for t in (self.header, self.units, self.counters, self.row_pos, self.row_slot, self.row_place,
                                                          self.part_o, self.part_ml, self.status))

    def describe(self, slots: torch.Tensor, new: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor, n_pages: int):
        """`slots`, `new`, `lengths`: 32-bit integers, one per request, on the device: page table row (negative: none), new tokens, tokens
        with them.  `page_table` [slots, pages]; the pool has `n_pages`.  Returns (row_pos, row_slot, row_place) [rows] each: the pass's
        own tensors, which the next call overwrites.  A request whose lengths cannot be, or whose slot there is not, counts as one without
        a slot, and rows beyond the pass's are left out; check_status() then raises."""
        n = slots.numel()
        for name, t in (("slots", slots), ("new", new), ("lengths", lengths)):
            if t.dtype is not I32 or t.dim() != 1 or not t.is_contiguous() or t.numel() != n:
                raise ValueError(f"{name} must be contiguous 32-bit integers, one per request")
        if n > self.requests:
            raise ValueError(f"a pass for {self.requests} requests does not take {n}")
        _table(page_table, n_pages, self.page_tokens)
        _here((("slots", slots), ("new", new), ("lengths", lengths), ("page_table", page_table), ("the pass", self.header)))
        lib.check(lib.kernels("stack").ds41_ragged_describe(self.args_ref, C.c_void_p(slots.data_ptr()), C.c_void_p(new.data_ptr()),
                                                            C.c_void_p(lengths.data_ptr()), n, C.c_void_p(page_table.data_ptr()),
                                                            page_table.shape[0], page_table.shape[1], n_pages, C.c_void_p(_stream())),
                  "ds41_ragged_describe")
        self.table_shape, self.n_pages = page_table.shape, n_pages
        return self.row_pos, self.row_slot, self.row_place

    def check_status(self, what: str = "ragged pass"):
        lib.raise_on_status(self.status, what)


def _table(page_table: torch.Tensor, n_pages: int, page_tokens: int):
    if page_table.dtype is not I32 or page_table.dim() != 2 or not page_table.is_contiguous() or page_table.numel() == 0:
        raise ValueError("page_table is a contiguous matrix of 32-bit integers, [slots, pages]")
    if n_pages <= 0 or n_pages * page_tokens >= 1 << 31 or page_table.shape[1] * page_tokens >= 1 << 31:
        raise ValueError("a pool and a request have fewer than 2^31 rows")


def _here(tensors):
    here = torch.cuda.current_device()
    for name, t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")


def _projection(name: str, x: torch.Tensor, rows: int, heads: int, dim: int) -> S.ProjArgs:
    if x.dim() != 3 or tuple(x.shape) != (rows, heads, dim) or x.dtype not in (BF16, F32):
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}] of bf16 or fp32")
    row, head, one = _steps(x)
    if one != 1 or head != dim or row < heads * dim or row >= 1 << 31:
        raise ValueError(f"{name}: a row's heads must lie side by side")
    return S.ProjArgs(x.data_ptr(), 0, row, 1, int(x.dtype == BF16), 0)


def _weight(name: str, w: Optional[torch.Tensor], heads: int, dim: int) -> int:
    if w is None:
        return 0
    if w.dtype is not F32 or not w.is_contiguous() or tuple(w.shape) not in ((dim,), (heads, dim)):
        raise ValueError(f"{name} must be contiguous fp32, [{dim}] or [{heads}, {dim}]")
    return dim if w.dim() == 2 else 0


def heads_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, row_pos: torch.Tensor, row_place: torch.Tensor, pool: torch.Tensor, *,
                   q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   freq: Optional[torch.Tensor] = None, width: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Queries [rows, heads, dim] as attention reads them; keys and values go into `pool`.

    q, k [rows, kv_heads, dim], v [rows, kv_heads, vdim]: bf16 or fp32, a row's heads side by side.  Every head of q and k becomes
    x / sqrt(mean(x^2) + eps) * weight where a weight (fp32, [dim], or [heads, dim]) is given, the mean over the first `width` values
    (0: all; the others are padding, zeros); its values j and j + len(freq), j < len(freq), are then turned by row_pos * freq[j].
    pool [pages * page_tokens, kv_heads * (dim + vdim)], bf16 or fp32: row row_place[r] becomes the keys of all heads, then the values.
    Rows with a negative place are left out.  Two rows with one place leave one of theirs."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v are [rows, heads, values]")
    R, H, D = q.shape
    G, V = k.shape[1], v.shape[2]
    if pool.dtype not in (BF16, F32) or pool.dim() != 2 or not pool.is_contiguous() or pool.shape[1] != G * (D + V) or pool.shape[0] == 0 \
            or pool.shape[0] >= 1 << 31:
        raise ValueError(f"pool must be contiguous rows of {G * (D + V)} values, bf16 or fp32, fewer than 2^31")
    if H == 0 or G == 0 or D == 0 or V == 0 or D > 1024 or max(H, G) > 4096 or (H + G) * D > 51200 - 512:
        raise ValueError("heads of 1 to 1024 values, of all queries and keys at most 50688")
    a = HeadsArgs()
    a.q, a.k, a.v = _projection("q", q, R, H, D), _projection("k", k, R, G, D), _projection("v", v, R, G, V)
    a.q_norm_stride, a.k_norm_stride = _weight("q_norm", q_norm, H, D), _weight("k_norm", k_norm, G, D)
    if freq is not None and (freq.dtype is not F32 or freq.dim() != 1 or not freq.is_contiguous() or 2 * freq.numel() > D):
        raise ValueError(f"freq must be at most {D // 2} contiguous fp32 values")
    if not 0 <= width <= D or not eps >= 0:
        raise ValueError(f"width is 0 to {D}, eps is not negative")
    for name, t in (("row_pos", row_pos), ("row_place", row_place)):
        if t.dtype is not I32 or t.dim() != 1 or not t.is_contiguous() or t.numel() < R:
            raise ValueError(f"{name} must be contiguous 32-bit integers, one per row")
    if out is None:
        out = torch.empty(R, H, D, dtype=pool.dtype, device=q.device)
    if tuple(out.shape) != (R, H, D) or out.dtype != pool.dtype:
        raise ValueError(f"out must be [{R}, {H}, {D}] of the pool's type")
    row, head, one = _steps(out)
    if one != 1 or head != D or row < H * D:
        raise ValueError("out: a row's heads must lie side by side, rows apart")
    _here((("q", q), ("k", k), ("v", v), ("row_pos", row_pos), ("row_place", row_place), ("pool", pool), ("q_norm", q_norm),
           ("k_norm", k_norm), ("freq", freq), ("out", out)))
    if R == 0:
        return out
    a.q_norm, a.k_norm, a.freq = lib.ptr(q_norm), lib.ptr(k_norm), lib.ptr(freq)
    a.row_pos, a.row_place, a.q_out, a.pool = row_pos.data_ptr(), row_place.data_ptr(), out.data_ptr(), pool.data_ptr()
    a.ld_q, a.eps, a.width, a.rows, a.heads, a.kv_heads, a.dim, a.vdim = row, eps, width or D, R, H, G, D, V
    a.rot_dim, a.pool_rows, a.f32 = 0 if freq is None else 2 * freq.numel(), pool.shape[0], int(pool.dtype == F32)
    lib.check(lib.kernels("stack").ds41_ragged_heads(C.byref(a), C.c_void_p(_stream())), "ds41_ragged_heads")
    return out


def attend(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, described: RaggedPass, *, scale: float,
           sink: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Grouped-query attention of a described pass over a paged cache: [rows, heads, vdim].

    q [rows, heads, dim]; pool [pages * page_tokens, kv_heads * (dim + vdim)]: keys of all key/value heads, then their values, the new
    tokens' among them.  `sink` [heads] fp32: an extra logit in a head's denominator; `gate` [rows, heads] fp32: a head's result times
    sigmoid(gate).  Rows behind the last request's are left as `out` has them."""
    p = described
    (q_row, q_head), R = _heads("q", q, p.heads, p.dtype), p.rows
    if tuple(q.shape) != (R, p.heads, p.dim):
        raise ValueError(f"q must be [{R}, {p.heads}, {p.dim}]")
    if p.table_shape is None:
        raise ValueError("the pass has not been described")
    if pool.dtype is not p.dtype or pool.dim() != 2 or not pool.is_contiguous() or pool.shape[1] != p.kv_heads * (p.dim + p.vdim) \
            or pool.data_ptr() % 16:
        raise ValueError(f"pool must be contiguous rows of {p.kv_heads * (p.dim + p.vdim)} values of {p.dtype}, 16-byte aligned")
    if pool.shape[0] != p.n_pages * p.page_tokens or page_table.shape != p.table_shape:
        raise ValueError(f"the pass was described for {p.n_pages} pages and a page table of {tuple(p.table_shape)}")
    _table(page_table, p.n_pages, p.page_tokens)
    if not scale > 0:
        raise ValueError("scale must be positive")
    if out is None:
        out = torch.empty(R, p.heads, p.vdim, dtype=p.dtype, device=q.device)
    if tuple(out.shape) != (R, p.heads, p.vdim) or out.dtype is not p.dtype:
        raise ValueError(f"out must be [{R}, {p.heads}, {p.vdim}] of {p.dtype}")
    step, head, one = _steps(out)
    if one != 1 or head != p.vdim or step % 8 or step < p.heads * p.vdim or out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned, a row's heads side by side and rows apart, at multiples of 8 values")
    if sink is not None and (sink.dtype is not F32 or tuple(sink.shape) != (p.heads,) or not sink.is_contiguous()):
        raise ValueError(f"sink must be {p.heads} contiguous fp32 values")
    if gate is not None and (gate.dtype is not F32 or tuple(gate.shape) != (R, p.heads) or (p.heads > 1 and gate.stride(1) != 1)):
        raise ValueError(f"gate must be fp32 [{R}, {p.heads}] with a row's values side by side")
    _here((("q", q), ("pool", pool), ("page_table", page_table), ("out", out), ("sink", sink), ("gate", gate), ("the pass", p.header)))
    a = AttendArgs(q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), out.data_ptr(), None if gate is None else gate.data_ptr(),
                   None if sink is None else sink.data_ptr(), q_row, q_head, step, 0 if gate is None else gate.stride(0), scale, R,
                   page_table.shape[1], p.n_pages)
    lib.check(lib.kernels("stack").ds41_ragged_attend(C.byref(a), p.args_ref, C.c_void_p(_stream())), "ds41_ragged_attend")
    return out
