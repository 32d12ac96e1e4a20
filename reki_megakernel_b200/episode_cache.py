"""Paged K/V cache of many episodes: placing new rows, storing them, and attention over them
(``include/mkx_cache.h``).

The expert reads K/V that are dense per episode ([SP, NH, HD] per layer, src/mk_expert.py:486-495);
episodes of different lengths then all take the longest one's memory. Here the rows of all episodes
share one pool of pages. One step of serving is

1. ``plan_rows``: pages for the new rows of each episode, block tables and slot maps, from the
   episodes' lengths, on the GPU (nothing is read back);
2. ``write_rows``: rotary positions (one to four axes: index, or time / height / width of image rows)
   on q and k, K and V rows to their slots, in one pass;
3. ``attend``: the new rows over all rows of their episode -- single rows to long chunks, causal or
   not, with a sliding window and first rows that stay visible.

``EpisodeCache`` keeps the pools, tables and counters of such a cache. ``rope_tables`` makes the
cos / sin tables of the same positions for ``RegisterPrepare.run`` and ``ExpertMegakernel.run``. All
calls are asynchronous on the current stream of the tensors' device and can be captured in a CUDA
graph. There is no CPU fallback: the CUDA library must load. Inference only: nothing records gradients, and a tensor that
requires grad is refused unless ``torch.no_grad()`` says that none are wanted.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import NamedTuple

import torch

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1}
PAGE_ROWS = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)          # of attend
MAX_EPISODES = 4096
MAX_ROWS = 1 << 30             # rows of one episode that a table can hold


class RowPlan(NamedTuple):
    """Where the new rows of a step go. start [B + 1] int32: first row of each episode; slot [rows] int64 (-1: none),
    episode and position [rows] int32; length [B] int32 and marks [3] int64: the state after the step."""
    start: torch.Tensor
    slot: torch.Tensor
    episode: torch.Tensor
    position: torch.Tensor
    length: torch.Tensor
    marks: torch.Tensor


# Calls go through ``_mkx_torch`` (csrc/mk_torch.cpp), which checks, allocates and launches in one step and answers None
# to arguments it does not accept; the checks below then say what is wrong.

def _vector(t, name: str, n: int, dtype, device) -> None:
    if t.dtype != dtype or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [{n}] tensor on {device}")


def _check_table(table, B: int, page_rows: int, device) -> None:
    shape = table.shape
    if (len(shape) != 2 or shape[0] != B or shape[1] < 1 or table.dtype != torch.int32 or table.device != device
            or not table.is_contiguous()):
        raise ValueError(f"table must be a contiguous int32 [{B}, pages] tensor on {device}")
    if shape[1] * page_rows > MAX_ROWS:
        raise ValueError(f"a table row may hold up to {MAX_ROWS} rows")


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device")
    return t.device


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _check_strides(t: torch.Tensor, name: str, apart: bool = False) -> None:
    """Dims must be contiguous, rows, heads and pages 16 bytes apart or a multiple, and the start 16-byte aligned. What is
    written to, and the pages that attend reads by TMA, are no expanded tensors (``apart``)."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dim must be contiguous")
    if t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        raise ValueError(f"{name}: rows, heads and pages must start on 16-byte boundaries")
    if apart and any(s == 0 for s, n in zip(t.stride(), t.shape) if n > 1):
        raise ValueError(f"{name} must not be expanded: several of its rows, heads or pages share a place")


def _check_gradients(**tensors) -> None:
    """Nothing here is differentiable: a tensor that requires grad is refused while gradients are recorded."""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} requires grad, and no gradients are recorded: call under torch.no_grad(), or detach it")


def _refused(what: str):
    return ValueError(f"{what}: these arguments are not supported")


# ---- placing ----------------------------------------------------------------------------------------

def check_plan_args(length, new, table, free, marks, page_rows: int, rows: int) -> None:
    """What ``plan_rows`` checks before it hands raw pointers to the library. Raises ValueError."""
    dev, B = length.device, length.numel()
    if not 1 <= B <= MAX_EPISODES:
        raise ValueError(f"1 to {MAX_EPISODES} episodes")
    if page_rows not in PAGE_ROWS:
        raise ValueError(f"page_rows must be one of {PAGE_ROWS}")
    if not 0 <= rows < 1 << 31:
        raise ValueError("rows must be in 0 .. 2^31 - 1")
    _vector(length, "length", B, torch.int32, dev)
    _vector(new, "new", B, torch.int32, dev)
    _vector(free, "free", max(1, free.numel()), torch.int32, dev)
    _vector(marks, "marks", 3, torch.int64, dev)
    _check_table(table, B, page_rows, dev)


def plan_rows(length: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, marks: torch.Tensor, *,
              page_rows: int, rows: int, ticket: torch.Tensor | None = None) -> RowPlan:
    """Places ``new[b]`` rows behind the ``length[b]`` rows that episode b holds: pages off the ring ``free``, their
    table entries (``table`` [B, pages] int32, written in place), and the new rows' start, slot, episode and position.

    ``marks`` [3] int64: pages ever taken, pages ever returned (their difference is free, the next at
    ``free[taken % len(free)]``), and, in the returned marks, the new rows that got no slot. ``rows``: how many rows
    the step has room for; rows behind the last new one get slot -1. The returned length and marks are the state after
    the step: new tensors, or, with a ``ticket`` ([1] int32, zero, a word that only plans of this state use), the
    arguments themselves, advanced in place."""
    r = _lib.load_torch().plan(length, new, table, free, marks, page_rows, rows, ticket)
    if type(r) is tuple:
        return RowPlan(*r)
    if r is None:
        _cuda(length, "length")
        check_plan_args(length, new, table, free, marks, page_rows, rows)
        if ticket is not None:
            _vector(ticket, "ticket", 1, torch.int32, length.device)
        raise _refused("plan_rows")
    _lib.check(r, "mkx_cache_plan")


# ---- rotary positions and storing -------------------------------------------------------------------

@functools.lru_cache(maxsize=64)
def _rotary(head_dim: int, sections, base: float, interleaved: bool):
    """(the struct ``mkx_rotary`` as bytes, number of axes)."""
    sections = sections if sections is not None else (head_dim // 2,)
    half = sum(sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or half < 8 or half % 8 or 2 * half > head_dim:
        raise ValueError(f"sections must be 1 to 4 counts whose sum is a multiple of 8 up to {head_dim // 2}")
    if not (base > 0 and math.isfinite(base) and math.isfinite(1 / base)):
        raise ValueError("base must be positive")
    return _lib.pack_rotary(base, len(sections), *sections, *(0,) * (4 - len(sections)), int(interleaved)), len(sections)


def _sections(sections):
    return sections if sections is None or type(sections) is tuple else tuple(sections)


def _positions(positions: torch.Tensor, axes: int, rows: int, device) -> torch.Tensor:
    if positions.dim() == 1:
        positions = positions[None]
    if (positions.dtype != torch.int32 or tuple(positions.shape) != (axes, rows) or positions.device != device
            or (rows > 1 and positions.stride(1) != 1)):
        raise ValueError(f"positions must be int32 [{axes}, {rows}] on {device}, each axis contiguous")
    return positions


def rope_tables(positions: torch.Tensor, head_dim: int, *, sections=None, base: float = 10000.0,
                interleaved: bool = False):
    """cos, sin [rows, head_dim] fp32 of ``positions`` [axes, rows] (or [rows]) int32. Frequency i of ``sum(sections)``
    (default: one axis, head_dim / 2) belongs to dims i and i + sum(sections), the others get 1 and 0; see ``write_rows``.
    ``RegisterPrepare.run`` and ``ExpertMegakernel.run`` turn dims i and i + head_dim / 2 together: for them the
    sections add up to head_dim / 2."""
    dev = _cuda(positions, "positions")
    if not 16 <= head_dim <= 256 or head_dim % 16:
        raise ValueError("head_dim must be a multiple of 16 up to 256")
    rot, axes = _rotary(head_dim, _sections(sections), base, interleaved)
    rows = positions.shape[-1]
    positions = _positions(positions, axes, rows, dev)
    cos = torch.empty((rows, head_dim), dtype=torch.float32, device=dev)
    sin = torch.empty_like(cos)
    _lib.check(_lib.load().mkx_rope_tables(rot, positions.data_ptr(), positions.stride(0), rows, head_dim,
                                           cos.data_ptr(), sin.data_ptr(), dev.index, _stream(dev)), "mkx_rope_tables")
    return cos, sin


def check_write_args(k, v, slot, k_pages, v_pages, q, positions, out) -> None:
    """What ``write_rows`` checks of shapes, types and devices. Raises ValueError."""
    shape, dtype, dev = k.shape, k.dtype, k.device
    if len(shape) != 3 or v.shape != shape or shape[1] < 1:
        raise ValueError("k and v must be [rows, kv_heads, head_dim] alike")
    rows, heads, hd = shape
    if dtype not in DTYPES or not 16 <= hd <= 256 or hd % 16:
        raise ValueError("k must be bf16 or fp16 with a head_dim that is a multiple of 16 up to 256")
    pool = k_pages.shape
    if (len(pool) != 4 or v_pages.shape != pool or pool[2] != heads or pool[3] != hd or pool[0] < 1
            or pool[1] not in PAGE_ROWS):
        raise ValueError(f"k_pages and v_pages must be [pages, page_rows, {heads}, {hd}] with page_rows in {PAGE_ROWS}")
    if v.dtype != dtype or v.device != dev:
        raise ValueError(f"v must be {dtype} on {dev}")
    for t in (k_pages, v_pages):
        if t.dtype != dtype or t.device != dev:
            raise ValueError(f"k_pages and v_pages must be {dtype} on {dev}")
    _vector(slot, "slot", rows, torch.int64, dev)
    _check_gradients(k=k, v=v, k_pages=k_pages, v_pages=v_pages, q=q, out=out)
    if q is None:
        if out is not None:
            raise ValueError("out belongs to q")
        return
    if positions is None:
        raise ValueError("q is only rotated: it needs positions")
    qs = q.shape
    if len(qs) != 3 or qs[0] != rows or qs[1] < 1 or qs[2] != hd or q.dtype != dtype or q.device != dev:
        raise ValueError(f"q must be {dtype} [{rows}, heads, {hd}] on {dev}")
    if out is not None and (out.shape != qs or out.dtype != dtype or out.device != dev):
        raise ValueError("out must be like q")


def write_rows(k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
               q: torch.Tensor | None = None, positions: torch.Tensor | None = None, sections=None,
               base: float = 10000.0, interleaved: bool = False, out: torch.Tensor | None = None):
    """Stores rows ``k``, ``v`` [rows, kv_heads, head_dim] at ``slot`` [rows] int64 of the pages [pages, page_rows,
    kv_heads, head_dim] (a slot outside of them is skipped; two rows must not share one). With ``positions``
    [axes, rows] (or [rows]) int32, k is rotated on the way, and so is ``q`` [rows, heads, head_dim] into the returned
    tensor (``out`` when given; ``out`` may be q).

    Dims i and i + h, h = sum(sections), turn by positions[axis(i)] * base^(-i / h); dims from 2 h on pass through.
    ``sections``: frequencies per axis (default: one axis with head_dim / 2); axis(i) goes through them one axis after
    the other, or, ``interleaved``, over the axes in turn while each has some left. Tensors may be slices: dims
    contiguous, rows, heads and pages on 16-byte boundaries."""
    rot = None
    if positions is not None:
        rot, axes = _rotary(k.shape[-1], _sections(sections), base, interleaved)
    r = _lib.load_torch().store(k, v, slot, k_pages, v_pages, q, positions, rot, out)
    if r is None:
        _cuda(k, "k")
        check_write_args(k, v, slot, k_pages, v_pages, q, positions, out)
        if positions is not None:
            _positions(positions, axes, k.shape[0], k.device)
        for name, t in (("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("q", q), ("out", out)):
            if t is not None:
                _check_strides(t, name, apart=name in ("k_pages", "v_pages", "out"))
        raise _refused("write_rows")
    if type(r) is int:
        _lib.check(r, "mkx_cache_store")
    return None if r is True else r


# ---- attention ----------------------------------------------------------------------------------------

def check_attend_args(q, k_pages, v_pages, table, length, start, max_rows, causal, window, sinks, scale, out) -> None:
    """What ``attend`` checks of shapes, types, devices and values. Raises ValueError."""
    shape, dtype, dev = q.shape, q.dtype, q.device
    if len(shape) != 3 or dtype not in DTYPES or shape[2] not in HEAD_DIMS:
        raise ValueError(f"q must be bf16 or fp16 [rows, heads, head_dim], head_dim in {HEAD_DIMS}")
    pool = k_pages.shape
    if (len(pool) != 4 or v_pages.shape != pool or pool[3] != shape[2] or pool[0] < 1 or pool[1] not in PAGE_ROWS
            or pool[2] < 1):
        raise ValueError(f"k_pages and v_pages must be [pages, page_rows, kv_heads, {shape[2]}] with page_rows in {PAGE_ROWS}")
    if shape[1] < 1 or shape[1] % pool[2]:
        raise ValueError("heads must be a multiple of kv_heads")
    for t in (k_pages, v_pages):
        if t.dtype != dtype or t.device != dev:
            raise ValueError(f"k_pages and v_pages must be {dtype} on {dev}")
    B = length.numel()
    if not 1 <= B <= MAX_EPISODES:
        raise ValueError(f"1 to {MAX_EPISODES} episodes")
    _vector(length, "length", B, torch.int32, dev)
    _vector(start, "start", B + 1, torch.int32, dev)
    _check_table(table, B, pool[1], dev)
    if max_rows is not None and max_rows < 0:
        raise ValueError("max_rows must not be negative")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if window > 0 and not causal:
        raise ValueError("a window needs causal=True")
    if sinks > 0 and window == 0:
        raise ValueError("sinks are the rows that stay visible beside a window")
    if scale is not None and not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if out is not None and (out.shape != shape or out.dtype != dtype or out.device != dev):
        raise ValueError("out must be like q")
    _check_gradients(q=q, k_pages=k_pages, v_pages=v_pages, out=out)


def attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, length: torch.Tensor,
           start: torch.Tensor, *, max_rows: int | None = None, causal: bool = True, window: int = 0, sinks: int = 0,
           scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new rows ``q`` [rows, heads, head_dim] over the pages [pages, page_rows, kv_heads, head_dim];
    heads / kv_heads query heads share a K/V head. Rows ``start[b] .. start[b + 1] - 1`` are the last ones of the
    ``length[b]`` rows of episode b (stored before: see ``write_rows``), whose row j lies in page
    ``table[b, j // page_rows]``.

    A row at position p sees the rows j < length[b] of its episode with j <= p (all of them if not ``causal``) and,
    with a ``window`` > 0, with j > p - window or j < ``sinks``. out = softmax(scale q k^T) v (scale: 1 / sqrt(head_dim)),
    zero for a row that sees nothing, NaN where a score is NaN or infinite; rows behind start[B] are left as they were. ``out`` may be q. What pages hold beyond an
    episode's length does not matter; the K and V rows below it are finite. ``max_rows``: no episode has more new rows
    (default: q's rows). The kernel is chosen by ``max_rows`` and by what a table row can hold, so tight values of both
    pick the one that fits; that of long chunks (more than 16 rows of a K/V head) rounds each probability to 16 bits
    before the second product, the other keeps twice as many. A wait that ran out on the device surfaces in
    ``check_device_error()``."""
    most = -1 if max_rows is None else max_rows if max_rows >= 0 else -2  # -1: q's rows; below: refused
    r = _lib.load_torch().attend(q, k_pages, v_pages, table, length, start, most, causal, window, sinks, scale, out)
    if r is None:
        _cuda(q, "q")
        check_attend_args(q, k_pages, v_pages, table, length, start, max_rows, causal, window, sinks, scale, out)
        for name, t in (("q", q), ("k_pages", k_pages), ("v_pages", v_pages), ("out", out)):
            if t is not None:
                _check_strides(t, name, apart=name != "q")
        raise _refused("attend")
    if r is False:
        raise RuntimeError("call attend once on this device before its first capture")
    if type(r) is int:
        _lib.check(r, "mkx_cache_attend")
    return r


def check_device_error(device=None) -> None:
    """Raises if a bounded wait of an ``attend`` on ``device`` ran out since the last check (synchronises)."""
    index = None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    code = _lib.load_torch().error_code(index, False)
    if code:
        raise _lib.MkxError("attend", _lib.MKX_ERR_DEVICE, f"error word {code:#x}")


# ---- the cache ------------------------------------------------------------------------------------------

class EpisodeCache:
    """Pools, tables and counters of a paged cache: ``EpisodeCache(layers=..., pages=..., episodes=...)``.

    k, v [layers, pages, page_rows, kv_heads, head_dim]; table [episodes, pages_per_episode] int32; length [episodes]
    int32; free [pages] int32 (a ring) and marks [3] int64. One step:

        plan = cache.plan(new, rows)                 # new [episodes] int32 rows per episode, sum <= rows
        q = cache.write(layer, k, v, plan, q=q, positions=..., sections=...)
        out = cache.attend(layer, q, plan, max_rows=..., window=..., sinks=...)

    ``plan`` advances the state in place (in stream order), so a captured step can be replayed. ``release`` returns
    the pages of episodes that ended."""

    def __init__(self, *, layers: int, pages: int, episodes: int, page_rows: int = 32, kv_heads: int = 12,
                 head_dim: int = 64, pages_per_episode: int | None = None, dtype=torch.bfloat16, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("EpisodeCache needs a CUDA device")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        if layers < 1 or pages < 1 or kv_heads < 1:
            raise ValueError("layers, pages and kv_heads must be positive")
        if not 1 <= episodes <= MAX_EPISODES:
            raise ValueError(f"1 to {MAX_EPISODES} episodes")
        if page_rows not in PAGE_ROWS:
            raise ValueError(f"page_rows must be one of {PAGE_ROWS}")
        if head_dim not in HEAD_DIMS or dtype not in DTYPES:
            raise ValueError(f"head_dim in {HEAD_DIMS}, bf16 or fp16")
        wide = pages if pages_per_episode is None else pages_per_episode
        if wide < 1 or wide * page_rows > MAX_ROWS:
            raise ValueError(f"an episode may hold up to {MAX_ROWS} rows")
        _lib.load_torch().error_code(dev.index, True)  # allocates the device's error word, which a capture could not
        self.device, self.page_rows, self.episodes = dev, page_rows, episodes
        self.k = torch.zeros((layers, pages, page_rows, kv_heads, head_dim), dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((episodes, wide), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(episodes, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.marks = torch.tensor([0, pages, 0], dtype=torch.int64, device=dev)
        self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)

    def plan(self, new: torch.Tensor, rows: int) -> RowPlan:
        """Places ``new`` [episodes] int32 rows (device); ``rows`` is the room of the step's row tensors. The plan's
        length and marks are the cache's own. Rows without a slot are counted in ``marks[2]``: their episodes grew by
        the stored rows alone, fewer than the plan's ``start`` says, so that step is not one to ``attend`` with."""
        return plan_rows(self.length, new, self.table, self.free, self.marks, page_rows=self.page_rows, rows=rows,
                         ticket=self._ticket)

    def release(self, ended: torch.Tensor) -> None:
        """Returns all pages of the episodes with ``ended`` [episodes] (bool) to the free ring, length 0."""
        _vector(ended, "ended", self.episodes, torch.bool, self.device)
        a = _lib.ReleaseInputs(ended.data_ptr(), self.length.data_ptr(), self.table.data_ptr(), self.free.data_ptr(),
                               self.marks.data_ptr(), self._ticket.data_ptr(), self.episodes, self.table.shape[1],
                               self.free.shape[0], self.page_rows)
        _lib.check(_lib.load().mkx_cache_release(C.byref(a), self.device.index, _stream(self.device)), "mkx_cache_release")
        for t in (self.length, self.table, self.free, self.marks, self._ticket):
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: RowPlan, **kw):
        """``write_rows`` into the pages of ``layer``."""
        return write_rows(k, v, plan.slot, self.k[layer], self.v[layer], **kw)

    def attend(self, layer: int, q: torch.Tensor, plan: RowPlan, **kw) -> torch.Tensor:
        """``attend`` over the pages of ``layer``."""
        return attend(q, self.k[layer], self.v[layer], self.table, self.length, plan.start, **kw)

    def check_device_error(self) -> None:
        check_device_error(self.device)
