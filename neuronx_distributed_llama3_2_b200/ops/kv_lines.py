"""Cache lines that continue other lines, and copies of pages, in all layers at once (``csrc/kv_lines.cu``).  ``inference.kv_cache.KVCache`` and its
``BeamLines`` are the callers of everyday use."""
from __future__ import annotations

import ctypes as _c
from typing import List, Optional, Sequence, Union

import torch

from . import _lib

MAX_BEAMS = 32
_P, _I, _L = _c.c_void_p, _c.c_int, _c.c_longlong
_ARGS = {
    "nxd_reorder_lines": [_P, _I, _I, _I, _P, _P, _P, _P, _I, _I, _P],
    "nxd_copy_pages": [_P, _I, _I, _I, _L, _L, _L, _L, _I, _P, _P, _P, _P],
}


def _entry(name: str):
    fn = getattr(_lib.lib(), name)
    if fn.argtypes is None:
        fn.argtypes = _ARGS[name]
    return fn


class _Kind(_c.Structure):          # nxd_lines
    _fields_ = [("base", _P), ("n", _I), ("heads", _I), ("rows", _L), ("row_bytes", _L), ("line_stride", _L), ("head_stride", _L), ("pages", _I),
                ("whole", _I)]


class _Alike:
    """Tensors of one shape: ``key`` is lines or pages, heads, rows, bytes of a row, strides of lines and heads in bytes."""

    def __init__(self, key: tuple, whole: bool):
        self.key, self.whole, self.tensors, self.at = key, whole, [], []

    def addresses(self):
        at = [f() for f in self.where]
        if at != self.at:          # ``t.data = ...`` moves a tensor
            self.at, self.base = at, (_c.c_void_p * len(at))(*at)
        return self.base


class CacheTensors:
    """The tensors of a cache, laid out for the kernels once: ``cache`` ``[lines or pages, heads, rows, dim]`` with rows side by side (heads and
    lines may be strided, shapes may differ from tensor to tensor), ``states`` ``[lines, ...]`` with a line's values side by side."""

    def __init__(self, cache: Sequence[torch.Tensor], states: Sequence[torch.Tensor] = ()):
        self.cache, self.states = list(cache), list(states)
        if not self.cache and not self.states:
            raise ValueError("a cache without tensors")
        self.device = (self.cache or self.states)[0].device
        if len({t.data_ptr() for t in self.cache + self.states if t.numel()}) < sum(t.numel() > 0 for t in self.cache + self.states):
            raise ValueError("two of the cache's tensors lie in one place")
        if any(n > 1 and s == 0 for t in self.cache + self.states for n, s in zip(t.shape, t.stride())):
            raise ValueError("lines of an expanded tensor lie in one place")
        kinds = {}, {}
        for t in self.cache:
            if t.dim() != 4 or (t.numel() and t.shape[3] > 1 and t.stride(3) != 1) or (t.numel() and t.shape[2] > 1 and t.stride(2) != t.shape[3]):
                raise ValueError(f"a cache tensor [lines, heads, rows, dim] with rows side by side is expected, not {tuple(t.shape)} with "
                                 f"strides {t.stride()}")
            if t.device != self.device:
                raise ValueError(f"cache tensors on {self.device} and on {t.device}")
            size = t.element_size()
            key = (t.shape[0], t.shape[1], t.shape[2], t.shape[3] * size, t.stride(0) * size, t.stride(1) * size)
            kinds[0].setdefault(key, _Alike(key, False)).tensors.append(t)
        for t in self.states:
            if t.dim() < 1 or (t.shape[0] and not t[0].is_contiguous()):
                raise ValueError(f"a state [lines, ...] with a line's values side by side is expected, not {tuple(t.shape)} with strides {t.stride()}")
            if t.device != self.device:
                raise ValueError(f"cache tensors on {self.device} and states on {t.device}")
            size = t.element_size()
            line = t[0].numel() * size if t.shape[0] else 0
            key = (t.shape[0], 1, 1, line, t.stride(0) * size, line)
            kinds[1].setdefault(key, _Alike(key, True)).tensors.append(t)
        self.kinds, self.state_kinds = list(kinds[0].values()), list(kinds[1].values())
        for kind in self.kinds + self.state_kinds:
            kind.where = [t.data_ptr for t in kind.tensors]
        # how many lines there are with and without a block table
        self.lines = min(t.shape[0] for t in self.cache + self.states)
        self.state_lines = min((t.shape[0] for t in self.states), default=None)
        self.cuda = self.device.type == "cuda"
        self.every = self.kinds + self.state_kinds
        self.table = (_Kind * len(self.every))(*[_Kind(0, len(k.tensors), k.key[1], k.key[2], k.key[3], k.key[4], k.key[5], k.key[0], k.whole)
                                                 for k in self.every])


def _laid_out(cache: Union[CacheTensors, Sequence[torch.Tensor]], states: Sequence[torch.Tensor] = ()) -> CacheTensors:
    if isinstance(cache, CacheTensors):
        if states:
            raise ValueError("the states are part of CacheTensors")
        return cache
    return CacheTensors(cache, states)


def _index(name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> torch.Tensor:
    if t.shape != shape or t.dtype not in (torch.int64, torch.int32) or t.device != device:
        raise ValueError(f"{name}: an int64 or int32 tensor {shape} on {device} is expected, not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def reorder_lines_(cache: Union[CacheTensors, Sequence[torch.Tensor]], parents: torch.Tensor, start: Optional[torch.Tensor] = None,
                   end: Optional[torch.Tensor] = None, *, states: Sequence[torch.Tensor] = (), block_table: Optional[torch.Tensor] = None,
                   page_size: int = 0) -> None:
    """Line ``b * W + w`` becomes what line ``b * W + parents[b, w]`` was, in place, in every tensor: rows ``[start[b], end[b])`` of the cache (all
    rows without them) and the states whole.  ``parents``: ``[B, W]``, any map; a parent outside ``[0, W)`` leaves its line as it is.  Lines
    behind ``B * W`` stay as they are, and a line that continues itself costs nothing.  With ``block_table`` ``[lines, pages a line]`` (int32) the
    cache tensors are pages: those that hold the rows must belong to one line each."""
    c = _laid_out(cache, states)
    if parents.dim() != 2 or not 1 <= parents.shape[1] <= MAX_BEAMS:
        raise ValueError(f"parents: [B, W] with up to {MAX_BEAMS} beams is expected, not {tuple(parents.shape)}")
    B, W = parents.shape
    parents = _index("parents", parents, (B, W), c.device)
    start = None if start is None else _index("start", start, (B,), c.device)
    end = None if end is None else _index("end", end, (B,), c.device)
    table = None
    if block_table is not None:
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or not block_table.is_contiguous() or block_table.device != c.device:
            raise ValueError("block_table: a contiguous int32 tensor [lines, pages a line] beside the cache is expected")
        if page_size < 1 or any(k.key[2] != page_size for k in c.kinds):
            raise ValueError(f"page_size {page_size} is not that of the cache's pages")
        table = block_table
    lines = c.lines if table is None else table.shape[0] if c.state_lines is None else min(table.shape[0], c.state_lines)
    if lines < B * W:
        raise ValueError(f"{B} groups of {W} lines are more than the {lines} that there are")
    if not c.cuda or not _lib.available():
        return _reorder_ref(c, parents, start, end, table, page_size)
    if B > 65535:
        raise ValueError(f"{B} groups are more than 65535")
    for kind, entry in zip(c.every, c.table):
        entry.base = _c.addressof(kind.addresses())
    with _lib.on_device_of(parents):
        rc = _entry("nxd_reorder_lines")(c.table, len(c.every), B, W, parents.data_ptr(), 0 if start is None else start.data_ptr(),
                                         0 if end is None else end.data_ptr(), 0 if table is None else table.data_ptr(), page_size,
                                         0 if table is None else table.shape[1], _lib.stream_ptr())
    _lib.check(rc, "nxd_reorder_lines")


def _reorder_ref(c: CacheTensors, parents, start, end, table, page_size) -> None:
    """The same in torch operations."""
    B, W = parents.shape
    for b in range(B):
        p = [x if 0 <= x < W else w for w, x in enumerate(parents[b].tolist())]
        moved = [w for w in range(W) if p[w] != w]
        if not moved:
            continue
        to, frm = [b * W + w for w in moved], [b * W + p[w] for w in moved]
        for t in c.cache:
            rows = t.shape[2] if table is None else table.shape[1] * page_size
            lo = 0 if start is None else max(0, int(start[b]))
            hi = rows if end is None else min(rows, int(end[b]))
            if hi <= lo:
                continue
            if table is None:
                t[to, :, lo:hi] = t[frm, :, lo:hi]
                continue
            pos = torch.arange(lo, hi, device=t.device)
            dst, src = (table[x].long()[:, pos // page_size] for x in (to, frm))          # [moved, rows]
            row = (pos % page_size).expand_as(dst)
            ok = (dst >= 0) & (dst < t.shape[0]) & (src >= 0) & (src < t.shape[0])
            t[dst[ok], :, row[ok]] = t[src[ok], :, row[ok]]
        for t in c.states:
            t[to] = t[frm]


def copy_pages_(cache: Union[CacheTensors, Sequence[torch.Tensor]], src: Union[torch.Tensor, Sequence[int]],
                dst: Union[torch.Tensor, Sequence[int]], *, rows: Union[torch.Tensor, Sequence[int], None] = None) -> None:
    """Page ``dst[i]`` becomes page ``src[i]`` in every tensor ``[pages, heads, rows, dim]``; with ``rows``, only its first ``rows[i]`` rows of every head.
    No page may be written twice or be among those that are read; lists are checked for that, and for pages that there are not.  Of tensors on the
    GPU a pair outside the pool is passed by."""
    c = _laid_out(cache)
    if not c.cache:
        return
    if not (isinstance(src, torch.Tensor) and isinstance(dst, torch.Tensor) and (rows is None or isinstance(rows, torch.Tensor))):
        src, dst, rows = _from_lists(c, src, dst, rows)
    n = src.shape[0] if src.dim() else -1
    src, dst = _index("src", src, (n,), c.device), _index("dst", dst, (n,), c.device)
    rows = None if rows is None else _index("rows", rows, (n,), c.device)
    if n == 0:
        return
    if not c.cuda or not _lib.available():
        return _copy_ref(c, src, dst, rows)
    fn = _entry("nxd_copy_pages")
    with _lib.on_device_of(src):
        for k in c.kinds:
            lead, heads, page, row, line, head = k.key
            rc = fn(k.addresses(), len(k.at), lead, heads, page, row, line, head, n, src.data_ptr(), dst.data_ptr(),
                    0 if rows is None else rows.data_ptr(), _lib.stream_ptr())
            _lib.check(rc, "nxd_copy_pages")


def _from_lists(c: CacheTensors, src, dst, rows):
    """What comes as lists is checked here and brought to the device, in one copy."""
    pages = min(k.key[0] for k in c.kinds)
    lists = [None if x is None or isinstance(x, torch.Tensor) else [int(i) for i in x] for x in (src, dst, rows)]
    if len(dst) != len(src) or (rows is not None and len(rows) != len(src)):
        raise ValueError(f"{len(src)} pages to copy, {len(dst)} to copy to" + ("" if rows is None else f", rows of {len(rows)}"))
    for name, x in zip(("src", "dst"), lists):
        if x is not None and any(not 0 <= i < pages for i in x):
            raise ValueError(f"{name}: page {next(i for i in x if not 0 <= i < pages)} is not one of the {pages} that there are")
    if lists[1] is not None:
        if len(set(lists[1])) != len(lists[1]):
            raise ValueError("dst: a page is written twice")
        if lists[0] is not None and set(lists[0]) & set(lists[1]):
            raise ValueError(f"page {min(set(lists[0]) & set(lists[1]))} is both read and written")
    packed = iter(torch.tensor([x for x in lists if x is not None], dtype=torch.int64).to(c.device, non_blocking=True))
    return tuple(next(packed) if x is not None else given for x, given in zip(lists, (src, dst, rows)))


def _copy_ref(c: CacheTensors, src, dst, rows) -> None:
    """The same in torch operations."""
    for t in c.cache:
        for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
            if 0 <= a < t.shape[0] and 0 <= b < t.shape[0]:
                n = t.shape[2] if rows is None else max(0, min(t.shape[2], int(rows[i])))
                t[b, :, :n] = t[a, :, :n]
