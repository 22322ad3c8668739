"""KV cache state for the inference graphs (reference keeps the cache as aliased parameters of the compiled
graph and re-emits the whole cache every step, ``examples/inference/modules/model_base.py:114-125,388-422``).

Here the cache is a plain device allocation per layer that the kernels update IN PLACE:
  contiguous  ``[lines, kv_heads_local, seq_len, head_dim]``
  paged       ``[pages, kv_heads_local, page_size, head_dim]`` + a block table ``[lines, max_pages]``

Paged mode has two flavours: the static identity mapping (every line owns ``max_pages`` pages up front) and, with
``num_pages``, a POOL smaller than ``lines * max_pages`` managed by the native page allocator
(``runtime.native.PagedKVPool``): lines get pages as they grow (``reserve``), give them back (``free``), can be forked
copy-on-write (``fork``) and rolled back (``truncate``).  The block table is a device tensor updated in place, so CUDA
graphs that captured it see the new mapping.

Layers need not be alike: ``layer_specs[i] = (kv_heads, key_dim, value_dim)`` gives layer ``i`` its own shapes (key and
value sizes may differ), and ``share_from[i] = j`` makes layer ``i`` read layer ``j``'s keys and values instead of
holding its own (cross-layer KV sharing: ``layer(i)`` returns ``j``'s tensors, nothing is allocated for ``i``).
A spec ``(kv_heads, key_dim, value_dim, "columns")`` keeps ONE tensor per layer whose value is the first ``value_dim``
columns of the key rows (the latent cache of a compressed key/value projection); a spec ``None`` is a layer without
keys and values; a spec ``(kv_heads, key_dim, value_dim, "heads", value_heads)`` gives the value tensor its own number
of heads (several attention maps -- key heads -- over the same values).

Recurrent layers keep a STATE per cache line instead: ``state_specs[i] = {name: shape}`` allocates fp32 tensors
``[lines, *shape]`` (``state(i)``).  State is per line, not per page: ``fork`` copies it, and a layer that starts a
sequence at position 0 starts from zero by itself, so a line that is handed out again needs no clearing.
"""
from __future__ import annotations

from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import torch

from ..ops.kv_lines import CacheTensors, copy_pages_, reorder_lines_


class KVCache:
    def __init__(self, num_layers: int, lines: int, kv_heads: int, seq_len: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None, paged: bool = False, page_size: int = 128,
                 num_pages: Optional[int] = None, layer_specs: Optional[List[Optional[Tuple[int, int, int]]]] = None,
                 share_from: Optional[Dict[int, int]] = None,
                 state_specs: Optional[Dict[int, Dict[str, Tuple[int, ...]]]] = None):
        self.num_layers, self.lines, self.kv_heads, self.seq_len, self.head_dim = num_layers, lines, kv_heads, seq_len, head_dim
        self.share_from = dict(share_from or {})
        for i, j in self.share_from.items():
            if j in self.share_from or not (0 <= j < num_layers) or j == i:
                raise ValueError(f"layer {i} cannot share the keys/values of layer {j}")
        specs = layer_specs if layer_specs is not None else [(kv_heads, head_dim, head_dim)] * num_layers
        self.paged, self.page_size = paged, page_size
        self.pool = None
        self._laid_out: Optional[CacheTensors] = None
        self._held: tuple = ()
        if paged:
            self.max_pages = (seq_len + page_size - 1) // page_size
            if num_pages is None:
                n_pages = lines * self.max_pages
                # static identity mapping: every line owns its pages up front
                self.block_table = torch.arange(n_pages, dtype=torch.int32, device=device).reshape(lines, self.max_pages)
            else:
                from ..runtime.native import PagedKVPool

                n_pages = num_pages
                self.pool = PagedKVPool(n_pages, page_size, lines, self.max_pages)
                self.block_table = torch.zeros(lines, self.max_pages, dtype=torch.int32, device=device)
            lead, rows = n_pages, page_size
        else:
            lead, rows = lines, seq_len
            self.block_table = None
        self.k: List[Optional[torch.Tensor]] = []
        self.v: List[Optional[torch.Tensor]] = []
        for i in range(num_layers):
            if i in self.share_from:
                self.k.append(None)
                self.v.append(None)
                continue
            if specs[i] is None:                       # a layer without keys and values (recurrent state only)
                self.k.append(None)
                self.v.append(None)
                continue
            g, dk, dv = specs[i][:3]
            self.k.append(torch.zeros((lead, g, rows, dk), dtype=dtype, device=device))
            if len(specs[i]) > 3 and specs[i][3] == "columns":
                self.v.append(self.k[-1][..., :dv])    # the values are columns of the key rows: one tensor
            elif len(specs[i]) > 4 and specs[i][3] == "heads":
                self.v.append(torch.zeros((lead, int(specs[i][4]), rows, dv), dtype=dtype, device=device))
            else:
                self.v.append(torch.zeros((lead, g, rows, dv), dtype=dtype, device=device))
        self.states: Dict[int, Dict[str, torch.Tensor]] = {
            i: {name: torch.zeros((lines,) + tuple(shape), dtype=torch.float32, device=device)
                for name, shape in spec.items()} for i, spec in (state_specs or {}).items()}

    def owns(self, i: int) -> bool:
        """False for a layer that reads another layer's keys and values."""
        return i not in self.share_from

    def layer(self, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        i = self.share_from.get(i, i)
        return self.k[i], self.v[i]

    def state(self, i: int) -> Dict[str, torch.Tensor]:
        """The recurrent state tensors ``[lines, ...]`` (fp32) of layer ``i``."""
        return self.states[i]

    def _tensors(self) -> List[torch.Tensor]:
        """Every allocation once (a value tensor that is a column range of its key tensor is not one)."""
        out = []
        for t in self.k + self.v:
            if t is not None and t._base is None:
                out.append(t)
        return out

    def _state_tensors(self) -> List[torch.Tensor]:
        return [t for d in self.states.values() for t in d.values()]

    def reset(self) -> None:
        for t in self._tensors() + self._state_tensors():
            t.zero_()
        if self.pool is not None:
            for line in range(self.lines):
                self.pool.free_line(line)
            self.block_table.zero_()

    # -- dynamic page pool (no-ops for the contiguous cache and the static mapping) ---------------------------------------
    def sync_lines(self, lines: Iterable[int]) -> None:
        """Copy the allocator's page lists of ``lines`` into the device block table."""
        if self.pool is None:
            return
        rows = list(lines)
        if not rows:
            return
        host = torch.tensor([self.pool.block_row(r)[0] for r in rows], dtype=torch.int32)
        self.block_table[torch.tensor(rows, dtype=torch.long, device=self.block_table.device)] = host.to(
            self.block_table.device, non_blocking=True)

    def reserve(self, line: int, n_tokens: int) -> None:
        """Room for ``n_tokens`` tokens in total on ``line`` (``MemoryError`` when the pool is exhausted)."""
        if self.pool is not None and self.pool.reserve(line, n_tokens) > 0:
            self.sync_lines([line])

    def free(self, line: int) -> None:
        if self.pool is not None:
            self.pool.free_line(line)

    def truncate(self, line: int, n_tokens: int) -> None:
        if self.pool is not None and self.pool.truncate(line, n_tokens) > 0:
            self.sync_lines([line])

    @property
    def tensors(self) -> CacheTensors:
        """The cache's tensors, laid out for the kernels that move lines and pages of all layers at once."""
        held = (*self.k, *self.v, *self._state_tensors())
        if self._laid_out is None or len(held) != len(self._held) or any(a is not b for a, b in zip(held, self._held)):
            self._laid_out, self._held = CacheTensors(self._tensors(), self._state_tensors()), held
        return self._laid_out

    def copy_pages(self, src: Sequence[int], dst: Sequence[int], rows: Optional[Sequence[int]] = None) -> None:
        """Page ``dst[i]`` becomes page ``src[i]`` in every layer (its first ``rows[i]`` rows); no page may be in both lists."""
        assert self.paged, "a contiguous cache has no pages"
        if len(src):
            copy_pages_(self.tensors, src, dst, rows=rows)

    def fork(self, src: int, dst: int) -> None:
        """``dst`` continues from ``src``'s content: full pages shared, the partial last page copied."""
        self.fork_lines(src, [dst])

    def fork_lines(self, src: int, dsts: Sequence[int], whole_pages: bool = True) -> None:
        """Every line of ``dsts`` continues from ``src``'s content: full pages are shared, the partial last page is copied for all of them in one
        launch (with ``whole_pages`` false only the rows of the reserved tokens).  If the pool has not enough pages no line is forked."""
        assert self.pool is not None, "fork needs the dynamic page pool (num_pages=...)"
        dsts, copies, forked = list(dsts), [], []
        try:
            for dst in dsts:
                copy = self.pool.fork(src, dst)
                forked.append(dst)
                if copy is not None:
                    copies.append(copy)
        except MemoryError:
            for dst in forked:
                self.pool.free_line(dst)
            raise
        rows = None if whole_pages else [self.pool.line_tokens(src) % self.page_size] * len(copies)
        self.copy_pages([a for a, _ in copies], [b for _, b in copies], rows)
        for t in self._state_tensors() if dsts else ():
            t[dsts] = t[src].clone()
        self.sync_lines(dsts)

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool, on the device in one launch a layer shape; the number of pages in use."""
        assert self.pool is not None, "compact needs the dynamic page pool (num_pages=...)"
        moves = self.pool.compact()
        self.copy_pages([a for a, _ in moves], [b for _, b in moves])
        self.sync_lines(range(self.lines))
        return self.pool.num_pages - self.pool.num_free

    def resize_pool(self, num_pages: int) -> None:
        """A pool of another size: the pages in use move to the front and into new tensors, the old ones are let go.  ``MemoryError`` if more are in
        use; where a new tensor cannot be had the cache keeps working and may be resized again.  What holds the old tensors (a captured graph,
        ``BeamLines``) has to be made again."""
        used = self.compact()
        if used > num_pages or num_pages < 1:
            raise MemoryError(f"{used} pages are in use, {num_pages} are not enough")
        # where memory runs out on the way, the allocator names no page that a tensor has not
        shrinks = num_pages < self.pool.num_pages
        if shrinks:
            self.pool.resize(num_pages)
        self._laid_out, self._held = None, ()          # they hold the old tensors
        for i in range(self.num_layers):
            if self.k[i] is None:
                continue
            dim, columns = self.v[i].shape[-1], self.v[i]._base is not None
            self.k[i] = self._resized(self.k[i], num_pages, used)
            self.v[i] = self.k[i][..., :dim] if columns else self._resized(self.v[i], num_pages, used)
        if not shrinks:
            self.pool.resize(num_pages)

    @staticmethod
    def _resized(t: torch.Tensor, num_pages: int, used: int) -> torch.Tensor:
        new = torch.zeros((num_pages,) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device)
        new[:used] = t[:used]
        return new

    def reorder_lines(self, parents: torch.Tensor, start: Optional[torch.Tensor] = None, end: Optional[torch.Tensor] = None) -> None:
        """Line ``b * W + w`` becomes what line ``b * W + parents[b, w]`` was (``parents [B, W]``): rows ``[start[b], end[b])`` of every layer, and its
        recurrent state.  With a dynamic pool ``end`` has to be given, within what the lines have reserved, and pages that hold these rows must not
        be shared (``BeamLines`` sees to both)."""
        if self.pool is not None and end is None:
            raise ValueError("end: the rows of a dynamic pool end where the lines' reservations do")
        reorder_lines_(self.tensors, parents, start, end, block_table=self.block_table, page_size=self.page_size if self.paged else 0)

    def beams(self, lengths: Sequence[int], width: int, new_tokens: int = 0) -> "BeamLines":
        """Lines ``b * width`` hold prompts of ``lengths[b]`` tokens: the ``width`` lines of each request continue it, with room for ``new_tokens``
        more."""
        return BeamLines(self, lengths, width, new_tokens)

    def prepare_write(self, line: int, pos: int) -> None:
        """Before writing position ``pos`` of ``line``: give the line a private copy of that page if it is shared."""
        if self.pool is None:
            return
        copy = self.pool.unshare(line, pos)
        if copy is not None:
            self.copy_pages([copy[0]], [copy[1]])
            self.sync_lines([line])

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._tensors() + self._state_tensors())


class BeamLines:
    """The cache lines of a beam search: line ``b * width + w`` is beam ``w`` of request ``b``.  A prompt is computed once, on its request's first
    line, and spread over the others here: shared pages with a dynamic pool (the beams' own rows are private), copied rows otherwise.  ``reorder`` then
    moves only what lies behind the prompts.  Where a pool has not enough pages (``MemoryError``) the prompts stay and the other lines are free."""

    def __init__(self, cache: KVCache, lengths: Sequence[int], width: int, new_tokens: int = 0):
        lengths = [int(n) for n in lengths]
        if not lengths or not 1 <= width <= 32 or len(lengths) * width > cache.lines:
            raise ValueError(f"{len(lengths)} requests of {width} beams: between 1 and 32 beams, {cache.lines} cache lines")
        if min(lengths) < 0 or new_tokens < 0 or max(lengths) + new_tokens > cache.seq_len:
            raise ValueError(f"prompts of up to {max(lengths)} tokens and {new_tokens} more do not fit a cache of {cache.seq_len}")
        self.cache, self.lengths, self.width = cache, lengths, width
        device = next(t.device for t in cache._tensors() + cache._state_tensors())
        self.start = torch.tensor(lengths, dtype=torch.int64, device=device)
        self.limit = self.start + new_tokens
        lines = range(len(lengths) * width)
        if cache.pool is None:
            if width > 1:
                cache.reorder_lines(torch.zeros(len(lengths), width, dtype=torch.int64, device=device), None, self.start)
            return
        for b, n in enumerate(lengths):
            if cache.pool.line_tokens(b * width) < n:
                raise ValueError(f"line {b * width} has room for {cache.pool.line_tokens(b * width)} tokens, its prompt has {n}")
        for line in lines:
            if line % width:
                cache.free(line)
        try:
            for b, n in enumerate(lengths):
                cache.truncate(b * width, n)
                if n % cache.page_size:
                    cache.prepare_write(b * width, n)          # a prompt may end in a page that it shares
                cache.fork_lines(b * width, range(b * width + 1, (b + 1) * width), whole_pages=False)
            for line in lines:
                cache.pool.reserve(line, lengths[line // width] + new_tokens)
        except MemoryError:
            for line in lines:
                if line % width:
                    cache.free(line)
                else:
                    cache.truncate(line, lengths[line // width])
            raise
        cache.sync_lines(lines)

    def reorder(self, parents: torch.Tensor, end: Optional[torch.Tensor] = None) -> None:
        """Beam ``w`` of request ``b`` continues its beam ``parents[b, w]``; ``end [B]``: the rows that have been written."""
        if self.cache.pool is not None:
            private = self.cache.pool.private_from(0, len(self.lengths) * self.width)
            shared = [i for i, at in enumerate(private) if at > self.lengths[i // self.width]]
            if shared:
                raise ValueError(f"line {shared[0]} shares pages behind its prompt with another line")
            end = self.limit if end is None else torch.minimum(end, self.limit)          # behind it the table names other lines' pages
        self.cache.reorder_lines(parents, self.start, end)
