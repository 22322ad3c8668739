"""Attention over packed sequences: the samples of a batch laid end to end in one row instead of padded to the longest.

``PackedSequences`` holds where the sequences of a step begin and the tile list that the kernels walk (``csrc/packed_plan.cu``);
it is made on the device from ``cu_seqlens`` without a copy to the host and serves every layer of the step, forward and
backward.  The kernels are ``csrc/packed_attention.cu`` and ``csrc/packed_attention_bwd.cu``.  ``ops.attention`` has the public
functions."""
from __future__ import annotations

import ctypes as _c
import math
from typing import List, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rope import _aligned as _rope_aligned, _launch as _rope_launch


class PackedSequences:
    """The sequences of a packed row of ``total`` tokens: sequence ``s`` takes rows ``cu_seqlens[s] .. cu_seqlens[s + 1]``.

    ``cu_seqlens [N + 1]``: int32 or int64, rising (equal neighbours are an empty sequence), inside ``[0, total]``; rows ahead of the
    first boundary or behind the last belong to no sequence, attend to nothing and give zeros.  On the CPU this is checked; on
    the GPU, where a check would wait for the device, a boundary that falls or leaves the row is taken as the nearest one
    that does not.  What is made of the boundaries (tile lists, positions) is made once for every stream, and once inside every
    captured graph, which reads ``cu_seqlens`` again in each replay; elsewhere lengths that change want a new object.  The object
    holds what it made for each stream and for the last capture there: what earlier captures made is their graphs' alone."""

    def __init__(self, cu_seqlens: torch.Tensor, total: int):
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"cu_seqlens: N + 1 boundaries as int32 or int64, not {tuple(cu_seqlens.shape)} {cu_seqlens.dtype}")
        if not 0 < total < 2 ** 31 - 256:
            raise ValueError(f"a packed row of {total} tokens")
        self.cu_seqlens, self.total, self.count = cu_seqlens.contiguous(), int(total), cu_seqlens.numel() - 1
        self._plans: dict = {}
        self._positions: dict = {}
        if not cu_seqlens.is_cuda:
            ends = cu_seqlens.tolist()
            if any(b < a for a, b in zip(ends, ends[1:])) or ends[0] < 0 or ends[-1] > total:
                raise ValueError(f"cu_seqlens have to rise inside [0, {total}]: {ends[:8]} ...")

    @property
    def device(self) -> torch.device:
        return self.cu_seqlens.device

    def _here(self) -> Tuple[int, int]:
        """The current stream, and which capture goes on there: another one's lists may be unwritten still, or gone with its graph."""
        if not self.cu_seqlens.is_cuda:
            return 0, 0
        stream = torch._C._cuda_getCurrentRawStream(self.cu_seqlens.get_device())
        if not _lib.available():
            return stream, 0
        capture_id = _lib.lib().nxd_capture_id
        capture_id.restype = _c.c_ulonglong
        return stream, capture_id(_c.c_void_p(stream))

    def plan(self, causal: bool, rows: int = 128) -> Tuple[torch.Tensor, int, int]:
        """``(list of tiles of that many rows, its entries, columns of the per-row scratch)`` for the kernels, made on first use."""
        stream, capture = self._here()
        key = (causal, rows, stream, capture != 0)
        if key not in self._plans or self._plans[key][0] != capture:
            most = min(self.count, self.total)
            entries = self.total // rows + most + 2                         # nxd_packed_plan_entries
            columns = (self.total + 3 * most + 3 & ~3) + 64                 # nxd_packed_plan_columns
            lists = torch.empty((entries + self.count + (entries + 3) // 4, 4), dtype=torch.int32, device=self.device)
            rc = _lib.lib().nxd_packed_plan(_lib.ptr(self.cu_seqlens), _c.c_int(self.cu_seqlens.dtype == torch.int64), _c.c_int(self.count),
                                            _c.c_longlong(self.total), _c.c_int(causal), _c.c_int(rows), _lib.ptr(lists),
                                            _c.c_void_p(lists.data_ptr() + 16 * entries), _which(lists, entries, self.count), _lib.stream_ptr())
            _lib.check(rc, "nxd_packed_plan")
            self._plans[key] = (capture, (lists, entries, columns))
        return self._plans[key][1]

    def positions(self) -> torch.Tensor:
        """int32 ``[total]``: every token's position in its own sequence (0 outside of them), for the rotation."""
        stream, capture = self._here()
        key = (stream, capture != 0)
        if key not in self._positions or self._positions[key][0] != capture:
            cu = self.cu_seqlens.long().clamp(0, self.total).cummax(0).values
            rows = torch.arange(self.total, device=self.device)
            s = torch.searchsorted(cu, rows, right=True) - 1
            inside = (s >= 0) & (s < self.count)
            pos = torch.where(inside, rows - cu[s.clamp(0, self.count)], 0)
            self._positions[key] = (capture, pos.to(torch.int32))
        return self._positions[key][1]

    def first_tokens(self) -> torch.Tensor:
        """int64 ``[N]``: the row of every sequence's first token."""
        return self.cu_seqlens[:-1].long().clamp(0, self.total - 1).cummax(0).values

    def last_tokens(self) -> torch.Tensor:
        """bool ``[total]``: the last token of a sequence (it has no next token to predict), and every row outside of them."""
        cu = self.cu_seqlens.long().clamp(0, self.total).cummax(0).values
        mask = torch.zeros(self.total + 1, dtype=torch.bool, device=self.device)
        mask[cu] = True
        return mask[1:] | ~self.inside()

    def inside(self) -> torch.Tensor:
        """bool ``[total]``: the tokens that belong to a sequence."""
        rows = torch.arange(self.total, device=self.device)
        cu = self.cu_seqlens
        return (rows >= cu[0]) & (rows < cu.max())

    def slices(self) -> List[slice]:
        """The sequences' rows, on the host (waits for the device)."""
        ends = self.cu_seqlens.long().clamp(0, self.total).cummax(0).values.tolist()
        return [slice(a, b) for a, b in zip(ends, ends[1:])]


def as_packed(sequences: Union[torch.Tensor, PackedSequences], total: int, device: torch.device) -> PackedSequences:
    packed = sequences if isinstance(sequences, PackedSequences) else PackedSequences(sequences, total)
    if packed.total != total:
        raise ValueError(f"sequences packed in {packed.total} rows, tensors of {total}")
    if packed.device != device:
        raise ValueError(f"cu_seqlens on {packed.device}, tensors on {device}")
    return packed


def _fix(t: torch.Tensor) -> torch.Tensor:
    """Unit stride on the head dimension, the others multiples of 8 elements that do not overlap, 16-byte aligned."""
    T, H, D = t.shape
    row, head, unit = t.stride()
    if unit == 1 and t.data_ptr() % 16 == 0 and (H == 1 or head % 8 == 0 and head >= D) and (T == 1 or row % 8 == 0 and row >= D):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(*ts: torch.Tensor):
    """(head, row) strides; a dimension of one has any."""
    vals = []
    for t in ts:
        T, H, D = t.shape
        row, head, _ = t.stride()
        vals += (head if H > 1 else D, row if T > 1 else H * D)
    return (_c.c_longlong * len(vals))(*vals)


def gave_up() -> bool:
    """Whether a call of packed attention gave up waiting inside its kernel since the last one that failed for it or was asked: its results
    are NaN.  Waits for the current stream."""
    flag = _c.c_int(0)
    _lib.check(_lib.lib().nxd_packed_attn_status(_c.byref(flag), _lib.stream_ptr()), "nxd_packed_attn_status")
    return bool(flag.value)


def _which(lists: torch.Tensor, entries: int, count: int) -> _c.c_void_p:
    """Where a plan's list has the sequences' numbers of its tiles: behind the tiles and the sequences."""
    return _c.c_void_p(lists.data_ptr() + 16 * (entries + count))


def _rest_of(rest: Optional[torch.Tensor], lists: torch.Tensor, entries: int, columns: int, count: int) -> tuple:
    """Of what the rounding took from the result: the sequences' numbers if it has 128 rows for each (``None``: one row a column), rows."""
    if rest is None or rest.shape[1] == columns:
        return None, _c.c_longlong(columns)
    return _which(lists, entries, count), _c.c_longlong(rest.shape[1])


def _forward(q, k, v, packed: PackedSequences, scale: float, causal: bool, grad: bool, wait_tries: int = -1):
    """``(o, lse, rest)``; the two that the backward pass takes are ``None`` without it.  ``wait_tries``: of a wait inside the kernel, -1: two
    seconds (``gave_up``; the next call raises)."""
    T, Hq, D = q.shape
    # an odd number of heads to a key head: two neighbouring tiles of one head are worked on together (csrc/packed_attention.cu)
    tiles, entries, columns = packed.plan(causal, 128 if Hq // k.shape[1] % 2 == 0 else 256)
    o = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((Hq, columns), dtype=torch.float32, device=q.device) if grad else None
    rest = torch.empty((Hq, min(columns, 128 * max(1, packed.count)), D), dtype=torch.uint8, device=q.device) if grad else None
    rc = _lib.lib().nxd_packed_attn_fwd(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(o), _lib.ptr(lse), _lib.ptr(rest), _strides(q, k, v, o), _lib.ptr(tiles),
        *_rest_of(rest, tiles, entries, columns, packed.count), _c.c_int(entries),
        _c.c_longlong(columns), _c.c_longlong(T), _c.c_int(Hq), _c.c_int(k.shape[1]), _c.c_int(D), _c.c_float(scale), _c.c_int(causal),
        _c.c_int(wait_tries), _lib.stream_ptr())
    _lib.check(rc, "nxd_packed_attn_fwd")
    return o, lse, rest


def _backward(q, k, v, o, lse, rest, do, dq, dk, dv, plan, count: int, scale: float, causal: bool, wait_tries: int = -1) -> None:
    """Every element of ``dq / dk / dv`` is written.  ``plan``: the list that the forward pass had, or one made with it."""
    q, k, v, o, do = (_fix(t) for t in (q, k, v, o, do))          # what was saved may have been moved
    T, Hq, D = o.shape
    Hkv = k.shape[1]
    tiles, entries, columns = plan
    if (q.shape != o.shape or do.shape != o.shape or k.shape != (T, Hkv, D) or v.shape != k.shape or not Hkv or Hq % Hkv
            or any(x.dtype != o.dtype or x.device != o.device for x in (q, k, v, do))):          # ``q.data = ...`` since
        raise RuntimeError(f"packed attention saved q, k and v for a result {tuple(o.shape)} {o.dtype} on {o.device}; they have become "
                           + ", ".join(f"{tuple(x.shape)} {x.dtype} on {x.device}" for x in (q, k, v)))
    delta = torch.empty(lse.numel() + 4, dtype=torch.float32, device=q.device)
    acc = torch.empty((Hq, D, columns), dtype=torch.float32, device=q.device)
    splits = _lib.lib().nxd_packed_attn_bwd_splits(_c.c_longlong(T), _c.c_int(count), _c.c_int(Hq), _c.c_int(Hkv))
    kv_acc = torch.zeros((2, Hkv, T, D), dtype=torch.float32, device=q.device) if splits > 1 else None
    rc = _lib.lib().nxd_packed_attn_bwd(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(o), _lib.ptr(rest), _lib.ptr(do), _lib.ptr(lse), _lib.ptr(delta), _lib.ptr(acc), _lib.ptr(kv_acc),
        _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _strides(q, k, v, o, do, dq, dk, dv), _lib.ptr(tiles),
        *_rest_of(rest, tiles, entries, columns, count), _c.c_int(entries),
        _c.c_longlong(columns), _c.c_longlong(T), _c.c_int(count), _c.c_int(Hq), _c.c_int(Hkv), _c.c_int(D), _c.c_float(scale),
        _c.c_int(causal), _c.c_int(wait_tries), _lib.stream_ptr())
    _lib.check(rc, "nxd_packed_attn_bwd")


class _PackedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packed, scale, causal):
        q, k, v = _fix(q), _fix(k), _fix(v)
        grad = any(ctx.needs_input_grad[:3])
        with _lib.on_device_of(q):
            o, lse, rest = _forward(q, k, v, packed, scale, causal, grad)
            if grad:
                ctx.save_for_backward(q, k, v, o, lse, rest)
                ctx.args = (packed.plan(causal), packed.count, scale, causal)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, rest = ctx.saved_tensors
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        with _lib.on_device_of(q):
            _backward(q, k, v, o, lse, rest, do, dq, dk, dv, *ctx.args)
        return dq, dk, dv, None, None, None


class _RopePackedAttnFn(torch.autograd.Function):
    """Rotation (positions that start again with every sequence) and causal attention of one projection output as one node: the
    three gradients are written side by side into one buffer and rotated back there, as in ``flash_attn.rope_flash_attn``."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, n_q, n_kv, packed, scale):
        T, heads, D = qkv.shape
        with _lib.on_device_of(qkv):
            qkv = _rope_aligned(qkv)
            rot = torch.empty_like(qkv)
            positions = packed.positions()
            if cos.shape[0] < packed.total:          # the bound keeps a sequence that is too long for the tables from reading behind them
                positions = positions.clamp(max=cos.shape[0] - 1)
            _rope_launch(qkv, cos, sin, n_q + n_kv, 1, 1 << 30, positions, False, rot)
            o, lse, rest = _forward(rot[:, :n_q], rot[:, n_q:n_q + n_kv], rot[:, n_q + n_kv:], packed, scale, True, ctx.needs_input_grad[0])
            if ctx.needs_input_grad[0]:
                ctx.save_for_backward(rot, o, lse, rest, cos, sin, positions)
                ctx.args = (n_q, n_kv, packed.plan(True), packed.count, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        rot, o, lse, rest, cos, sin, positions = ctx.saved_tensors
        n_q, n_kv, plan, count, scale = ctx.args
        parts = lambda x: (x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:])     # noqa: E731
        with _lib.on_device_of(rot):
            d = torch.empty_like(rot)
            _backward(*parts(rot), o, lse, rest, do, *parts(d), plan, count, scale, True)
            _rope_launch(d, cos, sin, n_q + n_kv, 1, 1 << 30, positions, True)
        return d, None, None, None, None, None, None


def packed_attn_nxd(q, k, v, packed: PackedSequences, softmax_scale: Optional[float], causal: bool) -> torch.Tensor:
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if scale <= 0.0:                # the kernels keep the maximum of the raw scores, which wants a positive scale
        q, scale = (-q, -scale) if scale < 0.0 else (q * 0.0, 1.0)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if not grad and not _lib.transformed(q, k, v):          # forward-mode derivatives and ``torch.func`` are refused by the node
        with _lib.on_device_of(q):
            return _forward(_fix(q), _fix(k), _fix(v), packed, scale, bool(causal), False)[0]
    return _PackedAttnFn.apply(q, k, v, packed, scale, bool(causal))


def rope_packed_attn(qkv, cos, sin, n_q: int, n_kv: int, packed: PackedSequences) -> torch.Tensor:
    return _RopePackedAttnFn.apply(qkv, cos, sin, n_q, n_kv, packed, 1.0 / math.sqrt(qkv.shape[-1]))
