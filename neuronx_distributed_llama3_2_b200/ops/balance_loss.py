"""Binding + autograd node of the load-balancing loss (``csrc/balance_loss.cu``): all layers' router logits where they are, one pass
forward (and a small one that adds up), one backward.  ``modules.moe.load_balancing_loss_func`` is the public function."""
from __future__ import annotations

import ctypes as _c
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_LAYERS, MAX_EXPERTS = 128, 1024


def _rows(t: torch.Tensor, E: int) -> torch.Tensor:
    """``[rows, E]`` with unit stride along the experts."""
    if t.dim() != 2 or t.shape[1] != E:
        t = t.reshape(-1, E)
    return t if t.stride(1) == 1 or E == 1 else t.contiguous()


def qualifies(logits: List[torch.Tensor], E: int) -> bool:
    x = logits[0]
    dtype, device = x.dtype, x.get_device()
    return (x.is_cuda and dtype in _DTYPES and len(logits) <= MAX_LAYERS and E <= MAX_EXPERTS
            and all(t.dtype is dtype and t.get_device() == device for t in logits) and _lib.available()
            and not _lib.transformed(*logits))          # forward-mode derivatives and ``torch.func`` take the torch form


def _table(rows: Sequence[torch.Tensor], mask: Optional[torch.Tensor], E: int, top_k: int) -> tuple:
    """The entry points' first arguments: pointers, row strides and rows of the layers, and what they share."""
    n = len(rows)
    return ((_c.c_void_p * n)(*[t.data_ptr() for t in rows]), (_c.c_longlong * n)(*[t.stride(0) for t in rows]),
            (_c.c_longlong * n)(*[t.shape[0] for t in rows]), _c.c_int(n), _c.c_int(_DTYPES[rows[0].dtype]), _lib.ptr(mask), _c.c_int(E),
            _c.c_int(top_k))


# what moves saved tensors: the innermost pair of hooks, None without one; whether the backward pass that goes on leaves the graph for another
_saved_hooks = getattr(torch._C._autograd, "_top_saved_tensors_default_hooks", lambda _: "unknown")
_keeps_graph = getattr(torch._C._autograd, "_get_current_graph_task_keep_graph", lambda: True)


class _Kept:
    """A call's table of addresses with the storages that it points into: ``logits.data = ...`` behind the loss, or hooks on what the node
    saved, give the saved tensors other storage, while the gradient wants the values that the loss saw."""

    def __init__(self, table: tuple, tensors: Sequence[torch.Tensor]):
        self.table, self.storages = table, [t.untyped_storage() for t in tensors]
        self.at = [s.data_ptr() for s in self.storages]

    def valid(self) -> bool:          # a storage can be resized
        return [s.data_ptr() for s in self.storages] == self.at


class _BalanceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, E, top_k, mask, *logits):
        rows = [_rows(t, E) for t in logits]
        sizes = [t.shape[0] for t in rows]
        n, x, lib = len(rows), rows[0], _lib.lib()
        loss = torch.empty((), dtype=torch.float32, device=x.device)
        counts = torch.empty(E, dtype=torch.int64, device=x.device)
        table = _table(rows, mask, E, top_k)
        with _lib.on_device_of(x):
            blocks = lib.nxd_balance_loss_num_blocks(_c.c_longlong(max(sizes)), _c.c_int(n), _c.c_int(E))
            share = torch.empty(E + 2 * blocks * E, dtype=torch.float32, device=x.device)     # the shares, then the call's scratch
            rc = lib.nxd_balance_loss_fwd(*table, _lib.ptr(loss), _lib.ptr(counts), _lib.ptr(share),
                                          _c.c_void_p(share.data_ptr() + 4 * E), _lib.stream_ptr())
        _lib.check(rc, "nxd_balance_loss_fwd")
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)         # no zeros for the counts' gradient
        ctx.save_for_backward(share, mask, *logits)
        # hooks (checkpointing, offloading) are there to let the memory go; what they give back is read where it lies
        ctx.kept = None if _saved_hooks(True) is not None else _Kept(table, rows if mask is None else [*rows, mask])
        ctx.args = (E, top_k, x.dtype, sizes, [None if r is t else t.shape for r, t in zip(rows, logits)])
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * len(ctx.needs_input_grad)
        saved = ctx.saved_tensors          # all of them: none may have been written since
        E, top_k, dtype, sizes, shapes = ctx.args
        share, mask, logits = saved[0], saved[1], saved[2:]
        kept, need = ctx.kept, ctx.needs_input_grad[3:]
        if not _keeps_graph():             # like what is saved, these go with the last pass
            ctx.kept = None
        if torch.is_grad_enabled():        # this gradient is differentiated itself: in torch operations, on the program's own tensors
            loss, _ = balance_loss_ref(list(logits), E, top_k, mask)
            grads = iter(torch.autograd.grad(loss, [t for t, x in zip(logits, need) if x], grad.to(loss.dtype), create_graph=True))
            return (None, None, None, *[next(grads) if x else None for x in need])
        if kept is not None and kept.valid():          # the table of 32 layers costs a tenth of the call
            table = kept.table
        else:
            rows = [_rows(t, E) for t in logits]
            if [(*t.shape, t.dtype, t.device) for t in rows] != [(n, E, dtype, share.device) for n in sizes]:
                raise RuntimeError(f"router logits saved for the balance loss have become {[(*t.shape, t.dtype, t.device) for t in rows]}")
            table = _table(rows, mask, E, top_k)
        dx = torch.empty((sum(sizes), E), dtype=dtype, device=share.device)
        grad = grad.float()
        with _lib.on_device_of(share):
            rc = _lib.lib().nxd_balance_loss_bwd(*table, _lib.ptr(share), _lib.ptr(grad), _lib.ptr(dx), _lib.stream_ptr())
        _lib.check(rc, "nxd_balance_loss_bwd")
        grads = dx.split(sizes)
        if any(s is not None for s in shapes):
            grads = [g if s is None else g.view(s) for g, s in zip(grads, shapes)]
        if not all(need):
            grads = [g if x else None for g, x in zip(grads, need)]
        return (None, None, None, *grads)


def balance_loss(logits: List[torch.Tensor], E: int, top_k: int, mask: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` of tensors that ``qualifies`` takes; ``mask``: bool, one per row of a tensor."""
    return _BalanceLossFn.apply(E, top_k, mask, *logits)


def balance_loss_ref(logits: List[torch.Tensor], E: int, top_k: int, mask: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The same in torch operations."""
    x = torch.cat([t.reshape(-1, E) for t in logits]).float() if len(logits) > 1 else logits[0].reshape(-1, E).float()
    rows = mask.repeat(len(logits)) if mask is not None else None
    if rows is not None:          # ahead of the softmax, whose gradient turns a zero into NaN where the row holds one
        x = torch.where(rows[:, None], x, 0.0)
    probs = torch.softmax(x, dim=-1)
    # the largest logits, ties to the lowest expert (a top-k leaves open which of two equal ones it takes)
    selected = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k]
    if rows is None:
        n = torch.full((), float(x.shape[0]), device=x.device)
        ones = torch.ones(selected.shape, dtype=torch.int64, device=x.device)
    else:
        n = rows.sum().float()
        ones = rows[:, None].expand_as(selected).long()
        probs = torch.where(rows[:, None], probs, 0.0)
    counts = torch.zeros(E, dtype=torch.int64, device=x.device).scatter_add_(0, selected.reshape(-1), ones.reshape(-1))
    n = n.clamp(min=1.0)
    loss = (counts.float() / n * (probs.sum(0) / n)).sum() * (E / top_k)
    return loss, counts
