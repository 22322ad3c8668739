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


def _where(mask: Optional[torch.Tensor], rows: Sequence[torch.Tensor]) -> list:
    """What the table says of its tensors but their sizes."""
    return [mask is not None and mask.data_ptr(), *[t.data_ptr() for t in rows], *[t.stride(0) for t in rows]]


# what moves saved tensors: the innermost pair of hooks, None without one
_saved_hooks = getattr(torch._C._autograd, "_top_saved_tensors_default_hooks", lambda _: "unknown")


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
        # Without hooks the program's own tensors are saved as they are, so that ``logits.data = ...`` gives them other storage: what is
        # saved is another tensor on the storage of this call (the gradient wants its values), and its writes are counted with theirs.  The
        # tensors themselves are for a gradient that is differentiated.
        where = None
        if _saved_hooks(True) is None:
            where = _where(mask, rows)
            ctx.save_for_backward(share, mask, *[r.detach() if r is t else r for r, t in zip(rows, logits)], *logits)
        else:
            ctx.save_for_backward(share, mask, *logits)
        ctx.args = (table, where, E, top_k, sizes, [None if r is t else t.shape for r, t in zip(rows, logits)])
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * len(ctx.needs_input_grad)
        saved = ctx.saved_tensors          # all of them: none may have been written since
        table, where, E, top_k, sizes, shapes = ctx.args
        n = len(sizes)
        share, mask, rows = saved[0], saved[1], saved[2:2 + n]
        if torch.is_grad_enabled():        # this gradient is differentiated itself: in torch operations, on the program's own tensors
            logits, need = saved[-n:], ctx.needs_input_grad[3:]
            loss, _ = balance_loss_ref(list(logits), E, top_k, mask)
            grads = iter(torch.autograd.grad(loss, [t for t, x in zip(logits, need) if x], grad.to(loss.dtype), create_graph=True))
            return (None, None, None, *[next(grads) if x else None for x in need])
        if where is None or _where(mask, rows) != where:    # checkpointing, offloading; the table of 32 layers costs a tenth of the call
            rows = [_rows(t, E) for t in rows]
            if [tuple(t.shape) for t in rows] != [(n, E) for n in sizes]:
                raise RuntimeError(f"router logits saved for the balance loss have become {[tuple(t.shape) for t in rows]}")
            table = _table(rows, mask, E, top_k)
        x = rows[0]
        dx = torch.empty((sum(sizes), x.shape[1]), dtype=x.dtype, device=x.device)
        grad = grad.float()
        with _lib.on_device_of(x):
            rc = _lib.lib().nxd_balance_loss_bwd(*table, _lib.ptr(share), _lib.ptr(grad), _lib.ptr(dx), _lib.stream_ptr())
        _lib.check(rc, "nxd_balance_loss_bwd")
        grads = dx.split(sizes)
        if any(s is not None for s in shapes):
            grads = [g if s is None else g.view(s) for g, s in zip(grads, shapes)]
        if not all(ctx.needs_input_grad[3:]):
            grads = [g if need else None for g, need in zip(grads, ctx.needs_input_grad[3:])]
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
