"""Binding + autograd node of the load-balancing loss (``csrc/balance_loss.cu``): all layers' router logits where they are, one pass
forward (and a small one that adds up), one backward.  ``modules.moe.load_balancing_loss_func`` is the public function."""
from __future__ import annotations

import ctypes as _c
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_LAYERS, MAX_EXPERTS = 128, 1024


def _rows(t: torch.Tensor, E: int) -> torch.Tensor:
    """``[rows, E]`` with unit stride along the experts."""
    t = t.reshape(-1, E)
    return t if E == 1 or t.stride(1) == 1 else t.contiguous()


def qualifies(logits: List[torch.Tensor], E: int) -> bool:
    x = logits[0]
    return (x.is_cuda and x.dtype in _DTYPES and len(logits) <= MAX_LAYERS and E <= MAX_EXPERTS
            and all(t.dtype == x.dtype and t.device == x.device for t in logits) and _lib.available())


def _table(rows: List[torch.Tensor]):
    n = len(rows)
    return ((_c.c_void_p * n)(*[t.data_ptr() for t in rows]), (_c.c_longlong * n)(*[t.stride(0) for t in rows]),
            (_c.c_longlong * n)(*[t.shape[0] for t in rows]), _c.c_int(n), _c.c_int(_DTYPES[rows[0].dtype]))


class _BalanceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, E, top_k, mask, *logits):
        rows = [_rows(t, E) for t in logits]
        dev = rows[0].device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty(E, dtype=torch.int64, device=dev)
        lib = _lib.lib()
        blocks = lib.nxd_balance_loss_num_blocks(_c.c_longlong(max(t.shape[0] for t in rows)), _c.c_int(len(rows)), _c.c_int(E))
        share = torch.empty(E + 2 * blocks * E, dtype=torch.float32, device=dev)          # the shares, then the call's scratch
        with torch.cuda.device(dev):
            rc = lib.nxd_balance_loss_fwd(*_table(rows), _lib.ptr(mask), _c.c_int(E), _c.c_int(top_k), _lib.ptr(loss), _lib.ptr(counts),
                                          _lib.ptr(share), _c.c_void_p(share.data_ptr() + 4 * E), _lib.stream_ptr())
        _lib.check(rc, "nxd_balance_loss_fwd")
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(share, mask, *rows)
        ctx.args = (E, top_k, [t.shape for t in logits])
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        share, mask, *rows = ctx.saved_tensors
        E, top_k, shapes = ctx.args
        sizes = [t.shape[0] for t in rows]
        dx = torch.empty((sum(sizes), E), dtype=rows[0].dtype, device=rows[0].device)
        grad = grad.float()
        with torch.cuda.device(dx.device):
            rc = _lib.lib().nxd_balance_loss_bwd(*_table(rows), _lib.ptr(mask), _c.c_int(E), _c.c_int(top_k), _lib.ptr(share),
                                                 _lib.ptr(grad), _lib.ptr(dx), _lib.stream_ptr())
        _lib.check(rc, "nxd_balance_loss_bwd")
        grads = [g.view(s) if need else None for g, s, need in zip(dx.split(sizes), shapes, ctx.needs_input_grad[3:])]
        return (None, None, None, *grads)


def balance_loss(logits: List[torch.Tensor], E: int, top_k: int, mask: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` of tensors that ``qualifies`` takes; ``mask``: bool, one per row of a tensor."""
    return _BalanceLossFn.apply(E, top_k, mask, *logits)


def balance_loss_ref(logits: List[torch.Tensor], E: int, top_k: int, mask: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The same in torch operations."""
    x = torch.cat([t.reshape(-1, E) for t in logits]).float() if len(logits) > 1 else logits[0].reshape(-1, E).float()
    probs = torch.softmax(x, dim=-1)
    # the largest logits, ties to the lowest expert (a top-k leaves open which of two equal ones it takes)
    selected = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k]
    if mask is None:
        n = torch.full((), float(x.shape[0]), device=x.device)
        ones = torch.ones(selected.shape, dtype=torch.int64, device=x.device)
    else:
        rows = mask.repeat(len(logits))
        n = rows.sum().float()
        ones = rows[:, None].expand_as(selected).long()
        probs = torch.where(rows[:, None], probs, 0.0)
    counts = torch.zeros(E, dtype=torch.int64, device=x.device).scatter_add_(0, selected.reshape(-1), ones.reshape(-1))
    n = n.clamp(min=1.0)
    loss = (counts.float() / n * (probs.sum(0) / n)).sum() * (E / top_k)
    return loss, counts
