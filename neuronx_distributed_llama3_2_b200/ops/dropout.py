"""Dropout from a counter-based generator (``csrc/dropout.cu``): no mask is stored, the backward pass draws it again.

Element ``i`` of the row-major tensor is kept when word ``i % 4`` of Philox4x32-7 (Salmon et al., SC 2011) at counter ``(i // 4,
offset)`` under the key ``seed`` is at least ``p 2^32``, so the mask is the same on every device, in every layout and type, and for
a call that activation checkpointing repeats (one whose seed is a tensor: as long as that holds what it held, see ``dropout``)."""
from __future__ import annotations

import ctypes as _c
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_M32, _M64 = 0xFFFFFFFF, 0xFFFFFFFFFFFFFFFF
Seed = Union[int, torch.Tensor, None]


def philox_words(n: int, seed: int, offset: int = 0, rounds: int = 7, device=None) -> torch.Tensor:
    """The first ``n`` 32-bit words (as int64) of the generator: four to a counter."""
    i = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = i & _M32, i >> 32
    c2, c3 = torch.full_like(i, offset & _M32), torch.full_like(i, offset >> 32 & _M32)
    k0, k1 = seed & _M32, seed >> 32 & _M32
    for _ in range(rounds):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # 64-bit products; the sign bit is a bit like the others
        c0, c1, c2, c3 = (b >> 32 & _M32) ^ c1 ^ k0, b & _M32, (a >> 32 & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = k0 + 0x9E3779B9 & _M32, k1 + 0xBB67AE85 & _M32
    return torch.stack((c0, c1, c2, c3), dim=1).view(-1)[:n]


def dropout_keep(shape, p: float, seed: int, offset: int = 0, device=None) -> torch.Tensor:
    """The keep mask of ``dropout`` for a tensor of that shape."""
    n = 1
    for s in shape:
        n *= int(s)
    return (philox_words(n, seed & _M64, offset & _M64, device=device) >= int(p * 2 ** 32)).view(shape)


def _launch(x, residual, p, seed, offset, state, used):
    y = torch.empty_like(x)
    with _lib.on_device_of(x):
        rc = _lib.lib().nxd_dropout(
            _lib.ptr(x), _lib.ptr(residual), _lib.ptr(y), _c.c_longlong(x.numel()), _c.c_int(_DTYPES[x.dtype]), _c.c_double(p),
            _c.c_ulonglong(seed), _c.c_ulonglong(offset), _lib.ptr(state), _c.c_int(0 if state is None else state.numel()),
            _lib.ptr(used), _lib.stream_ptr())
    _lib.check(rc, "nxd_dropout")
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, state):
        x = x.contiguous()
        used = None
        if state is not None and ctx.needs_input_grad[0]:      # the program may count its state on before the backward pass
            used = torch.empty(2, dtype=torch.int64, device=x.device)
        ctx.args, ctx.used = (p, seed, offset), used
        return _launch(x, residual.contiguous() if residual is not None else None, p, seed, offset, state, used)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, offset = ctx.args
        dx = None
        if ctx.needs_input_grad[0]:
            if ctx.used is not None:
                offset = 0
            dx = _launch(dy.contiguous(), None, p, seed, offset, ctx.used, None)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x: torch.Tensor, p: float = 0.5, seed: Seed = None, offset: int = 0, residual: Optional[torch.Tensor] = None,
            training: bool = True) -> torch.Tensor:
    """``x / (1 - p)`` where the generator keeps an element and 0 elsewhere, plus ``residual`` (of ``x``'s shape and type), rounded once.

    ``seed``: a number (64 bits); or an int64 tensor of one or two on ``x``'s device, the seed and a number that is added to
    ``offset``, read when the kernel runs, so that a captured step which counts it on draws another mask in every replay; or
    ``None``: drawn from torch's CPU generator, which activation checkpointing winds back.  Two calls with the same seed and
    offset drop the same elements: calls of one step take different offsets or seeds.

    The backward pass of a call takes the numbers that the call read, whatever a seed tensor holds by then.  Activation checkpointing
    calls again and reads again, and winds back torch's generators but no tensor of the program: under it a seed tensor is counted on
    behind the backward pass, or the call gets a copy that stays (``state.clone()``, made outside the repeated part)."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} not in [0, 1]")
    if not x.is_floating_point():
        raise ValueError(f"dropout of {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"a residual {tuple(residual.shape)} {residual.dtype} for {tuple(x.shape)} {x.dtype}")
    state = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() not in (1, 2) or seed.device != x.device or not seed.is_contiguous():
            raise ValueError(f"a seed tensor holds one or two int64 on {x.device}")
        state, seed = seed.detach(), 0
    if not training or p == 0.0 or x.numel() == 0:
        return x if residual is None else x + residual
    if p == 1.0:
        y = x.masked_fill(torch.ones((), dtype=torch.bool, device=x.device), 0.0)
        return y if residual is None else y + residual
    if seed is None:
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured dropout would drop the same elements in every replay: pass its seed as a tensor")
        seed = int(torch.randint(0, 2 ** 62, (1,)).item())
    if x.is_cuda and x.dtype in _DTYPES and _lib.available() and not _lib.transformed(x, residual):
        if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad):
            return _DropoutFn.apply(x, residual, p, seed & _M64, offset & _M64, state)
        return _launch(x.contiguous(), residual.contiguous() if residual is not None else None, p, seed & _M64, offset & _M64, state, None)
    if state is not None:
        numbers = state.view(-1).tolist()
        seed, offset = numbers[0], offset + (numbers[1] if len(numbers) > 1 else 0)
    keep = dropout_keep(x.shape, p, seed, offset, x.device)
    wide = x.float() if x.dtype in (torch.bfloat16, torch.float16) else x
    y = torch.where(keep, wide * (1.0 / (1.0 - p)), 0.0)
    return (y if residual is None else y + residual.to(y.dtype)).to(x.dtype)


class Dropout(torch.nn.Module):
    """``torch.nn.Dropout`` on this generator: every training call draws its seed from torch's CPU generator; ``offset`` tells
    apart what ranks with one generator state hold (the tensor-parallel rank where activations are sharded)."""

    _nxd_fx_leaf = True             # one node of a pipeline's graph

    def __init__(self, p: float = 0.5, offset: int = 0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} not in [0, 1]")
        self.p, self.offset = p, offset

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return dropout(x, self.p, None, self.offset, residual, self.training)

    def extra_repr(self) -> str:
        return f"p={self.p}, offset={self.offset}"
