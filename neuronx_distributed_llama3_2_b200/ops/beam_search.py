"""Beam search on the device (``csrc/beam_search.cu``): the candidates of a step, the books of the beams, the sequences at the end.

A search over ``B`` requests with ``W`` beams each is, per step: logits of all beams, ``beam_select`` for the ``2 W`` best continuations of
every request, ``beam_advance`` for the next tokens and the line that each beam continues, ``ops.kv_lines`` for the cache lines that
move; at the end ``beam_finish``.  Nothing of it needs the host.  ``inference.beam_search.BeamSearch`` holds the state of one search."""
from __future__ import annotations

import ctypes as _c
import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

MAX_BEAMS, MAX_CANDIDATES = 32, 64
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_P, _I, _L, _F = _c.c_void_p, _c.c_int, _c.c_longlong, _c.c_float
_ARGS = {
    "nxd_beam_select_scratch": [_I] * 5,
    "nxd_beam_select": [_I, _P, _L, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P],
    "nxd_beam_advance": [_P, _P, _P, _I, _I, _I, _P, _P, _P, _P, _P, _F, _L, _L, _I, _I] + [_P] * 10,
    "nxd_beam_finish_scratch": [_I] * 3,
    "nxd_beam_finish": [_P, _P, _P, _P, _P, _I, _I, _I, _F, _L, _L] + [_P] * 7,
}


def _entry(name: str):
    fn = getattr(_lib.lib(), name)
    if fn.argtypes is None:
        fn.restype = _L if name.endswith("scratch") else _I
        fn.argtypes = _ARGS[name]
    return fn


class BeamPool(NamedTuple):
    """Hypotheses that have ended, the best first; places without one have the score ``-inf`` and length and slot 0."""
    scores: torch.Tensor            # [B, W] fp32: summed log-probability / length ** penalty
    lengths: torch.Tensor           # [B, W] int32: generated tokens, the last of them the one that ends
    slots: torch.Tensor             # [B, W] int32: the line that held it before that token
    done: torch.Tensor              # [B] bool: the request is over


class BeamHistory(NamedTuple):
    """Of every step the token of each line and the line that it continued."""
    tokens: torch.Tensor            # [steps, B, W] int32
    parents: torch.Tensor           # [steps, B, W] int32


def new_beam_pool(B: int, W: int, device=None) -> BeamPool:
    return BeamPool(torch.full((B, W), -float("inf"), dtype=torch.float32, device=device), torch.zeros(B, W, dtype=torch.int32, device=device),
                    torch.zeros(B, W, dtype=torch.int32, device=device), torch.zeros(B, dtype=torch.bool, device=device))


def new_beam_history(steps: int, B: int, W: int, device=None) -> BeamHistory:
    return BeamHistory(*torch.zeros(2, steps, B, W, dtype=torch.int32, device=device).unbind(0))


def _kernel(t: torch.Tensor) -> bool:
    return t.is_cuda and _lib.available()


def _alike(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, like: torch.Tensor) -> None:
    if t.shape != shape or t.dtype is not dtype or t.get_device() != like.get_device() or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor {tuple(shape)} on {like.device} is expected, not {t.dtype} {tuple(t.shape)} on {t.device}"
                         + ("" if t.is_contiguous() else " with strides"))


# ---- the candidates ---------------------------------------------------------------------------------------------------

def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``n`` best continuations of every request: ``scores[b, w] + log_softmax(logits[b, w])[v]`` over beams and tokens, the best first and of
    equal ones the lowest ``w * V + v``.

    ``logits``: ``[B, W, V]`` or ``[B * W, V]``, fp32, bf16 or fp16, unit stride along the tokens; ``scores``: ``[B, W]`` fp32.  Tokens with the logit
    ``-inf`` and beams with the score ``-inf`` are left out, and so is a beam whose logits hold NaN or ``+inf``, or nothing finite; where fewer
    than ``n`` candidates are left the rest have the score ``-inf``, from the lowest ``w * V + v`` on.  Tokens of one beam are compared by their logits,
    those of different beams by their scores in 64 bits, in which a beam's log-sum-exp is good to 2^-20 with up to 2^18 tokens and to 2^-19 with 2^20 (equal
    rows have equal ones).  Returns ``(scores [B, n] fp32, beams [B, n] int64, tokens [B, n] int64)``; not differentiable."""
    shape, sizes = scores.shape, logits.shape
    if len(shape) != 2 or scores.dtype is not torch.float32:
        raise ValueError(f"scores: an fp32 tensor [B, W] is expected, not {scores.dtype} {tuple(shape)}")
    B, W = shape
    if not (len(sizes) == 3 and sizes[0] == B and sizes[1] == W or len(sizes) == 2 and sizes[0] == B * W):
        raise ValueError(f"logits {tuple(sizes)} do not go with scores of {B} x {W} beams")
    if not logits.is_floating_point():
        raise ValueError(f"logits of {logits.dtype} are no floating-point numbers")
    if logits.get_device() != scores.get_device():
        raise ValueError(f"logits on {logits.device}, scores on {scores.device}")
    V, n = sizes[-1], int(n)
    if not 1 <= n <= MAX_CANDIDATES:
        raise ValueError(f"between 1 and {MAX_CANDIDATES} candidates are taken, not {n}")
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams are taken, not {W}")
    if n > W * V:
        raise ValueError(f"{n} candidates are more than {W} beams of {V} tokens have")
    if not _kernel(logits):
        return beam_select_ref(logits, scores, n)
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError(f"logits of {logits.dtype} are not taken on the GPU: fp32, bf16 or fp16")
    strides = logits.stride()
    if (strides[-1] != 1 and V != 1) or len(sizes) == 3 and W > 1 and B > 1 and strides[0] != W * strides[1]:
        logits = logits.contiguous()
        strides = logits.stride()
    if not scores.is_contiguous():
        scores = scores.contiguous()
    tokens = torch.empty((B, n), dtype=torch.int64, device=logits.device)
    beams, best = torch.empty_like(tokens), scores.new_empty((B, n))
    if B:
        with _lib.on_device_of(logits):
            size = _scratch_bytes(code, B, W, V, n)
            if size <= 0:
                raise ValueError(f"{W} beams of {V} tokens are more than one call takes")
            scratch = scores.new_empty((size + 3) // 4)          # the call's own
            rc = _entry("nxd_beam_select")(code, logits.data_ptr(), strides[1] if len(sizes) == 3 and W > 1 else strides[0], scores.data_ptr(), B, W, V, n,
                                           scratch.data_ptr(), best.data_ptr(), beams.data_ptr(), tokens.data_ptr(), _lib.stream_ptr())
        _lib.check(rc, "nxd_beam_select")
    return best, beams, tokens


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(code: int, B: int, W: int, V: int, n: int) -> int:
    return _entry("nxd_beam_select_scratch")(code, B, W, V, n)


def beam_select_ref(logits: torch.Tensor, scores: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The same in torch operations, in 64 bits."""
    (B, W), V = scores.shape, logits.shape[-1]
    x, scores = logits.detach().reshape(B, W, V).double(), scores.detach()
    total = scores.double()[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    total = torch.where(x.isinf() | total.isnan(), -float("inf"), total).reshape(B, W * V)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    return best.float(), at // V, at % V


# ---- the books --------------------------------------------------------------------------------------------------------

def beam_advance(candidates: Tuple[torch.Tensor, torch.Tensor, torch.Tensor], scores: torch.Tensor, pool: BeamPool, history: BeamHistory,
                 step: int, *, eos_token_id: Optional[int] = None, pad_token_id: int = 0, length_penalty: float = 1.0,
                 early_stopping: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, BeamPool]:
    """What ``beam_select``'s candidates of step ``step`` (from 0 on) make of the beams.

    Candidates with the token ``eos_token_id`` end: those among the first ``W`` join the pool with ``score / (step + 1) ** length_penalty``, which keeps
    its best ``W`` (of equal ones the older).  The best ``W`` others are the new beams.  A beam's best continuation stays in its line and the
    others go to the lines that nobody continues, so the fewest cache lines move and none that is read is written.  A request is over once its pool
    is full and, without ``early_stopping``, none of its beams has a better score at its present length than the pool's last; it stays as it
    is from then on, its tokens are ``pad_token_id``.  Where fewer than ``W`` candidates go on (``2 W`` always do) the lines left have the score ``-inf``.

    ``candidates``: scores, beams, tokens ``[B, N]``, the best first; ``scores``: the running ``[B, W]`` (of a request that is over they are handed
    on).  Writes row ``step`` of the history.  Returns ``(scores [B, W], tokens [B, W], parents [B, W], pool)``, by line."""
    cand_scores, cand_beams, cand_tokens = candidates
    if scores.dim() != 2:
        raise ValueError(f"scores: [B, W] is expected, not {tuple(scores.shape)}")
    (B, W), N, dev = scores.shape, cand_scores.shape[-1], scores.device
    if not (1 <= W <= MAX_BEAMS and 1 <= N <= MAX_CANDIDATES):
        raise ValueError(f"{W} beams and {N} candidates: up to {MAX_BEAMS} and {MAX_CANDIDATES} are taken")
    step = int(step)
    if not (history.tokens.dim() == 3 and 0 <= step < history.tokens.shape[0]):
        raise ValueError(f"step {step} is outside a history of {tuple(history.tokens.shape)}")
    _alike("scores", scores, (B, W), torch.float32, scores)
    _check_books(pool, history, B, W, scores)
    for name, t, dtype in (("candidates' scores", cand_scores, torch.float32), ("candidates' beams", cand_beams, torch.int64),
                           ("candidates' tokens", cand_tokens, torch.int64)):
        _alike(name, t, (B, N), dtype, scores)
    eos, pad = _ids(eos_token_id, pad_token_id)
    norm = _norm(step + 1, length_penalty)
    if not _kernel(scores):
        return _advance_ref(cand_scores, cand_beams, cand_tokens, scores, pool, history, step, norm, eos, pad, early_stopping)
    running, tokens, parents = torch.empty_like(scores), cand_tokens.new_empty((B, W)), cand_beams.new_empty((B, W))
    pool_scores, lengths, slots, done = (torch.empty_like(t) for t in pool)
    row = 4 * step * B * W
    with _lib.on_device_of(scores):
        rc = _entry("nxd_beam_advance")(cand_scores.data_ptr(), cand_beams.data_ptr(), cand_tokens.data_ptr(), B, W, N, scores.data_ptr(),
                                        pool.scores.data_ptr(), pool.lengths.data_ptr(), pool.slots.data_ptr(), pool.done.data_ptr(), norm, eos, pad,
                                        int(bool(early_stopping)), step + 1, running.data_ptr(), tokens.data_ptr(), parents.data_ptr(),
                                        pool_scores.data_ptr(), lengths.data_ptr(), slots.data_ptr(), done.data_ptr(),
                                        history.tokens.data_ptr() + row, history.parents.data_ptr() + row, _lib.stream_ptr())
    _lib.check(rc, "nxd_beam_advance")
    return running, tokens, parents, BeamPool(pool_scores, lengths, slots, done)


def _ids(eos_token_id: Optional[int], pad_token_id: int) -> Tuple[int, int]:
    eos, pad = -1 if eos_token_id is None else int(eos_token_id), int(pad_token_id)
    if eos_token_id is not None and not 0 <= eos < 2 ** 31:
        raise ValueError(f"eos_token_id {eos_token_id} is no token")
    if not -2 ** 31 <= pad < 2 ** 31:
        raise ValueError(f"pad_token_id {pad_token_id} does not fit 32 bits")
    return eos, pad


def _norm(length: int, penalty: float) -> float:
    try:
        norm = float(length) ** float(penalty)
    except OverflowError:
        norm = float("inf")
    if not 1e-37 < norm < 3e38:
        raise ValueError(f"a length of {length} to the power of {penalty} is no fp32 number")
    return norm


def _check_books(pool: BeamPool, history: BeamHistory, B: int, W: int, scores: torch.Tensor) -> None:
    _alike("pool.scores", pool.scores, (B, W), torch.float32, scores)
    _alike("pool.lengths", pool.lengths, (B, W), torch.int32, scores)
    _alike("pool.slots", pool.slots, (B, W), torch.int32, scores)
    _alike("pool.done", pool.done, (B,), torch.bool, scores)
    T = history.tokens.shape[0]
    _alike("history.tokens", history.tokens, (T, B, W), torch.int32, scores)
    _alike("history.parents", history.parents, (T, B, W), torch.int32, scores)


def _merged(W: int, *sides):
    """The best ``W`` of the sides' entries ``(scores, others...)``, of equal ones the first; entries of ``-inf`` are zero."""
    scores = torch.cat([s[0] for s in sides], dim=1)
    scores, order = torch.sort(scores, dim=1, descending=True, stable=True)
    scores, order = scores[:, :W], order[:, :W]
    held = scores > -float("inf")
    return (scores.contiguous(), *[torch.cat(x, dim=1).gather(1, order) * held.to(x[0].dtype) for x in zip(*[s[1:] for s in sides])])


def _advance_ref(cand_scores, cand_beams, cand_tokens, scores, pool, history, step, norm, eos, pad, early_stopping):
    """The same in torch operations, request by request."""
    (B, W), N = scores.shape, cand_scores.shape[1]
    running, tokens = torch.full_like(scores, -float("inf")), torch.full((B, W), pad, dtype=torch.int64, device=scores.device)
    parents = torch.arange(W, device=scores.device).repeat(B, 1)
    cs, cb, ct, over = cand_scores.tolist(), cand_beams.tolist(), cand_tokens.tolist(), pool.done.tolist()
    for b in range(B):
        if over[b]:
            running[b] = scores[b]
            continue
        going = [r for r in range(N) if ct[b][r] != eos][:W]
        heirs = {}                         # line -> its best continuation
        for r in going:
            if 0 <= cb[b][r] < W:
                heirs.setdefault(cb[b][r], r)
        free = iter([w for w in range(W) if w not in heirs])
        for r in going:
            line = cb[b][r] if heirs.get(cb[b][r]) == r else next(free)
            running[b, line], tokens[b, line], parents[b, line] = cs[b][r], ct[b][r], cb[b][r]
    first = torch.arange(N, device=scores.device) < W
    ends = (cand_tokens == eos) & first & (cand_scores > -float("inf")) & ~pool.done[:, None]
    ended = torch.where(ends, cand_scores / torch.full_like(cand_scores, norm), -float("inf"))
    new_scores, lengths, slots = _merged(W, (pool.scores, pool.lengths, pool.slots),
                                         (ended, torch.full_like(cand_beams, step + 1).int(), cand_beams.int()))
    was = pool.done[:, None]
    new_scores, lengths, slots = (torch.where(was, a, b) for a, b in ((pool.scores, new_scores), (pool.lengths, lengths), (pool.slots, slots)))
    last = new_scores[:, -1]
    done = pool.done | ((last > -float("inf")) & (torch.full_like(was[:, 0], bool(early_stopping)) | (last >= running.amax(1) / torch.full_like(last, norm))))
    history.tokens[step], history.parents[step] = tokens.int(), parents.int()
    return running, tokens, parents, BeamPool(new_scores.contiguous(), lengths.contiguous(), slots.contiguous(), done)


# ---- the sequences ----------------------------------------------------------------------------------------------------

def beam_finish(scores: torch.Tensor, pool: BeamPool, history: BeamHistory, step: int, *, eos_token_id: Optional[int] = None,
                pad_token_id: int = 0, length_penalty: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The best ``W`` hypotheses of every request after ``step`` steps, the best first: what its pool holds and, where it is not over, its beams with
    ``scores / step ** length_penalty``.  Returns ``(tokens [B, W, step] int64, lengths [B, W] int64, scores [B, W] fp32)``; behind a sequence's
    length are ``pad_token_id``, a place without a hypothesis has the length 0 and the score ``-inf``."""
    if scores.dim() != 2:
        raise ValueError(f"scores: [B, W] is expected, not {tuple(scores.shape)}")
    (B, W), dev, step = scores.shape, scores.device, int(step)
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams are taken, not {W}")
    if not (history.tokens.dim() == 3 and 1 <= step <= history.tokens.shape[0]):
        raise ValueError(f"{step} steps are outside a history of {tuple(history.tokens.shape)}")
    _alike("scores", scores, (B, W), torch.float32, scores)
    _check_books(pool, history, B, W, scores)
    eos, pad = _ids(eos_token_id, pad_token_id)
    norm = _norm(step, length_penalty)
    if not _kernel(scores):
        return _finish_ref(scores, pool, history, step, norm, eos, pad)
    if B > 65535:
        raise ValueError(f"{B} requests are more than 65535")
    tokens = torch.empty((B, W, step), dtype=torch.int64, device=dev)
    lengths = tokens.new_empty((B, W))
    best = torch.empty_like(scores)
    with _lib.on_device_of(scores):
        scratch = None
        if W * step > 2 ** 16:          # lines of many steps do not fit shared memory
            scratch = torch.empty(_entry("nxd_beam_finish_scratch")(B, W, step), dtype=torch.uint8, device=dev)
        rc = _entry("nxd_beam_finish")(scores.data_ptr(), pool.scores.data_ptr(), pool.lengths.data_ptr(), pool.slots.data_ptr(),
                                       pool.done.data_ptr(), B, W, step, norm, eos, pad, history.tokens.data_ptr(), history.parents.data_ptr(),
                                       tokens.data_ptr(), lengths.data_ptr(), best.data_ptr(), 0 if scratch is None else scratch.data_ptr(), _lib.stream_ptr())
    _lib.check(rc, "nxd_beam_finish")
    return tokens, lengths, best


def _finish_ref(scores, pool, history, step, norm, eos, pad):
    """The same in torch operations."""
    B, W = scores.shape
    own = torch.where(pool.done[:, None] | scores.isnan(), -float("inf"), scores / torch.full_like(scores, norm))
    best, lengths, slots, ended = _merged(
        W, (pool.scores, pool.lengths.long().clamp(0, step), pool.slots.long().clamp(0, W - 1), torch.ones_like(pool.lengths)),
        (own, torch.full((B, W), step, device=scores.device), torch.arange(W, device=scores.device).repeat(B, 1), torch.zeros_like(pool.lengths)))
    tokens = torch.full((B, W, step), pad, dtype=torch.int64, device=scores.device)
    line = slots
    for t in range(step - 1, -1, -1):
        inside = lengths - ended > t          # the token that ends is in no history
        tokens[:, :, t] = torch.where(inside, history.tokens[t].long().gather(1, line), tokens[:, :, t])
        line = torch.where(inside, history.parents[t].long().clamp(0, W - 1).gather(1, line), line)
    tokens.scatter_(2, (lengths - 1).clamp(min=0)[..., None], torch.where((ended > 0) & (lengths > 0), eos, tokens.gather(
        2, (lengths - 1).clamp(min=0)[..., None])[..., 0])[..., None])
    return tokens, lengths, best
