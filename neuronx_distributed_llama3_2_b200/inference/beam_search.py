"""Beam search over the KV cache: the state of one search, and the loop that generates with it.

Per step: the logits of all beams, the ``2 W`` best continuations of every request (``ops.beam_search.beam_select``), the books
(``beam_advance``), and the cache lines that continue another line (``KVCache.beams`` / ``BeamLines.reorder``).  None of it waits for the device; every
``CHECK_EVERY`` steps the loop asks whether all requests are over (steps of a request that is over change nothing)."""
from __future__ import annotations

from typing import Callable, List, Optional, Tuple

import torch

from ..ops.beam_search import beam_advance, beam_finish, beam_select, new_beam_history, new_beam_pool
from .kv_cache import KVCache

CHECK_EVERY = 8


class BeamSearch:
    """``groups`` requests with ``width`` beams each, for up to ``max_new_tokens`` tokens.

    A continuation by ``eos_token_id`` among the best ``width`` ends a hypothesis, whose score is its summed log-probability divided by its
    length (generated tokens, the last one included) to the power of ``length_penalty``; a request keeps its best ``width`` hypotheses, and is over
    once it has so many and no beam could enter at its present length (``early_stopping``: once it has so many)."""

    def __init__(self, groups: int, width: int, max_new_tokens: int, *, eos_token_id: Optional[int] = None, pad_token_id: int = 0,
                 length_penalty: float = 1.0, early_stopping: bool = False, device=None):
        if not 1 <= width <= 32 or groups < 1 or max_new_tokens < 1:
            raise ValueError(f"{groups} requests, {width} beams (1 to 32), {max_new_tokens} tokens")
        self.groups, self.width, self.max_new_tokens, self.step = groups, width, max_new_tokens, 0
        self.early_stopping = bool(early_stopping)
        self._kw = dict(eos_token_id=eos_token_id, pad_token_id=pad_token_id, length_penalty=length_penalty)
        self.scores = torch.zeros(groups, 1, dtype=torch.float32, device=device)          # one beam before the first step
        self.pool = new_beam_pool(groups, width, device)
        self.history = new_beam_history(max_new_tokens, groups, width, device)

    def advance(self, logits: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``logits``: of the prompts' last tokens ``[groups, V]`` at first, then of every beam ``[groups * width, V]``.  Returns the beams' next
        tokens and the beams that they continue, ``[groups, width]`` each."""
        if self.step >= self.max_new_tokens:
            raise ValueError(f"the search has taken its {self.max_new_tokens} steps")
        B, W = self.groups, self.width
        have = self.scores.shape[1]
        found = beam_select(logits, self.scores, min(2 * W, have * logits.shape[-1]))
        running = self.scores if have == W else self.scores.expand(B, W).contiguous()
        self.scores, tokens, parents, self.pool = beam_advance(found, running, self.pool, self.history, self.step,
                                                               early_stopping=self.early_stopping, **self._kw)
        self.step += 1
        return tokens, parents

    def finished(self) -> bool:
        """Whether every request is over (waits for the device)."""
        return bool(self.pool.done.all())

    def finish(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(tokens [groups, width, steps], lengths, scores)`` of the best ``width`` hypotheses, the best first."""
        return beam_finish(self.scores, self.pool, self.history, self.step, **self._kw)


def search(search_: BeamSearch, cache: KVCache, lengths: List[int], prompt_logits: torch.Tensor,
           step: Callable[[torch.Tensor, torch.Tensor], torch.Tensor], check: Optional[Callable[[], None]] = None
           ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Runs a search to its end.  ``prompt_logits [B, V]``: request ``b``'s prompt of ``lengths[b]`` tokens lies in cache line ``b * width``;
    ``step(tokens [B * W], positions [B * W])`` writes the tokens into their lines and returns the logits behind them."""
    W, steps, ends = search_.width, search_.max_new_tokens, search_._kw["eos_token_id"] is not None
    lines = cache.beams(lengths, W, steps - 1)
    tokens, _ = search_.advance(prompt_logits)
    end = lines.start.clone()
    for t in range(1, steps):
        if ends and t % CHECK_EVERY == 0 and search_.finished():
            break
        logits = step(tokens.reshape(-1), end.repeat_interleave(W))
        end += 1
        tokens, parents = search_.advance(logits)
        if t + 1 < steps and W > 1:
            lines.reorder(parents, end)
        if check is not None:
            check()
    return search_.finish()


def sequences(input_ids: torch.Tensor, lengths: List[int], found: Tuple[torch.Tensor, torch.Tensor, torch.Tensor], n: int,
              pad_token_id: int) -> torch.Tensor:
    """Prompts with their best ``n`` continuations behind them, ``[B * n, T + the longest's tokens]``."""
    tokens = found[0][:, :n, : int(found[1][:, :n].max())]
    B, T = input_ids.shape
    out = torch.full((B, n, T + tokens.shape[2]), pad_token_id, dtype=input_ids.dtype, device=tokens.device)
    for b, length in enumerate(lengths):
        out[b, :, :length] = input_ids[b, :length].to(tokens.device)
        out[b, :, length:length + tokens.shape[2]] = tokens[b].to(out.dtype)
    return out.reshape(B * n, -1)
