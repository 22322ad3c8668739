"""Switch-Transformer load-balancing auxiliary loss (reference
``src/neuronx_distributed/modules/moe/loss_function.py:5-48``).

``loss = E / k * sum_e(fraction_of_tokens_routed_to_e * mean_router_prob_e)`` computed over all layers' router logits.
The reference concatenates them and builds the one-hot with an arange-compare in fp64 (an XLA workaround); here one kernel
reads every layer's logits where they are (``ops.balance_loss``), and another writes their gradients; on the CPU and for
other types it is torch in fp32.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from ...ops import balance_loss as ops


def load_balancing_loss_func(router_logits: Union[torch.Tensor, Sequence[torch.Tensor]], num_experts: int, top_k: int,
                             mask: Optional[torch.Tensor] = None, return_counts: bool = False
                             ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``router_logits``: ``[..., num_experts]``, or one such tensor per layer (``None`` entries are skipped).  A row's experts are
    its ``top_k`` largest logits, the lower one of two equal ones.  ``mask``: one truth value (or 0 / 1) per row of a layer, in
    the rows' order, the same for every layer; rows that it leaves out (padding) enter neither the shares nor the
    probabilities and get zero gradients, and with none left the loss is 0.  ``return_counts``: ``(loss, counts)`` with the
    int64 number of rows that chose each expert, all layers together."""
    logits = [router_logits] if isinstance(router_logits, torch.Tensor) else [t for t in router_logits if t is not None]
    if not logits:
        raise ValueError("no router logits")
    if not 0 < top_k <= num_experts:
        raise ValueError(f"Invalid top_k={top_k} for num_experts={num_experts}")
    if any(t.shape[-1:] != (num_experts,) and t.numel() % num_experts for t in logits):
        raise ValueError(f"router logits {[tuple(t.shape) for t in logits]} are no rows of {num_experts}")
    if mask is not None:
        mask = mask.reshape(-1).bool().contiguous()
        if mask.device != logits[0].device or any(t.numel() != mask.numel() * num_experts for t in logits):
            raise ValueError(f"a mask of {mask.numel()} rows for router logits {[tuple(t.shape) for t in logits]}")
    fn = ops.balance_loss if ops.qualifies(logits, num_experts) else ops.balance_loss_ref
    loss, counts = fn(logits, num_experts, top_k, mask)
    return (loss, counts) if return_counts else loss
