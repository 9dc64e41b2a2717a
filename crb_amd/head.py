"""Losses of a causal LM's output head over a large vocabulary, without
keeping the logits, on the crbq kernels.

    loss = linear_cross_entropy(h, head.weight, labels)        # h [..., C], labels [...]
    top = top_logits(teacher_logits, k=64)                     # TopLogits(val, idx, lse)
    loss = linear_distill(h, head.weight, top, temperature=2.0)

Both losses are differentiable in h and weight (once); the logits
scale * h W^T are computed in pieces of the vocabulary, again in the backward
pass.  h and weight are both fp16 or both bf16; losses are fp32.  The
reference has no counterpart: its perplexity forms all logits and calls a
cross entropy (eval_ppl_utils.py:626-636).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as fwad

from . import kernels
from ._lib import CrbqError


class TopLogits(NamedTuple):
    """A teacher's k largest logits of each row."""
    val: torch.Tensor                  # [..., k], descending, the logits' dtype
    idx: torch.Tensor                  # int32 [..., k]; outside [0, V): an empty slot
    lse: Optional[torch.Tensor]        # fp32 [...]: log sum exp of logits / temperature


class _Loss(torch.autograd.Function):
    """One of the losses; call, top and ignore_index as kernels takes them."""

    @staticmethod
    def forward(ctx, h, weight, call, top, ignore_index):
        loss, state = call.forward(top, ignore_index)
        ctx.save_for_backward(h, weight, call.labels, state)
        ctx.call = call
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        call, state = ctx.call, ctx.saved_tensors[3]   # (and the check that none was changed)
        dh, dW = call.grad(state, g.contiguous(), ctx.needs_input_grad[0],
                           ctx.needs_input_grad[1])
        return dh, dW, None, None, None


def _loss(h, weight, call, top=None, ignore_index=-100):
    # (a forward-mode tangent is refused by the Function, not dropped)
    if (torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad)
            or fwad._current_level >= 0):
        return _Loss.apply(h, weight, call, top, ignore_index)
    return call.forward(top, ignore_index)[0]


def _rows(x: torch.Tensor, lead, what: str, tail: int) -> torch.Tensor:
    """x [*lead, (k)] with its leading dimensions as one."""
    if x.shape[:x.dim() - tail] != lead:
        raise CrbqError(f"{what} of shape {tuple(x.shape)} do not fit hidden states of "
                        f"{tuple(lead)} tokens")
    return x if len(lead) == 1 else x.reshape(-1, *x.shape[x.dim() - tail:])


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                         scale: float = 1.0, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """torch's cross_entropy(scale * h @ weight.T, labels) in fp32, the logits
    never kept.  h [..., C], weight [V, C], labels [...] int64; a token whose
    label is ignore_index has loss 0 and is left out of the mean (a mean over
    no token is NaN) and of the gradients; a label outside the vocabulary
    makes loss and gradients NaN.  reduction "mean", "sum" or "none"."""
    lead = h.shape[:-1]
    x = h if len(lead) == 1 else h.reshape(-1, h.shape[-1])
    call = kernels.xent_call(x, weight, _rows(labels, lead, "labels", 0), scale, reduction,
                             "linear_cross_entropy")
    loss = _loss(x, weight, call, None, int(ignore_index))
    return loss if reduction != "none" or len(lead) == 1 else loss.reshape(lead)


def linear_distill(h: torch.Tensor, weight: torch.Tensor, top, temperature: float = 1.0,
                   scale: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """KL divergence from a teacher's top logits to the student's softmax of
    scale / temperature * h @ weight.T, whose logits are never kept.

    top: a TopLogits or (val, idx, lse).  lse None: the teacher is the
    softmax of its listed logits / temperature.  With lse (top_logits at the
    same temperature) the tokens not listed are one more outcome, of what the
    listed ones leave.  A row that lists nothing is left out (loss 0).  The
    loss has no factor temperature ** 2."""
    val, idx, lse = top
    lead = h.shape[:-1]
    x = h if len(lead) == 1 else h.reshape(-1, h.shape[-1])
    top = kernels.top_args(x, _rows(val, lead, "teacher logits", 1),
                           _rows(idx, lead, "teacher tokens", 1),
                           None if lse is None else _rows(lse, lead, "teacher log-sum-exps", 0),
                           "linear_distill")
    call = kernels.distill_call(x, weight, top[0].shape[1], scale, temperature, reduction,
                                "linear_distill")
    loss = _loss(x, weight, call, top)
    return loss if reduction != "none" or len(lead) == 1 else loss.reshape(lead)


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest of logits [..., V] (ties to the lowest index, NaN above
    everything) and the log-sum-exp of logits / temperature."""
    lead = logits.shape[:-1]
    if len(lead) == 1:
        return TopLogits(*kernels.top_logits(logits, k, temperature))
    val, idx, lse = kernels.top_logits(logits.reshape(-1, logits.shape[-1]), k, temperature)
    return TopLogits(val.reshape(*lead, k), idx.reshape(*lead, k), lse.reshape(lead))
