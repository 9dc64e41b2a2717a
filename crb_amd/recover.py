"""Tuning the output end of a quantized model against the dense model.

The decoder layers stay as the quantizer left them; the final norm and the
output head (which the quantizer does not touch) are tuned so that the quantized
model's predictions on the calibration windows come back to the dense
model's, of which only the top logits of each token are kept:

    top = teacher_top(model, windows, k=64)          # before quantization
    StackQuantizer(model, ...).run(windows)
    losses = recover_head(model, windows, top, steps=20)
    eval_ppl(model, ids, seqlen, fused=True)

The loss is head.linear_distill, its logits never kept; weights are held
in fp32 while they are tuned (AdamW) and rounded to the model's type for every
step.  No counterpart in the reference.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .evaluate import final_hidden, split_head
from .head import TopLogits, linear_distill, top_logits

LOSS_SCALE = 4096.0          # of fp16 gradients: a mean over many tokens is below their range


@torch.no_grad()
def teacher_top(model: nn.Module, windows: torch.Tensor, k: int = 64, temperature: float = 1.0,
                chunk: int = 8) -> TopLogits:
    """The top k logits of every token of windows [nsamples, seqlen], with the
    log-sum-exp of each token's logits / temperature: [nsamples, seqlen, (k)]."""
    mods, head, scale = split_head(model)
    hidden = final_hidden(model, windows, chunk)
    tops = []
    for h in hidden:                                 # a window's logits at a time
        for m in mods + [head]:
            h = m(h)
        tops.append(top_logits(h / scale if scale != 1.0 else h, min(k, h.shape[-1]),
                               temperature))
    return TopLogits(*(torch.stack(x) for x in zip(*tops)))


def _untie(model: nn.Module, head: nn.Linear) -> None:
    """A head that shares the embedding's weight gets its own: the embedding
    (and with it the hidden states) stays."""
    emb = getattr(model, "get_input_embeddings", lambda: None)()
    if emb is not None and emb.weight is head.weight:
        head.weight = nn.Parameter(head.weight.detach().clone())
        if hasattr(getattr(model, "config", None), "tie_word_embeddings"):
            model.config.tie_word_embeddings = False


def recover_head(model: nn.Module, windows: torch.Tensor, top: TopLogits, steps: int = 20,
                 lr: float = 1e-4, temperature: float = 1.0, batch: int = 4, chunk: int = 8,
                 seed: int = 0) -> list:
    """Tune the modules behind the decoder layers for ``steps`` steps on
    ``batch`` windows each, towards the teacher's ``top`` (teacher_top of the same
    windows and temperature).  Returns the losses (mean KL per token)."""
    mods, head, scale = split_head(model)
    _untie(model, head)
    hidden = final_hidden(model, windows, chunk)
    params = [p for m in mods + [head] for p in m.parameters()]
    masters = [p.detach().float().clone() for p in params]
    opt = torch.optim.AdamW(masters, lr=lr, weight_decay=0.0)
    up = LOSS_SCALE if head.weight.dtype == torch.float16 else 1.0
    g = torch.Generator().manual_seed(seed)
    wanted = [p.requires_grad for p in params]
    losses = []
    try:
        for p in params:
            p.requires_grad_(True)
        for _ in range(steps):
            pick = torch.randperm(windows.shape[0], generator=g)[:batch].to(hidden.device)
            with torch.enable_grad():
                h = hidden[pick]
                for m in mods:
                    h = m(h)
                loss = linear_distill(h, head.weight, [x[pick] for x in top], temperature,
                                      scale=1.0 / scale)
                grads = torch.autograd.grad(loss * up, params)
            for m, d in zip(masters, grads):
                m.grad = d.float() / up
            opt.step()
            with torch.no_grad():
                for p, m in zip(params, masters):
                    p.copy_(m)
            losses.append(loss.detach())
    finally:
        for p, w in zip(params, wanted):
            p.requires_grad_(w)
    return [float(x) for x in losses]
