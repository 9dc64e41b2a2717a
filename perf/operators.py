"""The measured operators of the output head: what a program that scores or
tunes a (quantized) causal LM asks of its last layer, over a large vocabulary.

  xent     crb_amd.head.linear_cross_entropy: softmax cross entropy of the
           logits h W^T without keeping them, forward or with gradients
  distill  crb_amd.head.linear_distill: KL from a teacher's top logits to the
           student h W^T, forward or with gradients
  top      crb_amd.head.top_logits: a teacher's k largest logits of each row,
           their indices and the row's log-sum-exp

``own`` false computes the same in plain 32-bit torch operations.
"""
import math

import torch

own = False

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"
IGNORE = -100
LOSS_SCALE = {"fp16": 4096.0, "bf16": 1.0}    # a tuning step in fp16 scales its loss


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def _xent(name, tokens, hidden, vocab, dtype, grad, scale=1.0):
    return {"name": name, "kind": "xent", "tokens": tokens, "hidden": hidden, "vocab": vocab,
            "dtype": dtype, "grad": grad, "scale": scale}


def _distill(name, tokens, hidden, vocab, k, dtype, grad, tail, temperature):
    return {"name": name, "kind": "distill", "tokens": tokens, "hidden": hidden, "vocab": vocab,
            "k": k, "dtype": dtype, "grad": grad, "tail": tail, "temperature": temperature}


def _top(name, tokens, vocab, k, dtype):
    return {"name": name, "kind": "top", "tokens": tokens, "vocab": vocab, "k": k, "dtype": dtype}


def listed():
    return [
        # A few tokens of a toy model (hidden 128, 200 tokens): nothing but latency.
        _xent("xent_tiny", 5, 128, 200, "fp16", False),
        # The score of one next token at the head of an 8B model: the head's weight read once.
        _xent("xent_one_token", 1, 4096, 128256, "bf16", False),
        # One perplexity window of a 125M model.
        _xent("xent_window_768", 2047, 768, 50272, "fp16", False),
        # Two perplexity windows of a 6.7B model.
        _xent("xent_windows_4096", 4094, 4096, 50272, "fp16", False),
        # A short ragged tuning step: hidden no multiple of 64, odd vocabulary, logits scaled down.
        _xent("xent_step_ragged", 333, 1000, 32007, "bf16", True, 0.25),
        # A tuning step of an 8B model's head on one window, the largest.
        _xent("xent_step_8b", 2047, 4096, 128256, "bf16", True),
        # KL of a quantized model on a few tokens, with the tail as one outcome.
        _distill("distill_few_tokens", 17, 2048, 50272, 64, "fp16", False, True, 1.0),
        # A short distillation step of a 125M model at temperature 2.
        _distill("distill_step_768", 250, 768, 50272, 20, "bf16", True, False, 2.0),
        # A distillation step of a 6.7B model's head on one window.
        _distill("distill_step_4096", 2047, 4096, 50272, 128, "fp16", True, True, 1.0),
        # The teacher's candidates for one next token.
        _top("top_one_token", 1, 50272, 16, "fp16"),
        # A ragged batch of 32-bit logits.
        _top("top_ragged_fp32", 301, 32007, 50, "fp32"),
        # The teacher's logits of one window of an 8B model.
        _top("top_window", 2047, 128256, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _hidden(rng):
    """A hidden size: mostly multiples of 64, as models have, some ragged."""
    c = _log(rng, 128, 4096)
    r = rng.random()
    return c // 64 * 64 if r < 0.6 else c // 8 * 8 if r < 0.85 else c


def draw(rng):
    kind = rng.choice(["xent", "xent", "distill", "distill", "top"])
    while True:
        tokens, vocab = _log(rng, 1, 4096), _log(rng, 200, 131072)
        dtype = rng.choice(["fp16", "bf16"])
        if kind == "top":
            c = _top("", tokens, vocab, min(vocab, _log(rng, 1, 128)), rng.choice(["fp16", "bf16", "fp32"]))
        elif kind == "xent":
            c = _xent("", tokens, _hidden(rng), vocab, dtype, rng.random() < 0.6, rng.choice([1.0, 1.0, 0.25]))
        else:
            c = _distill("", tokens, _hidden(rng), vocab, min(vocab // 2, _log(rng, 1, 128)), dtype,
                         rng.random() < 0.6, rng.random() < 0.5, rng.choice([1.0, 2.0]))
        del c["name"]
        most = {"flops": 6.0 * 2047 * 4096 * 128256, "bytes": 2.5e9 if kind != "top" else 2.0 * 2047 * 128256}
        w = work(c)
        if all(w[k] <= most[k] for k in most) and 3072 not in c.values():
            return c


def work(case):
    """Each input read and each output written once; products of the logits
    and, with gradients, of both gradients."""
    T, V = case["tokens"], case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "top":
        return {"bytes": T * V * size + T * (case["k"] * (size + 4) + 4), "flops": 3.0 * T * V}
    C = case["hidden"]
    targets = T * 8 if case["kind"] == "xent" else T * (case["k"] * (size + 4) + 4)
    once = (T + V) * C * size
    if case["grad"]:
        return {"bytes": 2 * once + targets + 4, "flops": 6.0 * T * V * C}
    return {"bytes": once + targets + 4 * T, "flops": 2.0 * T * V * C}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rows(V, K, T, g):
    """K distinct tokens of each row, in no order: one of each K-th part."""
    part = (torch.arange(K, device=DEV) + torch.rand((T, K), device=DEV, generator=g)) * (V / K)
    idx = part.long().clamp_(max=V - 1)
    return idx.gather(1, torch.rand((T, K), device=DEV, generator=g).argsort(1))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    T, V, dt = case["tokens"], case["vocab"], DT[case["dtype"]]
    if case["kind"] == "top":
        # logits of a language model: a wide bulk, a few tokens far above it
        z = torch.randn((T, V), device=DEV, generator=g) * 2.0
        few = torch.randint(0, V, (T, 8), device=DEV, generator=g)
        z.scatter_add_(1, few, 8.0 * torch.rand((T, 8), device=DEV, generator=g))
        return {"case": case, "logits": z.to(dt)}
    C = case["hidden"]
    # a head whose logits spread by 1.5, hidden states with uneven channels
    # that point at their target by anything from nothing to certainty
    W = torch.randn((V, C), device=DEV, generator=g) * (1.5 / math.sqrt(C))
    chan = torch.exp(0.3 * torch.randn(C, device=DEV, generator=g))
    chan = chan / chan.square().mean().sqrt()
    h = torch.randn((T, C), device=DEV, generator=g) * chan
    pull = 12.0 * torch.rand((T, 1), device=DEV, generator=g)
    state = {"case": case}
    if case["kind"] == "xent":
        # token frequencies fall off as they do in text; a prompt's labels are masked
        y = (V ** torch.rand(T, device=DEV, generator=g)).long().clamp_(1, V) - 1
        h = h + pull * W[y] / W[y].norm(dim=1, keepdim=True)
        y[:T // 8] = IGNORE
        state["labels"] = y
    else:
        K, tau = case["k"], case["temperature"]
        idx = _rows(V, K, T, g)
        h = h + pull * W[idx[:, 0]] / W[idx[:, 0]].norm(dim=1, keepdim=True)
        gaps = -torch.log(torch.rand((T, K), device=DEV, generator=g).clamp_(min=1e-6))
        val = (10.0 - torch.cumsum(gaps * (4.0 / (1 + torch.arange(K, device=DEV))), 1)).to(dt)
        tail = 0.02 + 0.3 * torch.rand(T, device=DEV, generator=g)
        lse = torch.logsumexp(val.float() / tau, 1) - torch.log1p(-tail)
        state["top"] = (val, idx.to(torch.int32), lse if case["tail"] else None)
    state["up"] = torch.tensor(LOSS_SCALE[case["dtype"]], device=DEV)      # the loss's own gradient
    state["h"] = h.to(dt).requires_grad_(case["grad"])
    state["W"] = W.to(dt).requires_grad_(case["grad"])
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    from crb_amd import head

    case = state["case"]
    if case["kind"] == "top":
        top = head.top_logits(state["logits"], case["k"])
        return [top.val, top.idx, top.lse]
    reduction = "mean" if case["grad"] else "none"
    if case["kind"] == "xent":
        loss = head.linear_cross_entropy(state["h"], state["W"], state["labels"], scale=case["scale"],
                                         ignore_index=IGNORE, reduction=reduction)
    else:
        loss = head.linear_distill(state["h"], state["W"], state["top"], temperature=case["temperature"],
                                   reduction=reduction)
    if not case["grad"]:
        return [loss]
    dh, dW = torch.autograd.grad(loss, (state["h"], state["W"]), state["up"])
    return [loss.detach(), dh, dW]


@torch.no_grad()
def _plain(state):
    case = state["case"]
    if case["kind"] == "top":
        return _plain_top(state["logits"], case["k"])
    h, W = state["h"].float(), state["W"].float()
    if case["kind"] == "xent":
        s = case["scale"]
        z = (h @ W.t()) * s
        y = state["labels"]
        live = y != IGNORE
        at = y.clamp(min=0)[:, None]
        m = z.max(1, keepdim=True).values
        e = torch.exp(z - m)
        total = e.sum(1, keepdim=True)
        loss = torch.where(live, (torch.log(total) + m - z.gather(1, at))[:, 0], 0.0)
        if not case["grad"]:
            return [loss]
        n = live.sum().clamp(min=1)
        dz = e / total
        dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
        dz *= live[:, None] * (s * state["up"] / n)
        loss = loss.sum() / n
    else:
        s = 1.0 / case["temperature"]
        z = (h @ W.t()) * s
        val, idx, lse = state["top"]
        at, t = idx.long(), val.float() * s
        if lse is None:
            p = torch.exp(t - t.max(1, keepdim=True).values)
            p = p / p.sum(1, keepdim=True)
            rest = torch.zeros_like(p[:, :1])
        else:
            p = torch.exp(t - lse[:, None])
            rest = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        zt = z.gather(1, at)
        m = z.max(1, keepdim=True).values
        e = torch.exp(z - m)
        tail = e.scatter(1, at, 0.0).sum(1, keepdim=True)
        total = e.sum(1, keepdim=True)
        full = torch.log(total) + m
        cross = torch.where(rest > 0, rest * (torch.log(rest.clamp(min=1e-38)) - torch.log(tail / total)), 0.0)
        loss = (p * (torch.log(p.clamp(min=1e-38)) - zt + full)).sum(1) + cross[:, 0]
        if not case["grad"]:
            return [loss]
        dz = e * ((tail / total - rest) / tail)
        dz.scatter_(1, at, torch.exp(zt - full) - p)
        dz *= s * state["up"] / h.shape[0]
        loss = loss.mean()
    return [loss, (dz @ W).to(state["h"].dtype), (dz.t() @ h).to(state["W"].dtype)]


def _plain_top(logits, k):
    """Values as ordered whole numbers with the index below them, so that ties
    go to the lowest index."""
    x = logits.float() + 0.0
    bits = x.view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    V = x.shape[1]
    key = (order.long() << 32) | (V - 1 - torch.arange(V, device=x.device))
    best = torch.topk(key, k, dim=1).values
    idx = V - 1 - (best & 0xFFFFFFFF)
    m = x.max(1, keepdim=True).values
    lse = torch.log(torch.exp(x - m).sum(1)) + m[:, 0]
    return [logits.gather(1, idx), idx.to(torch.int32), lse]


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "top":
        z = state["logits"].double()
        val, idx = torch.sort(z, dim=1, descending=True, stable=True)
        k = case["k"]
        return [val[:, :k].clone(), idx[:, :k].to(torch.int32).clone(), torch.logsumexp(z, 1)]
    h, W = state["h"].double(), state["W"].double()
    T = h.shape[0]
    if case["kind"] == "xent":
        s = case["scale"]
        logq = torch.log_softmax(s * (h @ W.t()), 1)
        y = state["labels"]
        live = torch.nonzero(y != IGNORE)[:, 0]
        rows = torch.zeros(T, dtype=torch.float64, device=DEV)
        rows[live] = -logq[live, y[live]]
        if not case["grad"]:
            return [rows]
        n = max(1, live.numel())
        loss = rows.sum() / n
        dz = torch.zeros_like(logq)
        dz[live] = logq[live].exp()
        dz[live, y[live]] = torch.expm1(logq[live, y[live]])
    else:
        s = 1.0 / case["temperature"]
        z = s * (h @ W.t())
        val, idx, lse = state["top"]
        idx = idx.long()
        if lse is None:
            logp = torch.log_softmax(s * val.double(), 1)
            rest = torch.zeros(T, 1, dtype=torch.float64, device=DEV)
        else:
            logp = s * val.double() - lse.double()[:, None]
            rest = -torch.expm1(torch.logsumexp(logp, 1, keepdim=True).clamp(max=0))
        full = torch.logsumexp(z, 1, keepdim=True)
        others = torch.logsumexp(z.scatter(1, idx, -math.inf), 1, keepdim=True)
        rows = (logp.exp() * (logp - z.gather(1, idx) + full)).sum(1)
        rows = rows + (torch.special.xlogy(rest, rest) - rest * (others - full))[:, 0]
        if not case["grad"]:
            return [rows]
        n = T
        loss = rows.mean()
        # the teacher spreads the tail's probability as the student does
        target = rest * torch.exp(z - others)
        target.scatter_(1, idx, logp.exp())
        dz = torch.exp(z - full) - target
    dz *= s * float(state["up"]) / n
    return [loss, dz @ W, dz.t() @ h]
