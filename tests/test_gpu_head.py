"""The output-head losses (linear_cross_entropy, linear_distill) and
top_logits against plain 64-bit implementations.

Tolerances.  z is a sum of C exact products in fp32: its error is taken as a
random walk of C roundings, dz0 = 4 sqrt(C) 2^-24 max sum_c |s h W|.  A
loss is a few exponentials and logarithms of such z (relative 2^-22 each)
away: |error| <= 2 dz0 + 2^-21 (1 + max |z| + |loss|).  A gradient adds one rounding
of every dz (d = u = 2^-8 bf16, 2^-11 fp16; up to 64 tokens dz has two parts, d = u^2),
fp32 sums, one rounding of the result and, in fp16, the spacing of subnormal numbers:
  |error| <= (d + 2 dz0 + 2^-20 (1 + max |z|)) sum (q + p) |factor| + u |result| + tiny.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def make(T, V, C, dtype, seed=0, pull=4.0):
    g = torch.Generator().manual_seed(seed)
    W = torch.randn(V, C, generator=g) * (1.5 / math.sqrt(C))
    h = torch.randn(T, C, generator=g)
    y = torch.randint(0, V, (T,), generator=g)
    h = h + pull * torch.rand(T, 1, generator=g) * W[y] / (W[y].norm(dim=1, keepdim=True) + 1e-6)
    return h.to(dtype).to(DEV), W.to(dtype).to(DEV), y.to(DEV)


def ref_z(h, W, s):
    """(z in 64 bits, bound of its fp32 error)"""
    hd, wd = h.double().cpu(), W.double().cpu()
    z = s * (hd @ wd.t())
    mag = abs(s) * (hd.abs() @ wd.abs().t())
    return z, 4 * math.sqrt(h.shape[1]) * 2.0 ** -24 * float(mag.max())


def loss_tol(z, dz0, loss):
    return 2 * dz0 + 2.0 ** -21 * (1 + float(z.abs().max()) + loss.abs())


def grad_refs(h, W, dz, both, dz0, z, s, dtype):
    """dz [T, V] (with the loss gradient's coefficient), both = q + p times
    its size: (dh, tolerance, dW, tolerance)."""
    hd, wd, u = h.double().cpu(), W.double().cpu(), U[dtype]
    d = u * u if h.shape[0] <= 64 else u
    e = d + 2 * dz0 + 2.0 ** -20 * (1 + float(z.abs().max()))
    dh, dW = s * dz @ wd, s * dz.t() @ hd
    th = abs(s) * e * (both @ wd.abs()) + u * dh.abs() + TINY[dtype]
    tw = abs(s) * e * (both.t() @ hd.abs()) + u * dW.abs() + TINY[dtype]
    return dh, th, dW, tw


def close(got, want, tol, what):
    got = got.double().cpu()
    bad = (got - want).abs() - tol
    assert not torch.isnan(got).any() and float(bad.max()) <= 0, (
        what, float(bad.max()), float((got - want).abs().max()))


def ref_xent(h, W, y, s, ignore, coef):
    z, dz0 = ref_z(h, W, s)
    logq = torch.log_softmax(z, 1)
    y = y.cpu()
    live = y != ignore
    at = torch.where(live, y, 0)[:, None]
    loss = torch.where(live, -logq.gather(1, at)[:, 0], 0.0)
    q = logq.exp()
    onehot = torch.zeros_like(q).scatter_(1, at, 1.0)
    w = (coef * live)[:, None]
    return z, dz0, loss, (q - onehot) * w, (q + onehot) * w.abs()


SIZES = [(1, 1, 8), (1, 200, 128), (2, 3, 33), (5, 203, 128), (16, 257, 64), (17, 300, 72),
         (64, 255, 200), (65, 511, 96), (129, 513, 264), (256, 256, 256), (257, 1025, 136),
         (300, 777, 1000), (513, 130, 61)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,C", SIZES)
def test_xent(T, V, C, dtype):
    from crb_amd.head import linear_cross_entropy
    h, W, y = make(T, V, C, dtype, T + V)
    if T > 4:
        y[1::4] = -100
    for s in (1.0, -0.5):
        n = int((y != -100).sum())
        z, dz0, loss, dz, both = ref_xent(h, W, y, s, -100, torch.full((T,), 1.0 / n).double())
        rows = linear_cross_entropy(h, W, y, scale=s, reduction="none")
        tol = loss_tol(z, dz0, loss)
        close(rows, loss, tol, "rows")
        total = linear_cross_entropy(h, W, y, scale=s, reduction="sum")
        close(total, loss.sum(), tol.sum(), "sum")
        h2, W2 = h.clone().requires_grad_(), W.clone().requires_grad_()
        mean = linear_cross_entropy(h2, W2, y, scale=s)
        close(mean, loss.sum() / n, tol.mean() * T / n, "mean")
        mean.backward()
        dh, th, dW, tw = grad_refs(h, W, dz, both, dz0, z, s, dtype)
        close(h2.grad, dh, th, "dh")
        close(W2.grad, dW, tw, "dW")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_xent_row_gradients(dtype):
    """reduction "none" with a gradient of its own for each row: large, tiny
    (far below fp16's range next to the largest), negative, zero."""
    from crb_amd.head import linear_cross_entropy
    T, V, C = 70, 300, 64
    h, W, y = make(T, V, C, dtype, 3)
    y[5] = -100
    g = torch.randn(T) * 10.0 ** torch.linspace(-6, 1, T)
    g[7] = 0.0
    z, dz0, loss, dz, both = ref_xent(h, W, y, 1.0, -100, g.double())
    h.requires_grad_(), W.requires_grad_()
    rows = linear_cross_entropy(h, W, y, reduction="none")
    got = torch.autograd.grad(rows, (h, W), g.to(DEV))
    dh, th, dW, tw = grad_refs(h.detach(), W.detach(), dz, both, dz0, z, 1.0, dtype)
    # a row's dz is rounded relative to the largest coefficient in fp16
    floor = (2.0 ** -25 / 16384 * float(g.abs().max()) if dtype == torch.float16 else 0.0)
    th = th + floor * W.detach().double().cpu().abs().sum(0)
    tw = tw + floor * h.detach().double().cpu().abs().sum(0)
    close(got[0], dh, th, "dh")
    close(got[1], dW, tw, "dW")
    assert not got[0][5].any() and not got[0][7].any()


def test_xent_many_pieces():
    """More tokens x vocabulary than one piece of the backward pass holds."""
    from crb_amd.head import linear_cross_entropy
    T, V, C, dtype = 4100, 20001, 64, torch.bfloat16
    h, W, y = make(T, V, C, dtype, 1)
    h.requires_grad_(), W.requires_grad_()
    loss = linear_cross_entropy(h, W, y, reduction="sum")
    dh, dW = torch.autograd.grad(loss, (h, W))
    with torch.no_grad():
        z = h.double() @ W.double().t()
        logq = torch.log_softmax(z, 1)
        want = -logq.gather(1, y[:, None]).sum()
        dz0 = 4 * math.sqrt(C) * 2.0 ** -24 * float((h.double().abs() @ W.double().abs().t()).max())
        q = logq.exp()
        one = torch.zeros_like(q).scatter_(1, y[:, None], 1.0)
        e = U[dtype] + 2 * dz0 + 2.0 ** -20 * (1 + float(z.abs().max()))
        assert abs(float(loss.double() - want)) <= T * 2 * dz0 + 2.0 ** -18 * float(want)
        for got, r, m in ((dh, (q - one) @ W.double(), (q + one) @ W.double().abs()),
                          (dW, (q - one).t() @ h.double(), (q + one).t() @ h.double().abs())):
            assert float(((got.double() - r).abs() - e * m - U[dtype] * r.abs()).max()) <= 0


def ref_distill(h, W, val, idx, lse, s, tau, coef):
    """Slot by slot, as the definition reads; idx outside [0, V) are empty."""
    z, dz0 = ref_z(h, W, s / tau)
    T, V = z.shape
    val, idx = val.double().cpu() / tau, idx.long().cpu()
    loss = torch.zeros(T, dtype=torch.float64)
    dz, both = torch.zeros_like(z), torch.zeros_like(z)
    for t in range(T):
        ok = (idx[t] >= 0) & (idx[t] < V)
        at, x = idx[t][ok], val[t][ok]
        if not at.numel():
            continue
        p = torch.softmax(x, 0) if lse is None else (x - float(lse[t])).exp()
        pt = 0.0 if lse is None else max(0.0, 1.0 - float(p.sum()))
        logq = torch.log_softmax(z[t], 0)
        out = torch.ones(V, dtype=torch.bool)
        out[at] = False
        if not out.any():
            pt = 0.0
        loss[t] = (torch.special.xlogy(p, p) - torch.where(p > 0, p * logq[at], 0.0)).sum()
        target = torch.zeros(V, dtype=torch.float64).index_add_(0, at, p)
        if pt > 0:
            lt = torch.logsumexp(logq[out], 0)
            loss[t] += pt * (math.log(pt) - lt)
            target[out] = pt * (logq[out] - lt).exp()
        total = target.sum()
        dz[t] = (logq.exp() * total - target) * coef[t]
        both[t] = (logq.exp() * total + target) * abs(coef[t])
    return z, dz0, loss, dz, both


def teacher(T, V, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    val = (3.0 * torch.randn(T, k, generator=g)).to(dtype)
    return val.to(DEV), idx.to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,C,k", [(1, 1, 8, 1), (1, 200, 128, 7), (3, 256, 40, 256),
                                     (17, 300, 72, 20), (65, 511, 96, 100), (130, 1025, 64, 255),
                                     (300, 777, 200, 3)])
def test_distill(T, V, C, k, dtype):
    from crb_amd.head import linear_distill
    h, W, _ = make(T, V, C, dtype, T + V)
    val, idx = teacher(T, V, k, 9, torch.float32 if k % 2 else dtype)
    for tail, tau, s in ((False, 1.0, 1.0), (True, 2.0, 0.5)):
        lse = None
        if tail:
            rest = torch.rand(T, generator=torch.Generator().manual_seed(4)).to(DEV) * 0.5
            rest[0] = 0.0
            lse = torch.logsumexp(val.float() / tau, 1) - torch.log1p(-rest)
        z, dz0, loss, dz, both = ref_distill(h, W, val, idx, lse, s, tau,
                                             torch.full((T,), 1.0 / T).double())
        # p and 1 - sum p are fp32: their rounding (2^-22 each, times |log q| <= 2 max|z| + log V)
        more = 2.0 ** -20 * (2 * float(z.abs().max()) + math.log(V) + 16)
        rows = linear_distill(h, W, (val, idx, lse), temperature=tau, scale=s, reduction="none")
        tol = loss_tol(z, dz0, loss) + more
        close(rows, loss, tol, "rows")
        h2, W2 = h.clone().requires_grad_(), W.clone().requires_grad_()
        mean = linear_distill(h2, W2, (val, idx, lse), temperature=tau, scale=s)
        close(mean, loss.mean(), tol.mean(), "mean")
        mean.backward()
        dh, th, dW, tw = grad_refs(h, W, dz, both, dz0, z, s / tau, dtype)
        close(h2.grad, dh, th, "dh")
        close(W2.grad, dW, tw, "dW")


def test_distill_many_pieces():
    """Lists over more than one piece of the backward pass."""
    from crb_amd.head import linear_distill
    T, V, C, k, dtype = 8200, 20001, 64, 12, torch.float16
    h, W, _ = make(T, V, C, dtype, 3)
    g = torch.Generator().manual_seed(7)
    idx = (torch.arange(k) * (V // k) + torch.randint(0, V // k, (T, k), generator=g)).to(DEV)
    idx = torch.where(torch.arange(T, device=DEV)[:, None] % 2 == 0, idx, idx.flip(1))
    val = torch.randn(T, k, generator=g).to(DEV)
    lse = torch.logsumexp(val, 1) + 0.5
    h.requires_grad_(), W.requires_grad_()
    loss = linear_distill(h, W, (val, idx.int(), lse), reduction="sum")
    dh, dW = torch.autograd.grad(loss, (h, W))
    with torch.no_grad():
        hd, wd = h.double(), W.double()
        z = hd @ wd.t()
        dz0 = 4 * math.sqrt(C) * 2.0 ** -24 * float((hd.abs() @ wd.abs().t()).max())
        big = float(z.abs().max())
        logq = torch.log_softmax(z, 1)
        p = (val.double() - lse.double()[:, None]).exp()
        pt = 1 - p.sum(1)
        lt = torch.logsumexp(logq.scatter(1, idx, -math.inf), 1)
        want = ((p * (p.log() - logq.gather(1, idx))).sum(1) + pt * (pt.log() - lt)).sum()
        target = (pt[:, None] * (logq - lt[:, None]).exp()).scatter(1, idx, p)
        q = logq.exp()
        del z, logq
        e = U[dtype] + 2 * dz0 + 2.0 ** -20 * (1 + big)
        # a row: z's error, and p's and 1 - sum p's (2^-22 each, times |log q|)
        row = 2 * dz0 + 2.0 ** -20 * (2 * big + math.log(V) + 16)
        assert abs(float(loss.double() - want)) <= T * row + 2.0 ** -18 * float(want)
        for got, r, m in ((dh, (q - target) @ wd, (q + target) @ wd.abs()),
                          (dW, (q - target).t() @ hd, (q + target).t() @ hd.abs())):
            tol = e * m + U[dtype] * r.abs() + TINY[dtype]
            assert float(((got.double() - r).abs() - tol).max()) <= 0


# more tiles of 64 tokens than CUs
MANY = [(300, 14001, 72), (65, 35001, 200), (513, 8001, 136), (1030, 4099, 328)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,C", MANY)
def test_xent_many_tiles(T, V, C, dtype):
    test_xent(T, V, C, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("T,V,C", MANY)
def test_distill_many_tiles(T, V, C, dtype):
    test_distill(T, V, C, T % 64 + 1, dtype)


def test_many_tiles_rows():
    """Gradients of their own for many rows, some of them 0, NaN hidden states where
    nothing is learned, a strided weight."""
    from crb_amd.head import linear_cross_entropy
    T, V, C, dtype = 300, 14001, 72, torch.bfloat16
    h, W, y = make(T, V, C, dtype, 23)
    y[7::9] = -100
    g = torch.randn(T, generator=torch.Generator().manual_seed(2))
    g[:128:2] = 0.0
    z, dz0, loss, dz, both = ref_xent(h, W, y, 1.0, -100, g.double())
    wide = torch.full((V, C + 16), math.nan, device=DEV, dtype=dtype)
    wide[:, 8:8 + C] = W
    dead = h.clone()
    dead[7::9] = math.nan
    dead.requires_grad_(), wide.requires_grad_()
    rows = linear_cross_entropy(dead, wide[:, 8:8 + C], y, reduction="none")
    close(rows.detach(), loss, loss_tol(z, dz0, loss), "rows")
    got = torch.autograd.grad(rows, (dead, wide), g.to(DEV))
    dh, th, dW, tw = grad_refs(h, W, dz, both, dz0, z, 1.0, dtype)
    close(got[0], dh, th, "dh")
    close(got[1][:, 8:8 + C], dW, tw, "dW")
    assert not got[0][7::9].any() and not got[0][:128:2].any()


def test_distill_odd_lists():
    """Empty slots, a row that lists nothing, a token listed twice, a teacher
    that gives a listed token no probability, one with all of it."""
    from crb_amd.head import linear_distill
    T, V, C, k = 6, 90, 32, 5
    h, W, _ = make(T, V, C, torch.float16, 2)
    val, idx = teacher(T, V, k, 5)
    idx[0, 1] = -1
    idx[0, 3] = V
    idx[1] = -1
    idx[2] = V + torch.arange(k, dtype=torch.int32, device=DEV)
    idx[3, 4] = idx[3, 0]
    idx[3, 2] = idx[3, 0]
    val[4, 2] = -math.inf
    val[5, 0] = 300.0
    for tail in (False, True):
        lse = torch.logsumexp(val, 1) + 0.3 if tail else None
        live = torch.tensor([1, 0, 0, 1, 1, 1]).double()
        z, dz0, loss, dz, both = ref_distill(h, W, val, idx, lse, 1.0, 1.0, live / 4)
        rows = linear_distill(h, W, (val, idx, lse), reduction="none")
        tol = loss_tol(z, dz0, loss) + 2.0 ** -20 * (2 * float(z.abs().max()) + 21)
        # exp(300 - 300.3) carries the rounding of 300 in fp32
        tol = tol + 300 * 2.0 ** -23 * 10 * tail
        close(rows, loss, tol, "rows")
        assert float(rows[1]) == 0 and float(rows[2]) == 0
        h2, W2 = h.clone().requires_grad_(), W.clone().requires_grad_()
        mean = linear_distill(h2, W2, (val, idx, lse))
        close(mean, loss.sum() / 4, tol.sum() / 4, "mean")
        mean.backward()
        dh, th, dW, tw = grad_refs(h, W, dz, both, dz0 + 1e-4 * tail, z, 1.0, torch.float16)
        close(h2.grad, dh, th, "dh")
        close(W2.grad, dW, tw, "dW")
        assert not h2.grad[1:3].any()


def test_distill_teacher_that_does_not_add_up():
    """A log-sum-exp below that of the listed logits: probabilities above 1 in
    sum, no tail; the gradient is still the loss's."""
    from crb_amd.head import linear_distill
    T, V, C, k = 70, 300, 64, 6
    h, W, _ = make(T, V, C, torch.bfloat16, 21)
    val, idx = teacher(T, V, k, 6)
    lse = torch.logsumexp(val, 1) - 0.25
    z, dz0, loss, dz, both = ref_distill(h, W, val, idx, lse, 1.0, 1.0, torch.ones(T).double())
    h.requires_grad_(), W.requires_grad_()
    rows = linear_distill(h, W, (val, idx, lse), reduction="none")
    more = 2.0 ** -20 * (2 * float(z.abs().max()) + math.log(V) + 16)
    close(rows.detach(), loss, 2 * (loss_tol(z, dz0, loss) + more), "rows")
    got = torch.autograd.grad(rows, (h, W), torch.ones(T, device=DEV))
    dh, th, dW, tw = grad_refs(h.detach(), W.detach(), dz, both, dz0, z, 1.0, torch.bfloat16)
    close(got[0], dh, th, "dh")
    close(got[1], dW, tw, "dW")


@pytest.mark.parametrize("T", [1, 64, 65, 200])
def test_tile_edges_of_tokens(T):
    """Token counts around the tiles' edges, hidden states of one stage."""
    from crb_amd.head import linear_cross_entropy
    V, C = 513, 64
    h, W, y = make(T, V, C, torch.float16, T)
    z, dz0, loss, dz, both = ref_xent(h, W, y, 1.0, -100, torch.ones(T).double())
    h.requires_grad_(), W.requires_grad_()
    out = linear_cross_entropy(h, W, y, reduction="sum")
    close(out.detach(), loss.sum(), loss_tol(z, dz0, loss).sum(), "sum")
    got = torch.autograd.grad(out, (h, W))
    dh, th, dW, tw = grad_refs(h.detach(), W.detach(), dz, both, dz0, z, 1.0, torch.float16)
    close(got[0], dh, th, "dh")
    close(got[1], dW, tw, "dW")


def test_distill_nothing_listed():
    from crb_amd.head import linear_distill
    h, W, _ = make(3, 40, 16, torch.bfloat16)
    h.requires_grad_(), W.requires_grad_()
    val, idx = torch.zeros(3, 2, device=DEV), torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    loss = linear_distill(h, W, (val, idx, None))
    assert math.isnan(float(loss))
    dh, dW = torch.autograd.grad(loss, (h, W))
    assert not dh.any() and not dW.any()


@pytest.mark.parametrize("kind", ["xent", "distill"])
def test_gradient_against_differences(kind):
    """Along a direction of h and W: the loss at both ends of a step that the
    16-bit inputs hold exactly against the gradient in between."""
    from crb_amd import head
    T, V, C = 40, 500, 64
    h, W, y = make(T, V, C, torch.float16, 8)
    val, idx = teacher(T, V, 9, 2)
    lse = torch.logsumexp(val, 1) + 0.2

    def f(a, b):
        if kind == "xent":
            return head.linear_cross_entropy(a, b, y, reduction="sum")
        return head.linear_distill(a, b, (val, idx, lse), reduction="sum")

    for which in (0, 1):
        x = (h, W)[which]
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
        step = 0.02 / math.sqrt(C) / (1.0 if which else 0.1)
        lo, hi = (x - step * d.half()), (x + step * d.half())
        mid = ((lo.double() + hi.double()) / 2).half()
        args = [h, W]
        args[which] = mid.requires_grad_()
        g, = torch.autograd.grad(f(*args), args[which])
        args[which] = lo
        l0 = float(f(*args))
        args[which] = hi
        l1 = float(f(*args))
        want = float((g.double() * (hi.double() - lo.double())).sum())
        size = float((g.double() * (hi.double() - lo.double())).abs().sum())
        # rounding of g (2^-11 of each term, and dz's again), of both losses, and the
        # third derivative: |z'|^3 / 24 per row with |z'| of one row's step
        dz1 = float(((hi.double() - lo.double()) @ W.double().t()).abs().max()) if which == 0 else \
            float((h.double() @ (hi.double() - lo.double()).t()).abs().max())
        tol = 2.0 ** -10 * size + 1e-5 * (abs(l0) + abs(l1)) + T * dz1 ** 3 / 12
        assert abs((l1 - l0) - want) <= tol, (l1 - l0, want, tol)
        assert tol < 0.2 * size


@pytest.mark.parametrize("T", [3, 40, 300])
def test_masked_rows_keep_their_nan(T):
    """A masked token's infinities and NaN reach neither loss nor gradients."""
    from crb_amd.head import linear_cross_entropy
    V, C = 300, 72
    h, W, y = make(T, V, C, torch.bfloat16, 6)
    y[1] = -100
    y[T - 1] = -100
    bad = h.clone()
    bad[1] = float("nan")
    bad[T - 1] = float("inf")
    out = []
    for x in (h, bad):
        x, w = x.clone().requires_grad_(), W.clone().requires_grad_()
        loss = linear_cross_entropy(x, w, y)
        out.append((loss.detach(), *torch.autograd.grad(loss, (x, w))))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_xent_all_masked_and_outside():
    from crb_amd.head import linear_cross_entropy
    h, W, y = make(20, 100, 24, torch.float16)
    h.requires_grad_(), W.requires_grad_()
    none = torch.full_like(y, -100)
    loss = linear_cross_entropy(h, W, none)
    assert math.isnan(float(loss))
    dh, dW = torch.autograd.grad(loss, (h, W))
    assert not dh.any() and not dW.any()
    assert float(linear_cross_entropy(h, W, none, reduction="sum")) == 0
    y[3], y[4] = 100, -1
    rows = linear_cross_entropy(h, W, y, reduction="none")
    assert torch.isnan(rows).nonzero().flatten().tolist() == [3, 4]
    # an index that is a token too
    y2 = torch.full_like(y, 7)
    assert not linear_cross_entropy(h, W, y2, ignore_index=7, reduction="none").any()


def test_confident_row_keeps_its_small_loss():
    """loss = log(1 + exp(a - z)) of a row whose label has all but 1e-9."""
    from crb_amd.head import linear_cross_entropy
    V, C = 300, 8
    W = torch.zeros(V, C, device=DEV, dtype=torch.float16)
    W[7, 0] = 1.0
    h = torch.zeros(1, C, device=DEV, dtype=torch.float16)
    h[0, 0] = 26.0
    h.requires_grad_()
    loss = linear_cross_entropy(h, W, torch.tensor([7], device=DEV))
    want = math.log1p(299 * math.exp(-26.0))
    assert abs(float(loss) / want - 1) < 1e-5
    dh, = torch.autograd.grad(loss, h, torch.tensor(65536.0, device=DEV))
    want = -65536.0 * 299 / (299 + math.exp(26.0))
    assert abs(float(dh[0, 0]) / want - 1) < 2.0 ** -9


def test_strides_alignment_and_shapes():
    from crb_amd.head import linear_cross_entropy
    T, V, C = 30, 90, 64
    h, W, y = make(T, V, C, torch.bfloat16, 4)
    want = linear_cross_entropy(h, W, y, reduction="none")
    wide = torch.empty(T, C + 24, device=DEV, dtype=h.dtype)
    wide[:, 8:8 + C] = h
    off = torch.empty(V * C + 1, device=DEV, dtype=h.dtype)[1:].view(V, C)
    off.copy_(W)
    col = h.t().contiguous().t()
    for hh in (wide[:, 8:8 + C], wide[:, 8:8 + C].clone(), col):
        for ww in (W, off, W.t().contiguous().t()):
            for yy in (y, torch.stack([y, y], 1)[:, 0]):
                assert torch.equal(linear_cross_entropy(hh, ww, yy, reduction="none"), want)
    cube = linear_cross_entropy(h.view(5, 6, C), W, y.view(5, 6), reduction="none")
    assert cube.shape == (5, 6) and torch.equal(cube.flatten(), want)
    one = linear_cross_entropy(h[3], W, y[3], reduction="none")
    assert one.shape == ()
    assert abs(float(one) - float(want[3])) <= 1e-5
    rows = h[:1].expand(4, C)
    got = linear_cross_entropy(rows, W, y[:1].expand(4), reduction="none")
    assert torch.equal(got, want[:1].expand(4)) or float((got - want[0]).abs().max()) <= 1e-5


def test_frozen_sides():
    from crb_amd.head import linear_cross_entropy, linear_distill
    h, W, y = make(33, 200, 40, torch.float16, 11)
    top = (*teacher(33, 200, 4, 1), None)
    for f in (lambda a, b: linear_cross_entropy(a, b, y), lambda a, b: linear_distill(a, b, top)):
        a, b = h.clone().requires_grad_(), W.clone().requires_grad_()
        dh, dW = torch.autograd.grad(f(a, b), (a, b))
        a = h.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(f(a, W), a)[0], dh)
        b = W.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(f(h, b), b)[0], dW)


def test_repeats_are_bitwise_equal():
    from crb_amd.head import linear_distill
    h, W, _ = make(300, 3000, 128, torch.bfloat16, 12)
    top = (*teacher(300, 3000, 30, 1), None)
    h.requires_grad_(), W.requires_grad_()
    first = None
    for _ in range(3):
        loss = linear_distill(h, W, top)
        out = (loss.detach(), *torch.autograd.grad(loss, (h, W)))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_other_stream():
    from crb_amd.head import linear_cross_entropy
    h, W, y = make(50, 400, 64, torch.float16, 13)
    h.requires_grad_(), W.requires_grad_()

    def step():
        loss = linear_cross_entropy(h, W, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, W)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["xent", "distill", "top"])
def test_graph_replays(kind):
    """The calls in a captured graph, without autograd: every replay on
    changed inputs against the eager call."""
    from crb_amd import kernels
    h, W, y = make(50, 400, 64, torch.float16, 13)
    val, idx = teacher(50, 400, 6, 3)
    one = torch.ones((), device=DEV)

    def step():
        if kind == "top":
            return kernels.top_logits(h, 5)
        if kind == "xent":
            loss, state = kernels.head_xent(h, W, y)
            return (loss, *kernels.head_xent_grad(h, W, y, state, one))
        loss, state = kernels.head_distill(h, W, val, idx)
        return (loss, *kernels.head_distill_grad(h, W, 6, state, one))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        for x in (h, y, val, idx):
            x.copy_(torch.roll(x, 1, 0))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


# ---------------------------------------------------------------------------
# top_logits
# ---------------------------------------------------------------------------
def check_top(x, k, tau=1.0):
    from crb_amd.head import top_logits
    got = top_logits(x, k, temperature=tau)
    # NaN above everything, ties to the lowest index: a stable sort of the negated values
    xd = x.double().cpu()
    val, idx = torch.sort(xd, dim=-1, descending=True, stable=True)
    assert got.idx.dtype == torch.int32 and got.val.dtype == x.dtype
    assert torch.equal(got.idx.cpu().long(), idx[..., :k])
    assert torch.equal(got.val.cpu(), x.cpu().gather(-1, idx[..., :k])) or torch.isnan(got.val).any()
    lse = torch.logsumexp(xd / tau, -1)
    g = got.lse.double().cpu()
    same = (g == lse) | (torch.isnan(g) & torch.isnan(lse))
    # exponentials: relative 2^-23 (1 + |x - max| log2 e) of terms below e^-(x - max): 2^-21
    # and the sum's walk over V terms
    tol = 2.0 ** -21 + 4 * math.sqrt(x.shape[-1]) * 2.0 ** -24 + 2.0 ** -23 * lse.abs()
    assert bool((same | ((g - lse).abs() <= tol)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16],
                         ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 2, 2), (5, 200, 200), (4, 256, 256), (2, 1023, 100),
                                   (7, 1025, 17), (3, 8192, 256), (3, 8193, 256), (2, 9001, 5),
                                   (2, 50272, 64), (3, 131073, 128)])
def test_top_logits(T, V, k, dtype):
    g = torch.Generator().manual_seed(V)
    x = (4 * torch.randn(T, V, generator=g)).to(dtype).to(DEV)
    check_top(x, k)
    check_top(x, k, 2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16],
                         ids=["fp32", "fp16", "bf16"])
def test_top_logits_ties_and_specials(dtype):
    V = 20011
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-2, 2, (12, V), generator=g).to(dtype)       # thousands of ties
    x[1] = 3.0                                                     # one value only
    x[2] = -math.inf
    x[3] = low
    x[4] = low
    x[4, 17000:17003] = 1.0
    x[5, :] = -0.0
    x[5, 5::7] = 0.0
    x[6, 100] = math.inf
    x[6, 200] = math.inf
    x[7, 300] = math.nan
    x[8] = torch.arange(V).to(dtype)                               # ascending
    x[9] = -torch.arange(V).to(dtype)
    x[10, 19999] = math.nan
    x[10, 19998] = -math.nan
    for k in (1, 50, 256):
        check_top(x.to(DEV), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,V,k", [(3, 90001, 200), (520, 1500, 128), (515, 50273, 20)])
def test_top_logits_rows_and_lengths(T, V, k, dtype):
    """Few long rows, many short and many long ones; ties, masked rows and NaN among them."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(T, V, generator=g).to(dtype)
    x[0] = 1.0
    x[1, : V - 3] = -math.inf
    x[2, V // 2] = math.nan
    check_top(x.to(DEV), k)


def test_top_logits_rows_of_any_stride():
    base = torch.randn(6, 30001, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    for a in range(1, 9):
        check_top(base[:, a:a + 20001], 40)
    check_top(base[::2, ::3], 40)
    check_top(base[:1].expand(3, -1), 9)
    check_top(base[:, :600].reshape(2, 3, 600), 9)


# ---------------------------------------------------------------------------
# more than 2^31 elements
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T", [5, 70])
def test_weight_beyond_32_bits(T):
    from crb_amd.head import linear_cross_entropy
    V, C, dtype = 140001, 16384, torch.bfloat16
    g = torch.Generator(device=DEV).manual_seed(T)
    W = torch.empty(V, C, device=DEV, dtype=dtype).normal_(0.0, 1.5 / math.sqrt(C), generator=g)
    h = torch.randn(T, C, device=DEV, generator=g).to(dtype)
    y = torch.randint(0, V, (T,), device=DEV, generator=g)
    y[0], y[1], y[2] = V - 1, V - 2, 0
    W[V - 1] = (0.05 * h[0].float()).to(dtype)                     # rows that are learned or wrong
    W[V - 3] = (0.06 * h[1].float()).to(dtype)
    h.requires_grad_(), W.requires_grad_()
    loss = linear_cross_entropy(h, W, y, reduction="sum")
    dh, dW = torch.autograd.grad(loss, (h, W))
    with torch.no_grad():
        hd, step = h.double(), 20000
        parts = range(0, V, step)
        z = torch.cat([hd @ W[v:v + step].double().t() for v in parts], 1)
        mag = max(float((hd.abs() @ W[v:v + step].double().abs().t()).max()) for v in parts)
        dz0 = 4 * math.sqrt(C) * 2.0 ** -24 * mag
        logq = torch.log_softmax(z, 1)
        rows = -logq.gather(1, y[:, None])[:, 0]
        assert abs(float(loss.double() - rows.sum())) <= float(loss_tol(z, dz0, rows).sum())
        q, one = logq.exp(), torch.zeros_like(logq).scatter_(1, y[:, None], 1.0)
        u = U[dtype]
        e = (u * u if T <= 64 else u) + 2 * dz0 + 2.0 ** -20 * (1 + float(z.abs().max()))
        want, size = torch.zeros_like(hd), torch.zeros_like(hd)
        for v in parts:
            w, d, m = W[v:v + step].double(), (q - one)[:, v:v + step], (q + one)[:, v:v + step]
            want += d @ w
            size += m @ w.abs()
            r = d.t() @ hd
            tol = e * (m.t() @ hd.abs()) + u * r.abs()
            assert float(((dW[v:v + step].double() - r).abs() - tol).max()) <= 0, v
        assert float(((dh.double() - want).abs() - e * size - u * want.abs()).max()) <= 0


def test_top_logits_beyond_32_bits():
    T, V, k = 20000, 120001, 40
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(T, V, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    from crb_amd.head import TopLogits, top_logits
    top = top_logits(x, k)
    for t in (0, 17000, 17897, T - 1):                             # 2^31 lies in row 17895
        val, idx = torch.sort(x[t].double(), descending=True, stable=True)
        lse = float(torch.logsumexp(x[t].double(), 0))
        assert torch.equal(top.idx[t].long(), idx[:k]), t
        assert torch.equal(top.val[t].double(), val[:k]), t
        assert abs(float(top.lse[t]) - lse) <= 2.0 ** -21 + 4 * math.sqrt(V) * 2.0 ** -24 + 2.0 ** -23 * lse
    assert isinstance(top, TopLogits)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    from crb_amd import head, kernels
    from crb_amd._lib import CrbqError
    h, W, y = make(4, 50, 16, torch.float16)
    val, idx = teacher(4, 50, 3, 0)
    bad = [
        lambda: head.linear_cross_entropy(h.float(), W.float(), y),
        lambda: head.linear_cross_entropy(h, W.bfloat16(), y),
        lambda: head.linear_cross_entropy(h, W[:, :8], y),
        lambda: head.linear_cross_entropy(h, W, y[:3]),
        lambda: head.linear_cross_entropy(h, W, y.int()),
        lambda: head.linear_cross_entropy(h, W, y, reduction="max"),
        lambda: head.linear_cross_entropy(h.cpu(), W.cpu(), y.cpu()),
        lambda: head.linear_cross_entropy(h, W, y.cpu()),
        lambda: head.linear_cross_entropy(h[:0], W, y[:0]),
        lambda: head.linear_cross_entropy(h, W, y, scale=0.0),
        lambda: head.linear_cross_entropy(h, W, y, scale=float("nan")),
        lambda: head.linear_distill(h, W, (val, idx.long(), None)),
        lambda: head.linear_distill(h, W, (val[:, :2], idx, None)),
        lambda: head.linear_distill(h, W, (val[:2], idx[:2], None)),
        lambda: head.linear_distill(h, W, (val, idx, None), temperature=0.0),
        lambda: head.linear_distill(h, W, (val, idx, torch.zeros(3, device=DEV))),
        lambda: head.linear_distill(h, W, (val.repeat(1, 100), idx.repeat(1, 100), None)),
        lambda: head.top_logits(h, 17),
        lambda: head.top_logits(h, 0),
        lambda: head.top_logits(h.cpu(), 2),
        lambda: head.top_logits(h.double(), 2),
        lambda: head.top_logits(h, 2, temperature=-1.0),
        lambda: head.top_logits(torch.zeros(2, 400, device=DEV), 257),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(CrbqError):
            f()
            pytest.fail(f"call {i} was not refused")
    _, state = kernels.head_xent(h, W, y)
    for g in (torch.ones(4, device=DEV), torch.ones((), device=DEV).double()):
        with pytest.raises(CrbqError):
            kernels.head_xent_grad(h, W, y, state, g)
    one = torch.ones((), device=DEV)
    for kw in (dict(need_h=False, need_w=False), dict(reduction="none"), dict(reduction="x")):
        with pytest.raises(CrbqError):
            kernels.head_xent_grad(h, W, y, state, one, **kw)
    with pytest.raises(CrbqError):
        kernels.head_xent_grad(h, W, y, state[1:], one)
    with pytest.raises(CrbqError):
        kernels.head_distill_grad(h, W, 3, state, one)
