"""Host side of the output-head entry points: sizes, and every refusal before
device work (no GPU needed: the pointers are never read)."""
import ctypes

import pytest
import torch

P = [ctypes.c_void_p(0x7f0000100000 + (i << 24)) for i in range(10)]
ARG, WS = -1, -3


def lib():
    from crb_amd import _lib
    return _lib.load()


def xent(**kw):
    a = dict(h=P[0], ldh=64, W=P[1], ldw=64, dtype=1, T=4, V=100, C=64, labels=P[2], ignore=-100,
             scale=1.0, red=1, loss=P[3], state=P[4], ws=None, nws=0, s=None)
    a.update(kw)
    return lib().crbq_head_xent(*a.values())


def xent_grad(**kw):
    a = dict(h=P[0], ldh=64, W=P[1], ldw=64, dtype=1, T=4, V=100, C=64, labels=P[2], scale=1.0,
             red=1, state=P[4], g=P[3], dh=P[5], ldd=64, dW=P[6], ldo=64, ws=None, nws=0, s=None)
    a.update(kw)
    return lib().crbq_head_xent_grad(*a.values())


def distill(**kw):
    a = dict(h=P[0], ldh=64, W=P[1], ldw=64, dtype=1, T=4, V=100, C=64, val=P[2], vd=0, ldv=8,
             idx=P[3], ldi=8, k=8, lse=None, scale=1.0, temp=1.0, red=1, loss=P[4], state=P[5],
             ws=None, nws=0, s=None)
    a.update(kw)
    return lib().crbq_head_distill(*a.values())


def distill_grad(**kw):
    a = dict(h=P[0], ldh=64, W=P[1], ldw=64, dtype=1, T=4, V=100, C=64, k=8, scale=1.0, temp=1.0,
             red=0, state=P[4], g=P[3], dh=P[5], ldd=64, dW=P[6], ldo=64, ws=None, nws=0, s=None)
    a.update(kw)
    return lib().crbq_head_distill_grad(*a.values())


def top(**kw):
    a = dict(x=P[0], dtype=1, T=4, V=100, ld=100, k=8, temp=1.0, val=P[1], idx=P[2], lse=P[3],
             s=None)
    a.update(kw)
    return lib().crbq_top_logits(*a.values())


ODD = ctypes.c_void_p(0x7f0000100002)
MATRIX = [dict(h=None), dict(W=None), dict(h=ODD), dict(W=ODD), dict(ldh=63), dict(ldh=56),
          dict(ldw=68), dict(ldw=1 << 22), dict(dtype=0), dict(dtype=3), dict(T=0), dict(V=0),
          dict(C=0), dict(C=60), dict(C=4), dict(T=1 << 22), dict(V=1 << 28),
          dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(ws=ODD, nws=1 << 40)]


@pytest.mark.parametrize("call", [xent, xent_grad, distill, distill_grad])
def test_matrix_refusals(call):
    for bad in MATRIX:
        assert call(**bad) == ARG, bad
    assert call() == WS                              # arguments fine, no workspace


def test_other_refusals():
    for bad in (dict(labels=None), dict(loss=None), dict(state=None), dict(red=3), dict(red=-1)):
        assert xent(**bad) == ARG, bad
    for call in (xent_grad, distill_grad):
        for bad in (dict(state=None), dict(g=None), dict(dh=None, dW=None), dict(dh=ODD),
                    dict(dW=ODD), dict(ldd=60), dict(ldo=8), dict(state=ODD), dict(red=3)):
            assert call(**bad) == ARG, bad
        assert call(dh=None) == WS and call(dW=None) == WS
    assert xent_grad(labels=None) == ARG
    for bad in (dict(val=None), dict(idx=None), dict(loss=None), dict(state=None), dict(k=0),
                dict(k=257), dict(ldv=7), dict(ldi=7), dict(temp=0.0), dict(temp=float("nan")),
                dict(vd=3), dict(red=7)):
        assert distill(**bad) == ARG, bad
    for bad in (dict(k=0), dict(k=257), dict(temp=-1.0)):
        assert distill_grad(**bad) == ARG, bad
    for bad in (dict(x=None), dict(val=None), dict(idx=None), dict(lse=None), dict(dtype=5),
                dict(T=0), dict(V=0), dict(ld=99), dict(k=0), dict(k=101), dict(V=400, ld=400, k=257),
                dict(temp=0.0), dict(V=1 << 31, ld=1 << 31)):
        assert top(**bad) == ARG, bad


def test_sizes():
    l = lib()
    assert l.crbq_head_state_floats(0, 0) == 0 and l.crbq_head_state_floats(5, 257) == 0
    assert l.crbq_head_workspace_size(0, 5, 8, 0, 0) == 0
    for T in (1, 16, 17, 64, 65, 2047, 65536):
        for V in (1, 200, 50272, 128256):
            for C in (8, 1000, 4096):
                fwd = l.crbq_head_workspace_size(T, V, C, 0, 0)
                lists = l.crbq_head_workspace_size(T, V, C, 64, 0)
                grad = l.crbq_head_workspace_size(T, V, C, 0, 1)
                assert 0 < fwd <= lists and grad > 0
                # the logits are not kept: well below T x V numbers where there are many
                if T >= 2047 and V >= 50272:
                    assert lists < T * V and grad < max(2 * T * 8192, 1 << 28) + 40 * T * C * 4


def test_cpu_tensors_are_refused():
    from crb_amd import head
    from crb_amd._lib import CrbqError
    h, W = torch.zeros(3, 16).half(), torch.zeros(9, 16).half()
    with pytest.raises(CrbqError):
        head.linear_cross_entropy(h, W, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(CrbqError):
        head.linear_distill(h, W, (torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), None))
    with pytest.raises(CrbqError):
        head.top_logits(h, 2)
