"""Refusals of the vocabulary projection's loss (host checks only, no GPU needed)."""
import pytest
import torch

import nnb
from nnb import TensorShapeError
from nnb import functional as F
from nnb.autograd import Value

P = 16          # an address that is never dereferenced: the checks come first


def _fwd(rows=4, D=8, V=8, groups=1, x=P, w=P, bias=P, targets=P, ls=0.0, loss=P, norm=P, dx=P, dw=P, dws=0, db=P, dbs=0):
    return nnb.lib().nnb_linear_ce_fwd(None, rows, D, V, groups, x, w, bias, targets, -100, ls, None, loss, norm, dx, dw, dws,
                                       db, dbs)


def test_refusals():
    INV, SHAPE, UNSUP = nnb.NNB_ERR_INVALID, nnb.NNB_ERR_SHAPE, nnb.NNB_ERR_UNSUPPORTED
    for k in ("rows", "D", "V"):
        assert _fwd(**{k: 0}) == SHAPE, k
    assert _fwd(groups=3) == SHAPE and _fwd(groups=0) == SHAPE
    for ls in (-0.1, 1.0, float("nan")):
        assert _fwd(ls=ls) == INV and "label_smoothing" in nnb.last_error()
    for k in ("x", "w", "targets", "loss", "norm"):
        assert _fwd(**{k: None}) == INV, k
    assert _fwd(bias=None) == INV and "bias" in nnb.last_error()
    assert _fwd(groups=2, dws=63) == INV and _fwd(groups=2, dbs=7) == INV and "overlap" in nnb.last_error()
    assert _fwd(V=2 ** 28, D=2 ** 10) == UNSUP and "tensor map" in nnb.last_error()
    assert _fwd(rows=2 ** 31) == UNSUP and _fwd(V=2 ** 31) == UNSUP and _fwd(D=2 ** 31) == UNSUP


def test_scaled_accumulate_refusals():
    def call(*entries, a=P, b=P):
        return nnb.lib().nnb_scaled_accumulate(None, len(entries), (nnb.ScaledGrad * max(1, len(entries)))(*entries), a, b)
    good = nnb.ScaledGrad(P, P, 4, 1, 0, 1)
    assert call() == nnb.NNB_OK
    assert call(nnb.ScaledGrad(None, None, 0, 1, 0, 1), nnb.ScaledGrad(None, None, 4, 0, 0, 1)) == nnb.NNB_OK
    for bad in (nnb.ScaledGrad(None, P, 4, 1, 0, 1), nnb.ScaledGrad(P, None, 4, 1, 0, 1), nnb.ScaledGrad(P, P, 4, 2, 3, 1)):
        assert call(good, bad) == nnb.NNB_ERR_INVALID and "tensor 1" in nnb.last_error()
    assert call(good, a=None) == nnb.NNB_ERR_INVALID and call(good, b=None) == nnb.NNB_ERR_INVALID
    assert call(*[good] * 9) == nnb.NNB_ERR_UNSUPPORTED


@pytest.mark.parametrize("op", [F.linear_cross_entropy, F.linear_token_losses])
def test_function_refusals(op):
    v = lambda *s: Value(torch.zeros(s))      # noqa: E731
    t = torch.zeros(2, 3, dtype=torch.int64)
    good = (v(2, 3, 8), v(5, 8), v(5))
    for x, w, b, tt in ((v(8), *good[1:], t), (good[0], v(5, 7), good[2], t), (good[0], v(8), good[2], t),
                        (*good[:2], v(6), t), (*good, t[:1]), (*good, t.view(-1)), (v(0, 3, 8), *good[1:], t[:0]),
                        (v(2, 3, 0), v(5, 0), good[2], t)):
        with pytest.raises(TensorShapeError):
            op(x, w, b, tt)
    with pytest.raises(ValueError, match="current CUDA device"):
        op(*good, t)


def test_grad_norm_refusals():
    v = lambda *s: Value(torch.zeros(s))      # noqa: E731
    args = (v(2, 3, 8), v(5, 8), v(5), torch.zeros(2, 3, dtype=torch.int64))
    assert F._check_grad_norm(None) is None
    with pytest.raises(ValueError, match="current CUDA device"):
        F._check_grad_norm(torch.ones(1))
    for bad in (torch.ones(2), torch.ones(0)):
        with pytest.raises(TensorShapeError, match="one value"):
            F.linear_cross_entropy(*args, grad_norm=bad)


def test_gradient_buffers_and_groups():
    """Buffers that the current parameter groups do not fit are refused without being marked as written."""
    def leaf(shape, grad):
        v = Value.leaf(torch.zeros(shape), True)
        v.grad = torch.zeros(grad) if grad else None
        return v

    for groups, shape, grad, fits in ((1, (4, 8), (4, 8), True), (1, (4, 8), (1, 32), True), (1, (4, 8), None, True),
                                      (1, (4, 8), (4, 32), False), (4, (4, 8), (4, 8), False), (4, (4, 8), None, False),
                                      (4, (4, 8), (4, 32), True), (4, (4, 8), (4, 4, 8), True), (4, (4, 8), (3, 32), False),
                                      (4, (1,), (4, 1), True)):
        v = leaf(shape, grad)
        with F.param_groups(groups):
            if fits:
                F._check_grouped("op", (None, v, Value(torch.zeros(3))))
                assert F._gstride(v.grad, v) == (v.data.numel() if grad else 0)
            else:
                with pytest.raises(TensorShapeError, match="does not hold"):
                    F._check_grouped("op", (v,))
                if groups > 1 and grad:
                    with pytest.raises(TensorShapeError, match="cannot hold"):
                        F._gstride(v.grad, v)
        assert v.grad_fresh
    v = leaf((4, 8), (4, 32))
    v.grad = torch.zeros(4, 40)[:, :32]                  # views of a flat buffer, as the sharded trainer's
    with F.param_groups(4):
        F._check_grouped("op", (v,))
        assert F._gstride(v.grad, v) == 40
