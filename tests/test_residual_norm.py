"""Refusals of the residual norm (host checks only, no GPU needed)."""
import pytest
import torch

import nnb
from nnb import NORM_LAYER, NORM_RMS, TensorShapeError, grad_outs
from nnb import functional as F
from nnb.autograd import Value, backward

P = 16          # an address that is never dereferenced: the checks come first


def _fwd(R=4, D=8, gate_rows=0, kind=NORM_LAYER, x=P, branch=P, pg=None, pb=None, gate=None, gamma=P, beta=P, h=P, y=P,
         stats=P):
    return nnb.lib().nnb_residual_norm_fwd(None, R, D, gate_rows, kind, 1e-5, 1.0, x, branch, pg, pb, gate, gamma, beta, h,
                                           y, stats)


def _bwd(R=4, D=8, groups=1, gate_rows=0, kind=NORM_LAYER, dh=P, dy=P, h=P, branch=P, pg=None, pb=None, gate=None, gamma=P,
         stats=P, outs=()):
    outs = dict(outs)
    names = ("dx", "dbranch", "dpost_gamma", "dpost_beta", "dgate", "dgamma", "dbeta")
    return nnb.lib().nnb_residual_norm_bwd(None, R, D, groups, gate_rows, kind, 1.0, dh, dy, h, branch, pg, pb, gate, gamma,
                                           stats, grad_outs(*[outs.get(n) for n in names]))


def test_forward_refusals():
    INV, SHAPE, UNSUP = nnb.NNB_ERR_INVALID, nnb.NNB_ERR_SHAPE, nnb.NNB_ERR_UNSUPPORTED
    assert _fwd(kind=2) == INV and "unknown norm" in nnb.last_error()
    assert _fwd(D=0) == SHAPE
    assert _fwd(D=16385) == UNSUP and "16384" in nnb.last_error()
    assert _fwd(R=2 ** 31) == UNSUP
    for name in ("x", "branch", "gamma", "beta", "h", "y"):        # (branch and h go together)
        assert _fwd(**{name: None}) == INV, name
    assert _fwd(branch=None, h=None, gate=P, gate_rows=1) == INV and _fwd(branch=None, h=None, pg=P, pb=P) == INV
    assert _fwd(kind=NORM_RMS) == INV                                  # an rms norm with a beta
    assert _fwd(pg=P) == INV and _fwd(pb=P) == INV                     # half a layer norm after the block
    assert _fwd(kind=NORM_RMS, beta=None, pg=P, pb=P) == INV
    assert _fwd(gate=P, gate_rows=3) == SHAPE and _fwd(gate=P, gate_rows=0) == SHAPE
    assert _fwd(stats=8) == INV and "aligned" in nnb.last_error()
    assert _fwd(R=0) == nnb.NNB_OK


def test_backward_refusals():
    INV, SHAPE, UNSUP = nnb.NNB_ERR_INVALID, nnb.NNB_ERR_SHAPE, nnb.NNB_ERR_UNSUPPORTED
    assert _bwd(kind=-1) == INV and _bwd(D=0) == SHAPE and _bwd(D=20000) == UNSUP
    assert _bwd(groups=0) == SHAPE and _bwd(groups=3) == SHAPE
    assert _bwd(R=2 ** 18, groups=2 ** 17) == UNSUP
    assert _bwd(dh=None, dy=None) == INV and _bwd(h=None) == INV and _bwd(stats=None) == INV and _bwd(gamma=None) == INV
    assert _bwd(gate=P, gate_rows=2, branch=None) == INV
    assert _bwd(gate=P, gate_rows=3) == SHAPE
    assert _bwd(gate=P, gate_rows=2, groups=4) == SHAPE               # a span that straddles groups
    assert _bwd(kind=NORM_RMS, outs={"dbeta": (P, 0, 1)}) == INV
    assert _bwd(outs={"dpost_gamma": (P, 0, 1)}) == INV and _bwd(outs={"dgate": (P, 0, 1)}) == INV
    assert _bwd(groups=2, outs={"dgamma": (P, 7, 1)}) == INV and "overlap" in nnb.last_error()
    assert _bwd(outs={"dgamma": (P, 0, 1), "dbeta": (P, 0, 1)}) == INV and "share" in nnb.last_error()
    assert _bwd(R=0) == nnb.NNB_OK


def _values(*shapes):
    return [Value(torch.zeros(s)) for s in shapes]


def test_function_refusals():
    x, b, g, be = _values((2, 3, 8), (2, 3, 8), (8,), (8,))
    with pytest.raises(ValueError, match="kind"):
        F.residual_norm(x, b, g, be, kind="group")
    with pytest.raises(ValueError, match="beta"):
        F.residual_norm(x, b, g)
    with pytest.raises(ValueError, match="beta"):
        F.residual_norm(x, b, g, be, post_gamma=g)
    with pytest.raises(ValueError, match="beta"):
        F.residual_norm(x, b, g, be, kind="rms")
    with pytest.raises(ValueError, match="beta"):
        F.residual_norm(x, b, g, be, post_beta=be)
    bad, narrow, empty = _values((2, 3, 9), (7,), (0, 8))
    for args, kw in (((x, bad, g, be), {}), ((x, b, narrow, be), {}), ((x, b, g, narrow), {}), ((empty, empty, g, be), {}),
                     ((x, b, g, be), {"gate": narrow}), ((x, b, g, be), {"gate": _values((4, 8))[0]}),
                     ((x, b, g, be), {"gate": empty})):
        with pytest.raises(TensorShapeError):
            F.residual_norm(*args, **kw)
    with pytest.raises(ValueError, match="current CUDA device"):
        F.residual_norm(x, b, g, be)


def test_one_parameter_in_two_places():
    """Refused when the sum is built, before any gradient buffer is taken; where no gradient is wanted the check of
    the buffers is the next."""
    x, b, be, be2 = _values((2, 3, 8), (2, 3, 8), (8,), (8,))
    for train, match in ((True, "two places"), (False, "current CUDA device")):
        g, row = Value.leaf(torch.ones(8), train), Value.leaf(torch.ones(1, 8), train)
        with pytest.raises(ValueError, match=match):
            F.residual_norm(x, b, g, be, post_gamma=g, post_beta=be2)
        with pytest.raises(ValueError, match=match):
            F.residual_norm(x, b, g, kind="rms", gate=g)
        with pytest.raises(ValueError, match="current CUDA device"):
            F.residual_norm(x, b, g, kind="rms", gate=row)


def test_rmsnorm_refusals():
    x, g = _values((3, 8), (8,))
    for args in ((x, _values((7,))[0], 1e-5), (_values((0, 8))[0], g, 1e-5)):
        with pytest.raises(TensorShapeError):
            F.rmsnorm(*args)
    with pytest.raises(ValueError, match="current CUDA device"):
        F.rmsnorm(x, g, 1e-5)


def test_backward_from_several_roots_refusals():
    a, b = _values((2,), (1,))
    with pytest.raises(ValueError, match="as many seeds"):
        backward((a,), ())
    with pytest.raises(ValueError, match="twice"):
        backward((b, b), (None, None))
    with pytest.raises(ValueError, match="single-element"):
        backward((b, a), (None, None))
    with pytest.raises(ValueError, match="element count"):
        backward((a,), (torch.zeros(3),))
    with pytest.raises(ValueError, match="type and device"):
        backward((a,), (torch.zeros(2, dtype=torch.float64),))
