"""Refusals of the parameter-list AdamW step (host checks only, no GPU needed)."""
import ctypes

import pytest
import torch

import nnb
from nnb import nn
from nnb.autograd import Value


def _arrays(count, n=4, skip=()):
    p = ctypes.c_void_p * count
    ptrs = {k: p(*([16] * count)) for k in "wgmvab"}      # never dereferenced: the checks come first
    for k, i in skip:
        ptrs[k][i] = None
    return (ctypes.c_size_t * count)(*([n] * count)), ptrs


def _step32(count, sizes, p, step=1):
    return nnb.lib().nnb_adamw_multi_step(None, count, sizes, p["w"], p["g"], p["m"], p["v"], 1e-3, 0.9, 0.999, 1e-8,
                                          0.0, step)


def _step8(count, sizes, p, step=1):
    return nnb.lib().nnb_adamw8_multi_step(None, count, sizes, p["w"], p["g"], p["m"], p["v"], p["a"], p["b"], 1e-3, 0.9,
                                           0.999, 1e-8, 0.0, step)


@pytest.mark.parametrize("step", [_step32, _step8])
def test_list_refusals(step):
    sizes, p = _arrays(3)
    assert step(3, sizes, p, 0) == nnb.NNB_ERR_INVALID and "step counts from 1" in nnb.last_error()
    for missing in ("w", "m", "v") + (("a", "b") if step is _step8 else ()):
        sizes, p = _arrays(3, skip=[(missing, 1)])
        assert step(3, sizes, p) == nnb.NNB_ERR_INVALID and "tensor 1" in nnb.last_error()
    sizes, p = _arrays(3)
    assert step(3, None, p) == nnb.NNB_ERR_INVALID
    sizes, p = _arrays(2, n=2 ** 43)
    assert step(2, sizes, p) == nnb.NNB_ERR_UNSUPPORTED
    sizes, p = _arrays(2)
    assert step(0, sizes, p) == nnb.NNB_OK                   # an empty list does nothing
    sizes, p = _arrays(2, n=0, skip=[("w", 0), ("m", 1)])
    assert step(2, sizes, p) == nnb.NNB_OK                   # nor do empty tensors


def test_moments_refusals():
    f = nnb.lib().nnb_adamw8_moments
    assert f(None, 0, *([None] * 6)) == nnb.NNB_OK
    for i in range(6):
        assert f(None, 8, *[None if j == i else 16 for j in range(6)]) == nnb.NNB_ERR_INVALID


def test_optimizer_refusals():
    with pytest.raises(ValueError, match="state_bits"):
        nn.AdamW([], state_bits=16)
    with pytest.raises(ValueError, match="current CUDA device"):
        nn.AdamW([Value(torch.zeros(4))])


def test_buffers_that_share_memory():
    apart = nn._apart
    assert apart([], []) and apart([64], [16]) and apart([128, 64], [4, 16]) and apart([64, 64, 96], [0, 8, 4])
    assert not apart([64, 64], [4, 4]) and not apart([124, 64], [4, 16]) and not apart([64, 80, 400], [100, 1, 3])
