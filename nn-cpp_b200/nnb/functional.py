"""Differentiable ops over the C ABI, mirroring nn's autograd ops (include/nn/autograd/ops.hpp).

Each function runs the forward kernel(s), returns a Value, and installs a backward rule that
calls the matching backward entry point with the grad_accum `first` flag of every parent that
needs a gradient. Names and argument meaning follow the reference; shape errors raise
nnb.TensorShapeError as the reference throws TensorShapeError.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import os
import weakref

import torch

from . import NORM_LAYER, NORM_RMS, ScaledGrad, TensorShapeError, check, grad_outs, lib
from .autograd import Value, current_stream as _s, empty, running


def _p(t):
    return None if t is None else t.data_ptr()


def _need(v: Value) -> bool:
    return v.requires_grad


# Parameter-gradient groups: with n > 1 the rows of every op's batch are n consecutive groups (the
# data-parallel step's virtual shards) and each parameter's gradient buffer is a [n, size] view; the
# ops then write one gradient per group (the *_grouped entry points).
_GROUPS = 1


@contextlib.contextmanager
def param_groups(n: int):
    global _GROUPS
    old, _GROUPS = _GROUPS, n
    try:
        yield
    finally:
        _GROUPS = old


def _holds_groups(buf, n: int) -> bool:
    """Whether a gradient buffer has room for the current groups' gradients of n elements each."""
    if _GROUPS == 1:
        return buf.numel() == n
    if buf.numel() != _GROUPS * n:
        return False
    return buf.is_contiguous() or (buf.dim() == 2 and buf.shape[0] == _GROUPS and buf.stride(0) >= n and
                                   (n == 1 or buf.stride(1) == 1))


def _gstride(buf, param: Value) -> int:
    """Elements between consecutive groups' gradients in a parameter's gradient buffer."""
    if buf is None:
        return 0
    n = param.data.numel()
    if _GROUPS == 1:
        return n
    if not _holds_groups(buf, n):
        raise TensorShapeError(f"a gradient buffer of shape {tuple(buf.shape)} cannot hold {_GROUPS} groups of {n} elements")
    return buf.stride(0) if buf.dim() == 2 and buf.shape[0] == _GROUPS else n


def _check_grouped(who: str, params) -> None:
    """Refuses a backward rule whose parameters' gradient buffers are not laid out for the current parameter
    groups, before any of them is taken (grad_accum would mark it as written)."""
    for p in params:
        if p is None or not p.requires_grad:
            continue
        n, buf = p.data.numel(), p.grad
        if buf is None or p.grad_borrowed:               # grad_accum makes one like the data
            buf = p.data
        if (_GROUPS > 1 or buf.numel() != n) and not _holds_groups(buf, n):
            raise TensorShapeError(f"{who}: a gradient buffer of shape {tuple(buf.shape)} does not hold {_GROUPS} group(s) of "
                                   f"{n} elements")


# ---- linear (ops.cpp:714-745) -------------------------------------------------------------------

def linear(x: Value, weight: Value, bias: Value) -> Value:
    xs, ws = x.shape, weight.shape
    if len(xs) < 2 or len(ws) != 2 or xs[-1] != ws[1] or bias.shape != (ws[0],):
        raise TensorShapeError("linear: shapes do not agree")
    n, K = ws
    M = x.data.numel() // K
    y = empty(xs[:-1] + (n,))
    pack, mode = _input_pack(weight, M, K)
    check(lib().nnb_linear_fwd_ex(_s(), 1, M, K, n, _p(x.data), _p(weight.data), 0, _p(bias.data), 0, _p(y), 0, None,
                                  _p(pack)))

    def backward(g):
        _linear_backward(g, x, weight, bias, M, K, n, pack, mode)

    return Value.node(y, (x, weight, bias), backward)


def _input_pack(weight: Value, M: int, K: int):
    """A buffer that keeps the forward GEMM's packed copy of the input x [M, K] for the weight
    gradient G^T x (nnb_linear_fwd_ex / nnb_linear_bwd_ex: x is then packed once per step instead of
    twice, with the same bits), when that gradient will be taken and the tensor core can read the
    pack for it (every parameter-gradient group a whole number of 16-row blocks); else (None, 0)."""
    if not _need(weight) or M % _GROUPS or (M // _GROUPS) % 16:
        return None, 0
    mode = lib().nnb_get_math_mode()
    return empty((lib().nnb_linear_pack_bytes(M, K, mode),), dtype=torch.uint8), mode


def linear_multi(x: Value, layers) -> list[Value]:
    """[linear(x, w_i, b_i) for (w_i, b_i) in layers] (the q, k, v projections of a self-attention,
    src/nn/attention.cpp:34). When the weights (and the biases) sit at one constant stride in memory --
    the data-parallel trainer's flat parameter buffer lays each Linear out as weight then bias -- the
    products run as one launch that packs x once (nnb_linear_multi_fwd); otherwise one linear per
    layer. Either way every output has linear's bits and linear's backward."""
    ws = [w for w, _ in layers]
    bs = [b for _, b in layers]
    if not ws or any(w.shape != ws[0].shape for w in ws) or any(b.shape != (ws[0].shape[0],) for b in bs):
        return [linear(x, w, b) for w, b in layers]
    xs = x.shape
    if len(xs) < 2 or len(ws[0].shape) != 2 or xs[-1] != ws[0].shape[1]:
        raise TensorShapeError("linear: shapes do not agree")
    n, K = ws[0].shape
    M = x.data.numel() // K

    def stride(ts):
        if any(not t.data.is_contiguous() for t in ts):
            return None
        d = [t.data.data_ptr() - ts[0].data.data_ptr() for t in ts]
        if len(ts) == 1:
            return 0
        if d[1] <= 0 or d[1] % 4 or any(d[i] != i * d[1] for i in range(len(ts))):
            return None
        return d[1] // 4

    w_stride, b_stride = stride(ws), stride(bs)
    if len(layers) == 1 or w_stride is None or b_stride is None or w_stride < n * K or b_stride < n:
        return [linear(x, w, b) for w, b in layers]
    y = empty((len(layers),) + xs[:-1] + (n,))
    pack, mode = _input_pack(ws[0], M, K)      # x's pack, shared by every product and its backward
    check(lib().nnb_linear_fwd_ex(_s(), len(layers), M, K, n, _p(x.data), _p(ws[0].data), w_stride,
                                  _p(bs[0].data), b_stride, _p(y), M * n, None, _p(pack)))
    outs = []
    for i, (w, b) in enumerate(layers):
        def backward(g, w=w, b=b):
            _linear_backward(g, x, w, b, M, K, n, pack if _need(w) else None, mode)
        outs.append(Value.node(y[i], (x, w, b), backward))
    return outs


def _linear_backward(g, x, weight, bias, M, K, n, pack=None, mode=0):
    """nnb_linear_bwd_ex: nnb_linear_bwd (one group) or nnb_linear_bwd_grouped, the weight gradient
    reading x's pack from the forward when it was kept."""
    dx, fx = x.grad_accum() if _need(x) else (None, 0)
    dw, fw = weight.grad_accum() if _need(weight) else (None, 0)
    db, fb = bias.grad_accum() if _need(bias) else (None, 0)
    check(lib().nnb_linear_bwd_ex(_s(), M, K, n, _GROUPS, _p(g), _p(x.data), _p(pack), mode, _p(weight.data), _p(dx),
                                  fx, _p(dw), _gstride(dw, weight), fw, _p(db), _gstride(db, bias), fb))


def linear_gelu(x: Value, weight: Value, bias: Value) -> Value:
    """gelu(linear(x, w, b)) as one GEMM with the GELU in its epilogue (same bits as the two ops)."""
    xs, ws = x.shape, weight.shape
    if len(xs) < 2 or len(ws) != 2 or xs[-1] != ws[1] or bias.shape != (ws[0],):
        raise TensorShapeError("linear: shapes do not agree")
    n, K = ws
    M = x.data.numel() // K
    y = empty(xs[:-1] + (n,))
    pre = empty(xs[:-1] + (n,))
    pack, mode = _input_pack(weight, M, K)
    check(lib().nnb_linear_fwd_ex(_s(), 1, M, K, n, _p(x.data), _p(weight.data), 0, _p(bias.data), 0, _p(y), 0,
                                  _p(pre), _p(pack)))

    def backward(g):
        dpre = empty(pre.shape)
        check(lib().nnb_gelu_bwd(_s(), pre.numel(), _p(pre), None, _p(g), _p(dpre), 1))
        _linear_backward(dpre, x, weight, bias, M, K, n, pack, mode)

    return Value.node(y, (x, weight, bias), backward)


# ---- matmul / matmul_bt (ops.cpp:683-712, 747-773) ------------------------------------------------

def _sum_to_shape_into(g: torch.Tensor, target: tuple, dst: torch.Tensor, first: int) -> None:
    """accumulate_grad (ops.cpp:110-117) of a gradient with the broadcast shape g.shape into dst (the
    gradient of a value shaped `target`): the leading axes are summed away one at a time (each a
    Tensor::sum(0), src/tensor.cpp:422-455), then every axis where target has 1 and g does not, in
    axis order (sum_to_shape, ops.cpp:35-53); the result is stored (first) or added into dst."""
    cur = g
    while cur.dim() > len(target):
        red = empty(cur.shape[1:])
        check(lib().nnb_column_sum(_s(), cur.shape[0], red.numel(), _p(cur), _p(red), 1))
        cur = red
    for i, t in enumerate(target):
        if t == 1 and cur.shape[i] != 1:
            sh = list(cur.shape)
            red = empty(sh[:i] + [1] + sh[i + 1:])
            check(lib().nnb_reduce_axis_fwd(_s(), math.prod(sh[:i]), sh[i], math.prod(sh[i + 1:]), _p(cur), 0, _p(red)))
            cur = red
    if tuple(cur.shape) != tuple(target):
        raise TensorShapeError("matmul: gradient does not reduce to the operand's shape")
    check(lib().nnb_accumulate(_s(), cur.numel(), _p(cur), _p(dst), first, 0))


def _accumulate_grad(v: Value, grad: torch.Tensor) -> None:
    dst, first = v.grad_accum()
    if tuple(grad.shape) == v.shape:
        check(lib().nnb_accumulate(_s(), grad.numel(), _p(grad), _p(dst), first, 0))
    else:
        _sum_to_shape_into(grad, v.shape, dst, first)


def _sgemm_into(ta, tb, m, n, k, a, lda, b, ldb, c, ldc, first):
    check(lib().nnb_sgemm(_s(), ta, tb, m, n, k, _p(a), lda, _p(b), ldb, _p(c), ldc, 0 if first else 1))


def _matmul_value(a: Value, b: Value, bt: bool) -> Value:
    from . import matmul as tensor_matmul
    y = tensor_matmul(a.data, b.data, False, bt)

    def backward(g):
        if len(b.shape) == 2 and len(a.shape) >= 2:
            # b a plain matrix: a's leading axes fold into M rows and both gradients come from one
            # GEMM each, stored (first) or accumulated (ops.cpp:686-700, 750-761)
            if bt:
                n, K = b.shape
            else:
                K, n = b.shape
            M = a.data.numel() // K
            if _need(a):
                da, fa = a.grad_accum()
                if bt:
                    _sgemm_into(0, 0, M, K, n, g, n, b.data, K, da, K, fa)
                else:
                    _sgemm_into(0, 1, M, K, n, g, n, b.data, n, da, K, fa)
            if _need(b):
                db, fb = b.grad_accum()
                if bt:
                    _sgemm_into(1, 0, n, K, M, g, n, a.data, K, db, K, fb)
                else:
                    _sgemm_into(1, 0, K, n, M, a.data, K, g, n, db, n, fb)
            return
        # batched b: the batched products, then the broadcast axes summed away (ops.cpp:703-710)
        if _need(a):
            _accumulate_grad(a, tensor_matmul(g, b.data, False, not bt))
        if _need(b):
            _accumulate_grad(b, tensor_matmul(g, a.data, True, False) if bt else tensor_matmul(a.data, g, True, False))

    return Value.node(y, (a, b), backward)


def matmul(a: Value, b: Value) -> Value:
    """a @ b with batch axes broadcast (nn::matmul(const Value&, const Value&), ops.cpp:683)."""
    return _matmul_value(a, b, False)


def matmul_bt(a: Value, b: Value) -> Value:
    """a @ b^T over the last two axes (nn::matmul_bt, ops.cpp:747)."""
    return _matmul_value(a, b, True)


def scaled_masked_softmax(x: Value, scale: float, key_padding_mask: torch.Tensor | None = None,
                          causal: bool = False) -> Value:
    """softmax(masked(x * scale)) over the last axis of x [N, H, Tq, Tk] (ops.cpp:1298-1343): padded
    keys (mask 0) get -1e9 and causally hidden keys (j > i) -2e9 before the softmax."""
    if len(x.shape) != 4 or x.shape[3] == 0:
        raise TensorShapeError("scaled_masked_softmax: x must be [N, H, Tq, Tk]")
    N, H, Tq, Tk = x.shape
    if key_padding_mask is not None and key_padding_mask.numel() and tuple(key_padding_mask.shape) != (N, Tk):
        raise TensorShapeError("scaled_masked_softmax: key_padding_mask must be [N, Tk]")
    pad = key_padding_mask if key_padding_mask is not None and key_padding_mask.numel() else None
    y = empty(x.shape)
    check(lib().nnb_scaled_masked_softmax_fwd(_s(), N, H, Tq, Tk, _p(x.data), _p(y), _p(pad), int(causal),
                                              ctypes.c_float(scale)))

    def backward(g):
        if _need(x):
            dx, f = x.grad_accum()
            check(lib().nnb_scaled_masked_softmax_bwd(_s(), N, H, Tq, Tk, _p(y), _p(g), _p(dx), f, _p(pad), int(causal),
                                                      ctypes.c_float(scale)))

    return Value.node(y, (x,), backward)


# ---- elementwise ------------------------------------------------------------------------------

def add(a: Value, b: Value) -> Value:
    """a + b for equal shapes, or b broadcast over a's leading axes (b's shape a suffix of a's)."""
    if a.shape != b.shape and (len(b.shape) > len(a.shape) or a.shape[len(a.shape) - len(b.shape):] != b.shape):
        raise TensorShapeError("add: shapes do not broadcast")
    y = empty(a.shape)
    check(lib().nnb_add_fwd(_s(), a.data.numel(), _p(a.data), _p(b.data), b.data.numel(), _p(y)))
    same = a.shape == b.shape

    def backward(g):
        if _need(a):
            da, f = a.grad_accum()
            check(lib().nnb_accumulate(_s(), g.numel(), _p(g), _p(da), f, 0))
        if _need(b):
            db, f = b.grad_accum()
            if same:
                check(lib().nnb_accumulate(_s(), g.numel(), _p(g), _p(db), f, 0))
            else:   # sum over the broadcast leading axes (sum_to_shape, ops.cpp:35-53)
                rows = g.numel() // b.data.numel()
                check(lib().nnb_column_sum(_s(), rows, b.data.numel(), _p(g), _p(db), f))

    return Value.node(y, (a, b), backward)


def relu(x: Value) -> Value:
    y = empty(x.shape)
    check(lib().nnb_relu_fwd(_s(), x.data.numel(), _p(x.data), _p(y)))

    def backward(g):
        dx, f = x.grad_accum()
        check(lib().nnb_relu_bwd(_s(), g.numel(), _p(x.data), _p(g), _p(dx), f))

    return Value.node(y, (x,), backward)


def gelu(x: Value) -> Value:
    y, th = empty(x.shape), empty(x.shape)
    check(lib().nnb_gelu_fwd(_s(), x.data.numel(), _p(x.data), _p(y), _p(th)))

    def backward(g):
        dx, f = x.grad_accum()
        check(lib().nnb_gelu_bwd(_s(), g.numel(), _p(x.data), _p(th), _p(g), _p(dx), f))

    return Value.node(y, (x,), backward)


def reshape(x: Value, shape) -> Value:
    shape = tuple(shape)
    n = 1
    for d in shape:
        n *= d
    if n != x.data.numel():
        raise TensorShapeError("reshape: element count differs")
    y = x.data.view(shape)

    def backward(g):
        dx, f = x.grad_accum()
        check(lib().nnb_accumulate(_s(), g.numel(), _p(g), _p(dx), f, 0))

    return Value.node(y, (x,), backward)


# ---- normalisation ------------------------------------------------------------------------------

def layernorm(x: Value, gamma: Value, beta: Value, eps: float) -> Value:
    D = x.shape[-1] if x.shape else 0
    if not x.shape or gamma.shape != (D,) or beta.shape != (D,):
        raise TensorShapeError("layernorm: shapes do not agree")
    R = x.data.numel() // D
    y, mean, inv = empty(x.shape), empty((R,)), empty((R,))
    check(lib().nnb_layernorm_fwd(_s(), R, D, _p(x.data), _p(gamma.data), _p(beta.data), ctypes.c_float(eps), _p(y),
                                  _p(mean), _p(inv)))

    def backward(g):
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dg, fg = gamma.grad_accum() if _need(gamma) else (None, 0)
        db, fb = beta.grad_accum() if _need(beta) else (None, 0)
        check(lib().nnb_layernorm_bwd_grouped(_s(), R, D, _GROUPS, _p(g), _p(x.data), _p(gamma.data), _p(mean), _p(inv),
                                              _p(dx), fx, _p(dg), _gstride(dg, gamma), fg, _p(db), _gstride(db, beta),
                                              fb))

    return Value.node(y, (x, gamma, beta), backward)


def _check_buffers(who: str, values, dtype=torch.float32) -> None:
    """Refuses values that are not contiguous buffers of `dtype` on the current CUDA device (None: skipped)."""
    dev = None
    for v in values:
        if v is None:
            continue
        t = v.data if isinstance(v, Value) else v
        at = t.get_device()
        if dev is None and at >= 0:
            dev = torch.cuda.current_device()
        if at != dev:
            raise ValueError(f"{who}: tensors must be on the current CUDA device, one is on {t.device}")
        if t.dtype is not dtype or not t.is_contiguous():
            raise ValueError(f"{who}: tensors must be contiguous {dtype}, one is {t.dtype}")


def residual_norm(x: Value, branch: Value, gamma: Value, beta: Value | None = None, eps: float = 1e-5, *,
                  kind: str = "layer", post_gamma: Value | None = None, post_beta: Value | None = None,
                  gate: Value | None = None, scale: float = 1.0) -> tuple[Value, Value]:
    """(h, y) with h = x + scale * gate * p and y = norm(h; gamma, beta): the residual sum after a block
    and the norm before the next one in one pass. p is the branch, or norm(branch; post_gamma, post_beta)
    when post_gamma is given.

    kind "layer" normalises by mean and variance and needs the betas, "rms" by the mean square and has
    none; `eps` serves both norms. The gate's last axis is the width D; its other axes hold n rows in all
    (none: [D], one row), each for rows / n consecutive rows of x: [D] or [1, D] is a parameter per
    channel (its gradient kept per parameter group as a norm's is), [N, 1, D] one row per sequence of an
    x of [N, T, D], x's own shape one per token.

    The backward runs when h's turn comes, with what reached y held until then. h's whole gradient is formed in
    registers on the way to x's and the branch's: h.grad, whose buffer held only what h's other consumers gave, is
    None after a backward pass."""
    if kind not in ("layer", "rms"):
        raise ValueError('residual_norm: kind must be "layer" or "rms"')
    layer = kind == "layer"
    shape = x.data.shape
    if not shape or 0 in shape or branch.data.shape != shape:
        raise TensorShapeError("residual_norm: x and branch need one non-empty shape")
    D = shape[-1]
    R = x.data.numel() // D
    if layer != (beta is not None) or (post_beta is not None) != (layer and post_gamma is not None):
        raise ValueError("residual_norm: a layer norm needs a beta, an rms norm has none")
    for p in (gamma, beta, post_gamma, post_beta):
        if p is not None and p.data.shape != (D,):
            raise TensorShapeError("residual_norm: norm parameters must be [D]")
    gate_rows = 0
    if gate is not None:
        if not gate.shape or gate.shape[-1] != D or gate.data.numel() == 0 or R % (gate.data.numel() // D):
            raise TensorShapeError("residual_norm: the gate must be rows of D that divide x's rows")
        gate_rows = gate.data.numel() // D
        if gate_rows > 1 and gate_rows % _GROUPS:
            raise TensorShapeError("residual_norm: the gate's rows do not divide into the parameter groups")
    if R % _GROUPS:
        raise TensorShapeError("residual_norm: the rows do not divide into the parameter groups")
    params = (gamma, beta, post_gamma, post_beta, gate if gate_rows == 1 else None)
    if post_gamma is not None or gate_rows == 1 or gamma is beta:
        trained = [id(v) for v in params if v is not None and _need(v)]
        if len(set(trained)) != len(trained):
            raise ValueError("residual_norm: one parameter in two places would share a gradient buffer")
    _check_buffers("residual_norm", (x, branch, gamma, beta, post_gamma, post_beta, gate))
    k = NORM_LAYER if layer else NORM_RMS
    opt = lambda v: None if v is None else v.data.data_ptr()
    h_data, y_data = torch.empty_like(x.data), torch.empty_like(x.data)
    stream_parents = tuple(v for v in (x, branch, post_gamma, post_beta, gate) if v is not None)
    norm_parents = tuple(v for v in (gamma, beta) if v is not None)
    train = any(_need(v) for v in stream_parents + norm_parents)
    stats = x.data.new_empty((R, 4)) if train else None
    check(lib().nnb_residual_norm_fwd(_s(), R, D, gate_rows, k, eps, scale, _p(x.data), _p(branch.data), opt(post_gamma),
                                      opt(post_beta), opt(gate), _p(gamma.data), opt(beta), _p(h_data), _p(y_data),
                                      _p(stats)))
    held = []          # (backward pass, what reached y in it)

    def run(dh, dy):
        _check_grouped("residual_norm", params)

        def out(v, grouped):
            if v is None or not _need(v):
                return None
            buf, first = v.grad_accum()
            return buf.data_ptr(), _gstride(buf, v) if grouped else 0, first
        norm = (out(gamma, True), out(beta, True)) if dy is not None else (None, None)
        grads = grad_outs(out(x, False), out(branch, False), out(post_gamma, True), out(post_beta, True),
                          out(gate, gate_rows == 1), *norm)
        check(lib().nnb_residual_norm_bwd(_s(), R, D, _GROUPS, gate_rows, k, scale, _p(dh), _p(dy), _p(h_data),
                                          _p(branch.data), opt(post_gamma), opt(post_beta), opt(gate), _p(gamma.data),
                                          _p(stats), grads))

    def h_backward(g):
        at, dy = held.pop() if held else (None, None)
        if at is not running():
            dy = None
        node = h_ref()
        run(None if node is not None and node.grad_fresh else g, dy)
        if node is not None:
            node.grad, node.grad_fresh, node.grad_borrowed = None, False, False

    def y_backward(g):
        if h.requires_grad:
            held[:] = [(running(), g)]
        else:
            run(None, g)

    h = Value.node(h_data, stream_parents, h_backward)
    h_ref = weakref.ref(h)
    return h, Value.node(y_data, (h,) + norm_parents, y_backward)


def rmsnorm(x: Value, gamma: Value, eps: float) -> Value:
    """x / sqrt(mean(x^2) + eps) * gamma over the last axis (residual_norm's "rms" norm on its own)."""
    if not x.shape or 0 in x.shape or gamma.shape != (x.shape[-1],):
        raise TensorShapeError("rmsnorm: shapes do not agree")
    _check_buffers("rmsnorm", (x, gamma))
    D = x.shape[-1]
    R = x.data.numel() // D
    if R % _GROUPS:
        raise TensorShapeError("rmsnorm: the rows do not divide into the parameter groups")
    y, stats = empty(x.shape), empty((R, 4))
    check(lib().nnb_residual_norm_fwd(_s(), R, D, 0, NORM_RMS, eps, 1.0, _p(x.data), None, None, None, None, _p(gamma.data),
                                      None, None, _p(y), _p(stats)))

    def backward(g):
        _check_grouped("rmsnorm", (gamma,))
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dg, fg = gamma.grad_accum() if _need(gamma) else (None, 0)
        check(lib().nnb_residual_norm_bwd(_s(), R, D, _GROUPS, 0, NORM_RMS, 1.0, None, _p(g), _p(x.data), None, None, None,
                                          None, _p(gamma.data), _p(stats),
                                          grad_outs((_p(dx), 0, fx), None, None, None, None,
                                                    (_p(dg), _gstride(dg, gamma), fg), None)))

    return Value.node(y, (x, gamma), backward)


def batchnorm(x: Value, weight: Value, bias: Value, eps: float, fuse_relu: bool = False,
              mean_out: torch.Tensor | None = None, var_out: torch.Tensor | None = None) -> Value:
    """batchnorm in training mode (ops.cpp:900-1001); mean_out / var_out receive the batch statistics
    (biased variance), as the reference's Tensor* outputs."""
    if len(x.shape) < 2:
        raise TensorShapeError("batchnorm: needs N and C axes")
    N, C = x.shape[0], x.shape[1]
    S = x.data.numel() // max(1, N * C)
    y = empty(x.shape)
    alive = empty(x.shape, dtype=torch.uint8) if fuse_relu else None
    mean = mean_out if mean_out is not None else empty((C,))
    var = var_out if var_out is not None else empty((C,))
    inv = empty((C,))
    check(lib().nnb_batchnorm_fwd(_s(), N, C, S, _p(x.data), _p(weight.data), _p(bias.data), ctypes.c_float(eps),
                                  int(fuse_relu), _p(y), _p(alive), _p(mean), _p(var), _p(inv)))

    def backward(g):
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dw, fw = weight.grad_accum() if _need(weight) else (None, 0)
        db, fb = bias.grad_accum() if _need(bias) else (None, 0)
        check(lib().nnb_batchnorm_bwd(_s(), N, C, S, _p(g), _p(x.data), _p(weight.data), _p(mean), _p(inv), _p(alive),
                                      _p(dx), fx, _p(dw), fw, _p(db), fb))

    out = Value.node(y, (x, weight, bias), backward)
    out.name = "batchnorm"
    return out


def batchnorm_eval(x: Value, weight: Value, bias: Value, running_mean: torch.Tensor, running_var: torch.Tensor,
                   eps: float, fuse_relu: bool = False) -> Value:
    """Evaluation-mode batch normalisation from the running statistics (batchnorm.cpp:51-55)."""
    if len(x.shape) < 2:
        raise TensorShapeError("batchnorm: needs N and C axes")
    N, C = x.shape[0], x.shape[1]
    S = x.data.numel() // max(1, N * C)
    if len(x.shape) > 4:
        raise TensorShapeError("batchnorm: at most four axes")
    Hs = x.shape[2] if len(x.shape) > 2 else 1      # the axes the parameter gradients sum over, in order
    Ws = x.shape[3] if len(x.shape) > 3 else 1
    y = empty(x.shape)
    alive = empty(x.shape, dtype=torch.uint8) if fuse_relu else None
    check(lib().nnb_batchnorm_eval_fwd(_s(), N, C, S, _p(x.data), _p(running_mean), _p(running_var),
                                       ctypes.c_float(eps), _p(weight.data), _p(bias.data), int(fuse_relu), _p(y),
                                       _p(alive)))

    def backward(g):
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dw, fw = weight.grad_accum() if _need(weight) else (None, 0)
        db, fb = bias.grad_accum() if _need(bias) else (None, 0)
        check(lib().nnb_batchnorm_eval_bwd(_s(), N, C, Hs, Ws, _p(g), _p(x.data), _p(running_mean), _p(running_var),
                                           ctypes.c_float(eps), _p(weight.data), _p(alive), _p(dx), fx, _p(dw), fw,
                                           _p(db), fb))

    return Value.node(y, (x, weight, bias), backward)


# ---- attention (ops.cpp:1226-1296) --------------------------------------------------------------

def attention(q: Value, k: Value, v: Value, heads: int, key_padding_mask: torch.Tensor | None = None,
              causal: bool = False, fused: bool | None = None) -> Value:
    """Multi-head attention (ops.cpp:1226-1296). Head size 64 runs the fused kernels (no
    [N, heads, Tq, Tk] probabilities kept; the backward recomputes them from the row max and sum);
    other head sizes, or fused=False (or NNB_ATTENTION=composed), run the reference's composition:
    head-batched GEMMs around the masked softmax, keeping the probabilities."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or qs[0] != ks[0] or qs[2] != ks[2]:
        raise TensorShapeError("attention: shapes do not agree")
    N, Tq, D = qs
    Tk = ks[1]
    if fused is None:
        fused = FUSED_ATTENTION
    if fused and heads > 0 and lib().nnb_flash_attention_supported(D, heads):
        return _flash_attention(q, k, v, heads, key_padding_mask, causal, N, Tq, Tk, D)
    out, probs = empty((N, Tq, D)), empty((N, heads, Tq, Tk))
    check(lib().nnb_attention_fwd(_s(), N, Tq, Tk, D, heads, _p(q.data), _p(k.data), _p(v.data),
                                  _p(key_padding_mask), int(causal), _p(out), _p(probs)))

    def backward(g):
        # fetched in the reference's order (v, q, k: ops.cpp:1273-1275)
        dv, fv = v.grad_accum() if _need(v) else (None, 0)
        dq, fq = q.grad_accum() if _need(q) else (None, 0)
        dk, fk = k.grad_accum() if _need(k) else (None, 0)
        check(lib().nnb_attention_bwd(_s(), N, Tq, Tk, D, heads, _p(g), _p(q.data), _p(k.data), _p(v.data),
                                      _p(probs), _p(key_padding_mask), int(causal), _p(dq), fq, _p(dk), fk, _p(dv),
                                      fv))

    return Value.node(out, (q, k, v), backward)


FUSED_ATTENTION = os.environ.get("NNB_ATTENTION", "fused").lower() != "composed"


def _flash_attention(q, k, v, heads, key_padding_mask, causal, N, Tq, Tk, D) -> Value:
    out, stats = empty((N, Tq, D)), empty((N, heads, Tq, 2))
    check(lib().nnb_flash_attention_fwd(_s(), N, Tq, Tk, D, heads, _p(q.data), _p(k.data), _p(v.data),
                                        _p(key_padding_mask), int(causal), _p(out), _p(stats)))

    def backward(g):
        dv, fv = v.grad_accum() if _need(v) else (None, 0)
        dq, fq = q.grad_accum() if _need(q) else (None, 0)
        dk, fk = k.grad_accum() if _need(k) else (None, 0)
        check(lib().nnb_flash_attention_bwd(_s(), N, Tq, Tk, D, heads, _p(g), _p(q.data), _p(k.data), _p(v.data),
                                            _p(out), _p(stats), _p(key_padding_mask), int(causal), _p(dq), fq, _p(dk),
                                            fk, _p(dv), fv))

    return Value.node(out, (q, k, v), backward)


# ---- dropout (src/nn/dropout.cpp:20-31) and attention with dropout (src/nn/attention.cpp:36-47) ------

# Batch slice of a data-parallel rank: (rows of the whole batch, first row, end row) while a rank runs
# its rows of a batch whose dropout masks the reference draws over all rows at once.
_BATCH_SLICE = None


@contextlib.contextmanager
def batch_slice(total_rows: int, row_lo: int, row_hi: int):
    """Inside, every dropout mask is drawn as this rank's rows [row_lo, row_hi) of the mask the whole
    batch of total_rows rows would draw (dropout.cpp:20-31 draws row-major from one generator), and
    the generator advances past the whole batch's draws: ranks stay in step and every rank's masks are
    the single-process masks' rows."""
    global _BATCH_SLICE
    old = _BATCH_SLICE
    _BATCH_SLICE = None if (row_lo == 0 and row_hi == total_rows) else (total_rows, row_lo, row_hi)
    try:
        yield
    finally:
        _BATCH_SLICE = old


def dropout_mask(state: torch.Tensor, n: int, p: float) -> torch.Tensor:
    """Dropout::forward's n keep / drop decisions drawn from the device generator `state` (advanced
    in place): (n + 31) // 32 words, bit e % 32 of word e // 32 set when element e is kept. Inside
    batch_slice, n covers this rank's rows and the draw is that slice of the whole batch's."""
    keep = empty(((n + 31) // 32,), dtype=torch.int32, device=state.device)
    if _BATCH_SLICE is None:
        check(lib().nnb_dropout_mask(_s(), _p(state), n, ctypes.c_float(p), _p(keep)))
    else:
        total_rows, lo, hi = _BATCH_SLICE
        if hi <= lo or n % (hi - lo):
            raise ValueError("dropout under batch_slice: the tensor's leading axis is not the rank's rows")
        per_row = n // (hi - lo)
        check(lib().nnb_dropout_mask_slice(_s(), _p(state), per_row * total_rows, per_row * lo, n, ctypes.c_float(p),
                                           _p(keep)))
    return keep


def dropout(x: Value, p: float, state: torch.Tensor) -> Value:
    """x * m, m = 0 with probability p else 1 / (1 - p), the mask drawn from `state` in row-major order."""
    n = x.data.numel()
    keep = dropout_mask(state, n, p)
    y = empty(x.shape, device=x.data.device)
    check(lib().nnb_dropout_apply(_s(), n, ctypes.c_float(p), _p(x.data), _p(keep), _p(y)))

    def backward(g):
        if _need(x):
            dx, f = x.grad_accum()
            check(lib().nnb_dropout_bwd(_s(), n, ctypes.c_float(p), _p(g), _p(keep), _p(dx), f))

    return Value.node(y, (x,), backward)


def attention_dropout(q: Value, k: Value, v: Value, heads: int, key_padding_mask: torch.Tensor | None, causal: bool,
                      p: float, state: torch.Tensor) -> Value:
    """MultiHeadAttention's core with its Dropout active: per head scores = q k^T, scaled_masked_softmax
    (ops.cpp:1298-1343), the dropout mask drawn over the [N, heads, Tq, Tk] weights, then weights v.
    The probabilities and the dropped weights are kept for the backward, as the reference's graph
    keeps them."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or qs[0] != ks[0] or qs[2] != ks[2]:
        raise TensorShapeError("attention: shapes do not agree")
    N, Tq, D = qs
    Tk = ks[1]
    if heads == 0 or D % heads or (causal and Tq != Tk):
        raise TensorShapeError("attention: bad heads or causal shape")
    if key_padding_mask is not None and tuple(key_padding_mask.shape) != (N, Tk):
        raise TensorShapeError("attention: key padding mask must be [N, Tk]")
    keep = dropout_mask(state, N * heads * Tq * Tk, p)
    out, probs, weights = empty((N, Tq, D)), empty((N, heads, Tq, Tk)), empty((N, heads, Tq, Tk))
    check(lib().nnb_attention_dropout_fwd(_s(), N, Tq, Tk, D, heads, _p(q.data), _p(k.data), _p(v.data),
                                          _p(key_padding_mask), int(causal), ctypes.c_float(p), _p(keep), _p(out),
                                          _p(probs), _p(weights)))

    def backward(g):
        dv, fv = v.grad_accum() if _need(v) else (None, 0)
        dq, fq = q.grad_accum() if _need(q) else (None, 0)
        dk, fk = k.grad_accum() if _need(k) else (None, 0)
        check(lib().nnb_attention_dropout_bwd(_s(), N, Tq, Tk, D, heads, _p(g), _p(q.data), _p(k.data), _p(v.data),
                                              _p(probs), _p(weights), ctypes.c_float(p), _p(keep),
                                              _p(key_padding_mask), int(causal), _p(dq), fq, _p(dk), fk, _p(dv), fv))

    return Value.node(out, (q, k, v), backward)


# ---- convolution and pooling ---------------------------------------------------------------------

def conv2d(x: Value, weight: Value, bias: Value, stride: int, padding: int, fuse_relu: bool = False,
           dilation: int = 1, groups: int = 1) -> Value:
    if dilation != 1 or groups != 1:
        if fuse_relu:
            raise ValueError("conv2d: the folded ReLU needs dilation 1 and groups 1 (conv2d.hpp:72)")
        return _conv2d_general(x, weight, bias, stride, padding, dilation, groups)
    if len(x.shape) != 4 or len(weight.shape) != 4:
        raise TensorShapeError("conv2d: needs 4-D input and weight")
    N, Cin, H, W = x.shape
    Cout, wc, kh, kw = weight.shape
    if wc != Cin or bias.shape != (Cout,):
        raise TensorShapeError("conv2d: channels do not agree")
    if stride <= 0 or padding < 0 or kh > H + 2 * padding or kw > W + 2 * padding:
        raise TensorShapeError("conv2d: bad window")
    ho, wo = (H + 2 * padding - kh) // stride + 1, (W + 2 * padding - kw) // stride + 1
    y = empty((N, Cout, ho, wo))
    alive = empty((N, Cout, ho, wo), dtype=torch.uint8) if fuse_relu else None
    check(lib().nnb_conv2d_fwd(_s(), N, Cin, H, W, Cout, kh, kw, stride, padding, _p(x.data), _p(weight.data),
                               _p(bias.data), int(fuse_relu), _p(y), _p(alive)))

    def backward(g):
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dw, fw = weight.grad_accum() if _need(weight) else (None, 0)
        db, fb = bias.grad_accum() if _need(bias) else (None, 0)
        check(lib().nnb_conv2d_bwd(_s(), N, Cin, H, W, Cout, kh, kw, stride, padding, _p(g), _p(x.data),
                                   _p(weight.data), _p(alive), _p(dx), fx, _p(dw), fw, _p(db), fb))

    return Value.node(y, (x, weight, bias), backward)


def _conv2d_general(x: Value, weight: Value, bias: Value, stride: int, padding: int, dilation: int,
                    groups: int) -> Value:
    """conv2d with dilation / groups (ops.cpp:1525-1607): per sample and group, im2col + GEMM."""
    if len(x.shape) != 4 or len(weight.shape) != 4:
        raise TensorShapeError("conv2d: needs 4-D input and weight")
    N, Cin, H, W = x.shape
    Cout, Cg, kh, kw = weight.shape
    if bias.shape != (Cout,) or groups <= 0 or dilation <= 0 or stride <= 0 or padding < 0 or Cin % groups \
            or Cout % groups or Cg != Cin // groups:
        raise TensorShapeError("conv2d: shapes do not agree")
    ekh, ekw = dilation * (kh - 1) + 1, dilation * (kw - 1) + 1
    if ekh > H + 2 * padding or ekw > W + 2 * padding:
        raise TensorShapeError("conv2d: bad window")
    ho, wo = (H + 2 * padding - ekh) // stride + 1, (W + 2 * padding - ekw) // stride + 1
    y = empty((N, Cout, ho, wo))
    check(lib().nnb_conv2d_ex_fwd(_s(), N, Cin, H, W, Cout, kh, kw, stride, padding, dilation, groups, _p(x.data),
                                  _p(weight.data), _p(bias.data), _p(y)))

    def backward(g):
        dx, fx = x.grad_accum() if _need(x) else (None, 0)
        dw, fw = weight.grad_accum() if _need(weight) else (None, 0)
        db, fb = bias.grad_accum() if _need(bias) else (None, 0)
        check(lib().nnb_conv2d_ex_bwd(_s(), N, Cin, H, W, Cout, kh, kw, stride, padding, dilation, groups, _p(g),
                                      _p(x.data), _p(weight.data), _p(dx), fx, _p(dw), fw, _p(db), fb))

    return Value.node(y, (x, weight, bias), backward)


def conv2d_relu(x: Value, weight: Value, bias: Value, stride: int, padding: int) -> Value:
    return conv2d(x, weight, bias, stride, padding, fuse_relu=True)


def maxpool2d(x: Value, kernel_size: int, stride: int) -> Value:
    if len(x.shape) != 4 or kernel_size == 0 or stride == 0:
        raise TensorShapeError("maxpool2d: bad input")
    N, C, H, W = x.shape
    if kernel_size > H or kernel_size > W:
        raise TensorShapeError("maxpool2d: window larger than the input")
    ho, wo = (H - kernel_size) // stride + 1, (W - kernel_size) // stride + 1
    y = empty((N, C, ho, wo))
    arg = empty((N, C, ho, wo), dtype=torch.int32)
    check(lib().nnb_maxpool2d_fwd(_s(), N, C, H, W, kernel_size, stride, _p(x.data), _p(y), _p(arg)))

    def backward(g):
        dx, f = x.grad_accum()
        check(lib().nnb_maxpool2d_bwd(_s(), N, C, H, W, kernel_size, stride, _p(g), _p(arg), _p(dx), f))

    return Value.node(y, (x,), backward)


def avgpool2d(x: Value, kernel_size: int, stride: int) -> Value:
    """avgpool2d (ops.cpp:1707-1772)."""
    if len(x.shape) != 4 or kernel_size == 0 or stride == 0:
        raise TensorShapeError("avgpool2d: bad input")
    N, C, H, W = x.shape
    if kernel_size > H or kernel_size > W:
        raise TensorShapeError("avgpool2d: window larger than the input")
    ho, wo = (H - kernel_size) // stride + 1, (W - kernel_size) // stride + 1
    y = empty((N, C, ho, wo))
    check(lib().nnb_avgpool2d_fwd(_s(), N, C, H, W, kernel_size, stride, _p(x.data), _p(y)))

    def backward(g):
        if _need(x):
            dx, fx = x.grad_accum()
            check(lib().nnb_avgpool2d_bwd(_s(), N, C, H, W, kernel_size, stride, _p(g), _p(dx), fx))

    return Value.node(y, (x,), backward)


def _reduce_axis(x: Value, axis: int, keepdim: bool, average: bool) -> Value:
    """sum / mean over one axis (reduce_axis, ops.cpp:284-376)."""
    shape = list(x.shape)
    nd = len(shape)
    if axis < -nd or axis >= nd:
        raise IndexError("reduce over an axis out of range")     # the reference throws TensorIndexError
    ax = axis + nd if axis < 0 else axis
    n = shape[ax]
    if n == 0:
        raise TensorShapeError("reduce over an empty axis")
    outer = math.prod(shape[:ax])
    inner = math.prod(shape[ax + 1:])
    out_shape = [d for i, d in enumerate(shape) if i != ax] if not keepdim else \
        [1 if i == ax else d for i, d in enumerate(shape)]
    y = empty(tuple(out_shape) if out_shape else (1,))
    check(lib().nnb_reduce_axis_fwd(_s(), outer, n, inner, _p(x.data), int(average), _p(y)))

    def backward(g):
        if _need(x):
            dx, fx = x.grad_accum()
            check(lib().nnb_reduce_axis_bwd(_s(), outer, n, inner, _p(g), int(average), _p(dx), fx))

    return Value.node(y, (x,), backward)


def sum(x: Value, axis: int, keepdim: bool = False) -> Value:      # noqa: A001 - the reference's name
    return _reduce_axis(x, axis, keepdim, False)


def mean(x: Value, axis: int, keepdim: bool = False) -> Value:
    return _reduce_axis(x, axis, keepdim, True)


# ---- embedding and losses -----------------------------------------------------------------------

def embedding(weight: Value, ids: torch.Tensor) -> Value:
    """ids: a CUDA int64 tensor of any shape; returns ids.shape + (D,) (ops.cpp:1991-2015)."""
    if len(weight.shape) != 2:
        raise TensorShapeError("embedding: weight must be 2-D")
    V, D = weight.shape
    cnt = ids.numel()
    out = empty(tuple(ids.shape) + (D,))
    check(lib().nnb_embedding_fwd(_s(), V, D, _p(weight.data), _p(ids), cnt, _p(out)))

    def backward(g):
        dw, f = weight.grad_accum()
        if _GROUPS > 1:
            check(lib().nnb_embedding_bwd_grouped(_s(), V, D, _GROUPS, _p(ids), cnt, _p(g), _p(dw), _gstride(dw, weight),
                                                  f))
        else:
            check(lib().nnb_embedding_bwd(_s(), V, D, _p(ids), cnt, _p(g), _p(dw), f))

    return Value.node(out, (weight,), backward)


def cross_entropy_loss(logits: Value, targets: torch.Tensor) -> Value:
    if len(logits.shape) != 2 or targets.dim() != 1 or targets.numel() != logits.shape[0]:
        raise TensorShapeError("cross_entropy_loss: shapes do not agree")
    N, C = logits.shape
    sm, loss, norm = empty((N, C)), empty((1,)), empty((1,))
    check(lib().nnb_cross_entropy_fwd(_s(), N, C, _p(logits.data), _p(targets), _p(sm), _p(loss), _p(norm)))

    def backward(g):
        dl, f = logits.grad_accum()
        check(lib().nnb_cross_entropy_bwd(_s(), N, C, _p(sm), _p(targets), _p(g), _p(norm), _p(dl), f))

    return Value.node(loss, (logits,), backward)


def sequence_cross_entropy(logits: Value, targets: torch.Tensor, ignore_index: int = -100,
                           label_smoothing: float = 0.0, grad_norm: torch.Tensor | None = None) -> Value:
    """grad_norm: a device scalar used by the backward pass in place of 1/(positions counted here),
    e.g. 1/(positions of the global batch) when this call sees one rank's part of it."""
    if len(logits.shape) != 3 or tuple(targets.shape) != logits.shape[:2]:
        raise TensorShapeError("sequence_cross_entropy: shapes do not agree")
    N, T, V = logits.shape
    P = N * T
    sm, loss, norm = empty((P, V)), empty((1,)), empty((1,))
    check(lib().nnb_sequence_ce_fwd(_s(), P, V, _p(logits.data), _p(targets), ignore_index,
                                    ctypes.c_float(label_smoothing), _p(sm), _p(loss), _p(norm)))

    def backward(g):
        dl, f = logits.grad_accum()
        check(lib().nnb_sequence_ce_bwd(_s(), P, V, _p(sm), _p(targets), ignore_index, ctypes.c_float(label_smoothing),
                                        _p(g), _p(norm if grad_norm is None else grad_norm), _p(dl), f))

    return Value.node(loss, (logits,), backward)


def _linear_ce_args(who: str, x, weight, bias, targets):
    """Shapes and buffers of a vocabulary projection's loss: (P, D, V)."""
    xs, ws = x.shape, weight.shape
    if len(xs) < 2 or len(ws) != 2 or xs[-1] != ws[1] or 0 in xs or 0 in ws or (bias is not None and bias.shape != ws[:1]):
        raise TensorShapeError(f"{who}: shapes do not agree")
    if tuple(targets.shape) != xs[:-1]:
        raise TensorShapeError(f"{who}: targets must have x's shape without its last axis")
    _check_buffers(who, (x, weight, bias))
    _check_buffers(who, (targets,), torch.int64)
    return x.data.numel() // xs[-1], xs[-1], ws[0]


def _check_grad_norm(grad_norm) -> None:
    if grad_norm is not None and grad_norm.numel() != 1:
        raise TensorShapeError("linear_cross_entropy: grad_norm must hold one value")
    _check_buffers("linear_cross_entropy", (grad_norm,))


def linear_cross_entropy(x: Value, weight: Value, bias: Value | None, targets: torch.Tensor, ignore_index: int = -100,
                         label_smoothing: float = 0.0, grad_norm: torch.Tensor | None = None) -> Value:
    """sequence_cross_entropy(linear(x, weight, bias), targets) without keeping the logits: x [..., D],
    weight [V, D], bias [V] or None, targets (int64, on the device) of x's leading shape. The mean loss over
    the targets that are not ignore_index, label smoothing and grad_norm as sequence_cross_entropy's.

    The rows go through in pieces; where a gradient is needed it is computed with the loss, from the same
    logits, and the backward only scales it (nnb_linear_ce_fwd, include/nnb.h): a second copy of the gradients,
    per parameter group, is kept until the graph goes, also for a loss that is only read. For inputs that need
    none, see linear_token_losses. The backward runs in the parameter groups of the forward."""
    _check_grad_norm(grad_norm)
    P, D, V = _linear_ce_args("linear_cross_entropy", x, weight, bias, targets)
    parents = (x, weight) if bias is None else (x, weight, bias)
    params = any(_need(v) for v in parents[1:])
    groups = _GROUPS if params else 1
    if P % groups:
        raise TensorShapeError("linear_cross_entropy: the rows do not divide into the parameter groups")
    # the gradients wanted and the loss' norm in one buffer, each on a 256-byte boundary
    sizes = [n if v is not None and _need(v) else 0 for v, n in ((x, P * D), (weight, groups * V * D), (bias, groups * V))]
    starts, total = [], 64
    for n in sizes:
        starts.append(total)
        total += -(-n // 64) * 64
    loss, kept = x.data.new_empty(1), x.data.new_empty(total)
    norm_at = kept.data_ptr()
    at = [norm_at + 4 * lo if n else None for lo, n in zip(starts, sizes)]
    check(lib().nnb_linear_ce_fwd(_s(), P, D, V, groups, _p(x.data), _p(weight.data), None if bias is None else _p(bias.data),
                                  _p(targets), ignore_index, label_smoothing, None, _p(loss), norm_at, at[0], at[1],
                                  0, at[2], 0))

    def backward(g):
        if params and groups != _GROUPS:
            raise ValueError(f"linear_cross_entropy: the forward kept gradients for {groups} parameter group(s), the "
                             f"backward runs in {_GROUPS}")
        if params:
            _check_grouped("linear_cross_entropy", parents[1:])
        runs = (1, groups, groups)
        if any(n and n != v.data.numel() * k for v, n, k in zip((x, weight, bias), sizes, runs)):
            raise TensorShapeError("linear_cross_entropy: an operand changed its size since the forward")
        grads = []
        for v, n, lo, runs_of in zip((x, weight, bias), sizes, starts, runs):
            if n:
                buf, f = v.grad_accum()
                grads.append(ScaledGrad(kept.data_ptr() + 4 * lo, buf.data_ptr(), n // runs_of, runs_of,
                                        _gstride(buf, v) if runs_of > 1 else 0, f))
        k = norm_at if grad_norm is None else grad_norm.data_ptr()
        # (one launch, unless x is the weight itself: then its two gradients are added one after the other)
        for part in ([grads] if x is not weight else [[e] for e in grads]):
            check(lib().nnb_scaled_accumulate(_s(), len(part), (ScaledGrad * len(part))(*part), _p(g), k))

    return Value.node(loss, parents, backward)


def linear_token_losses(x: Value, weight: Value, bias: Value | None, targets: torch.Tensor, ignore_index: int = -100,
                        label_smoothing: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(each target's loss, their mean) of linear_cross_entropy, for evaluation: plain tensors, of the
    targets' shape (0 where the target is ignore_index) and [1], with no gradients and nothing kept."""
    P, D, V = _linear_ce_args("linear_token_losses", x, weight, bias, targets)
    losses, loss, norm = empty(tuple(targets.shape)), empty((1,)), empty((1,))
    check(lib().nnb_linear_ce_fwd(_s(), P, D, V, 1, _p(x.data), _p(weight.data), None if bias is None else _p(bias.data),
                                  _p(targets), ignore_index, label_smoothing, _p(losses), _p(loss), _p(norm), None, None, 0,
                                  None, 0))
    return losses, loss
