"""The vocabulary projection's loss and gradients against their definition in 64 bits.

E = 2^-24 is half a step of fp32. The bounds start from the product's. An operand goes in as two fp16 parts
of 11 bits: they leave out 2^-22 of a value, or 2^-39 of the matrix' largest magnitude where the value is
below 2^-17 of it (half of the last step 2^-24 of a part, the largest being scaled to 2^14 at least; G,
at most 1, is scaled by 2^15: 2^-40). The product of the low parts is left out, another 2^-22. The tensor
core adds 128 terms in 24 additions, each off by at most one part in 2^23 of the magnitudes; those sums
are then added in fp32. So a product of K terms is off by at most
  g(K) = 3 2^-22 + min(24, 3 ceil(K / 16)) 2^-23 + (ceil(K / 128) + 2) 2^-24
times the sum of the terms' magnitudes, and what the small values' absolute errors add.
"""
import math

import pytest
import torch

import nnb
from nnb import functional as F
from nnb.autograd import Value
from nnb.graph import GraphedStep

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
IGNORE = -100


def g(K):
    return 3 * 2.0 ** -22 + min(24, 3 * math.ceil(K / 16)) * 2.0 ** -23 + (math.ceil(K / 128) + 2) * 2.0 ** -24


def _make(P, D, V, bias=True, ignored=0.0, seed=0, shift=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0):
        n = math.prod(shape)
        return torch.empty(n + shift, device="cuda")[shift:].view(shape).copy_(
            torch.randn(*shape, generator=gen, device="cuda") * std)

    x, w, b = t(P, D), t(V, D, std=2.0 / D ** 0.5), t(V) if bias else None
    targets = torch.randint(0, V, (P,), generator=gen, device="cuda")
    targets[torch.rand(P, generator=gen, device="cuda") < ignored] = IGNORE
    return x, w, b, targets


def _want(x, w, b, t, ls, up=1.0, norm=None):
    """Loss, per-row losses and gradients in 64 bits, each with its bound."""
    x, w = x.double(), w.double()
    P, D = x.shape
    V = w.shape[0]
    bias = b.double() if b is not None else torch.zeros(V, dtype=torch.float64, device="cuda")
    l = x @ w.t() + bias
    # logits: the product, and the bias' addition (1 rounding)
    el = g(D) * (x.abs() @ w.abs().t()) + E * l.abs() * 2
    el += 2.0 ** -39 * (float(x.abs().max()) * w.abs().sum(1) + float(w.abs().max()) * x.abs().sum(1)[:, None])
    live = t != IGNORE
    at = t.clamp(min=0)[:, None]
    lse = torch.logsumexp(l, 1)
    q = torch.full_like(l, ls / V).scatter_add_(1, at, torch.full_like(at, 1 - ls, dtype=torch.float64))
    rows = torch.where(live, lse - (q * l).sum(1), 0.0)
    worst = el.amax(1)
    # a row's loss moves by at most twice its worst logit; the sums of V terms in fp32 (at most V / 256 + 16
    # roundings of the sum of exponentials, and of sum |l| / V with smoothing), and a few roundings
    sums = (V / 256 + 24) * E
    erows = torch.where(live, 2 * worst + sums * (1 + ls * l.abs().mean(1)) + 8 * E * (lse.abs() + l.abs().amax(1)), 0.0)
    count = int(live.sum())
    loss = rows.sum() / count if count else torch.tensor(float("nan"))
    eloss = erows.sum() / max(count, 1) + 2 * E * abs(float(loss))
    k = up * (1.0 / count if norm is None else norm)
    p = (l - lse[:, None]).exp()
    mask = live[:, None].double()
    G = (p - q) * mask
    # p: twice the worst logit, the sum's roundings, exponential, argument, quotient; then the subtractions
    eG = mask * (p * (2 * worst[:, None] + sums + 8 * E + E * (l - l.amax(1, keepdim=True)).abs()) + 4 * E * q)
    eG += 2.0 ** -40 * mask
    small_w = 2.0 ** -39 * float(w.abs().max()) * G.abs().sum(1, keepdim=True)
    small_x = 2.0 ** -39 * float(x.abs().max()) * G.abs().sum(0)[:, None]
    out = {"loss": (loss, eloss), "rows": (rows, erows)}
    for name, value, err in (
            ("x", G @ w, eG @ w.abs() + g(V) * (G.abs() @ w.abs()) + small_w),
            ("w", G.t() @ x, eG.t() @ x.abs() + g(P) * (G.abs().t() @ x.abs()) + small_x),
            ("b", G.sum(0), eG.sum(0) + (P + 8) * E * G.abs().sum(0))):
        out[name] = value * k, err * abs(k) + 4 * E * value.abs() * abs(k)
    return out


def _close(got, want, name):
    v, e = want
    bad = (got.double() - v).abs() > e + 1e-37
    assert not torch.as_tensor(bad).any(), (name, float(((got.double() - v).abs() / (e + 1e-300)).max()))


def _run(x, w, b, t, ls=0.0, seed=None, base=None, **kw):
    vals = {"x": Value.leaf(x, True), "w": Value.leaf(w, True)}
    if b is not None:
        vals["b"] = Value.leaf(b, True)
    if base is not None:
        for k, v in vals.items():
            v.grad, v.grad_fresh = base[k].clone(), False
    loss = F.linear_cross_entropy(vals["x"], vals["w"], vals.get("b"), t, IGNORE, ls, **kw)
    loss.backward(seed)
    return loss.data, {k: v.grad for k, v in vals.items()}


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (64, 64, 65), (100, 33, 300), (256, 128, 4096), (129, 16, 1000), (130, 2048, 48),
          (17, 100, 5003), (40, 24, 50001), (512, 96, 257), (1000, 64, 130), (5, 512, 20000), (2047, 40, 33)]


@pytest.mark.parametrize("ls", [0.0, 0.1])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("P,D,V", SHAPES)
def test_against_64_bits(cuda, P, D, V, bias, ls):
    data = _make(P, D, V, bias, ignored=0.2 if P > 2 else 0.0, seed=P + V)
    loss, grads = _run(*data, ls)
    want = _want(*data, ls)
    _close(loss, want["loss"], "loss")
    for k, got in grads.items():
        _close(got, want[k], k)
    args = [Value.leaf(v, False) if v is not None else None for v in data[:3]]
    rows, mean = F.linear_token_losses(*args, data[3], IGNORE, ls)
    _close(rows, want["rows"], "rows")
    _close(mean, want["loss"], "mean")
    assert nnb.device_error() == 0


@pytest.mark.parametrize("P,D,V", [(5000, 48, 20000), (3001, 64, 40000)])
def test_several_pieces(cuda, P, D, V):
    """More rows than one piece's logits may take."""
    data = _make(P, D, V, ignored=0.1, seed=1)
    loss, grads = _run(*data)
    want = _want(*data, 0.0)
    _close(loss, want["loss"], "loss")
    for k, got in grads.items():
        _close(got, want[k], k)
    again = _run(*data)
    assert torch.equal(loss, again[0]) and all(torch.equal(grads[k], again[1][k]) for k in grads)


@pytest.mark.parametrize("shift", [1, 2])
def test_unaligned_buffers(cuda, shift):
    data = _make(70, 36, 129, seed=3, shift=shift)
    loss, grads = _run(*data)
    want = _want(*data, 0.0)
    _close(loss, want["loss"], "loss")
    for k, got in grads.items():
        _close(got, want[k], k)


def test_upstream_gradient_norm_and_added_gradients(cuda):
    data = _make(50, 32, 70, seed=4)
    base = {"x": torch.randn(50, 32, device="cuda"), "w": torch.randn(70, 32, device="cuda"),
            "b": torch.randn(70, device="cuda")}
    norm = torch.tensor([0.01], device="cuda")
    _, grads = _run(*data, seed=torch.tensor([3.0], device="cuda"), base=base, grad_norm=norm)
    want = _want(*data, 0.0, up=3.0, norm=float(norm))
    for k, got in grads.items():
        v, e = want[k]
        v = v + base[k].double()
        _close(got, (v, e + E * (v.abs() + base[k].abs().double())), k)


def test_matches_the_composed_ops(cuda):
    """linear then sequence_cross_entropy, the ops that keep the logits."""
    x, w, b, t = _make(96, 64, 500, ignored=0.3, seed=5)
    loss, grads = _run(x.view(4, 24, 64), w, b, t.view(4, 24), 0.1)
    vals = [Value.leaf(v, True) for v in (x.view(4, 24, 64), w, b)]
    ref = F.sequence_cross_entropy(F.linear(*vals), t.view(4, 24), IGNORE, 0.1)
    ref.backward()
    want = _want(x, w, b, t, 0.1)
    assert abs(float(loss) - float(ref.data)) <= 2 * float(want["loss"][1])
    for k, v in zip(("x", "w", "b"), vals):
        assert torch.all((grads[k].double() - v.grad.double()).abs().view(want[k][1].shape) <= 2 * want[k][1] + 1e-37), k


def test_any_subset_needs_gradients(cuda):
    x, w, b, t = _make(200, 48, 333, seed=6)
    loss, full = _run(x, w, b, t)
    for only in ("x", "w", "b"):
        vals = {k: Value.leaf(v, k == only) for k, v in (("x", x), ("w", w), ("b", b))}
        part = F.linear_cross_entropy(vals["x"], vals["w"], vals["b"], t)
        part.backward()
        assert torch.equal(part.data, loss) and torch.equal(vals[only].grad, full[only]), only


def test_weight_as_input(cuda):
    """x and the weight are one Value: it receives the sum of both gradients."""
    _, w, b, _ = _make(1, 40, 64, seed=14)
    t = torch.arange(64, device="cuda") % 60
    want = _run(w.clone(), w, b, t)[1]
    both = Value.leaf(w, True)
    F.linear_cross_entropy(both, both, Value.leaf(b, False), t).backward()
    assert torch.equal(both.grad, want["x"] + want["w"])


def test_all_ignored_and_bad_targets(cuda):
    x, w, b, t = _make(20, 16, 30, seed=7)
    loss, grads = _run(x, w, b, torch.full_like(t, IGNORE))
    assert torch.isnan(loss).all() and all(torch.equal(v, torch.zeros_like(v)) for v in grads.values())
    assert nnb.device_error() == 0
    for bad in (30, -1, 2 ** 40):
        t2 = t.clone()
        t2[3] = bad
        loss, grads = _run(x, w, b, t2)
        assert torch.isnan(loss).all() and nnb.device_error() == 16
        assert torch.equal(grads["x"][3], torch.zeros(16, device="cuda"))
        assert torch.isfinite(grads["w"]).all()


def test_masked_vocabulary_and_bad_rows(cuda):
    """A bias of -inf takes tokens out of the vocabulary; a row with NaN or +inf, or with nothing left, is NaN
    in its loss and its gradient, and leaves the other rows' losses and gradients as they were."""
    x, w, b, t = _make(40, 32, 64, seed=8)
    b[40:] = -math.inf
    t %= 40
    loss, grads = _run(x, w, b, t)
    want = _want(x, w[:40], b[:40], t, 0.0)
    _close(loss, want["loss"], "loss")
    _close(grads["x"], want["x"], "x")
    _close(grads["w"][:40], want["w"], "w")
    assert torch.equal(grads["w"][40:], torch.zeros(24, 32, device="cuda"))
    args = [Value.leaf(v, False) for v in (x, w, b)]
    clean, _ = F.linear_token_losses(*args, t)
    x2 = x.clone()
    x2[5, 3], x2[9, 0] = math.nan, math.inf
    bad, mean = F.linear_token_losses(Value.leaf(x2, False), *args[1:], t)
    keep = [i for i in range(40) if i not in (5, 9)]
    assert torch.equal(bad[keep], clean[keep]) and torch.isnan(bad[[5, 9]]).all() and torch.isnan(mean).all()
    _, g2 = _run(x2, w, b, t)
    assert torch.equal(g2["x"][keep], grads["x"][keep]) and torch.isnan(g2["x"][[5, 9]]).all()
    assert torch.isnan(g2["w"]).all() and torch.isnan(g2["b"]).all()
    none, _ = F.linear_token_losses(*args[:2], Value.leaf(torch.full_like(b, -math.inf), False), t)
    assert torch.isnan(none).all()


def test_large_logits(cuda):
    """Logits of many thousands: the softmax is one-hot and the loss their difference."""
    x, w, b, t = _make(16, 64, 200, seed=9)
    loss, grads = _run(x * 300, w * 300, b, t)
    want = _want(x * 300, w * 300, b, t, 0.0)
    _close(loss, want["loss"], "loss")
    assert all(torch.isfinite(v).all() for v in grads.values())


def test_parameter_groups(cuda):
    """Gradients kept per group of rows: those of the group's rows alone, bit for bit."""
    G, P, D, V = 4, 4 * 48, 40, 90
    x, w, b, t = _make(P, D, V, seed=10)
    vals = {"x": Value.leaf(x, True), "w": Value.leaf(w, True), "b": Value.leaf(b, True)}
    for k, n in (("w", V * D), ("b", V)):
        vals[k].grad, vals[k].grad_fresh = torch.full((G, n + 8), math.nan, device="cuda")[:, :n], True
    norm = torch.tensor([1.0 / 48], device="cuda")
    with F.param_groups(G):
        F.linear_cross_entropy(vals["x"], vals["w"], vals["b"], t, grad_norm=norm).backward()
    for z in range(G):
        rows = slice(48 * z, 48 * z + 48)
        _, part = _run(x[rows].contiguous(), w, b, t[rows].contiguous(), grad_norm=norm)
        assert torch.equal(vals["x"].grad[rows], part["x"])
        assert torch.equal(vals["w"].grad[z].view(V, D), part["w"]) and torch.equal(vals["b"].grad[z], part["b"])


def test_backward_outside_the_forwards_groups(cuda):
    """The kept gradients have the forward's groups: a backward in other groups, or into buffers that do not hold
    them, is refused before anything is launched or marked as written."""
    G, P, D, V = 2, 2 * 8, 6, 10
    x, w, b, t = _make(P, D, V, seed=19)

    def forward(grouped):
        vals = [Value.leaf(v, True) for v in (x, w, b)]
        if grouped:
            for v in vals[1:]:
                v.grad = torch.empty(G, v.data.numel(), device="cuda")
        return vals, lambda: F.linear_cross_entropy(*vals, t)

    def refused(vals, loss, match):
        with pytest.raises(ValueError, match=match):
            loss.backward()
        assert all(v.grad_fresh for v in vals)

    vals, f = forward(False)
    with F.param_groups(G):
        loss = f()
    refused(vals, loss, "parameter group")
    vals, f = forward(True)
    loss = f()
    with F.param_groups(G):
        refused(vals, loss, "parameter group")
    for inside in (True, False):       # buffers that do not fit the groups
        vals, f = forward(not inside)
        with F.param_groups(G if inside else 1):
            refused(vals, f(), "does not hold")
    vals, f = forward(True)
    with F.param_groups(G):
        f().backward()
    assert torch.equal(vals[0].grad, _run(x, w, b, t)[1]["x"])


def test_groups_of_different_size(cuda):
    """A group's bits are its own whatever the other groups hold: here one 2^30 times larger, next to values
    that its scale would have lost."""
    G, P, D, V = 2, 2 * 32, 24, 50
    x, w, b, t = _make(P, D, V, seed=17)
    x[:32] *= 2.0 ** 30
    x[32:, ::3] *= 2.0 ** -12
    vals = {"x": Value.leaf(x, True), "w": Value.leaf(w, True), "b": Value.leaf(b, True)}
    for k, n in (("w", V * D), ("b", V)):
        vals[k].grad, vals[k].grad_fresh = torch.empty(G, n, device="cuda"), True
    norm = torch.tensor([1.0 / 32], device="cuda")
    with F.param_groups(G):
        F.linear_cross_entropy(vals["x"], vals["w"], vals["b"], t, grad_norm=norm).backward()
    _, part = _run(x[32:].contiguous(), w, b, t[32:].contiguous(), grad_norm=norm)
    assert torch.equal(vals["x"].grad[32:], part["x"])
    assert torch.equal(vals["w"].grad[1].view(V, D), part["w"]) and torch.equal(vals["b"].grad[1], part["b"])


def test_ignored_rows_may_hold_anything(cuda):
    x, w, b, t = _make(40, 32, 64, seed=18)
    t[7], t[20] = IGNORE, IGNORE
    want = _run(x, w, b, t)
    x2 = x.clone()
    x2[7], x2[20] = math.nan, math.inf
    got = _run(x2, w, b, t)
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[1][k], want[1][k]) for k in want[1])


@pytest.mark.parametrize("std", [30.0, 300.0])
def test_gradients_of_large_logits(cuda, std):
    """Gradients of a softmax that is close to one-hot, and one-hot, against their bounds."""
    x, w, b, t = _make(16, 64, 200, seed=9)
    _, grads = _run(x * std, w * std, b, t)
    want = _want(x * std, w * std, b, t, 0.0)
    for k, got in grads.items():
        _close(got, want[k], k)


def test_gradients_of_confident_rows(cuda):
    """Rows whose target has nearly all the probability: the target's own entry, p - 1, is a difference of fp32
    values next to 1, every other entry as small as its probability."""
    x, w, b, t = _make(32, 48, 300, seed=23)
    w[t] += 6.0 * x / x.square().sum(1, keepdim=True) * 4.0
    _, grads = _run(x, w, b, t)
    want = _want(x, w, b, t, 0.0)
    for k, got in grads.items():
        _close(got, want[k], k)


def test_a_large_row_costs_the_others_no_bits(cuda):
    """Operands are scaled by blocks of 128 rows: a row 2^40 times larger leaves the bits of the rows in other
    blocks, their losses and their gradients, as they were."""
    x, w, b, t = _make(400, 40, 300, seed=24)
    x2 = x.clone()
    x2[130] *= 2.0 ** 40
    keep = [i for i in range(400) if not 128 <= i < 256]
    norm = torch.tensor([1.0], device="cuda")
    rows, grads = [], []
    for data in (x, x2):
        rows.append(F.linear_token_losses(*[Value.leaf(v, False) for v in (data, w, b)], t)[0])
        grads.append(_run(data, w, b, t, grad_norm=norm)[1]["x"])
    assert torch.equal(rows[0][keep], rows[1][keep]) and torch.equal(grads[0][keep], grads[1][keep])
    _close(rows[0], _want(x, w, b, t, 0.0)["rows"], "rows")


@pytest.mark.parametrize("k", [100, -100, 60, -60])
def test_operands_of_extreme_size(cuda, k):
    """x 2^k and w 2^-k have the same logits: the same loss to the bit, dx and dw with their powers of two, also where
    the scales of two blocks together leave the range of one fp32 factor."""
    x, w, b, t = _make(300, 70, 260, seed=26)
    norm = torch.tensor([1.0], device="cuda")
    want = _run(x, w, b, t, grad_norm=norm)
    got = _run(x * 2.0 ** k, w * 2.0 ** -k, b, t, grad_norm=norm)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1]["b"], want[1]["b"])
    assert torch.equal(got[1]["x"].double() * 2.0 ** k, want[1]["x"].double())
    assert torch.equal(got[1]["w"].double() * 2.0 ** -k, want[1]["w"].double())


@pytest.mark.parametrize("drop", [10.0, 28.0, 60.0])
def test_rare_tokens_keep_their_bits(cuda, drop):
    """Tokens of small probabilities whose block of 128 has no target: their rows of dW are as exact, relative to the
    terms they sum, as any others. (One bound for the entries of G, relative to the probability.)"""
    P, D, V = 200, 48, 400
    x, w, b, t = _make(P, D, V, seed=25)
    t %= 128
    b[128:] -= drop
    _, grads = _run(x, w, b, t)
    X, W, B = (v.double() for v in (x, w, b))
    l = X @ W.t() + B
    top = l.amax(1, keepdim=True)
    p = torch.softmax(l, 1)[:, 128:]
    worst = (g(D) * (X.abs() @ W.abs().t()) + 2 * E * l.abs()).amax(1, keepdim=True)
    worst = worst + 2.0 ** -39 * (float(X.abs().max()) * W.abs().sum(1).max() + float(W.abs().max()) * X.abs().sum(1, keepdim=True))
    ep = 2 * worst + (V / 256 + 24) * E + 8 * E + 2 * E * (l - top).abs()[:, 128:]
    terms = p.t() @ X.abs()
    err = (p * ep).t() @ X.abs() + (g(P) + 6 * E) * terms
    err += 2.0 ** -39 * (float(X.abs().max()) * p.sum(0)[:, None] + float(p.max()) * X.abs().sum(0))
    want = p.t() @ X / P
    assert torch.all((grads["w"][128:].double() - want).abs() <= err / P)
    assert float((err / P).max()) < 1e-4 * float(want.abs().max())


@pytest.mark.parametrize("P,D,V", [(40, 32, 64), (64, 33, 50), (7, 2, 20), (300, 1, 9), (2, 3, 5)])
@pytest.mark.parametrize("value", [1e6, 1e20, 3e38])
def test_rows_that_do_not_count_may_hold_large_values(cuda, P, D, V, value):
    """What a row with an ignored target holds leaves every bit of the loss and the gradients alone, with rows
    that share a 16-byte load among them; so does a row whose target is no token, for the gradients."""
    x, w, b, t = _make(P, D, V, seed=21)
    dead = [i for i in range(P) if i % 3 == 1]
    t[dead] = IGNORE
    want = _run(x, w, b, t)
    _close(want[0], _want(x, w, b, t, 0.0)["loss"], "loss")
    x2 = x.clone()
    x2[dead] = value
    got = _run(x2, w, b, t)
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[1][k], want[1][k]) for k in want[1])
    rows = [F.linear_token_losses(*[Value.leaf(v, False) for v in (data, w, b)], t)[0] for data in (x, x2)]
    assert torch.equal(*rows)
    t2 = t.clone()
    t2[dead] = V
    loss, grads = _run(x2, w, b, t2)
    assert torch.isnan(loss).all() and nnb.device_error() == 16
    assert all(torch.equal(grads[k], want[1][k]) for k in want[1])


def test_ignored_rows_of_a_group_may_hold_large_values(cuda):
    G, P, D, V = 2, 2 * 36, 5, 30
    x, w, b, t = _make(P, D, V, seed=22)
    t[[3, 50]] = IGNORE
    norm = torch.tensor([1.0 / 36], device="cuda")
    out = []
    for value in (1.0, 1e30):
        x[[3, 50]] = value
        vals = {"x": Value.leaf(x, True), "w": Value.leaf(w, True), "b": Value.leaf(b, True)}
        for k, n in (("w", V * D), ("b", V)):
            vals[k].grad, vals[k].grad_fresh = torch.empty(G, n, device="cuda"), True
        with F.param_groups(G):
            F.linear_cross_entropy(vals["x"], vals["w"], vals["b"], t, grad_norm=norm).backward()
        out.append([v.grad for v in vals.values()])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_tf32_mode(cuda):
    """The fast mode: operands of 11 significant bits, 2^-11 of each term's two factors."""
    x, w, b, t = _make(300, 64, 500, seed=11)
    old = nnb.get_math_mode()
    nnb.set_math_mode(nnb.MATH_TF32)
    try:
        loss, grads = _run(x, w, b, t)
    finally:
        nnb.set_math_mode(old)
    want = _want(x, w, b, t, 0.0)
    el = float((x.double().abs() @ w.double().abs().t()).max()) * 2.0 ** -10
    assert abs(float(loss) - float(want["loss"][0])) <= 2 * el
    p = torch.softmax((x.double() @ w.double().t() + b.double()), 1)
    for k, other in (("x", w), ("w", x)):
        lim = (p @ w.double().abs()).max() if k == "x" else (p.t() @ x.double().abs()).max()
        scale = float(want[k][0].abs().max()) + float(lim) / 300
        assert float((grads[k].double() - want[k][0]).abs().max()) <= (2 * el + 2.0 ** -9) * scale * 2


def test_gradients_against_differences(cuda):
    """Along a random direction, the 64-bit loss's central difference and the operator's gradients; the bounds
    of the gradients allow far less than the 1e-4 here."""
    x, w, b, t = _make(24, 16, 40, ignored=0.2, seed=12)
    _, grads = _run(x, w, b, t, 0.1)
    step = {k: torch.randn_like(v).double() * 0.1 for k, v in (("x", x), ("w", w), ("b", b))}

    def value(e):
        return float(_want(x.double() + e * step["x"], w.double() + e * step["w"], b.double() + e * step["b"], t, 0.1)["loss"][0])

    numeric = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = [grads[k].double() * step[k] for k in step]
    assert abs(numeric - sum(float(v.sum()) for v in terms)) <= 1e-4 * sum(float(v.abs().sum()) for v in terms)


def test_captured_and_on_another_stream(cuda):
    data = _make(300, 64, 1000, ignored=0.1, seed=13)
    want = _run(*data)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(*data)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [GraphedStep(lambda: _run(*data)) for _ in range(2)]
    for res in (got, graphs[0](), graphs[1](), graphs[0]()):
        assert torch.equal(res[0], want[0]) and all(torch.equal(res[1][k], want[1][k]) for k in want[1])
