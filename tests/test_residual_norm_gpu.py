"""The residual norm against its definition in 64 bits, with tolerances that count roundings.

E = 2^-24 is half a step of fp32. A row sum of D values is taken over at most 16 values per thread in
order and a tree of at most 10 levels: 26 roundings of the sum of magnitudes, 28 with the mean's factor.
So with A = mean|a| / deviation
  hat = (a - mean) * inv       is off by at most (20 |hat| + 28 A) E   (inv: half of the variance's 30,
                               the root and the quotient; then the difference and the product)
and every other bound below follows from it and the formula beside it. The norm's output and gradients
are held to the 64-bit formulas on the h that the operator returned.
"""
import itertools

import pytest
import torch

from nnb import functional as F
from nnb.autograd import Value, backward
from nnb.graph import GraphedStep

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
EPS = 1e-5


class Norm64:
    """A norm of rows in 64 bits, its backward, and the bounds of both in fp32."""

    def __init__(self, a, gamma, beta, layer):
        self.layer, self.gamma = layer, gamma
        mu = a.mean(1, keepdim=True) if layer else torch.zeros_like(a[:, :1])
        self.inv = ((a - mu).square().mean(1, keepdim=True) + EPS).rsqrt()
        self.hat = (a - mu) * self.inv
        self.out = self.hat * gamma + (beta if beta is not None else 0.0)
        self.err_hat = E * (20 * self.hat.abs() + 28 * a.abs().mean(1, keepdim=True) * self.inv)
        self.err_out = self.err_hat * gamma.abs() + E * ((self.hat * gamma).abs() + self.out.abs())

    def back(self, dy, err_dy):
        """(gradient of the input, its bound): inv (d - mean d - hat mean(d hat)), d = dy gamma."""
        d = dy * self.gamma
        err_d = err_dy * self.gamma.abs() + E * d.abs()
        mean = lambda t: t.mean(1, keepdim=True)      # noqa: E731
        md, mb = mean(d) if self.layer else 0.0, mean(d * self.hat)
        abs_d, abs_b = mean(d.abs()), mean((d * self.hat).abs())
        g = self.inv * (d - md - self.hat * mb)
        err_b = 30 * E * abs_b + mean(d.abs() * self.err_hat + self.hat.abs() * err_d)
        err = err_d + 30 * E * abs_d + mean(err_d) + self.err_hat * abs_b + self.hat.abs() * err_b
        return g, self.inv * (err + 24 * E * (d.abs() + abs_d + self.hat.abs() * abs_b))


def _make(R, D, span, kind, post, gate, seed=0, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0, mean=0.0):
        n = 1
        for s in shape:
            n *= s
        buf = torch.empty(n + shift, device="cuda")[shift:].view(shape)
        return buf.copy_(torch.randn(*shape, generator=g, device="cuda") * std + mean)

    layer = kind == "layer"
    ops = {"x": t(R, D, std=2.0, mean=0.5), "branch": t(R, D), "gamma": t(D, std=0.2, mean=1.0)}
    if layer:
        ops["beta"] = t(D, std=0.2)
    if post:
        ops["post_gamma"] = t(D, std=0.2, mean=1.0)
        if layer:
            ops["post_beta"] = t(D, std=0.2)
    if gate != "none":
        ops["gate"] = t({"channel": 1, "sequence": R // span, "token": R}[gate], D, std=0.5, mean=0.5)
    return ops, t(R, D), t(R, D)


def _check(ops, h, y, grads, dh, dy, kind, scale, base=None):
    """Everything the operator returned against the definition. base: gradients that were there before."""
    o = {k: v.double() for k, v in ops.items()}
    R, D = h.shape
    layer = kind == "layer"
    zero = torch.zeros_like(h, dtype=torch.float64)
    p, err_p, post = o["branch"], zero, None
    if "post_gamma" in o:
        post = Norm64(o["branch"], o["post_gamma"], o.get("post_beta"), layer)
        p, err_p = post.out, post.err_out
    rows = o["gate"].repeat_interleave(R // o["gate"].shape[0], 0) if "gate" in o else torch.ones_like(p)
    want_h = o["x"] + scale * rows * p
    err = (scale * rows).abs() * err_p + E * ((scale * rows * p).abs() * 2 + want_h.abs())
    assert torch.all((h.double() - want_h).abs() <= err)
    norm = Norm64(h.double(), o["gamma"], o.get("beta"), layer)
    assert torch.all((y.double() - norm.out).abs() <= norm.err_out)
    if grads is None:
        return
    dh = dh.double() if dh is not None else zero
    dt, err_dt = dh, zero
    sums = {}
    row_roundings = (R + 60) * E             # rows in any order: at most one rounding each, and the trees
    if dy is not None:
        dy = dy.double()
        g, e = norm.back(dy, zero)
        dt, err_dt = dh + g, e + 4 * E * (dh.abs() + norm.inv * (dy * o["gamma"]).abs() + g.abs())
        sums["gamma"] = (dy * norm.hat, dy.abs() * norm.err_hat)
        sums["beta"] = (dy, zero)
    sums.setdefault("gamma", (zero, zero))
    sums.setdefault("beta", (zero, zero))
    sums["x"] = None
    want = {"x": (dt, err_dt)}
    dp, err_dp = scale * rows * dt, (scale * rows).abs() * err_dt + 2 * E * (scale * rows * dt).abs()
    sums["gate"] = (scale * p * dt, (scale * p).abs() * err_dt + (scale * dt).abs() * err_p + 2 * E * (scale * p * dt).abs())
    if post is not None:
        sums["post_gamma"] = (dp * post.hat, err_dp * post.hat.abs() + dp.abs() * post.err_hat)
        sums["post_beta"] = (dp, err_dp)
        want["branch"] = post.back(dp, err_dp)
    else:
        want["branch"] = dp, err_dp
    for k in ops:
        if k not in want:
            v, e = sums[k]
            n = ops[k].shape[0] if k == "gate" else 1
            fold = lambda t: t.view(n, R // n, D).sum(1)      # noqa: E731
            want[k] = fold(v).view(ops[k].shape), (fold(e) + row_roundings * fold(v.abs())).view(ops[k].shape)
    for k, got in grads.items():
        v, e = want[k]
        if base is not None:
            v = v + base[k].double()
            e = e + E * (v.abs() + base[k].double().abs())
        bad = (got.double() - v).abs() > e + E * v.abs()
        assert not bad.any(), (k, int(bad.sum()), float(((got.double() - v).abs() / (e + 1e-300)).max()))


def _run(ops, dh, dy, kind, scale, only=None, base=None):
    vals = {k: Value.leaf(v, only is None or k in only) for k, v in ops.items()}
    if base is not None:
        for k, v in vals.items():
            v.grad, v.grad_fresh = base[k].clone(), False
    h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals.get("beta"), EPS, kind=kind,
                           post_gamma=vals.get("post_gamma"), post_beta=vals.get("post_beta"), gate=vals.get("gate"),
                           scale=scale)
    roots = [(v, d) for v, d in ((h, dh), (y, dy)) if d is not None]
    backward([v for v, _ in roots], [d for _, d in roots])
    return h.data, y.data, {k: v.grad for k, v in vals.items() if v.requires_grad}


FORMS = list(itertools.product(("layer", "rms"), (False, True), ("none", "channel", "sequence", "token")))
SHAPES = [(1, 1, 1), (1, 64, 1), (6, 3, 2), (40, 33, 8), (33, 64, 33), (300, 100, 3), (96, 512, 32), (50, 1001, 25),
          (12, 1024, 4), (21, 2048, 7), (10, 2500, 5), (8, 4096, 4), (9, 4100, 3), (7, 5001, 7), (6, 8192, 2), (5, 16383, 5),
          (4, 16384, 2)]


@pytest.mark.parametrize("kind,post,gate", FORMS)
@pytest.mark.parametrize("R,D,span", SHAPES)
def test_against_64_bits(cuda, R, D, span, kind, post, gate):
    ops, dh, dy = _make(R, D, span, kind, post, gate, seed=R * 31 + D)
    h, y, grads = _run(ops, dh, dy, kind, 0.5)
    _check(ops, h, y, grads, dh, dy, kind, 0.5)


@pytest.mark.parametrize("kind,post,gate", [("layer", True, "sequence"), ("rms", False, "channel")])
@pytest.mark.parametrize("R,D,span", [(5000, 64, 1000), (4000, 512, 500), (3001, 257, 3001), (1500, 2048, 3)])
def test_many_rows(cuda, R, D, span, kind, post, gate):
    """Runs of several rows, spans cut into pieces and pieces of several spans."""
    ops, dh, dy = _make(R, D, span, kind, post, gate, seed=5)
    h, y, grads = _run(ops, dh, dy, kind, 1.0)
    _check(ops, h, y, grads, dh, dy, kind, 1.0)
    again = _run(ops, dh, dy, kind, 1.0)[2]
    assert all(torch.equal(grads[k], again[k]) for k in grads)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_unaligned_buffers(cuda, shift):
    ops, dh, dy = _make(20, 128, 5, "layer", True, "sequence", seed=2, shift=shift)
    h, y, grads = _run(ops, dh, dy, "layer", 1.0)
    _check(ops, h, y, grads, dh, dy, "layer", 1.0)


@pytest.mark.parametrize("given", ["h", "y"])
@pytest.mark.parametrize("kind,post,gate", FORMS)
def test_one_root(cuda, kind, post, gate, given):
    ops, dh, dy = _make(24, 48, 6, kind, post, gate, seed=3)
    dh, dy = (dh, None) if given == "h" else (None, dy)
    base = {k: torch.randn_like(v) for k, v in ops.items()}
    h, y, grads = _run(ops, dh, dy, kind, 0.25, base=base)
    if given == "h":        # the norm before the next block is not reached: its gradients stay untouched
        for k in {"gamma", "beta"} & set(grads):
            assert torch.equal(grads.pop(k), base[k])
    _check(ops, h, y, grads, dh, dy, kind, 0.25, base=base)


@pytest.mark.parametrize("kind,post,gate", FORMS)
def test_gradients_are_added(cuda, kind, post, gate):
    ops, dh, dy = _make(30, 40, 10, kind, post, gate, seed=4)
    base = {k: torch.randn_like(v) for k, v in ops.items()}
    h, y, grads = _run(ops, dh, dy, kind, 1.0, base=base)
    _check(ops, h, y, grads, dh, dy, kind, 1.0, base=base)


def test_any_subset_needs_gradients(cuda):
    ops, dh, dy = _make(12, 64, 3, "layer", True, "sequence", seed=6)
    full = _run(ops, dh, dy, "layer", 1.0)[2]
    for only in (["x"], ["branch"], ["gate"], ["gamma"], ["beta"], ["post_gamma", "beta"]):
        grads = _run(ops, dh, dy, "layer", 1.0, only=only)[2] if only[0] not in ("gamma", "beta") else None
        if grads is None:       # h needs no gradient: only y is a root
            vals = {k: Value.leaf(v, k in only) for k, v in ops.items()}
            _, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals["beta"], EPS,
                                   post_gamma=vals["post_gamma"], post_beta=vals["post_beta"], gate=vals["gate"])
            y.backward(dy)
            grads = {k: v.grad for k, v in vals.items() if v.requires_grad}
        assert set(grads) == set(only)
        for k in only:
            assert torch.equal(grads[k], full[k]), k


def test_inference_keeps_nothing(cuda):
    ops, dh, dy = _make(12, 64, 3, "rms", True, "token", seed=6)
    vals = {k: Value.leaf(v, False) for k, v in ops.items()}
    h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], None, EPS, kind="rms",
                           post_gamma=vals["post_gamma"], gate=vals["gate"], scale=0.5)
    assert not h.requires_grad and not y.requires_grad and not h.parents
    _check(ops, h.data, y.data, None, None, None, "rms", 0.5)


def test_same_value_as_x_and_branch(cuda):
    ops, dh, dy = _make(17, 96, 17, "layer", False, "none", seed=8)
    ops["branch"] = ops["x"].clone()
    apart = _run(ops, dh, dy, "layer", 0.5)[2]
    x, gamma, beta = (Value.leaf(ops[k], True) for k in ("x", "gamma", "beta"))
    h, y = F.residual_norm(x, x, gamma, beta, EPS, scale=0.5)
    backward((h, y), (dh, dy))
    assert torch.equal(x.grad, apart["x"] + apart["branch"])
    with pytest.raises(ValueError, match="share"):
        h, y = F.residual_norm(x, x, gamma, beta, EPS, post_gamma=gamma, post_beta=beta)
        backward((h, y), (dh, dy))


def test_parameter_groups(cuda):
    """Under F.param_groups every parameter's gradient is kept per group of rows: the gradients of a group's
    rows alone, bit for bit (a group's sums do not depend on how many groups there are)."""
    G, R, D = 4, 4 * 60, 64
    ops, dh, dy = _make(R, D, 20, "layer", True, "sequence", seed=9)
    params = [k for k in ops if k not in ("x", "branch", "gate")]
    vals = {k: Value.leaf(v, True) for k, v in ops.items()}
    for k in params:
        vals[k].grad = torch.full((G, D), float("nan"), device="cuda")
        vals[k].grad_fresh = True
    with F.param_groups(G):
        h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals["beta"], EPS, post_gamma=vals["post_gamma"],
                               post_beta=vals["post_beta"], gate=vals["gate"])
        backward((h, y), (dh, dy))
    for z in range(G):
        rows, spans = slice(z * 60, z * 60 + 60), slice(z * 3, z * 3 + 3)
        part = {k: v[rows] if k in ("x", "branch") else v[spans] if k == "gate" else v for k, v in ops.items()}
        grads = _run(part, dh[rows].contiguous(), dy[rows].contiguous(), "layer", 1.0)[2]
        for k in params:
            assert torch.equal(vals[k].grad[z], grads[k]), k
        assert torch.equal(vals["gate"].grad[spans], grads["gate"])


@pytest.mark.parametrize("R,D", [(1, 24), (9, 33), (6, 512), (5, 4100)])
def test_one_value_in_every_place_of_its_shape(cuda, R, D):
    """x, the branch and a gate per token are one Value: it receives the sum of the three gradients."""
    ops, dh, dy = _make(R, D, 1, "rms", False, "token", seed=34)
    ops["branch"] = ops["gate"] = ops["x"]
    apart = _run({k: v.clone() for k, v in ops.items()}, dh, dy, "rms", 0.5)[2]
    x, gamma = Value.leaf(ops["x"], True), Value.leaf(ops["gamma"], True)
    h, y = F.residual_norm(x, x, gamma, None, EPS, kind="rms", gate=x, scale=0.5)
    backward((h, y), (dh, dy))
    parts = [apart[k].double() for k in ("x", "branch", "gate")]
    assert torch.all((x.grad.double() - sum(parts)).abs() <= 2 * E * sum(v.abs() for v in parts))
    assert torch.equal(gamma.grad, apart["gamma"])


@pytest.mark.parametrize("roots", ["y", "hy", "h", "consumer"])
def test_no_partial_gradient_is_left_on_h(cuda, roots):
    """h's whole gradient is never stored: h.grad is None after a pass, and passes over the same graph repeat."""
    ops, dh, dy = _make(6, 20, 6, "layer", False, "none", seed=33)
    vals = {k: Value.leaf(v, True) for k, v in ops.items()}
    h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals["beta"], EPS)
    other = F.add(h, y)
    seen = []
    for _ in range(2):
        for v in vals.values():
            v.zero_grad()
        if roots == "consumer":
            other.backward(dh)
        else:
            backward([{"h": h, "y": y}[r] for r in roots], [{"h": dh, "y": dy}[r] for r in roots])
        assert h.grad is None
        seen.append([v.grad.clone() for k, v in vals.items() if roots != "h" or k in ("x", "branch")])
    assert all(torch.equal(a, b) for a, b in zip(*seen))
    _check(ops, h.data, y.data, {k: v.grad for k, v in vals.items() if roots != "h" or k in ("x", "branch")},
           dh if roots != "y" else None, dh if roots == "consumer" else dy if "y" in roots else None, "layer", 1.0)


def test_gradients_that_the_groups_do_not_fit(cuda):
    """Parameters whose buffers do not hold the backward's groups, an activation used as one among them, are
    refused before a gradient is taken."""
    G, R, D = 2, 8, 12
    ops, dh, dy = _make(R, D, R, "rms", False, "channel", seed=31)
    for bad in ("gamma", "gate"):
        vals = {k: Value.leaf(v, True) for k, v in ops.items()}
        for k in ("gamma", "gate"):
            if k != bad:
                vals[k].grad = torch.empty(G, D, device="cuda")
        if bad == "gate":
            vals["gate"] = F.add(vals["gate"], vals["gate"])
        with F.param_groups(G):
            h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], None, EPS, kind="rms", gate=vals["gate"])
            with pytest.raises(ValueError, match="does not hold"):
                backward((h, y), (dh, dy))
        assert vals["x"].grad_fresh and vals["branch"].grad_fresh and vals["gamma"].grad_fresh
    x, gamma = Value.leaf(ops["x"], True), Value.leaf(ops["gamma"], True)
    with F.param_groups(G), pytest.raises(ValueError, match="does not hold"):
        F.rmsnorm(x, gamma, EPS).backward(dy)
    assert x.grad_fresh and gamma.grad_fresh


def test_gradients_against_differences(cuda):
    """Along a random direction: the 64-bit function's central difference and the operator's gradients.
    The difference's own error is step^2 / 6 of a third derivative, far below the 1e-4 allowed."""
    ops, dh, dy = _make(8, 24, 4, "layer", True, "sequence", seed=10)
    grads = _run(ops, dh, dy, "layer", 0.5)[2]
    o = {k: v.double() for k, v in ops.items()}
    step = {k: torch.randn_like(v) * 0.1 for k, v in o.items()}

    def value(t):
        q = {k: v + t * step[k] for k, v in o.items()}
        p = Norm64(q["branch"], q["post_gamma"], q["post_beta"], True).out * q["gate"].repeat_interleave(4, 0)
        h = q["x"] + 0.5 * p
        y = Norm64(h, q["gamma"], q["beta"], True).out
        return float((h * dh.double()).sum() + (y * dy.double()).sum())

    numeric = (value(1e-4) - value(-1e-4)) / 2e-4
    along = sum(float((grads[k].double() * step[k]).sum()) for k in grads)
    size = sum(float((grads[k].double() * step[k]).abs().sum()) for k in grads)
    assert abs(numeric - along) <= 1e-4 * size


def test_bad_rows_stay_alone(cuda):
    """Rows with NaN or infinities, and rows of zeros, leave every other row's bits as they were."""
    ops, dh, dy = _make(16, 200, 4, "layer", True, "token", seed=12)
    clean = _run(ops, dh, dy, "layer", 1.0)
    ops["x"][3, 5], ops["branch"][7, 0] = float("nan"), float("inf")
    ops["x"][9], ops["branch"][9] = 0.0, 0.0
    h, y, grads = _run(ops, dh, dy, "layer", 1.0)
    keep = [r for r in range(16) if r not in (3, 7, 9)]
    for a, b in ((h, clean[0]), (y, clean[1]), (grads["x"], clean[2]["x"]), (grads["branch"], clean[2]["branch"]),
                 (grads["gate"], clean[2]["gate"])):
        assert torch.equal(a[keep], b[keep])
    assert torch.isnan(y[3]).all() and torch.isnan(y[7]).all() and torch.isfinite(y[9]).all()


def test_seeds_are_not_written(cuda):
    """h is a root and also feeds another op: its seed's tensor stays as it was, and both parts count."""
    ops, dh, dy = _make(10, 32, 10, "layer", False, "none", seed=13)
    vals = {k: Value.leaf(v, True) for k, v in ops.items()}
    h, y = F.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals["beta"], EPS)
    z = F.relu(h)
    keep = dh.clone()
    backward((h, y, z), (dh, dy, dh))
    assert torch.equal(dh, keep)
    both = torch.where(h.data > 0, dh + dh, dh)
    want = _run(ops, both, dy, "layer", 1.0)[2]
    assert all(torch.equal(vals[k].grad, want[k]) for k in want)


def test_seeds_of_any_strides(cuda):
    ops, _, _ = _make(10, 32, 10, "layer", False, "none", seed=16)
    dh, dy = torch.ones(1, device="cuda").expand(10, 32), torch.randn(32, 10, device="cuda").t()
    want = _run(ops, dh.clone(memory_format=torch.contiguous_format), dy.contiguous(), "layer", 1.0)[2]
    got = _run(ops, dh, dy, "layer", 1.0)[2]
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_captured_and_on_another_stream(cuda):
    ops, dh, dy = _make(400, 512, 100, "rms", True, "sequence", seed=14)
    want = _run(ops, dh, dy, "rms", 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(ops, dh, dy, "rms", 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [GraphedStep(lambda: _run(ops, dh, dy, "rms", 1.0)) for _ in range(2)]
    for res in (got, graphs[0](), graphs[1](), graphs[0]()):
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
        assert all(torch.equal(res[2][k], want[2][k]) for k in want[2])


@pytest.mark.parametrize("R,D", [(1, 16), (50, 33), (300, 512), (7, 4100)])
def test_rmsnorm(cuda, R, D):
    ops, _, dy = _make(R, D, 1, "rms", False, "none", seed=15)
    x, gamma = Value.leaf(ops["x"], True), Value.leaf(ops["gamma"], True)
    y = F.rmsnorm(x, gamma, EPS)
    y.backward(dy)
    norm = Norm64(ops["x"].double(), ops["gamma"].double(), None, False)
    assert torch.all((y.data.double() - norm.out).abs() <= norm.err_out)
    want, err = norm.back(dy.double(), torch.zeros_like(norm.hat))
    assert torch.all((x.grad.double() - want).abs() <= err + E * want.abs())
    terms = dy.double() * norm.hat
    err = (dy.double().abs() * norm.err_hat).sum(0) + (R + 60) * E * terms.abs().sum(0)
    assert torch.all((gamma.grad.double() - terms.sum(0)).abs() <= err)


def test_no_rows(cuda):
    """The C entry with R == 0: stored parameter gradients become zeros, added ones stay."""
    from nnb import check, grad_outs, lib
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    outs = grad_outs(None, None, None, None, None, (a.data_ptr(), 0, 1), (b.data_ptr(), 0, 0))
    check(lib().nnb_residual_norm_bwd(torch.cuda.current_stream().cuda_stream, 0, 8, 1, 0, 0, 1.0, None, None, None, None,
                                      None, None, None, a.data_ptr(), None, outs))
    assert torch.equal(a, torch.zeros(8, device="cuda")) and torch.equal(b, torch.ones(8, device="cuda"))


def test_backward_after_one_that_failed(cuda):
    """A pass that stops between y's rule and h's leaves nothing for the next pass, from h alone."""
    def leaves():
        g = torch.Generator(device="cuda").manual_seed(3)
        return [Value(torch.randn(*s, generator=g, device="cuda"), True) for s in ((6, 16), (6, 16), (16,), (16,))]

    def fail(_):
        raise RuntimeError("a rule that fails")

    seed = torch.ones(6, 16, device="cuda")
    broken, fresh = leaves(), leaves()
    h, y = F.residual_norm(*broken)
    failing = Value.node(seed.clone(), (h,), fail)
    with pytest.raises(RuntimeError, match="a rule that fails"):
        backward((y, failing), (seed, seed))       # rules run in the order y, failing, h or failing, y, h
    with pytest.raises(RuntimeError, match="a rule that fails"):
        backward((failing, y), (seed, seed))
    backward((h,), (seed,))
    h, _ = F.residual_norm(*fresh)
    backward((h,), (seed,))
    for a, b in zip(broken[:2], fresh[:2]):
        assert torch.equal(a.grad, b.grad)
