"""What is measured of the language-model training operators: cases, inputs, plain forms, exact values.

Three operators of a language model's training step, in the order the step meets them:

``residual_norm``   the residual sum after a block joined with the norm before the next one:
                    h = x + scale * gate * post(branch), y = norm(h), with its gradients;
``linear_cross_entropy``  the vocabulary projection and its softmax cross entropy without keeping the
                    logits, with its gradients (or each token's loss alone, for evaluation);
``adamw``           one AdamW step over a model's whole parameter list, the moments in 32 or in 8 bits.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true
it calls the framework. ``exact`` is the definition in 64 bits, written apart from the plain form.
"""
import pathlib
import sys

import torch

own = False

IGNORE = -100
EPS = 1e-5                      # the norms' epsilon
ADAMW = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 1e-2}
ADAMW_STEPS_BEFORE = 100        # the measured step is the 101st
BLOCK = 256                     # elements that share a scale in the 8-bit states
TINY = 2.0 ** -100              # a block whose largest value is below this is stored as zeros

# The parameter list of the 4-block decoder of this repository's training benchmark (width 512,
# feed-forward 2048, vocabulary 4096): weights, biases and norms as they come.
_DECODER = ("2097152;" + "512;512;262144;512;262144;512;262144;512;262144;512;512;512;1048576;2048;1048576;512;" * 4
            + "512;512;2097152;4096")
# The small image classifier of the same benchmark: two convolutions and two linear layers.
_CLASSIFIER = "288;32;18432;64;401408;128;1280;10"
# A larger decoder, eight blocks of width 1024 and a ragged vocabulary of 50001.
_LARGE = "51201024;" + "1024;1024;4*1048576;4*1024;1024;1024;4194304;4096;4194304;1024;" * 8 + "1024;1024;51201024;50001"


def listed():
    return [
        # a character model's head on a small batch: every launch's latency counts
        {"name": "ce_char_train", "op": "ce", "positions": 256, "dim": 64, "vocab": 65, "bias": True,
         "ignored": 0.0, "smoothing": 0.0, "train": True},
        # the training benchmark's head: 64 sequences of 512 tokens, vocabulary 4096
        {"name": "ce_decoder_train", "op": "ce", "positions": 32768, "dim": 512, "vocab": 4096, "bias": True,
         "ignored": 0.0, "smoothing": 0.0, "train": True},
        # a large, odd vocabulary with padded sequences and label smoothing: the logits would be 800 MB
        {"name": "ce_vocab50k_train", "op": "ce", "positions": 4095, "dim": 1024, "vocab": 50001, "bias": False,
         "ignored": 0.25, "smoothing": 0.1, "train": True},
        # evaluation over a very large vocabulary: each token's loss, no gradients
        {"name": "ce_vocab128k_eval", "op": "ce", "positions": 2048, "dim": 512, "vocab": 131072, "bias": True,
         "ignored": 0.1, "smoothing": 0.0, "train": False},
        # one sequence of a small model: latency
        {"name": "norm_small_train", "op": "norm", "rows": 32, "dim": 64, "kind": "layer", "post": False,
         "gate": "none", "span": 32, "scale": 1.0, "train": True},
        # the training benchmark's residual sums: plain pre-norm blocks
        {"name": "norm_decoder_train", "op": "norm", "rows": 32768, "dim": 512, "kind": "layer", "post": False,
         "gate": "none", "span": 512, "scale": 1.0, "train": True},
        # a wide model with a norm on both sides of the block and a learned gate per channel
        {"name": "norm_wide_gated_train", "op": "norm", "rows": 8190, "dim": 2048, "kind": "rms", "post": True,
         "gate": "channel", "span": 819, "scale": 0.5, "train": True},
        # inference with a gate per sequence (a conditioning vector), odd width
        {"name": "norm_conditioned_eval", "op": "norm", "rows": 12288, "dim": 1001, "kind": "layer", "post": True,
         "gate": "sequence", "span": 256, "scale": 1.0, "train": False},
        # a small classifier's eight tensors: one launch's latency
        {"name": "adamw32_classifier", "op": "adamw", "bits": 32, "tensors": _CLASSIFIER},
        # the training benchmark's decoder
        {"name": "adamw32_decoder", "op": "adamw", "bits": 32, "tensors": _DECODER},
        {"name": "adamw8_decoder", "op": "adamw", "bits": 8, "tensors": _DECODER},
        # a larger decoder with 8-bit moments
        {"name": "adamw8_large", "op": "adamw", "bits": 8, "tensors": _LARGE},
    ]


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is uniform over [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["ce", "norm", "adamw"])
    if op == "ce":
        while True:
            p, d, v = _log_int(rng, 1, 32768), _log_int(rng, 8, 2048), _log_int(rng, 2, 131072)
            if p * v * d <= 4095 * 50001 * 1024 and p * v <= 300_000_000:
                break
        if rng.random() < 0.5:
            d = -(-d // 16) * 16
        return {"op": "ce", "positions": p, "dim": d, "vocab": v, "bias": rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.0, 0.1, 0.9]), "smoothing": rng.choice([0.0, 0.0, 0.1]),
                "train": rng.random() < 0.7}
    if op == "norm":
        while True:
            span, seqs, d = _log_int(rng, 1, 4096), _log_int(rng, 1, 256), _log_int(rng, 16, 8192)
            if span * seqs * d <= 32768 * 512:
                break
        if rng.random() < 0.5:
            d = -(-d // 4) * 4
        return {"op": "norm", "rows": span * seqs, "dim": d, "kind": rng.choice(["layer", "rms"]),
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "sequence", "token"]), "span": span,
                "scale": rng.choice([1.0, 0.5, 0.25]), "train": rng.random() < 0.7}
    total = _log_int(rng, 1000, 100_000_000)
    sizes = []
    for _ in range(_log_int(rng, 1, 200)):
        sizes.append(_log_int(rng, 1, max(2, total // 2)))
        total -= sizes[-1]
        if total <= 2:
            break
    return {"op": "adamw", "bits": rng.choice([32, 8]), "tensors": ";".join(str(n) for n in sizes)}


def _sizes(text):
    """The tensors' lengths of a list such as "512;4*1024;10"."""
    out = []
    for part in text.strip(";").split(";"):
        count, _, n = part.rpartition("*")
        out += [int(n)] * (int(count) if count else 1)
    return out


def _offsets(case):
    """Where each tensor of the list starts in a flat buffer, and the buffer's length."""
    out = [0]
    for n in _sizes(case["tensors"]):
        out.append(out[-1] + -(-n // BLOCK) * BLOCK)
    return out


def work(case):
    if case["op"] == "ce":
        p, d, v = case["positions"], case["dim"], case["vocab"]
        ins = p * d + v * d + (v if case["bias"] else 0)
        passes, products = (2, 3) if case["train"] else (1, 1)
        return {"bytes": 4 * ins * passes + 8 * p + 4, "flops": 2 * products * p * v * d}
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        if case["train"]:       # x, branch, dh, dy in; h, y, dx, dbranch out
            return {"bytes": 4 * 8 * n, "flops": 40 * n}
        return {"bytes": 4 * 4 * n, "flops": 15 * n}
    n = sum(_sizes(case["tensors"]))
    if case["bits"] == 32:      # w, m, v in and out, g in
        return {"bytes": 28 * n, "flops": 15 * n}
    # w and the codes in and out, g in, a scale per block and state in and out, the two moments' values out
    return {"bytes": (8 + 4 + 4 + 8) * n + 16 * (n // BLOCK), "flops": 40 * n}


# ---- inputs ---------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _inputs(case, seed):
    """The case's data on the GPU as plain tensors, from the seed alone."""
    g = _generator(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    def uniform(*shape, lim=1.0):
        return (torch.rand(*shape, generator=g, device="cuda") * 2 - 1) * lim

    if case["op"] == "ce":
        p, d, v = case["positions"], case["dim"], case["vocab"]
        # normed activations, a projection as training makes it, frequent and rare tokens
        t = (torch.rand(p, generator=g, device="cuda") ** 3 * v).long().clamp_(max=v - 1)
        drop = torch.rand(p, generator=g, device="cuda") < case["ignored"]
        drop[0] = False
        t = torch.where(drop, torch.full_like(t, IGNORE), t)
        return {"x": normal(p, d), "w": uniform(v, d, lim=2.0 / d ** 0.5),
                "b": normal(v, std=0.5) if case["bias"] else None, "t": t}
    if case["op"] == "norm":
        r, d, span = case["rows"], case["dim"], case["span"]
        gate_rows = {"none": 0, "channel": 1, "sequence": r // span, "token": r}[case["gate"]]
        layer = case["kind"] == "layer"
        out = {"x": normal(r, d, std=2.0) + uniform(r, 1), "branch": normal(r, d, std=0.7),
               "gamma": 1.0 + uniform(d, lim=0.2), "beta": uniform(d, lim=0.2) if layer else None,
               "post_gamma": 1.0 + uniform(d, lim=0.2) if case["post"] else None,
               "post_beta": uniform(d, lim=0.2) if case["post"] and layer else None,
               "gate": 0.5 + uniform(gate_rows, d, lim=0.5) if gate_rows else None}
        if case["train"]:
            out["dh"], out["dy"] = normal(r, d, std=0.01), normal(r, d, std=0.01)
        return out
    sizes = _sizes(case["tensors"])
    n = sum(sizes)
    # gradients and moments whose size differs from row to row, as in embeddings and norms
    scale = 10.0 ** (uniform((n + 511) // 512, 1) - 3.0)
    spread = lambda a: (a.view(-1, 512) * scale).view(-1)[:n]      # noqa: E731
    padded = scale.numel() * 512
    data = {"w": normal(n, std=0.05), "g": spread(normal(padded)), "m": spread(normal(padded, std=0.3)),
            "v": spread(normal(padded)).square()}
    # one flat buffer per kind, every tensor's part starting on a whole block, zeros between the parts
    out = {}
    for k, t in data.items():
        out[k] = torch.zeros(_offsets(case)[-1], device="cuda")
        for part, lo in zip(t.split(sizes), _offsets(case)):
            out[k][lo:lo + part.numel()] = part
    return out


def prepare(case, seed):
    data = _inputs(case, seed)
    state = {"case": case, "data": data}
    if case["op"] == "adamw" and case["bits"] == 8:
        # the states as a program holds them: codes and one scale per block
        data["m"], data["m_unit"] = _encode_m(data["m"])
        data["v"], data["v_unit"] = _encode_r(data["v"].sqrt())
    if case["op"] == "adamw":
        data["t"] = ADAMW_STEPS_BEFORE
    if own:
        _prepare_own(state)
    return state


# ---- the framework's calls --------------------------------------------------------------------------


def _framework():
    path = str(pathlib.Path(__file__).resolve().parent.parent / "nn-cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nnb.autograd
    import nnb.functional
    import nnb.nn
    return nnb


def _prepare_own(state):
    nnb = state["nnb"] = _framework()
    case, data = state["case"], state["data"]
    leaf = nnb.autograd.Value.leaf
    if case["op"] == "adamw":
        spans = list(zip(_offsets(case), _sizes(case["tensors"])))
        params = [leaf(data["w"][lo:lo + n], True) for lo, n in spans]
        for p, (lo, n) in zip(params, spans):
            p.grad, p.grad_fresh = data["g"][lo:lo + n], False
        opt = nnb.nn.AdamW(params, **ADAMW, state_bits=case["bits"])
        opt.t = data["t"]
        opt.flat_m.copy_(data["m"])
        opt.flat_v.copy_(data["v"])
        if case["bits"] == 8:
            opt.unit_m.copy_(data["m_unit"])
            opt.unit_v.copy_(data["v_unit"])
        state["opt"] = opt
        return
    state["values"] = {k: leaf(t, case["train"]) for k, t in data.items()
                       if t is not None and k not in ("t", "dh", "dy")}


def _run_own(state):
    nnb = state["nnb"]
    case, data = state["case"], state["data"]
    if case["op"] == "adamw":
        opt = state["opt"]
        opt.step()
        m, v = opt.flat_moments()
        return {"w": data["w"], "m": m, "v": v}
    vals = state["values"]
    for v in vals.values():
        if v.requires_grad:
            v.zero_grad()
    if case["op"] == "ce":
        args = vals["x"], vals["w"], vals.get("b"), data["t"], IGNORE, case["smoothing"]
        if not case["train"]:
            tokens, loss = nnb.functional.linear_token_losses(*args)
            return {"loss": loss, "tokens": tokens}
        loss = nnb.functional.linear_cross_entropy(*args)
        loss.backward()
        out = {"loss": loss.data}
    else:
        h, y = nnb.functional.residual_norm(vals["x"], vals["branch"], vals["gamma"], vals.get("beta"), EPS,
                                            kind=case["kind"], post_gamma=vals.get("post_gamma"),
                                            post_beta=vals.get("post_beta"), gate=vals.get("gate"), scale=case["scale"])
        out = {"h": h.data, "y": y.data}
        if case["train"]:
            nnb.autograd.backward((h, y), (data["dh"], data["dy"]))
    if case["train"]:
        out.update({"d" + k: v.grad for k, v in vals.items()})
    return out


# ---- plain forms, 32 bits ------------------------------------------------------------------------------


def run(state):
    case, data = state["case"], state["data"]
    if own:
        out = _run_own(state)
    elif case["op"] == "ce":
        out = _plain_ce(case, data)
    elif case["op"] == "norm":
        out = _plain_norm(case, data)
    else:
        out = _plain_adamw(case, data)
    return dict(sorted(out.items()))


def _plain_ce(case, s):
    x, w, t, ls = s["x"], s["w"], s["t"], case["smoothing"]
    v = w.shape[0]
    logits = x @ w.t()
    if s["b"] is not None:
        logits += s["b"]
    live = t != IGNORE
    count = live.sum()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp_().sum(1).log_() + top[:, 0]
    at = t.clamp(min=0)[:, None]
    nll = lse - logits.gather(1, at)[:, 0]
    if ls:
        nll = (1 - ls) * nll + ls * (lse - logits.mean(1))
    nll = torch.where(live, nll, torch.zeros_like(nll))
    loss = nll.double().sum() / count
    out = {"loss": loss.float().view(1)}
    if not case["train"]:
        out["tokens"] = nll
    else:
        d = (logits - lse[:, None]).exp_()
        d -= ls / v
        d.scatter_add_(1, at, torch.full_like(at, -(1 - ls), dtype=torch.float32))
        d *= torch.where(live, 1.0 / count.float(), torch.zeros_like(lse))[:, None]
        out.update(dx=d @ w, dw=d.t() @ x)
        if s["b"] is not None:
            out["db"] = d.sum(0)
    return out


def _plain_norm_parts(kind, a):
    """The normalised rows and their inverse deviations."""
    c = a - a.mean(1, keepdim=True) if kind == "layer" else a
    inv = (c.square().mean(1, keepdim=True) + EPS).rsqrt()
    return c * inv, inv


def _plain_norm_back(kind, dhat, hat, inv):
    out = dhat - hat * (dhat * hat).mean(1, keepdim=True)
    if kind == "layer":
        out = out - dhat.mean(1, keepdim=True)
    return out * inv


def _plain_norm(case, s):
    kind, scale, d = case["kind"], case["scale"], case["dim"]
    p = s["branch"]
    if case["post"]:
        bhat, binv = _plain_norm_parts(kind, p)
        p = bhat * s["post_gamma"]
        if s["post_beta"] is not None:
            p = p + s["post_beta"]
    gate = s["gate"]
    rows = gate.repeat_interleave(case["rows"] // gate.shape[0], 0) if gate is not None else None
    h = s["x"] + scale * (p * rows if rows is not None else p)
    hat, inv = _plain_norm_parts(kind, h)
    y = hat * s["gamma"]
    if s["beta"] is not None:
        y = y + s["beta"]
    out = {"h": h, "y": y}
    if not case["train"]:
        return out
    dy = s["dy"]
    dx = s["dh"] + _plain_norm_back(kind, dy * s["gamma"], hat, inv)
    out["dx"] = dx
    out["dgamma"] = (dy * hat).sum(0)
    if s["beta"] is not None:
        out["dbeta"] = dy.sum(0)
    dp = dx * scale
    if rows is not None:
        out["dgate"] = (dp * p).view(gate.shape[0], -1, d).sum(1)
        dp = dp * rows
    if case["post"]:
        out["dpost_gamma"] = (dp * bhat).sum(0)
        if s["post_beta"] is not None:
            out["dpost_beta"] = dp.sum(0)
        dp = _plain_norm_back(kind, dp * s["post_gamma"], bhat, binv)
    out["dbranch"] = dp
    return out


def _encode(values, levels):
    """Square-law codes k of non-negative blocks: k^2 * unit is the nearest such value, unit = max / levels^2."""
    top = values.amax(1, keepdim=True)
    unit = torch.div(top, torch.full_like(top, float(levels * levels)))
    inv = torch.div(torch.full_like(top, float(levels * levels)), top)
    t = values * inv
    # the nearest square: k where k^2 - k + 1/2 <= t < k^2 + k + 1/2
    k = ((t.double() - 0.25).clamp_(min=0).sqrt_() + 0.5).floor_().clamp_(max=levels)
    small = top < TINY
    k = torch.where(small | ~(t >= 0.5), torch.zeros_like(k), k)
    return k, torch.where(small, torch.zeros_like(unit), unit)


def _encode_m(m):
    b = m.view(-1, BLOCK)
    k, unit = _encode(b.abs(), 127)
    return (k * b.sign().double()).to(torch.int8).view(-1), unit.view(-1)


def _encode_r(r):
    b = r.view(-1, BLOCK)
    k, unit = _encode(b, 255)
    k = torch.where((b > 0) & (unit > 0), k.clamp(min=1), k)       # a root above zero keeps a code above zero
    return k.to(torch.uint8).view(-1), unit.view(-1)


def _decode(codes, unit):
    k = codes.to(torch.float32).view(-1, BLOCK)
    return (k * k.abs() * unit[:, None]).view(-1)


def _plain_adamw(case, s):
    s["t"] += 1
    b1, b2 = torch.tensor(ADAMW["beta1"], dtype=torch.float32), torch.tensor(ADAMW["beta2"], dtype=torch.float32)
    c1, c2 = float(1 - b1 ** s["t"]), float(1 - b2 ** s["t"])
    keep1, keep2 = float(1 - b1), float(1 - b2)
    b1, b2 = float(b1), float(b2)
    lr = torch.tensor(ADAMW["lr"], dtype=torch.float32)
    shrink = float(1 - lr * torch.tensor(ADAMW["weight_decay"], dtype=torch.float32))
    w, g = s["w"], s["g"]
    if case["bits"] == 8:
        m0, v0 = _decode(s["m"], s["m_unit"]), _decode(s["v"], s["v_unit"]).square()
    else:
        m0, v0 = s["m"], s["v"]
    m = b1 * m0 + keep1 * g
    v = b2 * v0 + keep2 * g * g
    root = v.sqrt()
    w.mul_(shrink).sub_(float(lr) * (m / c1) / (root / c2 ** 0.5 + ADAMW["eps"]))
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        return {"w": w, "m": m, "v": v}
    s["m"], s["m_unit"] = _encode_m(m)
    s["v"], s["v_unit"] = _encode_r(root)
    return {"w": w, "m": _decode(s["m"], s["m_unit"]), "v": _decode(s["v"], s["v_unit"]).square()}


# ---- exact values, 64 bits -----------------------------------------------------------------------------


def exact(case, seed):
    form = {"ce": _exact_ce, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]]
    return dict(sorted(form(case, _inputs(case, seed)).items()))


def _exact_ce(case, s):
    f64 = torch.float64
    x, w = s["x"].to(f64), s["w"].to(f64)
    b = s["b"].to(f64) if s["b"] is not None else torch.zeros(w.shape[0], dtype=f64, device="cuda")
    ls, v, t = case["smoothing"], w.shape[0], s["t"]
    count = int((t != IGNORE).sum())
    tokens = torch.zeros(x.shape[0], dtype=f64, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, 2 ** 27 // v)
    for lo in range(0, x.shape[0], step):
        part, tp = x[lo:lo + step], t[lo:lo + step]
        live = tp != IGNORE
        logp = torch.addmm(b, part, w.t())
        logp = logp - torch.logsumexp(logp, 1, keepdim=True)
        # the target distribution: 1 - ls on the label, ls spread over the vocabulary
        q = torch.full_like(logp, ls / v)
        rows = torch.arange(len(tp), device="cuda")
        q[rows, torch.where(live, tp, 0)] += 1 - ls
        tokens[lo:lo + step] = torch.where(live, -(q * logp).sum(1), 0.0)
        if case["train"]:
            d = (logp.exp() - q) * live[:, None].to(f64) / count
            dx[lo:lo + step] = torch.mm(d, w)
            dw.addmm_(d.t(), part)
            db += d.sum(0)
    out = {"loss": (tokens.sum() / count).view(1)}
    if not case["train"]:
        out["tokens"] = tokens
    else:
        out.update(dx=dx, dw=dw)
        if s["b"] is not None:
            out["db"] = db
    return out


def _exact_norm(case, s):
    f64 = torch.float64
    s = {k: t.to(f64) if t is not None else None for k, t in s.items()}
    names = [k for k in ("x", "branch", "gamma", "beta", "post_gamma", "post_beta", "gate") if s[k] is not None]
    for k in names:
        s[k].requires_grad_(case["train"])

    def norm(a, gamma, beta):
        if case["kind"] == "layer":
            var, mean = torch.var_mean(a, 1, correction=0, keepdim=True)
            return (a - mean) / torch.sqrt(var + EPS) * gamma + beta
        return a / torch.sqrt((a * a).mean(1, keepdim=True) + EPS) * gamma

    p = norm(s["branch"], s["post_gamma"], s["post_beta"]) if case["post"] else s["branch"]
    if s["gate"] is not None:
        n = s["gate"].shape[0]
        p = (p.view(n, case["rows"] // n, case["dim"]) * s["gate"][:, None, :]).view(p.shape)
    h = s["x"] + p * case["scale"]
    y = norm(h, s["gamma"], s["beta"])
    out = {"h": h.detach(), "y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad((h, y), [s[k] for k in names], (s["dh"], s["dy"]))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def _exact_adamw(case, s):
    f64 = torch.float64
    f32 = {k: float(torch.tensor(x, dtype=torch.float32)) for k, x in ADAMW.items()}
    b1, b2, t = f32["beta1"], f32["beta2"], ADAMW_STEPS_BEFORE + 1
    w, g, m, v = (s[k].to(f64) for k in ("w", "g", "m", "v"))
    if case["bits"] == 8:       # the codes that prepare hands over
        (m, m_unit), (r, r_unit) = _encode_m(s["m"]), _encode_r(s["v"].sqrt())
        block = torch.arange(m.numel(), device="cuda") // BLOCK
        m = m.to(f64) * m.to(f64).abs() * m_unit.to(f64)[block]
        v = (r.to(f64) ** 2 * r_unit.to(f64)[block]) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    step = f32["lr"] / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + f32["eps"])
    w = w * (1 - f32["lr"] * f32["weight_decay"]) - step
    if case["bits"] == 8:
        # a few in a million moments lie so near the border between two codes that the sums in 32 and in
        # 64 bits fall on different sides, one code apart: the stored moments have no value in 64 bits
        m = v = None
    return {"w": w, "m": m, "v": v}
