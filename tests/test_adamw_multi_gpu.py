"""The AdamW step over a parameter list, moments in 32 and in 8 bits, against nnb_adamw_step's bits and
against the formulas in 64 bits.

eps = 2^-24 is half a step of fp32 relative to the value; the 8-bit tolerances count roundings of it.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import nnb
from nnb import TensorShapeError, check, lib, nn
from nnb.autograd import Value
from nnb.graph import GraphedStep

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.02)
LISTS = {
    "one": [1], "block": [256], "odd": [255, 257, 1, 4099, 31], "chunks": [4096, 4097, 8192 + 5, 12],
    "empty": [0, 7, 0, 300], "many": [1 + (i * 37) % 700 for i in range(60)],
    "more than one launch": [1 + (i * 11) % 50 for i in range(1000)],
}


def _params(sizes, seed, shift=0):
    """Parameters and gradients with rows of very different size; shift: elements that the buffers are
    moved off their 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n in sizes:
        scale = 10.0 ** (torch.rand(-(-n // 64) * 64, generator=g, device="cuda").view(-1, 64)[:, :1] * 4 - 4)
        w, gr = (torch.empty(n + shift, device="cuda")[shift:] for _ in range(2))
        w.copy_(torch.randn(n, generator=g, device="cuda"))
        gr.copy_((torch.randn(scale.shape[0], 64, generator=g, device="cuda") * scale).view(-1)[:n])
        p = Value(w, True)
        p.grad = gr
        out.append(p)
    return out


def _corrections(t):
    table = np.zeros(2 * t, np.float32)
    n = lib().nnb_adam_bias_table(HYPER["beta1"], HYPER["beta2"], table.ctypes.data, t)
    return (float(table[2 * n - 2]), float(table[2 * n - 1])) if n < t else (float(table[2 * t - 2]), float(table[-1]))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", LISTS.values(), ids=LISTS.keys())
def test_list_is_bitwise_the_single_steps(cuda, sizes, shift):
    params = _params(sizes, 3, shift)
    opt = nn.AdamW(params, **HYPER)
    single = [(p.data.clone(), torch.zeros_like(p.data), torch.zeros_like(p.data)) for p in params]
    for t in range(1, 4):
        opt.step()
        for p, (w, m, v) in zip(params, single):
            check(lib().nnb_adamw_step(torch.cuda.current_stream().cuda_stream, w.numel(), w.data_ptr(),
                                       p.grad.data_ptr(), m.data_ptr(), v.data_ptr(),
                                       *[ctypes.c_float(x) for x in HYPER.values()], t))
    for p, m, v, want in zip(params, opt.m, opt.v, single):
        for got, ref in zip((p.data, m, v), want):
            assert torch.equal(got.view(torch.int32), ref.view(torch.int32))


def _decode(opt, i):
    """Parameter i's codes, units per element and decoded (m, root) in 64 bits."""
    n, lo = opt.params[i].data.numel(), opt.offsets[i]
    block = torch.arange(n, device="cuda") // opt.BLOCK + lo // opt.BLOCK
    km, kr = opt.m[i].view(-1).double(), opt.v[i].view(-1).double()
    um, ur = opt.unit_m.double()[block], opt.unit_v.double()[block]
    return km, kr, um, ur, km * km.abs() * um, kr * kr * ur


def _check_step8(opt, i, w0, m0, r0, g, t, shrink):
    """Parameter i after a step from the stored (m0, r0): the update in 64 bits and the nearest codes."""
    b1, b2, lr, eps = (float(np.float32(HYPER[k])) for k in ("beta1", "beta2", "lr", "eps"))
    c1, c2 = _corrections(t)
    k1, k2 = float(np.float32(1) - np.float32(b1)), float(np.float32(1) - np.float32(b2))
    m, r = b1 * m0 + k1 * g, torch.sqrt(b2 * r0 * r0 + k2 * g * g)
    # m': the code's value (1), two products and a sum: 4 roundings of at most |b1 m0| + |k1 g|
    em = 4 * E * (b1 * m0.abs() + k1 * g.abs())
    # r': the value (1), its square (twice that, +1), the products (1 and 2), the sum (1): 6 in v, half in r, + sqrt
    er = 4 * E * r
    km, kr, um, ur, ms, rs = _decode(opt, i)
    # stored: within half the gap to the neighbouring square, plus the sums' roundings, plus inverse,
    # product and unit of the code (3 roundings of the value) and the unit's own in both decodings (2)
    assert torch.all((ms - m).abs() <= um * (km.abs() + 0.5) + em + 5 * E * m.abs() + 1e-37)
    assert torch.all((rs - r).abs() <= ur * (kr + 0.5) + er + 5 * E * r + 1e-37)
    # the unit: the computed maximum differs from the exact one by at most the largest error of the block's
    # sums (|max x' - max x| <= max |x' - x|; em does not shrink where b1 m0 and k1 g cancel), plus the
    # division's rounding
    for units, top, err, levels in ((um, m.abs(), em, 127.0 ** 2), (ur, r, er, 255.0 ** 2)):
        for b in range(-(-len(m) // 256)):
            part = slice(256 * b, 256 * b + 256)
            best = float(top[part].max())
            if best < 2.0 ** -101:
                assert float(units[256 * b]) == 0.0
            else:
                assert abs(float(units[256 * b]) - best / levels) <= (float(err[part].max()) + 2 * E * best) / levels
    assert torch.all((kr >= 1) | (r == 0) | (ur == 0))
    # update: lr / c1 and its product (2), m' (em), r' (4), its scale (3), the sum with eps (1), the division (2 ulp
    # = 4): 14 of the step, and two roundings of w
    den = r / math.sqrt(c2) + eps
    step = lr / c1 * m / den
    w = w0 * shrink - step
    tol = lr / c1 * em / den + 14 * E * step.abs() + 2 * E * (w0.abs() + w.abs()) + 1e-37
    assert torch.all((opt.params[i].data.view(-1).double() - w).abs() <= tol)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("sizes", LISTS.values(), ids=LISTS.keys())
def test_8bit_step_against_64_bits(cuda, sizes, shift):
    params = _params(sizes, 5, shift)
    opt = nn.AdamW(params, **HYPER, state_bits=8)
    shrink = float(np.float32(1) - np.float32(HYPER["lr"]) * np.float32(HYPER["weight_decay"]))
    for t in range(1, 4):
        before = [(p.data.view(-1).double(), *_decode(opt, i)[4:]) for i, p in enumerate(params)]
        opt.step()
        for i in [i for i, n in enumerate(sizes) if n][:: max(1, len(sizes) // 20)]:
            _check_step8(opt, i, *before[i], params[i].grad.view(-1).double(), t, shrink)
        for p in params:
            p.grad.mul_(-0.7).add_(p.data, alpha=1e-4)
    for (m, v), i in zip(opt.moments(), range(len(sizes))):
        _, _, _, _, ms, rs = _decode(opt, i)
        assert torch.all((m.view(-1).double() - ms).abs() <= E * ms.abs())
        assert torch.all((v.view(-1).double() - rs * rs).abs() <= 3 * E * rs * rs + 1e-45)


def test_8bit_blocks_keep_to_themselves(cuda):
    """A NaN or an infinity in a gradient spoils its own block of its own tensor and nothing else."""
    for bad in (float("nan"), float("inf")):
        params, clean = _params([600, 600], 9), _params([600, 600], 9)
        params[0].grad[300] = bad
        a, b = nn.AdamW(params, **HYPER, state_bits=8), nn.AdamW(clean, **HYPER, state_bits=8)
        for _ in range(2):
            a.step()
            b.step()
        rest = torch.ones(600, dtype=torch.bool, device="cuda")
        rest[256:512] = False
        for (m, v), (mc, vc), p, c in zip(a.moments(), b.moments(), params, clean):
            keep = rest if p is params[0] else torch.ones_like(rest)
            for x, y in ((m, mc), (v, vc), (p.data, c.data)):
                assert torch.equal(x[keep], y[keep])
        assert torch.isnan(a.moments()[0][0][256:512]).all()


def test_zero_tiny_and_missing_gradients(cuda):
    params = _params([512, 300], 11)
    params[0].grad[:256] = 0.0
    params[0].grad[256:] = 1e-38
    params[1].grad_fresh = True                 # nothing reached it
    start = [p.data.clone() for p in params]
    opt = nn.AdamW(params, **HYPER, state_bits=8)
    opt.step()
    shrink = np.float32(1) - np.float32(HYPER["lr"]) * np.float32(HYPER["weight_decay"])
    for got, p0 in ((params[0].data[:256], start[0][:256]), (params[1].data, start[1])):
        assert torch.equal(got, p0 * float(shrink))
    assert all(torch.isfinite(p.data).all() for p in params)
    assert int(opt.m[0].abs().max()) == 0 and float(opt.unit_m[:2].max()) == 0.0
    assert torch.equal(params[1].grad, torch.zeros(300, device="cuda")) and not params[1].grad_fresh


def test_null_gradient_is_zeros(cuda):
    """The C entry's g[i] == NULL."""
    for bits in (32, 8):
        a, b = _params([700], 13), _params([700], 13)
        b[0].grad.zero_()
        oa, ob = nn.AdamW(a, **HYPER, state_bits=bits), nn.AdamW(b, **HYPER, state_bits=bits)
        ob.step()
        f = lib().nnb_adamw_multi_step if bits == 32 else lib().nnb_adamw8_multi_step
        check(f(torch.cuda.current_stream().cuda_stream, 1, oa._n, (ctypes.c_void_p * 1)(a[0].data.data_ptr()),
                (ctypes.c_void_p * 1)(None), *oa._states, *[ctypes.c_float(x) for x in HYPER.values()], 1))
        assert torch.equal(a[0].data, b[0].data)
        assert torch.equal(oa.flat_m, ob.flat_m) and torch.equal(oa.flat_v, ob.flat_v)


@pytest.mark.parametrize("n", [512, 256 * 5 + 77])
def test_8bit_update_is_rounded_like_the_32bit_one(cuda, n):
    """The first step from weights of zero and without eps is its quotient alone, every operation in it rounded to
    nearest: numpy's fp32 arithmetic gives the same bits."""
    f = np.float32
    g = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(41), device="cuda")
    p = Value(torch.zeros(n, device="cuda"), True)
    p.grad = g
    nn.AdamW([p], lr=3e-3, beta1=0.9, beta2=0.999, eps=0.0, weight_decay=0.0, state_bits=8).step()
    b1, b2, gn = f(0.9), f(0.999), g.cpu().numpy()
    c1, c2 = f(1) - b1, f(1) - b2
    m = (f(1) - b1) * gn
    r = np.sqrt((f(1) - b2) * gn * gn)
    want = (-f(3e-3) / c1 * m) / (r * (f(1) / np.sqrt(c2)))
    assert want.dtype == np.float32
    assert np.array_equal(p.data.cpu().numpy().view(np.int32), want.view(np.int32))


def test_a_refused_step_writes_nothing(cuda):
    """A gradient that nothing reached stands for zeros; where the step is refused, no buffer is filled with them."""
    params = _params([40, 30], 12)
    opt = nn.AdamW(params, **HYPER)
    flat = torch.arange(200.0, device="cuda")
    for grad in (flat.view(4, 50)[:, :10], flat[:50], flat[:80:2]):
        params[0].grad, params[0].grad_fresh = grad, True
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(flat, torch.arange(200.0, device="cuda")) and params[0].grad_fresh and opt.t == 0
    params[0].grad = flat[:40]
    opt.step()
    assert torch.equal(flat[:40], torch.zeros(40, device="cuda")) and float(flat[40]) == 40.0


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_share_memory(cuda, bits):
    """Slices of one buffer that overlap are updated one after the other in the list's order, each with its own
    moments, as one step per entry does."""
    runs = []
    for together in (True, False):
        g = torch.Generator(device="cuda").manual_seed(8)
        flat = torch.randn(20000, generator=g, device="cuda")
        params = []
        for lo, hi in ((0, 9000), (300, 20000), (100, 101), (8999, 9100)):
            params.append(Value(flat[lo:hi], True))
            params[-1].grad = torch.randn(hi - lo, generator=g, device="cuda")
        opts = [nn.AdamW(params, **HYPER, state_bits=bits)] if together else \
            [nn.AdamW([p], **HYPER, state_bits=bits) for p in params]
        for _ in range(3):
            for opt in opts:
                opt.step()
        runs.append([flat] + [t for k in ("m", "v") for opt in opts for t in getattr(opt, k)])
    assert len(runs[0]) == 9 and all(torch.equal(a, b) for a, b in zip(*runs))


def test_same_parameter_twice(cuda):
    """A parameter listed twice is updated twice in order, as one step per entry does."""
    p, = _params([1000], 17)
    q, = _params([1000], 17)
    opt = nn.AdamW([p, p], **HYPER)
    opt.step()
    states = [(torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")) for _ in range(2)]
    for m, v in states:
        check(lib().nnb_adamw_step(torch.cuda.current_stream().cuda_stream, 1000, q.data.data_ptr(), q.grad.data_ptr(),
                                   m.data_ptr(), v.data_ptr(), *[ctypes.c_float(x) for x in HYPER.values()], 1))
    assert torch.equal(p.data, q.data)


def test_8bit_checkpoint_round_trip(cuda):
    params, other = _params([500, 256, 3], 19), _params([500, 256, 3], 23)
    a, b = nn.AdamW(params, **HYPER, state_bits=8), nn.AdamW(other, state_bits=8)
    for _ in range(3):
        a.step()
    saved = [(n, t.cpu().numpy()) for n, t in a.state()]
    b.load_state(saved)
    assert b.t == 3 and math.isclose(b.lr, HYPER["lr"], rel_tol=1e-7)
    for x, y in ((a.flat_m, b.flat_m), (a.flat_v, b.flat_v), (a.unit_m, b.unit_m), (a.unit_v, b.unit_v)):
        assert torch.equal(x, y)
    for name, value in (("m.1", 127.5), ("m.1", -128.0), ("v.1", 256.0), ("v.1", float("nan"))):
        bad = dict(saved)
        bad[name] = bad[name].copy()
        bad[name][0] = value
        before = b.flat_m.clone()
        with pytest.raises(RuntimeError, match="not-codes"):
            b.load_state(list(bad.items()))
        assert torch.equal(before, b.flat_m)
    with pytest.raises(RuntimeError, match="unexpected"):
        nn.AdamW(_params([500, 256, 3], 1)).load_state(saved)


def test_captured_step_and_another_stream(cuda):
    """Replays of a captured step equal eager steps (at the captured step count), on a side stream too."""
    for bits in (32, 8):
        a, b = _params([5000, 77], 29), _params([5000, 77], 29)
        oa, ob = nn.AdamW(a, **HYPER, state_bits=bits), nn.AdamW(b, **HYPER, state_bits=bits)
        oa.step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ob.step()
        torch.cuda.current_stream().wait_stream(side)

        def captured():
            oa.t = 1
            oa.step()

        graph = GraphedStep(captured, warmup=1)
        graph()
        graph()
        for _ in range(3):
            ob.t = 1
            ob.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p.data, q.data)
        assert torch.equal(oa.flat_m, ob.flat_m) and torch.equal(oa.flat_v, ob.flat_v)


def test_step_refusals(cuda):
    p, = _params([64], 31)
    opt = nn.AdamW([p])
    p.grad = torch.zeros(32, device="cuda")
    with pytest.raises(TensorShapeError):
        opt.step()
    p.grad = torch.zeros(64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="float32"):
        opt.step()
    p.grad = torch.zeros(64)
    with pytest.raises(ValueError, match="current CUDA device"):
        opt.step()
    p.grad = torch.zeros(128, device="cuda")[::2]
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()


def test_trainer_refuses_8bit_states(cuda):
    from nnb.train import ShardedTrainer
    model = nn.Transformer(nn.TransformerConfig(vocab_size=16, dim=16, heads=1, layers=1, max_len=8))
    with pytest.raises(ValueError, match="32-bit"):
        ShardedTrainer(model, nn.AdamW(model.parameters(), state_bits=8))
