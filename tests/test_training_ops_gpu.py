"""The residual norm, the vocabulary projection's loss and the list AdamW together, as a training step of a
Transformer runs them."""
import itertools
import math

import pytest
import torch

from nnb import functional as F
from nnb import nn
from nnb.autograd import Value
from nnb.train import ShardedTrainer

pytestmark = pytest.mark.gpu

CONFIGS = [nn.ResidualConfig(norm, post, scale, rs)
           for norm, post, (scale, rs) in itertools.product(("layer", "rms"), (False, True), ((None, 1.0), (0.3, 0.5)))]


def _model(residual, layers=2, V=97, T=16, dropout=0.0, seed=3):
    cfg = nn.TransformerConfig(vocab_size=V, dim=64, heads=1, layers=layers, max_len=T, residual=residual, dropout=dropout)
    return nn.Transformer(cfg, seed=seed)


def _batch(V, B=8, T=16, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(0, V, (B, T), generator=g, device="cuda") for _ in range(2))


def _reference(model, ids, targets, r):
    """The same network with torch's own operations in 64 bits: (loss, gradients by name)."""
    params = {n: p.data.double().requires_grad_() for n, p in model.named_parameters()}
    D, T = model.config.dim, ids.shape[1]

    def norm(a, name):
        if r.norm == "layer":
            var, mean = torch.var_mean(a, -1, correction=0, keepdim=True)
            return (a - mean) / torch.sqrt(var + 1e-5) * params[name + "gamma"] + params[name + "beta"]
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-5) * params[name + "gamma"]

    def linear(a, name):
        return a @ params[name + "weight"].t() + params[name + "bias"]

    def join(x, branch, post, gate):
        if r.post_norm:
            branch = norm(branch, post)
        if r.layer_scale is not None:
            branch = branch * params[gate]
        return x + r.residual_scale * branch

    h = params["embed.weight"][ids] + model.pos.pe.data[:T].double()
    causal = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    for i in range(len(model.blocks)):
        b = f"blocks.{i}."
        y = norm(h, b + "ln1.")
        q, k, v = (linear(y, f"{b}attn.{c}.") for c in "qkv")
        s = (q @ k.transpose(1, 2) / math.sqrt(D)).masked_fill(~causal, -math.inf)
        h = join(h, linear(torch.softmax(s, -1) @ v, b + "attn.o."), b + "post1.", b + "scale1")
        y = linear(norm(h, b + "ln2."), b + "fc1.")
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        h = join(h, linear(y, b + "fc2."), b + "post2.", b + "scale2")
    logits = linear(norm(h, "ln_f."), "head.")
    loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten())
    return loss, dict(zip(params, torch.autograd.grad(loss, list(params.values()))))


@pytest.mark.parametrize("residual", CONFIGS, ids=str)
def test_model_gradients(cuda, residual):
    """Loss and every gradient of a two-block model. Each of its about forty products, norms and softmaxes is
    off by at most about 2e-6 of its values' size (the bounds of their own tests), so 40 x 2e-6 of each
    tensor's largest entry, doubled for the paths that join in the residual stream."""
    model = _model(residual)
    ids, targets = _batch(97)
    want, grads = _reference(model, ids, targets, residual)
    loss = model.loss(ids, targets)
    loss.backward()
    assert abs(float(loss.data) - float(want.detach())) <= 1.6e-4
    for name, p in model.named_parameters():
        assert not p.grad_fresh, name
        top = float(grads[name].abs().max())
        # (the attention's key bias has no gradient but rounding: its size is the other biases')
        if name.endswith("attn.k.bias"):
            top = float(grads[name.replace(".k.", ".v.")].abs().max())
        assert float((p.grad.double() - grads[name]).abs().max()) <= 1.6e-4 * top, name


def test_default_blocks_are_as_before(cuda):
    """Without a ResidualConfig the forward is add and layernorm, and loss() agrees with the kept logits'."""
    model = _model(None)
    ids, targets = _batch(97)
    h = model.pos(model.embed(ids))
    for b in model.blocks:
        h = F.add(h, b.attn(b.ln1(h)))
        h = F.add(h, b.fc2(F.linear_gelu(b.ln2(h), b.fc1.weight, b.fc1.bias)))
    logits = model.head(model.ln_f(h))
    assert torch.equal(model(ids).data, logits.data)
    kept = F.sequence_cross_entropy(logits, targets)
    assert abs(float(model.loss(ids, targets).data) - float(kept.data)) <= 1e-5 * float(kept.data)


def test_standalone_block(cuda):
    model = _model(CONFIGS[-1], layers=1)
    ids, _ = _batch(97)
    h = model.pos(model.embed(ids))
    block = model.blocks[0]
    alone = block(h)
    chained, y = block.advance(h, block.ln1(h), model.ln_f)
    assert torch.equal(alone.data, chained.data) and torch.equal(y.data, model.features(ids).data)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(cuda, bits):
    """Several steps: the optimizer moves every parameter by the formula's step from the gradients it was
    given, and a second run of the same steps has the same bits."""
    runs = []
    for _ in range(2):
        model = _model(CONFIGS[-1], seed=9)
        opt = nn.AdamW(model.parameters(), lr=1e-3, state_bits=bits)
        for step in range(3):
            ids, targets = _batch(97, seed=step)
            model.zero_grad()
            model.loss(ids, targets).backward()
            before = [p.data.clone() for p in model.parameters()]
            opt.step()
            assert all(torch.isfinite(p.data).all() for p in model.parameters())
            # a step is at most lr (1 - beta1) / sqrt(1 - beta2) = 3.17 lr, and the decay lr 0.01 |w|, |w| < 10 here;
            # an 8-bit root may be stored half a code (0.2 % near the top) low
            moved = [float((p.data - b).abs().max()) for p, b in zip(model.parameters(), before)]
            assert all(0 < m <= 1e-3 * (3.3 + 0.01 * 10) for m in moved)
        runs.append([p.data.clone() for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_sharded_trainer_with_the_fused_loss(cuda):
    """The data-parallel step with the model's own loss: close to the step with kept logits, captured and
    replayed with the same bits, and one shard's gradients independent of the others."""
    ids, targets = _batch(97)
    flats = []
    for fused, captured in ((True, False), (True, True), (False, False)):
        model = _model(CONFIGS[5], seed=11)
        trainer = ShardedTrainer(model, nn.AdamW(model.parameters(), lr=1e-3), shards=4, fused_loss=fused)
        if captured:
            step = trainer.capture(ids, targets, warmup=1)
            losses = [float(step()) for _ in range(2)][-1:]
        else:
            losses = [float(trainer.step(ids, targets)) for _ in range(3)][-1:]
        flats.append((losses, trainer.flat_w.clone(), trainer.shard_grads.clone()))
    assert flats[0][0] == flats[1][0] and torch.equal(flats[0][1], flats[1][1])
    scale = float(flats[2][2].abs().max())
    assert float((flats[0][2] - flats[2][2]).abs().max()) <= 5e-3 * scale
    # after three Adam steps of 1e-3 no weight may differ by more than their whole way
    assert float((flats[0][1] - flats[2][1]).abs().max()) <= 6e-3


def test_token_losses_of_a_model(cuda):
    model = _model(CONFIGS[4])
    ids, targets = _batch(97)
    targets[0, :5] = -100
    features = Value.leaf(model.features(ids).data, False)
    rows, mean = F.linear_token_losses(features, Value.leaf(model.head.weight.data), Value.leaf(model.head.bias.data), targets)
    assert rows.shape == targets.shape and float(rows[0, :5].abs().max()) == 0.0
    assert abs(float(mean) - float(model.loss(ids, targets).data)) <= 1e-6 * float(mean)


def _first_step(fused, ids, targets, shards=4):
    """(shard gradients by parameter name, flat shard gradients) of a trainer's first step."""
    model = _model(CONFIGS[5], seed=11)
    trainer = ShardedTrainer(model, nn.AdamW(model.parameters(), lr=1e-3), shards=shards, fused_loss=fused)
    trainer.step(ids, targets)
    names = [n for n, _ in model.named_parameters()]
    return dict(zip(names, trainer.shard_grads.split(trainer.sizes, dim=1))), trainer.shard_grads


def test_fused_loss_gradients_per_parameter(cuda):
    """Each shard's gradient of each parameter, with and without the kept logits: both are within 1.6e-4 of the
    exact one's largest entry (test_model_gradients), so within twice that of one another's (and 1.6e-4 of the
    tolerance for taking the other form's entry as the size)."""
    ids, targets = _batch(97)
    fused, kept = (_first_step(f, ids, targets)[0] for f in (True, False))
    for name, want in kept.items():
        size = kept[name.replace(".k.", ".v.")] if name.endswith("attn.k.bias") else want
        top = size.abs().amax(1)
        assert torch.all(top > 0), name
        assert torch.all((fused[name] - want).abs().amax(1) <= 3.3e-4 * top), name


def test_fused_loss_shards_do_not_depend_on_one_another(cuda):
    """A shard's gradients have the same bits whatever the other shards' rows are, and when the batch is split over
    two ranks (two groups of a half batch each, as a rank runs them)."""
    ids, targets = _batch(97)
    _, want = _first_step(True, ids, targets)
    other_ids, other_targets = _batch(97, seed=77)
    for z in range(4):
        rows = slice(2 * z, 2 * z + 2)
        mixed, mixed_targets = other_ids.clone(), other_targets.clone()
        mixed[rows], mixed_targets[rows] = ids[rows], targets[rows]
        assert torch.equal(_first_step(True, mixed, mixed_targets)[1][z], want[z])
    norm = torch.tensor([1.0 / ids.numel()], device="cuda")
    for half in (0, 1):
        model = _model(CONFIGS[5], seed=11)
        for p in model.parameters():
            p.grad, p.grad_fresh = torch.empty(2, p.data.numel(), device="cuda"), True
        rows = slice(4 * half, 4 * half + 4)
        with F.param_groups(2):
            model.loss(ids[rows], targets[rows], grad_norm=norm).backward()
        got = torch.cat([p.grad for p in model.parameters()], dim=1)
        assert torch.equal(got, want[2 * half: 2 * half + 2])
