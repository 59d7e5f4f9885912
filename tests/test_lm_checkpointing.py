"""Activation checkpointing of a Loopback LM with dropout: a forward that its backward computes again draws the masks it drew."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from loopback_amd import lm

CFG = dict(hidden_size=128, num_heads=2, vocab_size=97, prelude=1, loop_blocks=2, loops=2, coda=1, hidden_ratio=2, residual=None,
           dropout=0.2, gate=0.5, post_norm=True)


def make(device="cpu", dtype=torch.float32, **more):
    torch.manual_seed(0)
    return lm.LoopbackLM(lm.LMConfig(**(CFG | more))).to(device, dtype)


def run(model, ids, forward):
    model.zero_grad()
    model.rng[1] = 3
    loss = forward(model, ids, model.next_rng())
    loss.backward()
    return loss.detach(), [p.grad.clone() for p in model.parameters()]


FORWARDS = {
    "model": lambda model, ids, rng, **kw: checkpoint(model, ids, rng, **kw),
    "hidden": lambda model, ids, rng, **kw: lm.ops.next_token_loss(model.head(checkpoint(model.hidden, ids, rng, **kw)), ids),
}


@pytest.mark.parametrize("what", FORWARDS)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_checkpointed_forward(what, device):
    """Loss and gradients are the plain forward's, and the model's generator moves on once; with the next step's masks the
    gradients are others."""
    model = make(device, torch.float32 if device == "cpu" else torch.bfloat16)
    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(5)).to(device)
    want = run(model, ids, lambda m, i, r: m(i, r))
    assert model.rng[1] == 4
    got = run(model, ids, lambda m, i, r: FORWARDS[what](m, i, r, use_reentrant=False))
    assert model.rng[1] == 4 and torch.equal(got[0], want[0])
    assert all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    # the same step without naming its generator
    model.rng[1] = 3
    assert torch.equal(model(ids), want[0]) and model.rng[1] == 4
    other = run(model, ids, lambda m, i, r: m(i))   # the generator after r
    assert not all(torch.equal(a, b) for a, b in zip(other[1], want[1])) and model.rng[1] == 5


def test_repeated_without_its_generator():
    """A forward inside a backward pass that is not given the generator of the one it repeats is refused, and moves nothing on."""
    model, ids = make(), torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(5))
    # a reentrant checkpoint records where an input needs a gradient
    for forward in (lambda: checkpoint(model, ids, use_reentrant=False),
                    lambda: checkpoint(lambda i, one: model(i) * one, ids, torch.ones((), requires_grad=True), use_reentrant=True)):
        model.rng[1] = 0
        loss = forward()
        assert model.rng[1] == 1
        with pytest.raises(RuntimeError, match="next_rng"):
            loss.backward()
        assert model.rng[1] == 1


def test_without_dropout():
    """Models that drop nothing, and evaluation, need no generator, in a repeated forward either."""
    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(5))
    for model in (make(dropout=0.0), make().eval()):
        assert model.next_rng() is None
        want = torch.autograd.grad(model(ids), list(model.parameters()))
        got = torch.autograd.grad(checkpoint(model, ids, use_reentrant=False), list(model.parameters()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_training_forward():
    """The training forward with dropout under torch.compile in one graph: the eager loss, and one step of the generator."""
    model, ids = make(), torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(5))
    want = model(ids)
    model.rng[1] = 0
    torch._dynamo.reset()
    got = torch.compile(model, backend="eager", fullgraph=True)(ids)
    assert torch.allclose(got, want, atol=1e-5) and model.rng[1] == 1
