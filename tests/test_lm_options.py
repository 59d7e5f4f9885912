"""The language model's options from block_ops (fused feed-forward, norms after a block, gates, residual scale, dropout): on the
CPU in torch operations, on the GPU on the kernels, one training step of everything together."""
import pytest
import torch

from loopback_amd import block_ops, lm

SMALL = dict(hidden_size=128, num_heads=2, vocab_size=97, prelude=1, loop_blocks=2, loops=2, coda=1, hidden_ratio=2)
ALL = dict(ffn="fused", post_norm=True, gate=0.5, residual_scale=0.7, dropout=0.2)


def make(device="cpu", dtype=torch.float32, seed=0, residual=None, **options):
    """residual None, plain addition: Loopback's read runs on the GPU alone, and not in fp64."""
    torch.manual_seed(seed)
    return lm.LoopbackLM(lm.LMConfig(**SMALL, residual=residual, **options)).to(device, dtype)


def ids_of(b, t, device="cpu"):
    return torch.randint(0, 97, (b, t), generator=torch.Generator().manual_seed(5)).to(device)


def test_defaults_are_what_they_were():
    """Without options the model has the parameters, buffers and results it had; an option adds its own alone."""
    plain = make()
    names = set(plain.state_dict())
    assert not any(w in n for n in names for w in ("post", "gate.", "rng")) and not any(b.joined for b in plain.prelude)
    more = make(**ALL)
    added = set(more.state_dict()) - names
    assert added == {f"{b}.{p}" for b in ("prelude.0", "middle.0", "middle.1", "coda.0")
                     for p in ("attn_post.weight", "mlp_post.weight", "attn_gate", "mlp_gate")} | {"rng"}
    ids = ids_of(2, 9)
    fused = make(ffn="fused")
    assert torch.allclose(fused(ids), plain(ids), atol=1e-6)   # the same products; the CPU runs torch's
    scaled = make(residual_scale=1.0, gate=1.0)
    assert torch.allclose(scaled(ids), plain(ids), atol=1e-6)
    for bad in ({"ffn": "x"}, {"dropout": 1.0}, {"dropout": -0.1}):
        with pytest.raises(ValueError):
            lm.LMConfig(**bad)


def test_block_formula():
    """A block with every option is its formula, and a norm that is hooked is called."""
    cfg = lm.LMConfig(**SMALL, **(ALL | {"dropout": 0.0}))
    torch.manual_seed(1)
    blk = lm.Block(cfg)
    with torch.no_grad():
        for p in blk.parameters():
            p += 0.1 * torch.randn(p.shape)
    x = torch.randn(2, 5, 128)
    h = x + 0.7 * blk.attn_gate * blk.attn_post(blk.attn(blk.attn_norm(x)))
    ref = h + 0.7 * blk.mlp_gate * blk.mlp_post(blk.mlp(blk.mlp_norm(h)))
    assert torch.allclose(blk(x), ref, atol=1e-5)
    seen = []
    for m in (blk.mlp_norm, blk.attn_post, blk.mlp.down):
        m.register_forward_hook(lambda m, i, o: seen.append(m))
    assert torch.allclose(blk(x), ref, atol=1e-5) and len(seen) == 3


def test_dropout_steps():
    """Training forwards draw new masks and count them; the same state gives the same loss; evaluation drops nothing. A later
    forward does not change an earlier one's backward."""
    model, ids = make(dropout=0.3), ids_of(2, 9)
    state = {k: v.clone() for k, v in model.state_dict().items()}
    a, b = model(ids), model(ids)
    assert a != b and model.rng[1] == 2
    a.backward()
    first = model.embed.weight.grad.clone()
    model.load_state_dict(state)
    model.zero_grad()
    again = model(ids)
    again.backward()
    assert again == a and torch.equal(model.embed.weight.grad, first)
    model.eval()
    with torch.no_grad():
        assert model(ids) == model(ids) == make()(ids) and model.rng[1] == 1


def test_gradients_against_differences():
    """The model's gradient along a random direction is the loss's central difference, in fp64."""
    model, ids = make(dtype=torch.float64, **ALL), ids_of(2, 7)
    state = model.rng.clone()

    def loss():
        model.rng.copy_(state)
        logits = model.head(model.hidden(ids))   # the model's own loss is fp32
        return torch.nn.functional.cross_entropy(logits[:, :-1].reshape(-1, 97), ids[:, 1:].reshape(-1))

    params = [p for p in model.parameters()]
    grads = torch.autograd.grad(loss(), params)
    g = torch.Generator().manual_seed(3)
    way = [torch.randn(p.shape, generator=g, dtype=torch.float64) for p in params]
    exact = sum((a * b).sum() for a, b in zip(grads, way))
    eps, got = 1e-5, []
    with torch.no_grad():
        for sign in (1, -1):
            for p, w in zip(params, way):
                p += sign * eps * w
            got.append(loss())
            for p, w in zip(params, way):
                p -= sign * eps * w
    # The difference is off by its next term, quadratic in the step: norms of outputs that weights of 0.02 make (0.02^2 times
    # sums of 128, some 1e-2) bend over that size, so the step is far below it. The rotation rounds q and k to fp32, 6e-8 of
    # them, which a step of 1e-5 turns into up to 6e-8 / 2e-5 = 3e-3.
    assert abs((got[0] - got[1]) / (2 * eps) - exact) <= 5e-3 * max(1.0, abs(exact))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("options", [ALL, {"ffn": "fused"}, {"post_norm": True, "dropout": 0.1}, {"gate": 0.3}])
def test_training_step_on_the_kernels(dtype, options, monkeypatch):
    """Loss and gradients on the kernels are no further from the same model in fp64 than on torch's operations (the same masks),
    to a fifth."""
    print(f"case lm options {options} {dtype}", flush=True)
    model, ids = make("cuda", dtype, **options), ids_of(3, 65, "cuda")
    state = {k: v.clone() for k, v in model.state_dict().items()}

    def step(m):
        m.load_state_dict({k: v.to(m.embed.weight.dtype) if v.is_floating_point() else v for k, v in state.items()})
        loss = m(ids)
        return loss.detach().double(), [g.double() for g in torch.autograd.grad(64.0 * loss, list(m.parameters()))]

    nodes, H = [], block_ops.H
    counted = lambda name: lambda *a: nodes.append((name, a[-1])) or getattr(H, name)(*a)
    monkeypatch.setattr(block_ops, "H", type("Counted", (), {n: staticmethod(counted(n)) for n in ("join", "dropout", "gated_ffn")}))
    got = step(model)
    assert set(nodes) == {(n, True) for n, on in (("gated_ffn", "ffn" in options), ("join", len(options) > 1 or "ffn" not in options),
                                                  ("dropout", "dropout" in options)) if on}
    again = step(model)
    assert got[0] == again[0] and all(torch.equal(a, b) for a, b in zip(got[1], again[1]))
    monkeypatch.setattr(block_ops, "native", lambda *a, **k: False)
    ref = step(model)
    monkeypatch.undo()
    monkeypatch.setattr(lm.ops, "native", lambda *a, **k: False)
    monkeypatch.setattr(block_ops, "native", lambda *a, **k: False)
    big = make("cpu", torch.float64, **options)
    ids = ids.cpu()
    state = {k: v.cpu() for k, v in state.items()}
    exact = step(big)
    far = lambda a: torch.stack([(p.cpu() - q).norm() / (q.norm() + 1e-9) for p, q in zip(a[1], exact[1])])
    # gradients pass through the model's other 16-bit operations alike: the largest distance of any parameter's
    assert far(got).max() <= 1.2 * far(ref).max() + 1e-3, (far(got), far(ref))
    assert abs(got[0].cpu() - exact[0]) <= 1.2 * abs(ref[0].cpu() - exact[0]) + 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("residual", ["delta_attnres", None])
def test_captured_training_pass(residual):
    """Loss and gradients of the model with every option as one captured graph: each replay gives what the eager pass gives from
    the same generator's state, with eager work between the replays."""
    model, ids = make("cuda", torch.bfloat16, residual=residual, **ALL), ids_of(2, 64, "cuda")
    params = list(model.parameters())

    def step():
        loss = model(ids)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    start = model.rng.clone()
    eager = [[t.clone() for t in step()] for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    model.rng.copy_(start)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager[k]):
            assert torch.equal(a, b), k
        assert model.rng[1] == start[1] + k + 1 and torch.isfinite(torch.randn(1000, device="cuda").sum())
