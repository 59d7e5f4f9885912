"""The block operators' autograd nodes (block_ops) outside an ordinary backward pass: called by themselves, on other streams, with
gradients and saved tensors that are not what their forward had."""
import pytest
import torch

from gpu_helpers import DEV

pytestmark = pytest.mark.gpu


def rnd(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def rng_of(seed, step=3):
    return torch.tensor([seed, step], device=DEV)


def nodes(dtype=torch.bfloat16):
    """(name, its node, its upstream gradients) of each operator."""
    from loopback_amd import block_ops as ops
    x, y, w, g = (rnd(s, dtype, k).requires_grad_() for k, s in enumerate(((3, 50, 136), (3, 50, 136), (136,), (3, 1, 136))))
    dh, dn = rnd((3, 50, 136), dtype, 6), rnd((3, 50, 136), dtype, 7)
    yield "dropout", ops.dropout(x, 0.3, rng_of(1)).grad_fn, [dh]
    h, _ = ops.block_join(x, y, post_weight=w, gate=g, dropout=0.1, rng=rng_of(2), pre_weight=w)
    yield "join", h.grad_fn, [dh, dn]
    if dtype is not torch.float32:
        up, down = rnd((2 * 72, 136), dtype, 8, 0.1).requires_grad_(), rnd((136, 72), dtype, 9, 0.1).requires_grad_()
        yield "ffn", ops.gated_ffn(x, up, down).grad_fn, [dh]


def test_on_the_callers_stream():
    """A node that is called by itself works on its caller's stream: captured there, each replay gives the eager call's results for
    what the gradients then hold."""
    for name, node, grads in nodes():
        print(f"case stream {name}", flush=True)
        call = lambda: [t for t in node(*grads) if t is not None]
        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                call()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = call()
            for k in range(3):
                for g in grads:
                    g.mul_(-0.5)
                want = [t.clone() for t in call()]
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), (name, k)


def test_a_gradient_of_another_shape_or_type():
    """What a program hands to a node itself is checked before a kernel indexes by it: dropout takes the gradient's own type and rows,
    the feed-forward block's has to be its output's."""
    from loopback_amd import block_ops as ops
    x, rng = rnd((6, 40), torch.bfloat16, 1).requires_grad_(), rng_of(3)
    node = ops.dropout(x, 0.5, rng).grad_fn
    *_, (_, *block) = nodes()
    scale = torch.tensor(2.0, device=DEV)
    with torch.no_grad():
        for g in (rnd((6, 40), torch.float32, 2), rnd((6, 40), torch.float16, 3), rnd((3, 24), torch.bfloat16, 4),
                  rnd((6, 40), torch.float64, 5), rnd((0, 40), torch.bfloat16, 6), rnd((6, 0), torch.bfloat16, 7), rnd((), torch.float32, 8)):
            got, _ = node(g)   # and of rng
            keep = ops.keep_mask(g.shape, 0.5, rng)
            assert got.dtype is g.dtype and torch.equal(got, torch.where(keep, g * scale.to(g.dtype), 0.0)), g.shape
        node, (dy,) = block
        assert "Ffn" in node.name()
        node(dy)
        for bad in (dy[:2], dy[..., :64], dy.view(-1)):
            with pytest.raises(RuntimeError, match="wrong shape"):
                node(bad)


@pytest.mark.parametrize("change", [lambda t: t.flatten()[:1].clone(), lambda t: t.repeat(*t.shape[:-1], 2) if t.dim() else t,
                                    lambda t: t.to(torch.int16), lambda t: t.cpu()])
def test_saved_tensors_that_a_hook_changed(change):
    """Each saved tensor in turn comes back from a saved-tensor hook with another shape, type or device: the backward is refused."""
    from loopback_amd import block_ops as ops
    x, y, w, g = (rnd(s, torch.bfloat16, k).requires_grad_() for k, s in enumerate(((6, 40), (6, 40), (40,), (6, 40))))
    up, down = rnd((2 * 20, 40), torch.bfloat16, 8, 0.1).requires_grad_(), rnd((40, 20), torch.bfloat16, 9, 0.1).requires_grad_()
    odd, odd_up = rnd((6, 39), torch.bfloat16, 5).requires_grad_(), rnd((2 * 20, 39), torch.bfloat16, 6, 0.1).requires_grad_()
    odd_down = rnd((40, 19), torch.bfloat16, 7, 0.1).requires_grad_()
    calls = {"dropout": lambda: ops.dropout(x, 0.5, rng_of(1)),
             "join": lambda: sum(ops.block_join(x, y, post_weight=w, gate=g, dropout=0.5, rng=rng_of(2), pre_weight=w)),
             "ffn": lambda: ops.gated_ffn(x, up, down), "odd": lambda: ops.gated_ffn(odd, odd_up[:38], odd_down)}
    for name, call in calls.items():
        counted = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: counted.append(t) or t, lambda t: t):
            out = call()
        out.float().sum().backward()
        for k in range(len(counted)):
            print(f"case changed {name} {k}", flush=True)
            seen = []

            def unpack(t, k=k):
                seen.append(t)
                return change(t) if len(seen) - 1 == k else t

            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
                out = call()
            with pytest.raises((RuntimeError, IndexError)):
                out.backward(torch.ones_like(out))
                torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [8, 40, 200, 768, 1001])
def test_infinite_in_the_last_row(d, dtype):
    """An infinity in the last of a few rows, which the lanes of rows past the end look at too, gives the gate the gradient of the
    formula: infinite in its column, finite in the others."""
    from loopback_amd import block_ops as ops
    print(f"case infinite {d} {dtype}", flush=True)
    for shape, gshape in (((3, d), (d,)), ((2, 3, d), (2, 1, d)), ((1, d), (d,))):
        x, y, dh = (rnd(shape, dtype, k) for k in (1, 2, 3))
        gate = rnd((d,), dtype, 4).expand(gshape).contiguous().requires_grad_()
        y.view(-1, d)[-1, 5] = float("inf")
        dh.view(-1, d)[-1, 5] = 2.0
        h, _ = ops.block_join(x, y, gate=gate)
        got, = torch.autograd.grad(h, gate, dh)
        want = (dh.double() * y.double()).flatten(0, -2).sum(0) if len(gshape) == 1 else (dh.double() * y.double()).sum(1, keepdim=True)
        assert want.isinf().sum() == 1 and torch.equal(got.isinf(), want.isinf()) and not got.isnan().any(), (shape, got, want)


def test_offloaded_and_checkpointed():
    """Saved tensors kept on the host, and a pass computed again by checkpointing (both kinds), give the plain pass's bits."""
    from torch.utils.checkpoint import checkpoint
    from loopback_amd import block_ops as ops
    for d, n in ((136, 72), (65, 31)):   # aligned rows, and copies that are
        x, y, w = (rnd(s, torch.bfloat16, k).requires_grad_() for k, s in enumerate(((70, d), (70, d), (d,))))
        up, down = rnd((2 * n, d), torch.bfloat16, 8, 0.1).requires_grad_(), rnd((d, n), torch.bfloat16, 9, 0.1).requires_grad_()
        dh, rng, leaves = rnd((70, d), torch.bfloat16, 6), rng_of(4), (x, y, w, up, down)

        def run(x, y, w, up, down):
            h, m = ops.block_join(x, y, post_weight=w, gate=w, dropout=0.2, rng=rng, site=1, pre_weight=w)
            return h + ops.dropout(ops.gated_ffn(m, up, down), 0.3, rng, site=2)

        want = torch.autograd.grad(run(*leaves), leaves, dh)
        with torch.autograd.graph.save_on_cpu():
            out = run(*leaves)
        got = [torch.autograd.grad(out, leaves, dh)]
        got += [torch.autograd.grad(checkpoint(run, *leaves, use_reentrant=False), leaves, dh)]
        for p in leaves:
            p.grad = None
        checkpoint(run, *leaves, use_reentrant=True).backward(dh)
        got += [[p.grad for p in leaves]]
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(g, want)), d
