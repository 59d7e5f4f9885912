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
