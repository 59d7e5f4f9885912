"""The feed-forward block's backward far out on its activations: finite gates have finite gradients, whichever form computes them."""
import pytest
import torch

from loopback_amd import block_ops as ops

GATES = [1e19, -1e19, 3e38, -3e38, 1e13, -1e13, 101.0, -101.0, 99.0, -99.0, 3.0, -3.0, 0.0]


def operands(dtype, device="cpu"):
    """One inner column: the gate is x's first column, the up projection half of its second, 1."""
    x = torch.tensor(GATES, dtype=dtype, device=device).unsqueeze(1)
    x = torch.cat((x, torch.ones_like(x)), 1)
    gu = torch.tensor([[1.0, 0.0], [0.0, 0.5]], dtype=dtype, device=device)
    return x, gu, torch.ones(1, 1, dtype=dtype, device=device), torch.ones(len(GATES), 1, dtype=dtype, device=device)


def exact(x, act):
    """The gradients of x's two columns in fp64 (dy 1): u a'(g) and a(g) / 2."""
    g = x[:, 0].detach().double().cpu().requires_grad_()
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    da, = torch.autograd.grad(a.sum(), g)
    return torch.stack((0.5 * da, 0.5 * a.detach()), 1)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_torch_backward(act):
    """The torch form of the backward: fp64's gradients to fp32 round-off (the activation's terms are of at most twice the
    result's size; eight operations, 2^-20), and second derivatives that are finite."""
    x, gu, d, dy = operands(torch.float32)
    x.requires_grad_()
    dx = ops._ffn_backward(dy, x, gu, d, ops.ACTIVATIONS[act], 1)[0]
    ref = exact(x, act)
    assert ((dx.double() - ref).abs() <= 2.0 ** -20 * ref.abs() + 1e-30).all()
    second, = torch.autograd.grad(dx[:, 0].sum(), x)
    assert second.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_kernels_and_torch_form(act):
    """A bf16 backward on the kernels and the same one differentiated (torch operations): both within the two roundings of
    fp64's gradients (2^-8 each, of the projections' gradient and of the result)."""
    x, gu, d, dy = operands(torch.bfloat16, "cuda")
    ref = exact(x, act)
    for create in (False, True):
        v = x.clone().requires_grad_()
        dx, = torch.autograd.grad(ops.gated_ffn(v, gu, d, act), v, dy, create_graph=create)
        off = (dx.double().cpu() - ref).abs()
        assert (off <= 2.02 * 2.0 ** -8 * ref.abs() + 1e-30).all(), (create, dx, ref)

