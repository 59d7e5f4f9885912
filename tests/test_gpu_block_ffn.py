"""The gated feed-forward block (block_ops.gated_ffn) against its formulas in fp64 on the same 16-bit inputs.

Each stage's result is an fp32 sum rounded once, and the stages' roundings before it enter it as independent errors of at most
half a step u (2^-8 in bf16, 2^-11 in fp16) of each term. A result y = sum_k a_k b_k whose a_k carry r such roundings is
therefore within u |y| (its own rounding) + r u sum_k |a_k b_k| (the terms', all at once; never reached) + 1e-5 of the RMS of
sum |a_k b_k| (fp32 round-off). Rounded before: the activations for y and for the down projection's gradient (r = 1); the
gradients of the projections for dx and the gate/up gradient (r = 1, and 2^-15 for the 24-bit values they are formed from)."""
import pytest
import torch

from gpu_helpers import DEV

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rnd(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def unaligned(t):
    out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    out.copy_(t)
    return out


def close(got, ref, terms, dtype, what):
    """ref: the exact sums; terms: the sums of the terms' sizes."""
    u, tiny = HALF[dtype], 2.0 ** -25 if dtype is torch.float16 else 0.0
    tol = u * ref.abs() + (u * (1 + u) + 2.0 ** -15) * terms + 1e-5 * terms.pow(2).mean().sqrt() + tiny
    off = (got.double() - ref).abs()
    assert got.dtype is dtype and got.shape == ref.shape
    assert not (off > tol).any(), (what, (off / tol).max().item(), off.max().item())
    # and on the whole the errors average out: one rounding of the result and one of the terms, 2^-0.5 of half a step each
    assert ref.numel() < 64 or off.norm() <= 1.6 * u * ref.norm() + 1e-30, (what, (off.norm() / ref.norm()).item() / u)


def exact(x, wgu, wd, dy, act):
    n = wd.shape[1]
    x, wgu, wd, dy = (t.detach().double() for t in (x, wgu, wd, dy))
    x, dy = x.reshape(-1, x.shape[-1]), dy.reshape(-1, dy.shape[-1])
    g, u = x @ wgu[:n].t(), x @ wgu[n:].t()
    if act == "silu":
        s = torch.sigmoid(g)
        a, da = g * s, s * (1 + g * (1 - s))
    else:
        k = (2 / torch.pi) ** 0.5
        th = torch.tanh(k * (g + 0.044715 * g ** 3))
        a, da = 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g)
    h, dact = a * u, dy @ wd
    dgu = torch.cat((dact * u * da, dact * a), 1)
    pairs = {"y": (h, wd.t()), "dx": (dgu, wgu), "dw_gate_up": (dgu.t(), x), "dw_down": (dy.t(), h)}
    return {k: (p @ q, p.abs() @ q.abs()) for k, (p, q) in pairs.items()}


def check(t, d, n, m, dtype, act="silu", place=lambda v: v, lead=None):
    from loopback_amd import block_ops as ops
    print(f"case ffn {t}x{d}x{n}x{m} {dtype} {act}", flush=True)
    shape = (t,) if lead is None else lead
    x, wgu, wd = (place(rnd(s, dtype, k, std)).requires_grad_() for s, k, std in
                  (((*shape, d), 1, 1.0), ((2 * n, d), 2, 1.5 * d ** -0.5), ((m, n), 3, n ** -0.5)))
    dy = place(rnd((*shape, m), dtype, 4))
    y = ops.gated_ffn(x, wgu, wd, act)
    assert type(y.grad_fn).__name__ == "_GatedFfnBackward"
    grads = torch.autograd.grad(y, (x, wgu, wd), dy)
    torch.cuda.synchronize()
    ref = exact(x, wgu, wd, dy, act)
    got = dict(zip(("y", "dx", "dw_gate_up", "dw_down"), (y.detach(), *grads)))
    for k, (r, terms) in ref.items():
        close(got[k], r.view(got[k].shape), terms.view(got[k].shape), dtype, k)
    with torch.no_grad():
        y2 = ops.gated_ffn(x, wgu, wd, act)
    close(y2, ref["y"][0].view(y2.shape), ref["y"][1].view(y2.shape), dtype, "y without a backward")
    return y, grads


@pytest.mark.parametrize("t,d,n,m", [(1, 1, 1, 1), (1, 8, 8, 8), (2, 64, 32, 64), (33, 65, 31, 63), (65, 128, 96, 40),
                                     (128, 192, 128, 192), (129, 200, 264, 136), (257, 72, 520, 328), (300, 1001, 333, 77)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_sizes(t, d, n, m, dtype, act):
    check(t, d, n, m, dtype, act)


@pytest.mark.parametrize("t,d,n", [(4096, 768, 2048), (4100, 1032, 1544), (1000, 2048, 5632)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large(t, d, n, dtype):
    """The large tiles, with remainders of a tile in every direction; weight gradients split over the tokens."""
    check(t, d, n, d, dtype)


@pytest.mark.parametrize("t", [1, 2, 3, 7, 8, 16, 17, 31, 32, 48, 64, 65, 100])
def test_few_tokens(t):
    check(t, 768, 2048, 768, torch.bfloat16)


def test_unaligned_and_strided():
    """Rows past an aligned address, and strided inputs and gradients, give the aligned ones' results to the same bound."""
    check(140, 256, 160, 128, torch.bfloat16, place=unaligned)
    check(140, 256, 160, 128, torch.float16, "gelu", place=lambda v: v.t().contiguous().t())
    check(12, 64, 40, 64, torch.bfloat16, lead=(3, 4))
