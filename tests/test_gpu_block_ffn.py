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
    assert "FfnNode" in y.grad_fn.name()
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
                                     (128, 192, 128, 192), (5, 1001, 333, 77), (31, 135, 1000, 129), (129, 200, 264, 136), (257, 72, 520, 328), (300, 1001, 333, 77)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_sizes(t, d, n, m, dtype, act):
    check(t, d, n, m, dtype, act)


@pytest.mark.parametrize("t,d,n", [(4096, 768, 2048), (4100, 1032, 1544), (1000, 2048, 5632)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large(t, d, n, dtype):
    """The large tiles, with remainders of a tile in every direction; weight gradients split over the tokens."""
    check(t, d, n, d, dtype)


@pytest.mark.parametrize("columns,rows,k", [(2504, 4001, 300), (760, 16001, 264), (528, 3040, 6061), (200, 300, 72), (1496, 4104, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_products(columns, rows, k, dtype):
    """Each product of the block by itself, its result of `columns` x `rows`, every tile shape among the sizes, whole and in splits;
    one rounding of the fp32 sum (k products, errors of 2^-24 of the partial sums' size each), and nothing past the result."""
    from loopback_amd import block_ops as ops
    lib, code, st = ops.LIB, 1 if dtype is torch.bfloat16 else 2, torch.cuda.current_stream().cuda_stream
    print(f"case products {columns} {rows} {k} {dtype}", flush=True)

    def operand(r, c, seed):   # rows of c elements, in rows of a multiple of 8
        out = torch.zeros((r, (c + 7) // 8 * 8), dtype=dtype, device=DEV)
        out[:, :c] = rnd((r, c), dtype, seed)
        return out, out.shape[1], out[:, :c].double()

    def scratch():
        return torch.empty(max(4, lib.lbk_linear_scratch(columns, rows, k)), device=DEV)

    def test(name, call, ref, terms):
        outs = []
        for _ in range(2):
            out = torch.full((rows + 1, columns), 7.0, dtype=dtype, device=DEV)
            s = scratch()
            assert call(out.data_ptr(), s.data_ptr()) == 0
            torch.cuda.synchronize()
            assert (out[-1] == 7).all(), name
            outs.append(out[:-1])
        assert torch.equal(outs[0], outs[1]), name   # a fixed order
        tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
        off = (outs[0].double() - ref).abs()
        assert not (off > HALF[dtype] * ref.abs() + 1e-5 * terms + tiny).any(), (name, off.max().item())

    (p, lp, pv), (q, lq, qv) = operand(columns, k, 1), operand(rows, k, 2)          # k along both operands' rows
    (pt, lpt, ptv), (qt, lqt, qtv) = operand(k, columns, 3), operand(k, rows, 4)    # the columns, the rows along them
    test("forward", lambda o, s: lib.lbk_linear_fwd(q.data_ptr(), lq, p.data_ptr(), lp, o, columns, s, rows, k, columns, code, st),
         qv @ pv.t().contiguous(), qv.abs() @ pv.abs().t().contiguous())
    test("input gradient", lambda o, s: lib.lbk_linear_dx(q.data_ptr(), lq, pt.data_ptr(), lpt, o, columns, s, rows, k, columns, code, st),
         qv @ ptv, qv.abs() @ ptv.abs())
    test("weight gradient", lambda o, s: lib.lbk_linear_dw(qt.data_ptr(), lqt, pt.data_ptr(), lpt, s, o, k, rows, columns, code, st),
         qtv.t().contiguous() @ ptv, qtv.abs().t().contiguous() @ ptv.abs())


@pytest.mark.parametrize("t", [1, 2, 3, 7, 8, 16, 17, 31, 32, 48, 64, 65, 100])
def test_few_tokens(t):
    check(t, 768, 2048, 768, torch.bfloat16)


def test_unaligned_and_strided():
    """Rows past an aligned address, and strided inputs and gradients, give the aligned ones' results to the same bound."""
    check(140, 256, 160, 128, torch.bfloat16, place=unaligned)
    check(140, 256, 160, 128, torch.float16, "gelu", place=lambda v: v.t().contiguous().t())
    check(12, 64, 40, 64, torch.bfloat16, lead=(3, 4))


def test_gradients_one_at_a_time():
    """Each gradient alone has the bits it has beside the others, and a frozen projection's is not formed; aligned and not."""
    from loopback_amd import block_ops as ops
    for t, d, n, m in ((200, 256, 160, 128), (90, 65, 31, 70)):
        vals = [rnd(s, torch.bfloat16, k, std) for k, (s, std) in enumerate((((t, d), 1.0), ((2 * n, d), d ** -0.5), ((m, n), n ** -0.5)))]
        dy = rnd((t, m), torch.bfloat16, 9)

        def grads(need):
            v = [x.clone().requires_grad_(k in need) for k, x in enumerate(vals)]
            return dict(zip(need, torch.autograd.grad(ops.gated_ffn(*v), [v[k] for k in need], dy)))

        both = grads((0, 1, 2))
        for need in ((0,), (1,), (2,), (0, 2), (1, 2)):
            for k, g in grads(need).items():
                assert torch.equal(g, both[k]), (need, k)


def test_second_derivatives_hooks_and_modes():
    """A backward that is differentiated, batched or under a dispatch mode is torch's operations (a few roundings of 16 bits from
    the torch form's); saved tensors that a hook gives back strided or unaligned reach the kernels as they have to."""
    from loopback_amd import block_ops as ops
    vals = [rnd(s, torch.bfloat16, k, std) for k, (s, std) in enumerate((((5, 64), 1.0), ((48, 64), 0.125), ((64, 24), 0.2)))]
    dy = rnd((5, 64), torch.bfloat16, 9)
    leaf = lambda: [v.clone().requires_grad_() for v in vals]

    def second(fn):
        v = leaf()
        g = torch.autograd.grad(fn(*v), v, dy, create_graph=True)
        return torch.autograd.grad(sum(t.float().pow(2).sum() for t in g), v)

    for a, b in zip(second(ops.gated_ffn), second(lambda *v: ops._ffn_torch(*v, 0))):
        assert (a - b).float().norm() <= 3e-2 * b.float().norm()
    v = leaf()
    y = ops.gated_ffn(*v)
    want = torch.autograd.grad(y, v, dy, retain_graph=True)
    batched = torch.autograd.grad(y, v, torch.stack((dy, 2 * dy)), is_grads_batched=True)
    for a, b in zip(batched, want):
        assert (a[0] - b).float().norm() <= 2e-2 * b.float().norm() and (a[1] - 2 * b).float().norm() <= 4e-2 * b.float().norm()
    for unpack in (lambda t: t.t().contiguous().t() if t.dim() == 2 else t, lambda t: unaligned(t)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            y = ops.gated_ffn(*v)
        for a, b in zip(torch.autograd.grad(y, v, dy), want):
            assert torch.equal(a, b)
    out, tangent = torch.func.jvp(ops.gated_ffn, tuple(vals), tuple(vals))
    assert out.shape == tangent.shape == (5, 64)
    assert torch.func.vmap(ops.gated_ffn, in_dims=(0, None, None))(vals[0].view(5, 1, 64), *vals[1:]).shape == (5, 1, 64)


def test_captured_and_replayed():
    """Forward and backward in a captured graph: every replay gives the eager results, with eager work in between."""
    from loopback_amd import block_ops as ops
    for t, d, n in ((700, 768, 2048), (61, 65, 31), (1, 768, 2048)):
        v = [rnd(s, torch.bfloat16, k, std).requires_grad_() for k, (s, std) in enumerate((((t, d), 1.0), ((2 * n, d), d ** -0.5),
                                                                                            ((d, n), n ** -0.5)))]
        dy = rnd((t, d), torch.bfloat16, 9)

        def step():
            y = ops.gated_ffn(*v)
            with torch.no_grad():
                z = ops.gated_ffn(*v, activation="gelu")
            return [y.detach(), z, *torch.autograd.grad(y, v, dy)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for k in range(3):
            with torch.no_grad():
                v[0].mul_(-1.0)
            ref = [r.clone() for r in step()]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, ref):
                assert torch.equal(a, b), (t, k)


def test_not_finite_rows_stay_alone():
    """A token with an infinity or NaN does not reach the others, forward or backward."""
    from loopback_amd import block_ops as ops
    for t in (3, 40, 300):
        x, gu, d = rnd((t, 128), torch.bfloat16, 1), rnd((192, 128), torch.bfloat16, 2, 0.1), rnd((64, 96), torch.bfloat16, 3, 0.1)
        dy = rnd((t, 64), torch.bfloat16, 4)
        x2, dy2 = x.clone(), dy.clone()
        x2[1, 3], x2[2, 5], dy2[0, 7] = float("inf"), float("nan"), float("inf")

        def run(a, b):
            a = a.clone().requires_grad_()
            y = ops.gated_ffn(a, gu, d)
            return y.detach(), torch.autograd.grad(y, a, b)[0]

        (y, dx), (y2, dx2) = run(x, dy), run(x2, dy2)
        rest = [i for i in range(t) if i > 2]
        assert torch.equal(y[rest], y2[rest]) and torch.equal(dx[rest], dx2[rest]) and torch.equal(y[0], y2[0])
        assert y2[2].isnan().all() and not dx2[0].isfinite().all()


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last tokens' results and gradients are those of a call on them alone, to the
    roundings of two orders of summation (a step of the result each)."""
    from loopback_amd import block_ops as ops
    t, d, n = 262200, 64, 4104
    g = torch.Generator(device=DEV).manual_seed(1)
    x, gu, wd, dy = (torch.randn(s, device=DEV, generator=g, dtype=torch.bfloat16) * k for s, k in
                     (((t, d), 1.0), ((2 * n, d), 0.125), ((d, n), 0.02), ((t, d), 1.0)))
    print(f"case ffn {t}x{d}x{n}", flush=True)

    def run(a, b):
        a = a.clone().requires_grad_()
        y = ops.gated_ffn(a, gu, wd)
        return y.detach(), torch.autograd.grad(y, a, b)[0]

    got, ref = run(x, dy), run(x[-300:], dy[-300:])
    for a, b in zip(got, ref):
        assert (a[-300:] - b).float().norm() <= 2.0 ** -7 * b.float().norm()
