"""The block join and dropout (block_ops) against their formulas in fp64 on the same inputs: every result is an fp32 value
rounded once, so each element lies within half a step of the result's type (2^-8 of a bf16 value, 2^-11 of an fp16 one, 2^-24
of an fp32 one) plus fp32 round-off (1e-5 of the result's RMS; a dropped element is exactly 0). A norm's gradient is a difference r (t - v mean(t v)),
which cancels where a row has one or few elements: its fp32 round-off is that of its two terms, each of at most 16 roundings
(products, the row scale, a sum over up to 1024 lanes by pairs), 16 * 2^-24 = 2^-20 of r (|t| + |v| mean |t v|). The backward's formulas are
evaluated at the sum before its rounding. Sizes: one element, the edges of a vector, of the lanes
that share a row and of each row shape, odd widths, unaligned rows; gates whose runs of rows end inside and at a workgroup's."""
import pytest
import torch

from gpu_helpers import DEV

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def close(got, ref, dtype, what="", slack=0.0):
    ref = ref.double()
    rms = ref.pow(2).mean().sqrt() if ref.numel() else 0.0
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0   # half of fp16's smallest subnormal
    bad = (got.double() - ref).abs() > HALF[dtype] * ref.abs() + 1e-5 * rms + tiny + slack
    assert got.dtype is dtype and got.shape == ref.shape and not bad.any(), \
        (what, bad.sum().item(), (got.double() - ref).abs().max().item(), float(rms))


def rnd(shape, dtype, seed, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean
    return x.to(dtype).to(DEV)


def rng_of(seed, step=3):
    return torch.tensor([seed * 0x1234567 - 2 ** 60, step], device=DEV)


def unaligned(t):
    """The same values one element past an aligned address, contiguous."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    return out


def join64(x, y, post, gate, pre, mask, scale, eps, dh, dn):
    """(h, n) and the gradients of x, y, post, gate, pre in fp64 by their formulas."""
    f = lambda t: None if t is None else t.detach().double()
    x, y, post, gate, pre, dh, dn = map(f, (x, y, post, gate, pre, dh, dn))
    d = x.shape[-1]
    r1 = (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt() if post is not None else 1.0
    yh, w = y * r1, 1.0 if post is None else post
    gt = 1.0 if gate is None else gate
    h = x + scale * gt * yh * w * mask
    out, slack = {"h": h}, {}
    r2 = None
    terms = lambda t, v, r: 2.0 ** -20 * r * (t.abs() + v.abs() * (t * v).abs().mean(-1, keepdim=True))
    if pre is not None:
        r2 = (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        out["n"] = h * r2 * pre
    g = torch.zeros_like(x) if dh is None else dh
    if dn is not None:
        hh = h * r2
        t = dn * pre
        g = g + r2 * (t - hh * (t * hh).mean(-1, keepdim=True))
        slack["dx"] = terms(t, hh, r2)
        out["dpre"] = (dn * hh).flatten(0, -2).sum(0)
    out["dx"] = g
    dz = scale * mask * g
    t = dz * gt
    out["dy"] = t if post is None else r1 * (t * w - yh * (t * w * yh).mean(-1, keepdim=True))
    through = scale * mask * (gt if gate is None else gt.abs())   # what an error of dx is multiplied by on its way to dy
    slack["dy"] = slack.get("dx", 0.0) * through
    if post is not None:
        t_dx = slack["dy"] * w.abs() * r1
        slack["dy"] = terms(t * w, yh, r1) + t_dx + (t_dx * yh.abs()).mean(-1, keepdim=True) * yh.abs()
        out["dpost"] = (t * yh).flatten(0, -2).sum(0)
    if gate is not None:
        dg = dz * yh * w
        lead = [i for i, (a, b) in enumerate(zip((1,) * (x.dim() - gate.dim()) + tuple(gate.shape), x.shape)) if a == 1 and b != 1]
        out["dgate"] = (dg.sum(lead, keepdim=True) if lead else dg).reshape(gate.shape)
    return out, slack


def check_join(shape, dtype, post, gate, pre, p, scale=0.7, eps=1e-6, place=lambda t: t, dh_given=True, dn_given=True):
    from loopback_amd import block_ops as ops
    b, t, d = shape
    gshape = {"none": None, "column": (d,), "sequence": (b, 1, d), "full": shape}[gate]
    make = lambda s, k, **kw: None if s is None else place(rnd(s, dtype, k, **kw)).requires_grad_()
    x, y = make(shape, 1), make(shape, 2)
    pw, gw, nw = make((d,) if post else None, 3, std=0.2, mean=1.0), make(gshape, 4, std=0.3, mean=0.5), \
        make((d,) if pre else None, 5, std=0.2, mean=1.0)
    dh, dn = place(rnd(shape, dtype, 6)) if dh_given else None, place(rnd(shape, dtype, 7)) if pre and dn_given else None
    rng = rng_of(d + t)
    h, n = ops.block_join(x, y, post_weight=pw, gate=gw, scale=scale, dropout=p, rng=rng if p else None, site=9, pre_weight=nw,
                          eps=eps)
    assert "JoinNode" in h.grad_fn.name() and (n is None) == (not pre)
    outs = [(o, g) for o, g in ((h, dh), (n, dn)) if g is not None]
    torch.autograd.backward([o for o, _ in outs], [g for _, g in outs])
    torch.cuda.synchronize()
    mask = 1.0
    if p:
        drop = round(65536 * p)
        mask = ops.keep_mask(shape, p, rng, 9).double() * (65536 / max(1, 65536 - drop))   # p = 1 keeps nothing
    ref, slack = join64(x, y, pw, gw, nw, mask, scale, eps, dh, dn)
    got = {"h": h, "n": n, "dx": x.grad, "dy": y.grad, "dpost": pw is not None and pw.grad, "dgate": gw is not None and gw.grad,
           "dpre": nw is not None and nw.grad}
    for k, r in ref.items():
        close(got[k].detach(), r, dtype, k, slack.get(k, 0.0))
    with torch.no_grad():   # what records nothing gives the same bits
        h2, n2 = ops.block_join(x, y, post_weight=pw, gate=gw, scale=scale, dropout=p, rng=rng if p else None, site=9,
                                pre_weight=nw, eps=eps)
    assert torch.equal(h, h2) and (n is None or torch.equal(n, n2))


# widths: one vector and less, the edges of 4, 16, 64, 128, 256, 512 and 1024 lanes of eight columns, odd ones
@pytest.mark.parametrize("d", [1, 7, 8, 31, 32, 33, 40, 128, 136, 512, 520, 768, 1001, 1024, 1032, 2048, 2051, 4096, 4104, 8192])
@pytest.mark.parametrize("dtype", TYPES)
def test_join_widths(d, dtype):
    print(f"case join 3x7x{d} {dtype}", flush=True)
    check_join((3, 7, d), dtype, True, "column", True, 0.25)


@pytest.mark.parametrize("post,gate,pre,p", [(False, "none", False, 0.0), (True, "none", False, 0.0), (False, "none", True, 0.3),
                                             (False, "full", False, 0.1), (True, "full", True, 0.0), (True, "sequence", True, 0.1),
                                             (False, "sequence", False, 0.0), (False, "column", True, 0.5),
                                             (True, "column", False, 0.0), (True, "none", True, 1.0)])
@pytest.mark.parametrize("d", [96, 768, 1001, 1280])
def test_join_parts(post, gate, pre, p, d):
    """Every part alone and with others."""
    print(f"case join parts d={d} {post} {gate} {pre} {p}", flush=True)
    for dtype in TYPES:
        check_join((2, 37, d), dtype, post, gate, pre, p)


@pytest.mark.parametrize("b,t", [(1, 1), (1, 5), (5, 1), (2000, 1), (1000, 2), (37, 64), (37, 65), (6, 400), (3, 1365), (1, 4001)])
@pytest.mark.parametrize("d", [24, 200, 1032])
def test_join_gate_runs(b, t, d):
    """A gate per sequence: runs of one row, several in a workgroup's rows, runs cut between two and many workgroups."""
    print(f"case join gate runs {b}x{t}x{d}", flush=True)
    check_join((b, t, d), torch.bfloat16, True, "sequence", True, 0.1)
    check_join((b, t, d), torch.float32, False, "column", True, 0.0)


@pytest.mark.parametrize("d", [64, 768, 2048])
@pytest.mark.parametrize("dtype", TYPES)
def test_join_unaligned(d, dtype):
    print(f"case join unaligned {d} {dtype}", flush=True)
    check_join((2, 19, d), dtype, True, "column", True, 0.2, place=unaligned)


def test_join_one_upstream_gradient():
    """Only h, or only n, is used."""
    for kw in ({"dh_given": False}, {"dn_given": False}):
        for dtype in TYPES:
            check_join((2, 9, 776), dtype, True, "column", True, 0.1, **kw)


def test_join_gradients_one_at_a_time():
    """Each gradient alone has the bits it has beside the others."""
    from loopback_amd import block_ops as ops
    vals = {"x": rnd((2, 300, 768), torch.bfloat16, 1), "y": rnd((2, 300, 768), torch.bfloat16, 2),
            "post_weight": rnd((768,), torch.bfloat16, 3), "gate": rnd((2, 1, 768), torch.bfloat16, 4),
            "pre_weight": rnd((768,), torch.bfloat16, 5)}
    dh, dn = rnd((2, 300, 768), torch.bfloat16, 6), rnd((2, 300, 768), torch.bfloat16, 7)

    def grads(names):
        v = {k: t.clone().requires_grad_(k in names) for k, t in vals.items()}
        x, y = v.pop("x"), v.pop("y")
        out = ops.block_join(x, y, dropout=0.1, rng=rng_of(1), **v)
        v |= {"x": x, "y": y}
        return dict(zip(names, torch.autograd.grad(out, [v[k] for k in names], (dh, dn))))

    both = grads(list(vals))
    for k in vals:
        assert torch.equal(grads([k])[k], both[k]), k


def test_join_strides_and_types():
    """Strided inputs and upstream gradients (expanded, transposed) give the contiguous ones' results; fp64 and mixed types run
    the torch form."""
    from loopback_amd import block_ops as ops
    x, y, w = rnd((6, 4, 64), torch.bfloat16, 1), rnd((4, 6, 64), torch.bfloat16, 2), rnd((64, 2), torch.bfloat16, 3)
    xs, ys, ws = x.clone().requires_grad_(), y.transpose(0, 1).requires_grad_(), w[:, 1].requires_grad_()
    xc, yc, wc = (t.detach().contiguous().requires_grad_() for t in (xs, ys, ws))
    g = rnd((64,), torch.bfloat16, 4)
    a = ops.block_join(xs, ys, post_weight=ws, pre_weight=ws)
    b = ops.block_join(xc, yc, post_weight=wc, pre_weight=wc)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = torch.autograd.grad(a, (xs, ys, ws), (g.expand(6, 4, 64), g.expand(6, 4, 64)))
    gb = torch.autograd.grad(b, (xc, yc, wc), (g.expand(6, 4, 64).contiguous(), g.expand(6, 4, 64).contiguous()))
    for p, q in zip(ga, gb):
        assert torch.equal(p, q)
    h, _ = ops.block_join(x.double(), y.transpose(0, 1).double())
    assert torch.equal(h, x.double() + y.transpose(0, 1).double())
    h, _ = ops.block_join(x, y.transpose(0, 1).float())
    assert h.dtype is torch.bfloat16 and torch.equal(h, (x.float() + y.transpose(0, 1).float()).bfloat16())


def test_join_not_finite_and_empty():
    """A row with an infinity or NaN stays alone; a dropped one is gone; no rows give empty results and zero gradients."""
    from loopback_amd import block_ops as ops
    x, y = rnd((9, 776), torch.float32, 1), rnd((9, 776), torch.float32, 2)
    w = rnd((776,), torch.float32, 3)
    h0, n0 = ops.block_join(x, y, post_weight=w, pre_weight=w)
    y2 = y.clone()
    y2[3, 5], y2[6, 700] = float("inf"), float("nan")
    h, n = ops.block_join(x, y2, post_weight=w, pre_weight=w)
    rest = [0, 1, 2, 4, 5, 7, 8]
    assert torch.equal(h[rest], h0[rest]) and torch.equal(n[rest], n0[rest]) and h[3].isnan().any() and h[6].isnan().all()
    h, _ = ops.block_join(x, torch.full_like(y, float("nan")), dropout=1.0, rng=rng_of(1))
    assert torch.equal(h, x)
    e = torch.empty(0, 776, device=DEV, requires_grad=True)
    h, n = ops.block_join(e, e, post_weight=w, pre_weight=w, dropout=0.5, rng=rng_of(1))
    assert h.shape == n.shape == (0, 776)
    (h.sum() + n.sum()).backward()


@pytest.mark.parametrize("shape", [(1,), (5,), (8,), (3, 1), (4, 7), (2, 3, 40), (129, 8), (77, 1001), (3000, 768), (2, 100003)])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0, 2.0 ** -16])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout(shape, p, dtype):
    """Values and gradients element by element: one fp32 product, rounded; the mask that keep_mask gives."""
    from loopback_amd import block_ops as ops
    print(f"case dropout {shape} {p} {dtype}", flush=True)
    x, g, rng = rnd(shape, dtype, 1).requires_grad_(), rnd(shape, dtype, 2), rng_of(7, 2 ** 32 - 1)
    out = ops.dropout(x, p, rng, site=2 ** 32 - 1)
    out.backward(g)
    torch.cuda.synchronize()
    keep, drop = ops.keep_mask(shape, p, rng, 2 ** 32 - 1), round(65536 * p)
    s = torch.tensor(65536 / (65536 - drop) if drop < 65536 else 0.0, device=DEV)
    assert torch.equal(out, torch.where(keep, x.float() * s, 0.0).to(dtype))
    assert torch.equal(x.grad, torch.where(keep, g.float() * s, 0.0).to(dtype))
    y = unaligned(x.detach())
    assert torch.equal(ops.dropout(y, p, rng, site=2 ** 32 - 1), out)
    if x.dim() > 1:
        t = x.detach().transpose(0, -1).contiguous().transpose(0, -1)
        assert torch.equal(ops.dropout(t, p, rng, site=2 ** 32 - 1), out)


def test_dropout_not_finite():
    from loopback_amd import block_ops as ops
    x = torch.full((64, 64), float("inf"), device=DEV)
    out, keep = ops.dropout(x, 0.5, rng_of(1)), ops.keep_mask((64, 64), 0.5, rng_of(1))
    assert torch.equal(out, torch.where(keep, x, 0.0)) and 0.45 < keep.float().mean() < 0.55


def test_captured_and_replayed():
    """Join, its backward and dropout in a captured graph: every replay gives what the eager calls give at that step of the
    generator, with eager work between the replays."""
    from loopback_amd import block_ops as ops
    x, y, w = (rnd(s, torch.bfloat16, k).requires_grad_() for s, k in (((3, 500, 768), 1), ((3, 500, 768), 2), ((768,), 3)))
    dh, dn, rng = rnd((3, 500, 768), torch.bfloat16, 4), rnd((3, 500, 768), torch.bfloat16, 5), rng_of(11, 0)

    def step():
        r = rng.clone()
        out = ops.block_join(x, y, post_weight=w, gate=w, dropout=0.2, rng=r, site=1, pre_weight=w)
        grads = torch.autograd.grad(out, (x, y, w), (dh, dn))
        return [t.detach() for t in (*out, *grads, ops.dropout(dh, 0.3, r, site=2))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        rng[1] = 7 * k
        ref = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, ref):
            assert torch.equal(a, b), k


def test_second_derivatives_and_watchers():
    """A backward that is differentiated and forward mode run the torch form's operations: fp32 results to round-off."""
    from loopback_amd import block_ops as ops
    args = [rnd(s, torch.float32, k).requires_grad_() for s, k in (((2, 5, 40), 1), ((2, 5, 40), 2), ((40,), 3), ((2, 1, 40), 4),
                                                                  ((40,), 5))]
    rng = rng_of(2)

    def call(fn):
        x, y, post, gate, pre = args
        h, n = fn(x, y, post, gate, pre)
        u, v = torch.cos(torch.arange(400.0, device=DEV)).view(2, 5, 40), torch.sin(torch.arange(400.0, device=DEV)).view(2, 5, 40)
        g = torch.autograd.grad((h * u + n * v).sum(), args, create_graph=True)
        return torch.autograd.grad(sum(t.pow(2).sum() for t in g), args)

    got = call(lambda x, y, post, gate, pre: ops.block_join(x, y, post_weight=post, gate=gate, scale=0.5, dropout=0.2, rng=rng,
                                                           pre_weight=pre))
    ref = call(lambda x, y, post, gate, pre: ops._join_torch(x, y, post, gate, pre, rng, 0, round(65536 * 0.2), 0.5, 1e-6))
    for a, b in zip(got, ref):
        assert (a - b).norm() <= 1e-5 * b.norm()
    out, tangent = torch.func.jvp(lambda t: ops.dropout(t, 0.5, rng), (args[0].detach(),), (torch.ones_like(args[0]),))
    assert torch.equal(tangent != 0, ops.keep_mask((2, 5, 40), 0.5, rng)) and out.shape == (2, 5, 40)


def test_two_streams():
    """Calls on two streams at once give what each gives alone."""
    from loopback_amd import block_ops as ops
    xs = [rnd((4096, 776), torch.bfloat16, k) for k in (1, 2)]
    ws = [rnd((776,), torch.bfloat16, k) for k in (3, 4)]

    def work(k):
        x = xs[k].clone().requires_grad_()
        h, n = ops.block_join(x, xs[k], post_weight=ws[k], pre_weight=ws[k], dropout=0.1, rng=rng_of(k))
        return [h.detach(), n.detach(), *torch.autograd.grad((h, n), x, (xs[k], xs[1 - k]))]

    alone = [work(k) for k in (0, 1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                got[k] = work(k)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_hooks_batched_gradients_and_modes():
    """Saved tensors that a hook gives back strided or unaligned; batched gradients and a dispatch mode take torch's operations."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from loopback_amd import block_ops as ops
    args = [rnd(s, torch.float32, k) for k, s in enumerate(((3, 5, 40), (3, 5, 40), (40,), (3, 1, 40), (40,)))]
    u, v, rng = rnd((3, 5, 40), torch.float32, 8), rnd((3, 5, 40), torch.float32, 9), rng_of(2)
    leaf = lambda: [a.clone().requires_grad_() for a in args]
    call = lambda x, y, post, gate, pre: ops.block_join(x, y, post_weight=post, gate=gate, scale=0.5, dropout=0.2, rng=rng,
                                                        pre_weight=pre)
    ins = leaf()
    outs = call(*ins)
    want = torch.autograd.grad(outs, ins, (u, v), retain_graph=True)
    strided = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() > 1 else t
    for unpack in (strided, unaligned):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            other = call(*ins)
        for a, b in zip(torch.autograd.grad(other, ins, (u, v)), want):
            assert (a - b).norm() <= 1e-6 * b.norm()
    got = torch.autograd.grad(outs, ins, (torch.stack((u, 2 * u)), torch.stack((v, 2 * v))), is_grads_batched=True, retain_graph=True)
    for a, b in zip(got, want):
        assert (a[0] - b).norm() <= 1e-5 * b.norm() and (a[1] - 2 * b).norm() <= 1e-5 * b.norm()

    class Count(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Count.n += 1
            return func(*args, **(kwargs or {}))

    with Count():
        seen = torch.autograd.grad(outs, ins, (u, v), retain_graph=True)
        h, _ = call(*args)
    assert Count.n > 20 and (h - outs[0]).abs().max() <= 1e-6 * h.abs().max()
    for a, b in zip(seen, want):
        assert (a - b).norm() <= 1e-5 * b.norm()
    x = rnd((6, 40), torch.float32, 10).requires_grad_()
    y = ops.dropout(x, 0.5, rng)
    g, = torch.autograd.grad(y, x, torch.ones(2, 6, 40, device=DEV), is_grads_batched=True)
    assert torch.equal(g[0] != 0, ops.keep_mask((6, 40), 0.5, rng)) and torch.equal(g[0], g[1])


def test_generator_changed_in_place():
    """A generator that was changed before the backward of a call that took it is refused by autograd."""
    from loopback_amd import block_ops as ops
    x, rng = rnd((6, 40), torch.float32, 1).requires_grad_(), rng_of(3)
    y = ops.dropout(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_only_on_the_current_gpu(monkeypatch):
    """Tensors of a GPU that is not the current one run the torch form."""
    from loopback_amd import block_ops as ops
    x = rnd((6, 40), torch.float32, 1)
    want = ops.dropout(x, 0.5, rng_of(3)), ops.block_join(x, x)[0]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: x.device.index + 1)
    monkeypatch.setattr(ops, "H", None)   # a launch would fail
    assert torch.equal(ops.dropout(x, 0.5, rng_of(3)), want[0]) and torch.equal(ops.block_join(x, x)[0], want[1])


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last rows' results and gradients are those of a call on them alone; dropout's
    mask there is the generator's."""
    import numpy as np
    from loopback_amd import block_ops as ops
    rows, d = 262160, 8200
    print(f"case rows {rows}x{d}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((rows, d), device=DEV, generator=g, dtype=torch.bfloat16)
    out, last = ops.dropout(x, 0.25, rng_of(3), site=5), rows - 1
    u, m = np.uint64, np.uint64(0xFFFFFFFF)
    seed, step = (int(v) for v in rng_of(3).cpu())
    c = [np.arange(d // 8, dtype=u), np.full(d // 8, last, u), np.full(d // 8, 5, u), np.full(d // 8, step, u)]
    k = [u(seed & 0xFFFFFFFF), u((seed >> 32) & 0xFFFFFFFF)]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k[0], b & m, (a >> u(32)) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + u(0x9E3779B9)) & m, (k[1] + u(0xBB67AE85)) & m]
    keep = np.stack(c, -1).astype("<u4").view("<u2").reshape(d) >= 16384
    keep = torch.from_numpy(keep).to(DEV)
    assert torch.equal(out[last], torch.where(keep, x[last].float() * (65536 / 49152), 0.0).bfloat16())
    x, w = x.view(-1)[:rows * 8192].view(rows, 8192), rnd((8192,), torch.bfloat16, 2)
    del out

    def run(v):
        v = v.clone().requires_grad_()
        h, n = ops.block_join(v, v, post_weight=w, pre_weight=w)
        return h.detach(), n.detach(), torch.autograd.grad((h, n), v, (h.detach(), n.detach()))[0]

    for a, b in zip(run(x), run(x[-50:])):
        assert torch.equal(a[-50:], b)


def test_anomaly_mode():
    """The nodes under autograd's anomaly detection: a clean pass, and a NaN gradient that is found (in the first node it reaches)."""
    from loopback_amd import block_ops as ops
    x, w = rnd((4, 40), torch.float32, 1).requires_grad_(), rnd((40,), torch.float32, 2).requires_grad_()
    with torch.autograd.set_detect_anomaly(True, check_nan=True):
        h, n = ops.block_join(ops.dropout(x, 0.5, rng_of(1)), x, post_weight=w, pre_weight=w)
        (h.sum() + n.sum()).backward()
        h, n = ops.block_join(x, x, post_weight=w, pre_weight=w)
        with pytest.raises(RuntimeError, match="returned nan values"):
            (h.sum() * float("nan")).backward()


def test_inputs_changed_before_the_backward():
    """x and y are what the backward reads: changed in place, it refuses; h and n are not, and may be."""
    from loopback_amd import block_ops as ops
    x0, y0, w = (rnd(s, torch.bfloat16, k).requires_grad_() for k, s in enumerate(((40, 136), (40, 136), (136,))))
    dh, dn = rnd((40, 136), torch.bfloat16, 5), rnd((40, 136), torch.bfloat16, 6)

    def run(change):
        x, y = x0 * 1, y0 * 1
        h, n = ops.block_join(x, y, post_weight=w, pre_weight=w, dropout=0.1, rng=rng_of(2))
        f = (h * dh).sum() + (n * dn).sum()   # keeps dh and dn, not h and n
        with torch.no_grad():
            for t in change(x, y, h, n):
                t.add_(1.0)
        return torch.autograd.grad(f, (x0, y0, w))

    want = run(lambda x, y, h, n: ())
    for a, b in zip(run(lambda x, y, h, n: (h, n)), want):
        assert torch.equal(a, b)
    for change in (lambda x, y, h, n: (x,), lambda x, y, h, n: (y,)):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            run(change)
