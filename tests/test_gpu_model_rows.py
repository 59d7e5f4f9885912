"""Layer norm and the distillation loss (model_ops) against their formulas in fp64 on the same inputs.

A result is an fp32 value rounded once, so it lies within half a step of its type (2^-8 of a bf16 value, 2^-11 of an fp16 one, 2^-24
of an fp32 one) plus the round-off of the fp32 value. u = 2^-24. Layer norm: a row's sums go over at most 16 columns of a lane and
ten levels of lanes, 32 roundings of their terms' absolute values with the statistics' own, so hat = (h - m) r is within
E = 32 u r (|h| + mean|h|) and what is formed from it within the sums below. Distillation: a log-probability is a difference of
numbers no larger than A = max|z| / tau + max|x| / tau + log(vocab), each after at most 16 roundings, so within 16 u A, and a
probability within that share of itself (and 8 u more for the exponential)."""
import math

import pytest
import torch

from gpu_helpers import DEV
from loopback_amd import model_ops as M

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def close(got, ref, slack, what=""):
    dtype = got.dtype
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0   # half of fp16's smallest subnormal
    bad = (got.double() - ref).abs() > (HALF[dtype] * (ref.abs() + slack) + slack + tiny)
    assert got.shape == ref.shape and not bad.any() and got.isfinite().all(), \
        (what, int(bad.sum()), float((got.double() - ref).abs().max()), float(ref.abs().max()))


def rnd(shape, dtype, seed, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean
    return x.to(dtype).to(DEV)


def unaligned(t):
    """The same values one element past an aligned address, contiguous."""
    out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return out.copy_(t)


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
def norm_reference(x, add, w, b, dy, dh, eps):
    """{name: (value, slack)} in fp64."""
    dt = x.dtype
    X = x.double()
    h = (X + add.double()).to(dt).double() if add is not None else X
    z = h - h.mean(-1, keepdim=True)
    r = (z.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = z * r
    E = 32 * U * r * (h.abs() + h.abs().mean(-1, keepdim=True))
    W = w.double() if w is not None else torch.ones((), dtype=torch.float64, device=x.device)
    B = b.double() if b is not None else torch.zeros((), dtype=torch.float64, device=x.device)
    y = hat * W + B
    out = {"y": (y, E * W.abs() + 4 * U * (y.abs() + B.abs()))}
    if add is not None:
        out["h"] = (X + add.double(), 2 * U * (X.abs() + add.double().abs()))
    g = dy.double()
    over = lambda v: v.reshape(-1, v.shape[-1]).sum(0)  # noqa: E731
    t = g * W
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    dx = r * (t - mean(t) - hat * mean(t * hat))
    s = r * (32 * U * (t.abs() + mean(t.abs()) + 2 * hat.abs() * mean((t * hat).abs())) + E * mean((t * hat).abs())
             + hat.abs() * mean(t.abs() * E))
    if dh is not None:
        dx, s = dx + dh.double(), s + 4 * U * dh.double().abs()
    out["dx"] = (dx, s)
    n = 64 * U   # sums over the rows: at most 40 of a workgroup's in a row of adds, then ten levels
    out["dw"] = (over(g * hat), over(g.abs() * E + n * (g * hat).abs()))
    out["db"] = (over(g), n * over(g.abs()))
    return out


def check_norm(x, add, w, b, eps=1e-5, seed=9):
    leaves = [t.requires_grad_() for t in (x, add, w, b) if t is not None]
    dy = rnd(x.shape, x.dtype, seed)
    if add is None:
        dh, outs = None, (M.layer_norm(x, w, b, eps),)
        grads = torch.autograd.grad(outs, leaves, (dy,))
    else:
        dh, outs = rnd(x.shape, x.dtype, seed + 1), M.add_layer_norm(x, add, w, b, eps)
        grads = torch.autograd.grad(outs, leaves, (dh, dy))
    ref = norm_reference(*(None if t is None else t.detach() for t in (x, add, w, b)), dy, dh, eps)
    got = dict(zip(("h", "y") if add is not None else ("y",), outs))
    names = [k for k, t in zip(("dx", "dadd", "dw", "db"), (x, add, w, b)) if t is not None]
    got.update(zip(names, grads))
    for k, v in got.items():
        close(v.detach(), *ref["dx" if k == "dadd" else k], what=k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 7, 8, 31, 32, 33, 128, 136, 511, 512, 768, 1000, 1024, 2048, 2050, 4096, 5001, 8192, 8200, 16383, 16384])
def test_norm_widths(d, dtype):
    rows = 3 if d > 4096 else 37
    check_norm(rnd((rows, d), dtype, 1, 2.0, 0.5), None, rnd((d,), dtype, 2, 0.2, 1.0), rnd((d,), dtype, 3))
    check_norm(rnd((rows, d), dtype, 4), rnd((rows, d), dtype, 5, 0.5), rnd((d,), dtype, 6, 0.2, 1.0), rnd((d,), dtype, 7))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 64), (2, 1, 96), (5, 768), (3, 11, 40), (1500, 24), (4100, 768), (130, 2048), (64,)])
@pytest.mark.parametrize("affine", ["weight", "bias", "none"])
def test_norm_rows_and_parts(shape, affine, dtype):
    w = rnd(shape[-1:], dtype, 2, 0.2, 1.0) if affine == "weight" else None
    b = rnd(shape[-1:], dtype, 3) if affine == "bias" else None
    check_norm(rnd(shape, dtype, 1, 1.0, 2.0), None, w, b)
    check_norm(rnd(shape, dtype, 1), rnd(shape, dtype, 8), w, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_a_large_mean(dtype):
    """Differences from the mean, not a difference of squares: a mean a thousand times the spread."""
    x = rnd((9, 768), torch.float32, 1, 1.0, 1000.0).to(dtype)
    check_norm(x, None, rnd((768,), dtype, 2, 0.1, 1.0), rnd((768,), dtype, 3))


@pytest.mark.parametrize("d", [768, 1001])
def test_norm_strides_and_alignment(d):
    dt = torch.bfloat16
    base = rnd((6, 5, d), dt, 1)
    y = M.layer_norm(base, None, None)
    for x in (base.transpose(0, 1).contiguous().transpose(0, 1), unaligned(base), base.expand(2, 6, 5, d)[1],
              torch.cat((base, base), -1)[..., :d]):
        assert torch.equal(M.layer_norm(x, None, None), y)
    check_norm(unaligned(base), unaligned(base), unaligned(rnd((d,), dt, 2)), unaligned(rnd((d,), dt, 3)))
    x = base.detach().clone().requires_grad_()
    M.layer_norm(x.transpose(0, 1)).sum().backward()      # a gradient of one value for all, expanded
    assert x.grad.shape == x.shape and x.grad.isfinite().all()


def test_norm_of_one_tensor_twice():
    """A tensor added to itself, and one vector as weight and bias: both places' gradients come to it."""
    x, w = rnd((70, 136), torch.float32, 1).requires_grad_(), rnd((136,), torch.float32, 2).requires_grad_()
    h, y = M.add_layer_norm(x, x, w, w)
    a, b = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z = torch.nn.functional.layer_norm(2 * a, (136,), b, b)
    dy, dh = rnd(y.shape, torch.float32, 3), rnd(h.shape, torch.float32, 4)
    got = torch.autograd.grad([h, y], [x, w], [dh, dy])
    ref = torch.autograd.grad([2 * a, z], [a, b], [dh.double(), dy.double()])
    assert torch.equal(h, 2 * x)
    close(y, z, 1e-5), close(got[0], ref[0], 1e-4), close(got[1], ref[1], 1e-3)   # sums of 70 terms of up to 10: 70 10 2^-24 and less


def test_norm_gradients_that_are_asked_for():
    d = 256
    x, a, w, b = rnd((33, d), torch.bfloat16, 1), rnd((33, d), torch.bfloat16, 2), rnd((d,), torch.bfloat16, 3), rnd((d,), torch.bfloat16, 4)
    dy = rnd((33, d), torch.bfloat16, 5)
    full = [t.clone().requires_grad_() for t in (x, a, w, b)]
    h, y = M.add_layer_norm(*full)
    ref = torch.autograd.grad((h, y), full, (dy, dy))
    for need in range(1, 16):
        ts = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, a, w, b))]
        h, y = M.add_layer_norm(*ts)
        assert h.requires_grad == bool(need & 3)
        got = torch.autograd.grad((h, y) if need & 3 else (y,), [t for t in ts if t.requires_grad], (dy, dy) if need & 3 else (dy,))
        for g, r in zip(got, [r for i, r in enumerate(ref) if need >> i & 1]):
            assert torch.equal(g, r)
    # one result used alone
    ts = [t.clone().requires_grad_() for t in (x, a, w, b)]
    h, y = M.add_layer_norm(*ts)
    g = torch.autograd.grad(h, ts, dy, allow_unused=True, retain_graph=True)
    assert torch.equal(g[0], dy) and torch.equal(g[1], dy) and g[2] is None and g[3] is None
    # the stream itself as the first result
    s = x.clone().requires_grad_()
    h, y = M.add_layer_norm(s, None, w, b)
    assert torch.equal(h, s)
    g, = torch.autograd.grad((h, y), s, (dy, dy))
    t = x.clone().requires_grad_()
    g2, = torch.autograd.grad(M.layer_norm(t, w, b), t, dy)
    close(g, g2.double() + dy.double(), HALF[torch.bfloat16] * g2.double().abs() + 1e-6)


def test_norm_infinities_stay_in_their_rows():
    x = rnd((20, 96), torch.float32, 1)
    x[3, 5], x[7, 0] = math.inf, math.nan
    y = M.layer_norm(x)
    rows = torch.ones(20, dtype=torch.bool, device=DEV)
    rows[3] = rows[7] = False
    assert y[rows].isfinite().all() and not y[~rows].isfinite().any()


def test_empty_rows():
    x = torch.empty((0, 64), device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = M.layer_norm(x, w)
    assert y.shape == x.shape
    y.sum().backward()
    assert not w.grad.any()


# ---------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------
def teacher_of(rows, vocab, k, seed, pad=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    top = (torch.randn(rows, k, generator=g) * 2 + 3).sort(-1, descending=True).values
    if pad and rows > 2:
        kept = torch.randint(1, k + 1, (rows, 1), generator=g)
        ids = torch.where(torch.arange(k) < kept, ids, -1)
        ids[1] = -1                                   # a row that does not count
        top = torch.where(ids < 0, torch.nan, top)    # what is not named is not read into anything
    labels = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 3:
        labels[1] = labels[3] = -100
    return ids.to(DEV), top.to(DEV), labels.to(DEV)


def distill_reference(x, top, ids, lse, labels, tau, hard, g=1.0):
    """loss, its slack, the gradient and its slack, in fp64, row by row and class by class."""
    X = x.double()
    rows, vocab = X.shape
    valid = ids >= 0
    z = torch.where(valid, top.double() / tau, -math.inf)
    counts = valid.any(-1)
    ref = torch.logsumexp(z, -1) if lse is None else lse.double()
    p = torch.where(valid, torch.exp(z - ref.unsqueeze(-1)), 0.0)
    target = torch.zeros((rows, vocab), dtype=torch.float64, device=x.device)
    named = torch.zeros((rows, vocab), dtype=torch.bool, device=x.device)
    logq = torch.log_softmax(X / tau, -1)
    q = logq.exp()
    kl = torch.zeros(rows, dtype=torch.float64, device=x.device)
    for i in range(ids.shape[1]):
        at = ids[:, i].long().clamp_min(0).unsqueeze(-1)
        pi = p[:, i:i + 1]
        target.scatter_add_(1, at, pi)
        named |= torch.zeros_like(named).scatter(1, at, valid[:, i:i + 1])
        kl += torch.where(pi > 0, pi * (z[:, i:i + 1] - ref.unsqueeze(-1) - logq.gather(1, at)), 0.0).squeeze(-1)
    whole, parts = p.sum(-1, keepdim=True), target.clone()
    if lse is not None:
        rest = torch.where((~named).any(-1, keepdim=True), (1 - whole).clamp_min(0), 0.0)
        others = torch.where(named, 0.0, q)
        qr = others.sum(-1, keepdim=True)
        kl += torch.where(rest > 0, rest * (rest.log() - qr.log()), 0.0).squeeze(-1)
        target = target + torch.where(rest > 0, rest * others / qr, 0.0)
        whole, parts = whole + rest, target
    finite = torch.where(torch.isfinite(z), z, 0.0).abs().max() + X[X.isfinite()].abs().max() / tau + math.log(vocab)
    A = 16 * U * (finite + (0 if lse is None else lse.double().abs().max())) + 8 * U
    n, m = max(1, int(counts.sum())), 1
    loss = (1 - hard) * tau * tau * kl[counts].sum() / n
    # rest = 1 - P carries the roundings of P, at most 32 of sums no larger than 1, weighed by log(rest / q_rest)
    slack = (1 - hard) * tau * tau * (2 * A + 48 * U) * (1 + kl[counts].abs().sum() / n) * 2
    d = torch.where(counts.unsqueeze(-1), q * whole - target, 0.0) * ((1 - hard) * tau / n)
    ds = torch.where(counts.unsqueeze(-1), q * whole + parts, 0.0) * ((1 - hard) * tau / n)
    if lse is not None:   # the roundings of 1 - P, shared out as the others are
        ds = ds + torch.where(counts.unsqueeze(-1) & ~named, 48 * U / A * others / qr, 0.0) * ((1 - hard) * tau / n)
    if hard:
        there = labels >= 0
        m = max(1, int(there.sum()))
        l1 = torch.log_softmax(X, -1)
        loss = loss - hard * l1.gather(1, labels.clamp_min(0).unsqueeze(-1))[there].sum() / m
        slack = slack + hard * 2 * A * max(1.0, tau)
        one = torch.zeros_like(q).scatter(1, labels.clamp_min(0).unsqueeze(-1), 1.0)
        d = d + torch.where(there.unsqueeze(-1), l1.exp() - one, 0.0) * (hard / m)
        ds = ds + torch.where(there.unsqueeze(-1), l1.exp() + one, 0.0) * (hard / m) * max(1.0, tau)
    # a probability below fp32's smallest normal number, 2^-126, is 0
    return loss, float(slack), d * g, ds * A * 2 * g + 2.0 ** -126 * 2 * tau * g


def check_distill(x, top, ids, lse=None, labels=None, tau=1.0, hard=0.0, scale=1.0):
    x = x.detach().clone().requires_grad_()
    loss = M.distill_loss(x, top, ids, temperature=tau, teacher_lse=lse, labels=labels, hard_weight=hard)
    (loss * scale).backward()
    ref, slack, d, ds = distill_reference(x.detach(), top, ids, lse, labels, tau, hard, scale)
    assert loss.dtype is torch.float32 and loss.shape == ()
    assert abs(loss.item() - ref.item()) <= slack, (loss.item(), ref.item(), slack)
    close(x.grad, d, ds, "dlogits")
    return loss


def lse_of(top, ids, tau, more=0.2):
    z = torch.where(ids >= 0, top.double() / tau, -math.inf)
    return (torch.logsumexp(z, -1) + math.log1p(more)).float()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau,hard", [(1.0, 0.0), (2.0, 0.5), (1.0, 0.3)])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (5, 7, 3), (4, 8, 8), (6, 9, 1), (9, 101, 17), (7, 2049, 64), (5, 32003, 33),
                                          (600, 515, 12)])
def test_distill(rows, vocab, k, tau, hard, dtype):
    ids, top, labels = teacher_of(rows, vocab, k, 1)
    x = rnd((rows, vocab), dtype, 2, 3.0)
    scale = 1024.0 if dtype is torch.float16 else 1.0
    args = {"labels": labels if hard else None, "tau": tau, "hard": hard, "scale": scale}
    check_distill(x, top, ids, **args)
    check_distill(x, top.to(dtype), ids.to(torch.int32), lse=lse_of(top.to(dtype), ids, tau), **args)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [0.5, 3.0, 4.0, 7.5])
@pytest.mark.parametrize("rows,vocab,k", [(5, 2049, 64), (700, 9001, 12)])
def test_distill_temperatures(rows, vocab, k, tau, dtype):
    """The labels' softmax beside one at other temperatures."""
    ids, top, labels = teacher_of(rows, vocab, k, 5)
    x = rnd((rows, vocab), dtype, 6, 3.0)
    args = {"labels": labels, "tau": tau, "hard": 0.3, "scale": 1024.0 if dtype is torch.float16 else 1.0}
    check_distill(x, top, ids, **args)
    check_distill(x, top, ids, lse=lse_of(top, ids, tau), **args)


@pytest.mark.parametrize("tau,hard", [(1.0, 0.0), (1.0, 0.3), (2.0, 0.3), (4.0, 0.3), (3.0, 0.3)])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_past_the_caches(dtype, tail, tau, hard):
    """Logits of more than the caches hold, and the same rows in two calls of half as many: a row's gradient is the same value, less
    by the number of rows, a power of two."""
    rows, vocab, k = 4096, 16397, 7
    x = torch.empty(rows, vocab, dtype=dtype, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(2)).requires_grad_()
    ids, top, labels = teacher_of(rows, vocab, k, 3, pad=False)
    top, labels = top.to(dtype), labels.clamp_min(0) if hard else None
    lse = lse_of(top, ids, tau) if tail else None
    def run(at):
        part = [None if t is None else t[at] for t in (lse, labels)]
        loss = M.distill_loss(x[at], top[at], ids[at], temperature=tau, teacher_lse=part[0], labels=part[1], hard_weight=hard)
        return loss, torch.autograd.grad(loss, x)[0][at]
    whole, grad = run(slice(None))
    halves = [slice(0, rows // 2), slice(rows // 2, rows)]
    # a mean of 4096 fp32 terms within 16 roundings of their sum
    assert abs(whole - sum(run(at)[0] for at in halves) / 2) <= 64 * U * abs(whole)
    for at in halves:
        assert torch.equal(2 * grad[at], run(at)[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,m,shift", [(8, 2.0 ** 121, 0), (8, 2.0 ** 121, 1), (4, 2.0 ** 122, 0), (256, 2.0 ** 116, 0), (2048, 2.0 ** 115, 0)])
def test_norm_of_large_equal_values(d, m, shift, dtype):
    """Rows of one large value: they lie at their mean exactly, so y is the bias and dx is r (t - mean(t)), r eps^-1/2. What a lane past the
    row's end would form of the mean, 316 times it, is infinite."""
    x = torch.full((5, d), m, dtype=dtype, device=DEV)
    x = (unaligned(x) if shift else x).requires_grad_()
    w, b = (rnd((d,), dtype, i, 0.3, 1.0).requires_grad_() for i in (1, 2))
    y = M.layer_norm(x, w, b)
    dy = rnd((5, d), dtype, 3)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    t = dy.double() * w.detach().double()
    r = 1e-5 ** -0.5
    assert torch.equal(y.detach(), b.detach().expand(5, d)) and not dw.any()
    close(dx, r * (t - t.mean(-1, keepdim=True)), 32 * U * r * (t.abs() + t.abs().mean(-1, keepdim=True)), "dx")
    close(db, dy.double().sum(0), 8 * U * dy.double().abs().sum(0), "db")


@pytest.mark.parametrize("rows,vocab", [(3, M.DISTILL_MAX_TAIL - 512), (3, M.DISTILL_MAX_TAIL - 511), (3, M.DISTILL_MAX_TAIL),
                                        (513, M.DISTILL_MAX_TAIL), (3, M.DISTILL_MAX_TAIL + 1)])
def test_distill_the_largest_maps(rows, vocab):
    """The rest of a vocabulary whose map of named classes fills the 64 KiB of LDS that a launch may take unasked, with the waves' sums
    beside it more than fills it, and one whose map is too large for the kernels."""
    ids, top, labels = teacher_of(rows, vocab, 9, 5)
    ids[0, 0], ids[2, 0] = vocab - 1, vocab - 32     # the map's last word
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=DEV).normal_(0.0, 3.0, generator=torch.Generator(DEV).manual_seed(6))
    check_distill(x, top, ids, lse=lse_of(top, ids, 1.0), labels=labels, hard=0.3)


def test_rows_past_32_bits():
    """More than 2^31 elements: the last rows are what they are alone."""
    x = torch.empty(140000, 16384, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(4))
    last = x[-9:].clone()
    leaf, alone = x.requires_grad_(), last.clone().requires_grad_()
    y, z = M.layer_norm(leaf), M.layer_norm(alone)
    assert x.numel() > 2 ** 31 and torch.equal(y[-9:], z)
    g = torch.autograd.grad(y, leaf, y.detach())[0]
    assert torch.equal(g[-9:], torch.autograd.grad(z, alone, z.detach())[0])
    del y, g
    x = leaf.detach().view(-1)[:65536 * 35000].view(65536, 35000)
    ids, top, labels = teacher_of(8, 35000, 5, 3, pad=False)
    few, labels = x[-8:].clone().requires_grad_(), labels.clamp_min(0)
    loss = M.distill_loss(few, top, ids, temperature=2.0, labels=labels, hard_weight=0.5)
    want = torch.autograd.grad(loss, few)[0]
    many = lambda t: t.repeat(8192, *[1] * (t.dim() - 1))
    leaf = x.requires_grad_()
    loss = M.distill_loss(leaf, many(top), many(ids), temperature=2.0, labels=many(labels), hard_weight=0.5)
    assert torch.equal(torch.autograd.grad(loss, leaf)[0][-8:] * 8192, want) and loss.isfinite()


def test_distill_every_class_named():
    """Nothing is left for the others: the term is 0, not a logarithm of nothing."""
    x = rnd((3, 12), torch.float32, 1)
    ids = torch.stack([torch.randperm(12, generator=torch.Generator().manual_seed(i)) for i in range(3)]).to(DEV)
    top = rnd((3, 12), torch.float32, 2)
    lse = torch.logsumexp(top.double(), -1).float()
    a, b = check_distill(x, top, ids, lse=lse), check_distill(x, top, ids)
    assert abs(a.item() - b.item()) < 1e-5


def test_distill_a_class_named_twice():
    x = rnd((4, 50), torch.float32, 1)
    ids = torch.tensor([[3, 3, 7], [9, 3, 9], [1, 1, 1], [49, 0, 49]], device=DEV)
    top = rnd((4, 3), torch.float32, 2)
    check_distill(x, top, ids)
    check_distill(x, top, ids, lse=lse_of(top, ids, 1.0))


def test_distill_infinite_logits():
    """A masked class of the student (-inf), one of the teacher, and far ones."""
    x = rnd((4, 300), torch.float32, 1)
    x[:, 20:40] = -math.inf
    ids = torch.tensor([[1, 2, 3, 50]] * 4, device=DEV)
    top = rnd((4, 4), torch.float32, 2)
    top[1, 2] = -math.inf
    x[2, 100] = 300.0
    check_distill(x, top, ids)
    check_distill(x, top, ids, lse=lse_of(top, ids, 1.0))
    x[3, 50] = -math.inf      # a class that the teacher gives a probability: infinitely far
    assert M.distill_loss(x, top, ids).item() == math.inf
    x[3, 60] = math.nan
    assert math.isnan(M.distill_loss(x, top, ids).item())


def test_distill_others_far_below():
    """The others' share far below what a sum beside the named classes could hold (exp(-200))."""
    x = rnd((3, 400), torch.float32, 1) - 200.0
    ids = torch.tensor([[5, 6, 7, 300]] * 3, device=DEV)
    x[:, ids[0]] += 200.0
    top = rnd((3, 4), torch.float32, 2)
    check_distill(x, top, ids, lse=lse_of(top, ids, 1.0, 0.1))


def test_distill_nothing_counts():
    x = rnd((6, 40), torch.float32, 1).requires_grad_()
    ids = torch.full((6, 3), -1, device=DEV)
    top = torch.full((6, 3), math.nan, device=DEV)
    labels = torch.full((6,), -100, device=DEV)
    loss = M.distill_loss(x, top, ids, labels=labels, hard_weight=0.5)
    loss.backward()
    assert loss.item() == 0.0 and not x.grad.any()


def test_distill_ids_outside():
    """No read or write outside the row; the loss is NaN."""
    x = rnd((4, 40), torch.float32, 1)
    top = rnd((4, 3), torch.float32, 2)
    ids = torch.tensor([[1, 2, 40], [0, 1, 2], [2 ** 40, 1, 2], [-5, 3, 1]], device=DEV)
    labels = torch.tensor([1, 2, 3, 4], device=DEV)
    for lse in (None, torch.ones(4, device=DEV) * 5):
        t = x.clone().requires_grad_()
        loss = M.distill_loss(t, top, ids, teacher_lse=lse)
        loss.backward()
        assert math.isnan(loss.item())
    for bad in (40, -1, 2 ** 50):
        labels[2] = bad
        assert math.isnan(M.distill_loss(x, top, ids.clamp(max=3), labels=labels, hard_weight=0.5).item())


def test_distill_shapes_strides_alignment():
    dt = torch.bfloat16
    x, (ids, top, labels) = rnd((12, 333), dt, 1), teacher_of(12, 333, 5, 2)
    ref = M.distill_loss(x, top, ids, labels=labels, hard_weight=0.5, temperature=2.0)
    again = M.distill_loss(unaligned(x).view(3, 4, 333), top.view(3, 4, 5), ids.view(3, 4, 5), labels=labels.view(3, 4), hard_weight=0.5,
                           temperature=2.0)
    strided = M.distill_loss(torch.cat((x, x), -1)[:, :333], torch.stack((top, top), -1)[..., 0], torch.stack((ids, ids), -1)[..., 1],
                             labels=torch.stack((labels, labels), -1)[:, 0], hard_weight=0.5, temperature=2.0)
    assert torch.equal(ref, again) and torch.equal(ref, strided)
    assert M.distill_loss(torch.empty((0, 5), device=DEV), torch.empty((0, 2), device=DEV),
                          torch.empty((0, 2), device=DEV, dtype=torch.int64)).item() == 0.0
    one = M.distill_loss(x[0], top[0], ids[0])            # a single row of one dimension
    assert torch.equal(one, M.distill_loss(x[:1], top[:1], ids[:1]))


# ---------------------------------------------------------------------------------------------------------------
# both: streams, graphs, nodes outside an ordinary backward
# ---------------------------------------------------------------------------------------------------------------
def both(x, add, w, b, head, top, ids, labels):
    """A step's end: norm, head, loss."""
    h, y = M.add_layer_norm(x, add, w, b)
    return M.distill_loss(y @ head, top, ids, labels=labels, hard_weight=0.4, temperature=2.0) + 0.01 * h.float().pow(2).mean()


def operands(dtype=torch.bfloat16, rows=50, d=136, vocab=1000):
    ids, top, labels = teacher_of(rows, vocab, 9, 3)
    leaves = [rnd((rows, d), dtype, 1), rnd((rows, d), dtype, 2), rnd((d,), dtype, 4, 0.1, 1.0), rnd((d,), dtype, 5),
              rnd((d, vocab), dtype, 6, 0.2)]
    return [t.requires_grad_() for t in leaves], (top, ids, labels)


def test_on_another_stream_and_the_same_bits():
    leaves, rest = operands()
    want = torch.autograd.grad(both(*leaves, *rest), leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(both(*leaves, *rest), leaves)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    """Forward and backward in one graph, replayed on changed inputs with eager work between."""
    leaves, rest = operands()
    data = [t.detach().clone() for t in leaves]

    def step():
        ts = [t.detach().requires_grad_() for t in data]
        loss = both(*ts, *rest)
        return (loss.detach(), *torch.autograd.grad(loss, ts))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        data[0].copy_(rnd(data[0].shape, data[0].dtype, 20 + i))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_double_backward_and_watched_backward():
    """A backward that is differentiated, or batched, takes the torch form: its gradient against the kernels', and its own
    gradient against differences."""
    leaves, rest = operands(torch.float32, rows=6, d=24, vocab=30)
    loss = both(*leaves, *rest)
    plain = torch.autograd.grad(loss, leaves, retain_graph=True)
    graphed = torch.autograd.grad(loss, leaves, create_graph=True)
    for a, b in zip(plain, graphed):
        assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-7
    v = [rnd(t.shape, t.dtype, 40 + i) for i, t in enumerate(leaves)]
    hv = torch.autograd.grad(sum((g * u).sum() for g, u in zip(graphed, v)), leaves)
    f = [t.detach().double().cpu().requires_grad_() for t in leaves]
    cpu = [t.cpu() for t in rest]
    g64 = torch.autograd.grad(both(*f, *cpu), f, create_graph=True)
    h64 = torch.autograd.grad(sum((g * u.double().cpu()).sum() for g, u in zip(g64, v)), f)
    for a, b in zip(hv, h64):
        assert (a.double().cpu() - b).norm() <= 1e-4 * b.norm()
    out = M.layer_norm(leaves[0], leaves[2], leaves[3])
    eye = torch.eye(out.numel(), device=DEV).view(-1, *out.shape)[:5]
    rows = torch.autograd.grad(out, leaves[0], eye, is_grads_batched=True, retain_graph=True)[0]
    for e, r in zip(eye, rows):
        assert torch.allclose(torch.autograd.grad(out, leaves[0], e, retain_graph=True)[0], r, atol=1e-5)


def test_saved_tensors_from_hooks():
    leaves, rest = operands()
    want = torch.autograd.grad(both(*leaves, *rest), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = both(*leaves, *rest)
    for a, b in zip(torch.autograd.grad(loss, leaves), want):
        assert torch.equal(a, b)
    x = leaves[0]
    for bad in (lambda t: t.reshape(-1)[:8], lambda t: t.cpu(), lambda t: t.double()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            y, loss = M.layer_norm(x, leaves[2]), M.distill_loss(x, rest[0], rest[1].clamp(max=5))
        for o in (y, loss):
            with pytest.raises(RuntimeError, match="hook"):
                o.sum().backward()


def test_compile_and_tracing():
    from torch.fx.experimental.proxy_tensor import make_fx
    leaves, rest = operands()
    plain = [t.detach() for t in leaves]
    want = both(*plain, *rest)
    traced = make_fx(lambda *a: both(*a, *rest))(*plain)
    assert abs(traced(*plain).item() - want.item()) <= 0.02 * abs(want.item())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert M.layer_norm(plain[0], plain[2], plain[3]).dtype is torch.bfloat16
    mixed = M.layer_norm(plain[0], plain[2].float(), plain[3].float())   # mixed types: the torch form
    close(mixed, M.layer_norm(plain[0].float(), plain[2].float(), plain[3].float()).double(), 1e-5)
