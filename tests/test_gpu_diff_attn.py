"""Differential attention (model_ops.diff_attention) on the kernels against its formulas in fp64 on the same inputs.

h is half a step of the type (2^-8 of a bf16 value, 2^-11 of an fp16 one), u = 2^-24. Bounds, element by element:
  * a score is a sum of dh products in fp32, so it is within (dh + 8) u of the sum of their absolute values S; the probabilities, and
    the sums over at most n keys that divide them, are within e = 2 (dh + 8) u max S + (n / 64 + 64) u of themselves (a wave's lane
    adds the keys of a 64-key tile in four sums, then tile after tile);
  * forward: each probability enters the product rounded to the type, so P v is within (h + 2 e) sum p |v|, y within that for both
    maps, and is rounded once more;
  * backward: D1 and D2 come from the rounded y and P2 v, so they are within dy . (their bounds); a score gradient is within
    p (bound of D) + e |p (dA - D)| and is rounded to the type before the products that sum it, as the combined map is; dlam sums
    p dA in fp32. A result is rounded once;
  * what is rounded below a type's smallest normal number may lose all of it: 2^-25 in fp16 (half of its smallest subnormal), 2^-126
    in bf16 and fp32 (flushed), times a few for the products that it enters (FLOOR)."""
import math

import pytest
import torch

from gpu_helpers import DEV
from loopback_amd import model_ops as M

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]
U = 2.0 ** -24
FLOOR = {torch.bfloat16: 2.0 ** -124, torch.float16: 2.0 ** -25}


def rnd(shape, dtype, seed, std=1.0, mean=0.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean
    return x.to(dtype).to(DEV)


def close(got, ref, slack, what):
    half = HALF.get(got.dtype, U)
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0
    bad = (got.double() - ref).abs() > half * (ref.abs() + slack) + slack + tiny
    worst = ((got.double() - ref).abs() / (half * (ref.abs() + slack) + slack + tiny + 1e-300)).max().item()
    assert got.shape == ref.shape and got.isfinite().all() and not bad.any(), (what, int(bad.sum()), worst)


def reference(q, k, v, lam, dy, causal=True, scale=None, lengths=None, starts=None):
    """{name: (value, slack)}."""
    half, floor = HALF[q.dtype], FLOOR[q.dtype]
    f = lambda t: t.double()  # noqa: E731
    (b, tq, h2, dh), (tk, hk, dv) = q.shape, v.shape[1:]
    h = h2 // 2
    scale = dh ** -0.5 if scale is None else scale
    dev = q.device
    out = {n: (torch.zeros(s, dtype=torch.float64, device=dev), torch.zeros(s, dtype=torch.float64, device=dev))
           for n, s in (("y", (b, tq, h, dv)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("dlam", (b, tq, h)))}
    lam_all = f(lam).expand(b, tq, h)
    i, j = torch.arange(tq, device=dev).view(-1, 1), torch.arange(tk, device=dev)
    for n in range(b):
        length = tk if lengths is None else min(max(int(lengths[n]), 0), tk)
        start = tk - tq if starts is None else int(starts[n])
        seen = (j < length) & ((j <= start + i) if causal else torch.ones_like(i, dtype=torch.bool))
        for x in range(h):
            g = x // (h // hk)
            vv, vals = torch.where((j < length).view(-1, 1), f(v[n, :, g]), 0.0), []
            for m in range(2):
                kk = torch.where((j < length).view(-1, 1), f(k[n, :, 2 * g + m]), 0.0)
                qq = f(q[n, :, 2 * x + m])
                s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                size = torch.where(seen, qq.abs() @ kk.abs().T * scale, 0.0).amax(-1, keepdim=True)
                e = 2 * (dh + 8) * U * size + (tk / 64 + 64) * U
                vals.append((p, e, kk, qq))
            (p1, e1, k1, q1), (p2, e2, k2, q2) = vals
            lm = lam_all[n, :, x].unsqueeze(-1)
            pv1, pv2 = (half + 2 * e1) * (p1 @ vv.abs()), (half + 2 * e2) * (p2 @ vv.abs())
            z = p2 @ vv
            y = p1 @ vv - lm * z
            by = pv1 + lm.abs() * pv2 + 4 * U * (p1 @ vv.abs() + (lm * z).abs())
            by = by + floor * (1 + lm.abs()) * (seen.double() @ vv.abs())
            out["y"][0][n, :, x], out["y"][1][n, :, x] = y, by
            if dy is None:
                continue
            g_ = f(dy[n, :, x])
            da = g_ @ vv.T
            eda = (dv + 8) * U * (g_.abs() @ vv.abs().T)
            d1, d2 = (p1 * da).sum(-1, keepdim=True), (p2 * da).sum(-1, keepdim=True)
            b2 = (g_.abs() * (half * (z.abs() + pv2) + pv2 + (dv + 8) * U * z.abs())).sum(-1, keepdim=True)
            b1 = (g_.abs() * (half * (y.abs() + by) + by + (dv + 8) * U * (y.abs() + (lm * z).abs()))).sum(-1, keepdim=True) + lm.abs() * b2
            for m, (p, e, kk, qq, d, bd, w) in enumerate(((p1, e1, k1, q1, d1, b1, torch.ones_like(lm)), (p2, e2, k2, q2, d2, b2, -lm))):
                ds = p * (da - d) * w
                bs = w.abs() * p * (bd + eda + 4 * U * (da.abs() + d.abs())) + (half + e + 8 * U) * ds.abs()
                bs = bs + half * w.abs() * p * (bd + eda) + floor * seen * (1 + da.abs() + d.abs()) * (1 + w.abs())
                out["dq"][0][n, :, 2 * x + m], out["dq"][1][n, :, 2 * x + m] = ds @ kk * scale, (bs + tk * U * ds.abs()) @ kk.abs() * scale
                out["dk"][0][n, :, 2 * g + m] += ds.T @ qq * scale
                out["dk"][1][n, :, 2 * g + m] += (bs + tq * U * ds.abs()).T @ qq.abs() * scale
            a = p1 - lm * p2
            out["dv"][0][n, :, g] += a.T @ g_
            out["dv"][1][n, :, g] += (half * a.abs() + (e1 + 4 * U) * p1 * (1 + half) + (e2 + 4 * U) * p2 * lm.abs() * (1 + half)
                                      + tq * U * (p1 + lm.abs() * p2) + floor * seen * (1 + lm.abs())).T @ g_.abs()
            out["dlam"][0][n, :, x] = -d2.squeeze(-1)
            out["dlam"][1][n, :, x] = (p2 * ((e2 + 2 * U + tk * U) * da.abs() + eda)).sum(-1)
    if lam.dim() < 3:
        dims = (0, 1) if lam.dim() == 1 else (0, 1, 2)
        val, s = out["dlam"]
        out["dlam"] = (val.sum(dims), s.sum(dims) + (b * tq * h) * U * val.abs().sum(dims))
    return out


def operands(b, tq, tk, h, hk, dh, dv, dtype, lam="head", seed=1, std=1.0):
    shape = {"layer": (), "head": (h,), "token": (b, tq, h)}[lam]
    return [rnd((b, tq, 2 * h, dh), dtype, seed, std), rnd((b, tk, 2 * hk, dh), dtype, seed + 1, std), rnd((b, tk, hk, dv), dtype, seed + 2),
            rnd(shape, dtype, seed + 3, 0.3, 0.5)]


def ints(*v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def check(ts, train=True, **how):
    dy = rnd((*ts[0].shape[:2], ts[0].shape[2] // 2, ts[2].shape[3]), ts[0].dtype, 77) if train else None
    ref = reference(*ts, dy, **how)
    plain = M.diff_attention(*ts, **how)
    close(plain, *ref["y"], "y")
    if not train:
        return
    leaves = [t.detach().requires_grad_() for t in ts]
    y = M.diff_attention(*leaves, **how)
    close(y.detach(), *ref["y"], "recorded y")
    for name, g in zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(y, leaves, dy)):
        close(g, *ref[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh,dv", [(64, 128), (64, 64), (40, 80), (8, 8), (32, 64), (128, 256), (96, 192), (128, 128), (64, 192)])
@pytest.mark.parametrize("t", [1, 2, 31, 65, 200])
def test_widths_and_lengths(t, dh, dv, dtype):
    check(operands(2, t, t, 2, 1, dh, dv, dtype))


@pytest.mark.parametrize("lam", ["layer", "head", "token"])
@pytest.mark.parametrize("b,h,hk", [(1, 1, 1), (3, 4, 4), (2, 6, 2), (4, 8, 2)])
def test_heads_and_lambda(b, h, hk, lam):
    check(operands(b, 130, 130, h, hk, 64, 128, torch.bfloat16, lam))


@pytest.mark.parametrize("dtype", TYPES)
def test_lambda_in_fp32_negative_and_zero(dtype):
    ts = operands(2, 70, 70, 4, 2, 64, 128, dtype)
    for lam in (torch.tensor([0.7, -0.4, 0.0, 1.5], device=DEV), torch.tensor(-0.3, device=DEV), torch.randn(2, 70, 4, device=DEV)):
        check([*ts[:3], lam])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tq,tk", [(1, 1), (1, 700), (3, 64), (5, 333), (40, 41), (100, 300), (129, 1000), (70, 30)])
def test_chunks(tq, tk, causal):
    """Queries that are the last tokens; more queries than keys: the first ones see none."""
    check(operands(2, tq, tk, 4, 2, 64, 128, torch.bfloat16), causal=causal)


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_ragged(train, wide):
    """Lengths and positions of each sequence: none, one, inside and at a tile's end, past the tensor; queries before the first key."""
    b, tk = 8, 300
    lengths = ints(0, 1, 63, 64, 65, 300, 1000, -4, dtype=wide)
    for tq in (1, 5, 150):
        ts = operands(b, tq, tk, 4, 2, 64, 128, torch.bfloat16, "token")
        check(ts, train, lengths=lengths)
        check(ts, train, lengths=lengths, starts=lengths.clamp(0, tk) - tq)
        check(ts, train, lengths=lengths, starts=ints(-1000, 0, 5, -3, 64, 299, 2 ** 31 - 1, -2 ** 31, dtype=wide))
        check(ts, train, lengths=lengths, causal=False)


def test_what_is_past_the_lengths():
    """NaN and infinities in an unwritten cache reach nothing, and their gradient is zero."""
    lengths = ints(0, 1, 70, 128, 199)
    for tq in (1, 200):
        ts = operands(5, tq, 200, 4, 2, 64, 128, torch.bfloat16)
        how = {"lengths": lengths, "starts": lengths - tq if tq == 1 else ints(0, 0, 0, 0, 0)}
        ref = M.diff_attention(*ts, **how)
        for n, length in enumerate(lengths.tolist()):
            ts[1][n, length:], ts[2][n, length:] = math.nan, math.inf
        assert torch.equal(M.diff_attention(*ts, **how), ref) and not ref[0].any()
        leaves = [t.detach().requires_grad_() for t in ts]
        grads = torch.autograd.grad(M.diff_attention(*leaves, **how), leaves, torch.ones_like(ref))
        assert all(g.isfinite().all() for g in grads)
        for n, length in enumerate(lengths.tolist()):
            assert not grads[1][n, length:].any() and not grads[2][n, length:].any()
        assert not grads[0][0].any()


@pytest.mark.parametrize("b,tq,tk,h,hk", [(1, 1, 20000, 2, 1), (2, 8, 5000, 8, 2), (32, 1, 1500, 4, 4), (1, 32, 4097, 1, 1), (300, 1, 40, 2, 2)])
def test_few_queries_over_long_caches(b, tq, tk, h, hk):
    ts = operands(b, tq, tk, h, hk, 64, 128, torch.bfloat16)
    check(ts, False)
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, tk + 1, (b,), generator=g, dtype=torch.int32).to(DEV)
    check(ts, False, lengths=lengths, starts=lengths - tq)


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("b,tq,tk,h,hk,dh,dv,dtype", [
    (1, 333, 2049, 4, 2, 64, 128, torch.bfloat16), (2, 65, 5000, 2, 1, 40, 80, torch.float16), (1, 1, 3000, 2, 2, 64, 64, torch.bfloat16),
    (1, 700, 1100, 6, 3, 128, 256, torch.bfloat16), (3, 2000, 800, 1, 1, 32, 32, torch.float16)])
def test_few_blocks_over_long_keys(b, tq, tk, h, hk, dh, dv, dtype, train):
    """Blocks of queries too few for the CUs, whose keys go in chunks: sequences that end before a chunk, and within one."""
    ts = operands(b, tq, tk, h, hk, dh, dv, dtype, "token")
    check(ts, train)
    check(ts, train, causal=False)
    lengths = ints(*(min(tk, 255 + 300 * i) for i in range(b)))
    check(ts, train, lengths=lengths, starts=lengths - tq // 2)
    check(ts, train, lengths=ints(*(0 if i == 0 else tk for i in range(b))), starts=ints(*(-3 if i == 0 else 600 for i in range(b))))


def test_a_cache_past_32_bits():
    """Keys and values as parts of wide rows, 5 GB from the first to the last: the result and the gradients of compact copies."""
    tk, wide = 20000, 2 ** 17
    big = torch.empty(tk * wide, dtype=torch.bfloat16, device=DEV).view(1, tk, wide)
    q, k, v, lam = operands(1, 3, tk, 2, 1, 64, 128, torch.bfloat16)
    far = [big[:, :, 64:192].view(1, tk, 2, 64), big[:, :, wide - 128:].view(1, tk, 1, 128)]
    far[0].copy_(k), far[1].copy_(v)
    assert (tk - 1) * wide * 2 > 2 ** 32 and torch.equal(M.diff_attention(q, *far, lam), M.diff_attention(q, k, v, lam))
    leaves = [t.detach().requires_grad_() for t in (q, *far, lam)]
    near = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    a, b = M.diff_attention(*leaves), M.diff_attention(*near)
    dy = rnd(a.shape, torch.bfloat16, 7)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, leaves, dy), torch.autograd.grad(b, near, dy)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh,dv", [(64, 128), (128, 256), (40, 80)])
def test_a_single_key_has_no_score_gradient(dh, dv, dtype):
    """Sequences of one key, the first query of a causal one, and one key for many queries: zeros, as the probability is 1."""
    for t, causal, lengths in ((1, True, None), (70, True, None), (70, False, ints(1, 1)), (70, True, ints(1, 70))):
        leaves = [x.detach().requires_grad_() for x in operands(2, t, t, 4, 2, dh, dv, dtype, "token")]
        y = M.diff_attention(*leaves, causal=causal, lengths=lengths)
        dq, dk, dval, _ = torch.autograd.grad(y, leaves, rnd(y.shape, dtype, 8))
        assert (dq[:, 0] == 0).all() and dval[:, 0].abs().max() > 0
        if t == 1 or not causal:
            assert (dq == 0).all() and (dk == 0).all()
        elif lengths is not None:
            assert (dq[0] == 0).all() and (dk[0] == 0).all() and dq[1, 1:].abs().max() > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [2, 3, 4, 9, 40, 100, 128])
def test_score_gradients_of_short_sequences(t, dtype):
    """Of up to 128 keys the sums that a score's gradient is relative to are fp32: it is rounded once to the type, and its products'
    sum once. fp32's share: dA and D are sums of 128 products, P a score's exponential, within 64 u of |dy| |v| and of themselves."""
    q, k, v, lam = operands(2, t, t, 1, 1, 64, 128, dtype)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
    y = M.diff_attention(*leaves)
    dy = rnd(y.shape, dtype, 8)
    dq, dk = torch.autograd.grad(y, leaves[:2], dy)
    h, c = HALF[dtype], 64 ** -0.5
    q, k, v, g, lam = (x.detach().double() for x in (q, k, v, dy, lam))
    da, size = g[:, :, 0] @ v[:, :, 0].transpose(1, 2), g[:, :, 0].abs() @ v[:, :, 0].abs().transpose(1, 2)
    for e, f in ((0, 1.0), (1, -float(lam[0]))):
        s = q[:, :, e] @ k[:, :, e].transpose(1, 2) * c
        p = s.masked_fill(torch.ones(t, t, device=DEV).triu(1).bool(), -math.inf).softmax(-1)
        ds = c * f * p * (da - (p * da).sum(-1, keepdim=True))
        fp32 = 128 * U * c * abs(f) * p * (size + (p * size).sum(-1, keepdim=True))
        for got, other, left in ((dq[:, :, e], k[:, :, e], ds), (dk[:, :, e], q[:, :, e], ds.transpose(1, 2))):
            more = fp32 if left is ds else fp32.transpose(1, 2)
            bound = (h * left.abs() + (1 + h) * more) @ other.abs()
            ref = left @ other
            assert ((got.double() - ref).abs() <= h * (ref.abs() + bound) + bound + FLOOR[dtype] * (1 + other.abs().sum(1, keepdim=True))).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tq,tk,starts", [(128, 129, None), (130, 131, None), (200, 201, None), (200, 280, None), (200, 264, (1, 64)),
                                          (200, 200, (-3, -150)), (150, 300, (64, 0)), (300, 300, (-100, 2))])
def test_score_gradients_of_queries_that_see_few_keys(tq, tk, starts, dtype):
    """As of short sequences, whatever the other queries see: those that see more than 128 keys have no gradient here, so that dk is
    the few ones' too."""
    q, k, v, lam = operands(2, tq, tk, 1, 1, 64, 128, dtype)
    start = torch.full((2,), tk - tq, device=DEV) if starts is None else ints(*starts, dtype=torch.int64)
    keys = (start.view(2, 1) + torch.arange(tq, device=DEV) + 1).clamp(0, tk)          # that each query sees
    dy = rnd((2, tq, 1, 128), dtype, 8) * (keys <= 128).view(2, tq, 1, 1)
    assert (keys.amax() > 128) and ((keys >= 2) & (keys <= 128)).any()
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
    y = M.diff_attention(*leaves, starts=None if starts is None else start)
    dq, dk = torch.autograd.grad(y, leaves[:2], dy)
    h, c = HALF[dtype], 64 ** -0.5
    q, k, v, g, lam = (x.detach().double() for x in (q, k, v, dy, lam))
    da, size = g[:, :, 0] @ v[:, :, 0].transpose(1, 2), g[:, :, 0].abs() @ v[:, :, 0].abs().transpose(1, 2)
    hidden = torch.arange(tk, device=DEV) >= keys.unsqueeze(-1)
    for e, f in ((0, 1.0), (1, -float(lam[0]))):
        s = q[:, :, e] @ k[:, :, e].transpose(1, 2) * c
        p = torch.nan_to_num(s.masked_fill(hidden, -math.inf).softmax(-1), nan=0.0)
        ds = c * f * p * (da - (p * da).sum(-1, keepdim=True))
        fp32 = 128 * U * c * abs(f) * p * (size + (p * size).sum(-1, keepdim=True))
        for got, other, left in ((dq[:, :, e], k[:, :, e], ds), (dk[:, :, e], q[:, :, e], ds.transpose(1, 2))):
            more = fp32 if left is ds else fp32.transpose(1, 2)
            bound = (h * left.abs() + (1 + h) * more) @ other.abs()
            ref = left @ other
            assert ((got.double() - ref).abs() <= h * (ref.abs() + bound) + bound + FLOOR[dtype] * (1 + other.abs().sum(1, keepdim=True))).all()


def powers(shape, seed):
    """+-1, 2 or 4: a power of two times them is exact in fp16 down to its smallest number, 2^-24."""
    g = torch.Generator().manual_seed(seed)
    return (torch.exp2(torch.randint(0, 3, shape, generator=g).float()) * (torch.randint(0, 2, shape, generator=g) * 2 - 1)).to(DEV)


def gradients(ts, dy, **how):
    leaves = [t.detach().requires_grad_() for t in ts]
    return torch.autograd.grad(M.diff_attention(*leaves, **how), leaves, dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lam", ["head", "token"])
@pytest.mark.parametrize("t,h,hk,dh,dv", [(1, 1, 1, 64, 128), (100, 2, 1, 64, 128), (300, 2, 2, 64, 128), (700, 4, 1, 40, 80), (300, 2, 1, 128, 256)])
def test_gradients_of_small_and_large_upstreams(t, h, hk, dh, dv, lam, dtype):
    """Gradients are linear: those of 2^k dy are 2^k times those of dy, each rounded once, from upstreams of 2^-24 to some with which
    a score gradient before its scale is past 65504. Nothing between the two roundings depends on 2^k: an intermediate in the type
    would, below its smallest normal number and past its largest."""
    ts = operands(2, t, t, h, hk, dh, dv, dtype, lam)
    ts[1], ts[2] = ts[1] * 0.25, ts[2] * 0.5      # the largest results are of some thousands
    lengths = ints(t, (t + 1) // 2)
    dy = powers((2, t, h, dv), 5)
    one = gradients(ts, dy.to(dtype), lengths=lengths)
    half, tiny = HALF[dtype], 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126
    for k in (-24, -17, -10, 9, 12):
        for name, got, ref in zip(("dq", "dk", "dv", "dlam"), gradients(ts, (dy * 2.0 ** k).to(dtype), lengths=lengths), one):
            ref = ref.double() * 2.0 ** k
            if dtype is torch.float16 and ref.abs().max() > 60000:
                assert name in ("dv", "dlam") and k > 0   # past the range
                continue
            off = ((got.double() - ref).abs() - (2.1 * half * ref.abs() + tiny * (1 + 2.0 ** k))).max().item()
            assert off <= 0, (name, k, off, ref.abs().max().item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh,dv", [(64, 128), (128, 256)])
def test_gradients_of_queries_of_different_sizes(dh, dv, dtype):
    """A query's own gradient is as near beside queries whose upstreams are 2^20 times as large; and of the keys that see only small
    ones, those of the last block."""
    t, half, tiny = 400, HALF[dtype], 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126
    ts = operands(2, t, t, 2, 1, dh, dv, dtype, "token")
    ts[1], ts[2] = ts[1] * 0.25, ts[2] * 0.5
    dy, k = powers((2, t, 2, dv), 5), torch.full((2, t, 1, 1), -11.0, device=DEV)
    k[:, 100:120], k[:, 7], k[:, 150] = 9.0, -24.0, -20.0
    one, got = (gradients(ts, (dy * f).to(dtype)) for f in (1.0, torch.exp2(k)))
    ref = one[0].double() * torch.exp2(k).double()
    off = ((got[0].double() - ref).abs() - (2.1 * half * ref.abs() + tiny * (1 + torch.exp2(k).double()))).max().item()
    assert off <= 0
    for a, b in zip(got[1:3], one[1:3]):
        a, b = a[:, 384:].double(), b[:, 384:].double() * 2.0 ** -11
        off = ((a - b).abs() - (2.1 * half * b.abs() + tiny)).max().item()
        assert off <= 0


@pytest.mark.parametrize("dtype", TYPES)
def test_large_lambdas_and_infinite_upstreams(dtype):
    """Lambdas of hundreds and thousands; a query whose upstream is infinite leaves the others' gradients as they are without it."""
    ts = operands(2, 150, 150, 2, 1, 64, 128, dtype)
    for lam in (torch.tensor([300.0, -3000.0], device=DEV), torch.tensor([0.001, 2000.0], device=DEV).expand(2, 150, 2)):
        check([*ts[:3], lam])
    dy = rnd((2, 150, 2, 128), dtype, 9)
    dy[:, 70, 1] = 0.0
    ref = gradients(ts, dy)[0]
    dy[:, 70, 1, 5] = math.inf
    got = gradients(ts, dy)[0]
    assert not got[:, 70, 2:].isfinite().any()
    got[:, 70, 2:] = 0.0
    assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, 0.75 * 2.0 ** -8), (torch.float16, 0.75 * 2.0 ** -11)])
def test_values_gradient_of_many_keys(dtype, bound):
    """32768 keys whose probabilities are about 2^-15: dv is a sum over the queries of P dy, whose factors' roundings are independent, of
    half a step at most and 0.41 of it in the norm (over a binade: 1 / 3 of its square by 7 / 3 or less), and so is its own rounding:
    together sqrt(2) 0.41 = 0.58 of half a step, here below 0.75."""
    t = 32768
    q, k, v, lam = operands(1, t, t, 1, 1, 64, 128, dtype, "layer")
    dy = rnd((1, t, 1, 128), dtype, 9)
    got = gradients([q, k, v, lam], dy, causal=False)[2][0, :, 0].double()
    ref = torch.zeros_like(got)
    for at in range(0, t, 4096):   # blocks of queries
        p = [torch.softmax(q[0, at:at + 4096, m].double() @ k[0, :, m].double().T.contiguous() / 8, -1) for m in (0, 1)]
        ref += (p[0] - lam.double() * p[1]).T.contiguous() @ dy[0, at:at + 4096, 0].double()
    off = ((got - ref).norm() / ref.norm()).item()
    assert off <= bound, off


def test_one_tensor_twice():
    """The queries as the keys too, and keys that are the values' storage: the same results and gradients as from copies."""
    q, _, _, lam = operands(2, 100, 100, 2, 2, 64, 128, torch.bfloat16)
    far = lam.detach()[0].expand(2, 100, 2)   # one value for every query, without strides
    def run(q, k, v, lam):
        y = M.diff_attention(q, k, v, lam)
        return y, torch.autograd.grad(y, [q], rnd(y.shape, torch.bfloat16, 5))[0]
    one = q.detach().requires_grad_()
    two = [q.detach().clone().requires_grad_() for _ in range(3)]
    y, g = run(one, one, one.view(2, 100, 2, 128), far)
    z = M.diff_attention(two[0], two[1], two[2].view(2, 100, 2, 128), far.contiguous())
    grads = torch.autograd.grad(z, two, rnd(z.shape, torch.bfloat16, 5))
    assert torch.equal(y, z)
    # the three gradients are added in bf16, in any order
    total, size = sum(t.double() for t in grads), sum(t.double().abs() for t in grads)
    assert ((g.double() - total).abs() <= 2 * 2.0 ** -8 * size).all()


def test_far_scores():
    """Scores of hundreds, rising and falling along the keys: the running maximum moves at every tile, or never."""
    for sign in (1.0, -1.0):
        q, k, v, lam = operands(1, 200, 200, 2, 1, 64, 128, torch.bfloat16)
        ramp = torch.linspace(0, 30, 200, device=DEV).view(1, -1, 1, 1)
        k = (k * 0.1 + sign * ramp * 0.25).to(k.dtype)
        q = (q * 0.1 + 3.0).to(q.dtype)
        check([q, k, v, lam])


def test_scale_strides_alignment():
    dt = torch.bfloat16
    q, k, v, lam = operands(2, 90, 90, 4, 2, 64, 128, dt)
    ref = M.diff_attention(q, k, v, lam, scale=0.3)
    check([q, k, v, lam], scale=0.3)
    fused = torch.cat((q.flatten(2), k.flatten(2), v.flatten(2)), -1)      # one projection's output, split
    parts = fused.split([512, 256, 256], -1)
    views = [parts[0].view(2, 90, 8, 64), parts[1].view(2, 90, 4, 64), parts[2].view(2, 90, 2, 128)]
    assert torch.equal(M.diff_attention(*views, lam, scale=0.3), ref)
    odd = [torch.empty(t.numel() + 1, dtype=dt, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(M.diff_attention(*odd, lam, scale=0.3), ref)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]      # heads before tokens
    assert torch.equal(M.diff_attention(*turned, lam, scale=0.3), ref)
    last = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]        # columns apart
    assert torch.equal(M.diff_attention(*last, lam, scale=0.3), ref)
    shared = M.diff_attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), lam.unsqueeze(0).expand(2, 90, 4), scale=0.3)
    assert torch.equal(shared[0], ref[0])
    leaves = [t.detach().requires_grad_() for t in (*odd, lam)]
    a = torch.autograd.grad(M.diff_attention(*leaves, scale=0.3).transpose(1, 2), leaves, torch.ones(2, 4, 90, 128, device=DEV, dtype=dt))
    leaves = [t.detach().requires_grad_() for t in (*last, lam)]
    b = torch.autograd.grad(M.diff_attention(*leaves, scale=0.3), leaves, torch.ones((), device=DEV, dtype=dt).expand(2, 90, 4, 128))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_strides_of_dimensions_of_one():
    """A dimension of one may have any stride, which a contiguous copy keeps: one sequence and one token of a projection of an odd
    width, one sequence cut from odd rows, one head of keys cached heads first and further than 2^23 elements apart."""
    dt = torch.bfloat16
    def same(ts, views, **how):
        for n, (t, x) in enumerate(zip(ts, views)):
            assert torch.equal(t, x), n
        assert torch.equal(M.diff_attention(*views, **how), M.diff_attention(*ts, **how))
        a, b = ([t.detach().requires_grad_() for t in x] for x in (views, ts))
        ya, yb = M.diff_attention(*a, **how), M.diff_attention(*b, **how)
        dy = rnd(ya.shape, dt, 9)
        assert torch.equal(ya, yb)
        for x, y in zip(torch.autograd.grad(ya, a, dy), torch.autograd.grad(yb, b, dy)):
            assert torch.equal(x, y)

    ts = operands(1, 1, 1, 4, 2, 64, 128, dt, "token")
    row, at, views = torch.cat([t.flatten() for t in ts]), 0, []
    for t in ts:
        views.append(row.as_strided(t.shape, (1028, 1028, *t.stride()[2:]), at))
        at += t.numel()
    same(ts, views)
    *rows, lam = operands(1, 2, 2, 2, 2, 64, 128, dt)
    same([*rows, lam], [*(t.as_strided(t.shape, (517, *t.stride()[1:])) for t in rows), lam])
    for tq in (1, 3):   # a kernel of few queries, and for a backward the others
        q, k, v, lam = operands(1, tq, 70000, 2, 1, 64, 128, dt)
        far = v.transpose(1, 2).contiguous().transpose(1, 2)
        far = far.as_strided(far.shape, (70000 * 128, 128, 70000 * 128, 1))
        assert far.stride(2) > 2 ** 23
        same([q, k, v, lam], [q, k, far, lam])


def test_rows_too_far_apart_for_the_kernels():
    """Rows of more than 2^23 elements: torch operations."""
    q = torch.zeros(1, 2, 2 ** 17 + 2, 64, dtype=torch.bfloat16, device=DEV)
    k, v = rnd((1, 2, 2, 64), torch.bfloat16, 1), rnd((1, 2, 1, 128), torch.bfloat16, 2)
    lam = torch.tensor(0.5, device=DEV)
    assert not M.attention_native(q, k, v, lam) and M.attention_native(q[:, :1], k, v, lam) and M.attention_native(q[:, :, 2:], k, v, lam)
    close(M.diff_attention(q, k, v, lam)[:, :, :2], *reference(q[:, :, :4], k, v, lam, None)["y"], "y")
    one = M.diff_attention(q[:, :1], k, v, lam)
    close(one[:, :, -2:], *reference(q[:, :1, -4:], k, v, lam, None)["y"], "y")


def test_wide_results_take_torch_operations():
    """Results of more than 2^26 elements a token, whose gradient's rows the kernels do not reach."""
    def native(tq, h, dv):
        one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
        return M.attention_native(one.expand(1, tq, 2 * h, 8), one.expand(1, tq, 2, 8), one.expand(1, tq, 1, dv), one.expand(1, tq, h))
    assert native(20, 2 ** 19, 128) and not native(20, 2 ** 19, 136) and native(1, 2 ** 19, 256)


def test_gradients_that_are_asked_for():
    ts = operands(2, 77, 77, 4, 2, 64, 128, torch.bfloat16)
    dy = rnd((2, 77, 4, 128), torch.bfloat16, 9)
    leaves = [t.clone().requires_grad_() for t in ts]
    full = torch.autograd.grad(M.diff_attention(*leaves), leaves, dy)
    for need in range(1, 16):
        leaves = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate(ts)]
        got = torch.autograd.grad(M.diff_attention(*leaves), [t for t in leaves if t.requires_grad], dy)
        for a, b in zip(got, [g for i, g in enumerate(full) if need >> i & 1]):
            assert torch.equal(a, b)


def test_against_differences():
    """The kernels' gradient along a direction against differences of the plain forward in fp64."""
    ts = operands(1, 40, 40, 2, 1, 64, 128, torch.float16)
    dy = rnd((1, 40, 2, 128), torch.float16, 9)
    leaves = [t.clone().requires_grad_() for t in ts]
    got = torch.autograd.grad(M.diff_attention(*leaves), leaves, dy)
    f = [t.double().cpu() for t in ts]
    eps = 1e-5
    for i, g in enumerate(got):
        d = torch.randn(f[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        side = [M.diff_attention(*[t + s * eps * d if n == i else t for n, t in enumerate(f)]) for s in (1, -1)]
        want = ((side[0] - side[1]) / (2 * eps) * dy.double().cpu()).sum()
        # the bounds above, each element's, along the direction
        ref = reference(*ts, dy)[("dq", "dk", "dv", "dlam")[i]]
        slack = ((HALF[torch.float16] * ref[0].abs() + 2 * ref[1]).cpu() * d.abs()).sum() + 1e-6 * want.abs()
        assert abs((g.double().cpu() * d).sum() - want) <= slack


def test_streams_graphs_and_the_same_bits():
    ts = operands(3, 150, 150, 4, 2, 64, 128, torch.bfloat16, "token")
    lengths = ints(150, 20, 0)
    dy = rnd((3, 150, 4, 128), torch.bfloat16, 9)

    def step(n):
        leaves = [t.detach().requires_grad_() for t in ts]
        y = M.diff_attention(*leaves, lengths=n)
        few = M.diff_attention(ts[0][:, -1:].detach(), *(t.detach() for t in ts[1:3]), torch.ones((), device=DEV), lengths=n)
        return (y.detach(), few, *torch.autograd.grad(y, leaves, dy))

    want = step(lengths)
    for a, b in zip(step(lengths), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(lengths)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(lengths)
    for n in ((150, 20, 0), (3, 150, 64), (0, 0, 1)):
        lengths.copy_(ints(*n))
        ts[0].add_(0.125)
        want = [t.clone() for t in step(lengths)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_watched_and_differentiated_backwards():
    ts = operands(1, 9, 9, 2, 1, 16, 32, torch.bfloat16)
    leaves = [t.requires_grad_() for t in ts]
    y = M.diff_attention(*leaves)
    dy = rnd(y.shape, y.dtype, 9)
    plain = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    graphed = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for a, b in zip(plain, graphed):
        assert (a.double() - b.double()).norm() <= 0.02 * b.double().norm()
    again = torch.autograd.grad(sum((g.float() ** 2).sum() for g in graphed), leaves)
    assert all(g.isfinite().all() and g.any() for g in again)
    rows = torch.autograd.grad(y, leaves[0], torch.stack((dy, 2 * dy)), is_grads_batched=True, retain_graph=True)[0]
    assert (rows[0].double() - plain[0].double()).norm() <= 0.02 * plain[0].double().norm()
    for bad in (lambda t: t.reshape(-1)[:8], lambda t: t.cpu(), lambda t: t.double()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
            o = M.diff_attention(*leaves)
        with pytest.raises(RuntimeError, match="hook"):
            o.sum().backward()
    with torch.autograd.graph.save_on_cpu():
        o = M.diff_attention(*leaves)
    for a, b in zip(torch.autograd.grad(o, leaves, dy), plain):
        assert torch.equal(a, b)


def test_empty():
    for b, tq, tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        ts = [t.requires_grad_() for t in operands(b, tq, tk, 2, 1, 64, 128, torch.bfloat16)]
        y = M.diff_attention(*ts)
        assert y.shape == (b, tq, 2, 128) and not y.any()
        y.sum().backward()
        assert all(t.grad is not None and not t.grad.any() for t in ts)


def test_autocast_changes_nothing():
    """Torch operations in 32 bits, and their backward: no 16-bit products of what autocast would cast."""
    ts = operands(2, 40, 40, 4, 2, 64, 128, torch.bfloat16)
    dy = rnd((2, 40, 4, 128), torch.bfloat16, 9)
    leaves = [t.requires_grad_() for t in ts]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = M.diff_attention(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    ref = reference(*[t.detach() for t in ts], dy)
    close(y.detach(), *ref["y"], "y")
    for name, g in zip(("dq", "dk", "dv", "dlam"), got):
        close(g, *ref[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,tq,tk,h,hk,dh,dv", [(3, 333, 1001, 6, 3, 40, 80), (1, 333, 2049, 4, 2, 64, 128), (1, 200, 4000, 2, 1, 128, 256),
                                                (32, 1, 1500, 4, 4, 64, 128), (2, 8, 5000, 8, 2, 64, 64)])
def test_results_over_a_cache_are_rounded_once(b, tq, tk, h, hk, dh, dv, dtype):
    """Chunks of new tokens and single ones: their probabilities enter the products in two parts of 16 bits, 2^-16 (bf16) and 2^-22 of
    them left, so the error is the result's own rounding in the norm; a single part's would make it 1.4 to 1.5 of that."""
    ts = operands(b, tq, tk, h, hk, dh, dv, dtype, "token")
    ref = M.diff_attention(*(t.double() for t in ts))
    norm = lambda t: (t.double() - ref).norm().item()  # noqa: E731
    assert norm(M.diff_attention(*ts)) <= 1.1 * norm(ref.to(dtype))


def test_captured_gradients_follow_their_upstreams():
    """A captured fp16 pass, whose powers of two come from its tensors: each replay gives the eager pass's bits, on another stream too,
    for upstreams and values of other sizes and other lengths, eager work between the replays."""
    ts = operands(3, 300, 300, 4, 2, 64, 128, torch.float16, "token")
    lengths, dy = ints(300, 20, 0), rnd((3, 300, 4, 128), torch.float16, 9)

    def step():
        leaves = [t.detach().requires_grad_() for t in ts]
        y = M.diff_attention(*leaves, lengths=lengths)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for up, size, n in ((1.0, 1.0, (300, 20, 0)), (2.0 ** -12, 0.5, (3, 150, 64)), (2.0 ** 10, 0.25, (0, 300, 1)), (2.0 ** -3, 1.0, (129, 128, 2))):
        lengths.copy_(ints(*n))
        dy.copy_(rnd(dy.shape, torch.float16, 9) * up)
        ts[2].copy_(rnd(ts[2].shape, torch.float16, 3) * size)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(out, want)):
            assert torch.equal(a, b), (up, k)
