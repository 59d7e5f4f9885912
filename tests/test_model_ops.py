"""model_ops on the CPU (the torch forms): values against their definitions, gradients against differences, what is refused; and
the library's exports and host-side argument checks."""
import ctypes
import math
import os
import re

import pytest
import torch
import torch.nn.functional as F

from loopback_amd import model_ops as M
from loopback_amd import rocprof_summary as RS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared():
    with open(os.path.join(ROOT, "include", "loopback_model.h")) as f:
        txt = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    return set(re.findall(r"\b(lmo_\w+)\s*\(", txt))


def test_exports_and_abi():
    assert declared() == set(M.SIGNATURES)
    with open(os.path.join(ROOT, "include", "loopback_model.h")) as f:
        txt = f.read()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", txt).group(1))  # noqa: E731
    assert M.LIB.lmo_abi_version() == M.ABI_VERSION == value("LMO_ABI_VERSION")
    assert (M.NORM_MAX_WIDTH, M.DISTILL_MAX_TOP, M.DISTILL_MAX_TAIL, M.DISTILL_SAVED) == tuple(
        value("LMO_" + n) for n in ("NORM_MAX_WIDTH", "DISTILL_MAX_TOP", "DISTILL_MAX_TAIL", "DISTILL_SAVED"))


def test_argument_checks_before_launch():
    L, p, null = M.LIB, ctypes.c_void_p(4096), None
    assert L.lmo_layer_norm_fwd(null, null, null, null, null, null, null, 0, 8, 1e-5, 1, null) == 0       # no rows
    assert L.lmo_layer_norm_fwd(p, null, null, null, null, p, null, 4, 8, 1e-5, 7, null) == -4
    for d in (0, -8, M.NORM_MAX_WIDTH + 1):
        assert L.lmo_layer_norm_fwd(p, null, null, null, null, p, null, 4, d, 1e-5, 1, null) == -2
    assert L.lmo_layer_norm_fwd(p, p, null, null, null, p, null, 4, 8, 1e-5, 1, null) == -1              # no h_out
    assert L.lmo_layer_norm_fwd(ctypes.c_void_p(4097), null, null, null, null, p, null, 4, 8, 1e-5, 1, null) == -3
    assert L.lmo_layer_norm_bwd(p, p, null, p, null, null, p, null, null, 4, 8, 1, null) == -1            # no scratch
    assert L.lmo_layer_norm_bwd(p, p, null, p, null, null, null, null, null, 4, 8, 1, null) == 0          # nothing wanted
    assert L.lmo_layer_norm_scratch(0, 8) == 0 and L.lmo_layer_norm_scratch(100, 8) >= 16

    def fwd(x=p, top=p, top_dtype=0, ids=p, lse=null, labels=null, tau=1.0, hard=0.0, saved=p, coef=p, loss=p, rows=4, vocab=10, k=2, dt=1):
        return L.lmo_distill_fwd(x, top, top_dtype, ids, 1, lse, labels, tau, hard, saved, coef, loss, rows, vocab, k, dt, null)

    assert fwd(dt=5) == -4 and fwd(top_dtype=9) == -4
    assert fwd(vocab=0) == -2 and fwd(k=0) == -2 and fwd(k=M.DISTILL_MAX_TOP + 1) == -2 and fwd(vocab=2 ** 31) == -2
    assert fwd(lse=p, vocab=M.DISTILL_MAX_TAIL + 1) == -2
    for tau in (0.0, -1.0, math.inf, math.nan):
        assert fwd(tau=tau) == -1
    for hard in (-0.1, 1.1, math.nan):
        assert fwd(hard=hard) == -1
    assert fwd(x=null) == -1 and fwd(ids=null) == -1 and fwd(loss=null) == -1 and fwd(saved=null) == -1
    assert fwd(ids=ctypes.c_void_p(4100)) == -3 and fwd(labels=ctypes.c_void_p(4100)) == -3 and fwd(saved=ctypes.c_void_p(4100)) == -3
    assert L.lmo_distill_bwd(p, p, 0, p, 1, null, 1.0, p, p, null, p, 4, 10, 2, 0, 1, null) == -1
    assert L.lmo_distill_bwd(null, null, 0, null, 1, null, 1.0, null, null, null, null, 0, 10, 2, 0, 1, null) == 0


def test_every_kernel_has_a_family():
    names = set()
    for src in M._build.MODEL_SRC:
        with open(src) as f:
            names |= set(re.findall(r"__global__[^;{]*?\bvoid\s+(k_\w+)\s*\(", f.read(), flags=re.S))
    assert {"k_layer_norm_fwd", "k_layer_norm_bwd", "k_layer_norm_sum", "k_distill_fwd", "k_distill_mean", "k_distill_bwd"} <= names
    assert all(RS.family(f"void (anonymous namespace)::{n}<float, 1>(...)") != "torch / runtime" for n in names)


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
def rnd(*shape, seed=1, dtype=torch.float64):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("affine", [(True, True), (True, False), (False, True), (False, False)])
def test_norm_values(affine, dtype):
    x, a = rnd(3, 5, 12, dtype=dtype), rnd(3, 5, 12, seed=2, dtype=dtype)
    w = rnd(12, seed=3, dtype=dtype) if affine[0] else None
    b = rnd(12, seed=4, dtype=dtype) if affine[1] else None
    half = {torch.float64: 1e-15, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    h, y = M.add_layer_norm(x, a, w, b, eps=1e-3)
    assert torch.equal(h, x + a) and y.dtype is dtype and torch.equal(y, M.layer_norm(h, w, b, eps=1e-3))
    ref = F.layer_norm(h.double(), (12,), None if w is None else w.double(), None if b is None else b.double(), 1e-3)
    assert ((y.double() - ref).abs() <= half * ref.abs() + 64 * (2.0 ** -24 if dtype is not torch.float64 else 2.0 ** -53) * 10).all()
    s, n = M.add_layer_norm(x, None, w, b, eps=1e-3)
    assert s is x and torch.equal(n, M.layer_norm(x, w, b, eps=1e-3))


def test_norm_gradients():
    x, a, w, b = (t.requires_grad_() for t in (rnd(3, 7), rnd(3, 7, seed=2), rnd(7, seed=3), rnd(7, seed=4)))
    assert torch.autograd.gradcheck(lambda *t: M.add_layer_norm(*t, eps=1e-3), (x, a, w, b))
    assert torch.autograd.gradgradcheck(lambda *t: M.layer_norm(*t, eps=1e-3), (x, w, b))
    # the node's torch form, by its formulas, against autograd's
    h, dh, dy = rnd(4, 3, 7).requires_grad_(), rnd(4, 3, 7, seed=5), rnd(4, 3, 7, seed=6)
    want = torch.autograd.grad((h, M.layer_norm(h, w, b, eps=1e-3)), (h, w, b), (dh, dy))
    got = M._norm_backward(dh, dy, h.detach(), w.detach(), 7, 1e-3)
    for g, r in zip(got, want):
        assert torch.allclose(g, r, atol=1e-12)
    assert M._norm_backward(None, dy, h.detach(), None, 0, 1e-3) == (None, None, None)


def test_norm_refusals():
    x = torch.randn(2, 8)
    for bad in (lambda: M.layer_norm(x, torch.ones(7)), lambda: M.layer_norm(x, None, torch.ones(2, 8)), lambda: M.layer_norm(x.long()),
                lambda: M.layer_norm(torch.ones(())), lambda: M.add_layer_norm(x, x[:1]), lambda: M.add_layer_norm(x, torch.ones(8))):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------
def test_distill_is_the_divergence():
    """Every class named: the divergence of two distributions as torch forms it."""
    x, z = rnd(6, 11), rnd(6, 11, seed=2)
    ids = torch.stack([torch.randperm(11, generator=torch.Generator().manual_seed(i)) for i in range(6)])
    for tau in (1.0, 3.0):
        want = tau * tau * F.kl_div(F.log_softmax(x / tau, -1), F.log_softmax(z / tau, -1), reduction="batchmean", log_target=True)
        got = M.distill_loss(x, z.gather(1, ids), ids, temperature=tau)
        assert torch.allclose(got, want, atol=1e-12)
        lse = torch.logsumexp(z / tau, -1)
        assert torch.allclose(M.distill_loss(x, z.gather(1, ids), ids, temperature=tau, teacher_lse=lse), want, atol=1e-12)


def test_distill_labels_and_rest():
    """The rest as one event: two distributions of k + 1 events; the labels' cross entropy as torch forms it."""
    x, z = rnd(5, 40), rnd(5, 40, seed=2)
    top, ids = z.topk(6, -1)
    p, q = torch.softmax(z, -1), torch.softmax(x, -1)
    P = torch.cat((p.gather(1, ids), 1 - p.gather(1, ids).sum(-1, keepdim=True)), -1)
    Q = torch.cat((q.gather(1, ids), 1 - q.gather(1, ids).sum(-1, keepdim=True)), -1)
    kl = (P * (P.log() - Q.log())).sum(-1).mean()
    got = M.distill_loss(x, top, ids, teacher_lse=torch.logsumexp(z, -1))
    assert torch.allclose(got, kl, atol=1e-12)
    labels = torch.tensor([3, -100, 39, 0, 7])
    both = M.distill_loss(x, top, ids.int(), teacher_lse=torch.logsumexp(z, -1), labels=labels, hard_weight=0.3)
    assert torch.allclose(both, 0.7 * kl + 0.3 * F.cross_entropy(x, labels), atol=1e-12)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("hard", [0.0, 0.4])
def test_distill_gradients(tail, hard):
    x = rnd(5, 13).requires_grad_()
    ids = torch.tensor([[1, 2, 5], [12, 0, -1], [-1, -1, -1], [4, 4, 7], [3, 8, 9]])
    top = rnd(5, 3, seed=2)
    top[1, 2] = math.nan
    labels = torch.tensor([0, 12, 3, -100, 5]) if hard else None
    lse = torch.logsumexp(torch.where(ids >= 0, top / 2.0, -math.inf), -1) + 0.3 if tail else None
    f = lambda x: M.distill_loss(x, top, ids, temperature=2.0, teacher_lse=lse, labels=labels, hard_weight=hard)  # noqa: E731
    assert torch.autograd.gradcheck(f, x) and torch.autograd.gradgradcheck(f, x)
    want, = torch.autograd.grad(f(x), x)
    got, = M._distill_backward(torch.ones(()), x.detach(), top, ids, lse, labels, 2.0, hard)
    assert torch.allclose(got, want, atol=1e-12)
    if not hard:
        assert not want[2].any()


def test_distill_no_rows_and_one():
    assert M.distill_loss(torch.empty(0, 5), torch.empty(0, 2), torch.empty(0, 2, dtype=torch.int64)).item() == 0.0
    x, top, ids = rnd(9), rnd(3, seed=2), torch.tensor([1, 4, 8])
    assert torch.equal(M.distill_loss(x, top, ids), M.distill_loss(x[None], top[None], ids[None]))


def test_distill_refusals():
    x, top, ids = torch.randn(4, 9), torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    labels = torch.zeros(4, dtype=torch.int64)
    for bad in (lambda: M.distill_loss(x.long(), top, ids), lambda: M.distill_loss(x, top[:3], ids[:3]), lambda: M.distill_loss(x, top, ids[:, :2]),
                lambda: M.distill_loss(x, top, ids.float()), lambda: M.distill_loss(x, top.long(), ids),
                lambda: M.distill_loss(x, top[:, :0], ids[:, :0]), lambda: M.distill_loss(x, top[0], ids[0]),
                lambda: M.distill_loss(x, top, ids, temperature=0.0), lambda: M.distill_loss(x, top, ids, temperature=math.nan),
                lambda: M.distill_loss(x, top, ids, hard_weight=0.5), lambda: M.distill_loss(x, top, ids, labels=labels, hard_weight=1.5),
                lambda: M.distill_loss(x, top, ids, labels=labels[:3], hard_weight=0.5),
                lambda: M.distill_loss(x, top, ids, labels=labels.int(), hard_weight=0.5),
                lambda: M.distill_loss(x, top, ids, teacher_lse=torch.ones(3)), lambda: M.distill_loss(x, top, ids, teacher_lse=labels),
                lambda: M.distill_loss(x[:, :0], top, ids), lambda: M.distill_loss(x, top.to("meta"), ids)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------------------------------------------
# differential attention
# ---------------------------------------------------------------------------------------------------------------
def attn(b=2, tq=5, tk=5, h=4, g=2, dh=4, dv=6, lam=(4,)):
    return rnd(b, tq, 2 * h, dh), rnd(b, tk, 2 * g, dh, seed=2), rnd(b, tk, g, dv, seed=3), rnd(*lam, seed=4)


def test_attention_is_the_difference_of_two():
    """Against torch's attention over each map, its heads of keys repeated."""
    q, k, v, lam = attn()
    maps = [F.scaled_dot_product_attention(q[:, :, m::2].transpose(1, 2), k[:, :, m::2].transpose(1, 2).repeat_interleave(2, 1),
                                           v.transpose(1, 2).repeat_interleave(2, 1), is_causal=True) for m in (0, 1)]
    want = (maps[0] - lam.view(1, 4, 1, 1) * maps[1]).transpose(1, 2)
    assert torch.allclose(M.diff_attention(q, k, v, lam), want, atol=1e-12)
    assert torch.allclose(M.diff_attention(q, k, v, lam.expand(2, 5, 4)), want, atol=1e-12)
    one = M.diff_attention(q, k, v, torch.tensor(0.25, dtype=torch.float64), causal=False, scale=0.7)
    maps = [F.scaled_dot_product_attention(q[:, :, m::2].transpose(1, 2), k[:, :, m::2].transpose(1, 2).repeat_interleave(2, 1),
                                           v.transpose(1, 2).repeat_interleave(2, 1), scale=0.7) for m in (0, 1)]
    assert torch.allclose(one, (maps[0] - 0.25 * maps[1]).transpose(1, 2), atol=1e-12)


def test_attention_masks():
    """A token at a time over a growing cache gives what the whole sequence gives; rows that see nothing are zeros; what is past
    the lengths is not read into anything."""
    q, k, v, lam = attn()
    whole = M.diff_attention(q, k, v, lam)
    for i in range(5):
        n = torch.tensor([i + 1, i + 1])
        cache = k.clone(), v.clone()
        for c in cache:
            c[:, i + 1:] = math.nan
        assert torch.allclose(M.diff_attention(q[:, i:i + 1], *cache, lam, lengths=n, starts=n.int() - 1), whole[:, i:i + 1], atol=1e-12)
    assert torch.allclose(M.diff_attention(q[:, 3:], k, v, lam), whole[:, 3:], atol=1e-12)
    more = M.diff_attention(q, k[:, :2], v[:, :2], lam)          # more queries than keys: the first three see none
    assert not more[:, :3].any() and more[:, 3:].ne(0).all()
    none = M.diff_attention(q, k, v, lam, lengths=torch.tensor([0, 5]))
    assert not none[0].any() and torch.equal(none[1], whole[1])
    for tq, tk in ((0, 3), (3, 0)):
        ts = [t.requires_grad_() for t in attn(tq=tq, tk=tk)]
        y = M.diff_attention(*ts)
        assert y.shape == (2, tq, 4, 6) and not y.any()
        y.sum().backward()


@pytest.mark.parametrize("lam", [(), (4,), (2, 3, 4)])
def test_attention_gradients(lam):
    ts = [t.requires_grad_() for t in attn(tq=3, lam=lam)]
    how = {"lengths": torch.tensor([5, 2]), "starts": torch.tensor([2, -2])}
    f = lambda *a: M.diff_attention(*a, **how)  # noqa: E731
    assert torch.autograd.gradcheck(f, ts)
    if lam == (4,):
        assert torch.autograd.gradgradcheck(f, ts)
    dy = rnd(2, 3, 4, 6, seed=9)
    want = torch.autograd.grad(f(*ts), ts, dy)
    got = M._diff_backward(dy, *(t.detach() for t in ts), how["lengths"], how["starts"], 1, 15, 0.5)
    for a, b in zip(got, want):
        assert a.shape == b.shape and torch.allclose(a, b, atol=1e-12)


def test_attention_refusals():
    q, k, v, lam = attn()
    n = torch.tensor([1, 2])
    for bad in (lambda: M.diff_attention(q[0], k, v, lam), lambda: M.diff_attention(q.long(), k, v, lam), lambda: M.diff_attention(q, k[:1], v, lam),
                lambda: M.diff_attention(q, k[:, :4], v, lam), lambda: M.diff_attention(q, k[..., :3], v, lam),
                lambda: M.diff_attention(q[:, :, :7], k, v, lam), lambda: M.diff_attention(q[:, :, :6], k, v, lam[:3]),
                lambda: M.diff_attention(q, k[:, :, :3], v, lam), lambda: M.diff_attention(q, k, v, lam[:3]),
                lambda: M.diff_attention(q, k, v, 0.5), lambda: M.diff_attention(q, k, v, lam.long()),
                lambda: M.diff_attention(q, k, v, lam.view(1, 4)), lambda: M.diff_attention(q, k, v, lam, scale=0.0),
                lambda: M.diff_attention(q, k, v, lam, scale=-1.0), lambda: M.diff_attention(q, k, v, lam, scale=math.inf),
                lambda: M.diff_attention(q, k, v, lam, lengths=n.float()), lambda: M.diff_attention(q, k, v, lam, lengths=n[:1]),
                lambda: M.diff_attention(q, k, v, lam, starts=n.view(1, 2)), lambda: M.diff_attention(q, k, v, lam, starts=n.to("meta")),
                lambda: M.diff_attention(q, k.to("meta"), v, lam)):
        with pytest.raises(ValueError):
            bad()


class Strides(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("b", ctypes.c_int64), ("t", ctypes.c_int64), ("h", ctypes.c_int64)]


class Shape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("b", "tq", "tk", "h", "hk", "dh", "dv")] + [("causal", ctypes.c_int), ("scale", ctypes.c_float)]


def test_attention_argument_checks_before_launch():
    L, p, ref = M.LIB, 4096, ctypes.byref

    def fwd(dtype=1, q=(p, 512, 512, 64), lam=p, out=p, second=None, lse=None, scratch=p, **s):
        sizes = {"b": 1, "tq": 8, "tk": 8, "h": 2, "hk": 1, "dh": 64, "dv": 128, "causal": 1, "scale": 0.125, **s}
        k, v, lm = Strides(p, 1024, 128, 64), Strides(p, 1024, 128, 128), Strides(lam, 0, 0, 0)
        return L.lmo_diff_attn_fwd(ref(Strides(*q)), ref(k), ref(v), ref(lm), 1, None, None, out, second, lse, scratch, ref(Shape(**sizes)),
                                   dtype, None)

    assert fwd(b=0) == 0 and fwd(tq=0) == 0
    assert fwd(dtype=0) == -4 and fwd(dtype=3) == -4
    for s in ({"dh": 0}, {"dh": 12}, {"dh": 136}, {"dv": 264}, {"dv": 4}):
        assert fwd(**s) == -2, s
    for s in ({"tk": 0}, {"hk": 0}, {"h": 3, "hk": 2}, {"h": 1, "hk": 2}, {"scale": 0.0}, {"scale": math.inf}, {"scale": math.nan}, {"tq": 2 ** 30},
              {"tk": 2 ** 30}, {"b": 2 ** 23}, {"b": -1}, {"lam": None}, {"out": None}, {"second": p}, {"lse": p}, {"q": (None, 512, 512, 64)}):
        assert fwd(**s) == -1, s
    for q in ((p + 8, 512, 512, 64), (p, 512, 516, 64), (p, 4, 512, 64), (p, 512, 512, 60)):
        assert fwd(q=q) == -3
    assert fwd(q=(p, 512, 2 ** 24, 64)) == -2 and fwd(q=(p, -512, 512, 64)) == -2
    assert fwd(out=p + 2) == -3
    few = Shape(1, 1, 100000, 2, 1, 64, 128, 1, 0.125)
    assert L.lmo_diff_attn_scratch(ref(few), 0) > 0 and L.lmo_diff_attn_scratch(ref(Shape(8, 4096, 4096, 2, 1, 64, 128, 1, 0.125)), 1) == 0
    assert fwd(tq=1, tk=100000, scratch=None) == -1
    s = Strides(p, 1024, 128, 64)
    assert L.lmo_diff_attn_bwd(ref(s), ref(s), ref(s), ref(s), 1, None, None, p, p, p, p, p, p, None, None, 0, p, ref(few), 1, None) == -1
    assert L.lmo_diff_attn_bwd(ref(s), ref(s), ref(s), ref(s), 1, None, None, p, p, p, p, p, p, p, p, 7, p, ref(few), 1, None) == -1


def test_attention_backward_refuses_wide_rows():
    """Rows of dy whose distances of 32 are past 32 bits of bytes."""
    p, ref = 4096, ctypes.byref
    s = Strides(p, 2 ** 23, 2 ** 23, 8)
    for h in (2 ** 18 + 1, 2 ** 19):
        assert M.LIB.lmo_diff_attn_bwd(ref(s), ref(s), ref(s), ref(s), 1, None, None, p, p, p, p, p, p, p, p, 0, p,
                                       ref(Shape(1, 20, 20, h, 1, 8, 256, 1, 0.125)), 1, None) == -2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autocast_changes_nothing(dtype):
    """The operators compute in 32 bits and keep their input's type under autocast, whose products would be of 16."""
    x, w, b = (rnd(*s, seed=i, dtype=dtype).requires_grad_() for i, s in enumerate(((3, 12), (12,), (12,))))
    top, ids = rnd(3, 4, seed=5, dtype=dtype), torch.tensor([[0, 3, 7, 9]] * 3)
    q, k, v, lam = (t.to(dtype).requires_grad_() for t in attn(dh=8))
    calls = [(lambda: M.add_layer_norm(x, x * 0.5, w, b)[1], (x, w, b)), (lambda: M.diff_attention(q, k, v, lam), (q, k, v, lam)),
             (lambda: M.distill_loss(x, top, ids, teacher_lse=torch.logsumexp(top.float(), -1) + 0.2, temperature=2.0), (x,))]
    for call, leaves in calls:
        want = call()
        with torch.autocast("cpu", dtype=torch.bfloat16):
            got = call()
        assert got.dtype is want.dtype and torch.equal(got, want)
        for a, r in zip(torch.autograd.grad(got.sum(), leaves), torch.autograd.grad(want.sum(), leaves)):
            assert torch.equal(a, r)
    dy = rnd(2, 5, 4, 6, seed=9, dtype=dtype)
    leaves = [t.detach() for t in (q, k, v, lam)]
    want = M._diff_backward(dy, *leaves, None, None, 1, 15, 8 ** -0.5)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = M._diff_backward(dy, *leaves, None, None, 1, 15, 8 ** -0.5)
    assert all(torch.equal(a, r) for a, r in zip(got, want))
