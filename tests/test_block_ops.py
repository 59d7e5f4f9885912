"""block_ops on the CPU: the library and its refusals, the generator's published test vectors, the torch forms against the
formulas in fp64 and against differences, the checks of arguments."""
import os
import re

import pytest
import torch

from loopback_amd import block_ops as ops
from loopback_amd import rocprof_summary as RS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rnd(shape, seed, dtype=torch.float64):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def test_library():
    """The library exports what include/loopback_block.h declares and the binding's table is the header's."""
    with open(os.path.join(ROOT, "include", "loopback_block.h")) as f:
        text = f.read()
    names = set(re.findall(r"\b(lbk_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(ops.SIGNATURES) and all(hasattr(ops.LIB, n) for n in names)
    define = lambda n: int(re.search(rf"#define {n} (\d+)", text).group(1))
    assert define("LBK_ABI_VERSION") == ops.ABI_VERSION and define("LBK_JOIN_MAX_WIDTH") == ops.JOIN_MAX_WIDTH
    assert define("LBK_FEW_TOKENS") == ops.FEW_TOKENS


def test_row_kernels_refuse():
    """Calls whose operands the kernels do not take are refused before any launch; empty ones return at once."""
    L, p, null = ops.LIB, 4096, None
    drop = lambda x=p, rng=p, d=16, rows=4, drop=100, dt=1: L.lbk_dropout(x, rng, 0, drop, p, rows, d, dt, null)
    assert drop(dt=3) == -4 and drop(rows=-1) == -1 and drop(d=0) == -1 and drop(drop=65537) == -1 and drop(drop=-1) == -1
    assert drop(rows=2 ** 31) == -2 and drop(x=null) == -1 and drop(rng=null) == -1 and drop(x=4097) == -3
    assert drop(rng=4100) == -3 and drop(rows=0) == 0 and drop(x=4098, dt=0) == -3
    fwd = lambda x=p, n=p, gate=null, gr=1, pre=p, rng=null, dr=0, rows=4, d=64, dt=1, h=p: L.lbk_join_fwd(
        x, p, p, gate, gr, pre, rng, 0, dr, 1.0, 1e-6, h, n, p, p, rows, d, dt, null)
    assert fwd(dt=7) == -4 and fwd(d=0) == -1 and fwd(rows=-1) == -1 and fwd(d=8193) == -2 and fwd(rows=2 ** 31) == -2
    assert fwd(x=null) == -1 and fwd(n=null) == -1 and fwd(h=null) == -1 and fwd(gate=p, gr=0) == -1 and fwd(dr=5) == -1
    assert fwd(x=4097) == -3 and fwd(rng=4100, dr=5) == -3 and fwd(rows=0, x=null) == 0
    bwd = lambda dh=p, dn=p, h=p, y=p, pre=p, post=p, rpo=p, gate=null, dgate=null, s=p, rows=4: L.lbk_join_bwd(
        dh, dn, h, y, post, gate, 1, pre, rpo, p, null, 0, 0, 1.0, p, p, p, dgate, p, s, rows, 64, 1, null)
    assert bwd(dh=null, dn=null) == -1 and bwd(h=null) == -1 and bwd(y=null) == -1 and bwd(pre=null) == -1
    assert bwd(rpo=null) == -1 and bwd(post=null) == -1 and bwd(dgate=p) == -1 and bwd(s=null) == -1 and bwd(rows=0) == 0
    assert bwd(dn=null) == -1 and bwd(dh=4097) == -3 and bwd(s=4098) == -3   # dpre without dn
    assert L.lbk_join_scratch(0, 64, 1) == 0 and L.lbk_join_scratch(4, 9000, 1) == 0
    assert L.lbk_join_scratch(1, 64, 1) == 4 * 64


def test_products_refuse():
    L, p, null = ops.LIB, 4096, None
    up = lambda x=p, w=p, act=p, saved=p, t=100, d=8, n=8, a=0, dt=1, ldx=8, ldw=8, ld=8: L.lbk_ffn_gate_up(
        x, ldx, w, ldw, act, ld, saved, t, d, n, a, dt, null)
    assert up(dt=0) == -4 and up(dt=3) == -4 and up(t=-1) == -1 and up(d=0) == -1 and up(n=0) == -1 and up(a=2) == -1
    assert up(x=null) == -1 and up(w=null) == -1 and up(act=null) == -1 and up(x=4097) == -3 and up(saved=4098) == -3
    assert up(t=2 ** 31) == -2 and up(d=2 ** 31) == -2 and up(n=2 ** 31, ld=2 ** 31) == -2 and up(t=0, x=null) == 0
    assert up(x=4098) == -3 and up(ldx=12) == -3 and up(ldw=7) == -2 and up(ldw=2 ** 23) == -2 and up(ld=7) == -1
    assert up(t=4, saved=null, ldx=7) == -2 and up(t=4, x=4097, saved=null) == -3
    dn = lambda dy=p, w=p, saved=p, out=p, t=4, dt=2, lw=8, lo=16: L.lbk_ffn_dgate_up(dy, 8, w, lw, saved, out, lo, t, 8, 8, dt, null)
    assert dn(dt=0) == -4 and dn(dy=null) == -1 and dn(w=null) == -1 and dn(saved=null) == -1 and dn(out=null) == -1
    assert dn(saved=4098) == -3 and dn(out=4097) == -3 and dn(t=0) == 0 and dn(lw=9) == -3 and dn(lo=15) == -1 and dn(w=4098) == -3
    for fn in (L.lbk_linear_fwd, L.lbk_linear_dx):
        call = lambda x=p, w=p, y=p, t=100, k=8, ld=8, dt=1, s=null: fn(x, ld, w, 8, y, 8, s, t, k, 8, dt, null)
        assert call(dt=0) == -4 and call(x=null) == -1 and call(w=null) == -1 and call(y=null) == -1 and call(y=4097) == -3
        assert call(k=0) == -1 and call(t=0) == 0 and call(t=-1) == -1 and call(ld=12) == -3 and call(x=4098) == -3 and call(s=4100) == -3
    assert L.lbk_linear_fwd(p, 7, p, 8, p, 8, null, 4, 8, 8, 1, null) == -2
    dw = lambda dy=p, s=p, out=p, t=4: L.lbk_linear_dw(dy, 8, p, 8, s, out, t, 8, 8, 1, null)
    assert dw(dy=null) == -1 and dw(out=null) == -1 and dw(s=null, t=1 << 20) == -1 and dw(s=4100) == -3 and dw(t=-1) == -1
    assert dw(t=0) == -1
    pad = lambda x=p, out=p, rows=4, cols=7, ld=8, dt=1: L.lbk_pad_rows(x, rows, cols, ld, out, dt, null)
    assert pad(x=null) == -1 and pad(out=null) == -1 and pad(rows=0) == 0 and pad(ld=6) == -2 and pad(ld=9) == -3 and pad(dt=0) == -4
    assert pad(out=4098) == -3 and pad(x=4097) == -3
    assert L.lbk_linear_scratch(0, 8, 8) == 0 and L.lbk_linear_scratch(8192, 8192, 8192) == 0
    assert L.lbk_linear_scratch(8, 9, 1 << 20) % (8 * 9) == 0 and L.lbk_linear_scratch(8, 9, 1 << 20) > 72
    assert L.lbk_ffn_saved_bytes(33, 1) == 2 * 6144


def test_ffn_form():
    """The torch form: its values by their formula and its gradients against differences, in fp64."""
    args = [rnd((3, 5), 1).requires_grad_(), rnd((8, 5), 2).requires_grad_(), rnd((6, 4), 3).requires_grad_()]
    for act in ("silu", "gelu"):
        assert torch.autograd.gradcheck(lambda *a: ops.gated_ffn(*a, activation=act), args)
        g, u = (args[0] @ args[1].t()).chunk(2, -1)
        q = g if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)
        assert torch.allclose(ops.gated_ffn(*args, activation=act), (g * torch.sigmoid(q) * u) @ args[2].t(), atol=1e-12)
    assert ops.gated_ffn(args[0][:0], *args[1:]).shape == (0, 6)


def test_generator_vectors():
    """Philox-4x32-10's published known answers, as the halves of its words: counters and keys of zeros and of ones."""
    def bits(seed, step, site, row, block):
        lo, hi = torch.zeros(8, dtype=torch.int64), torch.full((8,), 65537)
        rng = torch.tensor([seed, step])
        while (hi - lo > 1).any():   # the largest `drop` at which an element is kept is its 16 bits
            mid = (lo + hi) // 2
            keep = torch.stack([ops._mask(int(m), rng, site, row + 1, 8 * block + 8)[row, 8 * block + k] for k, m in enumerate(mid)])
            lo, hi = torch.where(keep, mid, lo), torch.where(keep, hi, mid)
        return [int(a) + (int(b) << 16) for a, b in zip(lo[::2], lo[1::2])]

    assert bits(0, 0, 0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    # counter (block, row, site, step) and key halves beyond 2^31: signs of 64-bit products
    import numpy as np

    def numpy_words(c, k):
        u, m = np.uint64, np.uint64(0xFFFFFFFF)
        c, k = [u(v) for v in c], [u(v) for v in k]
        for _ in range(10):
            a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
            c = [(b >> u(32)) ^ c[1] ^ k[0], b & m, (a >> u(32)) ^ c[3] ^ k[1], a & m]
            k = [(k[0] + u(0x9E3779B9)) & m, (k[1] + u(0xBB67AE85)) & m]
        return [int(v) for v in c]

    assert numpy_words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert numpy_words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    for seed, step, site, row, block in ((-1, 2 ** 32 - 1, 2 ** 32 - 1, 5, 3), (-2 ** 63, 7, 2 ** 31, 0, 1),
                                         (0x299F31D0A4093822, 0x03707344, 0x13198A2E, 2, 2)):
        assert bits(seed, step, site, row, block) == numpy_words([block, row, site, step & 0xFFFFFFFF],
                                                                 [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF])


def test_dropout_form():
    """The share that is kept, its scale, the mask's independence of type and strides, and of other places and steps."""
    x, rng = torch.ones(300, 1001), torch.tensor([5, 1])
    y = ops.dropout(x, 0.1, rng, site=2)
    keep = ops.keep_mask((300, 1001), 0.1, rng, site=2)
    s = 65536 / (65536 - round(65536 * 0.1))
    assert torch.equal(y, keep * torch.tensor(s)) and abs(keep.double().mean() - 1 / s) < 4 * (0.09 / 300300) ** 0.5
    assert torch.equal(ops.dropout(x.t().contiguous().t().double(), 0.1, rng, site=2), keep.double() * s)
    for other in (ops.keep_mask((300, 1001), 0.1, torch.tensor([5, 2]), 2), ops.keep_mask((300, 1001), 0.1, rng, 3),
                  ops.keep_mask((300, 1001), 0.1, torch.tensor([6, 1]), 2)):
        agree = (other == keep).double().mean()
        assert abs(agree - 0.82) < 4 * (0.82 * 0.18 / 300300) ** 0.5
    assert ops.dropout(x, 0.0, None) is x and not ops.dropout(x, 1.0, rng).any()
    assert torch.equal(ops.dropout(x.bfloat16(), 0.1, rng, site=2), y.bfloat16())
    assert ops.dropout(torch.ones(()), 0.5, rng).shape == () and ops.dropout(torch.ones(0, 4), 0.5, rng).shape == (0, 4)


@pytest.mark.parametrize("gate", [None, (6,), (2, 1, 6), (2, 3, 6)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("pre", [True, False])
def test_join_form_against_differences(gate, post, pre):
    """The torch form's gradients against central differences in fp64."""
    rng = torch.tensor([3, 4])
    args = [rnd((2, 3, 6), 1), rnd((2, 3, 6), 2), *([rnd((6,), 3)] if post else []), *([rnd(gate, 4)] if gate else []),
            *([rnd((6,), 5)] if pre else [])]

    def fn(x, y, *rest):
        it = iter(rest)
        h, n = ops.block_join(x, y, post_weight=next(it) if post else None, gate=next(it) if gate else None, scale=0.6,
                              dropout=0.3, rng=rng, site=1, pre_weight=next(it) if pre else None)
        return (h,) if n is None else (h, n)

    assert torch.autograd.gradcheck(fn, [a.requires_grad_() for a in args])


def test_join_form_values():
    x, y, w, g, v = rnd((4, 10), 1), rnd((4, 10), 2), rnd((10,), 3), rnd((4, 10), 4), rnd((10,), 5)
    h, n = ops.block_join(x, y, post_weight=w, gate=g, scale=-2.0, pre_weight=v, eps=0.1)
    z = torch.nn.functional.rms_norm(y, (10,), w, 0.1) * g * -2.0
    assert torch.allclose(h, x + z, atol=1e-12) and torch.allclose(n, torch.nn.functional.rms_norm(x + z, (10,), v, 0.1), atol=1e-12)
    h, n = ops.block_join(x.bfloat16(), y.bfloat16())
    assert n is None and torch.equal(h, (x.bfloat16().float() + y.bfloat16().float()).bfloat16())


def test_arguments():
    x, w, rng = torch.zeros(2, 3, 8), torch.ones(8), torch.tensor([1, 2])
    for bad in (lambda: ops.dropout(x, 1.5, rng), lambda: ops.dropout(x, -0.1, rng), lambda: ops.dropout(x, float("nan"), rng),
                lambda: ops.dropout(x, 0.5, None), lambda: ops.dropout(x, 0.5, rng.int()), lambda: ops.dropout(x, 0.5, rng[:1]),
                lambda: ops.dropout(x, 0.5, rng, site=-1), lambda: ops.dropout(x, 0.5, rng, site=2 ** 32),
                lambda: ops.dropout(x.long(), 0.5, rng), lambda: ops.block_join(x, x[:1]), lambda: ops.block_join(x, x.view(6, 8)),
                lambda: ops.block_join(x, x, post_weight=w[:4]), lambda: ops.block_join(x, x, pre_weight=w.view(1, 8)),
                lambda: ops.block_join(x, x, gate=torch.ones(3, 8)), lambda: ops.block_join(x, x, gate=torch.ones(1, 3, 8)),
                lambda: ops.block_join(x, x, gate=torch.ones(2, 3, 1)), lambda: ops.block_join(x, x, gate=torch.ones(())),
                lambda: ops.block_join(x, x, dropout=0.1),
                lambda: ops.gated_ffn(x, torch.ones(4, 8), torch.ones(8, 3)), lambda: ops.gated_ffn(x, torch.ones(4, 7), torch.ones(8, 2)),
                lambda: ops.gated_ffn(x, torch.ones(4, 8), torch.ones(8, 2), "relu"), lambda: ops.gated_ffn(x, w, w)):
        with pytest.raises(ValueError):
            bad()
    assert [ops._gate_rows(torch.empty(s), x) for s in ((8,), (1, 1, 8), (2, 1, 8), (2, 3, 8))] == [6, 6, 3, 1]


def test_every_kernel_has_a_family():
    names = set()
    for src in ("loopback_block.hip", "loopback_ffn.hip"):
        with open(os.path.join(ROOT, "loopback_amd", "csrc", src)) as f:
            names |= set(re.findall(r"__global__[^;{]*?\bvoid\s+(k_\w+)\s*\(", f.read(), flags=re.S))
    assert {"k_dropout", "k_join_fwd", "k_join_bwd", "k_join_sum", "k_product", "k_split_sum", "k_few_tokens", "k_pad_rows"} <= names
    assert all(RS.family(f"void (anonymous namespace)::{n}<float, 1>(...)") != "torch / runtime" for n in names)


@pytest.mark.parametrize("gate", [None, (6,), (2, 1, 6), (2, 3, 6)])
@pytest.mark.parametrize("post,pre,drop", [(True, True, 20000), (False, True, 0), (True, False, 20000), (False, False, 0)])
def test_join_backward_form(gate, post, pre, drop):
    """The backward that a node calls where it has to be torch operations: its gradients are autograd's of the forward's torch
    form, also with one upstream gradient missing, in fp64, and those that are not asked for are not formed."""
    rng = torch.tensor([3, 4])
    x, y, p, g, w = (None if s is None else rnd(s, k).requires_grad_() for k, s in enumerate(
        ((2, 3, 6), (2, 3, 6), (6,) if post else None, gate, (6,) if pre else None)))
    h, n = ops._join_torch(x, y, p, g, w, rng, 1, drop, 0.6, 1e-3)
    dh, dn = rnd((2, 3, 6), 8), rnd((2, 3, 6), 9) if pre else None
    ins = [t for t in (x, y, p, g, w) if t is not None]
    for a, b in ((dh, dn), (None, dn), (dh, None)):
        outs = [(o, u) for o, u in ((h, a), (n, b)) if u is not None]
        if not outs:
            continue
        ref = iter(torch.autograd.grad([o for o, _ in outs], ins, [u for _, u in outs], retain_graph=True, allow_unused=True))
        ref = [None if t is None else next(ref) for t in (x, y, p, g, w)]
        need = 3 + 4 * post + 8 * bool(gate) + 16 * (pre and b is not None)
        got = ops._join_backward(a, b, x, y, p, g, w, rng, 1, drop, need, 0.6, 1e-3)
        for k, (u, v) in enumerate(zip(got, ref)):
            assert (u is not None) == bool(need >> k & 1) and (u is None or torch.allclose(u, v, atol=1e-12)), k
    none = ops._join_backward(dh, dn, x, y, p, g, w, rng, 1, drop, 0, 0.6, 1e-3)
    assert none == (None,) * 5


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_ffn_backward_form(act):
    """The backward that a node calls where it has to be torch operations: autograd's gradients of the torch form, in fp64."""
    x, g, d, dy = rnd((2, 3, 5), 1).requires_grad_(), rnd((8, 5), 2).requires_grad_(), rnd((6, 4), 3).requires_grad_(), rnd((2, 3, 6), 4)
    code = ops.ACTIVATIONS[act]
    ref = torch.autograd.grad(ops._ffn_torch(x, g, d, code), (x, g, d), dy)
    for need in (7, 1, 2, 4, 0):
        for k, (a, b) in enumerate(zip(ops._ffn_backward(dy, x, g, d, code, need), ref)):
            assert (a is not None) == bool(need >> k & 1) and (a is None or torch.allclose(a, b, atol=1e-12))


def test_watched_calls_are_torch_operations():
    """torch.compile in one graph, make_fx and fake tensors see torch operations, with the eager results."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    rng = torch.tensor([3, 4])
    x, w, gu, d = rnd((2, 3, 8), 1, torch.float32), rnd((8,), 2, torch.float32), rnd((12, 8), 3, torch.float32), rnd((8, 6), 4, torch.float32)

    def fn(x):
        h, n = ops.block_join(x, ops.gated_ffn(x, gu, d), post_weight=w, gate=w, scale=0.5, dropout=0.3, rng=rng, site=2, pre_weight=w)
        return h + ops.dropout(n, 0.2, rng, site=3)

    ref = fn(x)
    torch._dynamo.reset()
    assert torch.allclose(torch.compile(fn, backend="eager", fullgraph=True)(x), ref, atol=1e-6)
    assert torch.allclose(make_fx(fn)(rnd((2, 3, 8), 7, torch.float32))(x), ref, atol=1e-6)
    with FakeTensorMode():
        y = torch.empty(2, 3, 64, device="cuda", dtype=torch.bfloat16)
        v, r = torch.empty(64, device="cuda", dtype=torch.bfloat16), torch.empty(2, device="cuda", dtype=torch.int64)
        h, n = ops.block_join(y, y, post_weight=v, pre_weight=v, dropout=0.1, rng=r)
        assert h.shape == n.shape == y.shape and ops.dropout(y, 0.1, r).device == y.device
        assert ops.gated_ffn(y, torch.empty(96, 64, device="cuda", dtype=torch.bfloat16),
                             torch.empty(32, 48, device="cuda", dtype=torch.bfloat16)).shape == (2, 3, 32)
    assert torch.func.vmap(fn)(x[None]).shape == (1, 2, 3, 8)


@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_join_backward_is_at_the_unrounded_sum(dtype, half):
    """The torch form's gradients in 16 bits, of one row, where no sum hides a rounding: one rounding of the exact ones each (and
    fp32 round-off, 1e-5 of their size), the weight's of the norm after the rounded sum among them."""
    g = torch.Generator().manual_seed(5)
    x, y, post, pre, dh, dn = (torch.randn(s, generator=g).to(dtype) for s in ((1, 64), (1, 64), (64,), (64,), (1, 64), (1, 64)))
    got = ops._join_backward(dh, dn, x, y, post, None, pre, None, 0, 0, 31 - 8, 0.7, 1e-6)
    leaves = [t.double().requires_grad_() for t in (x, y, post, pre)]
    h, n = ops._join_torch(leaves[0], leaves[1], leaves[2], None, leaves[3], None, 0, 0, 0.7, 1e-6)
    ref = torch.autograd.grad((h, n), leaves, (dh.double(), dn.double()))
    for a, b in zip((got[0], got[1], got[2], got[4]), ref):
        assert ((a.double() - b).abs() <= half * b.abs() + 1e-5 * b.pow(2).mean().sqrt()).all()
