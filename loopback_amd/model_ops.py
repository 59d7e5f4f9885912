"""Operators of a language model's step around its products, on the HIP kernels of libloopback_model.so
(include/loopback_model.h), beside the norm, the attention and the loss of lm_ops:

  * `layer_norm(x, weight, bias)` and `add_layer_norm(x, add, weight, bias)`, the latter with the residual's add before the
    norm and, in its backward, the gradient that comes back along the residual stream;
  * `diff_attention(q, k, v, lam)`: differential attention, (softmax(q1 k1^T) - lam softmax(q2 k2^T)) v, for whole sequences, chunks
    of new tokens and single ones (bf16 and fp16);
  * `distill_loss(logits, top_logits, top_ids, ...)`: the divergence of a model's logits from a teacher's highest ones, with
    the labels' cross entropy mixed in where they are given.

The row kernels take plain fp32, bf16 and fp16 tensors of the current GPU where nothing has to see torch operations (lm_ops.native
says what does); everything else -- the CPU, other types, mixed types, autocast, tracers, transforms -- runs the torch form of the
same operator. A backward that is itself differentiated, or watched, runs the torch form too. Tensors of any strides are taken.
Saved tensors that a hook gives back with another shape, type or device are refused.
"""
from __future__ import annotations

import contextlib
import ctypes
import os

import torch

from . import _host as H      # the launch path (csrc/host.cpp), bound below to the library
from . import build as _build
from .block_ops import _plain_rows, _records, _upcast
from .lm_ops import _stream, native

ABI_VERSION = 1
NORM_MAX_WIDTH = 16384
DISTILL_MAX_TOP, DISTILL_MAX_TAIL, DISTILL_SAVED = 1024, 524288, 12
MAX_ROWS = 2 ** 31 - 1
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_p, _i64, _i32, _f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
# name -> (restype, argtypes); one line per declaration of include/loopback_model.h
SIGNATURES = {
    "lmo_abi_version": (_i32, []),
    "lmo_layer_norm_fwd": (_i32, [_p, _p, _p, _p, _p, _p, _p, _i64, _i64, _f32, _i32, _p]),
    "lmo_layer_norm_scratch": (_i64, [_i64, _i64]),
    "lmo_layer_norm_bwd": (_i32, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _i64, _i32, _p]),
    "lmo_diff_attn_scratch": (_i64, [_p, _i32]),
    "lmo_diff_attn_fwd": (_i32, [_p, _p, _p, _p, _i32, _p, _p, _p, _p, _p, _p, _p, _i32, _p]),
    "lmo_diff_attn_bwd_scratch": (_i64, [_p, _i32]),
    "lmo_diff_attn_bwd": (_i32, [_p, _p, _p, _p, _i32, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i32, _p, _p, _i32, _p]),
    "lmo_distill_fwd": (_i32, [_p, _p, _i32, _p, _i32, _p, _p, _f32, _f32, _p, _p, _p, _i64, _i64, _i64, _i32, _p]),
    "lmo_distill_bwd": (_i32, [_p, _p, _i32, _p, _i32, _p, _f32, _p, _p, _p, _p, _i64, _i64, _i64, _i32, _i32, _p]),
}


def _load() -> ctypes.CDLL:
    path = _build.MODEL_LIB
    if not os.path.exists(path):
        raise ImportError(f"loopback_model: {path} is not built (run `python -m loopback_amd.build`)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)          # AttributeError -> the library is stale
        fn.restype, fn.argtypes = res, args
    if lib.lmo_abi_version() != ABI_VERSION:
        raise ImportError(f"loopback_model: {path} has ABI {lib.lmo_abi_version()}, expected {ABI_VERSION}; rebuild")
    return lib


LIB = _load()
for _name in SIGNATURES:
    H.bind(_name, ctypes.cast(getattr(LIB, _name), ctypes.c_void_p).value)


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
def _hat(h, eps):
    """(h - mean) rstd of unrounded rows, and rstd."""
    z = h - h.mean(-1, keepdim=True)
    r = torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + eps)
    return z * r, r


def _norm_torch(h, w, b, eps):
    y = _hat(_upcast(h), eps)[0]
    y = y if w is None else y * _upcast(w)
    y = y if b is None else y + _upcast(b)
    return y.to(h.dtype)


def _norm_backward(dh, dy, h, w, need, eps):
    """The torch form of the layer norm's backward, for the node (csrc/host.cpp), by its formulas: the gradients of h, the weight
    and the bias that need's bits ask for."""
    dt, out = h.dtype, [None] * 3
    hat, r = _hat(_upcast(h), eps)
    g = _upcast(dy)
    if need & 1:
        t = g if w is None else g * _upcast(w)
        dx = r * (t - t.mean(-1, keepdim=True) - hat * (t * hat).mean(-1, keepdim=True))
        out[0] = (dx if dh is None else dx + _upcast(dh)).to(dt)
    lead = list(range(h.dim() - 1))
    if need & 2:
        out[1] = (g * hat).sum(lead).to(dt) if lead else (g * hat).to(dt)
    if need & 4:
        out[2] = g.sum(lead).to(dt) if lead else g.to(dt)
    return tuple(out)


def _norm_args(x, add, weight, bias):
    if not isinstance(x, torch.Tensor) or not x.is_floating_point() or x.dim() < 1:
        raise ValueError("layer norm takes a floating point tensor of at least one dimension")
    d = x.shape[-1]
    for name, w in (("weight", weight), ("bias", bias)):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name} has the width's shape ({d},), got {tuple(w.shape)}")
    if add is not None and add.shape != x.shape:
        raise ValueError(f"add has x's shape {tuple(x.shape)}, got {tuple(add.shape)}")


def norm_native(x, add, weight, bias) -> bool:
    """Whether the kernels take the call."""
    ts = [t for t in (x, add, weight, bias) if t is not None]
    return (native(*ts, codes=_CODES) and x.numel() > 0 and x.shape[-1] <= NORM_MAX_WIDTH
            and x.numel() // x.shape[-1] <= MAX_ROWS)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) rsqrt(var + eps) weight + bias over the last dimension, var the mean square of the differences from the mean;
    weight and bias (d,) may be left out. Rounded once. Differentiable in x, weight and bias."""
    _norm_args(x, None, weight, bias)
    eps = float(eps)
    if not norm_native(x, None, weight, bias):
        return _norm_torch(x, weight, bias, eps)
    x, weight, bias = _plain_rows(x, weight, bias)   # recorded, where they copy
    return H.layer_norm(x, None, weight, bias, eps, _CODES[x.dtype], _stream(x), _records(x, weight, bias))[1]


def add_layer_norm(x: torch.Tensor, add: torch.Tensor | None, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5):
    """(h, layer_norm(h)) of h = x + add, rounded to its type as the residual stream carries it on; add None: h is x. In the
    backward the gradients of both results meet in one pass."""
    _norm_args(x, add, weight, bias)
    eps = float(eps)
    if add is None and not (torch.is_grad_enabled() and x.requires_grad):
        return x, layer_norm(x, weight, bias, eps)
    if not norm_native(x, add, weight, bias):
        h = x if add is None else x + add
        return h, _norm_torch(h, weight, bias, eps)
    x, add, weight, bias = _plain_rows(x, add, weight, bias)
    return H.layer_norm(x, add, weight, bias, eps, _CODES[x.dtype], _stream(x), _records(x, add, weight, bias))


# ---------------------------------------------------------------------------------------------------------------
# differential attention
# ---------------------------------------------------------------------------------------------------------------
ATTN_MAX_DH, ATTN_MAX_DV, ATTN_MAX_TOKENS, ATTN_MAX_HEADS, ATTN_MAX_ROWS = 128, 256, 2 ** 30 - 1, 0x7fffff, 2 ** 29
ATTN_MAX_STRIDE, ATTN_MAX_OUT = 2 ** 23, 2 ** 26   # between rows of q, k and v, and of y's gradient


def _seen(b, tq, tk, causal, lengths, starts, device):
    """(b, tq, tk): which keys each query sees."""
    j = torch.arange(tk, device=device)
    i = torch.arange(tq, device=device).view(-1, 1)
    seen = torch.ones((b, tq, tk), dtype=torch.bool, device=device)
    if causal:
        start = tk - tq if starts is None else starts.view(-1, 1, 1)
        seen = seen & (j <= start + i)
    return seen if lengths is None else seen & (j < lengths.view(-1, 1, 1))


def _maps(q, k, causal, scale, lengths, starts):
    """Both softmax maps (b, hk, group, 2, tq, tk) of the unrounded q and k."""
    (b, tq, h2, dh), tk, hk = q.shape, k.shape[1], k.shape[2] // 2
    q = q.reshape(b, tq, hk, h2 // (2 * hk), 2, dh).permute(0, 2, 3, 4, 1, 5)
    k = k.reshape(b, tk, hk, 1, 2, dh).permute(0, 2, 3, 4, 5, 1)
    s = q.matmul(k.expand(b, hk, q.shape[2], 2, dh, tk).contiguous()) * scale
    s = torch.where(_seen(b, tq, tk, causal, lengths, starts, q.device).view(b, 1, 1, 1, tq, tk), s, -torch.inf)
    if tk:
        s = s - s.detach().amax(-1, keepdim=True).clamp_min(-1e30)   # finite where no key is seen
    e = torch.exp(s)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _held(t, lengths):
    """t (b, tk, ...) with zeros past the lengths: what is there is not read into anything."""
    if lengths is None:
        return t
    there = torch.arange(t.shape[1], device=t.device) < lengths.view(-1, 1)
    return torch.where(there.view(*there.shape, *(1 for _ in t.shape[2:])), t, 0.0)


def _lam_of(lam, b, tq, hk, group):
    """lam as (b, hk, group, tq, 1)."""
    return lam.expand(b, tq, hk * group).reshape(b, tq, hk, group).permute(0, 2, 3, 1).unsqueeze(-1)


def _own_types(t):
    """Products of the types that they are given, where autocast would take 16 bits for them: scores keep 32, and no backward forms a
    16-bit batched product of a transposed operand."""
    kind = t.device.type
    on = kind in ("cuda", "cpu") and torch.is_autocast_enabled(kind)
    return torch.autocast(kind, enabled=False) if on else contextlib.nullcontext()


def _diff_torch(q, k, v, lam, causal, scale, lengths, starts):
    with _own_types(q):
        return _diff_formula(q, k, v, lam, causal, scale, lengths, starts)


def _diff_formula(q, k, v, lam, causal, scale, lengths, starts):
    dt, (b, tq), hk, group = q.dtype, q.shape[:2], v.shape[2], q.shape[2] // (2 * v.shape[2])
    k, v = _held(_upcast(k), lengths), _held(_upcast(v), lengths)
    p = _maps(_upcast(q), k, causal, scale, lengths, starts)
    a = p[:, :, :, 0] - _lam_of(_upcast(lam), b, tq, hk, group) * p[:, :, :, 1]
    y = a.matmul(v.permute(0, 2, 1, 3).unsqueeze(2).expand(b, hk, group, v.shape[1], v.shape[3]).contiguous())
    return y.permute(0, 3, 1, 2, 4).reshape(b, tq, hk * group, v.shape[3]).to(dt)


def _diff_backward(dy, q, k, v, lam, lengths, starts, causal, need, scale):
    """The torch form of differential attention's backward, for the node (csrc/host.cpp), by its formulas: the gradients of q, k, v
    and lam that need's bits ask for."""
    with _own_types(q):
        return _diff_gradients(dy, q, k, v, lam, lengths, starts, causal, need, scale)


def _diff_gradients(dy, q, k, v, lam, lengths, starts, causal, need, scale):
    dt, (b, tq, h2, dh), (tk, hk, dv) = q.dtype, q.shape, v.shape[1:]
    group = h2 // (2 * hk)
    qu, ku, vu = _upcast(q), _held(_upcast(k), lengths), _held(_upcast(v), lengths)
    p = _maps(qu, ku, causal, scale, lengths, starts)
    l1 = _lam_of(_upcast(lam), b, tq, hk, group)
    g = _upcast(dy).reshape(b, tq, hk, group, dv).permute(0, 2, 3, 1, 4)                   # (b, hk, group, tq, dv)
    da = g.matmul(vu.permute(0, 2, 3, 1).unsqueeze(2).expand(b, hk, group, dv, tk).contiguous())
    p1, p2 = p[:, :, :, 0], p[:, :, :, 1]
    d1, d2 = (p1 * da).sum(-1, keepdim=True), (p2 * da).sum(-1, keepdim=True)
    ds = torch.stack((p1 * (da - d1), -l1 * p2 * (da - d2)), 3) * scale                    # (b, hk, group, 2, tq, tk)
    out = [None] * 4
    if need & 1:
        kk = ku.reshape(b, tk, hk, 1, 2, dh).permute(0, 2, 3, 4, 1, 5).expand(b, hk, group, 2, tk, dh).contiguous()
        out[0] = ds.matmul(kk).permute(0, 4, 1, 2, 3, 5).reshape(q.shape).to(dt)
    if need & 2:
        qq = qu.reshape(b, tq, hk, group, 2, dh).permute(0, 2, 3, 4, 1, 5).contiguous()
        dk = ds.transpose(-1, -2).contiguous().matmul(qq).sum(2)                           # (b, hk, 2, tk, dh)
        out[1] = dk.permute(0, 3, 1, 2, 4).reshape(k.shape).to(dt)
    if need & 4:
        dval = (p1 - l1 * p2).transpose(-1, -2).contiguous().matmul(g.contiguous()).sum(2)
        out[2] = dval.permute(0, 2, 1, 3).reshape(v.shape).to(dt)
    if need & 8:
        dl = -d2.squeeze(-1).permute(0, 3, 1, 2).reshape(b, tq, hk * group)
        out[3] = (dl if lam.dim() == 3 else dl.sum((0, 1)) if lam.dim() == 1 else dl.sum()).to(lam.dtype)
    return tuple(out)


def attention_native(q, k, v, lam) -> bool:
    """Whether the kernels take the call: bf16 or fp16, widths that are multiples of 8 up to 128 and 256, lam of their type or fp32."""
    return (native(q, k, v) and (type(lam) is torch.Tensor or type(lam) is torch.nn.Parameter) and lam.dtype in (q.dtype, torch.float32)
            and q.numel() > 0 and k.numel() > 0 and q.shape[3] % 8 == 0 and q.shape[3] <= ATTN_MAX_DH and v.shape[3] % 8 == 0
            and 0 < v.shape[3] <= ATTN_MAX_DV and max(q.shape[1], k.shape[1]) <= ATTN_MAX_TOKENS and q.shape[0] * q.shape[2] <= ATTN_MAX_HEADS
            and q.shape[0] * q.shape[1] * q.shape[2] // 2 < ATTN_MAX_ROWS
            # a copy of rows has them that far apart
            and all(t.shape[1] == 1 or t.shape[2] * t.shape[3] <= ATTN_MAX_STRIDE for t in (q, k, v))
            and (q.shape[1] == 1 or q.shape[2] // 2 * v.shape[3] <= ATTN_MAX_OUT))


def diff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, *, causal: bool = True,
                   scale: float | None = None, lengths: torch.Tensor | None = None,
                   starts: torch.Tensor | None = None) -> torch.Tensor:
    """Differential attention of H heads, each of two maps: y = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v.

    q (b, tq, 2 H, dh), rows 2 h and 2 h + 1 head h's two queries; k (b, tk, 2 G, dh) and v (b, tk, G, dv), G dividing H: H / G heads
    in a row share a pair of keys and its values. lam is one value (), one per head (H,) or one per query and head (b, tq, H), of
    q's type or fp32. Returns (b, tq, H, dv). scale: dh^-0.5 unless given, above 0.

    A query i of batch row n sees the keys j < lengths[n] (all tk without it) and, where causal, j <= starts[n] + i: starts is the
    position of the first query among the keys, tk - tq without it (the queries are the last tokens). A query that sees no key has
    zeros and no gradient. What k and v hold at and past lengths is not read into anything, and its gradient is zero; an infinity or
    a NaN among the keys before that may also reach queries that do not see it yet, as a product with a probability of 0. lengths and
    starts are int32 or int64 (b,), read when a kernel runs. Differentiable in q, k, v and lam."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or not (q.is_floating_point() and k.is_floating_point() and v.is_floating_point()):
        raise ValueError(f"diff_attention takes floating point q (b, tq, 2 H, dh), k (b, tk, 2 G, dh), v (b, tk, G, dv), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    b, tq, h2, dh = q.shape
    tk, g = v.shape[1], v.shape[2]
    if k.shape != (b, tk, 2 * g, dh) or v.shape[0] != b or g < 1 or h2 % (2 * g) or h2 == 0 or dh == 0 or v.shape[3] == 0:
        raise ValueError(f"diff_attention takes q (b, tq, 2 H, dh), k (b, tk, 2 G, dh), v (b, tk, G, dv), G dividing H, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    h = h2 // 2
    if not isinstance(lam, torch.Tensor) or not lam.is_floating_point() or tuple(lam.shape) not in ((), (h,), (b, tq, h)):
        raise ValueError(f"lam is a floating point tensor (), ({h},) or ({b}, {tq}, {h}), got "
                         f"{tuple(lam.shape) if isinstance(lam, torch.Tensor) else lam!r}")
    for t in (k, v, lam):
        if t.device != q.device:
            raise ValueError(f"q is on {q.device}, k, v or lam on {t.device}")
    scale = dh ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale is above 0, got {scale}")
    for name, t in (("lengths", lengths), ("starts", starts)):
        if t is not None and (t.dtype not in (torch.int32, torch.int64) or t.shape != (b,) or t.device != q.device):
            raise ValueError(f"{name} is an int32 or int64 tensor ({b},) on {q.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    causal = bool(causal)
    plain = all(t is None or type(t) is torch.Tensor for t in (lengths, starts))
    if not (plain and attention_native(q, k, v, lam)):
        return _diff_torch(q, k, v, lam, causal, scale, lengths, starts)
    lengths, starts = (t if t is None or t.dtype is torch.int32 else t.clamp(-ATTN_MAX_TOKENS, ATTN_MAX_TOKENS).int()
                       for t in (lengths, starts))
    lengths, starts = _plain_rows(lengths, starts)
    return H.diff_attn(q, k, v, lam, lengths, starts, causal, scale, _CODES[q.dtype], _stream(q), _records(q, k, v, lam))


# ---------------------------------------------------------------------------------------------------------------
# distillation from a teacher's highest logits
# ---------------------------------------------------------------------------------------------------------------
IGNORED = -100


def _teacher(top, ids, lse, tau, vocab):
    """(which entries name a class, which rows count, log p, p): fp32, or fp64 where the logits are."""
    valid = ids >= 0
    counts = valid.any(-1)
    z = torch.where(valid, _upcast(top) / tau, -torch.inf)
    ref = torch.logsumexp(z, -1) if lse is None else lse
    logp = z - torch.where(counts, ref, 0.0).unsqueeze(-1)
    return valid, counts, logp, torch.exp(logp)


def _unnamed(x, valid, at):
    """Which classes of each row are not named (bool, x's shape)."""
    named = torch.zeros((x.shape[0], x.shape[1] + 1), dtype=torch.bool, device=x.device)
    return ~named.scatter(1, torch.where(valid, at, x.shape[1]), True)[:, :-1]


def _rest(p, lse, free):
    """What the teacher leaves to the classes that it does not name."""
    if lse is None:
        return None
    return torch.where(free.any(-1), (1 - p.sum(-1)).clamp_min(0), 0.0)


def _distill_torch(logits, top, ids, lse, labels, tau, hard):
    x = _upcast(logits)
    t, vocab = x.shape
    valid, counts, logp, p = _teacher(top, ids, lse, tau, vocab)
    at = ids.long().clamp(0, vocab - 1)
    scaled = x / tau
    logq = scaled - torch.logsumexp(scaled, -1, keepdim=True)
    kl = torch.where(p > 0, p * (logp - logq.gather(1, at)), torch.where(p == 0, 0.0, p)).sum(-1)
    if lse is not None:
        free = _unnamed(x, valid, at)
        rest = _rest(p, lse, free)
        some = rest > 0
        logr = torch.logsumexp(torch.where(free, logq, -torch.inf), -1)
        kl = kl + torch.where(some, rest * (torch.log(torch.where(some, rest, 1.0)) - logr), 0.0)
    bad = (ids >= vocab).any(-1)
    kl = torch.where(bad, torch.nan, kl)
    loss = (1 - hard) * tau * tau * torch.where(counts, kl, 0.0).sum() / counts.sum().clamp_min(1)
    if labels is not None:
        labelled = labels != IGNORED
        outside = labelled & ((labels < 0) | (labels >= vocab))
        nll = torch.logsumexp(x, -1) - x.gather(1, labels.clamp(0, vocab - 1).unsqueeze(-1)).squeeze(-1)
        nll = torch.where(outside, torch.nan, torch.where(labelled, nll, 0.0))
        loss = loss + hard * nll.sum() / labelled.sum().clamp_min(1)
    return loss


def _distill_backward(g, logits, top, ids, lse, labels, tau, hard):
    """The torch form of the loss's backward, for the node (csrc/host.cpp), by its formulas: the gradient of the logits."""
    shape, vocab = logits.shape, logits.shape[-1]
    x = _upcast(logits).reshape(-1, vocab)
    top, ids = top.reshape(x.shape[0], -1), ids.reshape(x.shape[0], -1).long()
    lse = None if lse is None else lse.reshape(-1)
    valid, counts, _, p = _teacher(top, ids, lse, tau, vocab)
    at = ids.clamp(0, vocab - 1)
    q = torch.softmax(x / tau, -1)
    target = torch.zeros((x.shape[0], vocab + 1), dtype=x.dtype, device=x.device)
    target = target.scatter_add(1, torch.where(valid & (ids < vocab), at, vocab), p.to(x.dtype))[:, :-1]
    whole = p.sum(-1)
    if lse is not None:
        free = _unnamed(x, valid, at)
        rest = _rest(p, lse, free)
        whole = whole + rest
        others = torch.softmax(torch.where(free, x / tau, -torch.inf), -1)
        target = target + torch.where(free & (rest > 0).unsqueeze(-1), others * rest.unsqueeze(-1), 0.0)
    d = (q * whole.unsqueeze(-1) - target) * ((1 - hard) * tau / counts.sum().clamp_min(1))
    d = torch.where(counts.unsqueeze(-1), d, 0.0)
    if labels is not None:
        labels = labels.reshape(-1)
        labelled = labels != IGNORED
        inside = labelled & (labels >= 0) & (labels < vocab)
        one = torch.zeros_like(target).scatter(1, labels.clamp(0, vocab - 1).unsqueeze(-1), inside.unsqueeze(-1).to(x.dtype))
        d = d + torch.where(labelled.unsqueeze(-1), (torch.softmax(x, -1) - one) * (hard / labelled.sum().clamp_min(1)), 0.0)
    return ((g * d).to(logits.dtype).view(shape),)


def distill_loss(logits: torch.Tensor, top_logits: torch.Tensor, top_ids: torch.Tensor, *, temperature: float = 1.0,
                 teacher_lse: torch.Tensor | None = None, labels: torch.Tensor | None = None,
                 hard_weight: float = 0.0) -> torch.Tensor:
    """The distillation loss of logits x (..., vocab) from a teacher's k highest logits (..., k) of the classes top_ids (..., k,
    int32 or int64), a scalar in fp32:

        (1 - hard_weight) temperature^2 mean(KL(p || q)) + hard_weight mean(-log softmax(x)[label])

    q = softmax(x / temperature). p is the softmax of the teacher's k logits / temperature, or, with teacher_lse (...,), the log
    of its sum of exp(logit / temperature) over every class, exp(logit / temperature - teacher_lse); what that leaves is one
    event, the classes that are not named, on both sides. An id below 0 names nothing (rows with fewer than k), a row that names
    nothing does not count, a class named twice has both its probabilities; labels (..., int64) of -100 are ignored; the means
    are over the rows that count and over those with a label, 0 over none. An id of vocab or more, or another label outside the
    vocabulary, makes the loss NaN. Differentiable in the logits alone, whose gradient is rounded once."""
    tau, hard = float(temperature), float(hard_weight)
    if logits.dim() < 1 or not logits.is_floating_point() or logits.shape[-1] < 1:
        raise ValueError(f"distill_loss takes floating point logits (..., vocab), got {logits.dtype} {tuple(logits.shape)}")
    lead = logits.shape[:-1]
    if top_logits.shape != top_ids.shape or top_logits.shape[:-1] != lead or top_logits.dim() != logits.dim() \
            or top_logits.shape[-1] < 1:
        raise ValueError(f"top_logits and top_ids have the shape {tuple(lead)} + (k,), got {tuple(top_logits.shape)} and "
                         f"{tuple(top_ids.shape)}")
    if not top_logits.is_floating_point() or top_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"top_logits are floating point and top_ids int32 or int64, got {top_logits.dtype} and {top_ids.dtype}")
    if not 0.0 < tau < float("inf"):
        raise ValueError(f"temperature is above 0, got {temperature}")
    if not 0.0 <= hard <= 1.0 or (hard > 0.0 and labels is None):
        raise ValueError(f"hard_weight lies in [0, 1], and above 0 needs labels, got {hard_weight}")
    if teacher_lse is not None and (teacher_lse.shape != lead or not teacher_lse.is_floating_point()):
        raise ValueError(f"teacher_lse is floating point of the shape {tuple(lead)}, got {teacher_lse.dtype} {tuple(teacher_lse.shape)}")
    if labels is not None and (labels.shape != lead or labels.dtype is not torch.int64):
        raise ValueError(f"labels are int64 of the shape {tuple(lead)}, got {labels.dtype} {tuple(labels.shape)}")
    given = [t for t in (top_logits, top_ids, teacher_lse, labels) if t is not None]
    for t in given:
        if t.device != logits.device:
            raise ValueError(f"the logits are on {logits.device}, what they are compared with on {t.device}")
    top_logits = top_logits.detach()
    teacher_lse = None if teacher_lse is None else teacher_lse.detach()
    labels = labels if hard > 0.0 else None
    vocab, rows = logits.shape[-1], lead.numel()
    if not (native(logits, codes=_CODES) and logits.numel() > 0 and rows <= MAX_ROWS and top_logits.shape[-1] <= DISTILL_MAX_TOP
            and vocab < 2 ** 31 - 8 and (teacher_lse is None or vocab <= DISTILL_MAX_TAIL) and top_logits.dtype in _CODES
            and all(type(t) is torch.Tensor for t in given)):
        flat = [t.reshape(rows, t.shape[-1]) for t in (logits, top_logits, top_ids)]
        one = [None if t is None else t.reshape(rows) for t in (teacher_lse, labels)]
        return _distill_torch(*flat, *one, tau, hard)
    teacher_lse = None if teacher_lse is None else teacher_lse.float()
    logits, top_logits, top_ids, teacher_lse, labels = _plain_rows(logits, top_logits, top_ids, teacher_lse, labels)
    return H.distill(logits, top_logits, top_ids, teacher_lse, labels, tau, hard, _CODES[logits.dtype], _stream(logits),
                     _records(logits))


H.model_forms(_norm_backward, _distill_backward, _diff_backward)
