"""Operators of a transformer block's training step on the HIP kernels of libloopback_block.so (include/loopback_block.h):

  * `gated_ffn(x, w_gate_up, w_down)`: the gated feed-forward block, both projections, the activation and the product in
    one kernel, the activation's gradient in the one that forms it (bf16 and fp16);
  * `block_join(x, y, ...)`: a block's output y back on the residual stream x, with the norm after the block, a gate, a
    residual scale and dropout before the add, and the next block's norm after it;
  * `dropout(x, p, rng, site)`: dropout whose mask comes from a counter-based generator and is never stored.

The row kernels take plain fp32, bf16 and fp16 tensors of the current GPU where nothing has to see torch operations (lm_ops.native
says what does); everything else -- the CPU, other types, mixed types, autocast (but for dropout), tracers, transforms -- runs
the torch form of the same operator: the same formulas and the same masks. A backward that is itself differentiated, or
watched, runs the torch form too. Tensors of any strides are taken (the kernels work on contiguous rows; others are copied). Saved tensors that a hook gives
back with another shape, type or device are refused.

Dropout's generator: `rng` is an int64 tensor (seed, step) on the inputs' device, read when a kernel runs: a captured graph
draws a new mask when the program has changed it, and a backward reads it again, so the program changes a copy, not the
tensor that a forward took, before that forward's backward (autograd refuses it otherwise). `site`, 0 to 2^32 - 1, tells the
places of one step apart. The mask depends on (seed, step, site, row, column) alone.
"""
from __future__ import annotations

import ctypes
import os

import torch
import torch.nn.functional as F

from . import _host as H      # the launch path (csrc/host.cpp), bound below to the library
from . import build as _build
from .lm_ops import _stream, _watched, native

ABI_VERSION = 3
JOIN_MAX_WIDTH = 8192
FEW_TOKENS = 32
FFN_MAX_WIDTH = 2 ** 22 - 8   # elements between rows of the tiled products' operands
MAX_ROWS = 2 ** 31 - 1
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_p, _i64, _i32, _u32, _f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_uint32, ctypes.c_float
# name -> (restype, argtypes); one line per declaration of include/loopback_block.h
SIGNATURES = {
    "lbk_abi_version": (_i32, []),
    "lbk_dropout": (_i32, [_p, _p, _u32, _i32, _p, _i64, _i64, _i32, _p]),
    "lbk_join_fwd": (_i32, [_p, _p, _p, _p, _i64, _p, _p, _u32, _i32, _f32, _f32, _p, _p, _p, _p, _i64, _i64, _i32, _p]),
    "lbk_join_scratch": (_i64, [_i64, _i64, _i64]),
    "lbk_join_bwd": (_i32, [_p, _p, _p, _p, _p, _p, _i64, _p, _p, _p, _p, _u32, _i32, _f32, _p, _p, _p, _p, _p, _p, _i64,
                            _i64, _i32, _p]),
    "lbk_ffn_saved_bytes": (_i64, [_i64, _i64]),
    "lbk_pad_rows": (_i32, [_p, _i64, _i64, _i64, _p, _i32, _p]),
    "lbk_ffn_gate_up": (_i32, [_p, _i64, _p, _i64, _p, _i64, _p, _i64, _i64, _i64, _i32, _i32, _p]),
    "lbk_ffn_dgate_up": (_i32, [_p, _i64, _p, _i64, _p, _p, _i64, _i64, _i64, _i64, _i32, _p]),
    "lbk_linear_scratch": (_i64, [_i64, _i64, _i64]),
    "lbk_product_tiling": (_i32, [_i32, _i64, _i64, _i64, ctypes.POINTER(_i32)]),
    "lbk_linear_fwd": (_i32, [_p, _i64, _p, _i64, _p, _i64, _p, _i64, _i64, _i64, _i32, _p]),
    "lbk_linear_dx": (_i32, [_p, _i64, _p, _i64, _p, _i64, _p, _i64, _i64, _i64, _i32, _p]),
    "lbk_linear_dw": (_i32, [_p, _i64, _p, _i64, _p, _p, _i64, _i64, _i64, _i32, _p]),
}


def _load() -> ctypes.CDLL:
    path = _build.BLOCK_LIB
    if not os.path.exists(path):
        raise ImportError(f"loopback_block: {path} is not built (run `python -m loopback_amd.build`)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)          # AttributeError -> the library is stale
        fn.restype, fn.argtypes = res, args
    if lib.lbk_abi_version() != ABI_VERSION:
        raise ImportError(f"loopback_block: {path} has ABI {lib.lbk_abi_version()}, expected {ABI_VERSION}; rebuild")
    return lib


LIB = _load()
for _name in SIGNATURES:
    H.bind(_name, ctypes.cast(getattr(LIB, _name), ctypes.c_void_p).value)


def _upcast(t: torch.Tensor) -> torch.Tensor:
    return t.float() if t.dtype in (torch.bfloat16, torch.float16) else t


def _plain_rows(*tensors):
    return [t if t is None or t.is_contiguous() else t.contiguous() for t in tensors]


def _records(*tensors) -> bool:
    """Whether a call on these records a backward."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------------------------
def _drop_of(p: float, rng, x, site) -> int:
    """The probability's 65536ths, after the checks of dropout's arguments."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"a dropout probability lies in [0, 1], got {p}")
    if not 0 <= site < 2 ** 32:
        raise ValueError(f"site lies in [0, 2^32), got {site}")
    drop = round(65536 * p)
    if drop:
        if not isinstance(rng, torch.Tensor) or rng.dtype is not torch.int64 or rng.shape != (2,):
            raise ValueError("dropout needs rng, an int64 tensor (seed, step)")
        if rng.device != x.device:
            raise ValueError(f"rng is on {rng.device}, the input on {x.device}")
    return drop


def keep_mask(shape, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
    """The kept elements (bool, `shape`) of dropout(x, p, rng, site) for an x of this shape, in torch operations."""
    shape = torch.Size(shape)
    drop = _drop_of(p, rng, rng, site)
    d = shape[-1] if shape else 1
    rows = shape[:-1].numel()
    return _mask(drop, rng, site, rows, d).view(shape)


def _mask(drop: int, rng, site: int, rows: int, d: int) -> torch.Tensor:
    """Philox-4x32-10 (Salmon et al., 2011) in 64-bit integers, a counter per row and eight columns, 16 bits a column."""
    nb, low, dev = (d + 7) // 8, 0xFFFFFFFF, rng.device
    c0 = torch.arange(nb, device=dev).expand(rows, nb)
    c1 = torch.arange(rows, device=dev).unsqueeze(1).expand(rows, nb)
    c2 = torch.full((rows, nb), site, device=dev, dtype=torch.int64)
    c3 = (rng[1] & low).expand(rows, nb)
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57      # modulo 2^64: the shifts below take the bits that are right
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack((c0, c1, c2, c3), -1)
    return (torch.stack((w & 0xFFFF, w >> 16), -1).reshape(rows, 8 * nb)[:, :d] >= drop)


def _dropout_torch(x, rng, site, drop):
    d = x.shape[-1] if x.dim() else 1
    keep = _mask(drop, rng, site, x.shape[:-1].numel(), d).view(x.shape)
    s = 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    return torch.where(keep, _upcast(x) * s, 0.0).to(x.dtype)


def _dropout_backward(dy, rng, site, drop):
    """The torch form of dropout's backward, for the node (csrc/host.cpp) where that has to be torch operations."""
    return (_dropout_torch(dy, rng, site, drop),)


def _dropout_native(x, rng) -> bool:
    # autocast changes nothing here: the operation keeps its input's type
    return ((native(x, codes=_CODES) or _autocast_only(x)) and x.dim() > 0 and x.numel() > 0
            and x.shape[:-1].numel() <= MAX_ROWS and type(rng) is torch.Tensor and rng.is_contiguous())


def _autocast_only(x) -> bool:
    if _watched() or not x.is_cuda or not torch.is_autocast_enabled("cuda"):
        return False
    with torch.autocast("cuda", enabled=False):
        return native(x, codes=_CODES)


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor | None, site: int = 0) -> torch.Tensor:
    """x with each element dropped with probability p (to its 65536ths; 0 returns x) and the others multiplied by 1 / (1 - p);
    what is dropped is 0, also where x is not finite. The rows of the generator are those of x's last dimension."""
    if not x.is_floating_point():
        raise ValueError(f"dropout takes floating point tensors, got {x.dtype}")
    drop = _drop_of(p, rng, x, site)
    if drop == 0:
        return x
    if not _dropout_native(x, rng):
        return _dropout_torch(x, rng, site, drop)
    return H.dropout(x.contiguous(), rng, site, drop, _CODES[x.dtype], _stream(x), _records(x))


# ---------------------------------------------------------------------------------------------------------------
# block join
# ---------------------------------------------------------------------------------------------------------------
def _rms_torch(x, w, eps):
    """rms_norm of unrounded rows (fp32, or fp64 where those are given)."""
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * _upcast(w)


def _branch_torch(y, post, gate, rng, site, drop, scale, eps):
    """What is added to the residual stream, unrounded."""
    z = _upcast(y)
    if post is not None:
        z = _rms_torch(z, post, eps)
    if gate is not None:
        z = z * _upcast(gate)
    z = z * scale
    return _dropout_torch(z, rng, site, drop) if drop else z


def _join_torch(x, y, post, gate, pre, rng, site, drop, scale, eps):
    h = _upcast(x) + _branch_torch(y, post, gate, rng, site, drop, scale, eps)
    return h.to(x.dtype), None if pre is None else _rms_torch(h, pre, eps).to(x.dtype)


def _norm_grad(g, v, r):
    """The gradient of v r, r = rsqrt(mean(v^2) + eps), from that of the product g."""
    vh = v * r
    return r * (g - vh * (g * vh).mean(-1, keepdim=True))


def _sum_like(t, like):
    """t summed over the dimensions that `like` is broadcast over."""
    lead = t.dim() - like.dim()
    dims = [*range(lead), *(i for i in range(lead, t.dim()) if like.shape[i - lead] == 1 and t.shape[i] != 1)]
    return (t.sum(dims, keepdim=True) if dims else t).reshape(like.shape)


def _join_backward(dh, dn, x, y, post, gate, pre, rng, site, drop, need, scale, eps):
    """The torch form of the join's backward, for the node (csrc/host.cpp): the gradients of x, y, post, gate and pre that need's
    bits ask for, by their formulas (not by autograd: the node is locked while it runs, and the engine would wait for it). The
    norm's gradient is formed at the sum before its rounding."""
    nx, ny, npost, ngate, npre = (bool(need & b) for b in (1, 2, 4, 8, 16))
    dt, out = y.dtype, [None] * 5
    g = None if dh is None else _upcast(dh)
    if dn is not None:
        hu, dnu = _upcast(x) + _branch_torch(y, post, gate, rng, site, drop, scale, eps), _upcast(dn)
        r2 = torch.rsqrt(hu.pow(2).mean(-1, keepdim=True) + eps)
        gn = _norm_grad(dnu * _upcast(pre), hu, r2)
        g = gn if g is None else g + gn
        if npre:
            out[4] = _sum_like(dnu * (hu * r2), pre).to(dt)
    if nx:
        out[0] = g.to(dt)
    t, yu = g * scale, _upcast(y)
    if drop:
        t = _dropout_torch(t, rng, site, drop)
    r1 = None if post is None else torch.rsqrt(yu.pow(2).mean(-1, keepdim=True) + eps)
    yh = yu if post is None else yu * r1
    if ngate:
        out[3] = _sum_like(t * yh if post is None else t * yh * _upcast(post), gate).to(dt)
    if gate is not None:
        t = t * _upcast(gate)
    if npost:
        out[2] = _sum_like(t * yh, post).to(dt)
    if ny:
        out[1] = (t if post is None else _norm_grad(t * _upcast(post), yu, r1)).to(dt)
    return tuple(out)


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """The consecutive rows of x that share a row of the gate: (d,), or x's dimensions with the last leading ones 1."""
    lead, gl = x.shape[:-1], gate.shape[:-1]
    if gate.dim() >= 1 and gate.shape[-1] == x.shape[-1]:
        if gate.dim() == 1:
            return max(1, lead.numel())
        if len(gl) == len(lead):
            for k in range(len(lead) + 1):
                if gl[:k] == lead[:k] and all(s == 1 for s in gl[k:]):
                    return max(1, lead[k:].numel())
    raise ValueError(f"a gate for {tuple(x.shape)} is ({x.shape[-1]},) or has x's dimensions, the last of those before the "
                     f"width 1: got {tuple(gate.shape)}")


def block_join(x: torch.Tensor, y: torch.Tensor, *, post_weight: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0, dropout: float = 0.0,
               rng: torch.Tensor | None = None, site: int = 0, pre_weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(h, n) of a residual stream x and a block's output y of one shape (..., d):

        h = x + drop(scale * gate * rms_norm(y) post_weight),   n = rms_norm(h) pre_weight

    Each of post_weight (d,), gate, dropout and pre_weight may be left out (n is then None, for pre_weight). The gate is one
    row (d,), a row for each of the leading dimensions ((b, 1, d) for (b, t, d): one per sequence), or x's shape. h and n are
    each rounded once, n from the unrounded sum. Differentiable in x, y, post_weight, gate and pre_weight."""
    if y.shape != x.shape or not x.is_floating_point() or x.dim() < 1:
        raise ValueError(f"block_join takes two floating point tensors of one shape, got {tuple(x.shape)} and {tuple(y.shape)}")
    d = x.shape[-1]
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None and w.shape != (d,):
            raise ValueError(f"{name} has the width's shape ({d},), got {tuple(w.shape)}")
    gate_rows = 1 if gate is None else _gate_rows(gate, x)
    drop = _drop_of(dropout, rng, x, site)
    scale, eps = float(scale), float(eps)
    ts = [t for t in (x, y, post_weight, gate, pre_weight) if t is not None]
    if not (native(*ts, codes=_CODES) and x.numel() > 0 and d <= JOIN_MAX_WIDTH and x.numel() // d <= MAX_ROWS
            and (not drop or (type(rng) is torch.Tensor and rng.is_contiguous()))):
        return _join_torch(x, y, post_weight, gate, pre_weight, rng, site, drop, scale, eps)
    x, y, post_weight, gate, pre_weight = _plain_rows(x, y, post_weight, gate, pre_weight)   # recorded, where they copy
    return H.join(x, y, post_weight, gate, gate_rows, pre_weight, rng, site, drop, scale, eps, _CODES[x.dtype], _stream(x),
                  _records(*ts))


# ---------------------------------------------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------
ACTIVATIONS = {"silu": 0, "gelu": 1}


def _ffn_torch(x, w_gate_up, w_down, activation):
    g, u = F.linear(x, w_gate_up).chunk(2, dim=-1)
    a = F.silu(g) if activation == 0 else F.gelu(g, approximate="tanh")
    return F.linear(a * u, w_down)


def _ffn_backward(dy, x, w_gate_up, w_down, activation, need):
    """The torch form of the block's backward, for the node (csrc/host.cpp), by its formulas: the gradients of x, w_gate_up and
    w_down that need's bits ask for."""
    dt, n = x.dtype, w_down.shape[1]
    x2, dy2 = x.reshape(-1, x.shape[-1]), dy.reshape(-1, dy.shape[-1])
    g, u = (_upcast(t) for t in (x2 @ w_gate_up.t()).chunk(2, dim=-1))
    if activation == 0:
        c, q, dq = g, g, 1.0
    else:
        c = g.clamp(-100.0, 100.0)   # past these s is 0 or 1 and its derivative 0, and dq would overflow
        q, dq = 1.5957691216057308 * (c + 0.044715 * c.pow(3)), 1.5957691216057308 * (1 + 0.134145 * c.pow(2))
    s = torch.sigmoid(q)
    a = g * s
    out = [None, None, None]
    if need & 3:
        dact = _upcast(dy2 @ w_down)
        dgu = torch.cat((dact * u * (s + c * s * dq * (1 - s)), dact * a), -1).to(dt)
        out[0] = (dgu @ w_gate_up).reshape(x.shape) if need & 1 else None
        out[1] = dgu.t() @ x2 if need & 2 else None
    if need & 4:
        out[2] = dy2.t() @ (a * u).to(dt)
    return tuple(out)


H.torch_forms(_dropout_backward, _join_backward, _ffn_backward)


def gated_ffn(x: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """(a(x Wg^T) * (x Wu^T)) Wd^T of x (..., d), w_gate_up (2 n, d) = [Wg; Wu] and w_down (m, n); a is "silu" or "gelu" (its
    tanh form). On the kernels the projections, the activation and their product are one fp32 value rounded once, and the
    backward's gradients of the two projections are formed from 24 bits of them. A recorded call keeps 8 bytes per token and
    inner column for its backward (the activations and those bits)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if w_gate_up.dim() != 2 or w_down.dim() != 2 or x.dim() < 1 or w_gate_up.shape[1] != x.shape[-1] \
            or w_gate_up.shape[0] != 2 * w_down.shape[1]:
        raise ValueError(f"gated_ffn takes x (..., d), w_gate_up (2 n, d) and w_down (m, n), got {tuple(x.shape)}, "
                         f"{tuple(w_gate_up.shape)} and {tuple(w_down.shape)}")
    code = ACTIVATIONS[activation]
    if not (native(x, w_gate_up, w_down) and x.numel() > 0 and w_down.numel() > 0
            and x.numel() // x.shape[-1] <= MAX_ROWS and max(*w_gate_up.shape, *w_down.shape) <= FFN_MAX_WIDTH):
        return _ffn_torch(x, w_gate_up, w_down, code)
    x, w_gate_up, w_down = _plain_rows(x, w_gate_up, w_down)   # recorded, where they copy
    return H.gated_ffn(x, w_gate_up, w_down, code, _CODES[x.dtype], _stream(x), _records(x, w_gate_up, w_down))
