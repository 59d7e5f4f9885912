"""The operators of a transformer block's training step, as measurable cases through `loopback_amd.block_ops`.

Three operators, that a block of the language model (`loopback_amd.lm.Block`) calls one after another:
  * `ffn`: the gated feed-forward block, y = (a(x Wg^T) * (x Wu^T)) Wd^T, with every gradient where it trains;
  * `join`: a block's output back on the residual stream, h = x + drop(scale gate rms(y) w_post), n = rms(h) w_pre;
  * `dropout`: a mask from a counter-based generator, formed again in the backward pass instead of stored.

Sizes are the repository's configurations (widths 768, 1024 and 2048, their SwiGLU widths 2048 and 5632, 16384 tokens), its
odd test widths, and generic ragged ones. The plain forms compute in 32 bits and round once.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def _ffn(name, t, d, n, dtype, act, train):
    return {"name": name, "op": "ffn", "t": t, "d": d, "n": n, "dtype": dtype, "act": act, "train": train}


def _join(name, b, t, d, dtype, post, gate, scale, p, pre, train):
    return {"name": name, "op": "join", "b": b, "t": t, "d": d, "dtype": dtype, "post": post, "gate": gate, "scale": scale,
            "p": p, "pre": pre, "train": train}


def _drop(name, rows, d, dtype, p, train):
    return {"name": name, "op": "dropout", "t": rows, "d": d, "dtype": dtype, "p": p, "train": train}


def listed() -> list[dict]:
    return [
        # one token of a served model of width 2048: the weights' stream and the launches are everything
        _ffn("ffn_token", 1, 2048, 5632, "bf16", "silu", False),
        # a few ragged prompts at the LM's width
        _ffn("ffn_prompt", 333, 768, 2048, "bf16", "silu", False),
        # a small odd-sized model in fp16 mixed precision with the other activation, trained on a ragged batch
        _ffn("ffn_train_odd_fp16", 1001, 1001, 2731, "fp16", "gelu", True),
        # the LM's training step: 8 sequences of 2048 tokens
        _ffn("ffn_train_lm", 16384, 768, 2048, "bf16", "silu", True),
        # a wide model's training step, the most work
        _ffn("ffn_train_wide", 8192, 2048, 5632, "bf16", "silu", True),
        # one token back on the residual stream of a served model
        _join("join_token", 1, 1, 2048, "bf16", True, "column", 1.0, 0.0, True, False),
        # the LM's training step with norms before and after a block, a learned gate per channel and dropout
        _join("join_train_lm", 8, 2048, 768, "bf16", True, "column", 1.0, 0.1, True, True),
        # a wide model with one gate per sequence and a residual scale, fp16, ragged sequences
        _join("join_train_gated", 5, 1365, 2048, "fp16", True, "sequence", 0.5, 0.0, True, True),
        # an odd width in fp32: no norm after the block, a gate per token, dropout
        _join("join_train_odd_fp32", 3, 683, 1001, "fp32", False, "full", 0.7, 0.2, True, True),
        # dropout alone: a short batch, where latency counts
        _drop("dropout_short", 512, 768, "bf16", 0.5, False),
        # embeddings of the LM's training step
        _drop("dropout_train_lm", 16384, 768, "bf16", 0.1, True),
        # the largest: the inner activations of a wide feed-forward block
        _drop("dropout_train_wide", 16384, 5632, "bf16", 0.1, True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo: int, hi: int) -> int:
    """A width: two of three a multiple of eight, as models have them, one of three any."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 1 / 3 else max(8, w // 8 * 8)


def draw(rng) -> dict:
    op = rng.choice(("ffn", "ffn", "join", "join", "dropout"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "ffn":
        most = 18.0 * 8192 * 2048 * 5632
        while True:
            c = _ffn("", _log_int(rng, 1, 16384), _width(rng, 64, 4096), _width(rng, 64, 8192), dtype,
                     rng.choice(("silu", "gelu")), rng.random() < 0.6)
            if work(c)["flops"] <= most:
                break
    else:
        dtype = rng.choice((dtype, dtype, "fp32"))
        while True:
            b, t = _log_int(rng, 1, 32), _log_int(rng, 1, 8192)
            d = _width(rng, 8, 8192)
            if b * t * d <= 1 << 26:
                break
        if op == "join":
            c = _join("", b, t, d, dtype, rng.random() < 0.6, rng.choice(("none", "column", "sequence", "full")),
                      rng.choice((1.0, 0.5, 0.22)), rng.choice((0.0, 0.1, 0.3)), rng.random() < 0.8, rng.random() < 0.7)
        else:
            c = _drop("", b * t, d, dtype, rng.choice((0.05, 0.1, 0.5)), rng.random() < 0.6)
    del c["name"]
    return c


def _gate_shape(c):
    return {"column": (c["d"],), "sequence": (c["b"], 1, c["d"]), "full": (c["b"], c["t"], c["d"])}[c["gate"]]


def prepare(c: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[c["dtype"]], c["train"]

    def rnd(*shape, std=1.0, mean=0.0):
        return (mean + std * torch.randn(shape, device="cuda", generator=g)).to(dt)

    def rows(*shape):   # activations: channels of different sizes
        spread = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=g))
        return (torch.randn(shape, device="cuda", generator=g) * spread).to(dt)

    s = {"case": c}
    if c["op"] == "ffn":
        t, d, n = c["t"], c["d"], c["n"]
        s["x"], s["w_gate_up"], s["w_down"] = rows(t, d), rnd(2 * n, d, std=d ** -0.5), rnd(d, n, std=n ** -0.5)
        leaves = ("x", "w_gate_up", "w_down")
        if train:
            s["dy"] = rnd(t, d)
    elif c["op"] == "join":
        shape = (c["b"], c["t"], c["d"])
        s["x"], s["y"] = rows(*shape), rows(*shape)
        s["post"] = rnd(c["d"], std=0.1, mean=1.0) if c["post"] else None
        s["gate"] = rnd(*_gate_shape(c), std=0.2, mean=0.5) if c["gate"] != "none" else None
        s["pre"] = rnd(c["d"], std=0.1, mean=1.0) if c["pre"] else None
        leaves = ("x", "y", "post", "gate", "pre")
        if train:
            s["dh"], s["dn"] = rnd(*shape), rnd(*shape) if c["pre"] else None
    else:
        s["x"] = rows(c["t"], c["d"])
        leaves = ("x",)
        if train:
            s["dy"] = rnd(c["t"], c["d"])
    if c.get("p"):   # the generator's seed and the training step's number; the number of the place in the model
        s["rng"] = torch.stack((torch.randint(-2 ** 62, 2 ** 62, (), device="cuda", generator=g),
                                torch.randint(0, 100000, (), device="cuda", generator=g)))
        s["site"] = seed % 40
    s["leaves"] = [k for k in leaves if s[k] is not None]
    if train:
        for k in s["leaves"]:
            s[k].requires_grad_()
    return s


# -----------------------------------------------------------------------------------------------------------------------
# the plain forms
# -----------------------------------------------------------------------------------------------------------------------
def _words(rng, site, rows, blocks):
    """Philox-4x32-10 (Salmon et al., 2011): the four words of every counter (column block, row, site, step)."""
    low = 0xFFFFFFFF
    dev = rng.device
    c = [torch.arange(blocks, device=dev).expand(rows, blocks), torch.arange(rows, device=dev).view(-1, 1).expand(rows, blocks),
         torch.full((rows, blocks), site, device=dev), (rng[1] & low).expand(rows, blocks)]
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # products of 64 bits, modulo 2^64
        c = [(b >> 32) & low ^ c[1] ^ k0, b & low, (a >> 32) & low ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _keep(rng, site, rows, d, p):
    """The kept elements: 16 bits each, eight consecutive columns from one counter's four words."""
    w = torch.stack(_words(rng, site, rows, (d + 7) // 8), -1)
    bits = torch.stack((w & 0xFFFF, w >> 16), -1).reshape(rows, -1)[:, :d]
    return bits >= round(65536 * p)


def _dropped(z, rng, site, p):
    d = z.shape[-1]
    keep = _keep(rng, site, z.numel() // d, d, p).view(z.shape)
    return torch.where(keep, z * (65536 / (65536 - round(65536 * p))), torch.zeros((), device=z.device))


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _act(g, act):
    q = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)
    return g / (1 + torch.exp(-q))


def _plain(c, s, v):
    """The outputs of one forward of the case's operator on the 32-bit values v."""
    if c["op"] == "ffn":
        n = c["n"]
        gu = v["x"] @ v["w_gate_up"].t()
        return ((_act(gu[:, :n], c["act"]) * gu[:, n:]) @ v["w_down"].t(),)
    if c["op"] == "dropout":
        return (_dropped(v["x"], s["rng"], s["site"], c["p"]),)
    z = v["y"] if s["post"] is None else _rms(v["y"], v["post"])
    z = z if s["gate"] is None else z * v["gate"]
    z = z * c["scale"]
    z = _dropped(z, s["rng"], s["site"], c["p"]) if c["p"] else z
    h = v["x"] + z
    return (h,) if s["pre"] is None else (h, _rms(h, v["pre"]))


def _own(c, s):
    from loopback_amd import block_ops
    if c["op"] == "ffn":
        return (block_ops.gated_ffn(s["x"], s["w_gate_up"], s["w_down"], activation=c["act"]),)
    if c["op"] == "dropout":
        return (block_ops.dropout(s["x"], c["p"], s["rng"], site=s["site"]),)
    h, n = block_ops.block_join(s["x"], s["y"], post_weight=s["post"], gate=s["gate"], scale=c["scale"], dropout=c["p"],
                                rng=s.get("rng"), site=s.get("site", 0), pre_weight=s["pre"], eps=EPS)
    return (h,) if n is None else (h, n)


def _upstream(c, s):
    if c["op"] == "join":
        return (s["dh"],) if s["pre"] is None else (s["dh"], s["dn"])
    return (s["dy"],)


def run(s: dict):
    """One forward; where the case trains, the gradients of every input too."""
    c = s["case"]
    if own:
        with torch.set_grad_enabled(c["train"]):
            out = _own(c, s)
            if not c["train"]:
                return out
            return (*(o.detach() for o in out), *torch.autograd.grad(out, [s[k] for k in s["leaves"]], _upstream(c, s)))
    dt = DTYPES[c["dtype"]]
    with torch.set_grad_enabled(c["train"]):
        v = {k: s[k].detach().float().requires_grad_(c["train"]) for k in s["leaves"]}
        out = _plain(c, s, v)
        got = [o.detach().to(dt) for o in out]
        if c["train"]:
            got += [g.to(dt) for g in torch.autograd.grad(out, list(v.values()), [g.float() for g in _upstream(c, s)])]
    return tuple(got)


def work(c: dict) -> dict:
    e, d = BYTES[c["dtype"]], c["d"]
    if c["op"] == "ffn":
        t, n = c["t"], c["n"]
        weights, rows = 3 * n * d, t * d
        if c["train"]:   # x, dy and the weights in; y, dx and the weights' gradients out
            return {"bytes": e * (4 * rows + 2 * weights), "flops": 18.0 * t * d * n}
        return {"bytes": e * (2 * rows + weights), "flops": 6.0 * t * d * n}
    if c["op"] == "dropout":
        rows = c["t"] * d
        return {"bytes": e * rows * (4 if c["train"] else 2), "flops": 2.0 * rows * (2 if c["train"] else 1)}
    rows = c["b"] * c["t"] * d
    gate = 0 if c["gate"] == "none" else math.prod(_gate_shape(c))
    vecs = d * (int(c["post"]) + int(c["pre"])) + gate
    if c["train"]:       # x, y, dh, dn in; h, n, dx, dy out; the vectors in, their gradients out
        return {"bytes": e * (rows * (8 if c["pre"] else 6) + 2 * vecs), "flops": 40.0 * rows}
    return {"bytes": e * (rows * (4 if c["pre"] else 3) + vecs), "flops": 14.0 * rows}


# -----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits: masks by numpy's unsigned words, gradients by their formulas
# -----------------------------------------------------------------------------------------------------------------------
def _exact_mask(s, c, rows):
    """0 where dropped, 1 / (1 - p) where kept (p as its 65536ths), fp64 (rows, d)."""
    import numpy as np
    d, nb = c["d"], (c["d"] + 7) // 8
    seed, step = (int(v) for v in s["rng"].cpu())
    u, m, half = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
    x0 = np.broadcast_to(np.arange(nb, dtype=u), (rows, nb)).copy()
    x1 = np.repeat(np.arange(rows, dtype=u), nb).reshape(rows, nb)
    x2, x3 = np.full((rows, nb), s["site"], u), np.full((rows, nb), step & 0xFFFFFFFF, u)
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for r in range(10):
        ka, kb = u((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), u((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        p, q = x0 * u(0xD2511F53), x2 * u(0xCD9E8D57)
        x0, x1, x2, x3 = (q >> half) ^ x1 ^ ka, q & m, (p >> half) ^ x3 ^ kb, p & m
    words = np.stack((x0, x1, x2, x3), -1).astype("<u4").view("<u2").reshape(rows, 8 * nb)[:, :d]
    drop = int(round(65536 * c["p"]))
    kept = torch.from_numpy(np.ascontiguousarray(words >= drop)).to(s["rng"].device)
    return kept.double() * (65536.0 / (65536.0 - drop))


def _norm64(v):
    r = (v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS).pow(-0.5)
    return v * r, r


def _norm64_grad(g, vh, r):
    return r * (g - vh * (g * vh).sum(-1, keepdim=True) / vh.shape[-1])


def exact(c: dict, seed: int):
    s = prepare(c, seed)
    f = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    with torch.no_grad():
        if c["op"] == "ffn":
            n = c["n"]
            wg, wu, wd = f["w_gate_up"][:n].contiguous(), f["w_gate_up"][n:].contiguous(), f["w_down"]
            g, u = f["x"].matmul(wg.T), f["x"].matmul(wu.T)
            if c["act"] == "silu":
                sg = torch.sigmoid(g)
                a, da = g * sg, sg * (1 + g * (1 - sg))
            else:
                k = math.sqrt(2 / math.pi)
                th = torch.tanh(k * (g + 0.044715 * g ** 3))
                a = 0.5 * g * (1 + th)
                da = 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g)
            y = (a * u).matmul(wd.T)
            if not c["train"]:
                return (y,)
            dact = f["dy"].matmul(wd)
            dg, du = dact * u * da, dact * a
            return (y, dg.matmul(wg) + du.matmul(wu), torch.cat((dg.T.matmul(f["x"]), du.T.matmul(f["x"]))),
                    f["dy"].T.matmul(a * u))
        if c["op"] == "dropout":
            m = _exact_mask(s, c, c["t"])
            return (f["x"] * m, f["dy"] * m) if c["train"] else (f["x"] * m,)
        shape = f["x"].shape
        m = _exact_mask(s, c, c["b"] * c["t"]).view(shape) if c["p"] else torch.ones((), dtype=torch.float64, device="cuda")
        yh, r1 = _norm64(f["y"]) if c["post"] else (f["y"], None)
        w1 = f["post"] if c["post"] else torch.ones((), dtype=torch.float64, device="cuda")
        gate = f["gate"] if c["gate"] != "none" else torch.ones((), dtype=torch.float64, device="cuda")
        h = f["x"] + c["scale"] * gate * yh * w1 * m
        hh, r2 = _norm64(h) if c["pre"] else (None, None)
        out = (h, hh * f["pre"]) if c["pre"] else (h,)
        if not c["train"]:
            return out
        dh = f["dh"] + _norm64_grad(f["dn"] * f["pre"], hh, r2) if c["pre"] else f["dh"]
        dz = c["scale"] * m * dh
        t = dz * gate
        grads = [dh, _norm64_grad(t * w1, yh, r1) if c["post"] else t]
        if c["post"]:
            grads.append((t * yh).sum((0, 1)))
        if c["gate"] != "none":
            dgate = dz * yh * w1
            grads.append({"column": lambda: dgate.sum((0, 1)), "sequence": lambda: dgate.sum(1, keepdim=True),
                          "full": lambda: dgate}[c["gate"]]())
        if c["pre"]:
            grads.append((f["dn"] * hh).sum((0, 1)))
        return (*out, *grads)
