"""Measured cases of the row operators: layer norm, 8-bit activation checkpoints, rotary positions
and the quantised key/value cache.

Every case runs in two forms.  With ``own`` false, ``run`` computes the operator from elementary
torch operations in binary32 (angles in binary64) and rounds once at the end; with ``own`` true it
makes the calls a program makes of this package.  torch tensors are row-major, the package's arrays
column-major, so a torch tensor of shape (rows, d) and an array of dims (d, rows) share one memory
layout: the first array dimension is the last torch dimension.

8-bit form of a row: blocks of 32 neighbours share one scale byte e (the scale is 2^(e-127), the
smallest power of two, at least 2^-127, that brings the block's largest magnitude to 127 for
"int8" or to 448 for "e4m3"); a code is the value over the scale, rounded to nearest, ties to even.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5
# bits of the mantissa above which the exponent goes up by one, and the exponent of the largest code
FORMATS = {"int8": (0x7FFFFF - 0x7E0000, 6), "e4m3": (0x7FFFFF - 0x600000, 8)}


# ---- the cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # layer norm of one decode batch: 16 tokens in flight, latency counts
        {"name": "norm decode 16x2048", "op": "norm", "direction": "forward", "rows": 16, "d": 2048, "type": "bf16", "params": "f32"},
        # a width that is no multiple of any vector, as a trimmed or concatenated feature has
        {"name": "norm odd 4099x1023", "op": "norm", "direction": "forward", "rows": 4099, "d": 1023, "type": "f16", "params": "same"},
        # gradient of a small model trained in binary32
        {"name": "norm grad 777x768", "op": "norm", "direction": "backward", "rows": 777, "d": 768, "type": "f32", "params": "f32"},
        # gradient in a training step: eight sequences of 2048 tokens, the largest of the set by rows
        {"name": "norm grad 16384x4096", "op": "norm", "direction": "backward", "rows": 16384, "d": 4096, "type": "bf16", "params": "f32"},
        # layer norm of a training step that keeps its normalised rows in 8 bits for the gradient
        {"name": "ckpt norm 8192x5120", "op": "checkpoint", "through": "norm", "rows": 8192, "d": 5120, "type": "bf16", "format": "int8"},
        # activation of a small odd feed-forward layer, kept as e4m3
        {"name": "ckpt gelu 333x1000", "op": "checkpoint", "through": "gelu", "rows": 333, "d": 1000, "type": "f16", "format": "e4m3"},
        # gated activation of a large feed-forward layer: both halves kept in 8 bits
        {"name": "ckpt gated 8192x8192", "op": "checkpoint", "through": "silu gated", "rows": 8192, "d": 8192, "type": "bf16", "format": "int8"},
        # queries and keys of a decode batch at far positions of a stretched context, part of the head rotated
        {"name": "rotary decode far", "op": "rotary", "tokens": 48, "q_heads": 16, "kv_heads": 4, "d": 96, "rot": 64,
         "layout": "interleaved", "scaling": "yarn", "far": 1 << 20, "type": "f16", "adjoint": False},
        # gradient of the rotation in a binary32 training step
        {"name": "rotary grad 4096 f32", "op": "rotary", "tokens": 4096, "q_heads": 12, "kv_heads": 12, "d": 64, "rot": 64,
         "layout": "half", "scaling": "none", "far": 2048, "type": "f32", "adjoint": True},
        # queries and keys of packed prompts, read out of the fused projection
        {"name": "rotary prompt 16384", "op": "rotary", "tokens": 16384, "q_heads": 32, "kv_heads": 8, "d": 128, "rot": 128,
         "layout": "half", "scaling": "linear", "far": 32768, "type": "bf16", "adjoint": False},
        # one token for each of 16 short sequences joins the cache, the contexts are read back
        {"name": "cache decode 16x512", "op": "cache", "seqs": 16, "ctx": 512, "new": 1, "heads": 4, "d": 64, "page": 16,
         "layout": "half", "type": "bf16", "format": "int8"},
        # a chunk of prompt for each of 8 long sequences
        {"name": "cache chunk 8x16384", "op": "cache", "seqs": 8, "ctx": 16384, "new": 1024, "heads": 8, "d": 128, "page": 64,
         "layout": "half", "type": "bf16", "format": "e4m3"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "checkpoint", "checkpoint", "rotary", "cache"])
    if op in ("norm", "checkpoint"):
        d = _log(rng, 64, 16384)
        d = d if rng.random() < 0.4 else max(64, d // 64 * 64)
        rows = _log(rng, 1, (1 << 26) // d)
        if op == "norm":
            return {"op": op, "direction": rng.choice(["forward", "backward"]), "rows": rows, "d": d,
                    "type": rng.choice(["bf16", "f16", "f32"]), "params": rng.choice(["f32", "same"])}
        return {"op": op, "through": rng.choice(["norm", "silu", "gelu", "silu gated", "gelu gated"]), "rows": rows, "d": d,
                "type": rng.choice(["bf16", "f16"]), "format": rng.choice(["int8", "e4m3"])}
    if op == "rotary":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        kv = rng.choice([1, 2, 4, 8])
        q = kv * rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, (1 << 26) // (d * (q + 2 * kv))), "q_heads": q, "kv_heads": kv, "d": d,
                "rot": rng.choice([d, d // 2, 2 * (d // 6)]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "far": _log(rng, 128, 1 << 20),
                "type": rng.choice(["bf16", "f16", "f32"]), "adjoint": rng.random() < 0.4}
    d, heads, seqs = rng.choice([64, 72, 96, 128, 256]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 64)
    ctx = _log(rng, 16, max(17, (1 << 26) // (d * heads * seqs * 2)))
    return {"op": op, "seqs": seqs, "ctx": ctx, "new": rng.choice([1, 1, max(1, ctx // 16), max(1, ctx // 4)]), "heads": heads,
            "d": d, "page": rng.choice([16, 32, 64, 128]), "layout": rng.choice(["half", "interleaved"]),
            "type": rng.choice(["bf16", "f16"]), "format": rng.choice(["int8", "e4m3"])}


# ---- inputs ------------------------------------------------------------------------------------------
_package = None


def _pkg():
    """This repository's package, working on torch's stream."""
    global _package
    if _package is None:
        import __graft_entry__
        _package = __graft_entry__.load_package()
        _package.device_(torch.cuda.current_device())
        _package.stream_(_package.Stream.wrap(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream))
    return _package


class _Shared:
    """An array's memory for torch; the tensor keeps the array alive."""

    def __init__(self, array, shape, kind):
        self.array = array
        self.__cuda_array_interface__ = {"data": (array.ptr, False), "shape": shape, "typestr": kind, "version": 3}


def _keep(s, name, value):
    """Puts a tensor into the state; the package's own arrays hold the memory where they are used."""
    t = value.contiguous()
    if own:
        p = _pkg()
        kinds = {torch.bfloat16: ("<i2", p._lib.bfloat16), torch.float16: ("<f2", np.float16), torch.float32: ("<f4", np.float32),
                 torch.int8: ("|i1", np.int8), torch.uint8: ("|u1", np.uint8), torch.int32: ("<i4", np.int32)}
        kind, dtype = kinds[t.dtype]
        a = p.ROCArray(dtype, tuple(reversed(t.shape)))
        u = torch.as_tensor(_Shared(a, tuple(t.shape), kind), device=DEVICE).view(t.dtype)
        u.copy_(t)
        s["array"][name] = a
        t = u
    s[name] = t


def _rows(rows, d, g, device=DEVICE):
    """Rows as a residual stream has them: an offset and a scale of each row, a few wide channels."""
    x = torch.randn(rows, d, generator=g, device=device)
    x *= 0.5 + 2.0 * torch.rand(rows, 1, generator=g, device=device)
    x += 0.3 + 0.5 * torch.rand(rows, 1, generator=g, device=device)
    x[:, :: max(1, d // 5)] *= 6.0
    return x


def _frequencies(rot, scaling):
    """Angles per position of the rot/2 pairs, binary64, and the factor on cosine and sine."""
    base, stretch, length = 10000.0, 8.0, 4096.0
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEVICE)
    if scaling == "ntk":
        base = base * stretch ** (rot / (rot - 2.0))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / stretch, 1.0
    if scaling == "yarn":                       # YaRN (Peng et al. 2023): mixed by the turns over the original length
        keep = ((length * f / (2.0 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / stretch * (1.0 - keep), 0.1 * math.log(stretch) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    s = {"case": case, "array": {}}
    t = TYPES[case["type"]]
    if case["op"] in ("norm", "checkpoint"):
        rows, d = case["rows"], case["d"]
        norm = case["op"] == "norm" or case["through"] == "norm"
        x = _rows(rows, d, g) if norm else 1.5 * torch.randn(rows, d, generator=g, device=DEVICE)
        _keep(s, "x", x.to(t))
        p = torch.float32 if case.get("params") == "f32" else t
        if norm:
            _keep(s, "gamma", (1.0 + 0.2 * torch.randn(d, generator=g, device=DEVICE)).to(p))
            _keep(s, "beta", (0.1 * torch.randn(d, generator=g, device=DEVICE)).to(p))
        if "gated" in case.get("through", ""):
            _keep(s, "gate", torch.randn(rows, d, generator=g, device=DEVICE).to(t))
            _keep(s, "dgate", torch.zeros(rows, d, dtype=t, device=DEVICE))
        train = case["op"] == "checkpoint" or case["direction"] == "backward"
        if train:
            _keep(s, "dy", torch.randn(rows, d, generator=g, device=DEVICE).to(t))
            _keep(s, "dx", torch.zeros(rows, d, dtype=t, device=DEVICE))
            if norm:
                _keep(s, "dgamma", torch.zeros(d, dtype=p, device=DEVICE))
                _keep(s, "dbeta", torch.zeros(d, dtype=p, device=DEVICE))
        if case["op"] == "checkpoint" or not train:
            _keep(s, "y", torch.zeros(rows, d, dtype=t, device=DEVICE))
        if norm:
            mean = torch.zeros(rows, device=DEVICE)
            rstd = torch.zeros(rows, device=DEVICE)
            if case["op"] == "norm" and train:  # what the forward pass of that step has kept
                xd = s["x"].double()
                mean = xd.mean(1).float()
                rstd = (xd.var(1, unbiased=False) + EPS).rsqrt().float()
            _keep(s, "mean", mean)
            _keep(s, "rstd", rstd)
        if own and case["op"] == "checkpoint":
            s["kept"] = _pkg().Quantized8((d, rows), case["format"])
            if "gate" in s:
                s["kept_gate"] = _pkg().Quantized8((d, rows), case["format"])
        return s
    rot = case.get("rot", case["d"])
    s["freq"], s["factor"] = _frequencies(rot, case.get("scaling", "none"))
    if own:
        s["plan"] = _pkg().rotary_plan(rot, layout=case["layout"], scaling=case.get("scaling", "none"), stretch=8.0, original_length=4096)
    if case["op"] == "rotary":
        n, q, kv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["d"]
        _keep(s, "qkv", torch.randn(n, q + 2 * kv, d, generator=g, device=DEVICE).to(t))
        # packed sequences: positions run up from a start of each sequence
        run = max(1, min(n, case["far"] // 2))
        starts = torch.randint(0, max(1, case["far"] - run), (n // run + 1,), generator=g, device=DEVICE)
        i = torch.arange(n, device=DEVICE)
        _keep(s, "positions", (starts[i // run] + i % run).int())
        _keep(s, "q", torch.zeros(n, q, d, dtype=t, device=DEVICE))
        _keep(s, "k", torch.zeros(n, kv, d, dtype=t, device=DEVICE))
        if own:                                 # views of the projection, as the program that made it holds them
            a = s["array"]["qkv"]
            s["q_in"] = a.subview(slice(None), slice(0, q), slice(None))
            s["k_in"] = a.subview(slice(None), slice(q, q + kv), slice(None))
        return s
    seqs, ctx, new, heads, d, page = (case[k] for k in ("seqs", "ctx", "new", "heads", "d", "page"))
    low = torch.rand(seqs, generator=g, device=DEVICE)
    lengths = (new + (ctx - new) * low).long().clamp(new, ctx)
    lengths[0] = ctx
    lengths = lengths.cpu()
    need = (lengths + page - 1) // page
    most, total = -(-ctx // page), int(need.sum())
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)) + 1
    at = torch.arange(most)[None, :]
    first = torch.cumsum(need, 0) - need
    pages = torch.where(at < need[:, None], order[(first[:, None] + at).clamp(max=total - 1)], 0)
    token = lengths[:, None] - new + torch.arange(new)[None, :]
    slots = (torch.gather(pages, 1, token // page) - 1) * page + token % page + 1
    _keep(s, "pages", pages.int().to(DEVICE))
    _keep(s, "lengths", lengths.int().to(DEVICE))
    _keep(s, "slots", slots.reshape(-1).int().to(DEVICE))
    _keep(s, "positions", token.reshape(-1).int().to(DEVICE))
    for name in ("k", "v"):
        past = torch.randn(total * page, heads, d, generator=g, device=DEVICE)
        codes, scales = _quantize(past, case["format"])
        del past
        _keep(s, name + "_codes", codes.reshape(total, page, heads, d))
        _keep(s, name + "_scales", scales.reshape(total, page, heads, -1))
        _keep(s, name + "_new", torch.randn(seqs * new, heads, d, generator=g, device=DEVICE).to(t))
        _keep(s, name + "_out", torch.zeros(seqs, ctx, heads, d, dtype=t, device=DEVICE))
    if own:
        p, a = _pkg(), s["array"]
        s["cache"] = p.QuantizedCache(p.Quantized8.wrap(a["k_codes"], a["k_scales"]), p.Quantized8.wrap(a["v_codes"], a["v_scales"]))
    return s


# ---- plain forms -------------------------------------------------------------------------------------
def _blocks(x):
    """(..., d) as (..., blocks, 32), the last block filled up with zeros."""
    d = x.shape[-1]
    n = -(-d // 32)
    return torch.nn.functional.pad(x, (0, n * 32 - d)).reshape(*x.shape[:-1], n, 32)


def _quantize(x, form):
    """binary32 rows to codes (int8, or the bytes of e4m3) and scale bytes."""
    up, top = FORMATS[form]
    b = _blocks(x)
    e = (((b.abs().amax(-1).view(torch.int32) + up) >> 23) - top).clamp(min=0)
    v = (b * torch.ldexp(torch.ones_like(e, dtype=torch.float32), 127 - e)[..., None]).flatten(-2)[..., : x.shape[-1]]
    codes = v.round().to(torch.int8) if form == "int8" else v.to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, e.to(torch.uint8)


def _restore(codes, scales):
    """binary32 rows that codes and scale bytes stand for."""
    v = codes.float() if codes.dtype == torch.int8 else codes.view(torch.float8_e4m3fn).float()
    two = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (_blocks(v) * two[..., None]).flatten(-2)[..., : v.shape[-1]]


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = ((c * c).mean(1, keepdim=True) + EPS).rsqrt()
    hat = c * rstd
    return hat, mean[:, 0], rstd[:, 0], (hat * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype)


def _plain_norm_grad(s, hat, rstd):
    dy = s["dy"].float()
    g = dy * s["gamma"].float()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * hat).sum(0).to(s["gamma"].dtype), "dbeta": dy.sum(0).to(s["gamma"].dtype)}


def _act(name, a):
    """An activation and its derivative; gelu in its tanh form."""
    if name == "silu":
        q = torch.sigmoid(a)
        return a * q, q * (1.0 + a * (1.0 - q))
    c = math.sqrt(2.0 / math.pi)
    q = torch.sigmoid(2.0 * c * (a + 0.044715 * a * a * a))      # (1 + tanh u)/2 = sigmoid(2u)
    return a * q, q + a * q * (1.0 - q) * 2.0 * c * (1.0 + 3.0 * 0.044715 * a * a)


def _turn(x, cos, sin, rot, layout):
    """Rotates the first `rot` of the last dimension, pairs (i, i+rot/2) or (2i, 2i+1)."""
    h = x[..., :rot]
    if layout == "half":
        a, b = h[..., : rot // 2], h[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)
    a, b = h[..., 0::2], h[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rot:]], -1)


def _angles(s):
    return (s["positions"].double()[:, None] * s["freq"][None, :])[:, None, :]


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        if case["direction"] == "forward":
            _, mean, rstd, y = _plain_norm(s)
            return {"y": y, "mean": mean, "rstd": rstd}
        return _plain_norm_grad(s, (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None], s["rstd"])
    if case["op"] == "checkpoint":
        if case["through"] == "norm":
            hat, _, rstd, y = _plain_norm(s)
            return {"y": y, "rstd": rstd, **_plain_norm_grad(s, _restore(*_quantize(hat, case["format"])), rstd)}
        t, name = s["x"].dtype, case["through"].split()[0]
        y = _act(name, s["x"].float())[0]
        f, df = _act(name, _restore(*_quantize(s["x"].float(), case["format"])))
        if "gate" not in s:
            return {"y": y.to(t), "dx": (s["dy"].float() * df).to(t)}
        g = _restore(*_quantize(s["gate"].float(), case["format"]))
        return {"y": (y * s["gate"].float()).to(t), "dx": (s["dy"].float() * g * df).to(t), "dgate": (s["dy"].float() * f).to(t)}
    a = _angles(s)
    cos, sin = (a.cos() * s["factor"]).float(), (a.sin() * s["factor"]).float()
    if case["op"] == "rotary":
        q, kv, t = case["q_heads"], case["kv_heads"], s["qkv"].dtype
        r = _turn(s["qkv"][:, : q + kv].float(), cos, -sin if case["adjoint"] else sin, case["rot"], case["layout"]).to(t)
        return {"q": r[:, :q], "k": r[:, q:]}
    slots = s["slots"].long() - 1
    out = {}
    for name in ("k", "v"):
        x = s[name + "_new"].float()
        codes, scales = _quantize(_turn(x, cos, sin, case["d"], case["layout"]) if name == "k" else x, case["format"])
        s[name + "_codes"].flatten(0, 1)[slots] = codes
        s[name + "_scales"].flatten(0, 1)[slots] = scales
        at = torch.arange(case["ctx"], device=DEVICE)
        page = (s["pages"].long() - 1).clamp(min=0)[:, at // case["page"]]
        row = page * case["page"] + at % case["page"]
        v = _restore(s[name + "_codes"].flatten(0, 1)[row], s[name + "_scales"].flatten(0, 1)[row]).to(s[name + "_out"].dtype)
        out[name] = torch.where((at[None, :] < s["lengths"][:, None])[..., None, None], v, s[name + "_out"])
    return out


# ---- the package's calls -----------------------------------------------------------------------------
def _calls(s):
    case, p, a = s["case"], _pkg(), s["array"]
    if case["op"] == "norm":
        if case["direction"] == "forward":
            p.layernorm_(a["y"], a["x"], a["gamma"], a["beta"], eps=EPS, mean=a["mean"], rstd=a["rstd"])
            return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
        p.layernorm_backward_(a["dx"], a["dy"], a["x"], a["gamma"], mean=a["mean"], rstd=a["rstd"], dgamma=a["dgamma"], dbeta=a["dbeta"])
        return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if case["op"] == "checkpoint":
        if case["through"] == "norm":
            p.layernorm_(a["y"], a["x"], a["gamma"], a["beta"], eps=EPS, rstd=a["rstd"], checkpoint=s["kept"])
            p.layernorm_backward_(a["dx"], a["dy"], s["kept"], a["gamma"], rstd=a["rstd"], dgamma=a["dgamma"], dbeta=a["dbeta"])
            return {"y": s["y"], "rstd": s["rstd"], "dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
        name = case["through"].split()[0]
        if "gate" not in s:
            p.activation_(name, a["y"], a["x"], checkpoint=s["kept"])
            p.activation_backward_(name, a["dx"], a["dy"], s["kept"])
            return {"y": s["y"], "dx": s["dx"]}
        p.activation_(name, a["y"], a["x"], a["gate"], checkpoint=s["kept"], gate_checkpoint=s["kept_gate"])
        p.activation_backward_(name, a["dx"], a["dy"], s["kept"], s["kept_gate"], dgate=a["dgate"])
        return {"y": s["y"], "dx": s["dx"], "dgate": s["dgate"]}
    if case["op"] == "rotary":
        p.rotary_(a["q"], s["q_in"], a["positions"], s["plan"], adjoint=case["adjoint"])
        p.rotary_(a["k"], s["k_in"], a["positions"], s["plan"], adjoint=case["adjoint"])
        return {"q": s["q"], "k": s["k"]}
    p.cache_write_(s["cache"], a["k_new"], a["v_new"], a["slots"], rotary=s["plan"], positions=a["positions"])
    p.cache_read_(a["k_out"], a["v_out"], s["cache"], a["pages"], a["lengths"])
    return {"k": s["k_out"], "v": s["v_out"]}


def run(state):
    return _calls(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    b = BYTES[case["type"]]
    if case["op"] in ("norm", "checkpoint"):
        n, d, rows = case["rows"] * case["d"], case["d"], case["rows"]
        if case["op"] == "norm":
            p = 4 if case["params"] == "f32" else b
            if case["direction"] == "forward":
                return {"bytes": 2 * n * b + 2 * d * p + 8 * rows, "flops": 8 * n}
            return {"bytes": 3 * n * b + 3 * d * p + 8 * rows, "flops": 14 * n}
        kept = n + rows * (-(-d // 32))         # written by the forward pass, read by the backward pass
        if case["through"] == "norm":
            return {"bytes": 4 * n * b + 2 * kept + 5 * d * b + 8 * rows, "flops": 26 * n}
        if "gated" in case["through"]:
            return {"bytes": 6 * n * b + 4 * kept, "flops": 40 * n}
        return {"bytes": 4 * n * b + 2 * kept, "flops": 30 * n}
    if case["op"] == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["d"] * b + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    row = case["heads"] * case["d"]
    kept = row + case["heads"] * (-(-case["d"] // 32))
    new = case["seqs"] * case["new"]
    read = case["ctx"] + (case["seqs"] - 1) * (case["new"] + (case["ctx"] - case["new"]) // 2)
    return {"bytes": 2 * (new * (row * b + kept) + read * (kept + row * b)) + 8 * new, "flops": 8 * new * row + 2 * read * row}


# ---- the definition in 64 bits -----------------------------------------------------------------------
def _exact_kept(x, form):
    """What the rows stand for once they have been through 8 bits, from the definition."""
    top = 127.0 if form == "int8" else 448.0
    d = x.shape[-1]
    n = -(-d // 32)
    b = torch.zeros(*x.shape[:-1], n * 32, dtype=torch.float64, device=x.device)
    b[..., :d] = x
    b = b.unflatten(-1, (n, 32))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))           # largest = m 2^e, 1/2 <= m < 1
    mt, et = math.frexp(top)
    k = (e - et + (m > mt).int()).clamp(min=-127)
    k = torch.where(m == 0, torch.full_like(k, -127), k)
    one = torch.ones_like(m)
    v = torch.ldexp(b, -k)
    if form == "int8":
        v = torch.round(v)
    else:
        step = torch.ldexp(one, (torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
        v = torch.round(v / step) * step
    return torch.ldexp(v, k).flatten(-2)[..., :d]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "checkpoint"):
        x = s["x"].double()
        norm = case["op"] == "norm" or case["through"] == "norm"
        if norm:
            gamma, beta = s["gamma"].double(), s["beta"].double()
            d = x.shape[1]
            if case["op"] == "norm" and case["direction"] == "backward":
                mean, rstd = s["mean"].double(), s["rstd"].double()
            else:
                mean = x.sum(1) / d
                rstd = 1.0 / torch.sqrt(((x - mean[:, None]) ** 2).sum(1) / d + EPS)
            hat = (x - mean[:, None]) * rstd[:, None]
            y = hat * gamma + beta
            if case["op"] == "norm" and case["direction"] == "forward":
                return {"y": y, "mean": mean, "rstd": rstd}
            if case["op"] == "checkpoint":
                hat = _exact_kept(hat, case["format"])
            dy = s["dy"].double()
            g = dy * gamma
            dx = rstd[:, None] * (g - g.sum(1, keepdim=True) / d - hat * ((g * hat).sum(1, keepdim=True) / d))
            r = {"dx": dx, "dgamma": (dy * hat).sum(0), "dbeta": dy.sum(0)}
            return r if case["op"] == "norm" else {"y": y, "rstd": rstd, **r}

        def f(a):
            if case["through"].startswith("silu"):
                return a / (1.0 + torch.exp(-a)), (1.0 + torch.exp(-a) * (1.0 + a)) / (1.0 + torch.exp(-a)) ** 2
            c = math.sqrt(2.0 / math.pi)
            th = torch.tanh(c * (a + 0.044715 * a ** 3))
            return 0.5 * a * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * a * a)

        kept, dy = _exact_kept(x, case["format"]), s["dy"].double()
        if "gate" not in s:
            return {"y": f(x)[0], "dx": dy * f(kept)[1]}
        gate = s["gate"].double()
        return {"y": f(x)[0] * gate, "dx": dy * _exact_kept(gate, case["format"]) * f(kept)[1], "dgate": dy * f(kept)[0]}
    rot = case.get("rot", case["d"])
    angle = (s["positions"].double()[:, None] * s["freq"])[:, None, :]
    wave = torch.polar(torch.full_like(angle, s["factor"]), -angle if case.get("adjoint") else angle)

    def turn(x):                                # the pairs as complex numbers, times e^(i angle)
        y = x.double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., : rot // 2], y[..., rot // 2: rot]) * wave
            y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
        else:
            z = torch.complex(y[..., 0:rot:2], y[..., 1:rot:2]) * wave
            y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
        return y

    if case["op"] == "rotary":
        q, kv = case["q_heads"], case["kv_heads"]
        return {"q": turn(s["qkv"][:, :q]), "k": turn(s["qkv"][:, q: q + kv])}
    out = {}
    l = torch.arange(case["ctx"], device=DEVICE)
    for name in ("k", "v"):
        new = s[name + "_new"]
        fresh = _exact_kept(turn(new) if name == "k" else new.double(), case["format"])
        codes = s[name + "_codes"]
        v = codes.double() if case["format"] == "int8" else codes.view(torch.float8_e4m3fn).double()
        e = s[name + "_scales"].int().repeat_interleave(32, -1)[..., : case["d"]]
        all_rows = torch.ldexp(v, e - 127).flatten(0, 1)
        all_rows[s["slots"].long() - 1] = fresh
        r = s[name + "_out"].double()
        for b, n in enumerate(s["lengths"].tolist()):
            r[b, :n] = all_rows[(s["pages"][b, l[:n] // case["page"]].long() - 1) * case["page"] + l[:n] % case["page"]]
        out[name] = r
    return out
