"""Operators of a serving step with 8-bit weights, rotated positions and a shared prompt, as a
serving program calls them: activations quantised in blocks, the product with weights held so, the
norms of queries and keys with their rotation, and attention over a prefix that all requests share.

A matrix in 8 bits is a pair: ``codes`` ``[rows, Kp]`` float8_e4m3fn with K rounded up to
``Kp``, a multiple of 128 (zeros past K), and ``scale`` ``[rows, S]`` float8_e8m0fnu, a power of
two for each 128 columns, S a multiple of 4 (ones past Kp / 128).  The cache is the one of
``perf/operators.py``: blocks of codes with one fp32 scale for each block and head.

A case is a dict of plain values:

``kind``        ``"quantize"``, ``"linear"``, ``"rope"`` or ``"prefix"``
``rows``, ``k``, ``n``  (quantize, linear) the activations' rows and columns, the product's columns
``dtype``       of the activations: ``"float16"``, ``"bfloat16"``
``codes``       (linear) the activations come quantised, as of a norm that several products share
``gelu``, ``resid``  (linear) GELU after the bias; an fp32 residual, and then an fp32 result
``heads``, ``kv_heads``, ``head_dim``  the attention's geometry
``norm``, ``rot``, ``inter``, ``far``  (rope) norms or none; rotated columns; pairs of neighbours or
                of halves; the largest position
``batch``, ``new_lo``, ``new_hi``, ``own_lo``, ``own_hi``, ``prefix``  (prefix) requests, new tokens and
                own tokens before them of each, tokens of the shared prefix
``block``, ``cache``, ``sharp``  (prefix) tokens of a block, the codes' type, the logits' deviation
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "cobra-gpu-kernel_amd")
if _PKG not in sys.path:
    sys.path.insert(1, _PKG)

_DEVICE = "cuda"
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3fn": torch.float8_e4m3fn,
           "int8": torch.int8}
_E4M3_MAX = 448.0
_WIDTHS = (32, 64, 96, 128, 192, 256)
_EPS = 1e-6
_THETA = 10000.0


def _quantize(rows, k, dtype="bfloat16"):
    return {"kind": "quantize", "rows": rows, "k": k, "dtype": dtype}


def _linear(rows, k, n, dtype="bfloat16", *, codes=False, gelu=False, resid=False):
    return {"kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "codes": codes, "gelu": gelu,
            "resid": resid}


def _rope(rows, heads, kv_heads, head_dim, dtype="bfloat16", *, norm=True, rot=None, inter=False, far=8191):
    return {"kind": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "norm": norm, "rot": head_dim if rot is None else rot, "inter": inter, "far": far}


def _prefix(batch, new, own_lens, prefix, heads, kv_heads, head_dim, block=64, *, dtype="bfloat16",
            cache="float8_e4m3fn", sharp=2.0):
    return {"kind": "prefix", "batch": batch, "new_lo": new[0], "new_hi": new[1], "own_lo": own_lens[0],
            "own_hi": own_lens[1], "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "block": block, "dtype": dtype, "cache": cache, "sharp": sharp}


def listed():
    cases = {
        # A server's step: one token of each of 64 requests, before the projections that share them.
        "quantize_b64": _quantize(64, 1024, "float16"),
        # The activations of a wide layer's prefill chunk.
        "quantize_chunk": _quantize(8192, 8192),
        # One token of one conversation through a narrow projection: a launch is all there is.
        "linear_one": _linear(1, 1024, 1024, "float16"),
        # A small batch through a wide layer's first feed-forward product: bound by the weights' bytes.
        "linear_b16": _linear(16, 4096, 8192, gelu=True),
        # Prompts of odd lengths through a layer whose sizes fit no tile, with the residual stream.
        "linear_odd": _linear(333, 1096, 1000, "float16", resid=True),
        # A prefill chunk through a wide layer: bound by the matrix cores.
        "linear_chunk": _linear(8192, 4096, 4096),
        # A server's step of a narrow model: queries and keys of 64 tokens.
        "rope_b64": _rope(64, 8, 8, 64, "float16"),
        # A prefill chunk with shared heads.
        "rope_chunk": _rope(16384, 32, 8, 128),
        # A server's ordinary step: short conversations behind one system prompt.
        "prefix_b64": _prefix(64, (1, 1), (10, 500), 1999, 8, 8, 64, dtype="float16"),
        # Many conversations about one long document, with shared heads.
        "prefix_long_gqa": _prefix(128, (1, 1), (100, 2000), 30000, 32, 8, 128),
        # A few draft tokens of each request are checked at once; wide heads, an int8 cache.
        "prefix_draft": _prefix(23, (2, 6), (0, 300), 4001, 6, 2, 256, 32, cache="int8"),
        # New prompts behind the shared one.
        "prefix_chunk": _prefix(4, (300, 1000), (0, 500), 9000, 16, 4, 64, dtype="float16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_GEOMETRY = ((4, 4, 32), (2, 1, 32), (6, 6, 40), (8, 8, 64), (16, 4, 64), (14, 2, 64), (12, 4, 80), (8, 4, 96),
             (32, 8, 128), (8, 1, 128), (20, 1, 128), (5, 5, 168), (6, 2, 256))


def draw(rng):
    """One more case of the same ranges, none larger than the listed largest of its kind."""
    kind = rng.choice(["quantize", "linear", "linear", "linear", "rope", "prefix", "prefix", "prefix"])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "quantize":
        k = _log(rng, 1, 8192)
        return _quantize(_log(rng, 1, 60_000_000 // k), k, dtype)
    if kind == "linear":
        k, n = _log(rng, 64, 8192), _log(rng, 64, 8192)
        few = rng.random() < 0.5
        rows = _log(rng, 1, 64) if few else _log(rng, 65, max(66, min(16384, 130_000_000_000 // (k * n))))
        return _linear(rows, k, n, dtype, codes=rng.random() < 0.3, gelu=rng.random() < 0.3, resid=rng.random() < 0.3)
    heads, kv, hd = rng.choice(_GEOMETRY)
    if kind == "rope":
        rot = rng.choice([hd, hd, hd // 2 // 2 * 2])
        return _rope(_log(rng, 1, max(1, 80_000_000 // ((heads + 2 * kv) * hd))), heads, kv, hd, dtype,
                     norm=rng.random() < 0.7, rot=rot, inter=rng.random() < 0.4, far=_log(rng, 1, 200000))
    new = (1, rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1000)]))
    own_hi = _log(rng, 1, 4000)
    prefix = _log(rng, 1, 60000)
    # the own caches below prefix_long_gqa's, the plain form's scores and the pairs small
    top = max(1, min(128, 200_000_000 // ((own_hi + new[1]) * kv * hd), 250_000_000 // ((prefix + own_hi) * heads * new[1])))
    return _prefix(_log(rng, 1, top), new, (rng.randint(0, own_hi), own_hi), prefix, heads, kv, hd,
                   rng.choice([16, 32, 64, 128]), dtype=dtype, cache=rng.choice(["float8_e4m3fn", "float8_e4m3fn", "int8"]),
                   sharp=round(rng.uniform(1.0, 3.0), 2))


# -- inputs -------------------------------------------------------------------------


def _up(n, m):
    return -(-n // m) * m


def _spread(lo, hi, n, phase):
    """n whole numbers over lo .. hi, the same for every seed (so that the work is the case's own)."""
    return [lo + int((hi - lo + 1) * ((phase + i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(case):
    """(own tokens before the call, new tokens) of each request."""
    return (_spread(case["own_lo"], case["own_hi"], case["batch"], 0.999999),
            _spread(case["new_lo"], case["new_hi"], case["batch"], 0.999999))


def _activations(rows, cols, g):
    """Rows of differing size with a few columns far above the others, as hidden states have them."""
    x = torch.randn(rows, cols, generator=g, device=_DEVICE)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=_DEVICE))
    x *= torch.where(torch.rand(1, cols, generator=g, device=_DEVICE) < 0.01, 20.0, 1.0)
    return x


def _contents(total, kv, bs, hd, cache, seen, g):
    """A pool's keys and values as appends leave them: magnitudes that differ from block to
    block, and memory that nobody wrote (NaN codes) where ``seen`` [total, bs] is false."""
    hdp = next(w for w in _WIDTHS if w >= hd)
    qmax = _E4M3_MAX if cache == "float8_e4m3fn" else 127.0
    out = []
    for _ in range(2):
        x = torch.randn(total, kv, bs, hd, generator=g, device=_DEVICE)
        x *= torch.exp(0.5 * torch.randn(total, kv, 1, 1, generator=g, device=_DEVICE)) * 0.7
        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / qmax)))
        x = (x / scale[:, :, None, None]).clamp(-qmax, qmax)
        x = torch.nn.functional.pad(x, (0, hdp - hd))
        code = (x.round().to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)).view(torch.uint8)
        code = torch.where(seen[:, None, :, None], code, torch.full_like(code, 0x80 if cache == "int8" else 0x7F))
        out += [code, scale]
    k, ks, v, vs = out
    return k.view(_DTYPES[cache]), ks, v.transpose(2, 3).contiguous().view(_DTYPES[cache]), vs


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    dt, kind = _DTYPES[case["dtype"]], case["kind"]
    if kind == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["k"], g).to(dt)}
    if kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s = {"case": case, "a": _activations(m, k, g).to(dt), "a_scale": None, "resid": None}
        s["w"], s["w_scale"] = _plain_quantize(torch.randn(n, k, generator=g, device=_DEVICE) * k ** -0.5)
        if case["codes"]:
            s["a"], s["a_scale"] = _plain_quantize(s["a"])
        s["bias"] = 0.1 * torch.randn(n, generator=g, device=_DEVICE)
        if case["resid"]:
            s["resid"] = torch.randn(m, n, generator=g, device=_DEVICE)
        return s
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        t, rot = case["rows"], case["rot"]
        s = {"case": case, "qkv": (torch.randn(t, (heads + 2 * kv) * hd, generator=g, device=_DEVICE) * 2.0).to(dt),
             "q_weight": None, "k_weight": None}
        s["pos"] = torch.randint(0, case["far"] + 1, (t,), generator=g, device=_DEVICE, dtype=torch.int32)
        if case["norm"]:
            s["q_weight"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=_DEVICE)
            s["k_weight"] = 1.0 + 0.2 * torch.randn(hd, generator=g, device=_DEVICE)
        turn = torch.arange(0, rot, 2, dtype=torch.float64, device=_DEVICE) / max(rot, 1)
        s["inv_freq"] = (_THETA ** -turn).float()
        return s
    # Row 0 of the tables is the prefix's, which has no new tokens; the call comes after the new
    # tokens' own append, so the cache holds them too.
    before, new = _lengths(case)
    held = [case["prefix"]] + [b + n for b, n in zip(before, new)]
    new = [0] + new
    bs = case["block"]
    need = [_up(h, bs) // bs for h in held]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=_DEVICE).to(torch.int32)
    width = max(need) + 1
    rows = torch.tensor(need, device=_DEVICE)
    col = torch.arange(width, device=_DEVICE)
    at = ((torch.cumsum(rows, 0) - rows)[:, None] + col).clamp(max=total - 1)
    table = torch.where(col < rows[:, None], order[at], torch.full_like(order[at], -1)).contiguous()
    lens = torch.tensor(held, dtype=torch.int32, device=_DEVICE)
    live = torch.arange(width * bs, device=_DEVICE).view(1, width, bs) < lens.view(-1, 1, 1)
    seen = torch.zeros(total + 1, bs, dtype=torch.bool, device=_DEVICE)
    seen[torch.where(table >= 0, table, torch.full_like(table, total)).long().view(-1)] = live.view(-1, bs)
    k, ks, v, vs = _contents(total, kv, bs, hd, case["cache"], seen[:total], g)
    qkv = torch.randn(sum(new), (heads + 2 * kv) * hd, generator=g, device=_DEVICE)
    qkv[:, : heads * hd] *= case["sharp"] * 1.2
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=_DEVICE)
    return {"case": case, "qkv": qkv.to(dt), "cu": cu, "lens": lens, "table": table, "k": k, "ks": ks, "v": v,
            "vs": vs, "max_new": max(new), "max_len": max(held[1:]), "scale": hd ** -0.5}


# -- one pass -----------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "quantize":
        codes, scale = _own_quantize(state) if own else _plain_quantize(state["x"])
        return {"codes": codes, "exponent": scale.view(torch.uint8)}
    if kind == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    if kind == "rope":
        if own:
            _own_rope(state)
        else:
            _plain_rope(state)
        return state["qkv"]
    return _own_prefix(state) if own else _plain_prefix(state)


def _own_quantize(s):
    from cobra_amd import ops

    return ops.quantize8(s["x"])


def _own_linear(s):
    from cobra_amd import ops

    c = s["case"]
    out = torch.float32 if c["resid"] else _DTYPES[c["dtype"]]
    return ops.linear8(s["a"], s["w"], s["w_scale"], s["bias"], gelu=c["gelu"], out_dtype=out, resid=s["resid"],
                       a_scale=s["a_scale"])


def _own_rope(s):
    from cobra_amd import ops

    c = s["case"]
    ops.qk_norm_rope(s["qkv"], c["heads"], c["kv_heads"], c["head_dim"], positions=s["pos"], inv_freq=s["inv_freq"],
                     q_weight=s["q_weight"], k_weight=s["k_weight"], interleaved=c["inter"], eps=_EPS)


def _own_prefix(s):
    from cobra_amd import ops

    c = s["case"]
    return ops.cache_prefix_attn(s["qkv"], s["cu"], s["lens"], s["table"], 0, c["heads"], c["head_dim"], s["scale"],
                                 s["k"], s["v"], s["ks"], s["vs"], max_new=s["max_new"], max_len=s["max_len"],
                                 max_prefix=c["prefix"])


def _plain_quantize(x):
    """Rows in blocks of 128 columns: the least power of two that brings a block within e4m3's
    range (exact: frexp and compare), and the nearest codes."""
    m, k = x.shape
    kp, s4 = _up(k, 128), _up(k, 512) // 128
    x = torch.nn.functional.pad(x.float(), (0, kp - k)).view(m, kp // 128, 128)
    amax = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(2)
    frac, e = torch.frexp(amax)  # amax = frac 2^e, 1/2 <= frac < 1; 448 = 7/8 2^9
    e = torch.where(frac <= 0.875, e - 9, e - 8).clamp(min=-126)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    codes = torch.ldexp(x, -e[:, :, None]).to(torch.float8_e4m3fn).view(m, kp)
    scale = torch.full((m, s4), 127, dtype=torch.uint8, device=x.device)
    scale[:, : kp // 128] = (e + 127).to(torch.uint8)
    return codes, scale.view(torch.float8_e8m0fnu)


def _values(codes, scale):
    m, kp = codes.shape
    e = scale.view(torch.uint8)[:, : kp // 128].int() - 127
    return torch.ldexp(codes.float().view(m, kp // 128, 128), e[:, :, None]).view(m, kp)


def _plain_linear(s):
    c = s["case"]
    a, scale = (s["a"], s["a_scale"]) if c["codes"] else _plain_quantize(s["a"])
    y = torch.matmul(_values(a, scale), _values(s["w"], s["w_scale"]).t()) + s["bias"]
    if c["gelu"]:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y + s["resid"] if c["resid"] else y.to(_DTYPES[c["dtype"]])


def _plain_rope(s):
    c = s["case"]
    heads, kv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rot"]
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    for first, n, w in ((0, heads, s["q_weight"]), (heads, kv, s["k_weight"])):
        x = s["qkv"][:, first * hd:(first + n) * hd].float().view(-1, n, hd)
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["inter"] else (x[..., : rot // 2], x[..., rot // 2:rot])
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1 if c["inter"] else -2).reshape(*x.shape[:2], rot)
        s["qkv"][:, first * hd:(first + n) * hd] = torch.cat((y, x[..., rot:]), -1).view(-1, n * hd).to(s["qkv"].dtype)


def _plain_prefix(s):
    c = s["case"]
    heads, kv, hd, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]
    lens, cu, dev = s["lens"][1:], s["cu"][1:], s["cu"].device
    bsz, group, held = c["batch"], heads // kv, c["prefix"]

    def values(codes, scale, tab, order, n):
        """[requests, kv, tokens, hd] of the blocks that tab lists, zeros from token n on."""
        x = codes.view(torch.uint8)[tab].view(codes.dtype).float() * scale[tab][..., None, None]
        x = x.permute(order).reshape(tab.shape[0], kv, tab.shape[1] * bs, -1)[..., :hd]
        there = torch.arange(x.shape[2], device=dev)[None, :] < n
        return torch.where(there[:, None, :, None], x, torch.zeros_like(x))

    pre = s["table"][:1, : -(-held // bs)].long()
    tab = s["table"][1:, : -(-s["max_len"] // bs)].clamp(min=0).long()
    pk = values(s["k"], s["ks"], pre, (0, 2, 1, 3, 4), held)[0, :, :held]
    pv = values(s["v"], s["vs"], pre, (0, 2, 1, 4, 3), held)[0, :, :held]
    k = values(s["k"], s["ks"], tab, (0, 2, 1, 3, 4), lens[:, None])
    v = values(s["v"], s["vs"], tab, (0, 2, 1, 4, 3), lens[:, None])
    # Rows of every request to its most new tokens: [batch, kv, group, new, hd].
    i = torch.arange(s["max_new"], device=dev)
    row = (cu[:-1, None] + i).clamp(max=s["qkv"].shape[0] - 1).long()
    q = s["qkv"][:, : heads * hd].float()[row].view(bsz, s["max_new"], kv, group, hd).permute(2, 0, 3, 1, 4)
    rows = group * s["max_new"]
    far = torch.matmul(q.reshape(kv, bsz * rows, hd), pk.transpose(1, 2).contiguous()) * s["scale"]
    far = far.view(kv, bsz, group, s["max_new"], held)
    near = torch.matmul(q.transpose(0, 1).reshape(bsz, kv, rows, hd), k.transpose(2, 3).contiguous()) * s["scale"]
    near = near.view(bsz, kv, group, s["max_new"], -1).transpose(0, 1)
    last = lens[:, None] - (cu[1:] - cu[:-1])[:, None] + i
    seen = torch.arange(near.shape[-1], device=dev) <= torch.minimum(last, lens[:, None] - 1)[:, :, None]
    near = near.masked_fill(~seen[None, :, None], -math.inf)
    top = torch.maximum(far.amax(-1), near.amax(-1))[..., None]
    far, near = torch.exp(far - top), torch.exp(near - top)
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    o = torch.matmul(far.view(kv, bsz * rows, held), pv).view(kv, bsz, group, s["max_new"], hd)
    mine = torch.matmul(near.transpose(0, 1).reshape(bsz, kv, rows, -1), v)
    o = (o + mine.view(bsz, kv, group, s["max_new"], hd).transpose(0, 1)) / total
    t = torch.arange(s["qkv"].shape[0], device=dev)
    b = torch.searchsorted(cu[1:], t.int(), right=True)
    return o.permute(1, 3, 0, 2, 4)[b, t - cu[b]].reshape(-1, heads * hd).to(s["qkv"].dtype)


# -- the work of a pass, and its exact result ------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        m, k = case["rows"], case["k"]
        return {"bytes": m * (2 * k + _up(k, 128) + _up(k, 512) // 128), "flops": 0}
    if kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        in8 = _up(k, 128) + _up(k, 512) // 128
        return {"bytes": m * (in8 if case["codes"] else 2 * k) + n * (in8 + 4) + m * n * (8 if case["resid"] else 2),
                "flops": 2 * m * n * k}
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        cols = hd if case["norm"] else case["rot"]
        return {"bytes": case["rows"] * ((heads + kv) * cols * 4 + 4) + case["rot"] * 2 + (8 * hd if case["norm"] else 0),
                "flops": 0}
    before, new = _lengths(case)
    bs = case["block"]
    pairs = sum(n * (case["prefix"] + b) + n * (n + 1) // 2 for b, n in zip(before, new))
    held = [case["prefix"]] + [b + n for b, n in zip(before, new)]
    pages = sum(_up(h, bs) // bs for h in held)
    return {"bytes": sum(held) * kv * hd * 2 + pages * (4 + kv * 8) + 4 * sum(new) * heads * hd + 8 * len(held),
            "flops": 4 * pairs * heads * hd}


def exact(case, seed):
    """The results in 64 bits."""
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "linear": _exact_linear, "rope": _exact_rope, "prefix": _exact_prefix}[
        case["kind"]](s)


def _blocks_of(x):
    """([rows, blocks, 128] values, [rows, blocks] exponents) in 64 bits: the exponent by
    counting up from the logarithm's floor until the block fits."""
    m, k = x.shape
    z = torch.zeros(m, _up(k, 128), dtype=torch.float64, device=x.device)
    z[:, :k] = x.double()
    z = z.view(m, -1, 128)
    big = z.abs().amax(2)
    e = torch.floor(torch.log2(big.clamp(min=2.0 ** -300) / 448)) - 1
    for _ in range(3):
        e = torch.where(big > 448 * torch.exp2(e), e + 1, e)
    return z, e.clamp(min=-126.0)


def _nearest(x):
    """The nearest e4m3 value, ties to the even one: 4 significant bits, steps of 2^-9 at least."""
    step = torch.exp2((torch.frexp(x)[1].double() - 4).clamp(min=-9.0))
    return torch.round(x / step) * step


def _exact_quantize(s):
    z, e = _blocks_of(s["x"])
    scale = torch.full((z.shape[0], _up(z.shape[1], 4)), 127, dtype=torch.uint8, device=z.device)
    scale[:, : z.shape[1]] = (e + 127).to(torch.uint8)
    return {"codes": _nearest(z / torch.exp2(e)[:, :, None]).view(z.shape[0], -1), "exponent": scale}


def _exact_linear(s):
    c = s["case"]

    def held(codes, scale):
        z = codes.float().double().view(codes.shape[0], -1, 128)
        return (z * torch.exp2(scale.view(torch.uint8)[:, : z.shape[1]].double() - 127)[:, :, None]).view(codes.shape)

    if c["codes"]:
        a = held(s["a"], s["a_scale"])
    else:
        z, e = _blocks_of(s["a"])
        p = torch.exp2(e)[:, :, None]
        a = (_nearest(z / p) * p).view(z.shape[0], -1)
    w = held(s["w"], s["w_scale"])
    y = a @ w.T + s["bias"].double()
    if c["gelu"]:
        y = y * torch.special.erfc(-y / math.sqrt(2.0)) / 2
    return y + s["resid"].double() if c["resid"] else y


def _exact_rope(s):
    """Pairs as complex numbers."""
    c = s["case"]
    heads, kv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rot"]
    out = s["qkv"].double()
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)
    for head in range(heads + kv):
        x = out[:, head * hd:(head + 1) * hd]
        if c["norm"]:
            w = s["q_weight"] if head < heads else s["k_weight"]
            x = x / torch.sqrt(x.square().sum(1, keepdim=True) / hd + _EPS) * w.double()
        if rot:
            i = torch.arange(rot // 2, device=x.device)
            re, im = (2 * i, 2 * i + 1) if c["inter"] else (i, i + rot // 2)
            z = torch.complex(x[:, re], x[:, im]) * turn
            x = x.clone()
            x[:, re], x[:, im] = z.real, z.imag
        out[:, head * hd:(head + 1) * hd] = x
    return out


def _exact_prefix(s):
    """Request by request, head by head: one softmax over the prefix's keys and its own."""
    c = s["case"]
    heads, kv, hd, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    group = heads // kv
    out = torch.zeros(s["qkv"].shape[0], heads * hd, dtype=torch.float64, device=s["qkv"].device)

    def held(b, h):
        n = lens[b]
        pages = s["table"][b, : _up(n, bs) // bs].long()
        k = s["k"].view(torch.uint8)[pages, h].view(s["k"].dtype).double() * s["ks"][pages, h].double()[:, None, None]
        v = s["v"].view(torch.uint8)[pages, h].view(s["v"].dtype).double() * s["vs"][pages, h].double()[:, None, None]
        return k.reshape(-1, k.shape[-1])[:n, :hd], v.transpose(1, 2).reshape(-1, v.shape[1])[:n, :hd]

    for h in range(kv):
        pk, pv = held(0, h)
        for b in range(1, len(lens)):
            n, new = lens[b], cu[b + 1] - cu[b]
            if not new:
                continue
            ok, ov = held(b, h)
            q = s["qkv"][cu[b]:cu[b + 1], h * group * hd:(h + 1) * group * hd].double()
            q = q.view(new, group, hd).transpose(0, 1)
            z = torch.cat((q @ pk.T, q @ ok.T), -1) * s["scale"]
            z = z.masked_fill(torch.ones(new, z.shape[-1], dtype=torch.bool, device=z.device)
                              .triu(len(pk) + n - new + 1), -math.inf)
            o = torch.softmax(z, -1) @ torch.cat((pv, ov))
            out[cu[b]:cu[b + 1], h * group * hd:(h + 1) * group * hd] = o.transpose(0, 1).reshape(new, -1)
    return out
