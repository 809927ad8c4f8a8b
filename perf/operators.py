"""The operators of a key/value cache held in 8 bits, as a serving program calls them: block
tables and slot maps built from request lengths, the write of new keys and values, and the
attention that reads them.

The cache of a layer is a pool of blocks of ``block_size`` tokens.  ``k`` is
``[num_blocks, kv_heads, block_size, hdp]``, ``v`` ``[num_blocks, kv_heads, hdp, block_size]``
(hdp: the head_dim rounded up to 32, 64, 96, 128, 192 or 256, the columns past head_dim zero),
float8_e4m3fn or int8, with an fp32 scale for each block and head, a power of two.

A case is a dict of plain values:

``kind``        ``"attn"``, ``"append"`` or ``"tables"``
``batch``       requests
``len_lo``, ``len_hi``  tokens a request holds before the call, spread over that range
``new_lo``, ``new_hi``  new tokens of a request, spread over that range
``heads``, ``kv_heads``, ``head_dim``, ``block``  the layer's and the cache's geometry
``dtype``       of the activations: ``"float16"``, ``"bfloat16"``
``cache``       ``"float8_e4m3fn"`` or ``"int8"``
``causal``      (attn) a new token sees the tokens up to itself, or all of its request
``sharp``       (attn) factor on the queries: the logits' standard deviation
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
_QMAX = {"float8_e4m3fn": 448.0, "int8": 127.0}
_WIDTHS = (32, 64, 96, 128, 192, 256)
_E_MIN, _E_MAX = -40, 40  # exponents of the scales


def _case(kind, batch, length, new, heads=1, kv_heads=1, head_dim=32, block=16, *, dtype="float16",
          cache="float8_e4m3fn", causal=True, sharp=1.0):
    return {"kind": kind, "batch": batch, "len_lo": length[0], "len_hi": length[1], "new_lo": new[0],
            "new_hi": new[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "dtype": dtype, "cache": cache, "causal": causal, "sharp": sharp}


def listed():
    cases = {
        # One conversation of the narrow model, a token at a time: launches are all there is.
        "attn_one": _case("attn", 1, (999, 999), (1, 1), 4, 4, 32, 16),
        # A server's ordinary step: many requests of every length, one new token each.
        "attn_b64": _case("attn", 64, (100, 2047), (1, 1), 8, 8, 64, 64, sharp=2.0),
        # Long conversations with shared heads, where the cache's bytes are what counts.
        "attn_long_gqa": _case("attn", 16, (16000, 32700), (1, 1), 32, 8, 128, 64, dtype="bfloat16", sharp=2.0),
        # The longest context of the benchmark, one request: the work has to be split over its length.
        "attn_s100000": _case("attn", 1, (99999, 99999), (1, 1), 16, 2, 64, 128, cache="int8", sharp=2.0),
        # A few draft tokens of each request are checked at once; wide heads.
        "attn_draft": _case("attn", 23, (257, 3001), (2, 6), 6, 2, 256, 32, dtype="bfloat16", cache="int8"),
        # A chunk of each of a few long prompts after what the cache holds of them (prefill by pieces).
        "attn_chunk": _case("attn", 5, (1, 6000), (301, 1024), 16, 4, 64, 64, sharp=2.0),
        # The same of a wide layer: bound by the matrix cores.
        "attn_chunk_wide": _case("attn", 2, (8000, 14001), (2000, 2048), 32, 8, 128, 64, dtype="bfloat16",
                                 sharp=2.0),
        # The step's own new keys and values, one token each.
        "append_b64": _case("append", 64, (100, 2047), (1, 1), 8, 8, 64, 64),
        # Prompts written into the cache, beginning and ending inside a block; an odd head size.
        "append_odd": _case("append", 7, (0, 333), (5, 700), 6, 6, 40, 16, cache="int8"),
        # A whole prefill chunk of a wide layer.
        "append_chunk": _case("append", 8, (0, 4000), (1500, 2048), 32, 8, 128, 64, dtype="bfloat16"),
        # A step's tables and slots: room for a few drafts of each request, then given back.
        "tables_b64": _case("tables", 64, (100, 2047), (1, 5), block=16),
        # Many prompts admitted at once.
        "tables_prefill": _case("tables", 200, (0, 1000), (1, 3001), block=32),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_GEOMETRY = ((4, 4, 32), (2, 1, 32), (6, 6, 40), (8, 8, 64), (16, 4, 64), (14, 2, 64), (12, 4, 80), (8, 4, 96),
             (32, 8, 128), (8, 1, 128), (20, 1, 128), (5, 5, 168), (6, 2, 256))


def draw(rng):
    """One more case of the same ranges, none larger than the listed largest of its family."""
    family = rng.choice(["decode", "decode", "decode", "draft", "chunk", "chunk", "append", "append", "tables"])
    heads, kv, hd = rng.choice(_GEOMETRY)
    block = rng.choice([16, 32, 64, 128])
    opt = {"dtype": rng.choice(["float16", "bfloat16"]), "cache": rng.choice(["float8_e4m3fn", "float8_e4m3fn", "int8"])}
    if family in ("decode", "draft"):
        opt["sharp"] = round(rng.uniform(1.0, 3.0), 2)
        opt["causal"] = rng.random() < 0.8
        new = (1, 1) if family == "decode" else (1, rng.randint(2, 12))
        hi = _log(rng, 1, 100000)
        # cache bytes below attn_long_gqa's, the plain form's score matrix small
        top = max(1, min(256, 800_000_000 // (hi * kv * hd * 2), 400_000_000 // (hi * heads * new[1])))
        return _case("attn", _log(rng, 1, top), (rng.randint(max(1, hi // 8), hi), hi), new, heads, kv, hd, block, **opt)
    if family == "chunk":
        opt["sharp"] = round(rng.uniform(1.0, 3.0), 2)
        opt["causal"] = rng.random() < 0.8
        new_hi = _log(rng, 17, 2048)
        hi = _log(rng, 1, 14000)
        top = max(1, min(32, 2_000_000_000 // ((hi + new_hi) * heads * new_hi)))
        return _case("attn", _log(rng, 1, top), (rng.randint(0, hi), hi), (rng.randint(1, new_hi), new_hi), heads, kv,
                     hd, block, **opt)
    if family == "append":
        new_hi = _log(rng, 1, 2048)
        hi = _log(rng, 1, 4000)
        top = max(1, min(256, 14_000_000 // (new_hi * kv * hd), 60_000_000 // ((hi + new_hi) * kv * hd)))
        return _case("append", _log(rng, 1, top), (rng.randint(0, hi), hi), (rng.randint(1, new_hi), new_hi), heads, kv,
                     hd, block, **opt)
    new_hi = _log(rng, 1, 3000)
    return _case("tables", _log(rng, 1, max(1, min(1024, 300_000 // new_hi))), (0, _log(rng, 1, 4000)),
                 (rng.randint(0, new_hi), new_hi), block=block)


# -- inputs -------------------------------------------------------------------------


def _spread(lo, hi, n, phase):
    """n whole numbers over lo .. hi, the same for every seed (so that the work is the case's own)."""
    return [lo + int((hi - lo + 1) * ((phase + i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(case):
    """(tokens before the call, new tokens) of each request."""
    return (_spread(case["len_lo"], case["len_hi"], case["batch"], 0.999999),
            _spread(case["new_lo"], case["new_hi"], case["batch"], 0.5))


def _hdp(head_dim):
    return next(w for w in _WIDTHS if w >= head_dim)


def _blocks(tokens, block):
    return -(-tokens // block)


def _pool(held, extra, block, g):
    """Block tables for ``held`` tokens of each request (width: what they hold after ``extra``
    more, and one), their blocks scattered over the pool, and the free blocks as a stack."""
    width = max(_blocks(h + e, block) for h, e in zip(held, extra)) + 1
    need = [_blocks(h, block) for h in held]
    total = sum(_blocks(h + e, block) for h, e in zip(held, extra)) + 3
    order = torch.randperm(total, generator=g, device=_DEVICE).to(torch.int32)
    rows = torch.tensor(need, device=_DEVICE)
    col = torch.arange(width, device=_DEVICE)
    first = torch.cumsum(rows, 0) - rows
    at = (first[:, None] + col).clamp(max=total - 1)
    table = torch.where(col < rows[:, None], order[at], torch.full_like(order[at], -1)).contiguous()
    used = sum(need)
    free = torch.full((total,), -1, dtype=torch.int32, device=_DEVICE)
    free[: total - used] = order[used:]
    return table, free, torch.tensor([total - used], dtype=torch.int32, device=_DEVICE), total


def _exponent(amax, qmax):
    """The least whole e in [_E_MIN, _E_MAX] with amax <= qmax 2^e (exact: frexp and compare)."""
    m, x = torch.frexp(amax)  # amax = m 2^x, 1/2 <= m < 1
    qm, qx = math.frexp(qmax)
    e = torch.where(m <= qm, x - qx, x - qx + 1)
    return torch.where(amax > 0, e, torch.full_like(e, _E_MIN)).clamp(_E_MIN, _E_MAX)


def _codes(x, cache):
    """Scaled values rounded to the nearest code (ties to even) and limited to its range."""
    q = _QMAX[cache]
    x = x.clamp(-q, q)
    return x.round().to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)


def _contents(case, total, g, seen):
    """A pool's keys and values as appends leave them: magnitudes that differ from block to
    block, and memory that nobody wrote (NaN codes) past the ends of the requests.
    ``seen``: [total, block] truth values, the tokens that were written."""
    kv, hd, hdp, bs, cache = case["kv_heads"], case["head_dim"], _hdp(case["head_dim"]), case["block"], case["cache"]
    out = []
    for _ in range(2):
        x = torch.randn(total, kv, bs, hd, generator=g, device=_DEVICE)
        x *= torch.exp(0.5 * torch.randn(total, kv, 1, 1, generator=g, device=_DEVICE)) * 0.7
        e = _exponent(x.abs().amax((2, 3)), _QMAX[cache])
        scale = torch.ldexp(torch.ones_like(x[:, :, 0, 0]), e)
        x /= scale[:, :, None, None]
        x = torch.nn.functional.pad(x, (0, hdp - hd))
        code = _codes(x, cache).view(torch.uint8)
        del x
        code = torch.where(seen[:, None, :, None], code, torch.full_like(code, 0x80 if cache == "int8" else 0x7F))
        out += [code.view(_DTYPES[cache]), scale]
    k, ks, v, vs = out
    v = v.view(torch.uint8).transpose(2, 3).contiguous().view(_DTYPES[cache])
    return k, ks, v, vs


def _written(table, lens, block, total):
    """[total, block]: which tokens of the pool the requests hold."""
    bsz, width = table.shape
    pos = torch.arange(width * block, device=_DEVICE).view(1, width, block)
    live = pos < lens.view(bsz, 1, 1)
    seen = torch.zeros(total + 1, block, dtype=torch.bool, device=_DEVICE)
    seen[torch.where(table >= 0, table, torch.full_like(table, total)).long().view(-1)] = live.view(-1, block)
    return seen[:total]


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    held, new = _lengths(case)
    block, kind = case["block"], case["kind"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=_DEVICE)  # noqa: E731
    if kind == "tables":
        table, free, count, _ = _pool(held, new, block, g)
        return {"case": case, "lens": i32(held), "keep": i32(held), "new": i32(new), "table": table, "free": free,
                "count": count, "tokens": sum(new)}
    heads, kv, hd, dt = case["heads"], case["kv_heads"], case["head_dim"], _DTYPES[case["dtype"]]
    tokens = sum(new)
    qkv = torch.randn(tokens, (heads + 2 * kv) * hd, generator=g, device=_DEVICE)
    if kind == "attn":
        # The call comes after the new tokens' own append: the cache holds them too.
        after = [h + n for h, n in zip(held, new)]
        table, _, _, total = _pool(after, [0] * len(held), block, g)
        lens = i32(after)
        k, ks, v, vs = _contents(case, total, g, _written(table, lens, block, total))
        qkv[:, : heads * hd] *= case["sharp"] * 1.2
        cu = i32([0] + [sum(new[: i + 1]) for i in range(len(new))])
        return {"case": case, "qkv": qkv.to(dt), "cu": cu, "lens": lens, "table": table, "k": k, "ks": ks, "v": v,
                "vs": vs, "max_new": max(new), "max_len": max(after), "scale": hd ** -0.5}
    table, free, count, total = _pool(held, new, block, g)
    lens = i32(held)
    k, ks, v, vs = _contents(case, total, g, _written(table, lens, block, total))
    # Now and then a token is far larger than its block has seen: its scale has to grow.
    qkv *= torch.exp(torch.randn(tokens, 1, generator=g, device=_DEVICE))
    slots, first = [], 0
    spare = free[: int(count)].flip(0).long()
    for b, (h, n) in enumerate(zip(held, new)):
        had, has = _blocks(h, block), _blocks(h + n, block)
        table[b, had:has] = spare[first:first + has - had].int()
        first += has - had
        pos = torch.arange(h, h + n, device=_DEVICE)
        slots.append(table[b].long()[pos // block] * block + pos % block)
    runs = sum(_blocks(h + n, block) - h // block for h, n in zip(held, new) if n > 0)
    return {"case": case, "qkv": qkv.to(dt), "slots": torch.cat(slots), "k": k, "ks": ks, "v": v, "vs": vs,
            "runs": runs}


# -- one pass -----------------------------------------------------------------------


def run(state):
    case = state["case"]
    if case["kind"] == "tables":
        return _own_tables(state) if own else _plain_tables(state)
    if case["kind"] == "append":
        if own:
            _own_append(state)
        else:
            _plain_append(state)
        return {"k": state["k"], "k_scale": state["ks"], "v": state["v"], "v_scale": state["vs"]}
    return _own_attn(state) if own else _plain_attn(state)


def _own_tables(s):
    from cobra_amd import ops

    block = s["case"]["block"]
    slots, cu, missing = ops.cache_reserve(s["lens"], s["new"], s["table"], s["free"], s["count"], block, s["tokens"])
    refused = ops.cache_trim(s["lens"], s["keep"], s["table"], s["free"], s["count"], block)
    return {"slots": slots, "cu": cu, "missing": missing, "refused": refused, "table": s["table"], "lens": s["lens"],
            "free": s["free"], "count": s["count"]}


def _own_append(s):
    from cobra_amd import ops

    c = s["case"]
    ops.cache_append(s["qkv"], s["slots"], c["heads"], c["head_dim"], s["k"], s["v"], s["ks"], s["vs"])


def _own_attn(s):
    from cobra_amd import ops

    c = s["case"]
    return ops.cache_attn(s["qkv"], s["cu"], s["lens"], s["table"], c["heads"], c["head_dim"], s["scale"], s["k"],
                          s["v"], s["ks"], s["vs"], causal=c["causal"], max_new=s["max_new"], max_len=s["max_len"])


def _plain_tables(s):
    block, lens, new, table, free, count = s["case"]["block"], s["lens"], s["new"], s["table"], s["free"], s["count"]
    had = (lens + block - 1) // block
    need = (lens + new + block - 1) // block - had
    first = torch.cumsum(need, 0) - need
    cu = torch.zeros(new.numel() + 1, dtype=torch.int32, device=new.device)
    cu[1:] = torch.cumsum(new, 0)
    # The k-th new block is the k-th from the top of the stack.
    col = torch.arange(table.shape[1], device=new.device)[None, :]
    mine = (col >= had[:, None]) & (col < (had + need)[:, None])
    at = (count - 1 - (first[:, None] + col - had[:, None])).clamp(min=0, max=free.numel() - 1)
    table.copy_(torch.where(mine, free[at.long()], table))
    t = torch.arange(s["tokens"], device=new.device)
    b = torch.searchsorted(cu[1:], t.int(), right=True)
    pos = lens[b] + (t - cu[b])
    slots = table[b, (pos // block).long()].long() * block + pos % block
    lens += new
    count -= need.sum().int()
    # The way back: the k-th block returned goes k places below the new top.
    kept = torch.minimum(lens, s["keep"])
    has, stay = (lens + block - 1) // block, (kept + block - 1) // block
    back = has - stay
    total = back.sum().int()
    first = torch.cumsum(back, 0) - back
    gone = (col >= stay[:, None]) & (col < has[:, None])
    to = count + total - 1 - (first[:, None] + col - stay[:, None])
    to = torch.where(gone, to, torch.full_like(to, free.numel()))
    wide = torch.cat([free, free[:1]])
    wide.scatter_(0, to.long().view(-1), table.reshape(-1))
    free.copy_(wide[:-1])
    count += total
    lens.copy_(kept)
    zero = torch.zeros(1, dtype=torch.int32, device=new.device)
    return {"slots": slots, "cu": cu, "missing": zero, "refused": zero.clone(), "table": table, "lens": lens,
            "free": free, "count": count}


def _plain_append(s):
    c = s["case"]
    heads, kv, hd, hdp, bs, cache = (c["heads"], c["kv_heads"], c["head_dim"], _hdp(c["head_dim"]), c["block"],
                                     c["cache"])
    slots, n = s["slots"], s["runs"]
    dev = slots.device
    blk, off = slots // bs, slots % bs
    head = torch.ones_like(blk, dtype=torch.bool)
    head[1:] = blk[1:] != blk[:-1]
    run_of = torch.cumsum(head, 0) - 1
    block_of = torch.zeros(n, dtype=torch.long, device=dev).scatter_(0, run_of, blk)
    lowest = torch.full((n,), bs, dtype=torch.long, device=dev).scatter_reduce_(0, run_of, off, "amin")
    put = torch.zeros(n, bs, dtype=torch.bool, device=dev)
    put[run_of, off] = True
    live = torch.arange(bs, device=dev)[None, :] < lowest[:, None]
    for name, part in (("k", 0), ("v", 1)):
        x = s["qkv"][:, (heads + part * kv) * hd:(heads + (part + 1) * kv) * hd].float().view(-1, kv, hd)
        x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
        amax = torch.where(torch.isinf(x), torch.zeros_like(x), x).abs().amax(2)
        amax = torch.zeros(n, kv, device=dev).scatter_reduce_(0, run_of[:, None].expand(-1, kv), amax, "amax")
        fresh = torch.ldexp(torch.ones_like(amax), _exponent(amax, _QMAX[cache]))
        old = s[name + "s"][block_of]
        scale = torch.where((lowest == 0)[:, None], fresh, torch.maximum(old, fresh))
        codes = s[name].view(torch.uint8)[block_of]
        codes = codes.transpose(2, 3) if name == "v" else codes  # [n, kv, bs, hdp]
        grown = _codes(codes.contiguous().view(_DTYPES[cache]).float() * (old / scale)[:, :, None, None], cache)
        grew = ((scale > old)[:, :, None] & live[:, None, :])[..., None]
        codes = torch.where(grew, grown.view(torch.uint8), codes)
        fill = torch.zeros(n, bs, kv, hdp, dtype=torch.uint8, device=dev)
        fill[run_of, off, :, :hd] = _codes(x / scale[run_of][:, :, None], cache).view(torch.uint8)
        codes = torch.where(put[:, None, :, None], fill.transpose(1, 2), codes)
        codes = codes.transpose(2, 3) if name == "v" else codes
        s[name].view(torch.uint8)[block_of] = codes
        s[name + "s"][block_of] = scale


def _plain_attn(s):
    c = s["case"]
    heads, kv, hd, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]
    lens, cu, dev = s["lens"], s["cu"], s["lens"].device
    bsz, group = lens.numel(), heads // kv
    nb = -(-s["max_len"] // bs)
    tab = s["table"][:, :nb].clamp(min=0).long()
    there = torch.arange(nb * bs, device=dev)[None, :] < lens[:, None]

    def values(codes, scale, order):
        x = codes.view(torch.uint8)[tab].view(codes.dtype).float() * scale[tab][..., None, None]
        x = x.permute(order).reshape(bsz, kv, nb * bs, -1)[..., :hd]
        return torch.where(there[:, None, :, None], x, torch.zeros_like(x))

    k = values(s["k"], s["ks"], (0, 2, 1, 3, 4))
    v = values(s["v"], s["vs"], (0, 2, 1, 4, 3))
    i = torch.arange(s["max_new"], device=dev)
    row = (cu[:-1, None] + i).clamp(max=s["qkv"].shape[0] - 1).long()
    q = s["qkv"][:, : heads * hd].float()[row].view(bsz, s["max_new"], kv, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(bsz, kv, group * s["max_new"], hd)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    new = cu[1:] - cu[:-1]
    last = lens[:, None] - new[:, None] + i if c["causal"] else lens[:, None] - 1 + 0 * i
    seen = torch.arange(nb * bs, device=dev)[None, None, :] <= last[:, :, None]
    seen = (seen & there[:, None, :])[:, None, None]
    score = score.view(bsz, kv, group, s["max_new"], nb * bs).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(bsz, kv, group * s["max_new"], nb * bs), v).view(bsz, kv, group, s["max_new"], hd)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    t = torch.arange(s["qkv"].shape[0], device=dev)
    b = torch.searchsorted(cu[1:], t.int(), right=True)
    o = o.permute(0, 3, 1, 2, 4)[b, t - cu[b]]
    return o.reshape(-1, heads * hd).to(s["qkv"].dtype)


# -- the work of a pass, and its exact result ------------------------------------------


def work(case):
    held, new = _lengths(case)
    block = case["block"]
    if case["kind"] == "tables":
        got = sum(_blocks(h + n, block) - _blocks(h, block) for h, n in zip(held, new))
        # lengths read and written twice, ids read and written twice, slots and offsets written
        return {"bytes": 4 * case["batch"] * 7 + 4 * got * 4 + 8 * sum(new), "flops": 0}
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        # 16-bit keys and values in, 8-bit codes and the scales out
        runs = sum(_blocks(h + n, block) - h // block for h, n in zip(held, new) if n > 0)
        return {"bytes": sum(new) * (kv * hd * 2 * 2 + kv * _hdp(hd) * 2 + 8) + runs * kv * 8, "flops": 0}
    pairs = sum(sum(h + i + 1 for i in range(n)) if case["causal"] else n * (h + n) for h, n in zip(held, new))
    cached = sum(h + n for h, n in zip(held, new))
    pages = sum(_blocks(h + n, block) for h, n in zip(held, new))
    return {"bytes": cached * kv * hd * 2 + pages * (4 + kv * 8) + 2 * 2 * sum(new) * heads * hd + 12 * case["batch"],
            "flops": 4 * pairs * heads * hd}


def exact(case, seed):
    """The results in 64 bits, request by request."""
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return None  # whole numbers
    return _exact_append(s) if case["kind"] == "append" else _exact_attn(s)


def _exact_append(s):
    """Block after block on the host's lists, every quantity exact in 64 bits."""
    c = s["case"]
    heads, kv, hd, bs, cache = c["heads"], c["kv_heads"], c["head_dim"], c["block"], c["cache"]
    if s["runs"] > 4000:
        return None
    qmax = _QMAX[cache]
    lists = {}
    for t, slot in enumerate(s["slots"].tolist()):
        lists.setdefault(slot // bs, []).append((slot % bs, t))
    out = {}
    for name, first in (("k", heads * hd), ("v", (heads + kv) * hd)):
        code, scale = s[name].double().cpu(), s[name + "s"].double().cpu()
        if name == "v":
            code = code.transpose(2, 3).contiguous()
        src = s["qkv"][:, first:first + kv * hd].double().cpu().view(-1, kv, hd)
        for blk, tokens in lists.items():
            offs, ts = [o for o, _ in tokens], [t for _, t in tokens]
            x = src[ts]
            big = x.abs().amax((0, 2))
            for h in range(kv):
                e = _E_MIN
                while float(big[h]) > qmax * 2.0 ** e:
                    e += 1
                new = 2.0 ** min(e, _E_MAX)
                had = float(scale[blk, h])
                if min(offs) > 0:
                    if new > had:
                        code[blk, h, :min(offs)] = _nearest(code[blk, h, :min(offs)] * (had / new), cache)
                    new = max(new, had)
                scale[blk, h] = new
                code[blk, h, offs, :hd] = _nearest(x[:, h] / new, cache)
                code[blk, h, offs, hd:] = 0
        if name == "v":
            code = code.transpose(2, 3).contiguous()
        out[name], out[name + "_scale"] = None if cache == "int8" else code, scale
    return out


def _nearest(x, cache):
    """The nearest value of the code, ties to the even one, from its definition: whole
    numbers; or 4 significant bits down to steps of 2^-9."""
    q = _QMAX[cache]
    if cache == "int8":
        return torch.round(x.clamp(-q, q))
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-q, q)


def _exact_attn(s):
    c = s["case"]
    heads, kv, hd, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].long()
    out = torch.zeros(s["qkv"].shape[0], heads * hd, dtype=torch.float64, device=s["qkv"].device)
    for b, n in enumerate(lens):
        new = cu[b + 1] - cu[b]
        if not new or not n:
            continue
        pages = table[b, : _blocks(n, bs)]
        for h in range(kv):
            k = s["k"].view(torch.uint8)[pages, h].view(s["k"].dtype).double() * s["ks"][pages, h].double()[:, None, None]
            v = s["v"].view(torch.uint8)[pages, h].view(s["v"].dtype).double() * s["vs"][pages, h].double()[:, None, None]
            k = k.reshape(-1, k.shape[-1])[:n, :hd]
            v = v.transpose(1, 2).reshape(-1, v.shape[1])[:n, :hd]
            for head in range(h * (heads // kv), (h + 1) * (heads // kv)):
                q = s["qkv"][cu[b]:cu[b + 1], head * hd:(head + 1) * hd].double()
                z = q @ k.T * s["scale"]
                if c["causal"]:
                    z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(n - new + 1), -math.inf)
                out[cu[b]:cu[b + 1], head * hd:(head + 1) * hd] = torch.softmax(z, -1) @ v
    return out
