"""Operators of a serving step in plain form, 64 bits, on the host: matrices in 8-bit blocks and
their product, norms and rotation of queries and keys, attention behind a shared prefix."""

from __future__ import annotations

import math

import torch

from . import cache as oc

E4M3 = torch.float8_e4m3fn


def quantize(x: torch.Tensor):
    """(values of the codes, NaN where x is not finite; scale bytes) of [M, K], padded."""
    m, k = x.shape
    kp, s = -(-k // 128) * 128, -(-k // 512) * 4
    z = torch.zeros(m, kp, dtype=torch.float64)
    z[:, :k] = x.double()
    z = z.view(m, kp // 128, 128)
    a = torch.where(torch.isfinite(z), z.abs(), torch.zeros_like(z)).amax(2)
    e = torch.full_like(a, -126)
    for _ in range(254):  # the least power of two that holds the block
        e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
    q = oc.nearest(z / torch.exp2(e)[:, :, None], E4M3)
    q = torch.where(torch.isfinite(z), q, torch.full_like(q, math.nan))
    scale = torch.full((m, s), 127, dtype=torch.int64)
    scale[:, : kp // 128] = e.long() + 127
    return q.view(m, kp), scale


def values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What codes (their values) and scale bytes stand for."""
    m, kp = codes.shape
    return (codes.double().view(m, kp // 128, 128) * torch.exp2(scale[:, : kp // 128].double() - 127)[:, :, None]).view(m, kp)


def gelu(x: torch.Tensor) -> torch.Tensor:
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))


def cut_of_eights(a: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """What products of [M, K] and [N, K] may lose where eight consecutive ones are added with every one
    cut under 2^-13 of the largest one's exponent: 7 of eight by less than 2^-13 of the largest."""
    m, n = a.shape[0], w.shape[0]
    out = torch.zeros(m, n, dtype=torch.float64)
    for x, y in zip(a.abs().view(m, -1, 8).unbind(1), w.abs().view(n, -1, 8).unbind(1)):
        out += (x[:, None] * y[None]).amax(2)
    return 7 * 2.0 ** -13 * out


def linear(a, w, bias=None, use_gelu=False, resid=None, rmask=None, mask_branch=False):
    """(result, sum |a w| + |bias|) from 64-bit values."""
    y, mag = a @ w.T, a.abs() @ w.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if use_gelu:
        y = gelu(y)
    keep = None if rmask is None else (rmask != 0)[:, None]
    if keep is not None and mask_branch:
        y = torch.where(keep, y, torch.zeros_like(y))
    if resid is not None:
        y = y + resid.double()
        if keep is not None and not mask_branch:
            y = torch.where(keep, y, torch.zeros_like(y))
    return y, mag


def norm_rope(x, head_dim, pos, inv_freq, weight, interleaved, eps):
    """One head's columns [T, head_dim] -> the same after its norm and rotation."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(1, keepdim=True) + eps) * weight.double()
    if inv_freq is not None:
        r = inv_freq.numel()
        t = pos.double()[:, None] * inv_freq.double()
        i = torch.arange(r)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
        ya, yb = y[:, a], y[:, b]
        y = y.clone()
        y[:, a], y[:, b] = ya * t.cos() - yb * t.sin(), yb * t.cos() + ya * t.sin()
    return y


def attend(q, cu, lens, table, prefix, heads, head_dim, scale, k, v, k_scale, v_scale, causal):
    """``oc.attend`` behind the prefix in row ``prefix``: (ctx, sum p |v|, largest |score|, largest sum
    |q k| scale)."""
    n_blocks, kv, bs, _ = k.shape
    group = heads // kv
    out = torch.zeros(q.shape[0], heads, head_dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    top = reach = 0.0

    def held(b, h):
        L = max(0, min(lens[b], len(table[b]) * bs))
        pages = table[b][: oc.blocks(L, bs)]
        ok = torch.tensor([0 <= p < n_blocks for p in pages], dtype=torch.bool).repeat_interleave(bs)[:L]
        ids = torch.tensor([p if 0 <= p < n_blocks else 0 for p in pages], dtype=torch.long)
        kk = (k[ids, h] * k_scale[ids, h][:, None, None].double()).reshape(-1, k.shape[3])[:L, :head_dim]
        vv = (v[ids, h] * v_scale[ids, h][:, None, None].double()).transpose(1, 2).reshape(-1, v.shape[2])[:L, :head_dim]
        return torch.where(ok[:, None], kk, torch.zeros_like(kk)), torch.where(ok[:, None], vv, torch.zeros_like(vv)), ok

    for b, L in enumerate(lens):
        new = cu[b + 1] - cu[b]
        if new == 0:
            continue
        for h in range(kv):
            kk, vv, ok = held(b, h)
            pos = L - new + torch.arange(new)
            j = torch.arange(kk.shape[0])
            seen = ok[None, :] & (j[None, :] <= pos[:, None] if causal else torch.ones(new, kk.shape[0], dtype=torch.bool))
            if b != prefix:
                pk, pv, pok = held(prefix, h)
                kk, vv = torch.cat((pk, kk)), torch.cat((pv, vv))
                seen = torch.cat((pok[None, :].expand(new, -1), seen), 1)
            if kk.shape[0] == 0:
                continue
            for g in range(h * group, (h + 1) * group):
                x = q[cu[b]:cu[b + 1], g * head_dim:(g + 1) * head_dim].double()
                s = (x @ kk.T) * scale
                if seen.any():
                    top = max(top, float(s[seen].abs().max()))
                    reach = max(reach, float((x.abs() @ kk.abs().T)[seen].max()) * scale)
                s = s.masked_fill(~seen, -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
                t = p.sum(-1, keepdim=True)
                p = p / torch.where(t > 0, t, torch.ones_like(t))
                out[cu[b]:cu[b + 1], g] = p @ vv
                mag[cu[b]:cu[b + 1], g] = p @ vv.abs()
    return out.view(q.shape[0], -1), mag.view(q.shape[0], -1), top, reach
