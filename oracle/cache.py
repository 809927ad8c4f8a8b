"""The 8-bit key/value cache in plain form, 64 bits, on the host: block tables as lists, the
quantised write token by token, and attention request by request."""

from __future__ import annotations

import math
from typing import List, Tuple

import torch

E_MIN, E_MAX = -40, 40
QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def blocks(tokens: int, block: int) -> int:
    return -(-tokens // block)


def reserve(lens, new, table, free, block, tokens, count, num_free) -> Tuple[int, List[int], List[int], int]:
    """Python lists in place -> (missing, slots, cu, new count)."""
    width = len(table[0]) if table else 0
    bad = not 0 <= count <= num_free or sum(n for n in new if n > 0) > tokens
    need = []
    for L, n in zip(lens, new):
        if L < 0 or n < 0 or L + n > 2 ** 31 - 1 or blocks(L + n, block) > width:
            bad = True
            need.append(0)
        else:
            need.append(blocks(L + n, block) - blocks(L, block))
    refused = [-1] * tokens, [0] * (len(lens) + 1), count
    if bad:
        return (-1, *refused)
    if sum(need) > count:
        return (sum(need) - count, *refused)
    slots, cu = [], [0]
    for b, n in enumerate(new):
        at = blocks(lens[b], block)
        for j in range(need[b]):
            count -= 1
            table[b][at + j] = free[count]
        for p in range(lens[b], lens[b] + n):
            slots.append(table[b][p // block] * block + p % block)
        lens[b] += n
        cu.append(cu[-1] + n)
    return 0, slots + [-1] * (tokens - len(slots)), cu, count


def trim(lens, keep, table, free, block, count, num_free) -> Tuple[int, int]:
    """Python lists in place -> (refused, new count)."""
    width = len(table[0]) if table else 0
    if count < 0 or any(L < 0 or blocks(L, block) > width for L in lens):
        return 1, count
    gone = []
    for b, (L, kp) in enumerate(zip(lens, keep)):
        gone += table[b][blocks(min(L, max(kp, 0)), block):blocks(L, block)]
    if count + len(gone) > num_free:
        return 1, count
    for b, kp in enumerate(keep):
        lens[b] = min(lens[b], max(kp, 0))
    free[count:count + len(gone)] = gone[::-1]
    return 0, count + len(gone)


def nearest(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The code value nearest to each x (ties to even), within range; NaN gives 0."""
    q = QMAX[dtype]
    x = torch.nan_to_num(x, nan=0.0, posinf=q, neginf=-q).clamp(-q, q)
    if dtype == torch.int8:
        return torch.round(x)
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-q, q)


def exponent(amax: float, dtype: torch.dtype) -> int:
    e = E_MIN
    while e < E_MAX and amax > QMAX[dtype] * 2.0 ** e:
        e += 1
    return e


def append(qkv, slots, heads, head_dim, k, v, k_scale, v_scale, dtype) -> None:
    """k [N, H, bs, w], v [N, H, w, bs] and the scales as 64-bit host tensors, in place."""
    n, kv, bs, _ = k.shape
    by_block = {}
    for t, s in enumerate(slots):
        if 0 <= s < n * bs:
            by_block.setdefault(s // bs, {})[s % bs] = t  # of two for one slot the later one stays
    for code, scale, first in ((k, k_scale, heads), (v.transpose(2, 3), v_scale, heads + kv)):
        x = qkv[:, first * head_dim:(first + kv) * head_dim].double().view(-1, kv, head_dim)
        for blk, at in by_block.items():
            offs = sorted(at)
            rows = x[[at[o] for o in offs]]
            for h in range(kv):
                a = rows[:, h].abs()
                a = a[torch.isfinite(a)]
                new = 2.0 ** exponent(float(a.max()) if a.numel() else 0.0, dtype)
                old = float(scale[blk, h])
                if offs[0] > 0:
                    if new > old:
                        code[blk, h, :offs[0]] = nearest(code[blk, h, :offs[0]] * (old / new), dtype)
                    new = max(new, old)
                scale[blk, h] = new
                code[blk, h, offs, head_dim:] = 0
                code[blk, h, offs, :head_dim] = nearest(rows[:, h] / new, dtype)


def attend(q, cu, lens, table, heads, head_dim, scale, k, v, k_scale, v_scale, causal):
    """(ctx, |ctx| bound sum_j p_j |v_j|, largest |score|, largest sum |q k| scale) in 64 bits.

    k, v: 64-bit code values; cu, lens, table: lists.  Table entries outside the pool mask
    their keys."""
    n_blocks, kv, bs, _ = k.shape
    group = heads // kv
    out = torch.zeros(q.shape[0], heads, head_dim, dtype=torch.float64)
    mag = torch.zeros_like(out)
    top = reach = 0.0
    for b, L in enumerate(lens):
        new = cu[b + 1] - cu[b]
        if new == 0 or L <= 0:
            continue
        pages = table[b][:blocks(L, bs)]
        ok = torch.tensor([0 <= p < n_blocks for p in pages]).repeat_interleave(bs)[:L]
        ids = torch.tensor([p if 0 <= p < n_blocks else 0 for p in pages])
        pos = L - new + torch.arange(new)
        j = torch.arange(L)
        seen = ok[None, :] & (j[None, :] <= pos[:, None] if causal else torch.ones(new, L, dtype=torch.bool))
        for h in range(kv):
            kk = (k[ids, h] * k_scale[ids, h][:, None, None].double()).reshape(-1, k.shape[3])[:L, :head_dim]
            vv = (v[ids, h] * v_scale[ids, h][:, None, None].double()).transpose(1, 2).reshape(-1, v.shape[2])
            vv = vv[:L, :head_dim]
            kk = torch.where(ok[:, None], kk, torch.zeros_like(kk))
            vv = torch.where(ok[:, None], vv, torch.zeros_like(vv))
            for g in range(h * group, (h + 1) * group):
                x = q[cu[b]:cu[b + 1], g * head_dim:(g + 1) * head_dim].double()
                s = (x @ kk.T) * scale
                top = max(top, float(s[seen].abs().max()) if seen.any() else 0.0)
                reach = max(reach, float((x.abs() @ kk.abs().T)[seen].max()) * scale if seen.any() else 0.0)
                s = s.masked_fill(~seen, -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
                t = p.sum(-1, keepdim=True)
                p = p / torch.where(t > 0, t, torch.ones_like(t))
                out[cu[b]:cu[b + 1], g] = p @ vv
                mag[cu[b]:cu[b + 1], g] = p @ vv.abs()
    return out.view(q.shape[0], -1), mag.view(q.shape[0], -1), top, reach
