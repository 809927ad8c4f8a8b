"""Shared pieces of the cache tests: filled pools, host copies, and the attention's tolerance
(not collected: no test_ prefix)."""

from __future__ import annotations

import math

import torch

from oracle import cache as oc

E4M3, I8 = torch.float8_e4m3fn, torch.int8


def codes_of(t: torch.Tensor) -> torch.Tensor:
    """The code values of a cache tensor as 64-bit host numbers (NaN codes as 0)."""
    return torch.nan_to_num(t.cpu().double(), nan=0.0)


def random_cache(num_blocks, kv_heads, block, head_dim, dtype, seed, spread=6):
    """A pool with every token written: (k, v, k_scale, v_scale) on the host, codes over the
    whole range, scales 2^-spread .. 2^spread."""
    from cobra_amd import ops

    w = ops.cache_width(head_dim)
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape in ((num_blocks, kv_heads, block, w), (num_blocks, kv_heads, w, block)):
        x = torch.randn(shape, generator=g) * (60.0 if dtype == E4M3 else 40.0)
        if shape[2] == w:
            x[:, :, head_dim:] = 0
        else:
            x[..., head_dim:] = 0
        out.append(x.clamp(-448, 448).to(dtype) if dtype == E4M3 else x.round().clamp(-127, 127).to(dtype))
        e = torch.randint(-spread, spread + 1, (num_blocks, kv_heads), generator=g) - 6
        out.append(torch.ldexp(torch.ones(num_blocks, kv_heads), e))
    k, ks, v, vs = out
    return k, v, ks, vs


def poison(k, v, blk, first):
    """Codes of tokens first .. of a block as memory that nobody wrote: NaN (int8: -128)."""
    bad = 0x80 if k.dtype == I8 else 0x7F
    k.view(torch.uint8)[blk, :, first:] = bad
    v.view(torch.uint8)[blk, :, :, first:] = bad


def attn_tolerance(want, mag, top, reach, keys, head_dim, dtype, v_scale_max):
    """Largest |got - want| by element.

    p_j = w_j / l: w_j rounded to fp16 (half a step: 2^-11 of it; under 2^-14, where the row's
    reference has 2^8, at most 2^-25), from a score in fp32.  A score is a sum of
    head_dim products: at most head_dim + 4 roundings of 2^-24 of sum |q k|; in log2 units it is
    multiplied, has the scale's logarithm (at most 40) and the reference taken away: 6 roundings
    of 2^-24 of at most |score| log2(e) + 40, each; exp2 adds 2^-22.  Sums over the keys in
    fp32: keys roundings of 2^-24 each in O and l.  The result rounds once more to its type."""
    u = 2.0 ** -24
    score = (head_dim + 4) * u * reach + 6 * u * (top * math.log2(math.e) + 40 + 14) * math.log(2.0)
    rel = 2.0 ** -11 + 2 * score + 2.0 ** -21 + 2 * (keys + 8) * u
    eps = torch.finfo(dtype).eps / 2
    return (eps * (1 + rel)) * want.abs() + rel * mag * 1.01 + keys * 2.0 ** -33 * 448 * v_scale_max + \
        (2.0 ** -25 if dtype == torch.float16 else 0.0)


def model_tables(batch, held, block, num_blocks, width, seed):
    """Host lists: table (entries past the held blocks arbitrary), free stack, count."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_blocks, generator=g).tolist()
    table, at = [], 0
    for b in range(batch):
        n = oc.blocks(held[b], block)
        row = order[at:at + n] + [1 << 30, -7, -1, 2 ** 31 - 1] * width
        table.append(row[:width])
        at += n
    free = order[at:]
    return table, free + [-1] * (num_blocks - len(free)), len(free)
