"""Attention over the cache for about as many requests as a launch has workgroups, few of them with new tokens."""

import random

import pytest
import torch

from _cache_util import E4M3, codes_of
from _gpu_util import DEV

PLACES = (1 << 24) - 1  # workgroups of a launch


def test_splits_leave_every_request_its_workgroups():
    """On the CPU, as far as the workspace shows it."""
    from cobra_amd import _lib

    q = _lib.lib().cobra_cache_attn_workspace_bytes
    rng = random.Random(5)
    cases = [(120, 8388607, 32, 2, 32, 40, 5000), (1, 16777215, 1, 1, 64, 200, 10 ** 6)]
    for _ in range(3000):
        kv = rng.choice([1, 2, 8, 32])
        cases.append((int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(16, 24)) // kv, kv * rng.choice([1, 4, 20]), kv,
                      8 * rng.randint(1, 32), rng.choice([1, 5, 100, 10 ** 6]), int(2 ** rng.uniform(0, 31))))
    for tokens, batch, heads, kv, hd, new, length in cases:
        width = next(w for w in (32, 64, 96, 128, 192, 256) if w >= hd)
        splits = q(tokens, batch, heads, kv, hd, new, length) // (tokens * heads * (4 * width + 8))
        assert batch * kv * max(1, splits) <= PLACES, (tokens, batch, heads, kv, hd, new, length, splits)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,batch", [(16, 16, 1048575), (32, 2, 8388607)])
@pytest.mark.parametrize("new", [1, 40])
def test_as_many_requests_as_a_launch_has_workgroups(heads, kv, batch, new):
    """The requests with new tokens get what they get alone."""
    from cobra_amd import ops

    from test_gpu_prefix import build, i32

    hd, where = 32, [0, 5, batch // 2, batch - 1]
    held, few = [90, 1030 + new, 2 + new, new], [0, new, new, new]
    table, pool, q, cu = build(held, few, 0, heads, kv, hd, 16, torch.float16, E4M3, 7)
    dev = [t.to(DEV) for t in pool]
    rest = [heads, hd, hd ** -0.5, *dev]
    want = ops.cache_attn(q.to(DEV), i32(cu), i32(held), i32(table), *rest)
    lens = torch.zeros(batch, dtype=torch.int32)
    fresh = torch.zeros(batch + 1, dtype=torch.int32)
    tables = torch.full((batch, len(table[0])), -1, dtype=torch.int32)
    for b, n, f, row in zip(where, held, few, table):
        lens[b], fresh[b + 1], tables[b] = n, f, torch.tensor(row)
    args = [t.to(DEV) for t in (torch.cumsum(fresh, 0, dtype=torch.int32), lens, tables)]
    # Another order of the sums: either result is off by under 2^-9 of the largest |v|.
    largest = float((codes_of(pool[1]).abs().amax((1, 2, 3)) * pool[3].double().amax(1)).max())
    for hints in ({}, dict(max_new=new, max_len=100), dict(max_new=new, max_len=5000)):
        got = ops.cache_attn(q.to(DEV), *args, *rest, **hints)
        assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -8 * largest
