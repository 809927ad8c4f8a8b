"""GPU tests of attention behind a shared prefix where a launch's limits, or its splits', are reached."""

import pytest
import torch

from oracle import serve

from _cache_util import E4M3, I8, attn_tolerance, codes_of
from _gpu_util import DEV, log
from test_gpu_prefix import build, check, i32

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("heads,kv,hd,batch,tokens,own", [(4, 2, 64, 19370, 59377, 3), (16, 16, 32, 2047, 68000, 33),
                                                          (2, 1, 128, 70000, 140000, 2)])
def test_as_many_workgroups_as_a_launch_has(heads, kv, hd, batch, tokens, own):
    """Without max_new every request might have nearly all of the tokens: the own keys' workgroups alone are
    a launch's most, and the prefix's come to them."""
    from cobra_amd import ops

    rest = tokens - own * (batch - 2)
    new = [0] + [own] * (batch - 2) + [rest]
    held = [60] + [own + i % 7 for i in range(batch - 2)] + [rest + 2]
    table, pool, q, cu = build(held, new, 0, heads, kv, hd, 16, F16, E4M3, 3)
    dev = [t.to(DEV) for t in pool]
    args = (q.to(DEV), i32(cu), i32(held), i32(table), 0, heads, hd, hd ** -0.5, *dev)
    got = ops.cache_prefix_attn(*args, max_len=500, max_prefix=30000).cpu().double()
    k, v, ks, vs = pool
    some = [1, 2, 3, batch // 2, batch - 2, batch - 1]
    rows = torch.cat([torch.arange(cu[b], cu[b + 1])[-40:] for b in some])
    part = [0]
    for b in some:
        part.append(part[-1] + min(40, new[b]))
    want, mag, top, reach = serve.attend(q[rows, : heads * hd].double(), [0] + part, [held[b] for b in [0] + some],
                                         [table[b] for b in [0] + some], 0, heads, hd, hd ** -0.5, codes_of(k), codes_of(v),
                                         ks, vs, True)
    room = attn_tolerance(want, mag, top, reach, 60 + max(held) + 128, hd, F16, float(vs.max()))
    used = float(((got[rows] - want).abs() / room).max())
    log(f"[prefix launch] {heads}/{kv} x {hd}, {batch} requests: {used:.3f}")
    assert used <= 1.0
    # Cut by hints that fit: either is off by at most 2^-11 of sum p |v| for its weights and as much for its
    # rounding, and the scores' error, well under that.
    near = ops.cache_prefix_attn(*args, max_new=max(own, rest), max_len=500, max_prefix=100).cpu().double()
    largest = float((codes_of(v).abs().amax((1, 2, 3)) * vs.double().amax(1)).max())
    assert float((got - near).abs().max()) <= 2.0 ** -8 * largest


@pytest.mark.parametrize("heads,kv,batch", [(16, 16, 1048575), (32, 2, 8388607)])
@pytest.mark.parametrize("new", [1, 40])
def test_as_many_requests_as_a_launch_has_workgroups(heads, kv, batch, new):
    """batch x kv_heads just under 2^24, a few requests with new tokens among them: as those few alone."""
    from cobra_amd import ops

    hd, where = 32, [0, 5, batch // 2, batch - 1]
    held, few = [90, 30 + new, 2 + new, new], [0, new, new, new]
    table, pool, q, cu = build(held, few, 0, heads, kv, hd, 16, F16, E4M3, 7)
    dev = [t.to(DEV) for t in pool]
    rest = [0, heads, hd, hd ** -0.5, *dev]
    want = ops.cache_prefix_attn(q.to(DEV), i32(cu), i32(held), i32(table), *rest)
    lens = torch.zeros(batch, dtype=torch.int32)
    fresh = torch.zeros(batch + 1, dtype=torch.int32)
    tables = torch.full((batch, len(table[0])), -1, dtype=torch.int32)
    for b, n, f, row in zip(where, held, few, table):
        lens[b], fresh[b + 1], tables[b] = n, f, torch.tensor(row)
    offsets = torch.cumsum(fresh, 0, dtype=torch.int32)
    for hints in ({}, dict(max_new=new, max_len=100, max_prefix=100), dict(max_new=new, max_len=5000, max_prefix=5000)):
        got = ops.cache_prefix_attn(q.to(DEV), offsets.to(DEV), lens.to(DEV), tables.to(DEV), *rest, **hints)
        largest = float((codes_of(pool[1]).abs().amax((1, 2, 3)) * pool[3].double().amax(1)).max())
        assert float((got.double() - want.double()).abs().max()) <= 2.0 ** -8 * largest


def shares(tokens, batch, heads, kv, hd, new, length, prefix):
    """Shares of a row in all, from the workspace."""
    from cobra_amd import _lib

    width = next(w for w in (32, 64, 96, 128, 192, 256) if w >= hd)
    return _lib.lib().cobra_cache_prefix_attn_workspace_bytes(tokens, batch, heads, kv, hd, new, length, prefix) // (
        tokens * heads * (4 * width + 8))


@pytest.mark.parametrize("batch", [2, 3, 4])
@pytest.mark.parametrize("heads,kv,hd,dtype,cache", [(4, 2, 64, F16, E4M3), (4, 1, 256, BF16, I8), (2, 2, 128, BF16, E4M3),
                                                     (2, 1, 40, F16, I8)])
def test_few_requests_behind_a_long_prefix_without_hints(batch, heads, kv, hd, dtype, cache):
    """A table as wide as the prefix's lets the requests' own keys be as many: they are cut in 64 at most,
    where a call without a prefix would take more."""
    held = [20000, 300, 1, 77][:batch]
    new = [0, 3, 1, 1][:batch]
    T = sum(new)
    width = 20000
    assert shares(T, batch, heads, kv, hd, max(1, T - batch + 2), width, width) > 65
    check(held, new, 0, heads, kv, hd, 32, dtype, cache, seed=batch)


@pytest.mark.parametrize("hd,block", [(64, 16), (128, 64), (256, 32)])
def test_all_shares_that_there_may_be(hd, block):
    """192 of a prefix and 64 of a request's own keys, few of them written, or most."""
    assert shares(2, 3, 2, 1, hd, 1, 98304, 98304) == 256
    for held in ([20000, 17500, 40], [700, 16, 3], [0, 17001, 1]):
        check(held, [0, 1, 1], 0, 2, 1, hd, block, F16, E4M3, seed=hd, max_new=1, max_len=98304, max_prefix=98304)
    check([150, 17500, 260], [1, 0, 1], 0, 2, 1, hd, block, BF16, E4M3, seed=hd, max_new=1, max_len=98304, max_prefix=98304)
    check([17500, 17100], [0, 2], 0, 2, 1, hd, block, BF16, I8, seed=hd)
