"""GPU tests of attention behind a shared prefix where a launch's limits, or its splits', are reached."""

import pytest
import torch

from oracle import serve

from _cache_util import E4M3, attn_tolerance, codes_of
from _gpu_util import DEV, log
from test_gpu_prefix import build, i32

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.mark.parametrize("heads,kv,hd,batch,tokens,own", [(4, 2, 64, 19370, 59377, 3), (16, 16, 32, 2047, 68000, 33),
                                                          (2, 1, 128, 70000, 140000, 2)])
def test_as_many_workgroups_as_a_launch_has(heads, kv, hd, batch, tokens, own):
    """Without max_new every request might have nearly all of the tokens: the own keys' workgroups alone are
    a launch's most, and go round their row tiles where the prefix's come to them."""
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
