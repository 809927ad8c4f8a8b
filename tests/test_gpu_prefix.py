"""GPU tests of attention behind a shared prefix against the plain form in 64 bits (oracle/serve.py),
within the cache attention's bound (``_cache_util.attn_tolerance``)."""

import random

import pytest
import torch

from oracle import cache as oc
from oracle import serve

from _cache_util import E4M3, I8, attn_tolerance, codes_of, model_tables, poison, random_cache
from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def build(held, new, prefix, heads, kv, hd, block, dtype, cache, seed, lead=0, tail=0):
    """Tables, cache and queries on the host; memory that no request holds is poisoned."""
    num = sum(oc.blocks(h, block) for h in held) + 2
    width = max(1, max(oc.blocks(h, block) for h in held))
    table, _, _ = model_tables(len(held), held, block, num, width, seed)
    k, v, ks, vs = random_cache(num, kv, block, hd, cache, seed, spread=2)
    used = {}
    for b, n in enumerate(held):
        for i in range(oc.blocks(n, block)):
            used[table[b][i]] = min(block, n - i * block)
    for blk in range(num):
        if used.get(blk, 0) < block:
            poison(k, v, blk, used.get(blk, 0))
    g = torch.Generator().manual_seed(seed + 1)
    cu = [lead]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + tail, (heads + 2 * kv) * hd, generator=g)
    kk = codes_of(k) * ks.double()[:, :, None, None]
    q[:, : heads * hd] *= 2.0 / max(float(kk.std()), 1e-6)
    return table, (k, v, ks, vs), q.to(dtype), cu


def check(held, new, prefix, heads, kv, hd, block, dtype, cache, seed=0, causal=True, lead=0, tail=0, **hints):
    from cobra_amd import ops

    table, pool, q, cu = build(held, new, prefix, heads, kv, hd, block, dtype, cache, seed, lead, tail)
    k, v, ks, vs = pool
    scale = hd ** -0.5
    want, mag, top, reach = serve.attend(q[:, : heads * hd].double(), cu, held, table, prefix, heads, hd, scale,
                                         codes_of(k), codes_of(v), ks, vs, causal)
    dev = [t.to(DEV) for t in pool]
    out = torch.full((q.shape[0], heads * hd), 7.0, dtype=dtype, device=DEV)
    got = ops.cache_prefix_attn(q.to(DEV), i32(cu), i32(held), i32(table), prefix, heads, hd, scale, *dev, causal=causal,
                                out=out, **hints)
    torch.cuda.synchronize()
    assert got is out
    got = got.cpu().double()
    # Joining shares of a row: an exponential, a product and an addition more for each of at most 128.
    room = attn_tolerance(want, mag, top, reach, max(held) + held[prefix] + 128, hd, dtype, float(vs.max()))
    live = slice(cu[0], cu[-1])
    err = (got - want).abs()[live]
    used = float((err / room[live]).max()) if err.numel() else 0.0
    log(f"[prefix] held {held[:4]}.. new {new[:4]}.. {heads}/{kv} x {hd} bs{block} {dtype} {cache}: {used:.3f}")
    assert used <= 1.0
    assert (got[: cu[0]] == 7).all() and (got[cu[-1]:] == 7).all()
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("heads,kv,hd,block", [(4, 4, 32, 16), (8, 2, 64, 64), (6, 6, 40, 16), (8, 2, 128, 32),
                                               (4, 2, 80, 128), (2, 1, 168, 32), (6, 2, 256, 64)])
def test_one_token_a_request(heads, kv, hd, block, cache, dtype):
    """Few rows (the direct kernel for both passes) and many (tiles in LDS for the prefix)."""
    for batch in (2, 7, 40):
        rng = random.Random(batch)
        held = [150] + [rng.randint(1, 90) for _ in range(batch)]
        check(held, [0] + [1] * batch, 0, heads, kv, hd, block, dtype, cache, seed=batch)


@pytest.mark.parametrize("prefix_len", [0, 1, 15, 16, 17, 63, 64, 65, 129, 1000, 3001])
@pytest.mark.parametrize("batch", [3, 30])
def test_prefix_lengths(prefix_len, batch):
    held = [(7 * i) % 50 + 1 for i in range(batch)] + [prefix_len]
    check(held, [1] * batch + [0], batch, 8, 2, 64, 16, F16, E4M3, seed=prefix_len)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new_hi,heads,kv,hd", [(5, 8, 2, 64), (5, 4, 4, 32), (40, 16, 2, 64), (200, 4, 2, 128), (90, 4, 1, 256),
                                                (130, 6, 6, 40)])
def test_drafts_and_chunks(new_hi, heads, kv, hd, dtype):
    rng = random.Random(new_hi)
    new = [rng.randint(1, new_hi) for _ in range(5)] + [0]
    held = [n + rng.choice([0, 0, 3, 77]) for n in new[:5]] + [210]
    for causal in (True, False):
        check(held, new, 5, heads, kv, hd, 32, dtype, E4M3, seed=new_hi, causal=causal)


def test_the_prefixs_own_new_tokens_see_only_it():
    check([100, 20, 30], [5, 1, 2], 0, 4, 2, 64, 16, F16, E4M3)
    check([100, 20, 30], [90, 20, 2], 0, 8, 2, 64, 16, BF16, I8)


def test_rows_of_no_request_and_empty_ones():
    """Rows before and behind the requests' stay as they are; requests without new tokens, or without keys."""
    check([64, 5, 0, 9], [0, 5, 0, 1], 0, 4, 2, 64, 16, F16, E4M3, lead=3, tail=70)
    check([0, 3, 2], [0, 1, 2], 0, 4, 2, 64, 16, F16, E4M3, lead=1, tail=2)
    # lengths that say less than the new tokens: those that see nothing of their own see the prefix
    check([20, 1], [0, 3], 0, 4, 2, 64, 16, F16, E4M3)
    # neither: a zero row
    got = check([0, 0], [0, 2], 0, 4, 2, 64, 16, F16, E4M3)
    assert (got == 0).all()


@pytest.mark.parametrize("hints", [dict(max_new=1, max_len=1, max_prefix=1), dict(max_new=500, max_len=9000, max_prefix=9000),
                                   dict(max_new=1, max_len=40, max_prefix=100000)])
def test_hints_are_only_hints(hints):
    for new in ([0, 1, 1, 1], [0, 3, 40, 1]):
        held = [700] + [n + 30 for n in new[1:]]
        check(held, new, 0, 8, 2, 64, 32, F16, E4M3, seed=3, **hints)


def test_pages_outside_the_pool_are_masked():
    from cobra_amd import ops

    held, new = [100, 40, 33], [0, 1, 2]
    table, pool, q, cu = build(held, new, 0, 4, 2, 64, 16, F16, E4M3, 5)
    table[0][2], table[1][0], table[0][6] = -1, 1 << 30, 10 ** 6
    k, v, ks, vs = pool
    want, mag, top, reach = serve.attend(q[:, :256].double(), cu, held, table, 0, 4, 64, 0.125, codes_of(k), codes_of(v),
                                         ks, vs, True)
    got = ops.cache_prefix_attn(q.to(DEV), i32(cu), i32(held), i32(table), 0, 4, 64, 0.125, *[t.to(DEV) for t in pool])
    room = attn_tolerance(want, mag, top, reach, 400, 64, F16, float(vs.max()))
    assert ((got.cpu().double() - want).abs() <= room).all()


@pytest.mark.parametrize("new,hints", [([0, 2, 3, 1], {}), ([0, 2, 3, 1], dict(max_new=300)),
                                       ([0, 2, 3, 1], dict(max_new=300, max_len=1, max_prefix=1))])
def test_bad_offsets_and_lengths_stay_inside(new, hints):
    """Offsets outside the rows, lengths past the table and negative ones: the other requests' rows are right."""
    from cobra_amd import ops

    held = [700, 40, 50, 60]
    table, pool, q, cu = build(held, new, 0, 8, 2, 64, 16, F16, E4M3, 13)
    k, v, ks, vs = pool
    dev = [t.to(DEV) for t in pool]
    for lens, off in (([700, 2 ** 31 - 1, 50, -4], cu), (held, [0, 0, 2, 5, 99]), (held, [-5, -5, 2, 5, 6]),
                      (held, [0, 0, 2, 5, 4])):
        out = torch.full((6, 512), 7.0, dtype=F16, device=DEV)
        ops.cache_prefix_attn(q.to(DEV), i32(off), i32(lens), i32(table), 0, 8, 64, 0.125, *dev, out=out, **hints)
        want, mag, top, reach = serve.attend(q[:, :512].double(), cu, held, table, 0, 8, 64, 0.125, codes_of(k), codes_of(v),
                                             ks, vs, True)
        room = attn_tolerance(want, mag, top, reach, 900, 64, F16, float(vs.max()))
        rows = slice(2, 4 if off[-1] == 4 else 5)  # falling offsets: the rows before the last
        assert ((out.cpu().double() - want).abs() <= room)[rows].all()


@pytest.mark.parametrize("hints", [{}, dict(max_new=300)])
def test_offsets_that_fall_to_the_lowest_value(hints):
    """The last request's rows would be 2^31 - 5 in number; it has none, with a prefix and without."""
    from cobra_amd import ops

    held, off = [700, 40, 50, 60], [0, 0, 2, 5, -2 ** 31]
    table, pool, q, cu = build(held, [0, 2, 3, 1], 0, 8, 2, 64, 16, F16, E4M3, 13)
    rest = [i32(held), i32(table)], [8, 64, 0.125] + [t.to(DEV) for t in pool]
    for prefix in (False, True):
        out = torch.full((6, 512), 7.0, dtype=F16, device=DEV)
        call, row = (ops.cache_prefix_attn, [0]) if prefix else (ops.cache_attn, [])
        call(q.to(DEV), i32(off), *rest[0], *row, *rest[1], out=out, **hints)
        if not prefix:
            want = ops.cache_attn(q.to(DEV), i32(cu), *rest[0], *rest[1], **hints)
            assert torch.equal(out[:5], want[:5])
        assert (out[5] == 7).all()


@pytest.mark.parametrize("heads,kv,hd,held,new", [(4, 4, 128, [200, 70, 5], [0, 1, 1]),
                                                  (32, 2, 128, [3000] + [50] * 70, [0] + [1] * 70),
                                                  (16, 2, 128, [400, 300, 290], [0, 300, 280])])
def test_offsets_past_32_bits(heads, kv, hd, held, new):
    """Blocks that stand more than 2^32 bytes into the pool."""
    from cobra_amd import ops

    table, pool, q, cu = build(held, new, 0, heads, kv, hd, 64, BF16, E4M3, 17)
    k, v, ks, vs = pool
    few, all_blocks = k.shape[0], 2 ** 32 // (kv * 64 * hd) + 2 * k.shape[0]
    dev = []
    for t in pool:
        big = torch.zeros((all_blocks, *t.shape[1:]), dtype=t.dtype, device=DEV)
        big[-few:] = t.to(DEV)
        dev.append(big)
    far = [[i + all_blocks - few if 0 <= i < few else i for i in row] for row in table]
    got = ops.cache_prefix_attn(q.to(DEV), i32(cu), i32(held), i32(far), 0, heads, hd, hd ** -0.5, *dev)
    near = ops.cache_prefix_attn(q.to(DEV), i32(cu), i32(held), i32(table), 0, heads, hd, hd ** -0.5,
                                 *[t.to(DEV) for t in pool])
    assert torch.equal(got, near)
    check(held, new, 0, heads, kv, hd, 64, BF16, E4M3, seed=17)


@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 32), (6, 6, 40), (8, 4, 96), (4, 1, 128), (5, 5, 168), (2, 1, 256)])
@pytest.mark.parametrize("prefix_len", [90, 700])
def test_joins_of_many_requests(heads, kv, hd, prefix_len):
    """Rows of one wave that are of several requests, some without new tokens."""
    new = [0] + [(0, 1, 1, 2, 0, 0, 3)[i % 7] for i in range(150)]
    held = [prefix_len] + [1 + n + 7 * i % 60 for i, n in enumerate(new[1:])]
    check(held, new, 0, heads, kv, hd, 32, BF16, E4M3, seed=hd, lead=5, tail=3)


def test_more_row_tiles_than_compute_units():
    """Prompts whose tiles of rows are more than the chip takes at once, so that the prefix is cut in a few."""
    check([9000, 700, 730, 720], [0, 700, 701, 720], 0, 18, 18, 32, 64, F16, E4M3, seed=2)


def test_two_streams_at_once():
    from cobra_amd import ops

    held, new = [900] + [40] * 30, [0] + [1] * 30
    table, pool, q, cu = build(held, new, 0, 8, 2, 64, 16, F16, E4M3, 19)
    dev = [t.to(DEV) for t in pool]
    rest = [i32(cu), i32(held), i32(table), 0, 8, 64, 0.125, *dev]
    qs = [q.to(DEV), (-0.5 * q).to(DEV)]
    want = [ops.cache_prefix_attn(x, *rest) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for s, x, y in zip(streams, qs, got):
            with torch.cuda.stream(s):
                y.append(ops.cache_prefix_attn(x, *rest))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_groups_with_a_prefix_each():
    """Two groups of neighbouring rows, a call each on views, one result."""
    from cobra_amd import ops

    held, new = [120, 30, 31, 77, 12, 13], [0, 1, 2, 0, 3, 1]
    table, pool, q, cu = build(held, new, 0, 4, 2, 64, 16, F16, E4M3, 9)
    k, v, ks, vs = pool
    dev = [t.to(DEV) for t in pool]
    d_q, d_cu, d_lens, d_table = q.to(DEV), i32(cu), i32(held), i32(table)
    out = torch.empty(q.shape[0], 256, dtype=F16, device=DEV)
    for lo, hi in ((0, 3), (3, 6)):
        ops.cache_prefix_attn(d_q, d_cu[lo:hi + 1], d_lens[lo:hi], d_table[lo:hi], 0, 4, 64, 0.125, *dev, out=out)
    got = out.cpu().double()
    for lo, hi in ((0, 3), (3, 6)):
        want, mag, top, reach = serve.attend(q[:, :256].double(), cu[lo:hi + 1], held[lo:hi], table[lo:hi], 0, 4, 64, 0.125,
                                             codes_of(k), codes_of(v), ks, vs, True)
        room = attn_tolerance(want, mag, top, reach, 400, 64, F16, float(vs.max()))
        at = slice(cu[lo], cu[hi])
        assert ((got - want).abs()[at] <= room[at]).all()


def test_prefix_in_a_graph():
    from cobra_amd import ops

    held, new = [300] + [60] * 20, [0] + [1] * 20
    table, pool, q, cu = build(held, new, 0, 8, 2, 64, 16, F16, E4M3, 11)
    dev = [t.to(DEV) for t in pool]
    d_q, d_cu, d_lens, d_table = q.to(DEV), i32(cu), i32(held), i32(table)
    call = lambda: ops.cache_prefix_attn(d_q, d_cu, d_lens, d_table, 0, 8, 64, 0.125, *dev)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for pre, own in ((300, 60), (17, 1), (299, 33), (0, 5)):
        d_lens.copy_(i32([pre] + [own] * 20))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
