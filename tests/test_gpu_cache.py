"""GPU tests of the 8-bit key/value cache against its plain form in 64 bits (oracle/cache.py):
tables and slots and the quantised write to the bit, the attention within a bound derived from
its roundings (``_cache_util.attn_tolerance``)."""

import random

import pytest
import torch

from oracle import cache as oc

from _cache_util import E4M3, I8, attn_tolerance, codes_of, model_tables, poison, random_cache
from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# -- tables ---------------------------------------------------------------------------


def run_tables(held, new, block, num_blocks, width, tokens, seed, steps=1):
    """reserve, trim to random lengths, reserve again .. against the plain form."""
    from cobra_amd import ops

    lens = list(held)
    table, free, count = model_tables(len(held), held, block, num_blocks, width, seed)
    rng = random.Random(seed)
    d_lens, d_table, d_free, d_count = i32(lens), i32(table), i32(free), i32([count])
    for step in range(steps):
        missing, slots, cu, count = oc.reserve(lens, new, table, free, block, tokens, count, num_blocks)
        got = ops.cache_reserve(d_lens, i32(new), d_table, d_free, d_count, block, tokens)
        assert got[0].tolist() == slots and got[1].tolist() == cu and got[2].tolist() == [missing], step
        assert d_lens.tolist() == lens and d_table.tolist() == table and d_count.tolist() == [count], step
        keep = [rng.choice([0, -5, n, max(0, n - rng.randint(0, 40)), n + 3]) for n in lens]
        refused, count = oc.trim(lens, keep, table, free, block, count, num_blocks)
        r = ops.cache_trim(d_lens, i32(keep), d_table, d_free, d_count, block)
        assert r.tolist() == [refused], step
        assert d_lens.tolist() == lens and d_count.tolist() == [count], step
        assert d_free.tolist()[:count] == free[:count] and d_table.tolist() == table, step
    return missing


@pytest.mark.parametrize("batch,block,hi_len,hi_new", [
    (1, 16, 0, 1), (1, 128, 40, 300), (3, 16, 100, 40), (64, 64, 700, 6), (37, 32, 60, 500), (1025, 16, 33, 5),
    (2050, 128, 10, 3), (5, 16, 200, 2500),
    (400, 16, 9, 700), (1100, 16, 33, 100)])
def test_tables_follow_the_plain_form(batch, block, hi_len, hi_new):
    rng = random.Random(batch * 1000 + block)
    held = [rng.choice([0, 1, block, block - 1, rng.randint(0, hi_len)]) for _ in range(batch)]
    new = [rng.choice([0, 1, block, rng.randint(0, hi_new)]) for _ in range(batch)]
    width = max(oc.blocks(h + 3 * n, block) for h, n in zip(held, new)) + 1
    need = sum(oc.blocks(h + 3 * n, block) for h, n in zip(held, new)) + 4
    tokens = sum(new) + 5
    log(f"[tables] B{batch} bs{block} tokens {tokens}")
    assert run_tables(held, new, block, need, width, tokens, seed=batch, steps=3) == 0


def test_reserve_refuses_whole_calls():
    """Too few blocks, too short a row, too few slots, bad lengths, a bad count: nothing changes."""
    from cobra_amd import ops

    base = dict(lens=[5, 20, 0], new=[12, 3, 40], count=6)
    table, free, _ = model_tables(3, [5, 20, 0], 16, 9, 4, 3)
    for kw, tokens, want in [
        (dict(count=3), 55, 1), (dict(count=0), 55, 4), (dict(new=[12, 3, 200]), 255, -1), (dict(), 54, -1),
        (dict(new=[12, -1, 40]), 55, -1), (dict(lens=[5, -20, 0]), 55, -1), (dict(count=-1), 55, -1),
        (dict(count=10), 55, -1), (dict(lens=[5, 2 ** 31 - 2, 0]), 55, -1), (dict(new=[0, 0, 0], lens=[5, 20, 65]), 9, -1),
        (dict(), 9000, 0)]:
        c = dict(base, **kw)
        state = [i32(c["lens"]), i32(table), i32(free), i32([c["count"]])]
        before = [t.clone() for t in state]
        slots, cu, missing = ops.cache_reserve(state[0], i32(c["new"]), state[1], state[2], state[3], 16, tokens)
        assert missing.tolist() == [want], (kw, tokens)
        if want:
            assert all(torch.equal(x, y) for x, y in zip(state, before)), kw
            assert slots.tolist() == [-1] * tokens and cu.tolist() == [0] * 4, kw
        else:
            assert slots.tolist()[55:] == [-1] * (tokens - 55) and min(slots.tolist()[:55]) >= 0


def test_trim_refuses_whole_calls():
    from cobra_amd import ops

    table, free, count = model_tables(3, [50, 20, 0], 16, 9, 4, 3)
    for lens, n, want in [([50, 20, 0], count, 0), ([50, 20, 65], count, 1), ([50, -1, 0], count, 1),
                          ([50, 20, 0], 4, 1), ([50, 20, 0], -1, 1)]:
        state = [i32(lens), i32(table), i32(free[:7] if n == 4 else free), i32([n])]
        before = [t.clone() for t in state]
        r = ops.cache_trim(state[0], i32([0, 0, 0]), state[1], state[2], state[3], 16)
        assert r.tolist() == [want], (lens, n)
        if want:
            assert all(torch.equal(x, y) for x, y in zip(state, before))


def test_tables_of_no_request():
    from cobra_amd import ops

    none, table, free, count = i32([]), torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([1, 2]), i32([2])
    slots, cu, missing = ops.cache_reserve(none, none, table, free, count, 16, 3)
    assert slots.tolist() == [-1] * 3 and cu.tolist() == [0] and missing.tolist() == [0]
    assert ops.cache_trim(none, none, table, free, count, 16).tolist() == [0]
    lens, table = i32([0, 0]), torch.zeros(2, 0, dtype=torch.int32, device=DEV)  # no column, nothing asked for
    slots, cu, missing = ops.cache_reserve(lens, i32([0, 0]), table, i32([]), i32([0]), 16, 0)
    assert slots.numel() == 0 and cu.tolist() == [0, 0, 0] and missing.tolist() == [0]


# -- append ---------------------------------------------------------------------------


def check_append(qkv, slots, heads, head_dim, cache):
    """One append on the GPU and in plain form, on host copies of ``cache``; every byte of the
    pool is compared.  Returns the new state."""
    from cobra_amd import ops

    k, v, ks, vs = cache
    want = [k.double(), v.double(), ks.double(), vs.double()]
    oc.append(qkv.double(), slots, heads, head_dim, *want, k.dtype)
    dev = [t.to(DEV) for t in (k, v, ks, vs)]
    ops.cache_append(qkv.to(DEV), torch.tensor(slots, dtype=torch.int64, device=DEV), heads, head_dim, *dev)
    torch.cuda.synchronize()
    got = [t.cpu() for t in dev]
    assert torch.equal(got[2].double(), want[2]) and torch.equal(got[3].double(), want[3])
    for g, w in zip(got[:2], want[:2]):
        # an unwritten NaN code stays one
        assert torch.equal(torch.nan_to_num(g.double(), nan=-1e9), torch.nan_to_num(w, nan=-1e9))
    return got


def append_inputs(tokens, heads, kv, head_dim, dtype, seed, grow=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, (heads + 2 * kv) * head_dim, generator=g)
    return (x * torch.exp(grow * torch.randn(tokens, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("heads,kv,head_dim,block", [
    (4, 4, 32, 16), (2, 1, 8, 128), (6, 6, 40, 16), (8, 2, 64, 64), (4, 2, 72, 32), (8, 1, 128, 128), (3, 3, 168, 64),
    (4, 2, 256, 32)])
def test_append_is_the_plain_form(heads, kv, head_dim, block, cache, dtype):
    """Requests that begin and end anywhere in a block, a token at a time and many at once,
    with magnitudes that make scales grow."""
    rng = random.Random(head_dim * 7 + block)
    pool = 11
    state = random_cache(pool, kv, block, head_dim, cache, seed=head_dim)
    for blk in (2, 5):
        poison(state[0], state[1], blk, 0)
    for step in range(4):
        slots = []
        for blk in rng.sample(range(pool), 6):
            lo = rng.choice([0, 0, 1, block - 1, rng.randrange(block)])
            hi = block if rng.random() < 0.4 else rng.randint(lo, block)
            if step == 3:
                hi = lo + 1
            slots += [blk * block + o for o in range(lo, hi)]
        if not slots:
            continue
        # a poisoned block is only ever begun at offset 0 first
        slots = [s for s in slots if step > 0 or s // block not in (2, 5)] or [0]
        if step == 1:
            slots = list(range(2 * block, 3 * block)) + [5 * block] + [s for s in slots if s // block not in (2, 5)]
        x = append_inputs(len(slots), heads, kv, head_dim, dtype, seed=step)
        state = check_append(x, slots, heads, head_dim, state)


@pytest.mark.parametrize("cache", [E4M3, I8])
def test_append_skips_and_repeats(cache):
    """Slots that are negative or past the pool, and one slot twice (the later token stays)."""
    heads, kv, hd, block, pool = 2, 2, 64, 16, 6
    state = random_cache(pool, kv, block, hd, cache, seed=1)
    slots = [-1, 3 * 16 + 2, 3 * 16 + 3, 3 * 16 + 3, -9, 16 * 6, 1 << 40, -(1 << 62), 0, 1, 0, 5 * 16 + 15, -1]
    x = append_inputs(len(slots), heads, kv, hd, torch.float16, seed=5)
    x[10] *= 30
    state = check_append(x, slots, heads, hd, state)
    check_append(x, [-1] * len(slots), heads, hd, state)
    # more tokens for one block than it has room, all of them repeats
    x = append_inputs(700, heads, kv, hd, torch.float16, seed=6)
    check_append(x, [2 * 16 + (i % 16) for i in range(700)], heads, hd, state)


@pytest.mark.parametrize("cache", [E4M3, I8])
def test_append_replaced_token_beside_a_gap(cache):
    """A run whose first token a later one replaces, with offsets that it leaves out: the replaced
    token's values, a hundred times the others', leave no trace in the scale."""
    heads, kv, hd, block = 2, 2, 64, 16
    state = random_cache(3, kv, block, hd, cache, seed=1)
    x = append_inputs(6, heads, kv, hd, torch.float16, seed=5)
    x[0] *= 100
    x[3] *= 100
    check_append(x, [16 + 5, 16 + 8, 16 + 5, 32, 32 + 9, 32], heads, hd, state)


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_of_extreme_values(cache, dtype):
    """NaN, infinities, zeros, subnormals, the type's largest values, and magnitudes past the
    scales' range (bf16)."""
    heads, kv, hd, block = 1, 1, 32, 16
    state = random_cache(4, kv, block, hd, cache, seed=2)
    x = append_inputs(8, heads, kv, hd, dtype, seed=3)
    big = torch.finfo(dtype).max
    x[0] = 0
    x[1, 40] = float("nan")
    x[1, 70] = float("inf")
    x[2] = float("nan")
    x[3] = float("-inf")
    x[4] = 6e-8 if dtype == torch.float16 else 1e-30
    x[5, ::3] = big
    x[6, 5::4] = -big
    x[7] = 448.0
    for slots in ([16 + 3], [16], [0, 1, 2, 3], [32 + 4]):
        for first in range(8):
            xs = x[first:first + len(slots)]
            if len(xs) == len(slots):
                state = check_append(xs, slots, heads, hd, state)
    check_append(x, [48 + i for i in range(8)], heads, hd, state)


@pytest.mark.parametrize("scale", [448.0, 448.25, 256.0, 127.0, 127.5, 126.0, 1.0])
@pytest.mark.parametrize("cache", [E4M3, I8])
def test_append_scale_borders(cache, scale):
    """Largest values at, next to and away from a border between two scales, in every binade
    that fp16 has."""
    state = random_cache(3, 1, 16, 32, cache, seed=4)
    for e in range(-20, 8):
        x = torch.zeros(1, 96)
        x[0, 32:] = torch.linspace(-1, 1, 64)
        x[0, 40] = x[0, 70] = 1.0
        x = (x * scale * 2.0 ** e).half()
        if torch.isfinite(x).all():
            state = check_append(x, [16 + (e + 20) % 16], 1, 32, state)


def test_append_many_tokens():
    """A prefill's worth: workgroups look through windows of tokens for the blocks' beginnings."""
    heads, kv, hd, block = 4, 4, 64, 32
    held, new = [7, 0, 64, 31, 500], [700, 33, 1, 0, 2000]
    table, free, count = model_tables(5, held, block, 200, 90, 9)
    lens = list(held)
    _, slots, _, _ = oc.reserve(lens, new, table, free, block, sum(new), count, 200)
    for cache, dtype in ((E4M3, torch.bfloat16), (I8, torch.float16)):
        state = random_cache(200, kv, block, hd, cache, seed=8)
        check_append(append_inputs(len(slots), heads, kv, hd, dtype, seed=9), slots, heads, hd, state)


# -- attention --------------------------------------------------------------------------


def attn_case(heads, kv, head_dim, block, held, new, dtype, cache, seed, extra_rows=0, sharp=2.0):
    """Host state of one call: the cache, its tables, the queries (packed q | k | v)."""
    total = [h + n for h, n in zip(held, new)]
    need = sum(oc.blocks(t, block) for t in total)
    width = max(1, max(oc.blocks(t, block) for t in total)) + 2
    table, _, _ = model_tables(len(held), total, block, need + 2, width, seed)
    state = random_cache(need + 2, kv, block, head_dim, cache, seed)
    used = set()
    for b, t in enumerate(total):
        pages = table[b][:oc.blocks(t, block)]
        used |= set(pages)
        if t % block:
            poison(state[0], state[1], pages[-1], t % block)
    for blk in set(range(need + 2)) - used:
        poison(state[0], state[1], blk, 0)
        state[2][blk] = float("nan")
        state[3][blk] = float("inf")
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(new) + extra_rows, (heads + 2 * kv) * head_dim, generator=g)
    # logits of standard deviation about `sharp` whatever the blocks' scales: k ~ 2^-6 .. 1 times 60
    q *= sharp / 8.0
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return {"q": q.to(dtype), "cu": cu, "lens": total, "table": table, "cache": state}


def check_attn(c, heads, head_dim, causal=True, scale=None, log_as="", extra_tol=0.0, **kw):
    from cobra_amd import ops

    scale = head_dim ** -0.5 if scale is None else scale
    k, v, ks, vs = c["cache"]
    dtype, T = c["q"].dtype, c["q"].shape[0]
    want, mag, top, reach = oc.attend(c["q"].double(), c["cu"], c["lens"], c["table"], heads, head_dim, scale,
                                      codes_of(k), codes_of(v), torch.nan_to_num(ks.double()),
                                      torch.nan_to_num(vs.double(), posinf=0.0), causal)
    out = torch.full((T, heads * head_dim), 7.0, dtype=dtype, device=DEV)
    log(f"[cache_attn] {log_as} H{heads} kv{k.shape[1]} hd{head_dim} bs{k.shape[2]} {k.dtype} {dtype} lens "
        f"{c['lens'][:4]} new {c['cu'][-1]} causal={causal}")
    got = ops.cache_attn(c["q"].to(DEV), i32(c["cu"]), i32(c["lens"]), i32(c["table"]), heads, head_dim, scale,
                         *[t.to(DEV) for t in (k, v, ks, vs)], causal=causal, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out
    got = got.cpu().double()
    lo, hi = c["cu"][0], c["cu"][-1]
    assert (got[:lo] == 7).all() and (got[hi:] == 7).all()  # rows of no request are left as they were
    tol = attn_tolerance(want, mag, top, reach, max(c["lens"] + [1]), head_dim, dtype,
                         float(torch.nan_to_num(vs, nan=0.0, posinf=0.0).max())) + extra_tol
    # Past the largest number of the type and half a step the nearest value is an infinity.
    border = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    over = want.abs() - tol > border
    assert torch.equal(got[over], torch.copysign(torch.full_like(want, float("inf")), want)[over])
    some = torch.zeros_like(over)
    some[lo:hi] = True
    some &= want.abs() + tol < border
    off = ((got - want).abs() / tol)[some]
    worst = float(off.max()) if off.numel() else 0.0
    log(f"[cache_attn] worst {worst:.3f} of the bound")
    assert not torch.isnan(got).any() and worst <= 1.0
    return got


GEOMETRIES = [(4, 4, 32, 16), (2, 1, 8, 32), (6, 6, 40, 64), (8, 2, 64, 128), (14, 2, 64, 16), (12, 4, 80, 32),
              (4, 1, 96, 64), (8, 8, 128, 16), (20, 1, 128, 64), (5, 5, 168, 128), (2, 2, 192, 32), (6, 2, 256, 16)]


@pytest.mark.parametrize("heads,kv,head_dim,block", GEOMETRIES)
@pytest.mark.parametrize("cache,dtype", [(E4M3, torch.float16), (E4M3, torch.bfloat16), (I8, torch.float16),
                                         (I8, torch.bfloat16)])
def test_attn_one_token(heads, kv, head_dim, block, cache, dtype):
    """One new token of each request, from an empty cache to several splits of the keys."""
    held = [0, 1, 15, 16, 62, 63, 64, 200, 1023, 1300]
    c = attn_case(heads, kv, head_dim, block, held, [1] * len(held), dtype, cache, seed=head_dim)
    check_attn(c, heads, head_dim, max_new=1, max_len=1301)


@pytest.mark.parametrize("heads,kv,head_dim,block", GEOMETRIES)
@pytest.mark.parametrize("cache,dtype", [(E4M3, torch.float16), (I8, torch.bfloat16)])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_some_tokens(heads, kv, head_dim, block, cache, dtype, causal):
    """Ragged new tokens: the split kernel's rows over several tiles, requests without new
    tokens or without any, the chunk kernel where a request brings many."""
    held = [0, 3, 130, 64, 0, 500]
    few, many = [1, 5, 2, 0, 0, 7], [70, 1, 131, 0, 0, 64]
    for new in (few, many):
        c = attn_case(heads, kv, head_dim, block, held, new, dtype, cache, seed=block, extra_rows=3)
        check_attn(c, heads, head_dim, causal=causal, max_new=max(new))


@pytest.mark.parametrize("max_new,max_len", [(None, None), (1, 1), (1, 64), (3, 700), (100000, 5), (1, 10 ** 12),
                                             (200, 1)])
def test_attn_hints_do_not_change_the_result(max_new, max_len):
    """Expected bounds far from the truth, both ways."""
    for new in ([1, 1, 1], [40, 0, 9], [150, 70, 3]):
        c = attn_case(8, 2, 64, 32, [700, 0, 90], new, torch.float16, E4M3, seed=3)
        check_attn(c, 8, 64, max_new=max_new, max_len=max_len, log_as=f"hints {max_new} {max_len}")


def test_attn_more_rows_than_keys_seen():
    """Lengths that say less than the new tokens: the first rows see no key and are zero."""
    for new in ([9, 4], [200, 70]):
        c = attn_case(4, 2, 64, 16, [0, 0], new, torch.float16, E4M3, seed=5)
        c["lens"] = [3, 0]
        got = check_attn(c, 4, 64)
        assert (got[: new[0] - 3] == 0).all() and (got[new[0]:] == 0).all()


def test_attn_masks_blocks_outside_the_pool():
    for new in ([1, 1], [90, 5]):
        c = attn_case(4, 2, 64, 16, [400, 300], new, torch.bfloat16, E4M3, seed=6)
        c["table"][0][3] = -1
        c["table"][0][7] = 1 << 30
        c["table"][1][0] = c["cache"][0].shape[0]
        check_attn(c, 4, 64)
        c["table"][1] = [-1] * len(c["table"][1])  # a request whose every block is none: zero rows
        got = check_attn(c, 4, 64)
        assert (got[c["cu"][1]:] == 0).all()


def test_attn_bad_lengths_stay_inside():
    """Lengths past the table, negative ones, and offsets outside the rows: bounded, and the
    other requests' rows are right."""
    from cobra_amd import ops

    c = attn_case(4, 4, 32, 16, [40, 50, 60], [2, 3, 1], torch.float16, E4M3, seed=7)
    check_attn(c, 4, 32)
    want, mag, top, reach = oc.attend(c["q"].double(), c["cu"], c["lens"], c["table"], 4, 32, 0.2,
                                      *[codes_of(t) for t in c["cache"][:2]],
                                      *[torch.nan_to_num(t.double(), posinf=0.0) for t in c["cache"][2:]], True)
    for lens, cu in (([2 ** 31 - 1, 53, -4], c["cu"]), (c["lens"], [0, 2, 5, 99]), (c["lens"], [-3, 2, 5, 4])):
        out = torch.full((6, 128), 7.0, dtype=torch.float16, device=DEV)
        ops.cache_attn(c["q"].to(DEV), i32(cu), i32(lens), i32(c["table"]), 4, 32, 0.2,
                       *[t.to(DEV) for t in c["cache"]], out=out)
        tol = attn_tolerance(want, mag, top, reach, 63, 32, torch.float16, 1.0)
        assert ((out.cpu().double() - want).abs() <= tol)[2:5].all()


def test_attn_of_plain_queries_and_wide_rows():
    """q alone, the packed buffer, and a wider one give the same rows."""
    from cobra_amd import ops

    c = attn_case(8, 2, 64, 32, [300, 20], [1, 6], torch.float16, E4M3, seed=8)
    got = check_attn(c, 8, 64)
    q = c["q"].to(DEV)
    rest = [i32(c["cu"]), i32(c["lens"]), i32(c["table"]), 8, 64, 0.125, *[t.to(DEV) for t in c["cache"]]]
    for x in (q[:, :512].contiguous(), torch.cat([q, q[:, :56]], 1).contiguous()):
        assert torch.equal(ops.cache_attn(x, *rest).cpu().double(), got)


def test_attn_nan_query_stays_in_its_row():
    c = attn_case(4, 2, 64, 16, [100, 30], [3, 2], torch.float16, E4M3, seed=9)
    clean = check_attn(c, 4, 64)
    from cobra_amd import ops

    q = c["q"].clone()
    q[1, 70] = float("nan")  # token 1, head 1
    out = ops.cache_attn(q.to(DEV), i32(c["cu"]), i32(c["lens"]), i32(c["table"]), 4, 64, 0.125,
                         *[t.to(DEV) for t in c["cache"]]).cpu().double()
    assert torch.isnan(out[1, 64:128]).all()
    out[1, 64:128] = clean[1, 64:128]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attn_scales_far_apart(cache, dtype):
    """Neighbouring blocks whose scales differ by 2^30 and more, for keys and values (in fp16
    some results are past its range)."""
    for new in ([1], [80]):
        c = attn_case(2, 2, 64, 16, [333], new, dtype, cache, seed=10)
        k, v, ks, vs = c["cache"]
        n = ks.shape[0]
        vs.copy_(torch.ldexp(torch.ones(n, 2), (torch.arange(n) % 5 - 2)[:, None] * torch.tensor([[8, 15]])))
        ks.copy_(torch.ldexp(torch.ones(n, 2), -(torch.arange(n) % 3)[:, None] * 10 - 5 + torch.tensor([[0, 1]])))
        poison(k, v, c["table"][0][oc.blocks(c["lens"][0], 16) - 1], c["lens"][0] % 16)
        check_attn(c, 2, 64)


def test_attn_scales_of_any_value():
    """Scales that are no powers of two, and some outside [2^-40, 2^40], which are taken as its ends."""
    for new in ([1, 1], [90, 4]):
        c = attn_case(4, 2, 64, 16, [300, 70], new, torch.bfloat16, E4M3, seed=12)
        k, v, ks, vs = c["cache"]
        g = torch.Generator().manual_seed(13)
        used = torch.isfinite(vs)
        ks.copy_(torch.where(used, torch.exp(torch.randn(ks.shape, generator=g)) * 0.01, ks))
        vs.copy_(torch.where(used, torch.exp(3 * torch.randn(vs.shape, generator=g)), vs))
        check_attn(c, 4, 64)
        first = c["table"][0][0]
        vs[first] = 1e-20
        vs[c["table"][1][0]] = 0.0
        want = [t.clone() for t in c["cache"]]
        want[3][first] = want[3][c["table"][1][0]] = 2.0 ** -40
        got = check_attn(dict(c, cache=want), 4, 64)
        assert torch.equal(got, check_attn(c, 4, 64, extra_tol=64 * 448 * 2.0 ** -40))


def test_attn_one_long_request_of_thousands():
    """Without max_new the launch is shaped for any request's having all the tokens: more row tiles
    than a grid takes, which workgroups go round.  The result is that of the fitting hint."""
    from cobra_amd import ops

    B, long, H, hd, keys = 6000, 60000, 8, 8, 30
    k, v, ks, vs = (t.to(DEV) for t in random_cache(2, H, 32, hd, E4M3, seed=3))
    T = B - 1 + long
    q = (torch.randn(T, H * hd, generator=torch.Generator().manual_seed(5)) / 8).to(DEV, torch.bfloat16)
    cu = torch.arange(B + 1, dtype=torch.int32)
    cu[4001:] += long - 1
    lens = torch.full((B,), keys, dtype=torch.int32, device=DEV)
    table = torch.ones(B, 1, dtype=torch.int32, device=DEV)

    def run(**kw):
        return ops.cache_attn(q, cu.to(DEV), lens, table, H, hd, 0.3, k, v, ks, vs, causal=False, **kw)

    got = run()
    assert torch.equal(got, run(max_new=long))
    kd = codes_of(k)[1, :, :keys, :hd] * ks[1].cpu().double()[:, None, None]
    vd = (codes_of(v)[1, :, :hd, :keys] * vs[1].cpu().double()[:, None, None]).transpose(1, 2)
    rows = torch.cat([torch.arange(3995, 4100), torch.arange(4000 + long - 90, 4000 + long + 90)])
    s = 0.3 * q.cpu().double()[rows].view(-1, H, hd).transpose(0, 1) @ kd.transpose(1, 2).contiguous()
    want = (torch.softmax(s, -1) @ vd).transpose(0, 1).reshape(len(rows), -1)
    # bf16's half step; every weight 2^-11 of itself for fp16, at most the largest |v| of a head
    err = (got.cpu().double()[rows] - want).abs()
    assert (err <= want.abs() * 2.0 ** -8 + vd.abs().max() * 2.0 ** -9).all()


def test_attn_refuses_an_output_over_its_queries():
    from cobra_amd import ops

    c = attn_case(4, 2, 64, 16, [30], [6], torch.float16, E4M3, seed=2)
    k, v, ks, vs = (t.to(DEV) for t in c["cache"])
    q = c["q"].to(DEV)
    a = (i32(c["cu"]), i32(c["lens"]), i32(c["table"]), 4, 64, 0.125, k, v, ks, vs)
    for x, out in ((q, q.view(-1)[:6 * 256].view(6, 256)), (q[:, :256].contiguous(), None)):
        with pytest.raises(RuntimeError):
            ops.cache_attn(x, *a, out=x if out is None else out)


def test_tensors_that_are_not_rows_are_refused():
    """Strided views, wrong types and shapes: an error before anything is launched or changed."""
    from cobra_amd import ops

    c = attn_case(4, 2, 64, 16, [30, 5], [6, 1], torch.float16, E4M3, seed=2)
    k, v, ks, vs = (t.to(DEV) for t in c["cache"])
    q, cu, lens, table = c["q"].to(DEV), i32(c["cu"]), i32(c["lens"]), i32(c["table"])
    wide = torch.cat([q, q], 1)
    good = dict(q=q, cu=cu, lens=lens, table=table, k=k, v=v, ks=ks, vs=vs)

    def attn(**kw):
        a = dict(good, **kw)
        return ops.cache_attn(a["q"], a["cu"], a["lens"], a["table"], 4, 64, 0.125, a["k"], a["v"], a["ks"], a["vs"])

    def append(**kw):
        a = dict(good, slots=torch.arange(7, device=DEV), **kw)
        ops.cache_append(a["q"], a["slots"], 4, 64, a["k"], a["v"], a["ks"], a["vs"])

    state = (k.view(torch.uint8), v.view(torch.uint8), ks.view(torch.int32))  # bits: unused scales are NaN
    before = [t.clone() for t in state]
    flat = q.view(-1)
    bad = [dict(q=wide[:, :512]), dict(q=wide[:, ::2]), dict(q=q.float()), dict(q=q.cpu()), dict(q=q[None]),
           dict(q=flat[4:4 + 6 * 512].view(6, 512)), dict(k=k.transpose(0, 1)), dict(k=k.view(torch.uint8)),
           dict(v=v.transpose(2, 3)), dict(v=v[:-1]), dict(ks=ks.t()), dict(vs=vs.double()), dict(vs=vs[:, :1])]
    for kw in bad:
        for fn in (attn, append):
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                fn(**kw)
    for kw in (dict(cu=cu.long()), dict(cu=cu[:-1]), dict(lens=i32(c["lens"] * 2)[::2]), dict(table=table.t()),
               dict(table=table[:, ::2]), dict(lens=lens.cpu())):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            attn(**kw)
    lens4 = i32([3, 3, 3, 3])
    for kw in (dict(lens=lens4[::2]), dict(new=lens4), dict(table=table.t()), dict(count=i32([1, 1])), dict(bs=24)):
        a = dict(dict(lens=lens, new=i32([1, 1]), table=table, count=i32([0]), bs=16), **kw)
        for call in (lambda: ops.cache_reserve(a["lens"], a["new"], a["table"], i32([0]), a["count"], a["bs"], 4),
                     lambda: ops.cache_trim(a["lens"], a["new"], a["table"], i32([0]), a["count"], a["bs"])):
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                call()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(before, state))
    assert lens.tolist() == c["lens"]


def test_reserve_without_memory_changes_nothing():
    from cobra_amd import ops

    lens, count = i32([3]), i32([1])
    table, free = i32([[0, 0]]), i32([1])
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.02)
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            ops.cache_reserve(lens, i32([1]), table, free, count, 16, 2 ** 31 - 1)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert lens.tolist() == [3] and count.tolist() == [1]


def test_attn_long_split():
    """One request of tens of thousands of keys over many splits, and a short one beside it."""
    for cache, dtype in ((E4M3, torch.float16), (I8, torch.bfloat16)):
        c = attn_case(4, 1, 64, 128, [40001, 5], [2, 1], dtype, cache, seed=11)
        check_attn(c, 4, 64, max_new=2, max_len=40003)


def test_attn_past_32_bit_offsets():
    """Blocks that lie more than 2^32 bytes into the pool, written and read."""
    from cobra_amd import ops

    heads, kv, hd, bs, n = 2, 2, 256, 128, 70000  # 64 KiB a block
    k = torch.empty(n, kv, bs, hd, dtype=I8, device=DEV)
    v = torch.empty(n, kv, hd, bs, dtype=I8, device=DEV)
    ks, vs = (torch.empty(n, kv, device=DEV) for _ in range(2))
    ids = [69999, 3, 69998, 40000]
    lens = [4 * bs - 3]
    slots = [ids[p // bs] * bs + p % bs for p in range(lens[0])]
    x = append_inputs(lens[0], heads, kv, hd, torch.float16, seed=1, grow=0.1)
    ops.cache_append(x.to(DEV), torch.tensor(slots, device=DEV), heads, hd, k, v, ks, vs)
    at = torch.tensor(ids, device=DEV)
    small = [t[at].cpu() for t in (k, v, ks, vs)]
    want = random_cache(4, kv, bs, hd, I8, seed=1)
    want = [codes_of(want[0]), codes_of(want[1]), want[2].double(), want[3].double()]
    oc.append(x.double(), list(range(lens[0])), heads, hd, *want, I8)
    live = torch.arange(4 * bs) < lens[0]
    for got, w, order in ((small[0], want[0], (0, 2, 1, 3)), (small[1], want[1], (0, 3, 1, 2))):
        assert torch.equal(codes_of(got).permute(order).reshape(4 * bs, -1)[live],
                           w.permute(order).reshape(4 * bs, -1)[live])
    q = x[-1:].contiguous()
    out = ops.cache_attn(q.to(DEV), i32([0, 1]), i32(lens), i32([ids]), heads, hd, 0.0625, k, v, ks, vs)
    ref, mag, top, reach = oc.attend(q.double(), [0, 1], lens, [[0, 1, 2, 3]], heads, hd, 0.0625, *want, True)
    tol = attn_tolerance(ref, mag, top, reach, lens[0], hd, torch.float16, float(vs[at].max()))
    assert ((out.cpu().double() - ref).abs() <= tol).all()


# -- together -----------------------------------------------------------------------------


def serve(steps, graph=False, stream=None):
    """A batch of requests through reserve, append and attention, with drafts taken back:
    every step's attention against the plain form over what the cache then holds."""
    from cobra_amd import ops

    heads, kv, hd, block, pool, B = 4, 2, 64, 16, 60, 3
    scale = hd ** -0.5
    lens, table, free, count = [0] * B, [[0] * 20 for _ in range(B)], list(range(pool))[::-1], pool
    state = [torch.zeros(pool, kv, block, hd, dtype=E4M3), torch.zeros(pool, kv, hd, block, dtype=E4M3),
             torch.ones(pool, kv), torch.ones(pool, kv)]
    want = [codes_of(state[0]), codes_of(state[1]), state[2].double(), state[3].double()]
    d = [t.to(DEV) for t in state]
    t_lens, t_table, t_free, t_count = i32(lens), i32(table), i32(free), i32([count])
    rng = random.Random(4)
    g = torch.Generator().manual_seed(4)
    for step in range(steps):
        new = [rng.choice([0, 1, 1, 4, 37]) if step else 50 for _ in range(B)]
        T = sum(new) + 2
        x = (torch.randn(T, (heads + 2 * kv) * hd, generator=g) * (1 + step)).half()
        t_new, xd = i32(new), x.to(DEV)
        slots, cu, missing = ops.cache_reserve(t_lens, t_new, t_table, t_free, t_count, block, T)
        ops.cache_append(xd, slots, heads, hd, *d)
        out = torch.zeros(T, heads * hd, dtype=torch.float16, device=DEV)
        ops.cache_attn(xd, cu, t_lens, t_table, heads, hd, scale, *d, out=out)
        miss, s, c, count = oc.reserve(lens, new, table, free, block, T, count, pool)
        oc.append(x.double(), s, heads, hd, *want, E4M3)
        ref, mag, top, reach = oc.attend(x.double(), c, lens, table, heads, hd, scale, *want, True)
        assert missing.tolist() == [0] and miss == 0 and slots.tolist() == s
        tol = attn_tolerance(ref, mag, top, reach, max(lens), hd, torch.float16, float(want[3].max()))
        off = ((out.cpu().double() - ref).abs() / tol)[: c[-1]]
        log(f"[serve] step {step} lens {lens} worst {float(off.max()) if off.numel() else 0:.3f}")
        assert not off.numel() or off.max() <= 1
        keep = [max(0, n - rng.choice([0, 0, 2])) if rng.random() < 0.9 else 0 for n in lens]
        assert ops.cache_trim(t_lens, i32(keep), t_table, t_free, t_count, block).tolist() == [0]
        _, count = oc.trim(lens, keep, table, free, block, count, pool)
        assert t_lens.tolist() == lens and t_free.tolist()[:count] == free[:count]


def test_serve_loop():
    serve(8)


def test_serve_loop_on_another_stream():
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        serve(4)


def test_captured_decode_step_replays():
    """A step of one token each (tables, write, attention) captured once and replayed with new
    tokens, against the same steps run eagerly, eager work and a synchronisation in between."""
    from cobra_amd import ops

    heads, kv, hd, block, pool, B = 8, 2, 64, 16, 80, 4
    g = torch.Generator().manual_seed(12)
    steps = [torch.randn(B, (heads + 2 * kv) * hd, generator=g).half().to(DEV) for _ in range(7)]
    prompt = torch.randn(300 * B, (heads + 2 * kv) * hd, generator=g).half().to(DEV)

    def fresh():
        t = {"lens": i32([0] * B), "table": torch.zeros(B, 24, dtype=torch.int32, device=DEV),
             "free": torch.arange(pool, dtype=torch.int32, device=DEV), "count": i32([pool]), "one": i32([1] * B),
             "x": steps[0].clone(),
             "cache": [torch.zeros(pool, kv, block, hd, dtype=I8, device=DEV),
                       torch.zeros(pool, kv, hd, block, dtype=I8, device=DEV),
                       torch.ones(pool, kv, device=DEV), torch.ones(pool, kv, device=DEV)]}
        slots, _, missing = ops.cache_reserve(t["lens"], i32([300, 17, 0, 250]), t["table"], t["free"], t["count"],
                                              block, 567)
        ops.cache_append(prompt[:567].contiguous(), slots, heads, hd, *t["cache"])
        assert missing.tolist() == [0]
        return t

    def step(t):
        slots, cu, _ = ops.cache_reserve(t["lens"], t["one"], t["table"], t["free"], t["count"], block, B)
        ops.cache_append(t["x"], slots, heads, hd, *t["cache"])
        return ops.cache_attn(t["x"], cu, t["lens"], t["table"], heads, hd, 0.125, *t["cache"], max_new=1, max_len=384)

    eager = fresh()
    want = []
    for x in steps:
        eager["x"].copy_(x)
        want.append(step(eager).clone())
    t = fresh()
    saved = {n: v.clone() for n, v in t.items() if torch.is_tensor(v)}, [c.clone() for c in t["cache"]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t)
    torch.cuda.current_stream().wait_stream(side)
    for n, v in saved[0].items():
        t[n].copy_(v)
    for c, v in zip(t["cache"], saved[1]):
        c.copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(t)
    for x, w in zip(steps, want):
        t["x"].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        (prompt[:64].float() @ prompt[:64].float().T).sum().item()
        assert torch.equal(out, w)
    assert torch.equal(t["lens"], eager["lens"]) and torch.equal(t["table"], eager["table"])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(t["cache"], eager["cache"]))
