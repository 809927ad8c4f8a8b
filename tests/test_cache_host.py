"""CPU tests of the 8-bit cache: refusals before any launch, widths, workspaces, and the plain
form the GPU tests compare with."""

import math

import pytest
import torch

from oracle import cache as oc


def _lib():
    from cobra_amd import _lib as m

    return m.lib(), m


def test_cache_width():
    from cobra_amd import ops

    for hd in range(8, 257, 8):
        assert ops.cache_width(hd) == next(w for w in (32, 64, 96, 128, 192, 256) if w >= hd)
    for hd in (0, -8, 4, 12, 33, 264, 1 << 40):
        with pytest.raises(ValueError, match="multiples of 8"):
            ops.cache_width(hd)


def test_abi_rejects_bad_tables():
    lib, _ = _lib()
    ok = dict(lens=64, new=64, table=64, w=4, free=64, nf=8, count=64, slots=64, t=4, cu=64, missing=64, ws=64, b=2,
              bs=16)

    def reserve(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_reserve(a["lens"], a["new"], a["table"], a["w"], a["free"], a["nf"], a["count"],
                                       a["slots"], a["t"], a["cu"], a["missing"], a["ws"], a["b"], a["bs"], None)

    def trim(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_trim(a["lens"], a["new"], a["table"], a["w"], a["free"], a["nf"], a["count"],
                                    a["missing"], a["ws"], a["b"], a["bs"], None)

    for fn in (reserve, trim):
        for kw in (dict(bs=8), dict(bs=48), dict(bs=256), dict(b=-1), dict(w=-1), dict(nf=-1), dict(lens=None),
                   dict(new=None), dict(table=None), dict(free=None), dict(count=None), dict(missing=None),
                   dict(ws=None), dict(lens=66), dict(table=66), dict(w=1 << 31), dict(nf=1 << 31), dict(b=1 << 31)):
            assert fn(**kw) != 0, kw
        assert fn(b=0, lens=None, new=None, table=None) == 0
    for kw in (dict(t=-1), dict(t=1 << 31), dict(slots=None), dict(slots=68), dict(cu=None), dict(cu=66)):
        assert reserve(**kw) != 0, kw


def test_abi_rejects_bad_append_and_attention():
    lib, m = _lib()
    ok = dict(q=256, dt=m.F16, ld=12 * 64, slots=256, k=256, v=256, ks=256, vs=256, cache=m.CACHE_E4M3, t=4, nb=8,
              bs=16, h=8, kv=2, hd=64, cu=256, lens=256, table=256, w=4, ctx=1 << 20, ws=None, wsb=0, b=2, new=1, len=64,
              scale=0.125)

    def append(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_append(a["q"], a["dt"], a["ld"], a["slots"], a["k"], a["v"], a["ks"], a["vs"],
                                      a["cache"], a["t"], a["nb"], a["bs"], a["h"], a["kv"], a["hd"], None)

    def attn(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_attn_fwd(a["q"], a["dt"], a["ld"], a["cu"], a["lens"], a["table"], a["w"], a["k"],
                                        a["v"], a["ks"], a["vs"], a["cache"], a["ctx"], a["ws"], a["wsb"], a["t"],
                                        a["b"], a["nb"], a["bs"], a["h"], a["kv"], a["hd"], a["new"], a["len"],
                                        a["scale"], 1, None)

    shared = (dict(dt=m.F32), dict(dt=9), dict(cache=2), dict(cache=-1), dict(bs=24), dict(hd=60), dict(hd=264),
              dict(hd=0), dict(kv=3), dict(kv=0), dict(h=0), dict(ld=12 * 64 + 4), dict(t=-1), dict(t=1 << 31),
              dict(nb=-1), dict(q=None), dict(q=264), dict(k=None), dict(k=260), dict(v=260), dict(ks=None),
              dict(vs=258))
    for kw in shared:
        assert append(**kw) != 0, kw
        assert attn(**kw) != 0, kw
    assert append(ld=11 * 64) != 0 and append(slots=None) != 0 and append(slots=260) != 0
    assert append(t=0, q=None, slots=None) == 0
    for kw in (dict(ld=7 * 64), dict(cu=None), dict(lens=None), dict(table=None), dict(w=0), dict(ctx=None),
               dict(ctx=264), dict(nb=0), dict(b=-1), dict(new=-1), dict(len=-1), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(cu=258)):
        assert attn(**kw) != 0, kw
    assert attn(t=1 << 30, b=1 << 30, ctx=1 << 50) != 0  # tokens x heads past 2^31
    assert attn(t=1 << 24, b=1 << 24, ctx=1 << 50) != 0  # more workgroups than a launch has
    for ctx in (256, 256 + 3 * 12 * 128 + 8 * 128 - 16, 16):  # over the queries
        assert attn(ctx=ctx) != 0, ctx
    assert attn(t=0, q=None, ctx=None) == 0 and attn(b=0, cu=None) == 0
    # a call that splits its keys needs the workspace it asks for
    need = lib.cobra_cache_attn_workspace_bytes(1, 1, 8, 2, 64, 1, 100000)
    assert need > 0
    assert attn(t=1, b=1, len=100000, w=8192, ws=None, wsb=need) != 0
    assert attn(t=1, b=1, len=100000, w=8192, ws=256, wsb=need - 1) != 0
    assert attn(t=1, b=1, len=100000, w=8192, ws=260, wsb=need) != 0


def test_workspace_query():
    lib, _ = _lib()
    q = lib.cobra_cache_attn_workspace_bytes
    assert q(0, 4, 8, 8, 64, 1, 1000) == 0 and q(4, 0, 8, 8, 64, 1, 1000) == 0
    assert q(4, 4, 8, 3, 64, 1, 1000) == -1 and q(4, 4, 8, 8, 60, 1, 1000) == -1
    assert q(-1, 4, 8, 8, 64, 1, 1000) == -1 and q(4, 4, 8, 8, 64, -1, 1000) == -1
    assert q(8192, 4, 32, 8, 64, 2048, 4096) == 0  # many rows of many heads: no split
    assert q(1 << 22, 1, 8, 8, 64, 1, 100000) == 0  # no workspace for every row of so many
    for length in (1, 1000, 100000, 2 ** 31 - 1, 2 ** 40):
        n = q(64, 64, 8, 8, 64, 1, length)
        assert 0 <= n <= 1025 * 64 * 8 * (64 * 4 + 8)


def test_ops_refuse_before_launch():
    from cobra_amd import ops

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    lens, new, table, free, count = i32(3), i32(3), i32(3, 4), i32(9), i32(1)
    with pytest.raises(ValueError, match="device tensor"):
        ops.cache_reserve(lens, new, table, free, count, 16, 4)
    with pytest.raises(ValueError, match="new_lens"):
        ops.cache_reserve(lens, i32(2), table, free, count, 16, 4)
    with pytest.raises(ValueError, match="lens"):
        ops.cache_reserve(lens.long(), new, table, free, count, 16, 4)
    with pytest.raises(ValueError, match="block_table"):
        ops.cache_trim(lens, new, i32(4, 4), free, count, 16)
    with pytest.raises(ValueError, match="free_count"):
        ops.cache_trim(lens, new, table, free, i32(2), 16)
    k = torch.zeros(5, 2, 16, 64, dtype=torch.int8)
    v = torch.zeros(5, 2, 64, 16, dtype=torch.int8)
    s = torch.ones(5, 2)
    qkv = torch.zeros(6, 8 * 64, dtype=torch.float16)
    slots = torch.zeros(6, dtype=torch.int64)
    with pytest.raises(ValueError, match="device tensor"):
        ops.cache_append(qkv, slots, 4, 64, k, v, s, s)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.cache_append(qkv, slots, 4, 64, k.half(), v, s, s)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.cache_append(qkv, slots, 4, 64, k, v.view(torch.uint8), s, s)
    with pytest.raises(ValueError, match="block_size"):
        ops.cache_append(qkv, slots, 4, 64, k[:, :, :8], v, s, s)
    with pytest.raises(ValueError, match="rows of 96"):
        ops.cache_append(qkv, slots, 4, 72, k, v, s, s)
    with pytest.raises(ValueError, match="v must be"):
        ops.cache_append(qkv, slots, 4, 64, k, k, s, s)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        ops.cache_append(qkv, slots, 5, 64, k, v, s, s)
    with pytest.raises(ValueError, match="v_scale"):
        ops.cache_append(qkv, slots, 4, 64, k, v, s, s.half())
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.cache_append(qkv.float(), slots, 4, 64, k, v, s, s)
    with pytest.raises(ValueError, match="slots"):
        ops.cache_append(qkv, slots[:5], 4, 64, k, v, s, s)
    with pytest.raises(ValueError, match="slots"):
        ops.cache_append(qkv, slots.int(), 4, 64, k, v, s, s)
    cu = i32(4)
    args = (4, 64, 0.125, k, v, s, s)
    with pytest.raises(ValueError, match="device tensor"):
        ops.cache_attn(qkv, cu, lens, table, *args)
    with pytest.raises(ValueError, match="cu must be"):
        ops.cache_attn(qkv, i32(3), lens, table, *args)
    with pytest.raises(ValueError, match="multiple of 8 columns"):
        ops.cache_attn(qkv[:, :252], cu, lens, table, *args)
    with pytest.raises(ValueError, match="multiple of 8 columns"):
        ops.cache_attn(qkv[:, :260], cu, lens, table, *args)
    with pytest.raises(ValueError, match="scale must be positive"):
        ops.cache_attn(qkv, cu, lens, table, 4, 64, 0.0, k, v, s, s)


def test_plain_form_codes_are_torchs():
    """The plain form's e4m3 rounding is torch's conversion for every fp16 value in range."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x.abs() <= 448]
    assert torch.equal(oc.nearest(x.double(), torch.float8_e4m3fn), x.float().to(torch.float8_e4m3fn).double())
    assert oc.nearest(torch.tensor([math.nan, math.inf, -math.inf, 1e30]).double(), torch.float8_e4m3fn).tolist() == \
        [0.0, 448.0, -448.0, 448.0]
    assert [oc.exponent(a, torch.float8_e4m3fn) for a in (0.0, 448.0, 448.1, 1e30, 1e-30)] == [-40, 0, 1, 40, -40]
    assert [oc.exponent(a, torch.int8) for a in (127.0, 127.1, 63.5, 63.6)] == [0, 1, -1, 0]


def test_plain_form_tables_round_trip():
    lens, table, free = [5, 0, 33], [[7, 0, 0], [0, 0, 0], [1, 2, 3]], [9, 8, 6, 5, 4, 0]
    before = [list(lens), list(free)]
    missing, slots, cu, count = oc.reserve(lens, [12, 1, 0], table, free, 16, 14, 5, 6)
    assert (missing, cu, count, lens) == (0, [0, 12, 13, 13], 3, [17, 1, 33])
    assert table[0][:2] == [7, 4] and table[1][0] == 5
    assert slots == [7 * 16 + i for i in range(5, 16)] + [4 * 16, 5 * 16, -1]
    assert oc.trim(lens, before[0], table, free, 16, count, 6) == (0, 5)
    assert [lens, free] == before


def test_cache_refuses_before_it_allocates():
    from cobra_amd import CobraCache

    ok = dict(layers=1, kv_heads=2, head_dim=64, requests=2, num_blocks=4, device="cpu")
    for kw, match in ((dict(layers=0), "layers"), (dict(kv_heads=0), "kv_heads"), (dict(requests=-1), "requests"),
                      (dict(num_blocks=0), "num_blocks"), (dict(block_size=48), "block_size"),
                      (dict(head_dim=60), "multiples of 8"), (dict(), "GPU")):
        with pytest.raises(ValueError, match=match):
            CobraCache(**dict(ok, **kw))
    with pytest.raises(TypeError, match="float8_e4m3fn or int8"):
        CobraCache(**dict(ok, dtype=torch.float16))
