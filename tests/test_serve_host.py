"""CPU tests of the serving step's operators: refusals before any launch, widths, workspaces, the
configuration's options, and the plain forms that the GPU tests compare with."""

import math

import pytest
import torch

from oracle import serve


def _lib():
    from cobra_amd import _lib as m

    return m.lib(), m


def test_width8():
    from cobra_amd import ops

    assert [ops.width8(k) for k in (1, 128, 129, 512, 513, 4096)] == [(128, 4), (128, 4), (256, 4), (512, 4), (640, 8),
                                                                      (4096, 32)]


def test_abi_rejects_bad_products():
    lib, m = _lib()
    ok = dict(a=1 << 20, dt=m.F16, asc=None, w=2 << 20, wsc=3 << 20, bias=None, resid=None, rdt=m.F32, mask=None, epi=0,
              c=4 << 20, cdt=m.F16, ws=None, wsb=0, M=4, N=64, K=256)

    def linear(**kw):
        a = dict(ok, **kw)
        return lib.cobra_linear8_fwd(a["a"], a["dt"], a["asc"], a["w"], a["wsc"], a["bias"], a["resid"], a["rdt"],
                                     a["mask"], a["epi"], a["c"], a["cdt"], a["ws"], a["wsb"], a["M"], a["N"], a["K"],
                                     None)

    for kw in (dict(dt=m.F32), dict(dt=9), dict(cdt=3), dict(cdt=9), dict(M=-1), dict(M=1 << 31), dict(N=0), dict(N=1 << 27),
               dict(K=0), dict(K=1 << 23), dict(a=None), dict(a=(1 << 20) + 8), dict(w=None), dict(w=(2 << 20) + 8),
               dict(wsc=None), dict(wsc=(3 << 20) + 2), dict(c=None), dict(c=(4 << 20) + 8), dict(bias=8), dict(resid=8),
               dict(resid=5 << 20, rdt=3), dict(epi=m.EPI_MASK_OUT), dict(epi=16), dict(epi=m.EPI_MASK_BRANCH),
               dict(epi=m.EPI_MASK_RESID), dict(dt=m.E4M3), dict(dt=m.E4M3, asc=(5 << 20) + 2),
               dict(c=1 << 20), dict(c=(1 << 20) + 4 * 512 - 16), dict(c=2 << 20), dict(c=3 << 20),
               dict(resid=(4 << 20) + 16, rdt=m.F16), dict(resid=4 << 20, rdt=m.F32),
               dict(dt=m.E4M3, asc=5 << 20, c=5 << 20)):
        assert linear(**kw) != 0, kw
    assert linear(M=0, a=None, w=None, c=None) == 0
    need = lib.cobra_linear8_workspace_bytes(100, 64, 256, m.F16)
    assert need == 100 * (256 + 4)
    for kw in (dict(ws=None, wsb=need), dict(ws=6 << 20, wsb=need - 1), dict(ws=(6 << 20) + 8, wsb=need),
               dict(ws=1 << 20, wsb=need), dict(ws=4 << 20, wsb=need)):
        assert linear(M=100, **kw) != 0, kw
    q = lib.cobra_linear8_workspace_bytes
    assert q(0, 64, 256, m.F16) == 0 and q(100, 64, 256, m.E4M3) == 0 and q(16, 64, 256, m.BF16) == 0
    assert q(16, 64, 250, m.BF16) == 0 and q(17, 64, 250, m.BF16) == 17 * 260
    assert q(16, 64, 7, m.BF16) == 16 * 132  # rows under a load's length are quantised first
    assert q(1, 64, 256, m.F32) == -1 and q(-1, 64, 256, m.F16) == -1 and q(1, 0, 256, m.F16) == -1


def test_abi_rejects_bad_quantisation():
    lib, m = _lib()
    ok = dict(x=1 << 20, dt=m.F16, codes=2 << 20, scale=3 << 20, M=4, K=256)

    def quantize(**kw):
        a = dict(ok, **kw)
        return lib.cobra_quantize8(a["x"], a["dt"], a["codes"], a["scale"], a["M"], a["K"], None)

    for kw in (dict(dt=m.E4M3), dict(M=-1), dict(M=1 << 31), dict(K=0), dict(K=1 << 23), dict(M=1 << 29, K=1),
               dict(x=None), dict(x=(1 << 20) + 1), dict(x=(1 << 20) + 2, dt=m.F32), dict(codes=None),
               dict(codes=(2 << 20) + 8), dict(scale=None), dict(scale=(3 << 20) + 2), dict(codes=1 << 20),
               dict(scale=1 << 20), dict(scale=2 << 20)):
        assert quantize(**kw) != 0, kw
    assert quantize(M=0, x=None, codes=None, scale=None) == 0


def test_abi_rejects_bad_rotation():
    lib, m = _lib()
    ok = dict(q=256, dt=m.F16, ld=6 * 64, pos=256, seq=0, freq=256, rot=64, inter=0, qw=None, kw=None, eps=1e-6, t=4, h=4,
              kv=1, hd=64, pitch=64)

    def rope(**kw):
        a = dict(ok, **kw)
        return lib.cobra_qk_norm_rope(a["q"], a["dt"], a["ld"], a["pos"], a["seq"], a["freq"], a["rot"], a["inter"],
                                      a["qw"], a["kw"], a["eps"], a["t"], a["h"], a["kv"], a["hd"], a["pitch"], None)

    for kw in (dict(dt=m.F32), dict(t=-1), dict(t=1 << 31), dict(h=0), dict(kv=0), dict(hd=0), dict(hd=257, pitch=257),
               dict(pitch=63), dict(rot=-2), dict(rot=63), dict(rot=66), dict(ld=5 * 64 - 1), dict(eps=-1.0),
               dict(eps=float("nan")), dict(qw=256), dict(kw=256), dict(q=None), dict(q=257), dict(pos=None),
               dict(pos=258), dict(freq=None), dict(freq=258), dict(qw=256, kw=258), dict(seq=-1), dict(seq=1 << 31)):
        assert rope(**kw) != 0, kw
    assert rope(t=0, q=None, pos=None) == 0
    assert rope(rot=0, q=None) == 0  # neither norm nor rotation


def test_abi_rejects_bad_prefix():
    lib, m = _lib()
    ok = dict(q=256, dt=m.F16, ld=12 * 64, cu=256, lens=256, table=256, w=4, pre=0, k=256, v=256, ks=256, vs=256,
              cache=m.CACHE_E4M3, ctx=1 << 20, ws=1 << 22, wsb=1 << 30, t=4, b=2, nb=8, bs=16, h=8, kv=2, hd=64, new=1,
              len=64, most=64, scale=0.125)

    def attn(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_prefix_attn_fwd(a["q"], a["dt"], a["ld"], a["cu"], a["lens"], a["table"], a["w"], a["pre"],
                                               a["k"], a["v"], a["ks"], a["vs"], a["cache"], a["ctx"], a["ws"], a["wsb"],
                                               a["t"], a["b"], a["nb"], a["bs"], a["h"], a["kv"], a["hd"], a["new"],
                                               a["len"], a["most"], a["scale"], 1, None)

    for kw in (dict(dt=m.F32), dict(cache=2), dict(bs=24), dict(hd=60), dict(kv=3), dict(ld=7 * 64), dict(ld=12 * 64 + 4),
               dict(t=-1), dict(t=1 << 31), dict(nb=0), dict(w=0), dict(b=-1), dict(new=-1), dict(len=-1), dict(most=-1),
               dict(scale=0.0), dict(scale=float("nan")), dict(pre=-1), dict(pre=2), dict(b=0), dict(q=None), dict(q=264),
               dict(k=None), dict(v=260), dict(ks=None), dict(vs=258), dict(cu=None), dict(cu=258), dict(lens=None),
               dict(table=None), dict(ctx=None), dict(ctx=264), dict(ctx=256), dict(ws=None), dict(ws=(1 << 22) + 8),
               dict(wsb=16), dict(t=1 << 30, b=1 << 30, ctx=1 << 50), dict(t=1 << 24, b=1 << 24, ctx=1 << 50)):
        assert attn(**kw) != 0, kw
    assert attn(t=0, q=None, ctx=None) == 0
    q = lib.cobra_cache_prefix_attn_workspace_bytes
    assert q(0, 4, 8, 8, 64, 1, 1000, 1000) == 0 and q(4, 4, 8, 3, 64, 1, 1000, 1000) == -1
    assert q(4, 4, 8, 8, 64, 1, 1000, -1) == -1
    assert q(16384, 8, 32, 8, 128, 2048, 4096, 8192) == 0  # prompts: one pass, nothing to join
    for tokens, batch in ((1, 1), (64, 64), (4096, 4096)):
        for length in (1, 1000, 100000, 2 ** 31 - 1, 2 ** 40):
            n = q(tokens, batch, 8, 8, 64, 1, length, length)
            assert 0 < n <= 256 * tokens * 8 * (64 * 4 + 8)


def test_abi_rejects_bad_positions():
    lib, _ = _lib()
    ok = dict(cu=256, lens=256, out=256, t=4, b=2, pre=-1)

    def positions(**kw):
        a = dict(ok, **kw)
        return lib.cobra_cache_positions(a["cu"], a["lens"], a["out"], a["t"], a["b"], a["pre"], None)

    for kw in (dict(t=-1), dict(t=1 << 31), dict(b=0), dict(b=1 << 31), dict(pre=-2), dict(pre=2), dict(cu=None),
               dict(cu=258), dict(lens=None), dict(lens=258), dict(out=None), dict(out=258)):
        assert positions(**kw) != 0, kw
    assert positions(t=0, cu=None) == 0


def test_ops_refuse_before_launch():
    from cobra_amd import ops

    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    with pytest.raises(ValueError, match="device tensor"):
        ops.quantize8(torch.zeros(4, 8))
    a, w, ws = torch.zeros(3, 200, dtype=torch.float16), torch.zeros(64, 256, dtype=e4m3), torch.zeros(64, 4, dtype=torch.uint8).view(e8m0)
    with pytest.raises(ValueError, match="device tensor"):
        ops.linear8(a, w, ws)
    with pytest.raises(ValueError, match="w must be float8_e4m3fn"):
        ops.linear8(a, w.half(), ws)
    with pytest.raises(ValueError, match="w must be float8_e4m3fn"):
        ops.linear8(a, w[:, :200], ws)
    with pytest.raises(ValueError, match="w_scale must be"):
        ops.linear8(a, w, ws[:, :2])
    with pytest.raises(ValueError, match="w_scale must be"):
        ops.linear8(a, w, ws.view(torch.uint8))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.linear8(a.float(), w, ws)
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.linear8(a[:, :100].contiguous(), w, ws)
    codes, scale = torch.zeros(3, 256, dtype=e4m3), torch.zeros(3, 4, dtype=torch.uint8).view(e8m0)
    with pytest.raises(ValueError, match="out_dtype"):
        ops.linear8(codes, w, ws, a_scale=scale)
    with pytest.raises(ValueError, match="a_scale must be"):
        ops.linear8(codes, w, ws, a_scale=ws, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bias"):
        ops.linear8(a, w, ws, torch.zeros(63))
    with pytest.raises(ValueError, match="resid"):
        ops.linear8(a, w, ws, resid=torch.zeros(3, 63))
    qkv, f = torch.zeros(5, 6 * 64, dtype=torch.float16), torch.ones(32)
    pos = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.qk_norm_rope(qkv.float(), 4, 1, 64, pos, f)
    with pytest.raises(ValueError, match="head_dim"):
        ops.qk_norm_rope(qkv, 4, 1, 264, pos, f)
    with pytest.raises(ValueError, match="head_dim"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f, pitch=32)
    with pytest.raises(ValueError, match="qkv must be"):
        ops.qk_norm_rope(qkv, 6, 1, 64, pos, f)
    with pytest.raises(ValueError, match="inv_freq"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, torch.ones(33))
    with pytest.raises(ValueError, match="inv_freq"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f.double())
    with pytest.raises(ValueError, match="needs positions"):
        ops.qk_norm_rope(qkv, 4, 1, 64, None, f)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos[:4], f)
    with pytest.raises(ValueError, match="seq_len"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f, seq_len=5)
    with pytest.raises(ValueError, match="both"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f, q_weight=torch.ones(64))
    with pytest.raises(ValueError, match="eps"):
        ops.qk_norm_rope(qkv, 4, 1, 64, pos, f, eps=-1.0)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="device tensor"):
        ops.cache_positions(i32(4), i32(3), 5)
    with pytest.raises(ValueError, match="cu must be"):
        ops.cache_positions(i32(3), i32(3), 5)
    k, v, s = torch.zeros(5, 2, 16, 64, dtype=torch.int8), torch.zeros(5, 2, 64, 16, dtype=torch.int8), torch.ones(5, 2)
    with pytest.raises(ValueError, match="device tensor"):
        ops.cache_prefix_attn(qkv, i32(4), i32(3), i32(3, 4), 0, 4, 64, 0.125, k, v, s, s)
    with pytest.raises(ValueError, match="scale must be positive"):
        ops.cache_prefix_attn(qkv, i32(4), i32(3), i32(3, 4), 0, 4, 64, 0.0, k, v, s, s)


def test_config_options_leave_the_model_as_it_is():
    """Without the options the state_dict and the draws are the reference's; the norms draw nothing."""
    from cobra_amd import CobraTransformer, TransformerConfig

    torch.manual_seed(0)
    plain = CobraTransformer(TransformerConfig(1, 8, 64, 4, 64, 2, True))
    torch.manual_seed(0)
    other = CobraTransformer(TransformerConfig(1, 8, 64, 4, 64, 2, True, rope_theta=1e4, qk_norm=True), weights8=True)
    a, b = plain.state_dict(), other.state_dict()
    assert set(b) - set(a) == {f"layers.{i}.{n}_norm.weight" for i in range(2) for n in "qk"}
    assert all(torch.equal(a[n], b[n]) for n in a)
    assert TransformerConfig(1, 8, 64, 4, 64, 2, True) == TransformerConfig(1, 8, 64, 4, 64, 2, True, None, False)


def test_plain_quantisation():
    x = torch.tensor([[448.0, 1.0, math.nan, math.inf, -449.0]])
    codes, scale = serve.quantize(x)
    assert scale.tolist() == [[128, 127, 127, 127]]  # 449 needs 2^1
    assert codes[0, :2].tolist() == [224.0, 0.5] and codes[0, 2:4].isnan().all() and codes[0, 4] == -224.0
    y = torch.randn(3, 300, generator=torch.Generator().manual_seed(0))
    codes, scale = serve.quantize(y)
    assert (serve.values(codes, scale)[:, :300] - y.double()).abs().max() <= 2.0 ** -4 * y.abs().max()
    assert (codes[:, 300:] == 0).all()
    assert torch.equal(codes, codes.to(torch.float8_e4m3fn).double())


def test_plain_rotation_turns():
    """A quarter turn of every pair, in both orders, and lengths kept."""
    x = torch.arange(1.0, 9.0)[None]
    f = torch.full((4,), math.pi / 2)
    one = torch.ones(1, dtype=torch.int32)
    half = serve.norm_rope(x, 8, one, f, None, False, 0.0)
    assert torch.allclose(half, torch.tensor([[-5.0, -6, -7, -8, 1, 2, 3, 4]], dtype=torch.float64), atol=1e-6)
    inter = serve.norm_rope(x, 8, one, f, None, True, 0.0)
    assert torch.allclose(inter, torch.tensor([[-2.0, 1, -4, 3, -6, 5, -8, 7]], dtype=torch.float64), atol=1e-6)
