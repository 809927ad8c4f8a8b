"""GPU tests of ``CobraTransformer`` with rotated and normed queries and keys, 8-bit weights and a shared
prefix: against the blocks in 64 bits (the reference's gate, for bf16 the absolute term at bf16's unit
roundoff), and with 8-bit weights against its operators called one by one, to the bit."""

import pytest
import torch
import torch.nn.functional as F

from oracle import OracleTransformerConfig, compare_outputs, make_model, quantize_like
from oracle import serve

from _cache_util import E4M3, I8, codes_of
from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def build(cfg, dtype, theta=None, norm=False, weights8=False, seed=3):
    """(64-bit reference, its norms' weights, model)."""
    from cobra_amd import CobraTransformer, TransformerConfig

    ref = make_model(OracleTransformerConfig(*cfg), seed=seed)
    if dtype != F32:
        quantize_like(ref, dtype)
    mod = CobraTransformer(TransformerConfig(*cfg, rope_theta=theta, qk_norm=norm), weights8=weights8)
    state = dict(ref.state_dict())
    hd = cfg[2] // cfg[3]
    g = torch.Generator().manual_seed(seed)
    norms = []
    for i in range(cfg[5]):
        w = [(1 + 0.3 * torch.randn(hd, generator=g)).to(dtype).float() for _ in range(2)]
        norms.append(w if norm else [None, None])
        if norm:
            state[f"layers.{i}.q_norm.weight"], state[f"layers.{i}.k_norm.weight"] = w
    mod.load_state_dict(state, strict=True)
    return ref.double(), norms, mod.to(device=DEV, dtype=dtype).eval()


def turn(x, H, hd, pos, theta, w):
    freq = None if theta is None else (float(theta) ** -(torch.arange(0, hd, 2).double() / hd)).float()
    return torch.stack([serve.norm_rope(x[:, h], hd, pos, freq, w, False, 1e-6) for h in range(H)], 1)


def blocks64(ref, norms, x, theta, pos, attend):
    """The stack in 64 bits on rows x at positions pos; attend(layer, q, k, v) -> ctx, all [T, H, hd]."""
    att = ref.layers[0].attention
    H, hd = att.num_heads, att.d_model // att.num_heads
    r = x.double()
    for i, blk in enumerate(ref.layers):
        a = blk.attention
        h = blk.norm1(r)
        q, k, v = (p(h).view(-1, H, hd) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = turn(q, H, hd, pos, theta, norms[i][0]), turn(k, H, hd, pos, theta, norms[i][1])
        r = r + a.out_proj(attend(i, q, k, v).reshape(-1, H * hd))
        r = r + blk.ffn_out(F.gelu(blk.ffn_in(blk.norm2(r))))
    return ref.final_norm(r)


@pytest.mark.parametrize("cfg,dtype,theta,norm", [
    ((2, 70, 128, 4, 128, 2, True), F16, 10000.0, False),
    ((2, 70, 128, 4, 128, 2, False), F32, 10000.0, True),
    ((3, 33, 100, 5, 60, 2, True), F16, 500.0, True),
    ((2, 130, 256, 2, 256, 2, True), BF16, 10000.0, True),
    ((1, 64, 64, 8, 96, 2, True), F16, None, True),
])
def test_forward_is_the_blocks_in_64_bits(cfg, dtype, theta, norm):
    ref, norms, mod = build(cfg, dtype, theta, norm)
    B, S, D, H = cfg[:4]
    g = torch.Generator().manual_seed(5)
    x = torch.randn(B, S, D, generator=g).to(dtype)
    mask = torch.rand(B, S, generator=g) < 0.8
    mask[:, 0] = True
    for m in (None, mask):
        with torch.inference_mode():
            y = mod(x.to(DEV), None if m is None else m.to(DEV)).float().cpu()
        want = torch.zeros(B, S, D, dtype=torch.float64)
        with torch.no_grad():
            for b in range(B):
                keep = torch.ones(S, dtype=torch.bool) if m is None else m[b]

                def attend(i, q, k, v):
                    s = torch.einsum("qhd,khd->hqk", q, k) * (D // H) ** -0.5
                    bad = ~keep[None, :].expand(S, S)
                    if cfg[6]:
                        bad = bad | torch.ones(S, S, dtype=torch.bool).triu(1)
                    p = torch.nan_to_num(torch.softmax(s.masked_fill(bad, -torch.inf), -1))
                    return torch.einsum("hqk,khd->qhd", p, v)

                # Rows are masked after each block only; masked rows are not keys, so the others do not see them.
                want[b] = blocks64(ref, norms, x[b], theta, torch.arange(S), attend)
                want[b][~keep] = 0
        res = compare_outputs(want.float(), y, atol=1.6e-2 if dtype == BF16 else 2e-3)
        log(f"[serve model] {cfg} {dtype} theta {theta} norm {norm}: max_abs={res.max_abs_error:.3e} "
            f"failed={res.failed_elements}")
        assert res.passed


@pytest.mark.parametrize("cfg,dtype,code,block,norm", [
    ((4, 256, 128, 4, 128, 2, True), F16, E4M3, 16, False),
    ((4, 256, 100, 5, 60, 2, True), F32, I8, 32, True),
    ((4, 256, 256, 2, 256, 1, True), BF16, E4M3, 64, True),
])
def test_extend_behind_a_prefix(cfg, dtype, code, block, norm):
    """Prompts and single tokens of three requests behind one prefix, over the codes in the cache."""
    ref, norms, mod = build(cfg, dtype, 10000.0, norm)
    cache = mod.make_cache(4, 60, block, code)
    H, D = cfg[3], cfg[2]
    hd, hdp = D // H, cache.head_dim
    g = torch.Generator().manual_seed(4)
    for step, (new, prefix) in enumerate([([0, 75, 0, 0], None), ([50, 0, 3, 1], 1), ([1, 0, 1, 33], 1), ([1, 4, 1, 0], 1),
                                          ([1, 0, 1, 1], 1)]):
        T = sum(new)
        x = torch.randn(T + 2, D, generator=g).to(dtype)
        with torch.inference_mode():
            y, missing = mod.extend(x.to(DEV), cache, torch.tensor(new, dtype=torch.int32, device=DEV), prefix=prefix)
            torch.cuda.synchronize()
        assert missing.tolist() == [0] and y.dtype == dtype
        lens, table = cache.lens.tolist(), cache.block_table.tolist()
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        pos = torch.cat([torch.arange(lens[b] - n, lens[b]) + (lens[1] if prefix is not None and b != 1 else 0)
                         for b, n in enumerate(new)])

        def attend(i, q, k, v):
            pad = torch.zeros(q.shape[0], H, hdp, dtype=torch.float64)
            pad[..., :hd] = q
            ctx = serve.attend(pad.view(-1, H * hdp), cu, lens, table, -1 if prefix is None else prefix, H, hdp,
                               hd ** -0.5, codes_of(cache.k[i]), codes_of(cache.v[i]), cache.k_scale[i].cpu().double(),
                               cache.v_scale[i].cpu().double(), True)[0]
            return ctx.view(-1, H, hdp)[..., :hd]

        if prefix is None:  # every request sees its own keys alone
            from oracle import cache as oc

            def attend(i, q, k, v):  # noqa: F811
                pad = torch.zeros(q.shape[0], H, hdp, dtype=torch.float64)
                pad[..., :hd] = q
                ctx = oc.attend(pad.view(-1, H * hdp), cu, lens, table, H, hdp, hd ** -0.5, codes_of(cache.k[i]),
                                codes_of(cache.v[i]), cache.k_scale[i].cpu().double(),
                                cache.v_scale[i].cpu().double(), True)[0]
                return ctx.view(-1, H, hdp)[..., :hd]

        with torch.no_grad():
            want = blocks64(ref, norms, x[:T], 10000.0, pos, attend)
        res = compare_outputs(want.float(), y[:T].float().cpu(), atol=1.6e-2 if dtype == BF16 else 2e-3)
        log(f"[serve extend] {cfg} {dtype} step {step} lens {lens}: max_abs={res.max_abs_error:.3e} "
            f"failed={res.failed_elements}")
        assert res.passed


def by_hand(mod, x, B, S, mask=None, cache=None, new=None, prefix=None):
    """What forward and extend do with 8-bit weights, operator by operator, from the parameters."""
    from cobra_amd import ops

    cfg = mod.config
    H, D = cfg.num_heads, cfg.d_model
    hd = D // H
    op = BF16 if x.dtype == BF16 else F16
    T = x.shape[0]
    freq = (float(cfg.rope_theta) ** -(torch.arange(0, hd, 2).double() / hd)).float().to(DEV)
    r = torch.zeros(T, D, dtype=F32, device=DEV)
    l0 = mod.layers[0].norm1
    h = ops.ln_strided(x, D, l0.weight, l0.bias, out_dtype=op, resid_out=r)
    bits = None if mask is None else ops.mask_bits(mask)
    rm = None if mask is None else mask.view(-1)
    pos = None
    if cache is not None:
        slots, cu, _ = cache.reserve(new, T)
        pos = cache.positions(cu, T, prefix)
    for i, blk in enumerate(mod.layers):
        a = blk.attention
        w = torch.cat([a.q_proj.weight, a.k_proj.weight, a.v_proj.weight]).detach()
        b = torch.cat([a.q_proj.bias, a.k_proj.bias, a.v_proj.bias]).detach()
        qkv = ops.linear8(h, *ops.quantize8(w), b)
        ops.qk_norm_rope(qkv, H, H, hd, positions=pos, seq_len=None if cache is not None else S, inv_freq=freq,
                         q_weight=blk.q_norm.weight.detach(), k_weight=blk.k_norm.weight.detach())
        if cache is None:
            ctx = ops.attn(qkv, B, S, H, hd, hd ** -0.5, causal=cfg.causal, key_bits=bits)
        else:
            cache.append(i, qkv, slots, H)
            ctx = torch.zeros(T, D, dtype=op, device=DEV)
            cache.attn(i, qkv, cu, H, hd ** -0.5, out=ctx, prefix=prefix)
        r = ops.linear8(ctx, *ops.quantize8(a.out_proj.weight.detach()), a.out_proj.bias.detach(), out_dtype=F32, resid=r,
                        rmask=rm, mask_branch=True)
        h2 = ops.ln_strided(r, D, blk.norm2.weight, blk.norm2.bias, out_dtype=op)
        hid = ops.linear8(h2, *ops.quantize8(blk.ffn_in.weight.detach()), blk.ffn_in.bias.detach(), gelu=True)
        r = ops.linear8(hid, *ops.quantize8(blk.ffn_out.weight.detach()), blk.ffn_out.bias.detach(), out_dtype=F32, resid=r,
                        rmask=rm)
        last = i == cfg.num_layers - 1
        nxt = mod.final_norm if last else mod.layers[i + 1].norm1
        h = ops.ln_strided(r, D, nxt.weight, nxt.bias, out_dtype=x.dtype if last else op, mask_row=rm if last else None,
                           mask_resid=last and rm is not None, mask_out=last and rm is not None)
    return h


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_weights8_are_the_operators(dtype):
    cfg = (3, 50, 256, 4, 384, 2, True)
    ref, norms, mod = build(cfg, dtype, 10000.0, True, weights8=True)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(3, 50, 256, generator=g).to(dtype).to(DEV)
    mask = (torch.rand(3, 50, generator=g) < 0.7).to(DEV)
    with torch.inference_mode():
        for m in (None, mask):
            y = mod(x, m).clone()
            assert torch.equal(y.view(150, 256), by_hand(mod, x.view(150, 256), 3, 50, m))
        one, two = mod.make_cache(3, 60, 16), mod.make_cache(3, 60, 16)
        for new, prefix in (([40, 0, 0], None), ([0, 30, 9], 0), ([0, 1, 1], 0)):
            T = sum(new)
            n = torch.tensor(new, dtype=torch.int32, device=DEV)
            x = torch.randn(T, 256, generator=g).to(dtype).to(DEV)
            y, missing = mod.extend(x, one, n, prefix=prefix)
            assert missing.tolist() == [0] and torch.equal(y, by_hand(mod, x, 0, 0, cache=two, new=n, prefix=prefix))


def test_weights8_are_near_the_16_bit_model():
    """A value is off by at most 2^-4 of itself after its rounding to e4m3, so a product of rounded
    operands by about that of its norm, twice; four products a block, each added to a stream at least as
    large, and a norm that keeps the ratio: 4 x 2^-3 a block at the very most."""
    cfg = (2, 64, 256, 4, 256, 1, True)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(2, 64, 256, generator=g).half().to(DEV)
    out = []
    for w8 in (False, True):
        _, _, mod = build(cfg, F16, 10000.0, True, weights8=w8)
        with torch.inference_mode():
            out.append(mod(x).float().clone())
    assert float((out[0] - out[1]).norm() / out[0].norm()) <= 4 * 2.0 ** -3
    assert not torch.equal(out[0], out[1])


def test_step_with_prefix_in_a_graph():
    cfg = (3, 64, 128, 4, 128, 2, True)
    _, _, mod = build(cfg, F16, 10000.0, True, weights8=True)
    one, two = mod.make_cache(3, 60, 16), mod.make_cache(3, 60, 16)
    g = torch.Generator().manual_seed(8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    with torch.inference_mode():
        p = torch.randn(45, 128, generator=g).half().to(DEV)
        for c in (one, two):
            mod.extend(p, c, i32([0, 45, 0]))
        x, new = torch.zeros(2, 128, dtype=F16, device=DEV), i32([1, 0, 1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, missing = mod.extend(x, one, new, prefix=1, max_new=1, max_len=64, max_prefix=64)
        for _ in range(20):
            x.copy_(torch.randn(2, 128, generator=g).half())
            graph.replay()
            torch.cuda.synchronize()
            want, _ = mod.extend(x, two, new, prefix=1, max_new=1, max_len=64, max_prefix=64)
            assert missing.tolist() == [0] and torch.equal(y, want)
    assert one.lens.tolist() == two.lens.tolist() == [20, 45, 20]


def test_norms_eps_is_the_modules_own():
    """A changed eps counts from the next call on, eager and captured; the two norms of a block share it."""
    cfg = (2, 33, 64, 4, 64, 1, True)
    _, _, mod = build(cfg, F16, 10000.0, True)
    x = torch.randn(2, 33, 64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    with torch.inference_mode():
        first = mod(x).clone()
        blk = mod.layers[0]
        blk.q_norm.eps = 30.0
        with pytest.raises(ValueError, match="eps"):
            mod(x)
        blk.k_norm.eps = 30.0
        other = mod(x).clone()
        fresh = build(cfg, F16, 10000.0, True)[2]
        fresh.layers[0].q_norm.eps = fresh.layers[0].k_norm.eps = 30.0
        assert torch.equal(other, fresh(x)) and not torch.equal(other, first)
        blk.q_norm.eps = blk.k_norm.eps = 1e-6
        assert torch.equal(mod(x), first)


def test_model_refuses():
    from cobra_amd import CobraTransformer, TransformerConfig

    with pytest.raises(ValueError, match="rope_theta"):
        CobraTransformer(TransformerConfig(1, 8, 64, 4, 64, 1, True, rope_theta=0.0))
    with pytest.raises(ValueError, match="even head_dim"):
        CobraTransformer(TransformerConfig(1, 8, 60, 4, 64, 1, True, rope_theta=1e4))
    _, _, mod = build((2, 64, 128, 4, 128, 1, True), F16)
    cache = mod.make_cache(2, 8)
    x, new = torch.zeros(1, 128, dtype=F16, device=DEV), torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    for prefix in (-1, 2):
        with pytest.raises(ValueError, match="prefix"):
            mod.extend(x, cache, new, prefix=prefix)
    assert cache.lens.tolist() == [0, 0]
