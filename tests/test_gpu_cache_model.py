"""GPU tests of ``CobraTransformer.extend``: the stack over new tokens with a ``CobraCache``.

The comparison runs the blocks in 64 bits on the same rounded weights, taking keys and values
from the codes that the GPU has in its cache (so that both sides attend over the same 8-bit
values), with the reference's gate for fp16 operands (abs <= 2e-3 or rel <= 2e-2, for bf16 the
absolute term at bf16's unit roundoff).  The codes are checked against the 64-bit keys and
values: half a step of the code plus the operand's own rounding.
"""

import pytest
import torch
import torch.nn.functional as F

from oracle import OracleTransformerConfig, compare_outputs, make_model, quantize_like
from oracle import cache as oc

from _cache_util import E4M3, I8, codes_of
from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu


def blocks64(ref, x, cache, lens, new, table, act):
    """(y, worst distance of a code from its value over what the rounding allows) of the new
    tokens, in 64 bits over the cache's codes."""
    att = ref.layers[0].attention
    H, hd = att.num_heads, att.d_model // att.num_heads
    hdp = cache.head_dim
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    r = x.double()
    worst = 0.0
    for i, blk in enumerate(ref.layers):
        a = blk.attention
        h = blk.norm1(r)
        q, k, v = (p(h).view(-1, H, hd) for p in (a.q_proj, a.k_proj, a.v_proj))
        kc, vc = codes_of(cache.k[i]), codes_of(cache.v[i])
        ks, vs = cache.k_scale[i].cpu().double(), cache.v_scale[i].cpu().double()
        t = 0
        for b, n in enumerate(new):
            for p in range(lens[b] - n, lens[b]):
                page, off = table[b][p // cache.block_size], p % cache.block_size
                for code, scale, want in ((kc[page, :, off, :hd], ks[page], k[t]), (vc[page, :, :hd, off], vs[page], v[t])):
                    if p >= lens[b] - 1 or lens[b] - n == 0:  # before any scale that grew later in the step
                        step = 2.0 ** -4 if cache.k[i].dtype == E4M3 else 0.0
                        least = 2.0 ** -10 if cache.k[i].dtype == E4M3 else 0.5
                        err = (code * scale[:, None] - want).abs()
                        # twice for codes rounded again, and the fp16 / bf16 projection
                        room = 2 * torch.maximum(want.abs() * step, least * scale[:, None].expand_as(want)) + \
                            torch.finfo(act).eps * (want.abs() + 4.0)
                        worst = max(worst, float((err / room).max()))
                t += 1
        pad = torch.zeros(q.shape[0], H, hdp, dtype=torch.float64)
        pad[..., :hd] = q
        ctx, _, _, _ = oc.attend(pad.view(-1, H * hdp), cu, lens, table, H, hdp, hd ** -0.5, kc, vc, ks, vs, True)
        r = r + a.out_proj(ctx.view(-1, H, hdp)[..., :hd].reshape(-1, H * hd))
        r = r + blk.ffn_out(F.gelu(blk.ffn_in(blk.norm2(r))))
    return ref.final_norm(r), worst


@pytest.mark.parametrize("cfg,dtype,code,block", [
    ((3, 256, 128, 4, 128, 2, True), torch.float16, E4M3, 16),
    ((3, 256, 128, 4, 256, 2, True), torch.float32, I8, 32),
    ((3, 256, 100, 4, 60, 2, True), torch.float16, E4M3, 64),
    ((3, 256, 256, 2, 256, 1, True), torch.bfloat16, I8, 128),
    ((3, 256, 128, 2, 128, 3, True), torch.bfloat16, E4M3, 16),
])
def test_extend_is_the_blocks_over_the_cache(cfg, dtype, code, block):
    from cobra_amd import CobraTransformer, TransformerConfig

    ref = make_model(OracleTransformerConfig(*cfg), seed=3)
    if dtype != torch.float32:
        quantize_like(ref, dtype)
    mod = CobraTransformer(TransformerConfig(*cfg))
    mod.load_state_dict(ref.state_dict(), strict=True)
    mod = mod.to(device=DEV, dtype=dtype).eval()
    ref = ref.double()
    cache = mod.make_cache(3, 60, block, code)
    g = torch.Generator().manual_seed(4)
    atol = 1.6e-2 if dtype == torch.bfloat16 else 2e-3
    with torch.inference_mode():
        for step, new in enumerate([[50, 3, 0], [1, 1, 33], [1, 1, 1], [4, 0, 1], [0, 130, 0]]):
            T = sum(new)
            x = torch.randn(T + 2, cfg[2], generator=g).to(dtype)
            y, missing = mod.extend(x.to(DEV), cache, torch.tensor(new, dtype=torch.int32, device=DEV))
            torch.cuda.synchronize()
            assert missing.tolist() == [0] and y.dtype == dtype and y.shape == x.shape
            lens, table = cache.lens.tolist(), cache.block_table.tolist()
            want, worst = blocks64(ref, x[:T], cache, lens, new, table, torch.float16 if dtype == torch.float32 else dtype)
            res = compare_outputs(want.float(), y[:T].float().cpu(), atol=atol)
            log(f"[extend] {cfg} {dtype} step {step} lens {lens} max_abs={res.max_abs_error:.3e} "
                f"failed={res.failed_elements} codes {worst:.3f}")
            assert res.passed and worst <= 1.0
    keep = torch.tensor([0, 5, 0], dtype=torch.int32, device=DEV)
    assert cache.trim(keep).tolist() == [0]
    assert cache.free_count.item() == 60 - oc.blocks(5, block)


def test_extend_refuses():
    from cobra_amd import CobraTransformer, TransformerConfig

    def model(causal=True, layers=1):
        return CobraTransformer(TransformerConfig(2, 64, 128, 4, 128, layers, causal)).to(DEV, torch.float16).eval()

    mod = model()
    cache = mod.make_cache(2, 4, 16)
    new = torch.tensor([3, 2], dtype=torch.int32, device=DEV)
    x = torch.zeros(5, 128, dtype=torch.float16, device=DEV)
    with torch.inference_mode():
        with pytest.raises(ValueError, match="causal"):
            model(causal=False).extend(x, cache, new)
        with pytest.raises(ValueError, match="the cache is for 1 layers"):
            model(layers=2).extend(x, cache, new)
        with pytest.raises(ValueError, match=r"x must be \[T, 128\]"):
            mod.extend(x[None], cache, new)
        with pytest.raises(TypeError):
            mod.extend(x.double(), cache, new)
        with pytest.raises(ValueError, match="new_lens"):
            mod.extend(x, cache, new[:1])
        with pytest.raises(ValueError, match="x is on cpu"):
            mod.extend(x.cpu(), cache, new)
        assert cache.lens.tolist() == [0, 0]
        # more than the pool has: nothing is reserved, no length changes
        big = torch.zeros(90, 128, dtype=torch.float16, device=DEV)
        y, missing = mod.extend(big, cache, torch.tensor([40, 50], dtype=torch.int32, device=DEV))
        assert missing.tolist() == [3] and cache.lens.tolist() == [0, 0] and y.shape == big.shape
        y, missing = mod.extend(x, cache, new)
        assert missing.tolist() == [0] and cache.lens.tolist() == [3, 2] and torch.isfinite(y).all()
        y, missing = mod.extend(x[:0], cache, torch.zeros_like(new))
        assert y.shape == (0, 128) and missing.tolist() == [0] and cache.lens.tolist() == [3, 2]


def test_captured_extend_replays():
    """A step of two tokens each captured once: every replay is the eager call on the same state."""
    from cobra_amd import CobraTransformer, TransformerConfig

    mod = CobraTransformer(TransformerConfig(3, 256, 128, 4, 128, 2, True)).to(DEV, torch.float16).eval()
    caches = [mod.make_cache(3, 40, 16) for _ in range(2)]
    new = torch.tensor([2, 2, 2], dtype=torch.int32, device=DEV)
    x = torch.zeros(6, 128, dtype=torch.float16, device=DEV)
    g = torch.Generator().manual_seed(6)
    with torch.inference_mode():
        prompt = torch.randn(70, 128, generator=g).to(DEV, torch.float16)
        for c in caches:
            mod.extend(prompt, c, torch.tensor([40, 0, 30], dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, missing = mod.extend(x, caches[0], new, max_new=2)
        for _ in range(5):
            x.copy_(torch.randn(6, 128, generator=g).to(torch.float16))
            graph.replay()
            want, none = mod.extend(x, caches[1], new, max_new=2)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(missing, none) and missing.item() == 0
            assert torch.equal(caches[0].lens, caches[1].lens)
    assert caches[0].lens.tolist() == [50, 10, 40]
