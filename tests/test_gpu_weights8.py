"""GPU tests of ``CobraTransformer(weights8=True)`` operator by operator against 64 bits, in geometries that
need padding too: every product from the parameters themselves, quantised by the plain form, and what it took
and gave; the norms, rotations and attention between them from the products' own results."""

import pytest
import torch

from oracle import cache as oc
from oracle import compare_outputs, serve

from _cache_util import E4M3, I8, codes_of
from _gpu_util import DEV, log
from test_gpu_linear8 import bound
from test_gpu_serve_model import build, turn

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture
def products(monkeypatch):
    """(activations, result, keywords) of every ``ops.linear8`` in order, on the host."""
    from cobra_amd import ops

    seen, call = [], ops.linear8

    def recorded(a, *args, **kw):
        y = call(a, *args, **kw)
        torch.cuda.synchronize()
        seen.append((a.cpu().clone(), y.cpu().clone(), kw))
        return y

    monkeypatch.setattr(ops, "linear8", recorded)
    return seen


def up8(n):
    return -(-n // 8) * 8


def padded(blk, cfg):
    """(weight, bias) of a block's four products in the kernels' layout, from the parameters: each head's
    rows or columns and each width filled up to a multiple of 8 with zeros."""
    D, H, Fd = cfg[2], cfg[3], cfg[4]
    hd, dp, fp = D // H, up8(D), up8(Fd)
    hp = up8(hd)
    att = blk.attention
    heads = torch.cat([torch.arange(h * hp, h * hp + hd) for h in range(H)])  # where columns of all heads stand
    out = []
    for layers, rows, to, cols, wide in (
            ((att.q_proj, att.k_proj, att.v_proj), heads, H * hp, torch.arange(D), dp),
            ((att.out_proj,), torch.arange(D), dp, heads, H * hp),
            ((blk.ffn_in,), torch.arange(Fd), fp, torch.arange(D), dp),
            ((blk.ffn_out,), torch.arange(D), dp, torch.arange(Fd), fp)):
        w, b = torch.zeros(len(layers) * to, wide, dtype=torch.float64), torch.zeros(len(layers) * to, dtype=torch.float64)
        for i, layer in enumerate(layers):
            at = i * to + rows
            w[at[:, None], cols] = layer.weight.detach().cpu().double()
            b[at] = layer.bias.detach().cpu().double()
        out.append((w, b))
    return out, heads


def norm64(r, ln):
    x = r.double()
    y = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + ln.eps)
    return y * ln.weight.detach().cpu().double() + ln.bias.detach().cpu().double()


def check_norm(got, r, ln, D):
    """The first D columns: fp32 sums of D values, a square root, a division and two operations, and one
    rounding to the result's type; the others zero."""
    want = norm64(r[:, :D], ln)
    e32 = (D + 16) * 2.0 ** -24 * (1 + r[:, :D].double().abs().amax(1, keepdim=True))
    scale = ln.weight.detach().cpu().double().abs().max() / torch.sqrt(r[:, :D].double().var(1, unbiased=False, keepdim=True)
                                                                       + ln.eps)
    least = 2.0 ** -25 if got.dtype == F16 else 0.0
    room = e32 * (scale + want.abs() + 1) + torch.finfo(got.dtype).eps / 2 * want.abs() + least
    assert ((got[:, :D].double() - want).abs() <= 1.01 * room).all()
    assert (got[:, D:] == 0).all()


def check_stack(mod, cfg, norms, seen, x, y, theta, pos, attend, keep=None):
    """Everything that a call did, from what its products took and gave; attend(layer, q, k, v) in 64 bits."""
    D, H, n = cfg[2], cfg[3], cfg[5]
    hd = D // H
    hp = up8(hd)
    op = BF16 if x.dtype == BF16 else F16
    T = x.shape[0]
    rm = None if keep is None else keep.cpu().view(-1)
    assert len(seen) == 4 * n
    r = torch.zeros(T, up8(D))
    r[:, :D] = x.float()
    for i, blk in enumerate(mod.layers):
        weights, heads = padded(blk, cfg)
        parts = seen[4 * i:4 * i + 4]
        for j, ((w, b), (a, out, _)) in enumerate(zip(weights, parts)):
            resid = (None, r, None, parts[1][1])[j]
            aq, wq = serve.values(*serve.quantize(a)), serve.values(*serve.quantize(w.to(blk.ffn_in.weight.dtype)))
            want, mag = serve.linear(aq, wq, b, j == 2, resid, rm if j in (1, 3) else None, j == 1)
            cut = serve.cut_of_eights(aq, wq) if T > 16 and out.dtype == BF16 else 0.0
            room = bound(want, mag, aq.shape[1], j == 2, out.dtype, cut)
            assert out.dtype == (F32 if j in (1, 3) else op) and a.dtype == op
            assert ((out.double() - want).abs() <= room).all(), (i, j)
        (h, qkv, _), (ctx, r1, _), (h2, hid, _), (a2, r2, _) = parts
        check_norm(h, r, blk.norm1, D)
        check_norm(h2, r1, blk.norm2, D)
        assert torch.equal(hid, a2)
        q, k, v = (qkv[:, j * H * hp:(j + 1) * H * hp][:, heads].double().view(T, H, hd) for j in range(3))
        # Rotated queries and keys are rounded to the operand type once.
        q, k = (turn(t, H, hd, pos, theta, w).to(op).double() for t, w in zip((q, k), norms[i]))
        res = compare_outputs(attend(i, q, k, v).reshape(T, H * hd).float(), ctx[:, heads].float(),
                              atol=1.6e-2 if op == BF16 else 2e-3)
        log(f"[weights8] {cfg} {x.dtype} layer {i}: ctx max_abs={res.max_abs_error:.3e} failed={res.failed_elements}")
        assert res.passed
        rest = torch.ones(H * hp, dtype=torch.bool)
        rest[heads] = False
        assert (ctx[:, rest] == 0).all()
        r = r2
    live = torch.ones(T, dtype=torch.bool) if rm is None else rm != 0
    check_norm(y[live], r[live], mod.final_norm, D)
    assert (y[~live] == 0).all()


@pytest.mark.parametrize("cfg,dtype", [((2, 70, 128, 4, 128, 2, True), F16), ((3, 33, 100, 5, 60, 2, True), F16),
                                       ((3, 33, 100, 5, 60, 2, True), BF16), ((2, 40, 84, 6, 130, 1, False), F32),
                                       ((1, 9, 50, 5, 30, 2, True), BF16), ((2, 30, 300, 2, 260, 1, True), F16)])
@pytest.mark.parametrize("masked", [False, True])
def test_forward(products, cfg, dtype, masked):
    B, S, D, H = cfg[:4]
    _, norms, mod = build(cfg, dtype, 10000.0, True, weights8=True)
    mod.graph = False
    g = torch.Generator().manual_seed(5)
    x = torch.randn(B, S, D, generator=g).to(dtype)
    keep = None
    if masked:
        keep = torch.rand(B, S, generator=g) < 0.8
        keep[:, 0] = True
    with torch.inference_mode():
        y = mod(x.to(DEV), None if keep is None else keep.to(DEV)).cpu()

    def attend(i, q, k, v):
        out = torch.zeros(B * S, H, D // H, dtype=torch.float64)
        for b in range(B):
            at = slice(b * S, b * S + S)
            s = torch.matmul(q[at].transpose(0, 1), k[at].permute(1, 2, 0)) * (D // H) ** -0.5
            bad = torch.zeros(S, S, dtype=torch.bool) if keep is None else ~keep[b][None, :].expand(S, S)
            if cfg[6]:
                bad = bad | torch.ones(S, S, dtype=torch.bool).triu(1)
            p = torch.nan_to_num(torch.softmax(s.masked_fill(bad, -torch.inf), -1))
            out[at] = torch.matmul(p, v[at].transpose(0, 1)).transpose(0, 1)
        return out

    check_stack(mod, cfg, norms, products, x.view(B * S, D), y.view(B * S, D), 10000.0, torch.arange(S).repeat(B),
                attend, keep)


@pytest.mark.parametrize("cfg,dtype,code,block", [((4, 256, 100, 5, 60, 2, True), F16, E4M3, 16),
                                                  ((4, 256, 100, 5, 60, 2, True), BF16, I8, 32),
                                                  ((4, 256, 84, 6, 130, 1, True), F32, E4M3, 64)])
def test_extend_behind_a_prefix(products, cfg, dtype, code, block):
    D, H = cfg[2], cfg[3]
    _, norms, mod = build(cfg, dtype, 10000.0, True, weights8=True)
    cache = mod.make_cache(4, 60, block, code)
    hd, hp = D // H, cache.head_dim
    g = torch.Generator().manual_seed(4)
    for new, prefix in (([0, 75, 0, 0], None), ([50, 0, 3, 1], 1), ([1, 4, 1, 33], 1), ([1, 0, 1, 1], 1)):
        T = sum(new)
        x = torch.randn(T, D, generator=g).to(dtype)
        del products[:]
        with torch.inference_mode():
            y, missing = mod.extend(x.to(DEV), cache, torch.tensor(new, dtype=torch.int32, device=DEV), prefix=prefix)
        assert missing.tolist() == [0]
        lens, table = cache.lens.tolist(), cache.block_table.tolist()
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        pos = torch.cat([torch.arange(lens[b] - n, lens[b]) + (lens[1] if prefix is not None and b != 1 else 0)
                         for b, n in enumerate(new)])

        def attend(i, q, k, v):
            """Over the codes in the cache.  The new keys and values among them are off by a rounding to their code,
            another where their block's scale grew since, and by one to 16 bits."""
            wide = torch.zeros(T, H, hp, dtype=torch.float64)
            wide[..., :hd] = q
            pool = [codes_of(cache.k[i]), codes_of(cache.v[i]), cache.k_scale[i].cpu().double(),
                    cache.v_scale[i].cpu().double()]
            for b, n in enumerate(new):
                for t in range(n):
                    p = lens[b] - n + t
                    page, slot = table[b][p // block], p % block
                    for what, want, axis in ((0, k, 1), (1, v, 2)):
                        got = pool[what][page, :, slot] if axis == 1 else pool[what][page, :, :, slot]
                        scale = pool[what + 2][page][:, None]
                        half = torch.clamp(got.abs() * 2.0 ** -4, min=2.0 ** -9) if code == E4M3 else 0.5
                        err = (got * scale)[:, :hd] - want[cu[b] + t]
                        room = (2.1 * half * scale).expand_as(got)[:, :hd] + 2.0 ** -7 * want[cu[b] + t].abs()
                        assert (err.abs() <= room).all()
            rest = (cu, lens, table)
            if prefix is None:
                ctx = oc.attend(wide.view(T, H * hp), *rest, H, hp, hd ** -0.5, *pool, True)[0]
            else:
                ctx = serve.attend(wide.view(T, H * hp), *rest, prefix, H, hp, hd ** -0.5, *pool, True)[0]
            return ctx.view(T, H, hp)[..., :hd]

        check_stack(mod, cfg, norms, products, x, y.cpu(), 10000.0, pos, attend)
