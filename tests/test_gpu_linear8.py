"""GPU tests of matrices in 8-bit blocks and their product against the plain form in 64 bits
(oracle/serve.py): codes and scales to the bit, products within a bound from their roundings."""

import math

import pytest
import torch

from oracle import serve

from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rows(m, k, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g))
    x *= torch.where(torch.rand(1, k, generator=g) < 0.02, 30.0, 1.0)
    return x.to(dtype)


def check_codes(x):
    from cobra_amd import ops

    codes, scale = ops.quantize8(x.to(DEV))
    want, byte = serve.quantize(x)
    assert codes.dtype == torch.float8_e4m3fn and scale.dtype == torch.float8_e8m0fnu
    assert codes.shape == want.shape and scale.shape == byte.shape
    assert torch.equal(scale.view(torch.uint8).cpu().long(), byte)
    got = codes.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))
    return codes, scale


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 8), (5, 127), (2, 128), (7, 136), (4, 511), (3, 512), (9, 520), (64, 1024),
                                 (33, 1096), (1, 5000), (700, 4100), (2100, 2048)])
def test_quantize_is_the_plain_form(m, k, dtype):
    log(f"[quantize8] {m} x {k} {dtype}")
    check_codes(rows(m, k, dtype, m * 10 + k))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 3), (9, 7), (7, 9), (13, 100), (6, 121), (1, 129), (5, 200), (3, 255), (8, 256), (5, 257),
                                 (9, 509), (5, 1023), (3, 4091), (33333, 5), (40001, 100), (30001, 129), (20001, 250),
                                 (9001, 301), (2001, 2049)])
def test_quantize_narrow_and_odd_rows(m, k, dtype):
    check_codes(rows(m, k, dtype, m + k))


@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("k", [7, 9, 100, 127, 129, 250, 1023, 2050])
@pytest.mark.parametrize("n", [17, 9000])
def test_linear8_few_rows_of_odd_lengths(m, k, n):
    check_linear(m, k, n, F16 if k % 2 else BF16, m + k, gelu=k == 100, out=F32 if m == 5 else None)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize_every_16_bit_pattern(dtype):
    """Every fp16 and bf16 value, subnormals, infinities and NaN among them, each beside a block's
    largest value that puts the border of a scale, and ties, on either side."""
    src = F16 if dtype == F32 else dtype
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(src).view(512, 128)
    check_codes(x.to(dtype))
    fin = torch.where(torch.isfinite(x.float()), x, torch.zeros_like(x)).float()
    for top in (448.0, 449.0, 447.5, 1.75, 1.7578125, 0.875, 57344.0):
        y = fin.clamp(-top, top)
        y[:, 5] = top
        check_codes(y.to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize_extremes(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(8, 300)
    x[1] = info.max
    x[2] = info.tiny
    x[3, ::2] = math.inf
    x[3, 1] = 3.0
    x[4] = math.nan
    x[5, 130] = -math.inf
    x[6] = torch.linspace(-1, 1, 300) * info.tiny * 4
    x[7, 299] = -0.0
    check_codes(x.to(dtype))


def bound(y, mag, kp, use_gelu, dtype, cut=0.0):
    """Products of codes and scales are exact; at most kp + 8 additions in fp32, each off by at most
    2^-23 (the matrix cores may cut) of sum |a w| + |bias|, and what the scaled instructions cut
    (``serve.cut_of_eights``); GELU's slope is at most 1.13 and its own error 4e-7 of at most the
    argument; one addition of the residual; one rounding of the result."""
    err = (kp + 8) * 2.0 ** -23 * mag + cut
    if use_gelu:
        err = 1.13 * err + 4e-7 * mag + 4e-7
    err = err + 2.0 ** -23 * y.abs()
    least = 2.0 ** -25 if dtype == F16 else 0.0  # half of fp16's smallest step
    return err + torch.finfo(dtype).eps / 2 * (y.abs() + err) + least


def check_linear(m, k, n, dtype, seed, codes=False, bias=True, gelu=False, out=None, resid=None, mask=None,
                 mask_branch=False, spread=0.7):
    from cobra_amd import ops

    g = torch.Generator().manual_seed(seed)
    a = rows(m, k, dtype, seed, spread)
    w = torch.randn(n, k, generator=g) * k ** -0.5
    wq, wb = serve.quantize(w)
    aq, ab = serve.quantize(a)
    dw = ops.quantize8(w.to(DEV))
    b = 0.2 * torch.randn(n, generator=g) if bias else None
    r = None if resid is None else torch.randn(m, n, generator=g).to(resid)
    rm = None if mask is None else torch.rand(m, generator=g) < mask
    out_type = out or dtype
    want, mag = serve.linear(serve.values(aq, ab), serve.values(wq, wb), b, gelu, r, rm, mask_branch)
    kw = dict(bias=None if b is None else b.to(DEV), gelu=gelu, resid=None if r is None else r.to(DEV),
              rmask=None if rm is None else rm.to(DEV), mask_branch=mask_branch)
    if codes:
        ca, sa = ops.quantize8(a.to(DEV))
        y = ops.linear8(ca, *dw, a_scale=sa, out_dtype=out_type, **kw)
    else:
        y = ops.linear8(a.to(DEV), *dw, out_dtype=out, **kw)
    torch.cuda.synchronize()
    assert y.dtype == out_type and y.shape == (m, n)
    # Up to 16 rows and for fp32 results the products are added in fp32 one by one.
    cut = serve.cut_of_eights(serve.values(aq, ab), serve.values(wq, wb)) if m > 16 and out_type != F32 else 0.0
    room = bound(want, mag, aq.shape[1], gelu, out_type, cut)
    if rm is not None and resid is not None and not mask_branch:
        want = torch.where(rm[:, None], want, torch.zeros_like(want))
    used = float(((y.cpu().double() - want).abs() / room).max())
    log(f"[linear8] {m} x {k} x {n} {dtype} codes={codes} out={out_type}: {used:.3f} of the bound")
    assert used <= 1.0
    return y


@pytest.mark.parametrize("m", [1, 2, 4, 5, 15, 16, 17, 31, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear8_rows(m, dtype):
    check_linear(m, 256, 192, dtype, m)


@pytest.mark.parametrize("m", [1, 20, 64, 90])
@pytest.mark.parametrize("k,n", [(1, 1), (8, 3), (100, 17), (128, 16), (136, 63), (200, 1000), (384, 129), (640, 65),
                                 (1096, 250), (2050, 96), (4096, 40)])
def test_linear8_odd_sizes(m, k, n):
    check_linear(m, k, n, F16 if (m + k) % 2 else BF16, m + k + n, codes=k % 3 == 0, gelu=n % 2 == 0)


@pytest.mark.parametrize("m,k,n", [(16, 1024, 9000), (40, 512, 16400), (64, 2200, 1000), (50, 640, 4090), (700, 512, 1100), (2000, 256, 4100),
                                   (4100, 384, 2056), (9000, 128, 520)])
@pytest.mark.parametrize("out", [F16, BF16, F32])
def test_linear8_tiles(m, k, n, out):
    check_linear(m, k, n, BF16, m, out=out, resid=F32 if out == F32 else None)


@pytest.mark.parametrize("m,n", [(7, 50), (7, 64), (90, 50), (90, 64), (300, 264)])
@pytest.mark.parametrize("resid", [None, F16, BF16, F32])
@pytest.mark.parametrize("mask_branch", [False, True])
def test_linear8_epilogue(m, n, resid, mask_branch):
    for out in (F16, F32):
        check_linear(m, 192, n, F16, m + n, resid=resid, mask=0.6, mask_branch=mask_branch, gelu=True, out=out)
    check_linear(m, 192, n, BF16, m + n, resid=resid, bias=False, mask=0.0, mask_branch=mask_branch)


def test_linear8_codes_are_the_calls_own_quantisation():
    """The call on 16-bit activations and on their codes gives the same bits, few rows and many."""
    from cobra_amd import ops

    for m in (3, 40, 200):
        for dtype in (F16, BF16):
            a = rows(m, 904, dtype, m).to(DEV)
            w = ops.quantize8(rows(300, 904, F32, 5, 0.1).to(DEV))
            ca, sa = ops.quantize8(a)
            one = ops.linear8(a, *w)
            two = ops.linear8(ca, *w, a_scale=sa, out_dtype=dtype)
            assert torch.equal(one, two)


def test_linear8_shows_what_is_not_finite():
    """A row of activations with an infinity or a NaN gives NaN, the others stay as they are."""
    from cobra_amd import ops

    for m in (6, 150):
        a = rows(m, 256, BF16, 1).to(DEV)
        w = ops.quantize8(rows(96, 256, F32, 2, 0.1).to(DEV))
        clean = ops.linear8(a, *w)
        a[1, 200], a[4, 3] = math.inf, math.nan
        got = ops.linear8(a, *w)
        keep = [i for i in range(m) if i not in (1, 4)]
        assert torch.isnan(got[[1, 4]]).all() and torch.equal(got[keep], clean[keep])


def test_linear8_far_scales():
    """Blocks whose scales lie 2^100 apart: the sums are fp32's, nothing of the larger block is lost."""
    from cobra_amd import ops

    for m in (5, 100):
        a = torch.ones(m, 256)
        a[:, :128] *= 2.0 ** 60
        a[:, 128:] *= 2.0 ** -40
        w = torch.ones(48, 256)
        w[:, :128] *= 2.0 ** -50
        w[:, 128:] *= 2.0 ** 50
        y = ops.linear8(a.to(BF16).to(DEV), *ops.quantize8(w.to(DEV)), out_dtype=F32)
        assert torch.equal(y.cpu(), torch.full((m, 48), 128.0 * 2 ** 10 + 128.0 * 2 ** 10))


def test_linear8_empty():
    from cobra_amd import ops

    w = ops.quantize8(rows(96, 256, F32, 2).to(DEV))
    assert ops.linear8(torch.empty(0, 256, dtype=F16, device=DEV), *w).shape == (0, 96)
    none = ops.quantize8(torch.empty(0, 256, dtype=F16, device=DEV))
    assert none[0].shape == (0, 256) and none[1].shape == (0, 4)
    assert ops.linear8(torch.empty(5, 256, dtype=F16, device=DEV), *none).shape == (5, 0)


def test_linear8_in_a_graph_and_on_another_stream():
    from cobra_amd import ops

    a = [rows(m, 520, F16, m).to(DEV) for m in (6, 200)]
    w = ops.quantize8(rows(300, 520, F32, 2, 0.1).to(DEV))
    want = [ops.linear8(x, *w) for x in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.linear8(x, *w) for x in a]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [ops.linear8(x, *w) for x in a]
    for seed in (3, 4, 5):
        for x in a:
            x.copy_(rows(*x.shape, F16, seed).to(DEV))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a, out):
            assert torch.equal(y, ops.linear8(x, *w))


def test_sizes_past_32_bits():
    """Results, weights and inputs of more than 2^32 bytes: rows that repeat give results that repeat."""
    from cobra_amd import ops

    base = rows(250, 128, BF16, 1).to(DEV)
    w = rows(33000, 128, F32, 2, 0.1)
    y = ops.linear8(base.repeat(264, 1), *ops.quantize8(w.to(DEV))).view(264, 250, 33000)
    for i in range(1, 264):
        assert torch.equal(y[i], y[0])
    at = [0, 1, 63, 16500, 32998, 32999]
    aq, wq = serve.values(*serve.quantize(base.cpu())), serve.values(*serve.quantize(w[at]))
    want, mag = serve.linear(aq, wq, None, False, None, None, False)
    room = bound(want, mag, 128, False, BF16, serve.cut_of_eights(aq, wq))
    assert ((y[0][:, at].cpu().double() - want).abs() <= room).all()
    del y

    base = rows(500, 8192, BF16, 3, 0.1).to(DEV)
    codes, scale = ops.quantize8(base.repeat(1060, 1))
    want = ops.quantize8(base)
    for i in range(1060):
        at = slice(500 * i, 500 * i + 500)
        assert torch.equal(codes[at].view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(scale[at].view(torch.uint8), want[1].view(torch.uint8))
    for m in (3, 40):
        a = rows(m, 8192, F16, m).to(DEV)
        y = ops.linear8(a, codes, scale).view(m, 1060, 500)
        assert torch.equal(y, y[:, :1].expand_as(y))
        aq, wq = serve.values(*serve.quantize(a.cpu())), serve.values(*serve.quantize(base.cpu()[:40]))
        ref, mag = serve.linear(aq, wq, None, False, None, None, False)
        room = bound(ref, mag, 8192, False, F16, serve.cut_of_eights(aq, wq) if m > 16 else 0.0)
        got = y[:, 0, :40].cpu().double()
        over = got.isinf()  # fp16 rounds what is not below 65520 to infinity
        assert (ref.abs() + room >= 65520)[over].all() and (got.sign() == ref.sign())[over].all()
        assert ((got - ref).abs() <= room)[~over].all()
