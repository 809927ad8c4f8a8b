"""GPU tests of 8-bit products whose scales stand at either end of their range, or far apart, against 64 bits."""

import pytest
import torch

from oracle import serve

from _gpu_util import DEV, log
from test_gpu_linear8 import bound

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ROWS = [1, 6, 16, 17, 40, 300]


def check(y, aq, wq, m, out, what, low=0.0):
    """Within ``bound``; ``low``: what values under bf16's least ones may be off by in all."""
    want, mag = serve.linear(aq, wq)
    cut = serve.cut_of_eights(aq, wq) if m > 16 and out == BF16 else 0.0
    room = bound(want, mag, aq.shape[1], False, out, cut) + 1.01 * low
    err = (y.cpu().double() - want).abs()
    log(f"[linear8 range] {what} m {m} {out}: {float((err / room)[room > 0].max()):.3f} of the bound")
    assert (err <= room).all()


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_the_largest_activations(m, out):
    """A block's largest value up to bf16's own rounds to 2^128; weights that are small, and zeros."""
    from cobra_amd import ops

    g = torch.Generator().manual_seed(m)
    a = torch.randn(m, 256, generator=g)
    a[:, 5], a[:, 200] = torch.finfo(BF16).max, -3.3e38
    a = a.to(BF16)
    w = torch.randn(96, 256, generator=g) * 2.0 ** -60
    w[:, 5] = 2.0 ** -60 * torch.arange(96)
    w[3] = 0
    aq, ab = serve.quantize(a)
    assert int(ab[:, :2].min()) == 247 and float(serve.values(aq, ab).abs().max()) == 2.0 ** 128
    y = ops.linear8(a.to(DEV), *ops.quantize8(w.to(DEV)), out_dtype=out)
    assert torch.isfinite(y).all() and (y[:, 3] == 0).all()
    check(y, serve.values(aq, ab), serve.values(*serve.quantize(w)), m, out, "largest activations")


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("out", [F16, F32])
def test_the_largest_weights(m, out):
    from cobra_amd import ops

    g = torch.Generator().manual_seed(m)
    a = torch.randn(m, 256, generator=g).half()
    a[0] = 0
    w = torch.randn(96, 256, generator=g)
    w[:, 130] = 3.4e38
    code, byte = serve.quantize(a)
    byte[1:, 1] -= 116  # so that the second block's products with 2^128 are some 2^12
    assert int(byte.min()) >= 1 and (m == 1 or 2 <= int(byte[1:, 1].min()))
    wq = serve.values(*serve.quantize(w))
    assert float(wq.max()) == 2.0 ** 128
    y = ops.linear8(code.to(torch.float8_e4m3fn).to(DEV), *ops.quantize8(w.to(DEV)), out_dtype=out,
                    a_scale=byte.to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu))
    assert torch.isfinite(y).all() and (y[0] == 0).all()
    aq = serve.values(code, byte)
    check(y, aq, wq, m, out, "largest weights", 2.0 ** -133 * wq.abs().sum(1)[None, :])


def codes(rows, blocks, byte, top, g):
    """Random codes below `top` of either sign and the bytes given for each row and block, as (device pair, values)."""
    c = torch.randint(0, top, (rows, 128 * blocks), generator=g) + 128 * torch.randint(0, 2, (rows, 128 * blocks), generator=g)
    c = c.to(torch.uint8).view(torch.float8_e4m3fn)
    s = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8)
    s[:, :blocks] = byte.to(torch.uint8)
    return (c.to(DEV), s.to(DEV).view(torch.float8_e8m0fnu)), serve.values(c.double(), s.long())


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_scales_far_apart(m, out, seed):
    """Blocks of scales from 2^-123 to 2^120 beside each other, products of one size: values under 2."""
    from cobra_amd import ops

    g = torch.Generator().manual_seed(seed)
    blocks, n = 7, 70
    mid = torch.randint(7, 245, (1, blocks), generator=g)
    mid[0, seed % blocks], mid[0, (seed + 3) % blocks] = 244, 7
    a, aq = codes(m, blocks, mid + torch.randint(-3, 4, (m, blocks), generator=g), 64, g)
    w, wq = codes(n, blocks, 251 - mid + torch.randint(-3, 4, (n, blocks), generator=g), 64, g)
    check(ops.linear8(a[0], *w, a_scale=a[1], out_dtype=out), aq, wq, m, out, "far apart")


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_the_least_scales(m, out):
    """Bytes 1 to 3: values are rounded to multiples of 2^-132, by at most half of that each."""
    from cobra_amd import ops

    g = torch.Generator().manual_seed(m)
    a, aq = codes(m, 3, torch.randint(1, 4, (m, 3), generator=g), 127, g)
    w, wq = codes(50, 3, torch.randint(230, 248, (50, 3), generator=g), 127, g)
    low = 2.0 ** -133 * wq.abs().sum(1)[None, :]
    check(ops.linear8(a[0], *w, a_scale=a[1], out_dtype=out), aq, wq, m, out, "least", low)
