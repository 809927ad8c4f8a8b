"""GPU tests of the norms and rotation of queries and keys, and of the positions of cached requests,
against the plain form in 64 bits (oracle/serve.py)."""

import pytest
import torch

from oracle import serve

from _gpu_util import DEV, log

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def check(t, heads, kv, hd, dtype, rot, inter, norm, pitch=None, far=4000, pad=0, seed=0, offset=0):
    from cobra_amd import ops

    g = torch.Generator().manual_seed(seed + t)
    pitch = pitch or hd
    cols = (heads + 2 * kv) * pitch + pad
    x = (torch.randn(t, cols, generator=g) * torch.exp(torch.randn(t, 1, generator=g))).to(dtype)
    pos = torch.randint(0, far + 1, (t,), generator=g, dtype=torch.int32)
    if t > 2:
        pos[1] = -1
    freq = (10000.0 ** -(torch.arange(rot // 2).double() * 2 / max(rot, 1))).float() if rot else None
    qw = 1 + 0.3 * torch.randn(hd, generator=g) if norm else None
    kw = 1 + 0.3 * torch.randn(hd, generator=g) if norm else None
    dev = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    flat = torch.zeros(t * cols + offset, dtype=dtype, device=DEV)
    y = flat[offset:].view(t, cols)
    y.copy_(x.to(DEV))
    ops.qk_norm_rope(y, heads, kv, hd, positions=dev(pos) if rot or t % 2 else None, inv_freq=dev(freq),
                     q_weight=dev(qw), k_weight=dev(kw), interleaved=inter, eps=1e-5, pitch=pitch if pitch != hd else None)
    torch.cuda.synchronize()
    got = y.cpu().double()
    live = pos >= 0 if rot or t % 2 else torch.ones(t, dtype=torch.bool)
    want = x.double()
    room = torch.zeros_like(want)
    for h in range(heads + kv):
        at = slice(h * pitch, h * pitch + hd)
        z = serve.norm_rope(x[:, at], hd, pos, freq, (qw if h < heads else kw) if norm else None, inter, 1e-5)
        want[:, at] = torch.where(live[:, None], z, want[:, at])
        # The squares' sum: hd + 2 roundings of 2^-24, half of that in its root; root, quotient and two
        # products 2^-22 in all.  Sine and cosine are off by at most 2^-22 and by the angle's own rounding
        # in turns, 2^-26 of one: 2 pi 2^-26 < 2^-23.  A pair's two products and their sum: 2^-22.
        plain = serve.norm_rope(x[:, at], hd, pos, None, (qw if h < heads else kw) if norm else None, inter, 1e-5)
        size = plain.abs()
        if rot:
            r = rot // 2
            i = torch.arange(r)
            a, b = (2 * i, 2 * i + 1) if inter else (i, i + r)
            s = size[:, a] + size[:, b]
            size[:, a], size[:, b] = s, s
        room[:, at] = size * ((hd + 2) * 2.0 ** -25 + 2.0 ** -20)
    room = room + torch.finfo(dtype).eps / 2 * (want.abs() + room) + (2.0 ** -25 if dtype == F16 else 0.0)
    err = (got - want).abs()
    assert (err <= room).all(), float((err / room).max())
    log(f"[rope] {t} x {heads}/{kv} x {hd} {dtype} rot {rot} inter {inter} norm {norm}: {float((err / room).max()):.3f}")
    rest = (heads + kv) * pitch
    assert torch.equal(got[:, rest:], x.double()[:, rest:])  # values and what stands behind them
    if pitch > hd:
        for h in range(heads + kv):
            assert torch.equal(got[:, h * pitch + hd:(h + 1) * pitch], x.double()[:, h * pitch + hd:(h + 1) * pitch])
    if not live.all():
        assert torch.equal(got[~live], x.double()[~live])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rot", [
    (8, 8, 64, 64), (32, 8, 128, 128), (6, 2, 256, 256), (4, 4, 32, 32), (6, 6, 40, 40), (12, 4, 80, 80), (8, 4, 96, 96),
    (5, 5, 168, 168), (4, 2, 128, 64), (3, 1, 64, 16), (3, 1, 64, 24), (2, 1, 24, 20), (7, 1, 16, 16), (4, 4, 8, 8),
    (2, 2, 128, 8), (3, 3, 8, 2)])
def test_norm_and_rotation(heads, kv, hd, rot, norm, inter, dtype):
    for t in (1, 7):
        check(t, heads, kv, hd, dtype, rot, inter, norm)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,rot,pitch,pad,offset", [
    (5, 4, 8, 0, 0), (33, 10, 40, 3, 0), (255, 254, 256, 0, 0), (20, 20, 24, 0, 0), (100, 100, 104, 8, 0), (30, 30, 32, 0, 0),
    (64, 64, 64, 1, 0), (64, 64, 64, 0, 1), (64, 64, 64, 0, 4), (128, 128, 128, 4, 0), (1, 0, 8, 0, 0), (66, 66, 66, 0, 0)])
def test_odd_geometries(hd, rot, pitch, pad, offset, inter):
    for norm in (False, True):
        if rot or norm:
            check(5, 3, 2, hd, F16 if norm else BF16, rot, inter, norm, pitch=pitch, pad=pad, offset=offset)


def test_norm_alone():
    for t in (1, 4, 5):
        check(t, 4, 2, 64, F16, 0, False, True)
        check(t, 4, 2, 40, BF16, 0, True, True)


@pytest.mark.parametrize("far", [0, 1, 100000, 2 ** 31 - 1])
def test_far_positions(far):
    check(9, 4, 4, 64, F16, 64, False, False, far=far)
    check(9, 2, 2, 40, F16, 20, True, True, far=far)


@pytest.mark.parametrize("t,rot,inter,norm", [(3000, 64, False, True), (5001, 64, True, False), (20003, 64, False, True),
                                              (20003, 16, True, True), (20003, 0, False, True)])
def test_many_tokens(t, rot, inter, norm):
    """Several tokens a workgroup, and a last one with fewer."""
    check(t, 2, 1, 64, BF16, rot, inter, norm)


def test_zero_rows_and_large_values():
    """A head of zeros stays zero (eps); values whose squares pass fp16's range are normed in fp32."""
    from cobra_amd import ops

    x = torch.zeros(2, 3 * 64, dtype=F16, device=DEV)
    x[1] = 60000.0
    w = torch.ones(64, device=DEV)
    ops.qk_norm_rope(x, 1, 1, 64, q_weight=w, k_weight=w)
    assert (x[0] == 0).all() and (x[1, :128] == 1).all() and (x[1, 128:] == 60000).all()


def positions(cu, lens, tokens, prefix):
    out = [-1] * tokens
    for b, n in enumerate(lens):
        new = cu[b + 1] - cu[b]
        for i in range(new):
            out[cu[b] + i] = n - new + i + (lens[prefix] if prefix is not None and b != prefix else 0)
    return out


@pytest.mark.parametrize("batch", [1, 2, 64, 300, 5000])
def test_positions(batch):
    from cobra_amd import ops

    g = torch.Generator().manual_seed(batch)
    new = torch.randint(0, 4, (batch,), generator=g)
    new[0] = 0 if batch > 1 else 3
    lens = (new + torch.randint(0, 100, (batch,), generator=g)).tolist()
    cu = [0] + torch.cumsum(new, 0).tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for prefix in (None, 0, batch - 1):
        got = ops.cache_positions(i32(cu), i32(lens), cu[-1] + 3, prefix)
        assert got.tolist() == positions(cu, lens, cu[-1] + 3, prefix)
    assert ops.cache_positions(i32(cu), i32(lens), 0).numel() == 0
    assert ops.cache_positions(i32([0]), i32([]), 3).tolist() == [-1] * 3


def test_rope_in_a_graph():
    from cobra_amd import ops

    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 6 * 64, generator=g).half().to(DEV)
    src = x.clone()
    pos = torch.arange(20, dtype=torch.int32, device=DEV)
    freq = (10000.0 ** -(torch.arange(32).double() / 32)).float().to(DEV)
    w = torch.ones(64, device=DEV)
    ops.qk_norm_rope(x, 4, 1, 64, pos, freq, w, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.qk_norm_rope(x, 4, 1, 64, pos, freq, w, w)
    for shift in (0, 7, 50):
        pos.copy_(torch.arange(20, dtype=torch.int32) + shift)
        x.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want = src.clone()
        ops.qk_norm_rope(want, 4, 1, 64, pos, freq, w, w)
        assert torch.equal(x, want)


@pytest.mark.parametrize("hd", [128, 126])
def test_rows_past_32_bits(hd):
    """More than 2^32 bytes of rows: those that repeat, at positions that repeat, turn alike."""
    from cobra_amd import ops

    g = torch.Generator().manual_seed(3)
    base = torch.randn(250, 60 * hd, generator=g).to(BF16).to(DEV)
    freq = (10000.0 ** -(torch.arange(hd // 2).double() * 2 / hd)).float().to(DEV)
    w = torch.ones(hd, device=DEV)
    x = base.repeat(1200, 1)
    ops.qk_norm_rope(x, 40, 10, hd, seq_len=250, inv_freq=freq, q_weight=w, k_weight=w)
    want = base.clone()
    ops.qk_norm_rope(want, 40, 10, hd, seq_len=250, inv_freq=freq, q_weight=w, k_weight=w)
    x = x.view(1200, 250, -1)
    for i in range(1200):
        assert torch.equal(x[i], want)
    assert not torch.equal(want, base)
