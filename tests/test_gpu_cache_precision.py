"""GPU tests of the cache attention's precision: with fp16 activations the weights are held in two
fp16 terms in both kernels, so that a result is off by little more than its own rounding, and a
call's hints move it by no more."""

import pytest
import torch

from oracle import cache as oc

from _cache_util import E4M3, I8, attn_tolerance, codes_of, poison
from _gpu_util import DEV, log
from test_gpu_cache import attn_case, i32

pytestmark = pytest.mark.gpu


def attend(c, heads, head_dim):
    """(result, sum p |v|, largest |score|, largest sum |q k|) of a case in 64 bits."""
    k, v, ks, vs = c["cache"]
    return oc.attend(c["q"].double(), c["cu"], c["lens"], c["table"], heads, head_dim, head_dim ** -0.5, codes_of(k),
                     codes_of(v), torch.nan_to_num(ks.double()), torch.nan_to_num(vs.double(), posinf=0.0), True)


def run(c, heads, head_dim, **kw):
    from cobra_amd import ops

    got = ops.cache_attn(c["q"].to(DEV), i32(c["cu"]), i32(c["lens"]), i32(c["table"]), heads, head_dim,
                         head_dim ** -0.5, *[t.to(DEV) for t in c["cache"]], **kw)
    return got.cpu().double()


def rms(x):
    return float(x.square().mean().sqrt())


# Requests of one new token: at most 16 rows to a kv head; of 40 to 130: the chunk kernel.
FEW = ([900, 333, 61, 1500, 17, 700, 1200, 2000], [1] * 8)
MANY = ([300, 61, 800, 5], [80, 130, 40, 120])


@pytest.mark.parametrize("held,new", [FEW, MANY])
@pytest.mark.parametrize("heads,kv,head_dim", [(8, 8, 32), (8, 2, 64), (4, 4, 96), (8, 4, 128), (2, 2, 192), (4, 1, 256)])
@pytest.mark.parametrize("cache", [E4M3, I8])
def test_fp16_results_are_off_by_their_own_rounding(heads, kv, head_dim, cache, held, new):
    """The root mean square of the error against 64 bits, by that of rounding the 64-bit result to
    fp16 (both over a row's sum p |v|, so that every row counts).

    Before its rounding a result is off by e: 2^-21 of each weight, and scores whose head_dim
    roundings of 2^-24 add up as a random walk does: 16 x 2^-24 of a score's terms, some 4, at head_dim
    256.  That is 5e-6 of the weights, a fiftieth of fp16's 2^-12; even four times that, in quadrature,
    is within a hundredth.  With the weights in one term e is as large as the rounding."""
    parts = []
    for seed in range(3):
        c = attn_case(heads, kv, head_dim, 32, held, new, torch.float16, cache, seed=100 + seed, sharp=3.0)
        want, mag, _, _ = attend(c, heads, head_dim)
        got = run(c, heads, head_dim, max_new=max(new))
        fine = (want.abs() < 60000) & (want.abs() > 2.0 ** -13)  # fp16's normal numbers
        parts.append(torch.stack([((got - want) / mag)[fine], ((want.half().double() - want) / mag)[fine]]))
    err, own = torch.cat(parts, 1)
    log(f"[precision] {cache} H{heads} kv{kv} hd{head_dim} rows {sum(new)}: {rms(err) / rms(own):.4f} of its own rounding")
    assert rms(err) <= 1.01 * rms(own)


@pytest.mark.parametrize("cache", [E4M3, I8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_far_apart_head_by_head(cache, dtype):
    """Neighbouring blocks whose scales differ by up to 2^60, each head held to the bound of its
    own blocks' scales."""
    for new in ([1], [80]):
        c = attn_case(2, 2, 64, 16, [333], new, dtype, cache, seed=10)
        k, v, ks, vs = c["cache"]
        n = ks.shape[0]
        vs.copy_(torch.ldexp(torch.ones(n, 2), (torch.arange(n) % 5 - 2)[:, None] * torch.tensor([[8, 15]])))
        ks.copy_(torch.ldexp(torch.ones(n, 2), -(torch.arange(n) % 3)[:, None] * 10 - 5 + torch.tensor([[0, 1]])))
        pages = c["table"][0][:oc.blocks(c["lens"][0], 16)]
        poison(k, v, pages[-1], c["lens"][0] % 16)
        want, mag, top, reach = attend(c, 2, 64)
        largest = vs[pages].amax(0).double().repeat_interleave(64)  # of each column's head
        tol = attn_tolerance(want, mag, top, reach, c["lens"][0], 64, dtype, largest)
        got = run(c, 2, 64, max_new=max(new))
        border = torch.finfo(dtype).max
        sure = want.abs() + tol < border
        assert sure.all() or dtype == torch.float16  # values of 60 x 2^16 and more are past fp16's range
        assert ((got - want).abs() <= tol)[sure].all()
        over = want.abs() - tol > border * 1.001
        assert torch.equal(got[over], torch.copysign(torch.full_like(want, float("inf")), want)[over])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("held,new", [([700, 0, 90], [1, 1, 1]), ([700, 64, 90], [40, 3, 9]), ([300, 0, 90], [150, 70, 3])])
def test_hints_move_a_result_within_its_rounding(held, new, dtype):
    """Hints choose the kernel and the splits, which changes the order of sums and no more.

    Two results that are off by e before they are rounded differ by a step where a border lies
    between them, with a probability of 2 e by the step, else not at all.  fp16: e is a three
    hundredth of a step (two terms), 0.007 of the results a step apart, root mean square 0.08 of a step,
    against 0.29 for the rounding itself; twice that is taken.  bf16: a weight's 2^-12 and a result's
    2^-9 (root mean squares of half a step each) leave e at an eighth of the rounding."""
    c = attn_case(8, 2, 64, 32, held, new, dtype, E4M3, seed=3)
    want, mag, top, reach = attend(c, 8, 64)
    hints = [(max(new), max(c["lens"])), (None, None), (1, 1), (1, 64), (3, 700), (100000, 5), (1, 10 ** 12), (200, 1)]
    got = [run(c, 8, 64, max_new=n, max_len=m) for n, m in hints]
    own = rms((want.to(dtype).double() - want) / mag.clamp(min=1e-30))
    step = torch.finfo(dtype).eps * want.abs()
    weight = 2.0 ** -21 if dtype == torch.float16 else 2.0 ** -11
    room = step + 2 * (weight + 2.0 ** -18) * mag + 2.0 ** -24
    for hint, g in zip(hints[1:], got[1:]):
        apart = rms((g - got[0]) / mag.clamp(min=1e-30)) / own
        log(f"[hints] {dtype} new {new} {hint}: {apart:.4f} of the rounding")
        assert ((g - got[0]).abs() <= room).all(), hint
        assert apart <= (0.6 if dtype == torch.float16 else 1.0), hint
