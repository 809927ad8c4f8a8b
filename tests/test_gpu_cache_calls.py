"""GPU tests of the cache operators' host calls: what they refuse, and that each is made once."""

import ctypes

import pytest
import torch

from _cache_util import random_cache
from _gpu_util import DEV

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def tables():
    """Two requests, three free blocks of 16 tokens: room for 2 and 1 more tokens takes none of them."""
    return dict(lens=i32([3, 5]), new=i32([2, 1]), table=i32([[0, 9, 9], [1, 9, 9]]), free=i32([2, 3, 4]), count=i32([3]))


def reserve(t, tokens=3):
    from cobra_amd import ops

    return ops.cache_reserve(t["lens"], t["new"], t["table"], t["free"], t["count"], 16, tokens)


@pytest.mark.parametrize("tokens", [2 ** 31, 2 ** 45, 2 ** 62, -1])
def test_reserve_refuses_more_tokens_than_it_counts(tokens):
    """Before it allocates their slots."""
    t = tables()
    with pytest.raises(ValueError, match="tokens must be"):
        reserve(t, tokens)
    assert t["lens"].tolist() == [3, 5] and t["count"].tolist() == [3]


# -- each call is made once -------------------------------------------------------------


def hip():
    """The HIP runtime that torch has loaded."""
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))


def layer():
    """One layer's cache of five blocks, and a call's keys, values and queries for two requests."""
    k, v, ks, vs = (t.to(DEV) for t in random_cache(5, 2, 16, 64, torch.int8, seed=1))
    x = torch.randn(3, 8 * 64, generator=torch.Generator().manual_seed(2)).to(DEV, torch.float16)
    return dict(x=x, slots=torch.tensor([3, 4, 21], device=DEV), cu=i32([0, 2, 3]), k=k, v=v, ks=ks, vs=vs)


def calls(t, c):
    """The four operators as calls without arguments, and the tensors that they change."""
    from cobra_amd import ops

    pool = (c["k"], c["v"], c["ks"], c["vs"])
    return {
        "reserve": (lambda: reserve(t), (t["lens"], t["table"], t["count"])),
        "trim": (lambda: ops.cache_trim(t["lens"], t["keep"], t["table"], t["free"], t["count"], 16),
                 (t["lens"], t["free"], t["count"])),
        "append": (lambda: ops.cache_append(c["x"], c["slots"], 4, 64, *pool), pool),
        "attn": (lambda: ops.cache_attn(c["x"], c["cu"], t["lens"], t["table"], 4, 64, 0.125, *pool), ()),
    }


@pytest.mark.parametrize("name", ["reserve", "trim", "append", "attn"])
def test_an_older_error_is_none_of_the_calls(name):
    """An error that an earlier call of the thread left behind: each operator runs once, as without it,
    and leaves it where it was."""
    got = []
    for pending in (False, True):
        t, c = dict(tables(), keep=i32([1, 5])), layer()
        call, changed = calls(t, c)[name]
        torch.cuda.synchronize()
        rt = hip()
        try:
            left = rt.hipSetDevice(4096) if pending else 0
            out = call()
        finally:
            kept = rt.hipGetLastError()
        assert kept == left
        out = out if isinstance(out, tuple) else () if out is None else (out,)
        got.append([x.clone() for x in (*out, *changed)])
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("name", ["reserve", "trim", "append", "attn"])
def test_a_launch_that_fails_raises_and_is_not_made_again(name, monkeypatch):
    """On a stream whose capture has become invalid every launch is refused by the runtime: the
    native call raises the library's error, and the general path does not make it a second time."""
    from cobra_amd import CobraError, ops

    t, c = dict(tables(), keep=i32([1, 5])), layer()
    call, changed = calls(t, c)[name]
    rt = hip()
    raw, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamCreate(ctypes.byref(raw)) == 0
    again = []
    try:
        stream = torch.cuda.ExternalStream(raw.value)
        with torch.cuda.stream(stream):
            call()  # its memory is there
            torch.cuda.synchronize()
            before = [x.clone() for x in changed]
            torch.cuda.synchronize()
            monkeypatch.setattr(ops, "call", lambda fn, *a: again.append(fn))
            assert rt.hipStreamBeginCapture(raw, 2) == 0  # relaxed
            assert rt.hipStreamSynchronize(raw) != 0      # not allowed in a capture, which it ends
            with pytest.raises(CobraError, match=f"cobra_cache_{name}"):
                call()
    finally:
        rt.hipStreamEndCapture(raw, ctypes.byref(graph))
        rt.hipGetLastError()
        rt.hipStreamDestroy(raw)
        rt.hipGetLastError()
    torch.cuda.synchronize()
    assert again == []
    assert all(torch.equal(x, y) for x, y in zip(changed, before))
