"""GPU tests of captured ``CobraTransformer.extend``: which captures are refused, and what a graph
reads after the model has gone on."""

import gc

import pytest
import torch

from _gpu_util import DEV

pytestmark = pytest.mark.gpu

CFG = (3, 256, 128, 4, 128, 2, True)


def model(seed=1):
    from cobra_amd import CobraTransformer, TransformerConfig

    torch.manual_seed(seed)
    return CobraTransformer(TransformerConfig(*CFG)).to(DEV, torch.float16).eval()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rows(n, seed, dtype=torch.float16):
    return torch.randn(n, CFG[2], generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


@pytest.mark.parametrize("first", [None, torch.bfloat16])
def test_extend_is_not_captured_before_its_weights_are_laid_out(first):
    """They would be in the graph's memory, and hold nothing until it is replayed."""
    mod, twin = model(), model()
    cache, new = mod.make_cache(2, 8, 16), i32([2, 1])
    with torch.inference_mode():
        if first is not None:
            mod.extend(rows(3, 1, first), cache, new)
        held, x = cache.lens.tolist(), rows(3, 2)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="before it is captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                mod.extend(x, cache, new)
        assert cache.lens.tolist() == held
        c1, c2 = mod.make_cache(2, 8, 16), twin.make_cache(2, 8, 16)
        y, want = mod.extend(rows(3, 3), c1, new)[0], twin.extend(rows(3, 3), c2, new)[0]
        assert torch.equal(y, want)


def test_captured_extend_keeps_its_weights():
    """The model lays its weights out for another type, and again for the first, and the memory of
    what it drops is given back: the graph still has its own."""
    mod, twin = model(), model()
    cache, other, plain = mod.make_cache(2, 8, 16), mod.make_cache(2, 8, 16), twin.make_cache(2, 8, 16)
    new, x = i32([2, 1]), torch.zeros(3, CFG[2], device=DEV, dtype=torch.float16)
    with torch.inference_mode():
        for m, c in ((mod, cache), (twin, plain)):
            m.extend(rows(9, 4), c, i32([5, 4]))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, missing = mod.extend(x, cache, new)
        for step in range(4):
            if step == 1:
                mod.extend(rows(3, 5, torch.bfloat16), other, new)
            if step == 2:
                mod.extend(rows(3, 6), other, new)
            gc.collect()
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            junk = [torch.full((n,), float("nan"), device=DEV) for n in (1 << 8, 1 << 14, 1 << 15, 1 << 20)]
            x.copy_(rows(3, 10 + step))
            graph.replay()
            want, none = twin.extend(rows(3, 10 + step), plain, new)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(missing, none) and missing.item() == 0, step
            del junk
    assert torch.equal(cache.lens, plain.lens)
