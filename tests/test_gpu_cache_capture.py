"""GPU tests of captured ``CobraTransformer.extend``: which captures are refused."""

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
