"""GPU tests of the cache operators' host calls: what they refuse, and that each is made once."""

import pytest
import torch

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
