"""CPU tests of how the cache attention's calls are cut, as far as the workspace shows it, and of the
longest request that a cache is made for."""

import random

import pytest


def _workspace():
    from cobra_amd import _lib

    return _lib.lib().cobra_cache_attn_workspace_bytes


def test_workspace_is_bounded_whatever_the_hints():
    """Hints shape the launch: one far too low for the call's tokens must not ask for more memory
    than a call is worth (partial results of 2^19 rows of a head, whatever their width)."""
    q = _workspace()
    rng = random.Random(1)
    cases = [(100000, 1, 32, 8, 128, 1, 100000), (20000, 1, 8, 8, 256, 1, 100000), (2048, 1, 32, 8, 128, 1, 32000)]
    for _ in range(3000):
        kv = rng.choice([1, 2, 8, 32])
        cases.append((int(2 ** rng.uniform(0, 23)), int(2 ** rng.uniform(0, 10)), kv * rng.choice([1, 4, 20]), kv,
                      8 * rng.randint(1, 32), rng.choice([0, 1, 1, 5, 100, 10 ** 6]), int(2 ** rng.uniform(0, 31))))
    for tokens, batch, heads, kv, hd, new, length in cases:
        n = q(tokens, batch, heads, kv, hd, new, length)
        width = next(w for w in (32, 64, 96, 128, 192, 256) if w >= hd)
        assert 0 <= n <= (1 << 19) * (4 * width + 8), (tokens, batch, heads, kv, hd, new, length, n)


def test_fitting_hints_keep_their_splits():
    """Few rows over long requests are split into 512 units of work; counted by hand.  The last has
    more rows than its hint says: 2^19 / (512 x 32) = 32 splits at most, of 3125 keys rounded up to 3328."""
    q = _workspace()
    for args, splits in (((1, 1, 16, 2, 64, 1, 100000), 196), ((16, 16, 32, 8, 128, 1, 32701), 4),
                         ((92, 23, 6, 2, 256, 6, 3007), 6), ((64, 64, 8, 8, 64, 1, 2048), 0),
                         ((512, 1, 32, 8, 128, 1, 100000), 31)):
        tokens, _, heads, _, hd = args[:5]
        assert q(*args) == splits * tokens * heads * (4 * hd + 8), args


@pytest.mark.parametrize("max_len", [0, -1, -5000])
def test_a_cache_for_requests_of_no_length_is_refused(max_len):
    """It would have had tables of one block."""
    from cobra_amd import CobraCache

    with pytest.raises(ValueError, match="max_len must be positive"):
        CobraCache(1, 2, 64, 2, 4, max_len=max_len, device="cpu")
