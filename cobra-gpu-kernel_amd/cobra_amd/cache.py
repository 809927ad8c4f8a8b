"""A key/value cache held in 8 bits, for requests that grow by some tokens a call.

``CobraCache`` owns the pool of blocks of every layer and the tables, lengths and free blocks
that all layers share, all on the device; its methods are ``ops.cache_reserve``, ``cache_trim``,
``cache_append``, ``cache_positions``, ``cache_attn`` and ``cache_prefix_attn`` on them, and wait for
nothing.  ``CobraTransformer.extend``
runs the stack over new tokens with one.  (The reference's attention sees whole sequences,
torch_transformer_benchmark.py:88-123; it keeps no cache.)
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops


class CobraCache:
    """``requests`` rows of block tables over a pool of ``num_blocks`` blocks of ``block_size``
    tokens for each of ``layers`` layers.

    ``dtype`` float8_e4m3fn or int8; ``max_len``: the most tokens of a request (default: the
    whole pool).  A row is free when its length is 0; what a row means is the caller's.
    """

    def __init__(self, layers: int, kv_heads: int, head_dim: int, requests: int, num_blocks: int,
                 block_size: int = 64, dtype: torch.dtype = torch.float8_e4m3fn, max_len: Optional[int] = None,
                 device=None) -> None:
        for name, v in (("layers", layers), ("kv_heads", kv_heads), ("requests", requests),
                        ("num_blocks", num_blocks)):
            if v <= 0:
                raise ValueError(f"{name} must be positive")
        if max_len is not None and max_len <= 0:
            raise ValueError(f"max_len must be positive, got {max_len}")
        if block_size not in ops.CACHE_BLOCKS:
            raise ValueError(f"block_size must be one of {ops.CACHE_BLOCKS}, got {block_size}")
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise TypeError(f"the cache is held in float8_e4m3fn or int8, got {dtype}")
        width = ops.cache_width(head_dim)
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise ValueError(f"the cache lives on a GPU, got {dev}")
        self.layers, self.kv_heads, self.head_dim, self.block_size = layers, kv_heads, head_dim, block_size
        shape = (num_blocks, kv_heads, block_size, width)
        self.k: List[torch.Tensor] = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.v: List[torch.Tensor] = [torch.zeros((num_blocks, kv_heads, width, block_size), dtype=dtype, device=dev)
                                      for _ in range(layers)]
        scale = (num_blocks, kv_heads)
        self.k_scale = [torch.ones(scale, dtype=torch.float32, device=dev) for _ in range(layers)]
        self.v_scale = [torch.ones(scale, dtype=torch.float32, device=dev) for _ in range(layers)]
        rows = num_blocks if max_len is None else min(num_blocks, -(-max_len // block_size))
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.block_table = torch.zeros((requests, max(1, rows)), dtype=torch.int32, device=dev)
        self.free_list = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), num_blocks, dtype=torch.int32, device=dev)
        self._held: List[object] = []

    def hold(self, *things: object) -> None:
        """Keeps what a captured step over this cache reads alive for as long as the cache lives."""
        self._held += [t for t in things if not any(t is h for h in self._held)]

    def reserve(self, new_lens: torch.Tensor, tokens: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Room for ``new_lens`` more tokens of each request -> ``(slots, cu, missing)`` (``ops.cache_reserve``)."""
        return ops.cache_reserve(self.lens, new_lens, self.block_table, self.free_list, self.free_count,
                                 self.block_size, tokens)

    def trim(self, keep_lens: torch.Tensor) -> torch.Tensor:
        """Requests cut to ``keep_lens`` tokens, 0 for those that are over -> ``refused`` (``ops.cache_trim``)."""
        return ops.cache_trim(self.lens, keep_lens, self.block_table, self.free_list, self.free_count,
                              self.block_size)

    def positions(self, cu: torch.Tensor, tokens: int, prefix: Optional[int] = None) -> torch.Tensor:
        """Where the new tokens of a reserve stand in their requests (``ops.cache_positions``)."""
        return ops.cache_positions(cu, self.lens, tokens, prefix)

    def append(self, layer: int, qkv: torch.Tensor, slots: torch.Tensor, heads: int) -> None:
        """A layer's new keys and values into their slots (``ops.cache_append``)."""
        ops.cache_append(qkv, slots, heads, self.head_dim, self.k[layer], self.v[layer], self.k_scale[layer],
                         self.v_scale[layer])

    def attn(self, layer: int, q: torch.Tensor, cu: torch.Tensor, heads: int, scale: float, causal: bool = True,
             max_new: Optional[int] = None, max_len: Optional[int] = None,
             out: Optional[torch.Tensor] = None, prefix: Optional[int] = None,
             max_prefix: Optional[int] = None) -> torch.Tensor:
        """Attention of the new tokens over what a layer's cache holds of their requests (``ops.cache_attn``),
        or of row ``prefix`` and their requests (``ops.cache_prefix_attn``)."""
        if prefix is not None:
            return ops.cache_prefix_attn(q, cu, self.lens, self.block_table, prefix, heads, self.head_dim, scale,
                                         self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                         causal=causal, max_new=max_new, max_len=max_len, max_prefix=max_prefix, out=out)
        return ops.cache_attn(q, cu, self.lens, self.block_table, heads, self.head_dim, scale, self.k[layer],
                              self.v[layer], self.k_scale[layer], self.v_scale[layer], causal=causal,
                              max_new=max_new, max_len=max_len, out=out)
