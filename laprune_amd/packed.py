"""Packed prompts: the tokens of prompts of different lengths side by side in one pass.

The reference prefills one length per batch (laprune/llm/modifiers/aq_evaluation.py:
150-155, 279-322).  Here a pass takes any prompts, each behind any number of tokens
already in its cache, and every sequence gets what it would get alone.  The tables of
such a pass (which sequence and cache row a packed token belongs to, and the blocks of
queries of the attention) are built on the GPU from the lengths, once for all layers
(``lap_pack_prompts``).
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _native as N
from ._ops import ops

MAX_SEQUENCES = 4096  # of one pass (csrc/pack.hip)


@functools.lru_cache(1024)
def prompt_shape(total: int, batch: int, max_keys: int, num_q_heads: int, num_kv_heads: int,
                 head_dim: int, tiles: int = 0) -> tuple[int, int, int]:
    """(tokens per tile, bound of the tiles, parts of a tile's keys) of a pass; tiles:
    their number, when the lengths are known."""
    out = [C.c_int(0) for _ in range(3)]
    N.call("lap_prompt_shape", total, batch, tiles, max_keys, num_q_heads, num_kv_heads, head_dim,
           *map(C.byref, out))
    return tuple(v.value for v in out)


class PackedPrompts:
    """Tables of one packed pass, on the device (:func:`pack_prompts` makes them).

    starts int32 [B + 1]  first packed token of each sequence
    seq    int32 [total]  sequence of a packed token (-1 behind the last one)
    pos    int64 [total]  its position, which is its cache row
    tiles  int32 [n, 4]   the attention's blocks of queries, for the heads given to
                          ``pack_prompts`` (None without them)
    lens, cached: the lengths as host lists, or None when they were device tensors
    longest: the most keys of a sequence, when the lengths are known (else max_keys)
    """

    def __init__(self, batch, total, max_keys, heads, shape, starts, seq, pos, tiles, lens, cached):
        self.B, self.total, self.max_keys = batch, total, max_keys
        self.heads, self.shape = heads, shape
        self.starts, self.seq, self.pos, self.tiles = starts, seq, pos, tiles
        self.lens, self.cached = lens, cached
        self.longest = max_keys if lens is None else max(map(int.__add__, lens, cached))


def _host(v, name: str, batch: int | None = None) -> list[int]:
    v = [int(x) for x in v]
    if any(x < 0 for x in v):
        raise ValueError(f"{name}: negative length")
    if batch is not None and len(v) != batch:
        raise ValueError(f"{name}: one length per sequence ({batch}), got {len(v)}")
    return v


def pack_prompts(lens, cached=None, total: int | None = None, max_keys: int | None = None, *,
                 num_q_heads: int | None = None, num_kv_heads: int | None = None,
                 head_dim: int | None = None, device=None) -> PackedPrompts:
    """Tables of a pass over ``lens[b]`` new tokens of each sequence b, behind
    ``cached[b]`` tokens that its cache holds already (none by default).

    Lengths are host lists, or int32 GPU tensors [B] (both alike).  Tensors are read by
    the kernel alone, without synchronising: ``total`` then gives the packed tokens (a
    sum below it leaves tokens of no sequence, tokens past it are cut off) and
    ``max_keys`` a bound of any sequence's cached and new tokens (by default total, or
    required with a cached tensor).  With the head counts and the head dim the tables
    include the attention's (:func:`laprune_amd.attention.prompt_attention`)."""
    if isinstance(lens, torch.Tensor):
        if cached is not None and not isinstance(cached, torch.Tensor):
            raise ValueError("pack_prompts: lengths both as tensors or both as lists")
        if total is None or (max_keys is None and cached is not None):
            raise ValueError("pack_prompts: tensor lengths need total, and max_keys with cached ones")
        if lens.dtype != torch.int32 or lens.dim() != 1 or lens.numel() == 0:
            raise ValueError("pack_prompts: lengths must be an int32 tensor [B]")
        B = lens.numel()
        host = None, None
        new_dev, cached_dev = lens, cached
        if max_keys is None:
            max_keys = total
    else:
        if isinstance(cached, torch.Tensor):
            raise ValueError("pack_prompts: lengths both as tensors or both as lists")
        new = _host(lens, "lens")
        B = len(new)
        if B == 0:
            raise ValueError("pack_prompts: no sequences")
        old = _host(cached, "cached", B) if cached is not None else [0] * B
        dev = torch.device(device if device is not None else "cuda")
        host = new, old
        if total is None:
            total = sum(new)
        elif total < sum(new):
            raise ValueError(f"pack_prompts: {sum(new)} tokens exceed total = {total}")
        most = max(n + c for n, c in zip(new, old))
        if max_keys is None:
            max_keys = most
        elif max_keys < most:
            raise ValueError(f"pack_prompts: {most} keys exceed max_keys = {max_keys}")
        both = torch.tensor([new, old], dtype=torch.int32).to(dev)
        new_dev, cached_dev = both[0], both[1]
    if total < 0 or max_keys < 0:
        raise ValueError("pack_prompts: negative total or max_keys")
    heads = shape = None
    if (num_q_heads, num_kv_heads, head_dim) != (None, None, None):
        if None in (num_q_heads, num_kv_heads, head_dim):
            raise ValueError("pack_prompts: num_q_heads, num_kv_heads and head_dim go together")
        heads = num_q_heads, num_kv_heads, head_dim
        shape = prompt_shape(total, B, max_keys, *heads)
        if host[0] is not None:
            n = sum(-(-t // shape[0]) for t in host[0])
            shape = prompt_shape(total, B, max_keys, *heads, n)
    bt, n_tiles, _ = shape or (1, -1, 1)
    starts, seq, pos, tiles = ops().pack_prompts(new_dev, cached_dev, total, bt, n_tiles)
    return PackedPrompts(B, total, max_keys, heads, shape, starts, seq, pos, tiles, *host)
