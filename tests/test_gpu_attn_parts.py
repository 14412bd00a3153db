"""Splits of the keys and their merge: values that show the share of every tile and of every
place within a tile in the output, so that one tile, part or key too few or too many is
visible at any length.

All values are 0 or 1, so an output is a share sum_{t in C} p_t / sum_t p_t and its roundings
count relatively: a weight's to the data type (half a step), the output's (half a step), and
fp32 throughout otherwise: a score of D products and the argument of its exponential (both
enter the weight in proportion: SCORE below), and sums of 16 weights in a lane per tile, of a lane's tiles,
rescaled once each, and of the parts, twice each for numerator and denominator."""
import math

import pytest
import torch

from _attn64 import FP32, half_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
WIDE, NARROW = "tiles", "places"


def _values(pattern, T, D, dtype, dev):
    """Column d is 1 on tiles d, d + D, ... of 64 keys, or on keys d, d + D, ..."""
    t = torch.arange(T, device=dev)
    at = (t // 64 if pattern == WIDE else t) % D
    return torch.nn.functional.one_hot(at, D).to(dtype)


def _shares(got, q, k, v, visible, dtype):
    """got, q [n, D] of one head, k and v [T, D]."""
    T, D = k.shape
    s = q.double() @ k.double().T / math.sqrt(D)
    s = s.masked_fill(~visible, -math.inf)
    want = s.softmax(-1) @ v.double()
    u = half_step(dtype)
    most = (q.double().abs() @ k.double().abs().T).max().item() / math.sqrt(D)
    score = 2 * (D + 4) * most + 8 + 4 * most
    tol = want * (2 * u + FP32 * (2 * score + 2 * (16 + 2 * (T // 64 + 1) + 1100)))
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # an output below fp16's normal range
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), (d / tol.clamp_min(1e-30)).max().item()


def _case(dev, dtype, B, Hkv, T, D, n, Hq, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    return (r(n, Hq, D) * 0.5).to(dtype), r(B, Hkv, T, D).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nsplit", [1, 2, 7, 16, 17, 26, 51, 102])
def test_prompt_parts(dev, dtype, D, nsplit):
    """Up to 16 parts are merged by one wave, more by four, 64 at a time; sequences that
    fill all of them, some, and one."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    lens, cached = [2, 1, 3], [6463, 64 * 40, 20]  # the last part of the longest: one key
    q, k = _case(dev, dtype, 3, 2, 6465, D, sum(lens), 4, nsplit)
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=4, num_kv_heads=2, head_dim=D)
    plan.shape = (*plan.shape[:2], nsplit)
    for pattern in (WIDE, NARROW):
        v = _values(pattern, 6465, D, dtype, dev).expand(3, 2, -1, -1)
        got = prompt_attention(q, k, v, plan)
        i = 0
        for b, (n, c) in enumerate(zip(lens, cached)):
            vis = torch.arange(n + c, device=dev) <= torch.arange(n, device=dev)[:, None] + c
            for h in range(4):
                _shares(got[i:i + n, h], q[i:i + n, h], k[b, h // 2, :n + c], v[b, h // 2, :n + c],
                        vis, dtype)
            i += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_of_many_keys(dev, dtype, D):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    lens, cached, T = [1, 3], [70001, 130000], 130003
    q, k = _case(dev, dtype, 2, 1, T, D, 4, 4, 9)
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=4, num_kv_heads=1, head_dim=D)
    assert plan.shape[2] > 16
    for pattern in (WIDE, NARROW):
        v = _values(pattern, T, D, dtype, dev).expand(2, 1, -1, -1)
        got = prompt_attention(q, k, v, plan)
        i = 0
        for b, (n, c) in enumerate(zip(lens, cached)):
            vis = torch.arange(n + c, device=dev) <= torch.arange(n, device=dev)[:, None] + c
            for h in range(4):
                _shares(got[i:i + n, h], q[i:i + n, h], k[b, 0, :n + c], v[b, 0, :n + c], vis, dtype)
            i += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 40, 2100])
def test_causal_prompts_of_whole_and_masked_tiles(dev, dtype, D, n):
    """Rows of many tokens: whole tiles, masked ones, and waves that see none of a tile."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    for Hq, cached in ((1, 0), (3, 77)):
        q, k = _case(dev, dtype, 1, 1, n + cached, D, n, Hq, n)
        plan = pack_prompts([n], [cached], device=dev, num_q_heads=Hq, num_kv_heads=1, head_dim=D)
        vis = torch.arange(n + cached, device=dev) <= torch.arange(n, device=dev)[:, None] + cached
        for nsplit in (1, 3):
            plan.shape = (*plan.shape[:2], nsplit)
            for pattern in (WIDE, NARROW):
                v = _values(pattern, n + cached, D, dtype, dev)[None, None]
                got = prompt_attention(q, k, v, plan)
                for h in range(Hq):
                    _shares(got[:, h], q[:, h], k[0, 0], v[0, 0], vis, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,Hkv,prefix,lens,parts", [
    (2, 1, 3000, [5000, 3001], 17), (2, 1, 15000, [20000, 15001], 65), (1, 1, 0, [200], 1),
    (3, 2, 64, [64, 300, 129], 1), (40, 1, 700, [700 + 31 * i for i in range(40)], 1)])
def test_shared_prefix_parts(dev, dtype, D, B, Hkv, prefix, lens, parts):
    """At least `parts` parts, those of the prefix and each sequence's own."""
    from laprune_amd import _native as N
    from laprune_amd.retrieval import DenseDecoder
    T, Hq = max(lens), 2 * Hkv
    ws = N.size_query("lap_shared_attn_decode_workspace_size", B, Hq, Hkv, D, T, prefix)
    assert ws >= parts * B * Hq * (D + 2) * 4 or parts == 1
    q, k = _case(dev, dtype, B, Hkv, T, D, B, Hq, prefix)
    k[1:, :, :prefix] = k[:1, :, :prefix]
    dec = DenseDecoder(B, Hq, Hkv, D, T, dev, dtype)
    for pattern in (WIDE, NARROW):
        v = _values(pattern, T, D, dtype, dev).expand(B, Hkv, -1, -1)
        if prefix:
            got = dec.step(q[:, :, None], k, v, lengths=lens, shared_prefix=prefix)[:, :, 0]
        else:
            got = torch.empty_like(q)
            dec._ops.shared_decode(q, k, v, T, 0, None, 1 / math.sqrt(D), got)
        for b, n in enumerate(lens):
            for h in range(Hq):
                _shares(got[b, h][None], q[b, h][None], k[b, h // 2, :n], v[b, h // 2, :n],
                        torch.ones(1, n, dtype=torch.bool, device=dev), dtype)
