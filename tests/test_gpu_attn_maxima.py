"""The running maximum of prompt attention and of decode over a shared prefix: every key of
a tile counts for it, whichever lane holds its score.  Against attention in 64 bits with the
bounds of _attn64."""
import math

import pytest
import torch

from _attn64 import attend64, check

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _prompt(q, k, v, lens, cached):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    plan = pack_prompts(lens, cached, device=q.device, num_q_heads=q.shape[1], num_kv_heads=k.shape[1],
                        head_dim=q.shape[2])
    return prompt_attention(q, k, v, plan)


def _check(got, q, k, v, cached):
    """got, q [n, Hq, D]: the last n tokens of one sequence behind `cached`."""
    n, Hq, D = q.shape
    T = n + cached
    vis = torch.arange(T, device=q.device) <= torch.arange(n, device=q.device)[:, None] + cached
    for h in range(Hq):
        kv = h // (Hq // k.shape[1])
        check(got[:, h], *attend64(q[:, h], k[0, kv, :T], v[0, kv, :T], vis, 1 / math.sqrt(D), q.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("back", [0, 1, 130])
def test_every_key_as_the_largest(dev, dtype, D, back):
    """Row i's score of key i + 130 - back is some 2^29 (D = 64) to 2^58 above the others', in a
    masked tile (its own key, the one before) or in one that all rows of the wave see."""
    n, cached = 200, 130
    g = torch.Generator(device=dev).manual_seed(D + back)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    k, v = r(1, 1, n + cached, D).to(dtype), r(1, 1, n + cached, D).to(dtype)
    top = torch.arange(n, device=dev) + cached - back
    q = (2.5 * k[0, 0, top].float())[:, None].repeat(1, 2, 1).to(dtype)
    _check(_prompt(q, k, v, [n], [cached]), q, k, v, cached)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("first", [0, 4])
def test_half_of_the_keys_without_a_finite_score(dev, dtype, D, first):
    """Of the first 128 keys `first` to first + 3 of every eight score -inf; the others keep
    their weights beside the keys behind, which all score."""
    n, T = 3, 192
    big = torch.finfo(dtype).max
    g = torch.Generator(device=dev).manual_seed(D + first)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    q, k, v = r(n, 2, D).to(dtype), r(1, 1, T, D).to(dtype), r(1, 1, T, D).to(dtype)
    # fp16 products do not overflow fp32: those keys score -4e6 at least, which weighs 0 as well
    q[..., 0] = 60.0
    k[..., 0] = 0.0
    t = torch.arange(T, device=dev)
    gone = ((t - first) % 8 < 4) & (t < 128)
    k[0, 0, gone, 0] = -big
    got = _prompt(q, k, v, [n], [T - n])
    finite = (t <= torch.arange(n, device=dev)[:, None] + T - n) & ~gone
    for h in range(2):
        kk = torch.where(gone[:, None], torch.zeros_like(k[0, 0]), k[0, 0])
        check(got[:, h], *attend64(q[:, h], kk, v[0, 0], finite, 1 / math.sqrt(D), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_every_key_as_the_largest_of_a_shared_prefix(dev, dtype, D):
    """Sequence b's largest score is at key 3 b, of the prefix or of its own keys."""
    from laprune_amd.retrieval import DenseDecoder
    B, prefix, T = 70, 150, 209
    g = torch.Generator(device=dev).manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    k, v = r(B, 1, T, D).to(dtype), r(B, 1, T, D).to(dtype)
    k[1:, :, :prefix], v[1:, :, :prefix] = k[:1, :, :prefix], v[:1, :, :prefix]
    b = torch.arange(B, device=dev)
    q = (2.5 * k[b, 0, 3 * b].float())[:, None, None].repeat(1, 4, 1, 1).to(dtype)
    got = DenseDecoder(B, 4, 1, D, T, dev, dtype).step(q, k, v, shared_prefix=prefix)
    all_keys = torch.ones(1, T, dtype=torch.bool, device=dev)
    for i in range(B):
        for h in (0, 3):
            check(got[i, h], *attend64(q[i, h], k[i, 0], v[i, 0], all_keys, 1 / math.sqrt(D), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("at", [0, 5, 40000])
@pytest.mark.parametrize("nsplit", [1, 5])
def test_many_small_weights_beside_a_large_one(dev, dtype, D, at, nsplit):
    """Key `at` weighs 1 and its value is 0; 65000 others weigh 2^-18 to 2^-30 each and their
    values are 1, so the output is the others' share.  A weight is off by half a step of its
    own in the normal range, and in fp16 below that by half a step of 2^-24 at weights that
    are at least 2^7 where the row's largest is 1 (half a step of 2^-31)."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    T, n = 65001, 5
    k = torch.zeros(1, 1, T, D, dtype=dtype, device=dev)
    k[..., at, 0] = 8.0
    v = torch.ones(1, 1, T, D, dtype=dtype, device=dev)
    v[..., at, :] = 0.0
    power = torch.tensor([18.0, 23.0, 25.2, 27.0, 30.0], device=dev)
    q = torch.zeros(n, 1, D, dtype=dtype, device=dev)
    q[:, 0, 0] = (power * math.log(2) * math.sqrt(D) / 8).to(dtype)
    plan = pack_prompts([n], [T - n], device=dev, num_q_heads=1, num_kv_heads=1, head_dim=D)
    plan.shape = (*plan.shape[:2], nsplit)
    got = prompt_attention(q, k, v, plan)[:, 0].double()
    seen = torch.arange(T - n + 1, T + 1, device=dev).double()[:, None] - 1
    w = (-8 * q[:, :, 0].double() / math.sqrt(D)).exp()
    want = (seen * w / (1 + seen * w)).expand(n, D)
    # fp32 (half steps): the score and the exponential's argument up to 30, each twice, and the
    # sums of 16 weights in a lane per tile, of its tiles and of the parts
    tol = want * (torch.finfo(dtype).eps + 2.0 ** -24 * (8 + 4 * 30 + 2 * (16 + 2 * (T // 64 + 1) + 8)))
    if dtype == torch.float16:
        tol = tol + seen * 2.0 ** -32 + 2.0 ** -25  # the weights' and the output's smallest steps
    d = (got - want).abs()
    assert bool((d <= tol).all()), (d / tol)[:, 0].tolist()
