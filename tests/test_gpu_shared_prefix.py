"""Dense decode of a batch whose sequences begin with the same tokens, against attention
in 64 bits over every sequence's own keys."""
import math

import pytest
import torch

from _attn64 import attend64, check

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _case(dev, dtype, B, Hq, Hkv, D, prefix, lens, cap=None, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    cap = cap or max(lens)
    q = (r(B, Hq, 1, D) * 1.5).to(dtype)
    k, v = r(B, Hkv, cap, D).to(dtype), r(B, Hkv, cap, D).to(dtype)
    return q, k, v


def _check(got, q, k, v, prefix, lens):
    B, Hq, _, D = q.shape
    G = Hq // k.shape[1]
    for b, n in enumerate(lens):
        P = min(prefix, n)
        for h in range(Hq):
            kk = torch.cat((k[0, h // G, :P], k[b, h // G, P:n]))
            vv = torch.cat((v[0, h // G, :P], v[b, h // G, P:n]))
            o, tol = attend64(q[b, h], kk, vv, torch.ones(1, n, dtype=torch.bool, device=q.device),
                              1 / math.sqrt(D), q.dtype)
            check(got[b, h], o, tol)


CASES = [  # B, Hq, Hkv, D, prefix, lens
    (1, 4, 1, 128, 5, [9]),
    (1, 1, 1, 64, 1, [1]),
    (3, 8, 2, 64, 64, [64, 65, 200]),
    (2, 32, 8, 128, 1000, [1003, 1000]),
    (5, 7, 1, 128, 129, [129, 130, 500, 131, 192]),
    (9, 8, 1, 256, 300, [300 + 17 * i for i in range(9)]),
    (40, 8, 2, 64, 333, [333 + i for i in range(40)]),   # more rows than one block
    (70, 4, 1, 128, 2000, [2001 + (i * 7) % 90 for i in range(70)]),
    (2, 40, 1, 64, 100, [150, 101]),                     # more heads than a wave has rows
    (16, 4, 2, 128, 9000, [9000 + 100 * (i % 5) for i in range(16)]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_shared_prefix(dev, dtype, case):
    """The other sequences' rows of the prefix hold something else: they are not read."""
    from laprune_amd.retrieval import DenseDecoder
    B, Hq, Hkv, D, prefix, lens = CASES[case]
    q, k, v = _case(dev, dtype, B, Hq, Hkv, D, prefix, lens, seed=case)
    k[1:, :, :prefix] = math.nan
    v[1:, :, :prefix] = math.nan
    dec = DenseDecoder(B, Hq, Hkv, D, k.shape[2], dev, dtype)
    got = dec.step(q, k, v, lengths=lens, shared_prefix=prefix)
    _check(got, q, k, v, prefix, lens)
    # device plans, a cache longer than any sequence whose other rows are not finite
    big_k = torch.full((B, Hkv, max(lens) + 300, D), math.nan, dtype=dtype, device=dev)
    big_v = big_k.clone()
    for b, n in enumerate(lens):
        big_k[b, :, :n], big_v[b, :, :n] = k[b, :, :n], v[b, :, :n]
    plans = torch.tensor([[n, n, 0, 0, 0, 0, 0, n] for n in lens], dtype=torch.int32, device=dev)
    dec2 = DenseDecoder(B, Hq, Hkv, D, big_k.shape[2], dev, dtype)
    _check(dec2.step_dev(q, big_k, big_v, plans, shared_prefix=prefix), q, k, v, prefix, lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_uniform_lengths(dev, dtype):
    from laprune_amd.retrieval import DenseDecoder
    q, k, v = _case(dev, dtype, 4, 8, 2, 128, 500, [700] * 4)
    k[1:, :, :500], v[1:, :, :500] = k[:1, :, :500], v[:1, :, :500]
    dec = DenseDecoder(4, 8, 2, 128, 700, dev, dtype)
    got = dec.step(q, k, v, shared_prefix=500).clone()
    _check(got, q, k, v, 500, [700] * 4)
    whole = dec.step(q, k, v)
    assert (got.float() - whole.float()).abs().max() < 1e-2 * whole.float().abs().max()
    _check(dec.step(q, k, v, shared_prefix=700), q, k, v, 700, [700] * 4)


def test_a_sequence_shorter_than_the_prefix(dev):
    """Device plans may hold one (the host form refuses it): it sees its own length of
    the prefix; a length past the cache is cut, an empty sequence gives zeros."""
    from laprune_amd.retrieval import DenseDecoder
    lens = [300, 100, 0, 400]
    q, k, v = _case(dev, torch.bfloat16, 4, 8, 2, 64, 200, [400] * 4)
    plans = torch.tensor([[n, n, 0, 0, 0, 0, 0, n] for n in [300, 100, 0, 10 ** 9]],
                         dtype=torch.int32, device=dev)
    dec = DenseDecoder(4, 8, 2, 64, 400, dev, torch.bfloat16)
    got = dec.step_dev(q, k, v, plans, shared_prefix=200)
    _check(got, q, k, v, 200, lens)
    assert bool((got[2] == 0).all())


def test_own_rows_that_are_not_finite_stay_with_their_sequence(dev):
    from laprune_amd.retrieval import DenseDecoder
    lens = [150, 161, 170]
    q, k, v = _case(dev, torch.float16, 3, 4, 2, 64, 100, lens)
    v[1, :, 140, 5] = math.inf
    dec = DenseDecoder(3, 4, 2, 64, 170, dev, torch.float16)
    got = dec.step(q, k, v, lengths=lens, shared_prefix=100)
    assert bool((got[1, :, 0, 5] == math.inf).all())
    assert bool(got[0].isfinite().all()) and bool(got[2].isfinite().all())
    _check(got, q, k, v, 100, lens)


def test_captured_steps(dev):
    """One captured step follows new lengths in the plans; two graphs of one decoder."""
    from laprune_amd.retrieval import DenseDecoder
    B, Hq, Hkv, D, cap = 3, 8, 2, 128, 700
    q, k, v = _case(dev, torch.bfloat16, B, Hq, Hkv, D, 256, [cap] * B)
    dec = DenseDecoder(B, Hq, Hkv, D, cap, dev)
    plans = torch.zeros(B, 8, dtype=torch.int32, device=dev)
    plans[:, 1] = 300
    graphs = []
    for prefix in (256, 64):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            dec.step_dev(q, k, v, plans, shared_prefix=prefix)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dec.step_dev(q, k, v, plans, shared_prefix=prefix)
        graphs.append((g, prefix))
    for lens in ([256, 300, 699], [700, 257, 256], [400, 400, 400]):
        plans[:, 1] = torch.tensor(lens, device=dev)
        for g, prefix in graphs:
            g.replay()
            torch.cuda.synchronize()
            got = dec.out.clone()
            want = dec.step_dev(q, k, v, plans, shared_prefix=prefix)
            torch.cuda.synchronize()
            assert torch.equal(got, want[:, :, 0])
            _check(want, q, k, v, prefix, lens)


def test_refusals(dev):
    from laprune_amd.retrieval import DenseDecoder
    q, k, v = _case(dev, torch.bfloat16, 2, 4, 2, 64, 5, [20, 20])
    dec = DenseDecoder(2, 4, 2, 64, 20, dev)
    with pytest.raises(RuntimeError, match="exceeds"):
        dec.step(q, k, v, lengths=[20, 10], shared_prefix=11)
    with pytest.raises(RuntimeError, match="exceeds"):
        dec.step(q, k, v, shared_prefix=21)
    with pytest.raises(RuntimeError, match="prefix"):
        dec.step(q, k, v, shared_prefix=-1)
    with pytest.raises(RuntimeError, match="geometry"):
        dec.step(q[:1], k, v, shared_prefix=5)
    with pytest.raises(RuntimeError, match="aligned"):
        kk = torch.empty(2 * 2 * 20 * 64 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 2, 20, 64)
        dec.step(q, kk, kk, shared_prefix=5)
