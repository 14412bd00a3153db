"""Packed prompts and shared-prefix decode without a GPU: the tile shape's arithmetic,
and refusals of the host checks and of the C ABI before any device call."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from laprune_amd import _native as N
    return N.lib()


def _err(lib):
    return lib.lap_last_error().decode()


@pytest.mark.parametrize("heads", [(1, 1, 64), (32, 8, 128), (28, 4, 128), (128, 1, 64), (40, 1, 256),
                                   (8, 8, 256), (33, 1, 64)])
@pytest.mark.parametrize("total,B,keys", [(0, 1, 0), (1, 1, 1), (7, 3, 70000), (777, 7, 400),
                                          (16384, 1, 16384), (131072, 256, 131072), (1, 1, 1 << 29)])
def test_prompt_shape(heads, total, B, keys):
    """A tile's rows fit a workgroup (128), the bound holds every split of the
    tokens over the sequences, and no part of the keys is without keys at the longest."""
    from laprune_amd.packed import prompt_shape
    Hq, Hkv, D = heads
    bt, n, ns = prompt_shape(total, B, keys, Hq, Hkv, D)
    G = Hq // Hkv
    assert bt >= 1 and bt * G <= 128 and ns >= 1
    assert n >= total // bt + min(B, total)
    assert ns == 1 or keys > 64 * (ns - 1)


def test_lengths_are_checked_before_any_device_call():
    from laprune_amd.packed import pack_prompts
    t = torch.zeros(2, dtype=torch.int32)
    for args, kw, match in [
            (([],), {}, "no sequences"), (([1, -1],), {}, "negative"), (([1], [1, 2]), {}, "one length"),
            (([1], t), {}, "both"), ((t, [1, 2]), dict(total=3), "both"), ((t,), {}, "need total"),
            ((t, t), dict(total=3), "max_keys"), ((t.long(),), dict(total=3), "int32"),
            (([5],), dict(total=4), "exceed total"), (([5], [3]), dict(max_keys=7), "exceed max_keys"),
            ((t,), dict(total=-1), "negative"), (([1],), dict(num_q_heads=4, device="cpu"), "together")]:
        with pytest.raises(ValueError, match=match):
            pack_prompts(*args, **kw)


def test_prompt_attention_refuses_host_tensors():
    from laprune_amd.attention import _prompt_kernel_fits, prompt_attention
    q, k = torch.zeros(3, 4, 64), torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, k, k, None)
    assert not _prompt_kernel_fits(q[None], k, k)


def test_invalid_arguments_of_the_c_abi(lib):
    from laprune_amd import _native as N
    al, odd, null = C.c_void_p(4096), C.c_void_p(4098), None  # never dereferenced
    i = C.c_int(0)

    def pack(lens=al, B=2, total=10, bt=4, n=6, starts=al, tiles=al):
        return lib.lap_pack_prompts(lens, null, B, total, bt, n, starts, al, al, tiles, null)

    for kw, code, msg in [(dict(lens=null), 1, "null"), (dict(B=0), 1, "sizes"), (dict(total=-1), 1, "sizes"),
                          (dict(B=5000), 2, "5000"), (dict(n=3), 1, "n_tiles"), (dict(bt=0), 1, "n_tiles"),
                          (dict(tiles=odd), 1, "aligned")]:
        assert pack(**kw) == code and msg in _err(lib), kw

    def rope(q=al, dtype=N.BF16, n=4, B=2, D=64, seq=al, st=512, cap=16):
        return lib.lap_qk_rope_append(q, st, D, al, st, D, al, st, D, al, al, D, null, 0.0, null, 0.0,
                                      dtype, n, B, 4, 2, D, seq, al, al, 4096, 2048, D, al, 4096, 2048, D,
                                      cap, al, null)

    for kw, code, msg in [(dict(q=null), 1, "null"), (dict(dtype=N.F32), 1, "fp16/bf16"),
                          (dict(D=72), 2, "multiple of 16"), (dict(D=272), 2, "multiple of 16"),
                          (dict(seq=null), 1, "more tokens"), (dict(q=odd), 1, "aligned"),
                          (dict(st=513), 1, "aligned"), (dict(cap=0), 1, "sizes"), (dict(n=-1), 1, "sizes")]:
        assert rope(**kw) == code and msg in _err(lib), kw
    assert rope(n=0) == 0

    def prompt(q=al, dtype=N.BF16, Hq=8, Hkv=2, D=128, Tq=5, Tk=9, tiles=null, nt=0, bt=8, ns=1,
               scale=0.1, st=1024, ws=null, wsb=0):
        return lib.lap_prompt_attention(q, 8 * st, st, 128, al, al, 4096, 2048, 128, 4096, 2048, 128, dtype,
                                        1, Hq, Hkv, D, Tq, Tk, tiles, nt, bt, ns, 9, scale, al, 8 * st, st,
                                        128, ws, wsb, null)

    for kw, code, msg in [(dict(q=null), 1, "null"), (dict(dtype=N.F32), 1, "fp16/bf16"),
                          (dict(Hq=7), 1, "GQA"), (dict(D=96), 2, "head dim"),
                          (dict(Hq=129, Hkv=1), 2, "group size"), (dict(Tq=10), 1, "exceed"),
                          (dict(scale=-1.0), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
                          (dict(q=odd), 1, "aligned"), (dict(st=1025), 1, "aligned"),
                          (dict(bt=33), 1, "tile"), (dict(bt=0), 1, "tile"), (dict(ns=0), 1, "tile"),
                          (dict(ns=2), 4, "workspace"), (dict(ns=2, ws=al, wsb=100), 4, "workspace"),
                          (dict(Tk=1 << 30), 1, "sizes")]:
        assert prompt(**kw) == code and msg in _err(lib), kw
    assert prompt(tiles=al, nt=0) == 0  # no tile: nothing to launch

    def shared(q=al, dtype=N.BF16, B=2, Hq=8, T=300, prefix=200, D=128, scale=0.1, kst=128):
        return lib.lap_shared_attn_decode(q, 1024, 128, al, al, dtype, B, Hq, 2, T, D, 1 << 20, 1 << 18,
                                          kst, 1 << 20, 1 << 18, 128, prefix, null, scale, al, null, 0, null)

    for kw, code, msg in [(dict(q=null), 1, "null"), (dict(dtype=N.F32), 1, "fp16/bf16"), (dict(B=0), 1, "sizes"),
                          (dict(T=0), 1, "sizes"), (dict(prefix=301), 1, "prefix"), (dict(prefix=-1), 1, "prefix"),
                          (dict(Hq=9), 1, "GQA"), (dict(D=80), 2, "head dim"), (dict(scale=0.0), 1, "scale"),
                          (dict(q=odd), 1, "aligned"), (dict(kst=132), 1, "aligned"), (dict(), 4, "workspace")]:
        assert shared(**kw) == code and msg in _err(lib), kw
    assert lib.lap_prompt_shape(-1, 1, 0, 1, 8, 2, 64, C.byref(i), C.byref(i), C.byref(i)) == 1
    assert lib.lap_prompt_shape(1, 1, 0, 1, 8, 3, 64, C.byref(i), C.byref(i), C.byref(i)) == 1
    assert lib.lap_prompt_shape(1, 1, 0, 1, 8, 2, 96, C.byref(i), C.byref(i), C.byref(i)) == 2


def test_launches_past_the_limit_are_refused(lib):
    """A launch takes fewer than 2^32 work-items: 2^24 workgroups of 256."""
    from laprune_amd import _native as N
    al, odd, null = C.c_void_p(4096), C.c_void_p(4100), None  # never dereferenced

    def prompt(tiles, nt, ns=1, ws=null, B=1, Hkv=2):
        return lib.lap_prompt_attention(al, 1024, 256, 64, al, al, 4096, 2048, 64, 4096, 2048, 64, N.BF16,
                                        B, 2 * Hkv, Hkv, 64, 1, 9, tiles, nt, 64, ns, 9, 0.1, al, 1024, 256,
                                        64, ws, 1 << 62, null)

    def shared(B, T, ws=al):
        return lib.lap_shared_attn_decode(al, 1024, 64, al, al, N.BF16, B, 4, 2, T, 64, 4096, 2048, 64, 4096,
                                          2048, 64, 0, null, 0.1, al, ws, 0, null)

    def rope(n):
        return lib.lap_qk_rope_append(al, 256, 64, al, 128, 64, al, 128, 64, al, al, 64, null, 0.0, null, 0.0,
                                      N.BF16, n, 2, 4, 2, 64, al, al, al, 4096, 2048, 64, al, 4096, 2048, 64, 16,
                                      al, null)

    for call in [lambda: prompt(al, 1 << 23), lambda: prompt(null, 0, B=1 << 23),
                 lambda: prompt(al, 1 << 20, ns=8, ws=al), lambda: prompt(al, 1 << 18, ns=17, ws=al),
                 lambda: shared(1 << 23, 64), lambda: rope(1 << 27)]:
        assert call() == 1 and "too many rows" in _err(lib)
    assert prompt(al, 1, ns=2, ws=odd) == 1 and "aligned" in _err(lib)
    assert shared(2, 5000, odd) == 1 and "aligned" in _err(lib)


def test_workspace_sizes(lib):
    from laprune_amd import _native as N
    assert N.size_query("lap_prompt_attention_workspace_size", 10, 8, 128, 1) == 0
    assert N.size_query("lap_prompt_attention_workspace_size", 10, 8, 128, 3) == 10 * 8 * 3 * 130 * 4
    assert N.size_query("lap_shared_attn_decode_workspace_size", 16, 32, 8, 128, 17000, 16384) % (512 * 130 * 4) == 0
