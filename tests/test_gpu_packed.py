"""Packed prompts: the tables built from request lengths, norms and rotation with the
cache append, and causal attention over the caches, each against its definition (the
floating ones in 64 bits, with bounds counted from the roundings of the contract)."""
import math

import pytest
import torch

from _attn64 import FP32, attend64, check, half_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _tables(lens, cached, total):
    starts, rows = [0], []
    for b, (n, c) in enumerate(zip(lens, cached)):
        rows += [(b, c + i) for i in range(n)]
        starts.append(len(rows))
    rows = rows[:total] + [(-1, 0)] * (total - len(rows))
    return [min(s, total) for s in starts], [r[0] for r in rows], [r[1] for r in rows]


LENS = [([1], [0]), ([5], [0]), ([64], [7]), ([3, 0, 1, 0, 0, 130], [0, 9, 5, 1, 0, 70000]),
        ([0, 0, 7], [1, 2, 3]), ([7, 0, 0], [1, 2, 3]), ([1] * 70, list(range(70))),
        ([i % 5 for i in range(1500)], [i % 77 for i in range(1500)]),
        ([4097, 1, 8192], [0, 0, 0]), ([1] * 4096, [2] * 4096)]


@pytest.mark.parametrize("case", range(len(LENS)))
@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (4, 4, 256)])
def test_pack_tables(dev, case, heads):
    from laprune_amd.packed import pack_prompts
    lens, cached = LENS[case]
    Hq, Hkv, D = heads
    p = pack_prompts(lens, cached, device=dev, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D)
    starts, seq, pos = _tables(lens, cached, sum(lens))
    assert p.starts.tolist() == starts and p.seq.tolist() == seq and p.pos.tolist() == pos
    # the tiles cover every token once, each tile in one sequence, most keys first
    bt, bound, _ = p.shape
    tiles = [t for t in p.tiles.tolist() if t[1]]
    assert p.tiles.shape[0] == bound and p.tiles.tolist()[:len(tiles)] == tiles
    covered = []
    for q0, n, b, key0 in tiles:
        assert 0 < n <= bt and starts[b] <= q0 and q0 + n <= starts[b + 1]
        assert key0 == cached[b] + q0 - starts[b]
        covered += range(q0, q0 + n)
    assert sorted(covered) == list(range(sum(lens)))
    cost, top = [k + n for _, n, _, k in tiles], max(n + c for n, c in zip(lens, cached) if n)
    assert all(a + top / 1023 + 1 >= b for a, b in zip(cost, cost[1:]))  # in steps of a 1024th


@pytest.mark.parametrize("total", [0, 100, 139, 150])
def test_pack_device_lengths_padded_and_cut(dev, total):
    """Device lengths: a sum below the total leaves tokens of no sequence, tokens past
    it are cut off, a negative length counts as zero."""
    from laprune_amd.packed import pack_prompts
    lens, cached = [3, -4, 1, 135], [0, 2, 5, 9]
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    p = pack_prompts(t(lens), t(cached), total=total, max_keys=144, num_q_heads=8, num_kv_heads=2,
                     head_dim=64)
    starts, seq, pos = _tables([max(n, 0) for n in lens], cached, total)
    assert p.starts.tolist() == starts and p.seq.tolist() == seq and p.pos.tolist() == pos
    tiles = p.tiles.tolist()
    assert sum(t[1] for t in tiles) == min(total, 139)
    assert all(t[0] + t[1] <= total for t in tiles)
    assert p.lens is None


# ------------------------------------------------------------------ norm, rotation, append

def _rope_inputs(dev, dtype, n, Hq, Hkv, D, seed=0, fused=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(1, n, (Hq + 2 * Hkv) * D + (0 if fused else 8), generator=g, device=dev)
    x = (x * (0.2 + 3 * torch.rand(x.shape[-1], generator=g, device=dev))).to(dtype)
    q, k, v = x[..., :(Hq + 2 * Hkv) * D].split([Hq * D, Hkv * D, Hkv * D], dim=-1)
    a = torch.rand(1, n, D // 2, generator=g, device=dev) * 6.3
    a = torch.cat((a, a), -1)
    w = [(1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dtype) for _ in range(2)]
    return q, k, v, a.cos().to(dtype), a.sin().to(dtype), w


def _cache(dev, dtype, B, Hkv, D, cap):
    from laprune_amd.cache import DecodeKVCache
    c = DecodeKVCache(None, B, Hkv, D, cap, dtype=dtype, device=dev)
    c.k.fill_(7.0)
    c.v.fill_(9.0)
    return c


GEOMETRY = [(8, 2, 64), (32, 8, 128), (7, 1, 128), (3, 3, 256), (2, 1, 16), (4, 2, 80), (2, 2, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", GEOMETRY)
@pytest.mark.parametrize("norms", ["both", "q", "k", "none"])
def test_rope_append_packed(dev, dtype, heads, norms):
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D = heads
    lens, cached = [5, 0, 1, 33], [0, 4, 70, 3]
    n, cap = sum(lens), 71
    q, k, v, cos, sin, (qw, kw) = _rope_inputs(dev, dtype, n, Hq, Hkv, D)
    c = _cache(dev, dtype, 4, Hkv, D, cap)
    plan = pack_prompts(lens, cached, device=dev)
    qn, kn = (qw, 1e-6) if norms in ("both", "q") else None, (kw, 1e-5) if norms in ("both", "k") else None
    out = c.rope_append_packed(q, k, v, cos, sin, plan, q_norm=qn, k_norm=kn)
    torch.cuda.synchronize()
    seq, pos = plan.seq.long(), plan.pos

    def want(x, norm):
        """(value, bound): fp32 throughout and one rounding, or the model's own ops."""
        x = x.reshape(n, -1, D)
        co, si = cos[0, :, None], sin[0, :, None]
        rot = lambda y: torch.cat((-y[..., D // 2:], y[..., :D // 2]), -1)
        if norm is None:
            return ((x * co) + (rot(x) * si)).double(), torch.zeros(1, device=dev)
        w, eps = norm
        x = x.double()
        y = w.double() * x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        o = y * co.double() + rot(y) * si.double()
        # fp32: the mean of D squares, the root and three products and a sum each
        mag = y.abs() * co.abs().double() + rot(y).abs() * si.abs().double()
        return o, half_step(dtype) * o.abs() + FP32 * (D + 12) * mag + 2.0 ** -25 * (dtype == torch.float16)

    def near(got, wanted, bound):
        d = (got.double() - wanted).abs()
        assert bool((d <= bound).all()), (d / bound.clamp_min(1e-30)).max().item()

    near(out, *want(q, qn))
    near(c.k[seq, :, pos], *want(k, kn))
    assert torch.equal(c.v[seq, :, pos], v.reshape(n, Hkv, D))
    # nothing else is touched
    c.k[seq, :, pos] = 7.0
    c.v[seq, :, pos] = 9.0
    assert bool((c.k == 7.0).all()) and bool((c.v == 9.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_form_equals_the_packed_form(dev, dtype):
    """One token per sequence: rope_append with norms writes what the packed call
    writes, and without norms the packed call writes what rope_append writes."""
    from laprune_amd.packed import pack_prompts
    B, Hq, Hkv, D = 5, 8, 2, 128
    q, k, v, cos, sin, (qw, kw) = _rope_inputs(dev, dtype, B, Hq, Hkv, D, seed=3)
    cached = [0, 9, 3, 12, 7]
    pos = torch.tensor(cached, device=dev)[:, None]
    plan = pack_prompts([1] * B, cached, device=dev)
    per = lambda x: x.reshape(B, 1, -1)
    for norms in ({}, dict(q_norm=(qw, 1e-6), k_norm=(kw, 1e-6))):
        a, b = _cache(dev, dtype, B, Hkv, D, 16), _cache(dev, dtype, B, Hkv, D, 16)
        qa = torch.empty(B, Hq, D, dtype=dtype, device=dev)
        a.rope_append(per(q), per(k), per(v), per(cos), per(sin), pos, qa, **norms)
        qb = b.rope_append_packed(q, k, v, cos, sin, plan, **norms)
        assert torch.equal(qa, qb) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_row_layouts(dev):
    """Tokens in two dimensions of one stride, and one table row for all tokens; tokens
    that do not lie at one stride are refused."""
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D = 4, 2, 64
    q, k, v, cos, sin, _ = _rope_inputs(dev, torch.float16, 12, Hq, Hkv, D, seed=6)
    plan = pack_prompts([6, 6], device=dev)
    two = lambda x: x.unflatten(1, (2, 6))[0]
    one = lambda x: x[:, :1].expand(1, 12, D)
    a, b = _cache(dev, torch.float16, 2, Hkv, D, 8), _cache(dev, torch.float16, 2, Hkv, D, 8)
    qa = a.rope_append_packed(two(q), two(k), two(v), one(cos), one(sin), plan)
    qb = b.rope_append_packed(q, k, v, one(cos).contiguous(), one(sin).contiguous(), plan)
    assert torch.equal(qa, qb) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    for bad in (two(cos)[:, :1].expand(2, 6, D), two(cos).transpose(0, 1)):
        with pytest.raises(RuntimeError, match="one stride"):
            a.rope_append_packed(q, k, v, bad, one(sin), plan)


def test_tokens_of_no_sequence_and_past_the_capacity(dev):
    """Tokens behind the last sequence leave everything as it was; a token past the
    capacity is rotated but not cached."""
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D, n = 4, 2, 64, 12
    q, k, v, cos, sin, _ = _rope_inputs(dev, torch.bfloat16, n, Hq, Hkv, D, seed=5)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    plan = pack_prompts(t([3, 5]), t([0, 14]), total=n, max_keys=20)
    c = _cache(dev, torch.bfloat16, 2, Hkv, D, 16)
    out = torch.full((n, Hq, D), 5.0, dtype=torch.bfloat16, device=dev)
    c.rope_append_packed(q, k, v, cos, sin, plan, out)
    assert bool((out[8:] == 5.0).all()) and not bool((out[:8] == 5.0).all(-1).any())
    assert torch.equal(c.v[0, :, :3].transpose(0, 1), v[0, :3].view(3, Hkv, D))
    assert torch.equal(c.v[1, :, 14:].transpose(0, 1), v[0, 3:5].view(2, Hkv, D))
    assert bool((c.v[0, :, 3:] == 9).all()) and bool((c.v[1, :, :14] == 9).all())


# ------------------------------------------------------------------ prompt attention

def _attn_case(dev, dtype, Hq, Hkv, D, lens, cached, seed=0, cap_more=0, scale=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    cap = max(n + c for n, c in zip(lens, cached)) + cap_more
    q = (r(sum(lens), Hq, D) * scale).to(dtype)
    k, v = r(len(lens), Hkv, cap, D).to(dtype), r(len(lens), Hkv, cap, D).to(dtype)
    return q, k, v


def _check_prompt(got, q, k, v, lens, cached, scale=None):
    Hq, D = q.shape[1:]
    G = Hq // k.shape[1]
    worst, i = 0.0, 0
    for b, (n, c) in enumerate(zip(lens, cached)):
        if not n:
            continue
        vis = torch.arange(n + c, device=q.device) <= torch.arange(n, device=q.device)[:, None] + c
        for h in range(Hq):
            o, tol = attend64(q[i:i + n, h], k[b, h // G, :n + c], v[b, h // G, :n + c], vis,
                              scale or 1 / math.sqrt(D), q.dtype)
            worst = max(worst, check(got[i:i + n, h], o, tol))
        i += n
    return worst


PROMPTS = [  # heads, new, cached
    ((1, 1, 64), [1], [0]),
    ((4, 1, 128), [1, 1, 1], [0, 63, 64]),
    ((8, 2, 64), [5, 0, 64, 65, 1, 200], [0, 3, 0, 0, 130, 1]),
    ((32, 8, 128), [31, 97, 1, 128], [0, 0, 500, 33]),
    ((7, 1, 128), [37, 36, 150], [0, 1, 64]),
    ((28, 4, 128), [40], [2000]),
    ((3, 3, 256), [70, 1], [0, 0]),
    ((8, 1, 256), [33, 130], [129, 0]),
    ((40, 1, 64), [9, 30], [5, 0]),       # more heads than a wave has rows
    ((128, 1, 256), [3], [10]),           # one token fills a workgroup's rows
    ((16, 8, 64), [700, 300, 411], [0, 0, 64]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompt_attention(dev, dtype, case):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    (Hq, Hkv, D), lens, cached = PROMPTS[case]
    q, k, v = _attn_case(dev, dtype, Hq, Hkv, D, lens, cached, seed=case)
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D)
    _check_prompt(prompt_attention(q, k, v, plan), q, k, v, lens, cached)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 32, 100, 128])
@pytest.mark.parametrize("nsplit", [1, 2, 5])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_every_tile_shape_and_split(dev, dtype, rows, nsplit, D):
    """Each tile height, with the keys whole and in parts (some of them empty)."""
    from laprune_amd import packed
    from laprune_amd.attention import prompt_attention
    Hq, Hkv, lens, cached = 6, 2, [150, 1, 61], [0, 300, 7]
    q, k, v = _attn_case(dev, dtype, Hq, Hkv, D, lens, cached, seed=rows)
    bt = rows // 3
    shape = (bt, sum(lens) // bt + len(lens), nsplit)
    plan = packed.pack_prompts(lens, cached, device=dev, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D)
    both = torch.tensor([lens, cached], dtype=torch.int32, device=dev)
    plan.shape = shape
    plan.tiles = packed.ops().pack_prompts(both[0], both[1], plan.total, bt, shape[1])[3]
    out = torch.full((plan.total + 5, Hq, D), 3.0, dtype=dtype, device=dev)
    prompt_attention(q, k, v, plan, out=out[:plan.total])
    _check_prompt(out[:plan.total], q, k, v, lens, cached)
    assert bool((out[plan.total:] == 3.0).all())


@pytest.mark.parametrize("nsplit", [1, 3])
def test_padded_pass_leaves_rows_of_no_sequence(dev, nsplit):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    lens, cached, total = [20, 0, 33], [5, 0, 0], 70
    q, k, v = _attn_case(dev, torch.bfloat16, 4, 2, 64, lens + [total - 53], cached + [0])
    k, v = k[:3], v[:3]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    plan = pack_prompts(t(lens), t(cached), total=total, max_keys=64, num_q_heads=4, num_kv_heads=2,
                        head_dim=64)
    plan.shape = (*plan.shape[:2], nsplit)
    out = torch.full((total, 4, 64), 3.0, dtype=torch.bfloat16, device=dev)
    prompt_attention(q, k, v, plan, out=out)
    _check_prompt(out[:53], q[:53], k, v, lens, cached)
    assert bool((out[53:] == 3.0).all())


def _poison(x, rows, value):
    x[..., rows, ::3] = value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128), (4, 1, 256)])
def test_unseen_rows_do_not_leak(dev, dtype, value, heads):
    """Not finite values in rows past the end and in rows of later tokens: the earlier
    tokens' outputs are what they are without them, the later ones' carry them."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D = heads
    lens, cached = [100, 30], [3, 40]
    q, k, v = _attn_case(dev, dtype, Hq, Hkv, D, lens, cached, seed=1, cap_more=60)
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D)
    for b, (n, c) in enumerate(zip(lens, cached)):
        _poison(k[b], slice(n + c, None), value)
        _poison(v[b], slice(n + c, None), value)
    clean = prompt_attention(q, k, v, plan)
    _check_prompt(clean, q, k, v, lens, cached)
    _poison(v[0], slice(60, 61), value)    # seen by tokens 57 and later
    _poison(v[1], slice(69, 70), value)    # seen by the last token alone
    got = prompt_attention(q, k, v, plan)
    _check_prompt(got[:57], q[:57], k, v, [57], [3])
    o = got[57:100].float()
    assert bool((~o[:, :, ::3].isfinite()).all()) and bool(o[:, :, 1::3].isfinite().all())
    _check_prompt(got[100:129], q[100:129], k[1:], v[1:], [29], [40])
    assert bool((~got[129, :, ::3].isfinite()).all()) and bool(got[129, :, 1::3].isfinite().all())
    # keys of later tokens: only scores, which are masked
    _poison(v[0], slice(60, 61), 0.5)
    _poison(k[0], slice(60, 61), value)
    got = prompt_attention(q, k, v, plan)
    _check_prompt(got[:57], q[:57], k, v, [57], [3])


def test_extreme_scores(dev):
    """Scores of one huge key, all scores -inf (zeros), and +inf (NaN as softmax has it)."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    q, k, v = _attn_case(dev, torch.bfloat16, 2, 1, 64, [70], [0], seed=2)
    plan = pack_prompts([70], device=dev, num_q_heads=2, num_kv_heads=1, head_dim=64)
    q[:, 0] = q[:, 0].abs() + 0.1
    k[0, 0, 3] = 1e4
    got = prompt_attention(q, k, v, plan)
    _check_prompt(got, q, k, v, [70], [0])
    k[0, 0] = -3e38
    got = prompt_attention(q, k, v, plan)
    assert bool((got[:, 0] == 0).all())
    k[0, 0, 69] = 3e38
    got = prompt_attention(q, k, v, plan)
    assert bool((got[:69, 0] == 0).all()) and bool(got[69, 0].isnan().all())


def test_strided_operands_and_scale(dev):
    """q inside a projection's rows, K/V inside a [T, heads] layout, another scale."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D, lens, cached = 8, 2, 64, [90, 45], [0, 20]
    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).half()
    x = r(sum(lens), (Hq + 4) * D + 16)
    q = x[:, 16:16 + Hq * D].view(-1, Hq, D)
    k, v = r(2, 100, Hkv, D).transpose(1, 2), r(2, Hkv, 100, D + 8)[..., :D]
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D)
    got = prompt_attention(q, k, v, plan, scale=0.3)
    _check_prompt(got, q, k, v, lens, cached, scale=0.3)


def test_one_query_many_keys(dev):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    lens, cached = [1, 3], [70001, 130000]
    q, k, v = _attn_case(dev, torch.bfloat16, 8, 2, 128, lens, cached)
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=8, num_kv_heads=2, head_dim=128)
    assert plan.shape[2] > 1
    _check_prompt(prompt_attention(q, k, v, plan), q, k, v, lens, cached)


def test_cache_past_32_bit_offsets(dev):
    """A sequence whose rows lie past 2^31 elements of the cache."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    Hkv, D, cap = 2, 128, 1 << 22  # 2^30 elements per sequence
    k = torch.empty(3, Hkv, cap, D, dtype=torch.float16, device=dev)
    lens, cached = [0, 0, 30], [0, 0, 50]
    q, ks, vs = _attn_case(dev, torch.float16, 4, Hkv, D, lens, cached)
    k[2, :, :80] = ks[2]
    v = torch.empty_like(k)
    v[2, :, :80] = vs[2]
    plan = pack_prompts(lens, cached, device=dev, num_q_heads=4, num_kv_heads=Hkv, head_dim=D)
    _check_prompt(prompt_attention(q, k, v, plan), q, k, v, lens, cached)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 4, 4, 64, 130, 130), (1, 8, 2, 128, 70, 333),
                                   (3, 7, 1, 128, 2, 2), (1, 4, 2, 256, 65, 65)])
def test_do_sdpa_attn_of_prompts(dev, dtype, shape):
    from laprune_amd.attention import _prompt_kernel_fits, do_sdpa_attn
    B, Hq, Hkv, D, Tq, Tk = shape
    g = torch.Generator(device=dev).manual_seed(Tk)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dtype)
    q, k, v = r(B, Tq, Hq, D).transpose(1, 2), r(B, Hkv, Tk, D), r(B, Hkv, Tk, D)
    assert _prompt_kernel_fits(q, k, v)
    got = do_sdpa_attn(q, k, v, already_rope=True)
    assert got.shape == (B, Tq, Hq * D)
    flat = q.transpose(1, 2).reshape(B * Tq, Hq, D)
    _check_prompt(got.view(B * Tq, Hq, D), flat, k, v, [Tq] * B, [Tk - Tq] * B)
    # a gradient, or a layout of other rows: the library's kernels
    q2 = q.detach().requires_grad_()
    assert not _prompt_kernel_fits(q2, k, v)
    do_sdpa_attn(q2, k, v, already_rope=True).float().sum().backward()
    assert q2.grad is not None
    with torch.autocast("cuda", dtype=torch.float16):
        assert not _prompt_kernel_fits(q, k, v)
    odd = torch.empty(B * Hq * Tq * D + 1, dtype=dtype, device=dev)[1:].view(B, Hq, Tq, D)
    assert not _prompt_kernel_fits(odd, k, v)


def test_captured_and_replayed(dev):
    """One captured pass of tables, append and attention replays on new lengths and
    inputs, the eager results beside it."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    Hq, Hkv, D, total, cap = 8, 2, 64, 96, 200
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    new, old = t([40, 56]), t([0, 0])
    q, k, v, cos, sin, (qw, kw) = _rope_inputs(dev, torch.bfloat16, total, Hq, Hkv, D)
    norms = dict(q_norm=(qw, 1e-6), k_norm=(kw, 1e-6))

    def body(c):
        plan = pack_prompts(new, old, total=total, max_keys=cap, num_q_heads=Hq, num_kv_heads=Hkv,
                            head_dim=D)
        qr = c.rope_append_packed(q, k, v, cos, sin, plan, **norms)
        return qr, prompt_attention(qr, c.k, c.v, plan)

    ca, cb = _cache(dev, torch.bfloat16, 2, Hkv, D, cap), _cache(dev, torch.bfloat16, 2, Hkv, D, cap)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(ca)
    torch.cuda.current_stream().wait_stream(side)
    ca.k.fill_(7.0), ca.v.fill_(9.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body(ca)
    for i, (a, b) in enumerate([([40, 56], [0, 0]), ([1, 95], [40, 56]), ([96, 0], [41, 151])]):
        new.copy_(t(a))
        old.copy_(t(b))
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        want = body(cb)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        assert torch.equal(ca.k, cb.k) and torch.equal(ca.v, cb.v)


def test_two_streams_at_once(dev):
    """Split calls on two streams, each with its own workspace."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    runs = []
    for s in range(2):
        lens, cached = [3, 2], [9000, 4000 + s]
        q, k, v = _attn_case(dev, torch.bfloat16, 8, 2, 128, lens, cached, seed=s)
        plan = pack_prompts(lens, cached, device=dev, num_q_heads=8, num_kv_heads=2, head_dim=128)
        assert plan.shape[2] > 1
        runs.append((q, k, v, plan, prompt_attention(q, k, v, plan)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    outs = [[] for _ in runs]
    for _ in range(5):
        for i, (st, (q, k, v, plan, _)) in enumerate(zip(streams, runs)):
            with torch.cuda.stream(st):
                outs[i].append(prompt_attention(q, k, v, plan))
    torch.cuda.synchronize()
    for i, r in enumerate(runs):
        assert all(torch.equal(o, r[4]) for o in outs[i])


def test_refusals_on_the_gpu(dev):
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    q, k, v = _attn_case(dev, torch.bfloat16, 4, 2, 64, [10], [0])
    plan = pack_prompts([10], device=dev, num_q_heads=4, num_kv_heads=2, head_dim=64)

    def bad(*a, match, **kw):
        with pytest.raises(RuntimeError, match=match):
            prompt_attention(*a, **kw)

    bad(q, k, v, pack_prompts([10], device=dev), match="without head counts")
    bad(q[:9], k, v, plan, match="10 tokens")
    bad(q, k[:, :1], v[:, :1], plan, match="the plan is for")
    bad(q, k[:, :, :9], v[:, :, :9], plan, match="exceed")
    bad(q.float(), k.float(), v.float(), plan, match="fp16/bf16")
    bad(q, k.half(), v.half(), plan, match="dtype")
    bad(q.cpu(), k, v, plan, match="CUDA")
    bad(q.clone().requires_grad_(), k, v, plan, match="gradients")
    bad(q, k, v, plan, scale=0.0, match="scale")
    bad(q, k, v, plan, scale=math.nan, match="scale")
    x = torch.empty(10 * 4 * 64 + 1, dtype=torch.bfloat16, device=dev)[1:].view(10, 4, 64)
    bad(x, k, v, plan, match="aligned")
    with pytest.raises(RuntimeError, match="tile"):
        from laprune_amd._ops import ops
        ops().prompt_attention(q, k, v, plan.tiles, 65, 1, 10, 0.1, torch.empty_like(q))
    c = _cache(dev, torch.bfloat16, 1, 2, 64, 16)
    rq, rk, rv, cos, sin, _ = _rope_inputs(dev, torch.bfloat16, 10, 4, 2, 64)
    with pytest.raises(RuntimeError, match="10 tokens expected"):
        c.rope_append_packed(rq[:, :9], rk, rv, cos, sin, plan)
    with pytest.raises(RuntimeError, match="cache dtype"):
        c.rope_append_packed(rq.half(), rk, rv, cos, sin, plan)
    with pytest.raises(RuntimeError, match="norm weights"):
        c.rope_append_packed(rq, rk, rv, cos, sin, plan, q_norm=(cos[0, 0, :32].contiguous(), 1e-6))
    with pytest.raises(RuntimeError, match="sequences"):
        c.rope_append_packed(rq, rk, rv, cos, sin, pack_prompts([5, 5], device=dev))
    with pytest.raises(RuntimeError, match="cached lengths"):
        c.append_packed(rq, rk, rv, cos, sin, pack_prompts([10], [3], device=dev))


@pytest.mark.parametrize("Hq,Hkv,Tq", [(1, 1, 2), (4, 2, 65), (28, 4, 19), (128, 1, 3)])
def test_batches_past_one_launch_keep_the_library(dev, Hq, Hkv, Tq):
    """A launch takes fewer than 2^24 workgroups (nothing runs here: broadcast views)."""
    from laprune_amd.attention import _prompt_kernel_fits
    most = ((1 << 24) - 1) // (Hkv * -(-Tq // (128 // (Hq // Hkv))))
    q = torch.zeros((1, Hq, Tq, 64), dtype=torch.bfloat16, device=dev)
    k = torch.zeros((1, Hkv, Tq, 64), dtype=torch.bfloat16, device=dev)
    for B, fits in [(most, True), (most + 1, False)]:
        x, y = (t.expand(B, -1, -1, -1) for t in (q, k))
        assert _prompt_kernel_fits(x, y, y) == fits


@pytest.mark.parametrize("D", [64, 256])
def test_a_loose_bound_of_the_keys(dev, D):
    """max_keys may pass the caches, with lengths of either kind; only real keys are checked."""
    from laprune_amd.attention import prompt_attention
    from laprune_amd.packed import pack_prompts
    lens, cached = [40, 0, 7], [30, 9, 3]
    q, k, v = _attn_case(dev, torch.bfloat16, 4, 2, D, lens, cached)
    heads = dict(num_q_heads=4, num_kv_heads=2, head_dim=D)
    for most in (70, 4096, 1 << 29):
        for plan in (pack_prompts(lens, cached, max_keys=most, device=dev, **heads),
                     pack_prompts(*(torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, cached)),
                                  total=47, max_keys=most, **heads)):
            _check_prompt(prompt_attention(q, k, v, plan), q, k, v, lens, cached)
    with pytest.raises(RuntimeError, match="70 keys exceed the 69 rows"):
        prompt_attention(q, k[:, :, :69], v[:, :, :69],
                         pack_prompts(lens, cached, max_keys=4096, device=dev, **heads))
