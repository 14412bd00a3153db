"""Operators of packed prompts and of decode over a shared prefix: inputs, plain
forms, the calls of this package, and the work that each cannot do without.

Kinds of case (``case["kind"]``):
  plan    request lengths to each packed token's sequence and cache position
  rope    norms of queries and keys per head and the rotation in one pass, keys and
          values into the cache; a prompt's packed tokens or one token per sequence
  prompt  causal attention of packed prompts over the cache, grouped heads
  shared  one query token per sequence over a cache whose first tokens are the same
          in every sequence
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ------------------------------------------------------------------ the cases

def _plan(B, total, cached):
    return dict(kind="plan", B=B, total=total, cached=cached)


def _rope(form, B, Hq, Hkv, D, total, cached, dtype):
    return dict(kind="rope", form=form, B=B, Hq=Hq, Hkv=Hkv, D=D, total=total, cached=cached,
                dtype=dtype)


def _prompt(B, Hq, Hkv, D, total, cached, dtype):
    return dict(kind="prompt", B=B, Hq=Hq, Hkv=Hkv, D=D, total=total, cached=cached, dtype=dtype)


def _shared(B, Hq, Hkv, D, prefix, suffix, dtype):
    return dict(kind="shared", B=B, Hq=Hq, Hkv=Hkv, D=D, prefix=prefix, suffix=suffix,
                dtype=dtype)


def listed():
    return [
        # a few users' turns behind their cached conversations: launch latency counts
        dict(_plan(6, 517, 4000), name="plan_turns"),
        # an offline batch's prompts packed into one pass
        dict(_plan(256, 131072, 0), name="plan_batch"),
        # one decode step of a served batch
        dict(_rope("step", 16, 32, 8, 128, 16, 4096, "bf16"), name="rope_step_b16"),
        # short prompts of a small model, an odd number of tokens
        dict(_rope("prompt", 7, 8, 2, 64, 2051, 0, "fp16"), name="rope_2k_d64"),
        # one layer of a long prefill
        dict(_rope("prompt", 2, 32, 8, 128, 32768, 0, "bf16"), name="rope_32k"),
        # short prompts of a small model: latency counts
        dict(_prompt(7, 8, 2, 64, 777, 0, "fp16"), name="prompt_short_d64"),
        # unequal prompts of a served batch in one pass
        dict(_prompt(8, 32, 8, 128, 16384, 0, "bf16"), name="prompt_batch_16k"),
        # one long prompt
        dict(_prompt(1, 32, 8, 128, 16384, 0, "bf16"), name="prompt_one_16k"),
        # a turn of a long conversation: few queries behind 65001 cached tokens, seven
        # query heads per KV head
        dict(_prompt(1, 28, 4, 128, 300, 65001, "fp16"), name="prompt_turn_65k_g7"),
        # a small model's batch behind a system prompt
        dict(_shared(4, 8, 2, 64, 2000, 200, "bf16"), name="shared_b4_2k_d64"),
        # a batch of questions on one long document
        dict(_shared(16, 32, 8, 128, 16384, 1024, "bf16"), name="shared_b16_16k"),
        # many samples of one prompt, seven query heads per KV head
        dict(_shared(48, 28, 4, 128, 8193, 512, "fp16"), name="shared_b48_8k_g7"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _geometry(rng):
    while True:
        D, Hkv, G = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.randint(1, 8)
        if Hkv * G * D <= 8192:
            return Hkv * G, Hkv, D


def draw(rng):
    kind = rng.choice(["plan", "rope", "prompt", "prompt", "shared", "shared"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "plan":
        B = _log(rng, 1, 600)
        return _plan(B, max(B, _log(rng, 16, 131072)), rng.choice([0, _log(rng, 1, 100000)]))
    Hq, Hkv, D = _geometry(rng)
    if kind == "rope":
        if rng.random() < 0.4:
            B = _log(rng, 1, 64)
            return _rope("step", B, Hq, Hkv, D, B, _log(rng, 1, 4096), dtype)
        B = _log(rng, 1, 32)
        return _rope("prompt", B, Hq, Hkv, D, max(B, _log(rng, 64, 32768 * 5120 // (Hq + Hkv) // D // 2)),
                     rng.choice([0, _log(rng, 1, 2000)]), dtype)
    if kind == "prompt":
        while True:
            B = _log(rng, 1, 16)
            c = _prompt(B, Hq, Hkv, D, max(B, _log(rng, 64, 16384)),
                        rng.choice([0, 0, _log(rng, 1, 65000)]), dtype)
            new, cached = _lengths(c)
            grid = B * Hq * max(new) * max(n + t for n, t in zip(new, cached))
            if grid <= 1 << 33 and work(c)["flops"] <= work(listed()[7])["flops"]:
                return c
    while True:
        c = _shared(_log(rng, 1, 64), Hq, Hkv, D, _log(rng, 64, 32768), _log(rng, 1, 2048), dtype)
        if c["B"] * Hkv * D * (c["prefix"] + c["suffix"]) <= 1 << 29 and \
                work(c)["flops"] <= 1 << 38:
            return c


def _split(rng, B, total):
    """total tokens over B sequences of unequal lengths, one of them empty when there
    are more than four."""
    w = [rng.uniform(0.1, 1.9) for _ in range(B)]
    if B > 4:
        w[1] = 0.0
    cut = [round(total * sum(w[:b]) / sum(w)) for b in range(B)] + [total]
    return [cut[b + 1] - cut[b] for b in range(B)]


def _lengths(c, seed=0):
    """New and cached tokens of each sequence: of the case, for a plan of the seed too."""
    rng = random.Random(f"{c['B']} {c.get('total')} {c.get('cached')} {seed}")
    B = c["B"]
    if c["kind"] == "shared":
        return [1] * B, [c["prefix"] + rng.randint(0, c["suffix"]) - 1 for _ in range(B)]
    new = [1] * B if c.get("form") == "step" else _split(rng, B, c["total"])
    return new, [rng.randint(c["cached"] // 2, c["cached"]) for _ in range(B)]


def work(case):
    c = case
    if c["kind"] == "plan":
        return {"bytes": 12 * c["total"] + 12 * c["B"] + 4, "flops": 2 * c["total"]}
    Hq, Hkv, D, B = c["Hq"], c["Hkv"], c["D"], c["B"]
    new, cached = _lengths(c)
    if c["kind"] == "rope":
        n = c["total"]
        return {"bytes": 2 * n * D * (2 * (Hq + 2 * Hkv) + 2), "flops": 8 * n * (Hq + Hkv) * D}
    if c["kind"] == "prompt":
        pairs = sum(n * t + n * (n + 1) // 2 for n, t in zip(new, cached))
        keys = sum(n + t for n, t in zip(new, cached) if n)
        return {"bytes": 4 * D * (Hq * c["total"] + Hkv * keys), "flops": 4 * D * Hq * pairs}
    keys = [t + 1 for t in cached]
    once = c["prefix"] + sum(k - c["prefix"] for k in keys)
    return {"bytes": 4 * D * (Hq * B + Hkv * once), "flops": 4 * D * Hq * sum(keys)}


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    c = case
    s = dict(case=c)
    new, cached = _lengths(c, seed if c["kind"] == "plan" else 0)
    s["new"], s["cached"] = new, cached
    ints = dict(dtype=torch.int32, device="cuda")
    s["new_dev"], s["cached_dev"] = torch.tensor(new, **ints), torch.tensor(cached, **ints)
    if c["kind"] == "plan":
        return s
    dt = DTYPES[c["dtype"]]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    cap = max(n + t for n, t in zip(new, cached))
    s["k"], s["v"] = randn(B, Hkv, cap, D), randn(B, Hkv, cap, D)
    if c["kind"] == "shared":
        P = c["prefix"]
        s["k"][1:, :, :P], s["v"][1:, :, :P] = s["k"][:1, :, :P], s["v"][:1, :, :P]
        s["q"] = randn(B, Hq, 1, D, scale=1.5)
        return s
    n = c["total"]
    starts = [sum(new[:b]) for b in range(B)]
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    s["seq"] = seq.cuda()
    s["local"] = (torch.arange(n) - torch.tensor(starts)[seq]).cuda()
    s["pos"] = s["local"] + torch.tensor(cached).cuda()[s["seq"]]
    if c["kind"] == "prompt":
        s["q"] = randn(n, Hq, D, scale=1.5)
        return s
    # a projection's output holds q, k and v of a token side by side; keys have
    # channels of very different size before their norm
    x = randn(1, n, (Hq + 2 * Hkv) * D)
    x *= (torch.rand((Hq + 2 * Hkv) * D, generator=g, device="cuda") * 4 + 0.1).to(dt)
    s["qkv"] = x.split([Hq * D, Hkv * D, Hkv * D], dim=-1)
    s["q_w"], s["k_w"] = (1 + randn(D, scale=0.2).float()).to(dt), (1 + randn(D, scale=0.2).float()).to(dt)
    f = 500000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    a = s["pos"].double()[:, None] * f
    a = torch.cat((a, a), -1)[None]
    s["cos"], s["sin"] = a.cos().to(dt), a.sin().to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] != "plan":
        c = case
        from laprune_amd.cache import DecodeKVCache
        from laprune_amd.packed import pack_prompts
        from laprune_amd.retrieval import DenseDecoder
        heads = dict(num_q_heads=c["Hq"], num_kv_heads=c["Hkv"], head_dim=c["D"])
        if c["kind"] == "shared":
            s["dec"] = DenseDecoder(c["B"], c["Hq"], c["Hkv"], c["D"], s["k"].shape[2],
                                    s["k"].device, s["k"].dtype)
        elif c.get("form") != "step":
            s["plan"] = pack_prompts(s["new"], s["cached"], device="cuda", **heads)
        if c["kind"] == "rope":
            s["cache"] = DecodeKVCache(None, c["B"], c["Hkv"], c["D"], s["k"].shape[2],
                                       dtype=s["k"].dtype, device="cuda")
            s["cache"].k, s["cache"].v = s["k"], s["v"]
            s["q_out"] = torch.empty(c["total"], c["Hq"], c["D"], dtype=s["k"].dtype, device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "plan":
        if own:
            from laprune_amd.packed import pack_prompts
            p = pack_prompts(s["new_dev"], s["cached_dev"], total=c["total"],
                             max_keys=c["total"] + c["cached"])
            return p.starts, p.seq, p.pos
        return _plain_plan(s["new_dev"], s["cached_dev"], c["total"])
    if kind == "rope":
        if own:
            q, k, v = s["qkv"]
            norms = dict(q_norm=(s["q_w"], EPS), k_norm=(s["k_w"], EPS))
            if c["form"] == "step":
                d = c["D"]
                s["cache"].rope_append(q.view(-1, 1, c["Hq"] * d), k.view(-1, 1, c["Hkv"] * d),
                                       v.view(-1, 1, c["Hkv"] * d), s["cos"].view(-1, 1, d),
                                       s["sin"].view(-1, 1, d), s["pos"][:, None], s["q_out"],
                                       **norms)
            else:
                s["cache"].rope_append_packed(q, k, v, s["cos"], s["sin"], s["plan"], s["q_out"],
                                              **norms)
            return s["q_out"], s["cache"].k, s["cache"].v
        return _plain_rope(s)
    if kind == "prompt":
        if own:
            from laprune_amd.attention import prompt_attention
            return prompt_attention(s["q"], s["k"], s["v"], s["plan"])
        return _plain_prompt(s)
    if own:
        return s["dec"].step(s["q"], s["k"], s["v"], lengths=[t + 1 for t in s["cached"]],
                             shared_prefix=c["prefix"])
    return _plain_shared(s)


def _plain_plan(new, cached, total):
    starts = torch.zeros(new.numel() + 1, dtype=torch.int32, device=new.device)
    starts[1:] = torch.cumsum(new, 0)
    seq = torch.repeat_interleave(torch.arange(new.numel(), dtype=torch.int32, device=new.device),
                                  new, output_size=total)
    pos = torch.arange(total, device=new.device) + (cached - starts[:-1])[seq]
    return starts, seq, pos


def _plain_rope(s):
    c = s["case"]
    D, n = c["D"], c["total"]
    cos, sin = s["cos"].view(n, 1, D).float(), s["sin"].view(n, 1, D).float()

    def turn(x, w):
        x = x.reshape(n, -1, D).float()
        x = w.float() * (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS))
        half = torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1)
        return (x * cos + half * sin).to(s["k"].dtype)

    q, k, v = s["qkv"]
    s["k"][s["seq"], :, s["pos"]] = turn(k, s["k_w"])
    s["v"][s["seq"], :, s["pos"]] = v.reshape(n, -1, D)
    return turn(q, s["q_w"]), s["k"], s["v"]


def _plain_prompt(s):
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    q = torch.zeros(B, max(s["new"]), Hq, D, device="cuda")
    q[s["seq"], s["local"]] = s["q"].float() * (1.0 / math.sqrt(D))
    q = q.transpose(1, 2).unflatten(1, (Hkv, Hq // Hkv))
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    x = q @ k.transpose(-1, -2)
    t = torch.arange(k.shape[3], device="cuda")
    last = torch.arange(max(s["new"]), device="cuda") + s["cached_dev"][:, None]
    x.masked_fill_((t > last[..., None])[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    o = (x @ v) / x.sum(-1, keepdim=True)
    return o.flatten(1, 2)[s["seq"], :, s["local"]].to(s["q"].dtype)


def _plain_shared(s):
    c = s["case"]
    B, Hq, Hkv, D, P = c["B"], c["Hq"], c["Hkv"], c["D"], c["prefix"]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D) * (1.0 / math.sqrt(D))
    k, v = s["k"].float(), s["v"].float()
    shared = q.transpose(0, 1).flatten(1, 2) @ k[0, :, :P].transpose(1, 2)
    shared = shared.view(Hkv, B, -1, P).transpose(0, 1)
    own_part = q @ k[:, :, P:].transpose(2, 3)
    t = torch.arange(P, k.shape[2], device="cuda")
    own_part.masked_fill_((t > s["cached_dev"][:, None])[:, None, None], -math.inf)
    x = torch.cat((shared, own_part), -1)
    x = (x - x.amax(-1, keepdim=True)).exp()
    o = x[..., P:] @ v[:, :, P:]
    o += (x[..., :P].transpose(0, 1).flatten(1, 2) @ v[0, :, :P]).view(Hkv, B, -1, D).transpose(0, 1)
    return (o / x.sum(-1, keepdim=True)).view(B, Hq, 1, D).to(s["q"].dtype)


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    c = case
    s = _inputs(case, seed)
    if c["kind"] == "plan":  # whole numbers: counted one token at a time
        starts, rows = [0], []
        for b, (n, t) in enumerate(zip(s["new"], s["cached"])):
            rows += [(b, t + i) for i in range(n)]
            starts.append(len(rows))
        seq, pos = zip(*rows)
        return (torch.tensor(starts, dtype=torch.int32), torch.tensor(seq, dtype=torch.int32),
                torch.tensor(pos))
    D, G = c["D"], c["Hq"] // c["Hkv"]
    if c["kind"] == "rope":
        def norm_and_turn(x, w):
            x = x[0].double().unflatten(-1, (-1, D))
            x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            a, b = x[..., :D // 2], x[..., D // 2:]
            co, si = s["cos"][0, :, None].double(), s["sin"][0, :, None].double()
            return torch.cat((a * co[..., :D // 2] - b * si[..., :D // 2],
                              b * co[..., D // 2:] + a * si[..., D // 2:]), -1)
        q, k, v = s["qkv"]
        keys, vals = s["k"].double(), s["v"].double()
        keys[s["seq"], :, s["pos"]] = norm_and_turn(k, s["k_w"])
        vals[s["seq"], :, s["pos"]] = v[0].double().unflatten(-1, (-1, D))
        return norm_and_turn(q, s["q_w"]), keys, vals
    shared = c["kind"] == "shared"
    q = s["q"][:, :, 0] if shared else s["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    i = 0
    for b, (n, t) in enumerate(zip(s["new"], s["cached"])):
        for h in range(c["Hq"]):
            keys, vals = s["k"][b, h // G, :t + n].double(), s["v"][b, h // G, :t + n].double()
            score = q[i:i + n, h].double() @ keys.T / math.sqrt(D)
            score += torch.full_like(score, -math.inf).triu(t + 1)
            out[i:i + n, h] = score.softmax(-1) @ vals
        i += n
    return out[:, :, None] if shared else out
