"""Packed prompts, prompts in pieces, shared prefixes and head norms inside a (tiny,
random) Llama model: logits against the unwrapped model's own full-sequence attention.

With ``mask_out = 0`` every candidate is selected, so a LAPrune layer attends to its whole
cache.  Tolerance: 3e-2 of the largest logit, that of tests/test_gpu_llama.py for the same
model in bf16 (two attentions that round differently)."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB = 1000
TOL = 3e-2


def _config(heads=8, kv_heads=2, D=64):
    from transformers import LlamaConfig
    hidden = 512 if 512 % heads == 0 else 64 * heads  # transformers wants heads | hidden
    return LlamaConfig(vocab_size=VOCAB, hidden_size=hidden, intermediate_size=1024,
                       num_hidden_layers=3, num_attention_heads=heads, num_key_value_heads=kv_heads,
                       head_dim=D, max_position_embeddings=4096, rope_theta=10000.0,
                       attn_implementation="sdpa")


def _rel(a, b):
    a, b = a.float(), b.float()
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-6))


def _wrap(model, batch, capacity=512, apply=(1, 2), D=64):
    from laprune_amd.llama import LAPruneLlama, LAPruneSettings
    from laprune_amd.retrieval import RetrievalConfig
    g = torch.Generator().manual_seed(5)
    books = {i: torch.randn(32, 256, D, generator=g) * 0.1 for i in apply}
    s = LAPruneSettings(apply_layers=list(apply),
                        retrieval=RetrievalConfig(mask_out=0.0, sink_size=4, local_window=64))
    return LAPruneLlama(model, books, s, batch=batch, capacity=capacity)


def _pair(dev, batch, seed=1, norms=False, heads=(8, 2), D=64, **kw):
    from laprune_amd.llama import random_model
    ref = random_model(_config(*heads, D), dev, seed=seed)
    if norms:
        _add_norms(ref, D)
    return ref, _wrap(copy.deepcopy(ref), batch, D=D, **kw)


def _add_norms(model, D):
    """Norms of q's and k's heads between projection and rotation, in the model's code."""
    from types import MethodType

    from transformers.models.llama.modeling_llama import LlamaRMSNorm, apply_rotary_pos_emb

    def forward(self, hidden_states, position_embeddings=None, attention_mask=None, **kw):
        B, T, _ = hidden_states.shape
        heads = lambda p: p(hidden_states).view(B, T, -1, self.head_dim)
        q, k = self.q_norm(heads(self.q_proj)), self.k_norm(heads(self.k_proj))
        q, k, v = (x.transpose(1, 2) for x in (q, k, heads(self.v_proj)))
        q, k = apply_rotary_pos_emb(q, k, *position_embeddings)
        o = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
        return self.o_proj(o.transpose(1, 2).reshape(B, T, -1)), None

    g = torch.Generator().manual_seed(11)
    p = next(model.parameters())
    for layer in model.model.layers:
        for name in ("q_norm", "k_norm"):
            n = LlamaRMSNorm(D, eps=1e-6).to(p.device, p.dtype)
            with torch.no_grad():
                n.weight.copy_(1 + 0.5 * torch.randn(D, generator=g))
            setattr(layer.self_attn, name, n)
        layer.self_attn.forward = MethodType(forward, layer.self_attn)


def _want(ref, ids):
    with torch.no_grad():
        return ref(input_ids=ids[None], use_cache=False, logits_to_keep=1).logits[:, -1]


def _ids(dev, n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).to(dev)


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("heads,D", [((8, 2), 64), ((4, 1), 128), ((7, 1), 64)])
def test_packed_prompts_in_pieces_then_steps(dev, norms, heads, D):
    ref, lm = _pair(dev, 4, norms=norms, heads=heads, D=D)
    seqs = [_ids(dev, n, i) for i, n in enumerate((150, 1, 90, 233))]
    got = lm.prefill_packed([seqs[2][:70], seqs[0], seqs[3][:5]], rows=[2, 0, 3])
    for g, s in zip(got, (seqs[2][:70], seqs[0], seqs[3][:5])):
        assert _rel(g, _want(ref, s)[0]) < TOL
    got = lm.prefill_packed([seqs[1], seqs[2][70:71], seqs[3][5:]], rows=[1, 2, 3])
    for g, s in zip(got, (seqs[1], seqs[2][:71], seqs[3])):
        assert _rel(g, _want(ref, s)[0]) < TOL
    assert _rel(lm.prefill_row(2, seqs[2][71:]), _want(ref, seqs[2])) < TOL
    assert lm.lengths == [150, 1, 90, 233]
    assert lm.states[1].cache.encoded_lens == [150, 1, 90, 233]
    more = [_ids(dev, 70, 20 + i) for i in range(4)]
    for i in range(70):  # crosses every sequence's flush
        tok = torch.stack([m[i:i + 1] for m in more])
        step = lm.decode_graph(tok) if i % 3 else lm.decode(tok)
        if i % 9 == 0:
            for b in range(4):
                want = _want(ref, torch.cat((seqs[b], more[b][:i + 1])))
                assert _rel(step[b:b + 1], want) < TOL, (i, b)


@pytest.mark.parametrize("norms", [False, True])
def test_shared_prefix(dev, norms):
    """The prefix runs once; eager and captured steps of the dense layer read it once."""
    ref, lm = _pair(dev, 3, seed=3, norms=norms)
    prefix = _ids(dev, 140, 30)
    own = [_ids(dev, n, 31 + n) for n in (20, 3, 75)]
    assert _rel(lm.prefill_shared(prefix[None]), _want(ref, prefix)) < TOL
    assert lm.lengths == [140] * 3 and lm.shared_prefix == 140
    seqs = [torch.cat((prefix, o)) for o in own]
    for g, s in zip(lm.prefill_packed(own), seqs):
        assert _rel(g, _want(ref, s)[0]) < TOL
    c = lm.states[0].cache
    c.k[1:, :, :140] = float("nan")  # a dense layer: read from sequence 0 alone
    c.v[1:, :, :140] = float("nan")
    more = [_ids(dev, 8, 60 + i) for i in range(3)]
    for i in range(8):
        tok = torch.stack([m[i:i + 1] for m in more])
        step = lm.decode_graph(tok) if i > 3 else lm.decode(tok)
        for b in range(3):
            assert _rel(step[b:b + 1], _want(ref, torch.cat((seqs[b], more[b][:i + 1])))) < TOL
    # a new batch without one: captured again
    lm.reset()
    assert lm.shared_prefix == 0
    for st in lm.states:
        st.cache.k.zero_(), st.cache.v.zero_()
    lm.prefill_packed(own)
    for i in range(2):
        tok = torch.stack([m[i:i + 1] for m in more])
        step = lm.decode_graph(tok)
        for b in range(3):
            assert _rel(step[b:b + 1], _want(ref, torch.cat((own[b], more[b][:i + 1])))) < TOL


def test_a_norm_of_another_class_runs_its_own_code(dev):
    from transformers.models.llama.modeling_llama import LlamaRMSNorm

    class Scaled(LlamaRMSNorm):
        def forward(self, x):
            return 0.5 * super().forward(x)

    ref, _ = _pair(dev, 1, norms=True)
    for layer in ref.model.layers:
        for name in ("q_norm", "k_norm"):
            getattr(layer.self_attn, name).__class__ = Scaled
    lm = _wrap(copy.deepcopy(ref), 1)
    seq = _ids(dev, 120, 4)
    assert _rel(lm.prefill(seq[None, :100]), _want(ref, seq[:100])) < TOL
    for t in range(100, 104):
        step = lm.decode(seq[t:t + 1]) if t < 102 else lm.decode_graph(seq[t:t + 1])
        assert _rel(step, _want(ref, seq[:t + 1])) < TOL


def test_refusals(dev):
    _, lm = _pair(dev, 2, capacity=64)
    ids = _ids(dev, 80, 1)
    for call, match in [(lambda: lm.prefill_packed([ids[:0]]), "at least one token"),
                        (lambda: lm.prefill_packed([]), "at least one token"),
                        (lambda: lm.prefill_packed([ids[:3]] * 2, rows=[0, 0]), "of its own"),
                        (lambda: lm.prefill_packed([ids[:3]] * 3), "out of range"),
                        (lambda: lm.prefill_packed([ids[:3], ids[:65]]), "capacity"),
                        (lambda: lm.prefill_shared(ids[None, :65]), "capacity")]:
        with pytest.raises(RuntimeError, match=match):
            call()
        assert lm.lengths == [0, 0]
    lm.prefill_packed([ids[:60], ids[:5]])
    with pytest.raises(RuntimeError, match="capacity"):
        lm.prefill_row(0, ids[:5])
    with pytest.raises(RuntimeError, match="empty caches"):
        lm.prefill_shared(ids[None, :3])
    lm.prefill_row(1, ids[:5])
    assert lm.lengths == [60, 10]


def test_one_token_prompt_without_the_packed_kernels(dev):
    """Alone it is no decode step of the batch, with head norms as without."""
    for norms in (False, True):
        _, lm = _pair(dev, 1, norms=norms)
        lm._packs = lambda: False
        with pytest.raises(RuntimeError, match="whole batch"):
            lm.prefill_row(0, _ids(dev, 1, 1)[None])
        assert lm.lengths == [0] and lm._row is None
