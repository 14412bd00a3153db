"""Prompts of a wrapped model whose forms the packed tests leave out, against the unwrapped
model (models, tolerance and helpers of test_gpu_packed_llama)."""
import pytest
import torch

from test_gpu_packed_llama import TOL, _ids, _pair, _rel, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_prompts_of_one_and_two_tokens(dev, norms, graph):
    """A batch of one-token prompts is a step of the whole batch; generate() of two-token
    prompts prefills one such token each."""
    B = 3
    ref, lm = _pair(dev, B, seed=7, norms=norms)
    ids = torch.stack([_ids(dev, 4, 40 + b) for b in range(B)])
    got = lm.prefill(ids[:, :1])
    assert lm.lengths == [1] * B
    for t in range(1, 5):
        for b in range(B):
            assert _rel(got[b:b + 1], _want(ref, ids[b, :t])) < TOL, (t, b)
        if t < 4:
            step = lm.decode_graph if graph else lm.decode
            got = step(ids[:, t:t + 1])
    out = lm.generate(ids[:, :2], 3, graph=graph)
    assert out.shape == (B, 5) and torch.equal(out[:, :2], ids[:, :2])
    for b in range(B):
        for t in range(2, 5):  # a token that the reference's logits put first, up to their tolerance
            want = _want(ref, out[b, :t])[0].float()
            assert want[out[b, t]] >= want.max() - 2 * TOL * want.abs().max()


def _qwen3(dev, D, heads, kv_heads):
    from transformers import Qwen3Config, Qwen3ForCausalLM
    torch.manual_seed(2)
    config = Qwen3Config(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
                         num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=D,
                         max_position_embeddings=4096, attn_implementation="sdpa")
    with torch.device(dev):
        model = Qwen3ForCausalLM(config).to(torch.bfloat16).eval()
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for layer in model.model.layers:
            for name in ("q_norm", "k_norm"):
                w = getattr(layer.self_attn, name).weight
                w.copy_(1 + 0.5 * torch.randn(D, generator=g))
    return model


@pytest.mark.parametrize("D,heads,kv_heads", [(64, 8, 2), (128, 4, 4)])
def test_a_stock_model_with_head_norms(dev, monkeypatch, D, heads, kv_heads):
    """Its norms run in the append's launch: packed prompts, eager and captured steps."""
    import copy

    from test_gpu_packed_llama import _wrap

    from laprune_amd.cache import DecodeKVCache
    ref = _qwen3(dev, D, heads, kv_heads)
    lm = _wrap(copy.deepcopy(ref), 2, D=D)
    fused, plain = [], DecodeKVCache._qk_rope

    def count(self, q, k, v, cos, sin, seq, pos, q_norm, k_norm, q_out):
        fused.append(q_norm is not None and k_norm is not None)
        return plain(self, q, k, v, cos, sin, seq, pos, q_norm, k_norm, q_out)

    monkeypatch.setattr(DecodeKVCache, "_qk_rope", count)
    seqs = [_ids(dev, n, n) for n in (90, 33)]
    got = lm.prefill_packed([seqs[0][:70], seqs[1]])
    for g, s in zip(got, (seqs[0][:70], seqs[1])):
        assert _rel(g, _want(ref, s)[0]) < TOL
    assert _rel(lm.prefill_row(0, seqs[0][70:]), _want(ref, seqs[0])) < TOL
    assert fused == [True] * 6
    more = [_ids(dev, 6, 50 + b) for b in range(2)]
    for i in range(6):
        step = (lm.decode if i < 3 else lm.decode_graph)(torch.stack([m[i:i + 1] for m in more]))
        for b in range(2):
            assert _rel(step[b:b + 1], _want(ref, torch.cat((seqs[b], more[b][:i + 1])))) < TOL
    assert len(fused) > 6 and all(fused)
    # a hook on a norm, or a forward of its own, is not passed by
    calls = []
    lm.layers[1].self_attn.q_norm.register_forward_hook(lambda *a: calls.append(1))
    step = lm.decode(torch.stack([m[:1] for m in more]))
    assert calls == [1] and fused[-3:] == [True, False, True]
