"""How a wrapped model's prompts are put into passes (CPU: the attention layers and the tables
are stand-ins that record what they get)."""
import types

import pytest
import torch

VOCAB = 40


def _lm(monkeypatch, cls="Llama", batch=2, own=None, **kw):
    """A LAPruneLlama of a tiny model without kernels; lm.calls: per pass the mask that the
    layer got and the positions, lm.out: hidden states that the layers leave as they are."""
    import transformers

    from laprune_amd import llama
    config = getattr(transformers, cls + "Config")(
        vocab_size=VOCAB, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
        num_attention_heads=1, num_key_value_heads=1, head_dim=64, attn_implementation="sdpa", **kw)
    torch.manual_seed(0)
    model = getattr(transformers, cls + "ForCausalLM")(config).bfloat16().eval()
    if own is not None:
        model.model.__class__ = own(type(model.model))
    lm = llama.LAPruneLlama(model, {}, llama.LAPruneSettings(), batch=batch, capacity=256)
    lm.calls = []

    def attention(hidden_states, position_embeddings=None, attention_mask=None, position_ids=None, **kw):
        lm.calls.append((attention_mask, lm._plan, position_embeddings))
        c = lm.states[0].cache
        if lm._plan is not None:
            c.lengths = [a + b for a, b in zip(c.lengths, lm._plan.lens)]
        else:
            c.lengths = [n + hidden_states.shape[1] for n in c.lengths]
        return hidden_states, None

    model.model.layers[0].self_attn.forward = attention

    def tables(lens, cached, **kw):
        pos = torch.tensor([c + i for n, c in zip(lens, cached) for i in range(n)])
        return types.SimpleNamespace(lens=list(lens), cached=list(cached), pos=pos)

    monkeypatch.setattr(llama, "pack_prompts", tables)
    return lm


def _ids(n, seed=0):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed))


def _small(mask):
    return mask is None or mask.numel() <= 4


@pytest.mark.parametrize("cls", ["Llama", "Qwen3"])
def test_a_packed_pass_builds_no_mask_of_its_length_squared(monkeypatch, cls):
    """Positions that start anew look like packed sequences to the model's code, which would
    build a mask of the whole pass."""
    lm = _lm(monkeypatch, cls)
    lm.prefill(torch.stack([_ids(25, 1), _ids(25, 2)]))
    assert len(lm.calls) == 1 and lm.calls[0][1] is not None and _small(lm.calls[0][0])
    lm.prefill_packed([_ids(30, 3), _ids(20, 4)])
    assert len(lm.calls) == 2 and _small(lm.calls[1][0])
    lm.prefill_row(1, _ids(9)[None])
    assert len(lm.calls) == 3 and _small(lm.calls[2][0])


def test_a_model_that_makes_its_masks_itself(monkeypatch):
    """No mask is handed to it, so sequences are not packed: a batch of one length runs as it
    came, other prompts one at a time."""
    def own(base):
        class Other(base):
            def forward(self, *a, attention_mask=None, **kw):
                assert attention_mask is None  # it would not know a 1 x 1 one
                return super().forward(*a, attention_mask=None, **kw)
        return Other

    lm = _lm(monkeypatch, own=own)
    got = lm.prefill(torch.stack([_ids(25, 1), _ids(25, 2)]))
    assert got.shape == (2, VOCAB) and lm.calls[0][1] is None and _small(lm.calls[0][0])
    one = lm.prefill_packed([_ids(30, 3), _ids(20, 4)])
    assert one.shape == (2, VOCAB) and [c[1].lens for c in lm.calls[1:]] == [[30, 0], [0, 20]]
    assert all(_small(c[0]) for c in lm.calls) and lm.lengths == [55, 45]


ROPES = [dict(rope_type="dynamic", factor=4.0),
         dict(rope_type="longrope", factor=4.0, original_max_position_embeddings=64,
              short_factor=[1.0] * 32, long_factor=[1.0 + i for i in range(32)])]


@pytest.mark.parametrize("rope", ROPES, ids=lambda r: r["rope_type"])
@pytest.mark.parametrize("lens", [(20, 150), (150, 20), (20, 20)])
def test_rotary_tables_that_go_by_the_length(monkeypatch, rope, lens):
    """Each prompt is rotated as it would be alone; those of one length still share a pass."""
    kw = dict(max_position_embeddings=64 if rope["rope_type"] == "dynamic" else 256, rope_scaling=dict(rope))
    prompts = [_ids(n, n) for n in lens]
    alone, packed = _lm(monkeypatch, **kw), _lm(monkeypatch, **kw)
    for b, p in enumerate(prompts):
        alone.prefill_row(b, p)
    packed.prefill_packed(prompts)
    assert len(packed.calls) == (1 if lens[0] == lens[1] else 2)
    for i in range(2):
        a, b = (torch.cat([c[2][i] for c in lm.calls], 1) for lm in (alone, packed))
        assert torch.equal(a, b)


def test_a_prompt_is_one_row_of_ids(monkeypatch):
    """Rows of several are not run together as one prompt."""
    lm = _lm(monkeypatch)
    two = _ids(6).view(2, 3)
    for call in (lambda: lm.prefill_packed([two]), lambda: lm.prefill_row(0, two),
                 lambda: lm.prefill_shared(two), lambda: lm.prefill_packed([_ids(3), two[None]]),
                 lambda: lm.prefill_packed([two[0, 0]])):
        with pytest.raises(RuntimeError, match=r"ids \[T\] or \[1, T\]"):
            call()
    assert lm.lengths == [0, 0] and not lm.calls
    lm.prefill_packed([two[0], two[1:]])
    assert lm.lengths == [3, 3]


def test_batches_past_the_packed_tables_run_as_they_came(monkeypatch):
    """The tables of a pass hold 4096 sequences."""
    lm = _lm(monkeypatch)
    assert lm._packs()
    lm.B = 4096
    assert lm._packs()
    lm.B = 4097
    for st in lm.states:
        st.cache.lengths = [0] * 4097
    lm.prefill(_ids(2 * 4097).view(4097, 2))
    assert len(lm.calls) == 1 and lm.calls[0][1] is None and lm.lengths == [2] * 4097
    with pytest.raises(RuntimeError, match="4096 sequences"):
        lm.prefill_packed([_ids(3)])


@pytest.mark.parametrize("known", [True, False])
def test_a_wrapped_forward_of_the_model(monkeypatch, known):
    """One that says what it wraps still hands masks through; any other replacement does not."""
    import functools
    from laprune_amd.llama import _hands_masks_through
    lm = _lm(monkeypatch)
    inner = lm.model.model.forward

    def outer(*a, **kw):
        return inner(*a, **kw)

    lm.model.model.forward = functools.update_wrapper(functools.partial(outer), inner) if known else outer
    assert _hands_masks_through(lm.model) == known
