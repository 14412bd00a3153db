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
