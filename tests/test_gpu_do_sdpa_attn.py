"""do_sdpa_attn of several queries: who else has a say in its kernel."""
import pytest
import torch
from torch.nn.attention import SDPBackend, sdpa_kernel
from torch.overrides import TorchFunctionMode

pytestmark = pytest.mark.gpu


def _qkv(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    return [torch.randn(1, 4, 70, 64, generator=g, device=dev).bfloat16() for _ in range(3)]


class Watcher(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.seen.append(getattr(func, "__name__", ""))
        return func(*args, **(kwargs or {}))


def test_a_function_mode_sees_the_attention(dev):
    from laprune_amd.attention import _prompt_kernel_fits, do_sdpa_attn
    q, k, v = _qkv(dev)
    plain = do_sdpa_attn(q, k, v, already_rope=True)
    with Watcher() as w:
        got = do_sdpa_attn(q, k, v, already_rope=True)
    assert "scaled_dot_product_attention" in w.seen
    assert (got.float() - plain.float()).abs().max() < 0.02 * plain.float().abs().max()
    with torch.device(dev):
        assert _prompt_kernel_fits(q, k, v)


@pytest.mark.parametrize("backend", [SDPBackend.MATH, SDPBackend.FLASH_ATTENTION,
                                     SDPBackend.EFFICIENT_ATTENTION])
def test_a_chosen_backend_computes_the_prompt(dev, backend):
    """Under sdpa_kernel(...) the library's kernel of that name runs, bit by bit."""
    from laprune_amd.attention import _prompt_kernel_fits, do_sdpa_attn
    q, k, v = _qkv(dev)
    assert _prompt_kernel_fits(q, k, v)
    with sdpa_kernel(backend):
        assert not _prompt_kernel_fits(q, k, v)
        got = do_sdpa_attn(q, k, v, already_rope=True)
        want = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True)
    assert torch.equal(got, want.transpose(1, 2).flatten(2))
    with sdpa_kernel([SDPBackend.MATH, SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
        assert _prompt_kernel_fits(q, k, v)  # a choice of all of them is none
    assert _prompt_kernel_fits(q, k, v)
