"""Which watchers of the calling ops make the framework step back to the model's own (CPU)."""
import torch
from torch.overrides import TorchFunctionMode


class Watcher(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_function_modes_watch():
    from laprune_amd._ops import untraced, unwatched
    with torch.no_grad():
        assert untraced() and unwatched()
        with Watcher():
            assert not untraced() and not unwatched()
            with torch.device("cpu"):
                assert not untraced()
        with torch.device("cpu"):  # says where factories allocate, and watches nothing
            assert untraced() and unwatched()
            with Watcher():
                assert not untraced()
        assert untraced()
