"""Packed copies of a model's weights follow optimizers that leave `Tensor._version` as it was (host half; the device half is test_gpu_packed_weights.py)."""
import pytest
import torch

from geneface_amd import fused


class _State:      # what the hook looks at of a FusedState
    def __init__(self, watch):
        self._watch = watch


@pytest.mark.parametrize("cls", [torch.optim.Adam, torch.optim.AdamW, torch.optim.SGD])
def test_a_fused_step_raises_the_version_of_what_is_watched(cls):
    ours, still, other = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    state = _State([ours, still])
    fused._live.add(state)
    opt = cls([ours, still, other], lr=0.1, fused=True)
    for _ in range(2):
        ours.grad, still.grad, other.grad = torch.ones(3), None, torch.ones(3)
        before = [p._version for p in (ours, still, other)]
        opt.step()
        assert ours._version > before[0] and still._version == before[1] and other._version == before[2]
    assert bool((ours != 0).all())


def test_other_optimizers_are_left_alone():
    p = torch.nn.Parameter(torch.zeros(3))
    state = _State([p])
    fused._live.add(state)
    p.grad = torch.ones(3)
    before = p._version
    torch.optim.SGD([p], lr=0.1).step()
    assert p._version == before + 1


def test_a_state_that_is_gone_is_forgotten():
    p = torch.nn.Parameter(torch.zeros(3))
    state = _State([p])
    fused._live.add(state)
    del state
    assert all(p is not t for st in fused._live for t in st._watch)
