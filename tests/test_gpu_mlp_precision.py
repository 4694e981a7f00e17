"""GPU: a model's MLPs in 8 bits are computed in 8 bits whichever way the model is called, and beside the native ones within what 8 bits round."""
import copy

import pytest
import torch

from helpers import frame_inputs, model_fixture, sequence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(torso=False):
    from geneface_amd.radnerf import RADNeRF
    from geneface_amd.radnerf_torso import RADNeRFTorso
    hp, sd = model_fixture(torso)
    model = (RADNeRFTorso if torso else RADNeRF)(hp)
    model.load_state_dict(sd, strict=True)
    return hp, model.to(DEV)


def _points(n):
    g = torch.Generator().manual_seed(1)
    return ((torch.rand(n, 3, generator=g) * 2 - 1).to(DEV), torch.nn.functional.normalize(torch.randn(n, 3, generator=g), dim=-1).to(DEV),
            torch.randn(1, 64, generator=g).to(DEV))


@pytest.mark.parametrize("grad", [True, False])
def test_field_of_a_default_model_goes_by_it(grad):
    _, model = _model()
    pos, dirs, cond = _points(600)

    def run(m):
        with torch.set_grad_enabled(grad):
            return [t.detach() for t in m(pos, dirs, cond, m.individual_embeddings[0])]
    native = run(model)
    for m in (model.ambient_net, model.sigma_net, model.color_net):
        m.precision = "fp8"
    ours = run(model)
    pinned = copy.deepcopy(model)
    pinned.field_impl = pinned.render_impl = "ops"
    assert all(torch.equal(a, b) for a, b in zip(ours, run(pinned))) and not torch.equal(ours[1], native[1])
    for m in (model.ambient_net, model.sigma_net, model.color_net):
        m.precision = "native"
    assert all(torch.equal(a, b) for a, b in zip(run(model), native))


@pytest.mark.parametrize("torso", [False, True])
def test_rendering_goes_by_it_or_refuses(torso):
    hp, model = _model(torso)
    model.eval()
    fi = frame_inputs(sequence(4, 24, 24), 1)
    to = lambda t: t.to(DEV)      # noqa: E731
    args = tuple(to(fi[k]) for k in ("rays_o", "rays_d", "cond", "bg_coords", "pose6"))
    run = lambda impl: model.render(*args, index=0, staged=False, bg_color=to(fi["bg"]), perturb=False, force_all_rays=True, render_impl=impl, **hp)["rgb_map"]      # noqa: E731
    with torch.no_grad():
        native = run("auto")
        model.sigma_net.precision = "fp8"
        assert torch.equal(run("auto"), run("ops")) and not torch.equal(run("auto"), native)
        with pytest.raises(NotImplementedError, match="precision"):
            run("fused")

