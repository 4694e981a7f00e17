"""GPU: the fused training field computes with the weights of the last optimizer step, whatever kind of optimizer took it."""
import copy

import pytest
import torch

from helpers import model_fixture

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

OPTIMIZERS = {"adam": lambda p: torch.optim.Adam(p, lr=1e-2), "adam-fused": lambda p: torch.optim.Adam(p, lr=1e-2, fused=True),
              "adamw-fused": lambda p: torch.optim.AdamW(p, lr=1e-2, fused=True)}


def _optimizer(name, params):
    if name == "library":
        from geneface_amd.optim import AdamW
        return AdamW(params, lr=1e-2)
    return OPTIMIZERS[name](params)


@pytest.mark.parametrize("amp", [False, True])
@pytest.mark.parametrize("name", [*OPTIMIZERS, "library"])
def test_head_field_follows_every_step(name, amp):
    """The field's outputs after a step are, bit for bit, those of a copy of the model that has packed nothing yet."""
    from geneface_amd.radnerf import RADNeRF
    hp, sd = model_fixture(False)
    model = RADNeRF(hp)
    model.load_state_dict(sd, strict=True)
    model = model.to(DEV).train()
    g = torch.Generator().manual_seed(1)
    pos, dirs = (torch.rand(700, 3, generator=g) * 2 - 1).to(DEV), torch.nn.functional.normalize(torch.randn(700, 3, generator=g), dim=-1).to(DEV)
    cond = torch.randn(1, 64, generator=g).to(DEV)
    opt = _optimizer(name, list(model.parameters()))

    def run(m):
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.float16, enabled=amp):
            sigma, rgb, amb = m(pos, dirs, cond, m.individual_embeddings[0])
        (sigma.clamp(max=50).mean() + rgb.square().mean() + amb.mean()).backward()
        return sigma.detach(), rgb.detach(), amb.detach()
    last = None
    for step in range(3):
        ours = run(model)
        theirs = run(copy.deepcopy(model))
        assert all(torch.equal(a, b) for a, b in zip(ours, theirs)), (name, step)
        assert last is None or not torch.equal(last, ours[1])
        last = ours[1]
        opt.step()


@pytest.mark.parametrize("name", ["adam-fused", "library"])
def test_torso_field_follows_every_step(name):
    from geneface_amd.radnerf_torso import RADNeRFTorso
    hp, sd = model_fixture(True)
    model = RADNeRFTorso(hp)
    model.load_state_dict(sd, strict=True)
    model = model.to(DEV).train()
    g = torch.Generator().manual_seed(2)
    x, pose = (torch.rand(500, 2, generator=g) * 2 - 1).to(DEV), torch.randn(1, 6, generator=g).to(DEV) * 0.1
    opt = _optimizer(name, [p for n, p in model.named_parameters() if "torso" in n])

    def run(m):
        m.zero_grad(set_to_none=True)
        assert m._fused_torso_train_ok(x, m.torso_individual_codes[0], None)
        a, c, dx = m.forward_torso(x, pose, m.torso_individual_codes[0])
        (a.mean() + c.square().mean() + dx.square().mean()).backward()
        return a.detach(), c.detach(), dx.detach()
    for step in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(model), run(copy.deepcopy(model)))), (name, step)
        opt.step()


@pytest.mark.parametrize("which", ["torso", "head", "code", "both", "table"])
def test_what_changed_is_repacked(which):
    """Weights of the torso, of the head, an identity code, both, a table: a frame is bit for bit that of a copy that has packed nothing yet."""
    from helpers import frame_inputs, sequence
    from geneface_amd.radnerf_torso import RADNeRFTorso
    hp, sd = model_fixture(True)
    model = RADNeRFTorso(hp)
    model.load_state_dict(sd, strict=True)
    model = model.to(DEV).eval()
    fi = frame_inputs(sequence(4, 32, 32), 1)
    to = lambda t: t.to(DEV)      # noqa: E731
    args = tuple(to(fi[k]) for k in ("rays_o", "rays_d", "cond", "bg_coords", "pose6"))

    def run(m):
        with torch.no_grad():
            return m.render(*args, index=0, staged=False, bg_color=to(fi["bg"]), perturb=False, force_all_rays=True, render_impl="fused", **hp)["rgb_map"].clone()
    names = {"torso": ["torso_canonicial_net.net.2.weight"], "head": ["sigma_net.net.1.weight"], "code": ["individual_embeddings", "torso_individual_codes"],
             "both": ["torso_deform_net.net.0.weight", "color_net.net.0.weight"], "table": ["position_embedder.embeddings", "torso_embedder.embeddings"]}[which]
    last = run(model)
    for _ in range(2):
        with torch.no_grad():
            for n, p in model.named_parameters():
                if n in names:
                    p.mul_(1.1)
        now = run(model)
        assert torch.equal(now, run(copy.deepcopy(model))) and not torch.equal(now, last)
        last = now
