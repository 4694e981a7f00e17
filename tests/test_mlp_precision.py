"""MLP.precision on a whole model: never ignored (host half; the device half is test_gpu_mlp_precision.py)."""
import pytest

from geneface_amd import fused
from geneface_amd import hparams as HP
from geneface_amd.radnerf import RADNeRF
from geneface_amd.radnerf_torso import RADNeRFTorso


@pytest.mark.parametrize("torso", [False, True])
def test_a_model_with_8_bit_layers_takes_the_op_by_op_path(torso):
    hp = HP.may_hparams(torso)
    model = (RADNeRFTorso if torso else RADNeRF)(hp)
    assert model._pick_impl("auto", False, 16) == "fused"
    nets = [model.ambient_net, model.sigma_net, model.color_net] + ([model.torso_deform_net, model.torso_canonicial_net] if torso else [])
    for net in nets:
        net.precision = "fp8"
        assert model._pick_impl("auto", False, 16) == "ops"
        with pytest.raises(NotImplementedError, match="precision"):
            fused.get_state(model)
        net.precision = "native"
        assert model._pick_impl("auto", False, 16) == "fused"
