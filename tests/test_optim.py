"""CPU: what the AdamW step and the gradient norm refuse, before anything reaches a device, and the library's side of the same checks."""
import ctypes as C

import pytest
import torch

from geneface_amd import lib as L
from geneface_amd import optim


def _lists(n=5, bits=32, dtype=torch.float32):
    z = lambda dt: torch.zeros(n, dtype=dt)      # noqa: E731
    a = dict(params=[z(dtype)], grads=[z(dtype)], exp_avgs=[z(torch.float32)], exp_avg_sqs=[z(torch.float32)], steps=[torch.zeros(())])
    if bits == 8:
        a["exp_avgs"], a["exp_avg_sqs"] = ([torch.zeros(n, dtype=torch.uint8).view(torch.float8_e4m3fn)] for _ in range(2))
        a["exp_avg_scales"], a["exp_avg_sq_scales"] = ([torch.zeros(-(-n // 128))] for _ in range(2))
    return a


@pytest.mark.parametrize("change, message", [
    (lambda a: a["grads"].append(torch.zeros(5)), "unlike lengths"),
    (lambda a: a.update(grads=[torch.zeros(5, dtype=torch.float16)]), "its parameter's dtype"),
    (lambda a: a.update(params=[torch.zeros(5, dtype=torch.float64)], grads=[torch.zeros(5, dtype=torch.float64)]), "float32, bfloat16 or float16"),
    (lambda a: a.update(grads=[torch.zeros(6)]), "its parameter's size|parameter's size"),
    (lambda a: a.update(exp_avgs=[torch.zeros(5, dtype=torch.float16)]), "moments must be"),
    (lambda a: a.update(exp_avg_sqs=[torch.zeros(4)]), "parameter's size"),
    (lambda a: a.update(steps=[torch.zeros((), dtype=torch.int64)]), "each step"),
    (lambda a: a.update(steps=[torch.zeros(2)]), "each step"),
    (lambda a: a.update(grads=[torch.zeros(5).to_sparse()]), "sparse"),
    (lambda a: a.update(betas=(0.9, 1.0)), "betas"),
    (lambda a: a.update(betas=(-0.1, 0.9)), "betas"),
    (lambda a: a.update(max_norm=1.0), "go together"),
    (lambda a: a.update(grad_norm=torch.zeros(())), "go together"),
    (lambda a: a.update(exp_avg_scales=[torch.zeros(1)]), "must both be given"),
    (lambda a: None, "CUDA"),
])
def test_adamw_step_refuses(change, message):
    a = _lists()
    change(a)
    with pytest.raises((RuntimeError, ValueError), match=message):
        optim.adamw_step(**{"lr": 1e-3, **a})


@pytest.mark.parametrize("change, message", [
    (lambda a: a.update(exp_avgs=[torch.zeros(200)]), "moments must be"),
    (lambda a: a.update(exp_avg_scales=[torch.zeros(1)]), "one value for each 128"),
    (lambda a: a.update(exp_avg_sq_scales=[torch.zeros(2, dtype=torch.float16)]), "one value for each 128"),
    (lambda a: None, "CUDA"),
])
def test_adamw_step_refuses_8_bit_state(change, message):
    a = _lists(200, 8)
    change(a)
    with pytest.raises(RuntimeError, match=message):
        optim.adamw_step(**{"lr": 1e-3, **a})


def test_no_tensors_is_no_work():
    optim.adamw_step([], [], [], [], [], lr=1e-3)


@pytest.mark.parametrize("grads, message", [([], "no gradients"), ([None], "no gradients"), ([torch.zeros(3)], "CUDA"),
                                            ([torch.zeros(3, dtype=torch.int32)], "must be float32"), ([torch.zeros(3).to_sparse()], "sparse")])
def test_grad_norm_refuses(grads, message):
    with pytest.raises(RuntimeError, match=message):
        optim.grad_norm(grads)


@pytest.mark.parametrize("kw", [dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0),
                                dict(max_grad_norm=0.0), dict(lr=float("nan"))])
def test_adamw_refuses_options(kw):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_adamw_refuses_parameters_off_the_gpu():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.AdamW([p]).step()


def test_adamw_without_gradients_does_nothing():
    p = torch.nn.Parameter(torch.ones(3))
    assert optim.AdamW([p]).step() is None and torch.equal(p.detach(), torch.ones(3))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_of_the_other_width_is_refused(bits):
    p = torch.nn.Parameter(torch.zeros(3))
    o = optim.AdamW([p], state_bits=bits)
    s = {"step": torch.tensor(1.0), "exp_avg": torch.zeros(3), "exp_avg_sq": torch.zeros(3)}
    if bits == 32:
        s["exp_avg"] = torch.zeros(3, dtype=torch.uint8).view(torch.float8_e4m3fn)
    d = {"state": {0: s}, "param_groups": o.state_dict()["param_groups"]}
    with pytest.raises(RuntimeError, match=f"{bits}-bit moments"):
        o.load_state_dict(d)


def test_state_of_torch_adam_loads_and_keeps_its_types():
    p = torch.nn.Parameter(torch.zeros(3, 2, dtype=torch.bfloat16))
    o = optim.AdamW([p])
    m, v = torch.randn(3, 2), torch.rand(3, 2)
    o.load_state_dict({"state": {0: {"step": 7, "exp_avg": m, "exp_avg_sq": v}}, "param_groups": o.state_dict()["param_groups"]})
    s = o.state[p]
    assert s["step"].dtype == torch.float32 and float(s["step"]) == 7
    assert torch.equal(s["exp_avg"], m) and torch.equal(s["exp_avg_sq"], v) and s["exp_avg"].data_ptr() != m.data_ptr()
    with pytest.raises(RuntimeError, match="of shape"):
        o.load_state_dict({"state": {0: {"step": 7, "exp_avg": m[:2], "exp_avg_sq": v}}, "param_groups": o.state_dict()["param_groups"]})


@pytest.mark.parametrize("group", [dict(amsgrad=True), dict(maximize=True), dict(weight_decay=0.1, decoupled_weight_decay=False)])
def test_state_of_another_update_is_refused(group):
    p = torch.nn.Parameter(torch.zeros(3))
    o = optim.AdamW([p], lr=0.5)
    d = o.state_dict()
    d["param_groups"][0].update(group, lr=0.25)
    with pytest.raises(RuntimeError, match="another update"):
        o.load_state_dict(d)
    assert o.param_groups[0]["lr"] == 0.5
    d["param_groups"][0].update(dict.fromkeys(group, False), weight_decay=0.0)
    o.load_state_dict(d)
    assert o.param_groups[0]["lr"] == 0.25


def test_a_refused_state_leaves_the_old_one():
    p = torch.nn.Parameter(torch.zeros(3, 2))
    o = optim.AdamW([p])
    held = {"step": 3, "exp_avg": torch.ones(3, 2), "exp_avg_sq": torch.ones(3, 2)}
    o.load_state_dict({"state": {0: held}, "param_groups": o.state_dict()["param_groups"]})
    with pytest.raises(RuntimeError, match="of shape"):
        o.load_state_dict({"state": {0: {**held, "step": 9, "exp_avg_sq": torch.ones(2, 3)}}, "param_groups": o.state_dict()["param_groups"]})
    assert float(o.state[p]["step"]) == 3


def test_the_library_refuses_bad_descriptors(hip_lib):
    def refused(rc, word):
        assert rc == 1 and word in hip_lib.gf_last_error(), hip_lib.gf_last_error()
    refused(hip_lib.gf_adamw_step(None, None), b"null")
    refused(hip_lib.gf_grad_norm(None, None), b"null")
    table = (C.c_uint64 * 8)(*([16] * 6 + [16, 5]))
    d = lambda **k: optim.GfAdamw(**{"tensors_host": C.addressof(table), "count": 1, "state_bits": 32, "beta1": 0.9, "beta2": 0.99, **k})      # noqa: E731
    assert hip_lib.gf_adamw_step(C.byref(d(count=0)), None) == 0
    refused(hip_lib.gf_adamw_step(C.byref(d(tensors_host=None)), None), b"null")
    refused(hip_lib.gf_adamw_step(C.byref(d(dtype=3)), None), b"dtype")
    refused(hip_lib.gf_adamw_step(C.byref(d(state_bits=4)), None), b"state_bits")
    refused(hip_lib.gf_adamw_step(C.byref(d(beta2=1.0)), None), b"betas")
    for k in (0, 1, 2, 3, 6):
        table[k] = 0
        refused(hip_lib.gf_adamw_step(C.byref(d()), None), b"null pointer in tensor 0")
        table[k] = 16
    table[4] = 0
    refused(hip_lib.gf_adamw_step(C.byref(d(state_bits=8)), None), b"null pointer in tensor 0")
    table[7] = 1 << 41
    refused(hip_lib.gf_adamw_step(C.byref(d()), None), b"too many")
    g = (C.c_uint64 * 3)(0, 5, 0)
    n = lambda **k: optim.GfGradNorm(**{"tensors_host": C.addressof(g), "count": 1, "norm_out": 16, "workspace": 16, **k})      # noqa: E731
    refused(hip_lib.gf_grad_norm(C.byref(n()), None), b"null pointer in tensor 0")
    refused(hip_lib.gf_grad_norm(C.byref(n(workspace=None)), None), b"null")
    g[0], g[2] = 16, 7
    refused(hip_lib.gf_grad_norm(C.byref(n()), None), b"dtype")
    assert hip_lib.gf_grad_norm_workspace_bytes(10) >= 8 * 10


def test_the_library_exports_the_training_header(hip_lib):
    raw = C.CDLL(L.LIB_PATH)
    names = [n for _, n, _ in L.header_prototypes(L.TRAIN_HEADER_PATH)]
    assert {"gf_adamw_step", "gf_grad_norm"} <= set(names) and len(names) == len(set(names))
    assert not set(names) & {n for _, n, _ in L.header_prototypes()}
    for name in names:
        assert hasattr(raw, name), name


def test_device_code_of_the_training_operators(hip_lib):
    """The properties that the other translation units are held to: no packed-FP32 instruction, no scratch, no spilled register."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "tools"))
    import kernel_resources as KR
    from geneface_amd.csrc import build
    if not KR.available():
        pytest.skip("ROCm LLVM binutils not present")
    census = KR.report(os.path.join(build.OBJ_DIR, "train"))
    assert set(census) == {os.path.basename(p) for p in build.train_sources() if p.endswith(".hip")}
    for tu, d in census.items():
        c = d["instructions"]
        assert not any(c[k] for k in ("v_pk_fma_f32", "v_pk_mul_f32", "v_pk_add_f32", "scratch_")), (tu, c)
        for k in d["kernels"]:
            assert k.get("private_segment_fixed_size", 0) == 0 and k.get("vgpr_spill_count", 0) == 0 and k.get("vgpr_count", 0) <= 512, (tu, k)
