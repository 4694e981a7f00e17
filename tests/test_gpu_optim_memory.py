"""GPU: an AdamW step reads nothing that it writes, except a gradient that is its own parameter."""
import pytest
import torch

from geneface_amd import optim

pytestmark = pytest.mark.gpu


def _params():
    flat = torch.randn(9000, generator=torch.Generator().manual_seed(1)).cuda()
    return flat, [flat[:3000], flat[3000:5000], flat[6000:9000]]


@pytest.mark.parametrize("case", ["another parameter", "part of another", "its own, moved", "over the end", "a moment", "a step count"])
def test_gradients_in_memory_that_is_written_are_refused(case):
    flat, ps = _params()
    gs = [torch.ones_like(p) for p in ps]
    ms = [torch.zeros_like(p) for p in ps]
    steps = [torch.zeros((), device="cuda") for _ in ps]
    bad = {"another parameter": (0, ps[2]), "part of another": (1, flat[500:2500]), "its own, moved": (2, flat[5999:8999]), "over the end": (0, flat[4990:7990]),
           "a moment": (1, ms[0][:2000]), "a step count": (0, None)}[case]
    if case == "a step count":
        block = torch.zeros(3000, device="cuda")
        steps[1], gs[0] = block[2999], block
    else:
        gs[bad[0]] = bad[1]
    before = [t.clone() for t in (flat, *ms, *steps)]
    with pytest.raises(RuntimeError, match="shares memory"):
        optim.adamw_step(ps, gs, ms, [torch.zeros_like(p) for p in ps], steps, lr=1e-2)
    assert all(torch.equal(a, b) for a, b in zip(before, (flat, *ms, *steps)))


@pytest.mark.parametrize("name", ["lr", "grad_scale", "found_inf", "grad_norm"])
def test_scalars_in_memory_that_is_written_are_refused(name):
    flat, ps = _params()
    steps = [torch.zeros((), device="cuda") for _ in ps]
    for where in (steps[1], flat[4000]):
        kw = {"lr": 1e-2, name: where, **({"max_norm": 1.0} if name == "grad_norm" else {})}
        with pytest.raises(RuntimeError, match="shares memory"):
            optim.adamw_step(ps, [torch.ones_like(p) for p in ps], [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps], steps, **kw)


def test_memory_beside_what_is_written_is_taken():
    """Gradients and scalars directly before and behind a parameter, a gradient of strides of its own inside another parameter (it is copied first), and a
    gradient that is its parameter."""
    flat, ps = _params()
    gs = [torch.ones_like(ps[0]), ps[1], torch.full_like(ps[2], 0.5)]
    beside = [flat[5000:5999], flat[5999]]
    params = [*ps, torch.zeros(999, device="cuda"), torch.zeros(1000, device="cuda")]
    grads = [*gs, beside[0], flat[:2000:2]]
    with torch.no_grad():
        beside[1].fill_(1e-2)
    twin = [p.clone() for p in params]
    twin_grads = [g.clone() for g in grads]
    state = lambda: [[torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params], [torch.zeros((), device="cuda") for _ in params]]      # noqa: E731
    a, b = state(), state()
    optim.adamw_step(params, grads, *a, lr=beside[1])
    optim.adamw_step(twin, twin_grads, *b, lr=beside[1].clone())
    assert all(torch.equal(x, y) for x, y in zip(params, twin)) and all(torch.equal(x, y) for u, v in zip(a, b) for x, y in zip(u, v))
