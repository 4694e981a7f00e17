"""GPU: AdamW with 8-bit moments on gradients whose squares leave float32's range, against the formulas in 64 bits.

A step is compared with the formula on the state that the step before left.  Codes are rounded down or up, by less than one spacing; scales and roots are
some ten 32-bit roundings off at most, the parameter twenty of its own size and of the update's, then half a step of its type."""
import pytest
import torch

from geneface_amd import optim

pytestmark = pytest.mark.gpu
BETA1, BETA2, LR, EPS, DECAY = 0.9, 0.99, 1e-2, 1e-8, 0.1
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _held(s):
    wide = lambda k: s[k].float().double().cpu() * s[k + "_scale"].double().cpu().repeat_interleave(128)[:s[k].numel()]      # noqa: E731
    return wide("exp_avg"), wide("exp_avg_sq")


def _close(state, key, want):
    n = want.numel()
    most = torch.nn.functional.pad(want.abs(), (0, -n % 128)).view(-1, 128).amax(1).clamp(min=2.0 ** -100)
    scale = state[key + "_scale"].double().cpu()
    assert bool(((scale * 448 / most - 1).abs() <= 16 * 2.0 ** -24).all()), (key, scale * 448, most)
    each = (most / 448).repeat_interleave(128)[:n]
    y = (want / each).abs()
    gap = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    got = state[key].float().double().cpu() * scale.repeat_interleave(128)[:n]
    assert bool(((got - want).abs() <= gap * each * (1 + 2.0 ** -3)).all()), key      # (a value that rounds up to the next power of two: its spacing is twice that)
    assert bool((got[want != 0] != 0).all()) or key == "exp_avg"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where, value", [([0], 1e25), ([130, 131, 190], -3e30), ([299], 3e19), ([5, 140], 1e38)])
def test_a_gradient_whose_square_overflows(dtype, where, value):
    g = torch.Generator().manual_seed(1)
    n = 300
    p = torch.nn.Parameter((0.3 * torch.randn(n, generator=g)).to(dtype).cuda())
    opt = optim.AdamW([p], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=8)
    # binary16 holds no such gradient: it comes by the factor that the gradients carry
    carried = 1e-34 if dtype == torch.float16 else 1.0
    opt.grad_scale = torch.tensor(carried, dtype=torch.float32, device="cuda")
    carried = float(opt.grad_scale)
    for step in range(5):
        grad = torch.randn(n, generator=g).double()
        grad[7], grad[200] = 0.0, 0.0
        if step in (1, 3):
            grad[where] = value
        p.grad = (grad * carried if dtype != torch.float16 else (grad * carried).clamp(-6e4, 6e4)).to(dtype).cuda()
        grad = p.grad.double().cpu() / carried
        old = p.detach().double().cpu()
        m, r = _held(opt.state[p]) if step else (torch.zeros(n).double(), torch.zeros(n).double())
        opt.step()
        t = step + 1
        m = m + (1 - BETA1) * (grad - m)
        r = (BETA2 * r ** 2 + (1 - BETA2) * grad ** 2).sqrt()
        _close(opt.state[p], "exp_avg", m)
        _close(opt.state[p], "exp_avg_sq", r)
        move = LR / (1 - BETA1 ** t) * m / (r / (1 - BETA2 ** t) ** 0.5 + EPS)
        want = old * (1 - LR * DECAY) - move
        allowed = 20 * 2.0 ** -24 * (old.abs() + move.abs()) + HALF[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        off = (p.detach().double().cpu() - want).abs()
        assert bool((off <= allowed).all()), (step, off.argmax().item(), float((off - allowed).max()))
    assert all(bool(torch.isfinite(v).all()) for v in _held(opt.state[p]))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_gradient_that_is_no_number_still_leaves_none_in_its_block(bad):
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = optim.AdamW([p], state_bits=8)
    for step in range(2):
        p.grad = torch.ones(300, device="cuda")
        if step == 0:
            p.grad[140], p.grad[141] = bad, 1e30
        opt.step()
        for v in _held(opt.state[p]):
            finite = torch.isfinite(v)
            assert not bool(finite[128:256].any()) and bool(finite[:128].all()) and bool(finite[256:].all())
