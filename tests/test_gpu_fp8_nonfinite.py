"""GPU: what infinities and NaN do to 8-bit products and their gradients, on every path.

A block that holds an infinity or a NaN is NaN as a whole.  So of a product a row (column) is NaN exactly where its operand's row (the other's row)
holds a block that is none, and everything else is what it would be without it."""
import math

import pytest
import torch

from geneface_amd import fp8, optim
from geneface_amd.cond_encoder import MLP

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# the thin layer, over several tiles and over more tiles than workgroups; operands that share a launch; splits; a weight gradient that is split; larger tiles
SHAPES = [(300, 128, 96), (3, 2, 5), (110000, 128, 128), (300, 140, 150), (30, 90, 12000), (5000, 140, 300), (2000, 600, 700)]


def _inputs(M, N, K, dtype):
    g = torch.Generator().manual_seed(M + N + K)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    return r(M, K).to(dtype).cuda(), (r(N, K) / math.sqrt(K)).cuda(), r(M, N).to(dtype).cuda()


def _run(x, w, dy):
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = fp8.linear(a, b)
    return (y.detach(), *torch.autograd.grad(y, (a, b), dy))


def _only(got, clean, rows, cols, what):
    """NaN exactly in `rows` and `cols`, elsewhere as without."""
    none = torch.zeros(tuple(got.shape), dtype=torch.bool, device="cuda")
    none[rows] = True
    none[:, cols] = True
    assert torch.equal(torch.isnan(got), none), what
    assert torch.equal(got[~none], clean[~none]), what


def _block(at, size):
    return slice(at // 128 * 128, min(size, at // 128 * 128 + 128))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_what_is_no_number_reaches_every_result_of_its_blocks(M, N, K, dtype, bad):
    x, w, dy = _inputs(M, N, K, dtype)
    clean = _run(x, w, dy)
    nothing = slice(0, 0)
    m, n, k = M * 2 // 3, N // 2, K * 2 // 3
    broken = x.clone()
    broken[m, k] = bad
    y, dx, dw = _run(broken, w, dy)
    _only(y, clean[0], m, nothing, "y of x")
    assert torch.equal(dx, clean[1])
    _only(dw, clean[2], nothing, k, "dw of x")
    broken = dy.clone()
    broken[m, n] = bad
    y, dx, dw = _run(x, w, broken)
    assert torch.equal(y, clean[0])
    _only(dx, clean[1], m, nothing, "dx of dy")
    _only(dw, clean[2], n, nothing, "dw of dy")
    broken = w.clone()
    broken[n, k] = bad
    y, dx, dw = _run(x, broken, dy)
    _only(y, clean[0], nothing, _block(n, N), "y of w")
    _only(dx, clean[1], nothing, _block(k, K), "dx of w")
    assert torch.equal(dw, clean[2])
    y = fp8.linear(x, fp8.quantize_weight(broken))
    _only(y, fp8.linear(x, fp8.quantize_weight(w)), nothing, _block(n, N), "y of a kept w")


@pytest.mark.parametrize("dtype", TYPES)
def test_a_few_rows_with_what_is_no_number(dtype):
    x, w, _ = _inputs(11, 300, 2050, dtype)
    q = fp8.quantize_weight(w)
    clean = fp8.linear(x, q)
    for bad in (math.inf, math.nan):
        broken = x.clone()
        broken[7, 1500] = bad
        _only(fp8.linear(broken, q), clean, 7, slice(0, 0), bad)


@pytest.mark.parametrize("bits", [8, 32])
def test_an_overflow_makes_the_gradient_scaler_skip_the_step(bits):
    torch.manual_seed(1)
    net = MLP(96, 3, 128, 3).cuda()
    net.precision = "fp8"
    opt = optim.AdamW(net.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 126, growth_interval=1000)
    x = torch.randn(1000, 96, device="cuda")
    skipped = 0
    for _ in range(100):
        before, scale = [p.detach().clone() for p in net.parameters()], scaler.get_scale()
        opt.zero_grad()
        scaler.scale(net(x).square().mean() * 1e4).backward()
        scaler.step(opt)
        scaler.update()
        same = all(torch.equal(a, b.detach()) for a, b in zip(before, net.parameters()))
        assert same == (scaler.get_scale() < scale) and all(bool(torch.isfinite(p).all()) for p in net.parameters())
        skipped += same
        if not same:
            break
    assert skipped >= 1 and not same
