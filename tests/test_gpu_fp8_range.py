"""GPU: 8-bit products of values at the lower end of float32, against the definition in 64 bits."""
import pytest
import torch

import fp8_reference as R
from geneface_amd import fp8

pytestmark = pytest.mark.gpu


def _run(x, w, dy):
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = fp8.linear(a, b)
    return (y.detach(), *torch.autograd.grad(y, (a, b), dy))


@pytest.mark.parametrize("M, N, K", [(5, 40, 300), (300, 128, 96), (300, 140, 160), (30, 90, 12000)])
@pytest.mark.parametrize("power", [-100, -110, -116, -118, -122, -130, -140])
def test_values_next_to_the_smallest(power, M, N, K):
    """float32 operands of 2^power beside ordinary ones.  A code's value below bfloat16's subnormal spacing of 2^-133 is rounded to it when the code is widened,
    by 2^-134 at most: the sum is off by that times the other operand's magnitudes, and by the roundings of its additions."""
    g = torch.Generator().manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
    near = lambda got, a, b: bool(((got.double().cpu() - a @ b.t()).abs() <= a.shape[1] * (2.0 ** -24 * (a.abs() @ b.abs().t()) + 2.0 ** -149)      # noqa: E731
                                   + 2.0 ** -134 * b.abs().sum(1)).all())
    x, w, dy = r(M, K), r(N, K), r(M, N) * 2.0 ** power
    small = x * 2.0 ** power
    q = fp8.quantize_weight(w.cuda())
    assert near(fp8.linear(small.cuda(), q), R.by_rows(small), R.by_tiles(w)) and near(fp8.linear(small.cuda(), w.cuda()), R.by_rows(small), R.by_tiles(w))
    _, dx, dw = _run(x.cuda(), w.cuda(), dy.cuda())
    assert near(dx, R.by_rows(dy), R.by_tiles(w).t()) and near(dw, R.by_columns(dy).t(), R.by_columns(x).t())
