"""GPU: how 8-bit products are added up -- small products beside large ones, and long sums of one sign, on every path a product can take.

float32 and binary16 results are added up in 32 bits.  bfloat16 results come from the 8-bit matrix instructions, which drop what a product has below
2^-13 of the largest of its eight neighbours': at most 7 x 2^-13 of each eight's largest product (`lost`).  Results are then rounded once, by at
most half a step of their type (2^-8, 2^-11, 2^-24 of the value)."""
import math

import pytest
import torch

import fp8_reference as R
from geneface_amd import fp8

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def lost(a, b, dtype):
    """Upper bound of what the products of a [M, K] with b [N, K] lose, by eights of K: the largest product of an eight is at most the product of the largest."""
    if dtype != torch.bfloat16:
        return torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64)
    most = lambda t: torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).unflatten(1, (-1, 8)).amax(-1)      # noqa: E731
    return 7 * 2.0 ** -13 * (most(a) @ most(b).t())


def outlying(rows, n, dtype, seed):
    """Every eighth value of a row is 1, the others 1.375 x 2^-7: the products of these with their like are 1.89 x 2^-14 of the large ones."""
    v = torch.where(torch.arange(n) % 8 == seed % 8, 1.0, 1.375 * 2.0 ** -7)
    scale = torch.tensor([1.0, 2.0, 0.5])[torch.arange(rows) % 3]
    return (v * scale[:, None]).to(dtype).cuda()


def check(got, a, b, dtype, what):
    """got = a b^T for operands that e4m3 holds exactly."""
    a, b = a.double().cpu(), b.double().cpu()
    want = a @ b.t()
    allowed = HALF[dtype] * want.abs() + lost(a, b, dtype) + a.shape[1] * 2.0 ** -24 * (a.abs() @ b.abs().t())
    assert got.dtype == dtype
    off = (got.double().cpu() - want).abs()
    assert bool((off <= allowed).all()), (what, float((off / want.abs()).max()), float((allowed / want.abs()).max()))


# a few rows; the thin layer; tiles of their own and a split sum; tiles that share a launch; larger tiles
@pytest.mark.parametrize("M, N, K", [(5, 40, 1024), (300, 128, 96), (64, 100, 2048), (300, 140, 160), (40, 30, 600), (2500, 2450, 256), (200, 5000, 384)])
@pytest.mark.parametrize("dtype", TYPES)
def test_small_products_beside_large_ones(dtype, M, N, K):
    x, w = outlying(M, K, dtype, 0), outlying(N, K, torch.float32, 0)
    check(fp8.linear(x, fp8.quantize_weight(w)), x, w, dtype, "kept weight")
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    check(fp8.linear(a, b).detach(), x, w, dtype, "y")


@pytest.mark.parametrize("M, N, K", [(300, 128, 96), (1000, 300, 140), (2048, 140, 300), (3000, 1500, 1400)])
@pytest.mark.parametrize("tw", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_small_products_beside_large_ones_in_the_gradients(dtype, tw, M, N, K):
    """dx adds up over N, dw over M: each operand has the pattern along the axis that is summed over, and one scale along the other."""
    w = outlying(K, N, tw, 0).t().contiguous()
    dy = outlying(M, N, dtype, 0)
    x = torch.ones(M, K, dtype=dtype, device="cuda")
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, = torch.autograd.grad(fp8.linear(a, b), a, dy)
    check(dx, dy, w.t(), dtype, "dx")
    dy, x = outlying(N, M, dtype, 0).t().contiguous(), outlying(K, M, dtype, 0).t().contiguous()
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(fp8.linear(a, b), b, dy)
    check(dw, dy.t(), x.t(), tw, "dw")


def one_sign(rows, n, dtype, seed, scale=1.0):
    """Values of [1/2, 3/2], rows of unlike size so that the results fall anywhere between the steps of their type."""
    g = torch.Generator().manual_seed(seed)
    return (scale * (0.5 + torch.rand(rows, n, generator=g)) * (1 + torch.rand(rows, 1, generator=g))).to(dtype).cuda()


def check_long(got, a, b, dtype, what):
    """a, b: on the 8-bit grid, in 64 bits.  Nothing drifts: the roundings of the results, independent of each other, have a standard deviation of at most
    half / sqrt(3), their mean over n of them one that is sqrt(n) times smaller, and six of those are not met; what the eights lose comes on top, and what 32-bit
    sums round is less than 1e-5 as long as they are rounded either way."""
    want = a @ b.t()
    off = (got.double().cpu() - want) / want
    share = lost(a, b, dtype) / want
    mean, n = float(off.mean()), off.numel()
    assert abs(mean) <= 6 * HALF[dtype] / math.sqrt(3 * n) + float(share.mean()) + 1e-5, (what, mean)
    assert bool((off.abs() <= HALF[dtype] * (1 + 2.0 ** -8) + share + 1e-4).all()), (what, float(off.abs().max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", [(7, 300, 100000), (1024, 1024, 8200), (40, 300, 100000), (2500, 2450, 3000)])
def test_long_sums_of_one_sign(dtype, M, N, K):
    x, w = one_sign(M, K, dtype, 1, 2.0 ** -6), one_sign(N, K, torch.float32, 2)
    q = fp8.quantize_weight(w)
    check_long(fp8.linear(x, q), R.by_rows(x), R.by_tiles(w), dtype, (M, N, K))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", [(100000, 200, 260), (100000, 120, 90), (100000, 2, 128)])
def test_long_weight_gradients_of_one_sign(dtype, M, N, K):
    """The sums over the rows of a training batch, to weights of the activations' type."""
    x, dy = one_sign(K, M, dtype, 3, 2.0 ** -6).t().contiguous().requires_grad_(True), one_sign(N, M, dtype, 4).t().contiguous()
    w = torch.ones(N, K, dtype=dtype, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(fp8.linear(x, w), w, dy)
    check_long(dw, R.by_columns(dy).t(), R.by_columns(x.detach()).t(), dtype, (M, N, K))
