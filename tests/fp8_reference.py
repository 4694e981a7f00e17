"""The block-scaled 8-bit format and its products from their definition, in 64 bits on the CPU (tests only)."""
import torch


def scale_of(a):
    """Smallest power of two s >= 2^-127 with a <= 448 s; NaN where a is no finite number."""
    a = a.double()
    f, x = torch.frexp(a)                       # a = f 2^x with f in [1/2, 1); 448 = 7/8 * 2^9
    e = torch.where(f <= 0.875, x - 9, x - 8).double()
    e = torch.where(a == 0, torch.full_like(e, -127.0), e).clamp(min=-127)
    return torch.where(torch.isfinite(a), torch.exp2(e), torch.full_like(e, float("nan")))


def to_grid(y):
    """The nearest e4m3 value, ties to even."""
    gap = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / gap) * gap


def by_rows(x):
    """x [R, K] with each 128 values of a row on their grid: what the product multiplies with, in 64 bits."""
    x = x.double().cpu()
    R, K = x.shape
    v = torch.nn.functional.pad(x, (0, -K % 128)).view(R, -1, 128)
    s = scale_of(v.abs().amax(-1, keepdim=True))
    return (to_grid(v / s) * s).view(R, -1)[:, :K]


def by_columns(x):
    return by_rows(x.t()).t()


def by_tiles(w):
    w = w.double().cpu()
    N, K = w.shape
    v = torch.nn.functional.pad(w, (0, -K % 128, 0, -N % 128)).view(-(-N // 128), 128, -(-K // 128), 128)
    s = scale_of(v.abs().amax((1, 3), keepdim=True))
    return (to_grid(v / s) * s).reshape(v.shape[0] * 128, -1)[:N, :K]


def allowed(terms, result, dtype, count):
    """How far a product of `count` terms may be off.  terms: the sum of the magnitudes of what is added up.  32-bit results: each of `count` additions
    rounds at 2^-24 of a partial sum, which is at most `terms`.  16-bit results: half a step of the type (2^-8 or 2^-11 of the value; binary16
    below 2^-14: 2^-25), and the 17 bits that the 8-bit matrix instructions add with, taken as 2^-13 of `terms`."""
    if dtype == torch.float32:
        return count * 2.0 ** -24 * terms + 1e-38
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    return (half + 2.0 ** -20) * result.abs() + 2.0 ** -13 * terms * (1 + half) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
